// Routing: the top-k experts of every row of router logits and their weights, as moe_forward takes them.
//
//   score   softmax(l) or 1 / (1 + exp(-l))
//   key     l itself without a bias (both scores rise with l, so their order is the logits' own, exactly), and
//           score + bias in 64 bits with one: two keys of a row are often closer than 32 bits tell apart (256 experts,
//           1,024 rows: a few rows per call would differ from the order in 64 bits)
//   groups  E / n_group neighbouring experts each; a group's value is its largest key, with a bias the sum of its two
//           largest; only the experts of the topk_group best groups compete
//   picks   keys descending, equal keys by index; NaN counts as the largest
//   weight  the pick's score (renormalised: over the picks' sum, the softmax taken over the picks' own logits, and sigmoids that
//           are all small relative to the largest pick's, so that nothing underflows), times scale; a sum of 0 (every pick at
//           -inf, or a sigmoid of less than -700) gives weights of 0
//
// One wave per row; the instructions of 8 waves per SIMD bound 8,192 rows (logits arrive at 1.9 TB/s), the chain of the picks
// one row. us per call out of a graph, medians, for 1 / 200 / 8,192 rows of fp32: 512 experts, top 10: 3.3 / 3.8 / 8.9, with a bias
// 5.0 / 5.6 / 17.0; 256 in 8 groups of which 4 compete, top 8, sigmoid: 3.4 / 3.8 / 7.3, with a bias 4.7 / 5.2 / 12.4; 128, top 8:
// 2.8 / 3.1 / 5.2, with a bias and sigmoid 3.6 / 4.1 / 8.0. (8,192 rows took 7.7 to 8.9 and with a bias 15.4 to 17.0 on the cards
// measured.)
//
// Lane i holds the E / 64 neighbouring experts from i * NPL, so the lowest lane of a tie holds the
// lowest index; it sorts their keys (a network of max and min, without the indices). A pick is then one maximum over the
// lanes' first keys (six DPP steps), the first lane that has it, and that lane's keys move up. What the picks were is found
// at the end, all at once: lane r looks up the place of pick r's key among the keys of the lane that it came from. Nothing is
// kept between calls and no row depends on another.
#include "exl3_common.cuh"
#include "exl3_kernels.h"

#include <type_traits>

namespace exl3 {
namespace {

constexpr int kRouteWaves = 4;

// Keys in the order of their values: the larger value has the larger key, -0 that of +0, NaN one above all others, and
// kNone (no expert, or one that was picked) is below all. 32 bits: the logit's bits, turned; 64 bits: the value itself, with
// places of their own for what has none among the finite ones (score + bias is below 1e39).
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f), k = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
    return v != v ? 0xFFFFFFFFu : k;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __builtin_bit_cast(float, (k & 0x80000000u) ? (k == 0xFFFFFFFFu ? 0x7FC00000u : k & 0x7FFFFFFFu) : ~k);
}
constexpr double kInf = 1e300, kNan = 2e300;
__device__ __forceinline__ double key_of(double v) {      // (no -0: a score is never one, and a sum of others is +0)
    const double k = __builtin_fmin(__builtin_fmax(v, -kInf), kInf);
    return v != v ? kNan : k;
}
__device__ __forceinline__ double value_of(double k) {
    return k == kNan ? __builtin_nan("") : k == kInf ? INFINITY : k == -kInf ? -INFINITY : k;
}
template <class Key> constexpr Key kNone = std::is_same_v<Key, double> ? (Key)-INFINITY : (Key)0;

__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
__device__ __forceinline__ uint32_t smaller(uint32_t a, uint32_t b) { return min(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return __builtin_fmin(a, b); }

// v of the lane that CTRL names, `none` where there is no such lane
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v, uint32_t none) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, 0xF, 0xF, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v, float none) {
    return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, none)));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v, double none) {
    const uint64_t a = __builtin_bit_cast(uint64_t, v), b = __builtin_bit_cast(uint64_t, none);
    return __builtin_bit_cast(double, (uint64_t)dpp<CTRL>((uint32_t)(a >> 32), (uint32_t)(b >> 32)) << 32 |
                                          dpp<CTRL>((uint32_t)a, (uint32_t)b));
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ float lane_value(float v, int l) {
    return __builtin_bit_cast(float, lane_value(__builtin_bit_cast(uint32_t, v), l));
}
__device__ __forceinline__ double lane_value(double v, int l) {
    const uint64_t a = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)lane_value((uint32_t)(a >> 32), l) << 32 | lane_value((uint32_t)a, l));
}
// f over the wave's values: row_shr 1, 2, 4, 8 (lane 15 of each row of 16 has the row's), row_bcast 15 and 31 (lane 63)
template <class T, class F>
__device__ __forceinline__ T over_wave(T v, T none, F f) {
    v = f(v, dpp<0x111>(v, none));
    v = f(v, dpp<0x112>(v, none));
    v = f(v, dpp<0x114>(v, none));
    v = f(v, dpp<0x118>(v, none));
    v = f(v, dpp<0x142>(v, none));
    v = f(v, dpp<0x143>(v, none));
    return lane_value(v, 63);
}
template <class Key>
__device__ __forceinline__ Key wave_max(Key v) {
    return over_wave(v, kNone<Key>, [](Key a, Key b) { return larger(a, b); });
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
    return over_wave(v, (T)0, [](T a, T b) { return a + b; });
}

template <class Key, int N>
__device__ __forceinline__ void sort_descending(Key (&k)[N]) {
    // odd-even merge sort of N = 2^i keys
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int q = p; q > 0; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const Key a = k[i + j], b = k[i + j + q];
                        k[i + j] = larger(a, b);
                        k[i + j + q] = smaller(a, b);
                    }
}

template <int DT>
__device__ __forceinline__ float logit_at(const void* p, size_t i) {
    if constexpr (DT == 0) return (float)((const _Float16*)p)[i];
    else if constexpr (DT == 1) return __builtin_bit_cast(float, (uint32_t)((const uint16_t*)p)[i] << 16);
    else return ((const float*)p)[i];
}

// a lane's logits in loads of up to 16 bytes (its share starts on its own size, up to 16 bytes, and is all there)
template <int DT, int NPL>
__device__ __forceinline__ void logits_wide(const void* p, size_t at, float (&v)[NPL]) {
    constexpr int kSize = DT == 2 ? 4 : 2, kBytes = NPL * kSize, kEach = kBytes < 16 ? kBytes : 16;
    struct alignas(kEach) Piece {
        uint8_t b[kEach];
    };
    union {
        Piece piece[kBytes / kEach];
        std::conditional_t<DT == 2, float, uint16_t> x[NPL];
    } u;
#pragma unroll
    for (int i = 0; i < kBytes / kEach; ++i) u.piece[i] = ((const Piece*)((const uint8_t*)p + at * kSize))[i];
#pragma unroll
    for (int j = 0; j < NPL; ++j) v[j] = logit_at<DT>(u.x, j);
}

// 1 / (1 + e^-l), 0 below kLeastLogit: the hardware's reciprocal (2^-23) and two steps of Newton's
constexpr float kLeastLogit = -700.0f;
__device__ __forceinline__ double sigmoid64(float l) {
    const bool low = l < kLeastLogit;
    const double d = 1.0 + exp(low ? 700.0 : -(double)l);
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
    r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
    return low ? 0.0 : r;
}

// the softmax is taken relative to the row's largest logit (to 0 where that is -inf, so that exp gives 0)
template <class T>
__device__ __forceinline__ T top_or_0(T top) { return top == -(T)INFINITY ? (T)0 : top; }

template <int NPL, bool BIAS, int DT>
__global__ void __launch_bounds__(64 * kRouteWaves) route_kernel(RouteArgs A, int wide) {
    using Key = std::conditional_t<BIAS, double, uint32_t>;
    using Val = std::conditional_t<BIAS, double, float>;
    __shared__ Key lkeys[kRouteWaves][64 * NPL];
    const int l = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x * kRouteWaves + wv;
    if (row >= A.M) return;
    const size_t base = (size_t)row * A.stride;
    const int e0 = l * NPL;
    Key* lk = lkeys[wv];

    float lg[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) lg[j] = -INFINITY;
    if (wide & 1) {
        if (e0 < A.E) logits_wide<DT>(A.logits, base + e0, lg);
    } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const float v = logit_at<DT>(A.logits, base + min(e0 + j, A.E - 1));
            lg[j] = e0 + j < A.E ? v : -INFINITY;
        }
    }
    [[maybe_unused]] float bias[NPL];
    if constexpr (BIAS) {                            // (all of it before the first score is needed)
#pragma unroll
        for (int j = 0; j < NPL; ++j) bias[j] = -INFINITY;
        if (wide & 2) {
            if (e0 < A.E) logits_wide<2>(A.bias, e0, bias);
        } else {
#pragma unroll
            for (int j = 0; j < NPL; ++j) {
                const float v = A.bias[min(e0 + j, A.E - 1)];
                bias[j] = e0 + j < A.E ? v : -INFINITY;
            }
        }
    }
    // the row's softmax where the keys or the weights need it
    Val top = 0, total = 1, e[NPL];
    if (!A.sigmoid && (BIAS || !A.renormalize)) {
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) most = max(most, key_of(lg[j]));
        top = top_or_0((Val)value_of(wave_max(most)));
        total = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            if constexpr (BIAS) e[j] = exp((double)lg[j] - top);
            else e[j] = expf(lg[j] - top);
            total += e[j];
        }
        total = wave_sum(total);
        if (total == 0) total = 1;
    }
    if constexpr (BIAS) {                            // (now the scores)
        if (A.sigmoid) {
#pragma unroll
            for (int j = 0; j < NPL; ++j) e[j] = sigmoid64(lg[j]);
        } else {
            const double each = 1.0 / total;
#pragma unroll
            for (int j = 0; j < NPL; ++j) e[j] *= each;
        }
    }
    // (places behind the last expert have the key of -inf, or, as every expert of a row with a NaN, of NaN: with no expert's are
    // theirs smaller, but where keys are equal the experts come first, and there are topk of them)
    Key key[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        if constexpr (BIAS) key[j] = key_of(e[j] + (double)bias[j]);
        else key[j] = key_of(lg[j]);
        lk[e0 + j] = key[j];
    }
    auto lds_ready = [] {                            // (a wave's own part of LDS)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    lds_ready();

    bool sorted = false;
    if (A.n_group > 1) {
        // The lanes P g .. P g + P - 1 find group g's two largest keys. Where the lanes' own shares make up whole groups, the
        // power of two of them that does; else (aligned false) the power of two up to 64 / G, by way of LDS
        const int G = A.n_group, gs = A.E / G, share = gs / NPL;
        const bool aligned = gs % NPL == 0 && (share & (share - 1)) == 0;
        const int P = aligned ? share : 1 << (31 - __builtin_clz(64 / G)), g = l / P;
        Key t1 = kNone<Key>, t2 = kNone<Key>;
        if (aligned) {
            sort_descending(key);
            t1 = key[0];
            if constexpr (NPL > 1) t2 = key[1];
        } else if (g < G) {
            for (int i = l & (P - 1); i < gs; i += P) {
                const Key k = lk[g * gs + i];
                t2 = larger(t2, smaller(t1, k));
                t1 = larger(t1, k);
            }
        }
        auto join = [&](Key o1, Key o2) {
            t2 = larger(smaller(t1, o1), larger(t2, o2));
            t1 = larger(t1, o1);
        };
        // the neighbour, the other pair of four, the other four of eight, the other eight of sixteen (a mirror reaches them:
        // they all have the same two by then)
        if (P > 1) join(dpp<0xB1>(t1, t1), dpp<0xB1>(t2, t2));
        if (P > 2) join(dpp<0x4E>(t1, t1), dpp<0x4E>(t2, t2));
        if (P > 4) join(dpp<0x141>(t1, t1), dpp<0x141>(t2, t2));
        if (P > 8) join(dpp<0x140>(t1, t1), dpp<0x140>(t2, t2));
        for (int d = 16; d < P; d *= 2) join(__shfl_xor(t1, d), __shfl_xor(t2, d));
        Key value = t1;
        if constexpr (BIAS) {
            const Key sum = key_of(value_of(t1) + value_of(t2));
            value = gs > 1 ? sum : t1;
        }
        int rank = 0;
        for (int h = 0; h < G; ++h) {
            const Key o = lane_value(value, h * P);
            rank += o > value || (o == value && h < g);
        }
        const bool keeps = g < G && rank < A.topk_group;
        if (aligned) {
            // (a lane's keys are all of its own group)
#pragma unroll
            for (int j = 0; j < NPL; ++j) key[j] = keeps ? key[j] : kNone<Key>;
            sorted = true;
        } else {
            const uint64_t kept = __ballot(keeps);              // (bit P i: group i)
            const uint32_t magic = ((1u << 20) + gs - 1) / gs;  // e / gs for e < 1024 (e * gs < 2^20)
#pragma unroll
            for (int j = 0; j < NPL; ++j) {
                const int of = (int)((uint32_t)(e0 + j) * magic >> 20);
                const bool out = of >= G || !(kept >> (of * P) & 1);
                if (out) lk[e0 + j] = kNone<Key>;
                key[j] = out ? kNone<Key> : key[j];
            }
            lds_ready();
        }
    }

    // the picks: lane r keeps pick r's key, the lane it came from, and how many picks before it took that key from that lane
    if (!sorted) sort_descending(key);
    Key picked = kNone<Key>, last = kNone<Key>;
    int source = 0, last_from = -1, n = 0;
    for (int r = 0; r < A.topk; ++r) {
        Key most;
        uint64_t have;
        if constexpr (BIAS) {
            // the upper halves first, as whole numbers in the values' order: most often only one lane has the largest
            const int hi = (int)(__builtin_bit_cast(uint64_t, key[0]) >> 32);
            const uint32_t h = (uint32_t)hi ^ ((uint32_t)(hi >> 31) | 0x80000000u), top_h = wave_max(h);
            have = __ballot(h == top_h);
            if (have & (have - 1)) {
                most = wave_max(h == top_h ? key[0] : kNone<Key>);
                have = __ballot(key[0] == most);
            } else {
                most = lane_value(key[0], __builtin_ctzll(have));
            }
        } else {
            most = wave_max(key[0]);
            have = __ballot(key[0] == most);
        }
        const int win = __builtin_ctzll(have);
        n = win == last_from && most == last ? n + 1 : 0;
        last = most;
        last_from = win;
        const bool here = l == r;
        picked = here ? most : picked;
        source = here ? n << 8 | win : source;
        if constexpr (BIAS && NPL > 1) {
            if (l == win) {
                asm volatile("");                    // (a branch: 64 bits move at once, and are chosen by halves)
#pragma unroll
                for (int j = 0; j < NPL; ++j) key[j] = j + 1 < NPL ? key[j + 1] : kNone<Key>;
            }
        } else {
            const bool mine = l == win;
#pragma unroll
            for (int j = 0; j < NPL; ++j) {
                const Key here = key[j], next = j + 1 < NPL ? key[j + 1] : kNone<Key>;
                key[j] = mine ? next : here;
            }
        }
    }
    const bool live = l < A.topk;
    const int from = source & 255;
    int nth = source >> 8, id = from * NPL;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {                  // the place of the nth (from 0) key of this value
        const bool same = lk[from * NPL + j] == picked;
        if (same && nth == 0) id = from * NPL + j;
        nth -= same;
    }

    float x, w;
    if constexpr (BIAS) x = live ? logit_at<DT>(A.logits, base + id) : -INFINITY;
    else x = live ? value_of(picked) : -INFINITY;
    if (A.sigmoid) w = 1.0f / (1.0f + expf(-x));
    else if (A.renormalize) w = expf(x - top_or_0(BIAS ? value_of(wave_max(live ? key_of(x) : 0u)) : lane_value(x, 0)));
    else w = (float)((BIAS ? exp((double)x - top) : (Val)expf(x - (float)top)) / total);
    if (!live) w = 0;
    if (A.renormalize) {
        float sum = wave_sum(w);
        if (A.sigmoid && sum < 0x1p-24f) {           // every pick's score is exp(x) to 2^-24, and may be below fp32's smallest
            const float most = BIAS ? value_of(wave_max(live ? key_of(x) : 0u)) : lane_value(x, 0);
            w = x < kLeastLogit ? 0.0f : expf(x - most);
            sum = wave_sum(w);
        }
        w /= sum == 0 ? 1.0f : sum;
    }
    if (live) {
        A.ids[(size_t)row * A.topk + l] = id;
        A.w[(size_t)row * A.topk + l] = w * A.scale;
    }
}

template <int NPL, bool BIAS>
void route_dt(const RouteArgs& a, int dtype, hipStream_t s) {
    const dim3 grid((unsigned)((a.M + (int64_t)kRouteWaves - 1) / kRouteWaves)), block(64 * kRouteWaves);
    const int esz = dtype == 2 ? 4 : 2, each = NPL * esz < 16 ? NPL * esz : 16;
    // (a lane's logits, and its biases, in wide loads)
    constexpr int kBiasEach = NPL * 4 < 16 ? NPL * 4 : 16;
    const int wide = (a.E % NPL == 0 && (uintptr_t)a.logits % each == 0 && a.stride * esz % each == 0) |
                     (BIAS && a.E % NPL == 0 && (uintptr_t)a.bias % kBiasEach == 0) << 1;
    if (dtype == 0) hipLaunchKernelGGL((route_kernel<NPL, BIAS, 0>), grid, block, 0, s, a, wide);
    else if (dtype == 1) hipLaunchKernelGGL((route_kernel<NPL, BIAS, 1>), grid, block, 0, s, a, wide);
    else hipLaunchKernelGGL((route_kernel<NPL, BIAS, 2>), grid, block, 0, s, a, wide);
}

template <int NPL>
void route_npl(const RouteArgs& a, int dtype, hipStream_t s) {
    if (a.bias) route_dt<NPL, true>(a, dtype, s);
    else route_dt<NPL, false>(a, dtype, s);
}

}  // namespace

hipError_t launch_route(const RouteArgs& a, int dtype, hipStream_t s) {
    if (a.E <= 64) route_npl<1>(a, dtype, s);
    else if (a.E <= 128) route_npl<2>(a, dtype, s);
    else if (a.E <= 256) route_npl<4>(a, dtype, s);
    else if (a.E <= 512) route_npl<8>(a, dtype, s);
    else route_npl<16>(a, dtype, s);
    return hipGetLastError();
}

}  // namespace exl3
