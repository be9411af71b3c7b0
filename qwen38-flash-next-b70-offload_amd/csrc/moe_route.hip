// Routing: the top-k experts of every row of router logits and their weights, as moe_forward takes them.
//
//   score   softmax(l) or 1 / (1 + exp(-l))
//   key     l itself without a bias (both scores rise with l, so their order is the logits' own, exactly), and
//           score + bias in 64 bits with one: two keys of a row are often closer than 32 bits tell apart (256 experts,
//           1,024 rows: a few rows per call would differ from the order in 64 bits)
//   groups  E / n_group neighbouring experts each; a group's value is its largest key, with a bias the sum of its two
//           largest; only the experts of the topk_group best groups compete
//   picks   keys descending, equal keys by index; NaN counts as the largest
//   weight  the pick's score (renormalised: over the picks' sum, the softmax taken over the picks' own logits, so that
//           nothing underflows), times scale; a sum of 0 (every pick at -inf) gives weights of 0
//
// One wave per row. Lane i holds the E / 64 neighbouring experts from i * NPL, so the lowest lane of a tie holds the
// lowest index. A pick is one maximum over the lanes (six DPP steps), the first lane that has it, and that lane's next
// maximum. Nothing is kept between calls and no row depends on another.
#include "exl3_common.cuh"
#include "exl3_kernels.h"

#include <type_traits>

namespace exl3 {
namespace {

constexpr int kRouteWaves = 4;

// order-preserving keys: larger value, larger key; -0 as +0, NaN above everything, 0 below everything (no expert)
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    return v != v ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
    return v != v ? ~0ull : (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __builtin_bit_cast(float, (k & 0x80000000u) ? (k == 0xFFFFFFFFu ? 0x7FC00000u : k & 0x7FFFFFFFu) : ~k);
}
__device__ __forceinline__ double value_of(uint64_t k) {
    return __builtin_bit_cast(double, (k >> 63) ? (k == ~0ull ? 0x7FF8000000000000ull : k & 0x7FFFFFFFFFFFFFFFull) : ~k);
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
// the largest value over the wave, in every lane
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = dpp_max<0x111>(v);      // row_shr 1, 2, 4, 8: lane 15 of each row of 16 has the row's
    v = dpp_max<0x112>(v);
    v = dpp_max<0x114>(v);
    v = dpp_max<0x118>(v);
    v = dpp_max<0x142>(v);      // row_bcast 15 and 31: lane 63 has the wave's
    v = dpp_max<0x143>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
    const uint32_t hi = (uint32_t)(v >> 32), m = wave_max(hi);
    return (uint64_t)m << 32 | wave_max(hi == m ? (uint32_t)v : 0u);
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

template <int DT>
__device__ __forceinline__ float logit_at(const void* p, size_t i) {
    if constexpr (DT == 0) return (float)((const _Float16*)p)[i];
    else if constexpr (DT == 1) return __builtin_bit_cast(float, (uint32_t)((const uint16_t*)p)[i] << 16);
    else return ((const float*)p)[i];
}

// softmax terms relative to the row's largest logit (0 where that is -inf, so that exp gives 0)
template <class T>
__device__ __forceinline__ T top_or_0(T top) { return top == -(T)INFINITY ? (T)0 : top; }

template <int NPL, bool BIAS, int DT>
__global__ void __launch_bounds__(64 * kRouteWaves) route_kernel(RouteArgs A) {
    using Key = std::conditional_t<BIAS, uint64_t, uint32_t>;
    using Val = std::conditional_t<BIAS, double, float>;
    __shared__ Key lkeys[kRouteWaves][64 * NPL];
    __shared__ Key gkeys[kRouteWaves][kRouteMaxGroups];
    const int l = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x * kRouteWaves + wv;
    if (row >= A.M) return;
    const size_t base = (size_t)row * A.stride;
    const int e0 = l * NPL;

    float lg[NPL];
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        lg[j] = e0 + j < A.E ? logit_at<DT>(A.logits, base + e0 + j) : -INFINITY;
        most = max(most, e0 + j < A.E ? key_of(lg[j]) : 0u);
    }
    // the row's softmax where the keys or the weights need it
    Val top = 0, total = 1;
    if (!A.sigmoid && (BIAS || !A.renormalize)) {
        top = top_or_0((Val)value_of(wave_max(most)));
        total = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (e0 + j < A.E) total += BIAS ? exp((double)lg[j] - top) : (Val)expf(lg[j] - (float)top);
        total = wave_sum(total);
        if (total == 0) total = 1;
    }
    Key key[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        if constexpr (BIAS) {
            const double v = lg[j];
            const double sc = A.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - top) / total;
            key[j] = e0 + j < A.E ? key_of(sc + (double)A.bias[e0 + j]) : 0;
        } else {
            key[j] = e0 + j < A.E ? key_of(lg[j]) : 0;
        }
    }

    if (A.n_group > 1) {
        const int G = A.n_group, gs = A.E / G;
        Key* lk = lkeys[wv];
        Key* gk = gkeys[wv];
#pragma unroll
        for (int j = 0; j < NPL; ++j) lk[e0 + j] = key[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        // P = the power of two up to 64 / G lanes per group; each lane the two largest of its share, then of the group's
        const int P = 1 << (31 - __builtin_clz(64 / G)), g = l / P;
        Key t1 = 0, t2 = 0;
        if (g < G)
            for (int i = l & (P - 1); i < gs; i += P) {
                const Key k = lk[g * gs + i];
                t2 = k > t1 ? t1 : k > t2 ? k : t2;
                t1 = k > t1 ? k : t1;
            }
        for (int d = 1; d < P; d *= 2) {
            const Key o1 = __shfl_xor(t1, d), o2 = __shfl_xor(t2, d);
            const Key lo = t1 > o1 ? o1 : t1, hi2 = t2 > o2 ? t2 : o2;
            t1 = t1 > o1 ? t1 : o1;
            t2 = lo > hi2 ? lo : hi2;
        }
        if (g < G && (l & (P - 1)) == 0) {
            if constexpr (BIAS) gk[g] = gs > 1 ? key_of(value_of(t1) + value_of(t2)) : t1;
            else gk[g] = t1;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const Key mine = l < G ? gk[l] : 0;
        int rank = 0;
        for (int h = 0; h < G; ++h) {
            const Key o = gk[h];
            rank += o > mine || (o == mine && h < l);
        }
        const uint64_t kept = __ballot(l < G && rank < A.topk_group);
        const uint32_t magic = ((1u << 20) + gs - 1) / gs;      // e / gs for e < 1024 (e * gs < 2^20)
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (!(kept >> (((uint32_t)(e0 + j) * magic) >> 20) & 1)) key[j] = 0;
    }

    // the picks: lane r keeps pick r
    Key m = 0;
    int jm = 0, id = 0;
    Key picked = 0;
#pragma unroll
    for (int j = 0; j < NPL; ++j)
        if (key[j] > m) m = key[j], jm = j;
    for (int r = 0; r < A.topk; ++r) {
        const Key wm = wave_max(m);
        const int win = __builtin_ctzll(__ballot(m == wm));
        const int e = win * NPL + __builtin_amdgcn_readlane(jm, win);
        if (l == r) id = e, picked = wm;
        const int gone = l == win ? jm : -1;
        m = 0;
        jm = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            if (j == gone) key[j] = 0;
            if (key[j] > m) m = key[j], jm = j;
        }
    }

    const bool live = l < A.topk;
    float x, w;
    if constexpr (BIAS) x = live ? logit_at<DT>(A.logits, base + id) : -INFINITY;
    else x = live ? value_of(picked) : -INFINITY;
    if (A.sigmoid) w = 1.0f / (1.0f + expf(-x));
    else if (A.renormalize) w = expf(x - top_or_0(value_of(wave_max(live ? key_of(x) : 0u))));
    else w = (float)((BIAS ? exp((double)x - top) : (Val)expf(x - (float)top)) / total);
    if (!live) w = 0;
    if (A.renormalize) {
        const float sum = wave_sum(w);
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
    if (dtype == 0) hipLaunchKernelGGL((route_kernel<NPL, BIAS, 0>), grid, block, 0, s, a);
    else if (dtype == 1) hipLaunchKernelGGL((route_kernel<NPL, BIAS, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((route_kernel<NPL, BIAS, 2>), grid, block, 0, s, a);
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
