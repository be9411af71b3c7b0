// torch.ops.exl3xpu_moe: the reference's op schemas (kernels/moe-a8/exl3_moe.a8.sycl:1555-1592) implemented on the HIP
// dispatch key (DispatchKey::CUDA under PyTorch-ROCm) as thin wrappers over the C-ABI of libexl3moe.so.
// Shape/dtype checks raise RuntimeError like the reference's TORCH_CHECKs (a8:1266-1271).
#include <ATen/hip/HIPContext.h>
#include <c10/hip/HIPStream.h>
#include <torch/all.h>
#include <torch/library.h>

#include <algorithm>
#include <atomic>
#include <map>
#include <mutex>
#include <tuple>
#include <vector>

#include "../../include/exl3moe.h"

namespace {

void* cur_stream(const at::Tensor& like) {
    return (void*)c10::hip::getCurrentHIPStream(like.device().index()).stream();
}

void check(int rc, const char* what) { TORCH_CHECK(rc == EXL3_OK, what, ": ", exl3_last_error()); }

int dtype_code(const at::Tensor& x) {
    if (x.scalar_type() == at::kBFloat16) return EXL3_DT_BF16;
    if (x.scalar_type() == at::kHalf) return EXL3_DT_F16;
    if (x.scalar_type() == at::kFloat) return EXL3_DT_F32;
    TORCH_CHECK(false, "x dtype: bf16, fp16 or fp32 expected, got ", x.scalar_type());
}

at::Tensor forward_checked(const at::Tensor& x, const at::Tensor& topk_ids, const at::Tensor& topk_w,
                           const at::Tensor& ptrs, int64_t I, int64_t K, int64_t n_experts, const int64_t* hbm) {
    TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1, "moe_forward: x must be [M, H] with unit column stride");
    TORCH_CHECK(topk_ids.scalar_type() == at::kInt && topk_ids.is_contiguous(), "moe_forward: topk_ids int32 contiguous");
    TORCH_CHECK(topk_w.scalar_type() == at::kFloat && topk_w.is_contiguous(), "moe_forward: topk_w fp32 contiguous");
    TORCH_CHECK(ptrs.scalar_type() == at::kLong && ptrs.is_contiguous(), "moe_forward: ptrs int64 contiguous");
    const int M = (int)x.size(0), H = (int)x.size(1), topk = (int)topk_ids.size(-1);
    TORCH_CHECK(topk_ids.numel() == (int64_t)M * topk && topk_w.numel() == topk_ids.numel(), "moe_forward: ids/w [M, topk]");
    TORCH_CHECK(ptrs.numel() >= n_experts, "moe_forward: ptrs [n_experts]");
    auto out = at::empty_like(x);
    if (M == 0) return out;
    const size_t ws = exl3_moe_forward_workspace(M, H, (int)I, topk, (int)n_experts);
    auto w = at::empty({(int64_t)ws}, x.options().dtype(at::kByte));
    const int32_t* ids = topk_ids.data_ptr<int>();
    const int64_t* table = ptrs.data_ptr<int64_t>();
    check(hbm ? exl3_moe_forward_host(x.data_ptr(), dtype_code(x), x.stride(0), M, H, ids, topk_w.data_ptr<float>(), topk,
                                      table, (int)I, (int)K, (int)n_experts, out.data_ptr(), out.stride(0), w.data_ptr(),
                                      ws, hbm[0], hbm[1], cur_stream(x))
              : exl3_moe_forward(x.data_ptr(), dtype_code(x), x.stride(0), M, H, ids, topk_w.data_ptr<float>(), topk,
                                 table, (int)I, (int)K, (int)n_experts, out.data_ptr(), out.stride(0), w.data_ptr(), ws,
                                 cur_stream(x)),
          "moe_forward");
    return out;
}

at::Tensor moe_forward(at::Tensor x, at::Tensor topk_ids, at::Tensor topk_w, at::Tensor ptrs, int64_t I, int64_t K,
                       int64_t n_experts) {
    return forward_checked(x, topk_ids, topk_w, ptrs, I, K, n_experts, nullptr);
}
// the same for a table with experts in host memory (outside the device memory [hbm_base, hbm_base + hbm_bytes))
at::Tensor moe_forward_host(at::Tensor x, at::Tensor topk_ids, at::Tensor topk_w, at::Tensor ptrs, int64_t I, int64_t K,
                            int64_t n_experts, int64_t hbm_base, int64_t hbm_bytes) {
    const int64_t hbm[2] = {hbm_base, hbm_bytes};
    return forward_checked(x, topk_ids, topk_w, ptrs, I, K, n_experts, hbm);
}

// moe_prefetch (a8:1194-1222): claim slots for predicted experts of `layer`, copy them from host, repoint the table,
// on the current stream (use a side stream; make the compute stream wait before the next MoE call)
void moe_prefetch(at::Tensor ids, at::Tensor ptrs_all, int64_t layer, at::Tensor slot_of, at::Tensor slot_key,
                  at::Tensor slot_last, at::Tensor tick, at::Tensor host_base, int64_t slot_base, at::Tensor pf_list,
                  at::Tensor pf_slot, int64_t max_fill, int64_t n_experts, int64_t blob) {
    TORCH_CHECK(ids.scalar_type() == at::kInt && ids.is_contiguous(), "moe_prefetch: ids int32 contiguous");
    TORCH_CHECK(ptrs_all.scalar_type() == at::kLong && slot_of.scalar_type() == at::kInt &&
                    pf_list.scalar_type() == at::kInt && pf_slot.scalar_type() == at::kInt,
                "moe_prefetch: ptrs_all int64, slot_of / pf_list / pf_slot int32");
    TORCH_CHECK(ptrs_all.numel() >= (layer + 1) * n_experts && slot_of.numel() == ptrs_all.numel() &&
                    host_base.numel() > layer && pf_list.numel() >= 1 + n_experts &&
                    slot_last.numel() == slot_key.numel(),
                "moe_prefetch: cache state sizes");
    const int64_t mf = std::min<int64_t>(max_fill, pf_slot.numel());
    check(exl3_moe_prefetch(ids.data_ptr<int>(), (int)ids.numel(), ptrs_all.data_ptr<int64_t>(), (int)layer,
                            slot_of.data_ptr<int>(), slot_key.data_ptr<int>(), slot_last.data_ptr<int>(),
                            tick.data_ptr<int>(), (int)slot_key.numel(), host_base.data_ptr<int64_t>(), slot_base,
                            pf_list.data_ptr<int>(), pf_slot.data_ptr<int>(), (int)mf, (int)n_experts, blob,
                            cur_stream(ids)),
          "moe_prefetch");
}

// copy-engine prefetch (a8:1047-1142): plan on the current (compute) stream; the worker copies on the stream that is
// current when it starts
void moe_prefetch_plan(at::Tensor ids, at::Tensor ptrs_all, int64_t layer, at::Tensor slot_of, at::Tensor slot_key,
                       at::Tensor slot_last, at::Tensor tick, at::Tensor host_base, int64_t slot_base, at::Tensor pf_list,
                       at::Tensor pf_slot, at::Tensor plans, at::Tensor plan_seq, at::Tensor pend, at::Tensor done_seq,
                       int64_t max_fill, int64_t n_experts, int64_t blob) {
    TORCH_CHECK(ids.scalar_type() == at::kInt && ids.is_contiguous(), "moe_prefetch_plan: ids int32 contiguous");
    const int64_t L = done_seq.numel();
    TORCH_CHECK(L > layer && plan_seq.numel() >= L && pend.numel() >= L * 35 &&
                    plans.nbytes() >= (size_t)(L * (4 + 2 * n_experts) * 4) && pf_list.numel() >= 1 + n_experts,
                "moe_prefetch_plan: plan state sizes (start_copy_prefetch first)");
    check(exl3_moe_prefetch_plan(ids.data_ptr<int>(), (int)ids.numel(), ptrs_all.data_ptr<int64_t>(), (int)layer,
                                 slot_of.data_ptr<int>(), slot_key.data_ptr<int>(), slot_last.data_ptr<int>(),
                                 tick.data_ptr<int>(), (int)slot_key.numel(), host_base.data_ptr<int64_t>(), slot_base,
                                 pf_list.data_ptr<int>(), pf_slot.data_ptr<int>(), (int32_t*)plans.data_ptr(),
                                 plan_seq.data_ptr<int>(), pend.data_ptr<int>(), done_seq.data_ptr<int>(), (int)L,
                                 (int)std::min<int64_t>(max_fill, pf_slot.numel()), (int)n_experts, blob,
                                 cur_stream(ids)),
          "moe_prefetch_plan");
}

void moe_prefetch_worker_start(at::Tensor plans, at::Tensor host_base_cpu, int64_t slot_base, int64_t blob,
                               at::Tensor ptrs_all, at::Tensor slot_last, at::Tensor commit_host, at::Tensor done_seq,
                               int64_t n_layers, int64_t n_experts) {
    (void)ptrs_all;
    (void)slot_last;       // the commit runs on the device (ensure); the worker only publishes done_seq
    TORCH_CHECK(host_base_cpu.device().is_cpu() && host_base_cpu.scalar_type() == at::kLong &&
                    host_base_cpu.numel() >= n_layers && commit_host.nbytes() >= (size_t)(n_layers * 2 * 4),
                "moe_prefetch_worker_start: host_base_cpu int64 [n_layers] on the CPU, commit_host pinned");
    auto hb = host_base_cpu.contiguous();
    check(exl3_prefetch_worker_start((int32_t*)plans.data_ptr(), hb.data_ptr<int64_t>(), slot_base, blob,
                                     done_seq.data_ptr<int>(), (int32_t*)commit_host.data_ptr(), (int)n_layers,
                                     (int)n_experts, cur_stream(done_seq)),
          "moe_prefetch_worker_start");
}

std::vector<int64_t> moe_prefetch_worker_stop() {
    int64_t c[2] = {0, 0};
    check(exl3_prefetch_worker_stop(c), "moe_prefetch_worker_stop");
    return {c[0], c[1]};
}

at::Tensor moe_forward_cached(at::Tensor x, at::Tensor topk_ids, at::Tensor topk_w, at::Tensor ptrs_all, int64_t layer,
                              at::Tensor slot_of, at::Tensor slot_key, at::Tensor slot_last, at::Tensor tick,
                              at::Tensor host_base, int64_t slot_base, at::Tensor fill_all, at::Tensor fill_list,
                              int64_t max_fill, int64_t I, int64_t K, int64_t n_experts, at::Tensor pend,
                              at::Tensor done_seq) {
    // plans of the copy-engine prefetch are committed by this call's ensure when done_seq is in use
    if (done_seq.numel() > 0) {
        TORCH_CHECK(pend.numel() >= done_seq.numel() * 35, "moe_forward_cached: pend [n_layers * 35]");
        check(exl3_set_prefetch_commit(pend.data_ptr<int>(), done_seq.data_ptr<int>(), (int)done_seq.numel()),
              "moe_forward_cached");
    } else {
        check(exl3_set_prefetch_commit(nullptr, nullptr, 0), "moe_forward_cached");
    }
    TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1, "moe_forward_cached: x must be [M, H] with unit column stride");
    TORCH_CHECK(ptrs_all.scalar_type() == at::kLong && fill_all.scalar_type() == at::kLong &&
                    slot_of.scalar_type() == at::kInt,
                "moe_forward_cached: ptrs_all/fill_all int64, slot_of int32");
    TORCH_CHECK(topk_ids.scalar_type() == at::kInt && topk_ids.is_contiguous() && topk_w.scalar_type() == at::kFloat &&
                    topk_w.is_contiguous(),
                "tier mask: int32 ids, fp32 w");
    const int M = (int)x.size(0), H = (int)x.size(1), topk = (int)topk_ids.size(-1);
    TORCH_CHECK(topk_ids.numel() == (int64_t)M * topk && topk_w.numel() == topk_ids.numel(), "moe_forward_cached: ids/w [M, topk]");
    TORCH_CHECK(ptrs_all.numel() >= (layer + 1) * n_experts && slot_of.numel() == ptrs_all.numel() &&
                    fill_all.numel() == ptrs_all.numel() && host_base.numel() > layer &&
                    fill_list.numel() >= 1 + n_experts && slot_last.numel() == slot_key.numel(),
                "moe_forward_cached: cache state sizes");
    auto out = at::empty_like(x);
    if (M == 0) return out;
    const size_t ws = exl3_moe_forward_workspace(M, H, (int)I, topk, (int)n_experts);
    auto w = at::empty({(int64_t)ws}, x.options().dtype(at::kByte));
    check(exl3_moe_forward_cached(x.data_ptr(), dtype_code(x), x.stride(0), M, H, topk_ids.data_ptr<int>(),
                                  topk_w.data_ptr<float>(), topk, ptrs_all.data_ptr<int64_t>(), (int)layer,
                                  slot_of.data_ptr<int>(), slot_key.data_ptr<int>(), slot_last.data_ptr<int>(),
                                  tick.data_ptr<int>(), (int)slot_key.numel(), host_base.data_ptr<int64_t>(), slot_base,
                                  fill_all.data_ptr<int64_t>(), fill_list.data_ptr<int>(), (int)max_fill, (int)I,
                                  (int)K, (int)n_experts, out.data_ptr(), out.stride(0), w.data_ptr(), ws,
                                  cur_stream(x)),
          "moe_forward_cached");
    return out;
}

std::vector<at::Tensor> moe_align(at::Tensor topk_ids, at::Tensor topk_w, int64_t n_experts, int64_t pad) {
    TORCH_CHECK(topk_ids.scalar_type() == at::kInt && topk_ids.is_contiguous() && topk_ids.dim() == 2, "moe_align: ids");
    TORCH_CHECK(topk_w.scalar_type() == at::kFloat && topk_w.is_contiguous(), "moe_align: w");
    const int M = (int)topk_ids.size(0), topk = (int)topk_ids.size(1), npairs = M * topk;
    const int A = std::min(npairs, (int)n_experts);
    auto ib = at::empty({4 * A + 1 + 2 * npairs + 16}, topk_ids.options());
    auto fb = at::empty({npairs}, topk_w.options());
    const size_t wsb = exl3_moe_align_workspace(M, topk, (int)n_experts);
    auto ws = at::empty({(int64_t)std::max<size_t>(wsb, 1)}, topk_ids.options().dtype(at::kByte));
    check(exl3_moe_align(topk_ids.data_ptr<int>(), topk_w.data_ptr<float>(), M, topk, (int)n_experts, (int)pad,
                         ib.data_ptr<int>(), fb.data_ptr<float>(), ws.data_ptr(), wsb, cur_stream(topk_ids)),
          "moe_align");
    return {ib, fb};
}

at::Tensor host_alloc(int64_t nbytes) {
    void* p = exl3_host_alloc(nbytes);
    TORCH_CHECK(p, "host_alloc failed for ", nbytes, " bytes: ", exl3_last_error());
    return at::from_blob(p, {nbytes}, [](void* q) { exl3_host_free(q); },
                         at::TensorOptions().dtype(at::kByte).device(at::kCPU));
}

int64_t usm_kind(int64_t ptr) { return exl3_usm_kind(reinterpret_cast<const void*>(ptr)); }

void memcpy_async(int64_t dst, int64_t src, int64_t nbytes) {
    void* s = (void*)c10::hip::getCurrentHIPStream().stream();
    check(exl3_memcpy_async(reinterpret_cast<void*>(dst), reinterpret_cast<const void*>(src), nbytes, s), "memcpy_async");
}

int64_t blob_bytes(int64_t H, int64_t I, int64_t K) { return exl3_blob_bytes((int)H, (int)I, (int)K); }

void moe_set_splits(int64_t gu_p, int64_t dn_p) { check(exl3_set_splits(gu_p, dn_p), "moe_set_splits"); }
void moe_set_mr(int64_t mr) { check(exl3_set_mr(mr), "moe_set_mr"); }
void moe_set_debug(int64_t v) { check(exl3_set_debug(v), "moe_set_debug"); }
void moe_set_pair_max_m(int64_t v) { check(exl3_set_pair_max_m(v), "moe_set_pair_max_m"); }
void moe_set_prefill_min_m(int64_t v) { check(exl3_set_prefill_min_m(v), "moe_set_prefill_min_m"); }
// moe_set_victim_ring (experimental/n111-victim-ring/a9.patch:17-30): meta int32 [4 + 2K], sel int32 [E], buf the
// K ring slots; an empty meta turns the ring off
void moe_set_victim_ring(at::Tensor meta, at::Tensor sel, at::Tensor buf) {
    if (!meta.numel()) return check(exl3_set_victim_ring(nullptr, nullptr, nullptr, 0, 0), "moe_set_victim_ring");
    TORCH_CHECK(meta.scalar_type() == at::kInt && sel.scalar_type() == at::kInt && meta.is_contiguous() &&
                    sel.is_contiguous() && meta.is_cuda() && sel.is_cuda() && buf.is_cuda(),
                "moe_set_victim_ring: device int32 meta and sel");
    const int64_t K = (meta.numel() - 4) / 2;
    TORCH_CHECK(K > 0 && meta.numel() == 4 + 2 * K && buf.numel() > 0, "victim ring: meta [4 + 2K], buf [K * blob]");
    check(exl3_set_victim_ring(meta.data_ptr<int>(), sel.data_ptr<int>(), buf.data_ptr(),
                               (int64_t)buf.numel() * (int64_t)buf.element_size(), K),
          "moe_set_victim_ring");
}

void moe_set_victims(at::Tensor v) {
    if (!v.numel()) return check(exl3_set_victims(nullptr), "moe_set_victims");
    TORCH_CHECK(v.scalar_type() == at::kInt && v.is_cuda(), "moe_set_victims: device int32 tensor");
    check(exl3_set_victims(v.data_ptr<int>()), "moe_set_victims");
}
void moe_set_tier(at::Tensor ram_res, at::Tensor miss, at::Tensor safe) {
    if (!ram_res.numel()) return check(exl3_set_tier(nullptr, nullptr, 0, nullptr), "moe_set_tier");
    TORCH_CHECK(ram_res.scalar_type() == at::kByte && miss.scalar_type() == at::kInt && safe.scalar_type() == at::kInt,
                "moe_set_tier: uint8 ram_res, int32 miss ring, int32 safe");
    check(exl3_set_tier(ram_res.data_ptr<uint8_t>(), miss.data_ptr<int>(), miss.numel(), safe.data_ptr<int>()),
          "moe_set_tier");
}
void moe_set_host_stride(int64_t s) { check(exl3_set_host_stride(s), "moe_set_host_stride"); }
void moe_set_slot_stride(int64_t s) { check(exl3_set_slot_stride(s), "moe_set_slot_stride"); }
void moe_set_fused_ensure(int64_t v) { check(exl3_set_fused_ensure(v), "moe_set_fused_ensure"); }
// pinned host memory is device-mapped on MI355X: nothing to prefetch (the reference maps xe-SVM pages, a8:777-781)
void moe_svm_prefetch(at::Tensor ptrs, int64_t nbytes, at::Tensor like) {
    (void)ptrs;
    (void)nbytes;
    (void)like;
}
void moe_set_decision_log(at::Tensor buf) {
    if (!buf.numel()) return check(exl3_set_decision_log(nullptr, 0), "moe_set_decision_log");
    TORCH_CHECK(buf.scalar_type() == at::kInt && buf.is_cuda() && buf.is_contiguous(), "decision log: device int32");
    check(exl3_set_decision_log(buf.data_ptr<int>(), buf.numel() - 1), "moe_set_decision_log");
}
at::Tensor dequant(at::Tensor trellis, int64_t k_tiles, int64_t n_tiles, int64_t K) {
    TORCH_CHECK(trellis.is_cuda() && trellis.is_contiguous(), "dequant: contiguous device words");
    auto out = at::empty({16 * k_tiles, 16 * n_tiles}, trellis.options().dtype(at::kHalf));
    check(exl3_dequant(reinterpret_cast<const uint32_t*>(trellis.data_ptr()), (int)k_tiles, (int)n_tiles, (int)K,
                       reinterpret_cast<uint16_t*>(out.data_ptr()), cur_stream(trellis)),
          "dequant");
    return out;
}

// ---- torch.ops.exl3xpu_C: the dense EXL3 linear (experimental/n111-victim-ring/csrc/exl3_ops.sycl:639-781, 784-815)

void linear_checks(const at::Tensor& trellis, const at::Tensor& suh, const at::Tensor& svh, const at::Tensor& sonb,
                   int64_t k, int64_t K, int64_t cb) {
    TORCH_CHECK(exl3_linear_supported((int)K, (int)cb), "exl3xpu_C.linear: K=", K, " cb=", cb, " not built");
    TORCH_CHECK(trellis.is_cuda() && trellis.is_contiguous() && trellis.dim() == 3 && trellis.size(0) * 16 == k &&
                    trellis.size(2) == 16 * K,
                "exl3xpu_C.linear: trellis [k/16, n/16, 16K] contiguous on the device");
    TORCH_CHECK(suh.scalar_type() == at::kHalf && suh.is_contiguous() && suh.dim() == 2 && suh.size(1) == k,
                "exl3xpu_C.linear: suh fp16 [S, k]");
    TORCH_CHECK(svh.scalar_type() == at::kHalf && svh.is_contiguous() && svh.size(0) == trellis.size(1) * 16,
                "exl3xpu_C.linear: svh fp16 [n]");
    TORCH_CHECK(sonb.scalar_type() == at::kInt && sonb.is_contiguous() && sonb.numel() * 128 == svh.size(0),
                "exl3xpu_C.linear: shard_of_nb int32 [n / 128]");
}

// The small-M workspace. Its tagged partials must be zero when a call starts; every call leaves them zero.
// Eager calls on one (device, stream) share one buffer, zeroed when it is allocated, and run in stream order. A call
// made while its stream is being captured into a HIP graph gets a buffer of that capture alone (keyed by the capture
// id), allocated and zeroed inside the capture: the zero fill (a fill kernel, not a memset node) is then a node of
// that graph, so each replay starts from zero whatever ran on the buffer of another graph or of eager calls, and
// graphs captured one after another on the same stream can be replayed in any order. Sized for 8 rows; a larger one
// replaces it when a call needs more. Buffers are kept until the process ends: a captured graph holds their
// addresses.
at::Tensor& small_workspace(const at::Tensor& x, size_t bytes) {
    static std::mutex mu;
    static auto* cache = new std::map<std::tuple<int, void*, unsigned long long>, at::Tensor>();
    static auto* retired = new std::vector<at::Tensor>();
    void* st = cur_stream(x);
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    unsigned long long cid = 0;
    TORCH_CHECK(hipStreamGetCaptureInfo((hipStream_t)st, &cs, &cid) == hipSuccess, "exl3_gemm_small: capture status");
    if (cs != hipStreamCaptureStatusActive) cid = 0;            // eager: the stream's own buffer
    else if (cid == 0) cid = ~0ull;                             // (capture ids start at 1; keep 0 for eager calls)
    std::lock_guard<std::mutex> lock(mu);
    auto& t = (*cache)[{(int)x.device().index(), st, cid}];
    if (!t.defined() || (size_t)t.numel() < bytes) {
        if (t.defined()) retired->push_back(t);
        t = at::zeros({(int64_t)bytes}, x.options().dtype(at::kByte));
    }
    return t;
}

void gemm_small(at::Tensor x2, at::Tensor trellis, at::Tensor suh, at::Tensor svh, at::Tensor shard_of_nb, at::Tensor out,
                int64_t K, int64_t cb) {
    const int64_t M = x2.size(0), k = x2.size(1), n = svh.size(0);
    linear_checks(trellis, suh, svh, shard_of_nb, k, K, cb);
    TORCH_CHECK(x2.stride(1) == 1 && out.dim() == 2 && out.size(0) == M && out.size(1) == n && out.stride(1) == 1,
                "exl3_gemm_small: x [M, k], out [M, n] with unit column strides");
    TORCH_CHECK(M <= 8, "exl3_gemm_small: at most 8 rows, got ", M);
    const size_t ws_bytes = exl3_linear_workspace(8, (int)k, (int)n);
    auto& ws = small_workspace(x2, ws_bytes);
    check(exl3_linear_small(x2.data_ptr(), dtype_code(x2), x2.stride(0), (int)M, (int)k, (int)n, trellis.data_ptr(),
                            (int)K, (int)cb, suh.data_ptr(), (int)suh.size(0), svh.data_ptr(),
                            shard_of_nb.data_ptr<int>(), out.data_ptr(), dtype_code(out), out.stride(0), ws.data_ptr(),
                            ws_bytes, cur_stream(x2)),
          "exl3xpu_C.exl3_gemm_small");
}

void had_in_rm(at::Tensor x, at::Tensor suh, at::Tensor xh) {
    TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1, "exl3_had_in_rm: x [M, k]");
    TORCH_CHECK(xh.scalar_type() == at::kHalf && xh.is_contiguous() && xh.dim() == 3 && xh.size(1) == x.size(0) &&
                    xh.size(2) == x.size(1) && suh.scalar_type() == at::kHalf && suh.dim() == 2 &&
                    suh.size(0) == xh.size(0) && suh.is_contiguous(),
                "exl3_had_in_rm: xh fp16 [S, M, k], suh fp16 [S, k]");
    check(exl3_had_in(x.data_ptr(), dtype_code(x), x.stride(0), (int)x.size(0), (int)x.size(1), suh.data_ptr(),
                      (int)suh.size(0), xh.data_ptr(), cur_stream(x)),
          "exl3xpu_C.exl3_had_in_rm");
}

void had_out_h(at::Tensor y, at::Tensor svh, at::Tensor out) {
    TORCH_CHECK(y.scalar_type() == at::kHalf && y.is_contiguous() && y.sizes() == out.sizes() && y.dim() == 2 &&
                    out.stride(1) == 1 && svh.scalar_type() == at::kHalf && svh.numel() == y.size(1),
                "exl3_had_out_h: y fp16 [M, n] contiguous, out [M, n], svh fp16 [n]");
    check(exl3_had_out(y.data_ptr(), (int)y.size(0), (int)y.size(1), svh.data_ptr(), out.data_ptr(), dtype_code(out),
                       out.stride(0), cur_stream(y)),
          "exl3xpu_C.exl3_had_out_h");
}

void reconstruct(at::Tensor trellis, at::Tensor w, int64_t n0, int64_t K, int64_t cb) {
    TORCH_CHECK(trellis.is_cuda() && trellis.is_contiguous() && trellis.dim() == 3, "exl3_reconstruct: trellis");
    TORCH_CHECK(w.scalar_type() == at::kHalf && w.is_contiguous() && w.dim() == 2 && w.size(0) == trellis.size(0) * 16,
                "exl3_reconstruct: w fp16 [k, width] contiguous");
    check(exl3_reconstruct(trellis.data_ptr(), (int)w.size(0), (int)trellis.size(1) * 16, (int)n0,
                           (int)(n0 + w.size(1)), (int)K, (int)cb, w.data_ptr(), cur_stream(w)),
          "exl3xpu_C.exl3_reconstruct");
}

// the W8A8 route's switch (exl3_set_int8, exl3_ops.sycl:524): off unless the caller turns it on
std::atomic<bool> g_int8{false};
void set_int8(int64_t on) { g_int8.store(on != 0); }

// the W8A8 route (exl3_ops.sycl:668-740, the path without oneDNN): int8 xh with one scale per (shard, row), then per
// shard group the int8 weights at the static scale, the library's int8 GEMM (int32 sums) and the output Hadamard of
// y * sx * sw into the group's columns of out
void linear_q8(const at::Tensor& x2, const at::Tensor& trellis, const at::Tensor& suh, const at::Tensor& svh,
               at::IntArrayRef group_bounds, int64_t K, at::Tensor& out) {
    const int64_t M = x2.size(0), k = x2.size(1), n = svh.size(0), S = suh.size(0);
    void* st = cur_stream(x2);
    auto xq = at::empty({S, M, k}, x2.options().dtype(at::kChar));
    auto sx = at::empty({S, M}, x2.options().dtype(at::kFloat));
    check(exl3_had_in_q8(x2.data_ptr(), dtype_code(x2), x2.stride(0), (int)M, (int)k, suh.data_ptr(), (int)S,
                         xq.data_ptr(), sx.data_ptr(), M, st),
          "exl3xpu_C.linear (int8 had_in)");
    const float sw = 3.453125f / 127.0f;
    for (int64_t g = 0; g < S; ++g) {
        const int64_t g0 = group_bounds[g], g1 = group_bounds[g + 1], ng = g1 - g0;
        TORCH_CHECK(g0 <= g1 && g1 <= n && g0 % 128 == 0 && ng % 128 == 0,
                    "exl3xpu_C.linear: int8 route needs shard groups of whole 128-column blocks");
        if (ng == 0) continue;
        auto w = at::empty({k, ng}, x2.options().dtype(at::kChar));
        check(exl3_reconstruct_q8(trellis.data_ptr(), (int)k, (int)n, (int)g0, (int)g1, (int)K, w.data_ptr(), st),
              "exl3xpu_C.linear (int8 weights)");
        auto y = at::_int_mm(xq[g], w);                               // [M, ng] int32
        auto og = out.narrow(1, g0, ng);
        check(exl3_had_out_q8(y.data_ptr<int32_t>(), (int)M, (int)ng, sx.data_ptr<float>() + g * M, sw,
                              svh.narrow(0, g0, ng).data_ptr(), og.data_ptr(), dtype_code(out), out.stride(0), st),
              "exl3xpu_C.linear (int8 had_out)");
    }
}

// exl3_linear (exl3_ops.sycl:651-757): M <= small_m_max (at most 8 rows here) -> the fused path; otherwise, with at most 16
// shards of whole 128-column blocks, S k up to 2^22 and a trellis below 2 GiB, exl3_linear_rows, which decodes the trellis
// inside the product (111 -> 26 us at 40 rows and 689 -> 557 us at 8,192 rows of 2048 -> 12,288 against the following);
// else the input Hadamards, per shard group the reconstructed fp16 weights in slices of slice_n columns times xh[g] (a
// library GEMM, fp16 output), then the output Hadamard. slice_n is the library GEMM's alone.
at::Tensor linear(at::Tensor x, at::Tensor trellis, at::Tensor suh, at::Tensor svh, at::Tensor shard_of_nb,
                  at::IntArrayRef group_bounds, int64_t K, int64_t cb, int64_t small_m_max, int64_t slice_n) {
    auto shape = x.sizes().vec();
    const int64_t k = shape.back(), n = svh.size(0);
    auto x2 = x.reshape({-1, k});
    if (!x2.is_contiguous()) x2 = x2.contiguous();
    const int64_t M = x2.size(0);
    shape.back() = n;
    auto out = at::empty({M, n}, x.options());
    if (M == 0) return out.view(shape);
    linear_checks(trellis, suh, svh, shard_of_nb, k, K, cb);
    if (M <= std::min<int64_t>(small_m_max, 8)) {
        gemm_small(x2, trellis, suh, svh, shard_of_nb, out, K, cb);
        return out.view(shape);
    }
    const int64_t S = suh.size(0);
    TORCH_CHECK((int64_t)group_bounds.size() == S + 1 && group_bounds[0] == 0 && group_bounds[S] == n,
                "exl3xpu_C.linear: group_bounds [0, ..., n] with one group per suh row");
    if (g_int8.load() && cb == 2 && (K == 4 || K == 6) && M > 16) {     // exl3_ops.sycl:668
        linear_q8(x2, trellis, suh, svh, group_bounds, K, out);
        return out.view(shape);
    }
    // (row slices keep xh below 2 GiB)
    int64_t width = S <= 16 && k * n / 8 * K < (int64_t)1 << 31 && S * k <= (int64_t)1 << 22 ? 256 : 0;
    for (int64_t g = 0; g < S && width; ++g) {
        TORCH_CHECK(group_bounds[g] <= group_bounds[g + 1], "exl3xpu_C.linear: group_bounds not ascending");
        width = group_bounds[g + 1] % 128 ? 0 : group_bounds[g + 1] % 256 ? 128 : width;
    }
    if (width) {
        const int64_t step = std::min<int64_t>(M, std::max<int64_t>(128, (((int64_t)1 << 30) - 1) / (S * k) / 128 * 128));
        const size_t wb = exl3_linear_rows_workspace((int)step, (int)k, (int)n, (int)S, (int)width);
        auto ws = at::empty({(int64_t)wb}, x.options().dtype(at::kByte));
        const int64_t esz = x2.element_size();
        for (int64_t m0 = 0; m0 < M; m0 += step) {
            const int64_t ms = std::min(step, M - m0);
            check(exl3_linear_rows((const char*)x2.data_ptr() + m0 * k * esz, dtype_code(x2), k, (int)ms, (int)k, (int)n,
                                   trellis.data_ptr(), (int)K, (int)cb, suh.data_ptr(), (int)S, svh.data_ptr(),
                                   group_bounds.data(), (int)width, (char*)out.data_ptr() + m0 * n * esz,
                                   dtype_code(out), n, ws.data_ptr(), wb, cur_stream(x2)),
                  "exl3xpu_C.linear (rows)");
        }
        return out.view(shape);
    }
    auto xh = at::empty({S, M, k}, x.options().dtype(at::kHalf));
    had_in_rm(x2, suh, xh);
    auto y = at::empty({M, n}, x.options().dtype(at::kHalf));
    const int64_t step = slice_n > 0 ? std::max<int64_t>(16, slice_n / 16 * 16) : n;
    // one reconstructed slice at a time, from the caching allocator (stream-ordered reuse across slices and calls)
    auto wbuf = at::empty({k * std::min(step, n)}, x.options().dtype(at::kHalf));
    for (int64_t g = 0; g < S; ++g) {
        const int64_t g0 = group_bounds[g], g1 = group_bounds[g + 1];
        TORCH_CHECK(g0 <= g1 && g1 <= n, "exl3xpu_C.linear: group_bounds not ascending");
        for (int64_t n0 = g0; n0 < g1; n0 += step) {
            const int64_t n1 = std::min(n0 + step, g1);
            auto w = wbuf.narrow(0, 0, k * (n1 - n0)).view({k, n1 - n0});
            reconstruct(trellis, w, n0, K, cb);
            auto ys = y.narrow(1, n0, n1 - n0);
            at::matmul_out(ys, xh[g], w);
        }
    }
    had_out_h(y, svh, out);
    return out.view(shape);
}

at::Tensor linear_meta(at::Tensor x, at::Tensor trellis, at::Tensor suh, at::Tensor svh, at::Tensor shard_of_nb,
                       at::IntArrayRef group_bounds, int64_t K, int64_t cb, int64_t small_m_max, int64_t slice_n) {
    auto shape = x.sizes().vec();
    shape.back() = svh.size(0);
    return at::empty(shape, x.options());
}

bool linear_supported(int64_t K, int64_t cb) { return exl3_linear_supported((int)K, (int)cb) != 0; }

// ---- exl3xpu_moe.moe_route and the 8-bit float linear of exl3xpu_C ----------------------------------------------------
// (no counterpart in the reference). Every tensor of a call lives on the first one's device, which the call's launches,
// allocations and stream are those of, whatever device is current.

void on_device_of(const at::Tensor& x, const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.device() == x.device(), what, ": tensors on ", x.device(), " and ", t.device());
}

// fp32, contiguous and of `n` values on x's device; null where there is none
const float* f32_or_null(const std::optional<at::Tensor>& t, const at::Tensor& x, int64_t n, const char* what) {
    if (!t) return nullptr;
    on_device_of(x, *t, what);
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 1 && t->numel() == n, what,
                ": bias fp32 [", n, "] contiguous");
    return t->data_ptr<float>();
}

// [..., n] as [rows, n] with unit column stride (a copy only where the strides are not those of such rows)
at::Tensor rows_of(const at::Tensor& x, const char* what) {
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, what, ": [..., n] with n > 0, got ", x.sizes());
    TORCH_CHECK(x.numel() / x.size(-1) <= INT32_MAX && x.size(-1) <= INT32_MAX, what, ": sizes ", x.sizes());
    auto x2 = x.dim() == 2 ? x : x.reshape({x.numel() / x.size(-1), x.size(-1)});
    return x2.size(0) == 0 || (x2.stride(1) == 1 && (x2.size(0) == 1 || x2.stride(0) >= x2.size(1))) ? x2 : x2.contiguous();
}
int64_t row_stride(const at::Tensor& x2) { return x2.size(0) > 1 ? x2.stride(0) : x2.size(1); }

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t n) {
    TORCH_CHECK(!sizes.empty(), "a tensor of at least one dimension, got a scalar");
    auto v = sizes.vec();
    v.back() = n;
    return v;
}
int64_t fp8_up(int64_t k) { return (k + 127) / 128 * 128; }

int scoring_code(c10::string_view scoring) {
    TORCH_CHECK(scoring == "softmax" || scoring == "sigmoid", "moe_route: scoring 'softmax' or 'sigmoid', got '", scoring, "'");
    return scoring == "sigmoid";
}

std::tuple<at::Tensor, at::Tensor> moe_route(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t topk,
                                             c10::string_view scoring, int64_t n_group, int64_t topk_group,
                                             bool renormalize, double scale) {
    const c10::DeviceGuard guard(logits.device());
    const int sc = scoring_code(scoring);
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) > 0 && logits.size(-1) <= 1024, "moe_route: 1 to 1024 experts, got ",
                logits.sizes());
    const int64_t E = logits.size(-1);
    for (int64_t v : {topk, n_group, topk_group})
        TORCH_CHECK(v >= 1 && v <= E, "moe_route: topk, n_group and topk_group in 1..", E, ", got ", v);
    const int dt = dtype_code(logits);
    auto x2 = rows_of(logits, "moe_route");
    const float* b = f32_or_null(bias, logits, E, "moe_route");
    auto ids = at::empty(with_last(logits.sizes(), topk), logits.options().dtype(at::kInt));
    auto w = at::empty(with_last(logits.sizes(), topk), logits.options().dtype(at::kFloat));
    check(exl3_moe_route(x2.data_ptr(), dt, row_stride(x2), (int)x2.size(0), (int)E, b, (int)topk, sc, (int)n_group,
                         (int)topk_group, renormalize, (float)scale, ids.data_ptr<int>(), w.data_ptr<float>(),
                         cur_stream(logits)),
          "moe_route");
    return {ids, w};
}

std::tuple<at::Tensor, at::Tensor> moe_route_meta(const at::Tensor& logits, const std::optional<at::Tensor>&, int64_t topk,
                                                  c10::string_view, int64_t, int64_t, bool, double) {
    return {at::empty(with_last(logits.sizes(), topk), logits.options().dtype(at::kInt)),
            at::empty(with_last(logits.sizes(), topk), logits.options().dtype(at::kFloat))};
}

std::tuple<at::Tensor, at::Tensor> fp8_rows_empty(const at::Tensor& x, int64_t k) {
    return {at::empty(with_last(x.sizes(), fp8_up(k)), x.options().dtype(at::kFloat8_e4m3fn)),
            at::empty(with_last(x.sizes(), fp8_up(k) / 128), x.options().dtype(at::kFloat))};
}
std::tuple<at::Tensor, at::Tensor> fp8_quant_meta(const at::Tensor& x) { return fp8_rows_empty(x, x.size(-1)); }
std::tuple<at::Tensor, at::Tensor> fp8_silu_mul_quant_meta(const at::Tensor& x) {
    return fp8_rows_empty(x, x.size(-1) / 2);
}

std::tuple<at::Tensor, at::Tensor> fp8_quant(const at::Tensor& x) {
    const c10::DeviceGuard guard(x.device());
    const int dt = dtype_code(x);
    auto x2 = rows_of(x, "fp8_quant");
    auto out = fp8_rows_empty(x, x.size(-1));
    check(exl3_fp8_quant(x2.data_ptr(), dt, row_stride(x2), (int)x2.size(0), (int)x2.size(1), std::get<0>(out).data_ptr(),
                         std::get<1>(out).data_ptr<float>(), cur_stream(x)),
          "fp8_quant");
    return out;
}

std::tuple<at::Tensor, at::Tensor> fp8_silu_mul_quant(const at::Tensor& x) {
    const c10::DeviceGuard guard(x.device());
    const int dt = dtype_code(x);
    auto x2 = rows_of(x, "fp8_silu_mul_quant");
    TORCH_CHECK(x2.size(1) % 2 == 0, "fp8_silu_mul_quant: gate|up rows of an even size, got ", x.sizes());
    const int64_t k = x2.size(1) / 2;
    auto out = fp8_rows_empty(x, k);
    check(exl3_fp8_silu_mul_quant(x2.data_ptr(), dt, row_stride(x2), (int)x2.size(0), (int)k, std::get<0>(out).data_ptr(),
                                  std::get<1>(out).data_ptr<float>(), cur_stream(x)),
          "fp8_silu_mul_quant");
    return out;
}

void fp8_weight_checks(const at::Tensor& x, const at::Tensor& w, const at::Tensor& sw, int64_t k, const char* what) {
    on_device_of(x, w, what);
    on_device_of(x, sw, what);
    TORCH_CHECK(w.scalar_type() == at::kFloat8_e4m3fn && w.is_contiguous() && w.dim() == 2 && w.size(1) == fp8_up(k) &&
                    w.size(0) > 0 && w.size(0) <= INT32_MAX,
                what, ": weight float8_e4m3fn [n, ", fp8_up(k), "] contiguous, got ", w.scalar_type(), " ", w.sizes());
    TORCH_CHECK(sw.scalar_type() == at::kFloat && sw.is_contiguous() && sw.dim() == 2 &&
                    sw.size(0) == fp8_up(w.size(0)) / 128 && sw.size(1) == w.size(1) / 128,
                what, ": weight_scale fp32 [", fp8_up(w.size(0)) / 128, ", ", w.size(1) / 128, "] contiguous, got ",
                sw.scalar_type(), " ", sw.sizes());
}

at::Tensor fp8_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& sw, const std::optional<at::Tensor>& bias) {
    const c10::DeviceGuard guard(x.device());
    const int dt = dtype_code(x);
    auto x2 = rows_of(x, "fp8_linear");
    const int M = (int)x2.size(0), k = (int)x2.size(1);
    fp8_weight_checks(x, w, sw, k, "fp8_linear");
    const int64_t n = w.size(0);
    const float* b = f32_or_null(bias, x, n, "fp8_linear");
    auto out = at::empty(with_last(x.sizes(), n), x.options());
    if (M == 0) return out;
    const size_t ws = exl3_fp8_linear_workspace(M, k, (int)n);
    auto buf = at::empty({(int64_t)ws}, x.options().dtype(at::kByte));
    check(exl3_fp8_linear(x2.data_ptr(), dt, row_stride(x2), M, k, (int)n, w.data_ptr(), sw.data_ptr<float>(), b,
                          out.data_ptr(), dt, n, buf.data_ptr(), ws, cur_stream(x)),
          "fp8_linear");
    return out;
}

at::Tensor fp8_mlp(const at::Tensor& x, const at::Tensor& gu, const at::Tensor& gu_scale,
                   const std::optional<at::Tensor>& gu_bias, const at::Tensor& dn, const at::Tensor& dn_scale,
                   const std::optional<at::Tensor>& dn_bias) {
    const c10::DeviceGuard guard(x.device());
    const int dt = dtype_code(x);
    auto x2 = rows_of(x, "fp8_mlp");
    const int M = (int)x2.size(0), k = (int)x2.size(1);
    fp8_weight_checks(x, gu, gu_scale, k, "fp8_mlp (gate|up)");
    TORCH_CHECK(gu.size(0) % 2 == 0, "fp8_mlp: gate|up weights of an even number of rows, got ", gu.sizes());
    const int64_t I = gu.size(0) / 2, n = dn.size(0);
    fp8_weight_checks(x, dn, dn_scale, I, "fp8_mlp (down)");
    const float* gb = f32_or_null(gu_bias, x, 2 * I, "fp8_mlp (gate|up)");
    const float* db = f32_or_null(dn_bias, x, n, "fp8_mlp (down)");
    auto out = at::empty(with_last(x.sizes(), n), x.options());
    if (M == 0) return out;
    const size_t ws = exl3_fp8_mlp_workspace(M, k, (int)I, (int)n, dt);
    auto buf = at::empty({(int64_t)ws}, x.options().dtype(at::kByte));
    check(exl3_fp8_mlp(x2.data_ptr(), dt, row_stride(x2), M, k, (int)I, (int)n, gu.data_ptr(), gu_scale.data_ptr<float>(),
                       gb, dn.data_ptr(), dn_scale.data_ptr<float>(), db, out.data_ptr(), n, buf.data_ptr(), ws,
                       cur_stream(x)),
          "fp8_mlp");
    return out;
}

at::Tensor fp8_mlp_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, const std::optional<at::Tensor>&,
                        const at::Tensor& dn, const at::Tensor&, const std::optional<at::Tensor>&) {
    return at::empty(with_last(x.sizes(), dn.size(0)), x.options());
}

at::Tensor fp8_linear_meta(const at::Tensor& x, const at::Tensor& w, const at::Tensor&, const std::optional<at::Tensor>&) {
    return at::empty(with_last(x.sizes(), w.size(0)), x.options());
}

at::Tensor fp8_matmul(const at::Tensor& q, const at::Tensor& s, const at::Tensor& w, const at::Tensor& sw,
                      const std::optional<at::Tensor>& bias, at::ScalarType dtype) {
    const c10::DeviceGuard guard(q.device());
    TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn && q.is_contiguous() && q.dim() >= 1 && q.size(-1) > 0 &&
                    q.size(-1) % 128 == 0 && q.size(-1) <= INT32_MAX && q.numel() / q.size(-1) <= INT32_MAX,
                "fp8_matmul: q float8_e4m3fn [..., a multiple of 128] contiguous, got ", q.scalar_type(), " ", q.sizes());
    const int k = (int)q.size(-1), M = (int)(q.numel() / k);
    on_device_of(q, s, "fp8_matmul");
    TORCH_CHECK(s.scalar_type() == at::kFloat && s.is_contiguous() && s.dim() == q.dim() &&
                    s.sizes().vec() == with_last(q.sizes(), k / 128),
                "fp8_matmul: s fp32 ", with_last(q.sizes(), k / 128), " contiguous, got ", s.scalar_type(), " ", s.sizes());
    fp8_weight_checks(q, w, sw, k, "fp8_matmul");
    const int64_t n = w.size(0);
    const float* b = f32_or_null(bias, q, n, "fp8_matmul");
    auto out = at::empty(with_last(q.sizes(), n), q.options().dtype(dtype));
    const int dt = dtype_code(out);
    if (M == 0) return out;
    check(exl3_fp8_matmul(q.data_ptr(), s.data_ptr<float>(), M, k, (int)n, w.data_ptr(), sw.data_ptr<float>(), b,
                          out.data_ptr(), dt, n, nullptr, 0, cur_stream(q)),
          "fp8_matmul");
    return out;
}

at::Tensor fp8_matmul_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor& w, const at::Tensor&,
                           const std::optional<at::Tensor>&, at::ScalarType dtype) {
    return at::empty(with_last(q.sizes(), w.size(0)), q.options().dtype(dtype));
}

// ---- the norm and the 4-bit float linear of exl3xpu_C (no counterpart in the reference) ---------------------------------

// The operators' autograd kernel: they are for inference. It stands above the device's kernels, where torch.func's transforms show
// their tensors too (below, those are plain ones); tangents count whether gradients are on or not, as torch.no_grad leaves them.
void no_gradients(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
    const bool grad = at::GradMode::is_enabled(), tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const c10::IValue& v : torch::jit::last(stack, op.schema().arguments().size())) {
        if (!v.isTensor() || !v.toTensor().defined()) continue;
        const at::Tensor& t = v.toTensor();
        if ((grad && t.requires_grad()) || (tangents && t._fw_grad(0).defined())) {
            const std::string& name = op.schema().name();
            TORCH_CHECK(false, name.substr(name.rfind(':') + 1),
                        ": no gradients; detach the inputs, or call it under torch.no_grad() where they have no tangents");
        }
    }
    op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

int64_t fp4_stages(int64_t k) { return (k + 255) / 256; }

// The strides of scales [..., stages, 8] whose stages are outermost in memory: those of `lead` rows of 8, the stages, 1
std::vector<int64_t> fp4_scale_strides(at::IntArrayRef lead, int64_t& rows) {
    std::vector<int64_t> v(lead.size() + 2);
    int64_t at = 8;
    for (size_t i = lead.size(); i-- > 0;) {
        v[i] = at;
        at *= lead[i];
    }
    v[lead.size()] = at;
    v[lead.size() + 1] = 1;
    rows = at / 8;
    return v;
}

// quantised rows of x's leading sizes and k columns: codes [..., kp / 2] and scales [..., stages, 8], the stages outermost in memory
std::tuple<at::Tensor, at::Tensor> fp4_rows_empty(const at::Tensor& x, int64_t k) {
    auto q = with_last(x.sizes(), fp8_up(k) / 2);
    auto sizes = x.sizes().vec();
    sizes.back() = fp4_stages(k);
    sizes.push_back(8);
    int64_t rows;
    const auto o = x.options().dtype(at::kByte);
    return {at::empty(q, o), at::empty_strided(sizes, fp4_scale_strides(x.sizes().slice(0, x.dim() - 1), rows), o)};
}

// Quantised rows as the C-ABI takes them (copies only where the strides or addresses do not fit)
struct Fp4Rows {
    at::Tensor q, s;
    int M = 0, kp = 0;
    int64_t s_stage = 0;
    Fp4Rows(const at::Tensor& q_, const at::Tensor& s_, const char* what) {
        TORCH_CHECK(q_.scalar_type() == at::kByte && q_.dim() >= 1 && q_.size(-1) > 0 && q_.size(-1) % 64 == 0 &&
                        q_.size(-1) <= INT32_MAX / 2 && q_.numel() / q_.size(-1) <= INT32_MAX,
                    what, ": q uint8 [..., a multiple of 64], got ", q_.scalar_type(), " ", q_.sizes());
        on_device_of(q_, s_, what);
        kp = (int)(2 * q_.size(-1));
        const int64_t d = q_.dim() - 1;
        TORCH_CHECK(s_.scalar_type() == at::kByte && s_.dim() == d + 2 && s_.size(d) == fp4_stages(kp) && s_.size(d + 1) == 8 &&
                        s_.sizes().slice(0, d) == q_.sizes().slice(0, d),
                    what, ": s uint8 [..., ", fp4_stages(kp), ", 8] with q's leading sizes, got ", s_.scalar_type(), " ", s_.sizes());
        q = q_.is_contiguous() ? q_ : q_.contiguous();
        if ((uintptr_t)q.const_data_ptr() % 16) q = q.clone();
        int64_t rows;
        const auto want = fp4_scale_strides(q_.sizes().slice(0, d), rows);
        M = (int)rows;
        const bool one = s_.size(d) == 1;
        bool fits = s_.stride(d + 1) == 1 && (one || (s_.stride(d) >= want[d] && s_.stride(d) % 8 == 0)) &&
                    (uintptr_t)s_.const_data_ptr() % 8 == 0;
        for (int64_t i = 0; i < d; ++i) fits = fits && (s_.size(i) == 1 || s_.stride(i) == want[i]);
        s = s_;
        if (!fits && M > 0) {
            s = at::empty_strided(s_.sizes(), want, s_.options());
            s.copy_(s_);
        }
        s_stage = one || M == 0 ? 8 * rows : s.stride(d);
    }
};

std::tuple<at::Tensor, at::Tensor> fp4_quant_meta(const at::Tensor& x) { return fp4_rows_empty(x, x.size(-1)); }
std::tuple<at::Tensor, at::Tensor> fp4_silu_mul_quant_meta(const at::Tensor& x) { return fp4_rows_empty(x, x.size(-1) / 2); }

std::tuple<at::Tensor, at::Tensor> fp4_quant(const at::Tensor& x) {
    const c10::DeviceGuard guard(x.device());
    const int dt = dtype_code(x);
    auto x2 = rows_of(x, "fp4_quant");
    auto out = fp4_rows_empty(x, x.size(-1));
    check(exl3_fp4_quant(x2.data_ptr(), dt, row_stride(x2), (int)x2.size(0), (int)x2.size(1), std::get<0>(out).data_ptr(),
                         std::get<1>(out).data_ptr(), 8 * x2.size(0), cur_stream(x)),
          "fp4_quant");
    return out;
}

std::tuple<at::Tensor, at::Tensor> fp4_silu_mul_quant(const at::Tensor& x) {
    const c10::DeviceGuard guard(x.device());
    const int dt = dtype_code(x);
    auto x2 = rows_of(x, "fp4_silu_mul_quant");
    TORCH_CHECK(x2.size(1) % 2 == 0, "fp4_silu_mul_quant: gate|up rows of an even size, got ", x.sizes());
    const int64_t k = x2.size(1) / 2;
    auto out = fp4_rows_empty(x, k);
    check(exl3_fp4_silu_mul_quant(x2.data_ptr(), dt, row_stride(x2), (int)x2.size(0), (int)k, std::get<0>(out).data_ptr(),
                                  std::get<1>(out).data_ptr(), 8 * x2.size(0), cur_stream(x)),
          "fp4_silu_mul_quant");
    return out;
}

at::Tensor fp4_dequant_meta(const at::Tensor& q, const at::Tensor&, int64_t k, at::ScalarType dtype) {
    return at::empty(with_last(q.sizes(), k), q.options().dtype(dtype));
}

at::Tensor fp4_dequant(const at::Tensor& q, const at::Tensor& s, int64_t k, at::ScalarType dtype) {
    const c10::DeviceGuard guard(q.device());
    const Fp4Rows r(q, s, "fp4_dequant");
    TORCH_CHECK(k > 0 && fp8_up(k) == r.kp, "fp4_dequant: rows of ", r.kp, " columns do not hold k=", k);
    auto out = fp4_dequant_meta(q, s, k, dtype);
    check(exl3_fp4_dequant(r.q.const_data_ptr(), r.s.const_data_ptr(), r.s_stage, r.M, (int)k, out.data_ptr(), dtype_code(out),
                           cur_stream(q)),
          "fp4_dequant");
    return out;
}

// weights [n, k] in the rows' form, laid out as the product takes them
void fp4_weight_checks(const at::Tensor& x, const at::Tensor& w, const at::Tensor& sw, int64_t k, const char* what) {
    on_device_of(x, w, what);
    on_device_of(x, sw, what);
    TORCH_CHECK(w.scalar_type() == at::kByte && w.dim() == 2 && w.is_contiguous() && w.size(1) == fp8_up(k) / 2 && w.size(0) > 0 &&
                    w.size(0) <= INT32_MAX,
                what, ": weight uint8 [n, ", fp8_up(k) / 2, "] contiguous, got ", w.scalar_type(), " ", w.sizes());
    TORCH_CHECK(sw.scalar_type() == at::kByte && sw.dim() == 3 && sw.size(0) == w.size(0) && sw.size(1) == fp4_stages(k) &&
                    sw.size(2) == 8 && sw.stride(2) == 1 && sw.stride(0) == 8 &&
                    (sw.size(1) == 1 || sw.stride(1) == 8 * sw.size(0)),
                what, ": weight_scale uint8 [", w.size(0), ", ", fp4_stages(k), ", 8] with the stages outermost in memory, got ",
                sw.scalar_type(), " ", sw.sizes());
}

at::Tensor fp4_linear_meta(const at::Tensor& x, const at::Tensor& w, const at::Tensor&, const std::optional<at::Tensor>&) {
    return at::empty(with_last(x.sizes(), w.size(0)), x.options());
}

at::Tensor fp4_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& sw, const std::optional<at::Tensor>& bias) {
    const c10::DeviceGuard guard(x.device());
    const int dt = dtype_code(x);
    auto x2 = rows_of(x, "fp4_linear");
    const int M = (int)x2.size(0), k = (int)x2.size(1);
    fp4_weight_checks(x, w, sw, k, "fp4_linear");
    const int64_t n = w.size(0);
    const float* b = f32_or_null(bias, x, n, "fp4_linear");
    auto out = fp4_linear_meta(x, w, sw, bias);
    if (M == 0) return out;
    const size_t ws = exl3_fp4_linear_workspace(M, k, (int)n);
    at::Tensor buf;
    if (ws) buf = at::empty({(int64_t)ws}, x.options().dtype(at::kByte));
    check(exl3_fp4_linear(x2.data_ptr(), dt, row_stride(x2), M, k, (int)n, w.const_data_ptr(), sw.const_data_ptr(), b,
                          out.data_ptr(), dt, n, ws ? buf.data_ptr() : nullptr, ws, cur_stream(x)),
          "fp4_linear");
    return out;
}

at::Tensor fp4_matmul_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor& w, const at::Tensor&,
                           const std::optional<at::Tensor>&, at::ScalarType dtype) {
    return at::empty(with_last(q.sizes(), w.size(0)), q.options().dtype(dtype));
}

at::Tensor fp4_matmul(const at::Tensor& q, const at::Tensor& s, const at::Tensor& w, const at::Tensor& sw,
                      const std::optional<at::Tensor>& bias, at::ScalarType dtype) {
    const c10::DeviceGuard guard(q.device());
    const Fp4Rows r(q, s, "fp4_matmul");
    fp4_weight_checks(q, w, sw, r.kp, "fp4_matmul");
    const int64_t n = w.size(0);
    const float* b = f32_or_null(bias, q, n, "fp4_matmul");
    auto out = fp4_matmul_meta(q, s, w, sw, bias, dtype);
    check(exl3_fp4_matmul(r.q.const_data_ptr(), r.s.const_data_ptr(), r.s_stage, r.M, r.kp, (int)n, w.const_data_ptr(),
                          sw.const_data_ptr(), b, out.data_ptr(), dtype_code(out), n, cur_stream(q)),
          "fp4_matmul");
    return out;
}

struct Fp4MlpSizes {
    int64_t I, n;
    const float *gb, *db;
    Fp4MlpSizes(const at::Tensor& x, int64_t k, int64_t I_, const at::Tensor& gu, const at::Tensor& gu_scale,
                const std::optional<at::Tensor>& gu_bias, const at::Tensor& dn, const at::Tensor& dn_scale,
                const std::optional<at::Tensor>& dn_bias, const char* what)
        : I(I_), n(dn.size(0)) {
        TORCH_CHECK(I > 0 && I <= (1 << 22), what, ": intermediate size ", I);
        fp4_weight_checks(x, gu, gu_scale, k, what);
        TORCH_CHECK(gu.size(0) == 2 * fp8_up(I), what, ": gate|up weights of ", 2 * fp8_up(I), " rows, got ", gu.sizes());
        fp4_weight_checks(x, dn, dn_scale, I, what);
        gb = f32_or_null(gu_bias, x, 2 * fp8_up(I), what);
        db = f32_or_null(dn_bias, x, n, what);
    }
};

at::Tensor fp4_mlp(const at::Tensor& x, int64_t I, const at::Tensor& gu, const at::Tensor& gu_scale,
                   const std::optional<at::Tensor>& gu_bias, const at::Tensor& dn, const at::Tensor& dn_scale,
                   const std::optional<at::Tensor>& dn_bias) {
    const c10::DeviceGuard guard(x.device());
    const int dt = dtype_code(x);
    auto x2 = rows_of(x, "fp4_mlp");
    const int M = (int)x2.size(0), k = (int)x2.size(1);
    const Fp4MlpSizes z(x, k, I, gu, gu_scale, gu_bias, dn, dn_scale, dn_bias, "fp4_mlp");
    auto out = at::empty(with_last(x.sizes(), z.n), x.options());
    if (M == 0) return out;
    const size_t ws = exl3_fp4_mlp_workspace(M, k, (int)I);
    auto buf = at::empty({(int64_t)ws}, x.options().dtype(at::kByte));
    check(exl3_fp4_mlp(x2.data_ptr(), dt, row_stride(x2), M, k, (int)I, (int)z.n, gu.const_data_ptr(), gu_scale.const_data_ptr(),
                       z.gb, dn.const_data_ptr(), dn_scale.const_data_ptr(), z.db, out.data_ptr(), dt, z.n, buf.data_ptr(), ws,
                       cur_stream(x)),
          "fp4_mlp");
    return out;
}

at::Tensor fp4_mlp_meta(const at::Tensor& x, int64_t, const at::Tensor&, const at::Tensor&, const std::optional<at::Tensor>&,
                        const at::Tensor& dn, const at::Tensor&, const std::optional<at::Tensor>&) {
    return at::empty(with_last(x.sizes(), dn.size(0)), x.options());
}

at::Tensor fp4_mlp_matmul(const at::Tensor& q, const at::Tensor& s, int64_t I, const at::Tensor& gu, const at::Tensor& gu_scale,
                          const std::optional<at::Tensor>& gu_bias, const at::Tensor& dn, const at::Tensor& dn_scale,
                          const std::optional<at::Tensor>& dn_bias, at::ScalarType dtype) {
    const c10::DeviceGuard guard(q.device());
    const Fp4Rows r(q, s, "fp4_mlp_matmul");
    const Fp4MlpSizes z(q, r.kp, I, gu, gu_scale, gu_bias, dn, dn_scale, dn_bias, "fp4_mlp_matmul");
    auto out = at::empty(with_last(q.sizes(), z.n), q.options().dtype(dtype));
    const int dt = dtype_code(out);
    if (r.M == 0) return out;
    const size_t ws = exl3_fp4_mlp_matmul_workspace(r.M, (int)I);
    auto buf = at::empty({(int64_t)ws}, q.options());
    check(exl3_fp4_mlp_matmul(r.q.const_data_ptr(), r.s.const_data_ptr(), r.s_stage, r.M, r.kp, (int)I, (int)z.n,
                              gu.const_data_ptr(), gu_scale.const_data_ptr(), z.gb, dn.const_data_ptr(), dn_scale.const_data_ptr(),
                              z.db, out.data_ptr(), dt, z.n, buf.data_ptr(), ws, cur_stream(q)),
          "fp4_mlp_matmul");
    return out;
}

at::Tensor fp4_mlp_matmul_meta(const at::Tensor& q, const at::Tensor&, int64_t, const at::Tensor&, const at::Tensor&,
                               const std::optional<at::Tensor>&, const at::Tensor& dn, const at::Tensor&,
                               const std::optional<at::Tensor>&, at::ScalarType dtype) {
    return at::empty(with_last(q.sizes(), dn.size(0)), q.options().dtype(dtype));
}

// form 0, 1 or 2 as exl3_rms_norm's, `rows`: y too. The outputs there are, in the order q, s, y, held
std::vector<at::Tensor> rms_norm_empty(const at::Tensor& x, const std::optional<at::Tensor>& residual, int64_t form, bool rows) {
    TORCH_CHECK(form >= 0 && form <= 2 && (form || rows), "rms_norm: form ", form, " without rows");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "rms_norm: [..., k] with k > 0, got ", x.sizes());
    std::vector<at::Tensor> out;
    if (form) {
        auto [q, s] = form == 1 ? fp8_rows_empty(x, x.size(-1)) : fp4_rows_empty(x, x.size(-1));
        out.push_back(q);
        out.push_back(s);
    }
    if (rows) out.push_back(at::empty(x.sizes(), x.options()));
    if (residual) out.push_back(at::empty(x.sizes(), residual->options()));
    return out;
}

std::vector<at::Tensor> rms_norm_meta(const at::Tensor& x, const std::optional<at::Tensor>& residual,
                                      const std::optional<at::Tensor>&, double, int64_t form, bool rows, bool) {
    return rms_norm_empty(x, residual, form, rows);
}

std::vector<at::Tensor> rms_norm(const at::Tensor& x, const std::optional<at::Tensor>& residual,
                                 const std::optional<at::Tensor>& weight, double eps, int64_t form, bool rows,
                                 bool unit_offset) {
    const c10::DeviceGuard guard(x.device());
    const int dt = dtype_code(x);
    auto out = rms_norm_empty(x, residual, form, rows);
    const int64_t k = x.size(-1);
    const float* w = f32_or_null(weight, x, k, "rms_norm (weight)");
    int rdt = dt;
    at::Tensor r2;
    if (residual) {
        on_device_of(x, *residual, "rms_norm");
        TORCH_CHECK(residual->sizes() == x.sizes(), "rms_norm: residual ", x.sizes(), ", got ", residual->sizes());
        rdt = dtype_code(*residual);
        TORCH_CHECK(rdt == dt || rdt == EXL3_DT_F32, "rms_norm: residual of x's dtype or fp32, got ", residual->scalar_type());
        r2 = rows_of(*residual, "rms_norm");
    }
    // rows inside wider ones ([tokens, heads, k] cut out of a fused projection) as they are: a stride within and one between
    at::Tensor x2;
    int64_t inner = 1, stride = 0, outer = 0;
    if (x.dim() == 3 && x.stride(2) == 1 && x.numel() > 0 && x.size(0) > 1 && x.size(1) > 1 && x.stride(1) >= k &&
        x.stride(0) != x.size(1) * x.stride(1) && x.stride(0) >= 0 && x.size(1) <= INT32_MAX && x.numel() / k <= INT32_MAX) {
        x2 = x;
        inner = x.size(1);
        stride = x.stride(1);
        outer = x.stride(0);
    } else {
        x2 = rows_of(x, "rms_norm");
        stride = row_stride(x2);
    }
    const int M = (int)(x.numel() / k);
    auto ptr = [&](size_t i) { return out[i].data_ptr(); };
    const size_t y = form ? 2 : 0, held = y + rows;
    check(exl3_rms_norm(x2.const_data_ptr(), dt, stride, (int)inner, outer, residual ? r2.const_data_ptr() : nullptr, rdt,
                        residual ? row_stride(r2) : 0, residual ? ptr(held) : nullptr, w, unit_offset, (float)eps, M, (int)k,
                        rows ? ptr(y) : nullptr, (int)form, form ? ptr(0) : nullptr, form ? ptr(1) : nullptr, 8 * (int64_t)M,
                        cur_stream(x)),
          "rms_norm");
    return out;
}

}  // namespace

TORCH_LIBRARY(exl3xpu_C, m) {
    m.def("linear(Tensor x, Tensor trellis, Tensor suh, Tensor svh, Tensor shard_of_nb, int[] group_bounds, int K, "
          "int cb, int small_m_max, int slice_n) -> Tensor");
    m.impl("linear", c10::DispatchKey::CUDA, &linear);
    m.impl("linear", c10::DispatchKey::Meta, &linear_meta);
    m.def("exl3_gemm_small(Tensor x, Tensor trellis, Tensor suh, Tensor svh, Tensor shard_of_nb, Tensor(a!) out, "
          "int K, int cb) -> ()");
    m.impl("exl3_gemm_small", c10::DispatchKey::CUDA, &gemm_small);
    m.def("exl3_supported(int K, int cb) -> bool", &linear_supported);
    m.def("exl3_set_int8(int on) -> ()", &set_int8);
    m.def("exl3_had_in_rm(Tensor x, Tensor suh, Tensor(a!) xh) -> ()");
    m.impl("exl3_had_in_rm", c10::DispatchKey::CUDA, &had_in_rm);
    m.def("exl3_had_out_h(Tensor y, Tensor svh, Tensor(a!) out) -> ()");
    m.impl("exl3_had_out_h", c10::DispatchKey::CUDA, &had_out_h);
    m.def("exl3_reconstruct(Tensor trellis, Tensor(a!) w, int n0, int K, int cb) -> ()");
    m.impl("exl3_reconstruct", c10::DispatchKey::CUDA, &reconstruct);
    m.def("fp8_quant(Tensor x) -> (Tensor q, Tensor s)");
    m.impl("fp8_quant", c10::DispatchKey::CUDA, &fp8_quant);
    m.impl("fp8_quant", c10::DispatchKey::Meta, &fp8_quant_meta);
    m.def("fp8_silu_mul_quant(Tensor gate_up) -> (Tensor q, Tensor s)");
    m.impl("fp8_silu_mul_quant", c10::DispatchKey::CUDA, &fp8_silu_mul_quant);
    m.impl("fp8_silu_mul_quant", c10::DispatchKey::Meta, &fp8_silu_mul_quant_meta);
    m.def("fp8_linear(Tensor x, Tensor weight, Tensor weight_scale, Tensor? bias=None) -> Tensor");
    m.impl("fp8_linear", c10::DispatchKey::CUDA, &fp8_linear);
    m.impl("fp8_linear", c10::DispatchKey::Meta, &fp8_linear_meta);
    m.def("fp8_mlp(Tensor x, Tensor gate_up, Tensor gate_up_scale, Tensor? gate_up_bias, Tensor down, Tensor down_scale, "
          "Tensor? down_bias) -> Tensor");
    m.impl("fp8_mlp", c10::DispatchKey::CUDA, &fp8_mlp);
    m.impl("fp8_mlp", c10::DispatchKey::Meta, &fp8_mlp_meta);
    m.def("fp8_matmul(Tensor q, Tensor s, Tensor weight, Tensor weight_scale, Tensor? bias, ScalarType dtype) -> Tensor");
    m.impl("fp8_matmul", c10::DispatchKey::CUDA, &fp8_matmul);
    m.impl("fp8_matmul", c10::DispatchKey::Meta, &fp8_matmul_meta);
    m.def("rms_norm(Tensor x, Tensor? residual, Tensor? weight, float eps, int form, bool rows, bool unit_offset=False) -> "
          "Tensor[]");
    m.impl("rms_norm", c10::DispatchKey::CUDA, &rms_norm);
    m.impl("rms_norm", c10::DispatchKey::Meta, &rms_norm_meta);
    m.def("fp4_quant(Tensor x) -> (Tensor q, Tensor s)");
    m.impl("fp4_quant", c10::DispatchKey::CUDA, &fp4_quant);
    m.impl("fp4_quant", c10::DispatchKey::Meta, &fp4_quant_meta);
    m.def("fp4_silu_mul_quant(Tensor gate_up) -> (Tensor q, Tensor s)");
    m.impl("fp4_silu_mul_quant", c10::DispatchKey::CUDA, &fp4_silu_mul_quant);
    m.impl("fp4_silu_mul_quant", c10::DispatchKey::Meta, &fp4_silu_mul_quant_meta);
    m.def("fp4_dequant(Tensor q, Tensor s, int k, ScalarType dtype) -> Tensor");
    m.impl("fp4_dequant", c10::DispatchKey::CUDA, &fp4_dequant);
    m.impl("fp4_dequant", c10::DispatchKey::Meta, &fp4_dequant_meta);
    m.def("fp4_linear(Tensor x, Tensor weight, Tensor weight_scale, Tensor? bias=None) -> Tensor");
    m.impl("fp4_linear", c10::DispatchKey::CUDA, &fp4_linear);
    m.impl("fp4_linear", c10::DispatchKey::Meta, &fp4_linear_meta);
    m.def("fp4_matmul(Tensor q, Tensor s, Tensor weight, Tensor weight_scale, Tensor? bias, ScalarType dtype) -> Tensor");
    m.impl("fp4_matmul", c10::DispatchKey::CUDA, &fp4_matmul);
    m.impl("fp4_matmul", c10::DispatchKey::Meta, &fp4_matmul_meta);
    m.def("fp4_mlp(Tensor x, int I, Tensor gate_up, Tensor gate_up_scale, Tensor? gate_up_bias, Tensor down, "
          "Tensor down_scale, Tensor? down_bias) -> Tensor");
    m.impl("fp4_mlp", c10::DispatchKey::CUDA, &fp4_mlp);
    m.impl("fp4_mlp", c10::DispatchKey::Meta, &fp4_mlp_meta);
    m.def("fp4_mlp_matmul(Tensor q, Tensor s, int I, Tensor gate_up, Tensor gate_up_scale, Tensor? gate_up_bias, Tensor down, "
          "Tensor down_scale, Tensor? down_bias, ScalarType dtype) -> Tensor");
    m.impl("fp4_mlp_matmul", c10::DispatchKey::CUDA, &fp4_mlp_matmul);
    m.impl("fp4_mlp_matmul", c10::DispatchKey::Meta, &fp4_mlp_matmul_meta);
    for (const char* name : {"rms_norm", "fp4_quant", "fp4_silu_mul_quant", "fp4_dequant", "fp4_linear", "fp4_matmul", "fp4_mlp",
                             "fp4_mlp_matmul"})
        m.impl(name, c10::DispatchKey::Autograd, torch::CppFunction::makeFromBoxedFunction<&no_gradients>());
}

TORCH_LIBRARY(exl3xpu_moe, m) {
    m.def("moe_forward(Tensor x, Tensor topk_ids, Tensor topk_w, Tensor ptrs, int I, int K, int n_experts) -> Tensor");
    m.impl("moe_forward", c10::DispatchKey::CUDA, &moe_forward);
    m.def("moe_forward_host(Tensor x, Tensor topk_ids, Tensor topk_w, Tensor ptrs, int I, int K, int n_experts, "
          "int hbm_base, int hbm_bytes) -> Tensor");
    m.impl("moe_forward_host", c10::DispatchKey::CUDA, &moe_forward_host);
    m.def("moe_forward_cached(Tensor x, Tensor(i!) topk_ids, Tensor(j!) topk_w, Tensor(a!) ptrs_all, int layer, "
          "Tensor(b!) slot_of, Tensor(c!) slot_key, Tensor(d!) slot_last, Tensor(e!) tick, Tensor host_base, "
          "int slot_base, Tensor(f!) fill_all, Tensor(g!) fill_list, int max_fill, int I, int K, int n_experts, "
          "Tensor(h!) pend, Tensor done_seq) -> Tensor");
    m.impl("moe_forward_cached", c10::DispatchKey::CUDA, &moe_forward_cached);
    m.def("moe_prefetch(Tensor ids, Tensor(a!) ptrs_all, int layer, Tensor(b!) slot_of, Tensor(c!) slot_key, "
          "Tensor(d!) slot_last, Tensor tick, Tensor host_base, int slot_base, Tensor(e!) pf_list, Tensor(f!) pf_slot, "
          "int max_fill, int n_experts, int blob) -> ()");
    m.impl("moe_prefetch", c10::DispatchKey::CUDA, &moe_prefetch);
    m.def("moe_prefetch_plan(Tensor ids, Tensor(a!) ptrs_all, int layer, Tensor(b!) slot_of, Tensor(c!) slot_key, "
          "Tensor(d!) slot_last, Tensor tick, Tensor host_base, int slot_base, Tensor(e!) pf_list, Tensor(f!) pf_slot, "
          "Tensor(g!) plans, Tensor(h!) plan_seq, Tensor(i!) pend, Tensor done_seq, int max_fill, int n_experts, "
          "int blob) -> ()");
    m.impl("moe_prefetch_plan", c10::DispatchKey::CUDA, &moe_prefetch_plan);
    m.def("moe_prefetch_worker_start(Tensor plans, Tensor host_base_cpu, int slot_base, int blob, Tensor ptrs_all, "
          "Tensor slot_last, Tensor commit_host, Tensor done_seq, int n_layers, int n_experts) -> ()",
          &moe_prefetch_worker_start);
    m.def("moe_prefetch_worker_stop() -> int[]", &moe_prefetch_worker_stop);
    m.def("moe_align(Tensor topk_ids, Tensor topk_w, int n_experts, int pad) -> Tensor[]");
    m.impl("moe_align", c10::DispatchKey::CUDA, &moe_align);
    m.def("moe_route(Tensor logits, Tensor? bias, int topk, str scoring, int n_group, int topk_group, bool renormalize, "
          "float scale) -> (Tensor ids, Tensor w)");
    m.impl("moe_route", c10::DispatchKey::CUDA, &moe_route);
    m.impl("moe_route", c10::DispatchKey::Meta, &moe_route_meta);
    m.def("host_alloc(int nbytes) -> Tensor", &host_alloc);
    m.def("usm_kind(int ptr) -> int", &usm_kind);
    m.def("memcpy_async(int dst, int src, int nbytes) -> ()", &memcpy_async);
    m.def("blob_bytes(int H, int I, int K) -> int", &blob_bytes);
    m.def("moe_set_splits(int gu_p, int dn_p) -> ()", &moe_set_splits);
    m.def("moe_set_mr(int mr) -> ()", &moe_set_mr);
    m.def("moe_set_debug(int v) -> ()", &moe_set_debug);
    m.def("moe_set_pair_max_m(int v) -> ()", &moe_set_pair_max_m);
    m.def("moe_set_prefill_min_m(int v) -> ()", &moe_set_prefill_min_m);
    m.def("moe_set_victims(Tensor v) -> ()", &moe_set_victims);
    m.def("moe_set_victim_ring(Tensor meta, Tensor sel, Tensor buf) -> ()", &moe_set_victim_ring);
    m.def("moe_set_tier(Tensor ram_res, Tensor miss, Tensor safe) -> ()", &moe_set_tier);
    m.def("moe_set_host_stride(int s) -> ()", &moe_set_host_stride);
    m.def("moe_set_slot_stride(int s) -> ()", &moe_set_slot_stride);
    m.def("moe_set_fused_ensure(int v) -> ()", &moe_set_fused_ensure);
    m.def("moe_svm_prefetch(Tensor ptrs, int nbytes, Tensor like) -> ()", &moe_svm_prefetch);
    m.def("moe_set_decision_log(Tensor buf) -> ()", &moe_set_decision_log);
    m.def("dequant(Tensor trellis, int k_tiles, int n_tiles, int K) -> Tensor");
    m.impl("dequant", c10::DispatchKey::CUDA, &dequant);
}
