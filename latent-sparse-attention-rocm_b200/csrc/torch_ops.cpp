// torch_ops.cpp - the hot-path operators as torch.library ops (namespace "lsa").
//
// A thin C++ layer over the C ABI (include/lsa_b200.h): each op checks its tensors, takes the
// workspace of the current (device, stream), and launches the library's kernels on
// at::cuda::getCurrentCUDAStream(). Registered ops (drop-ins for the reference's operators):
//   lsa::regroup(q, k) -> (index_queries, index_keys)        make_index_space, port/gates.py:50-59
//   lsa::select_fused(index_queries, positions, centroids, members, block, bpb, top_p, window,
//                     sink, top_k) -> (lists, lengths)          flat_select fused, pipeline.py:274-316
//                     (index_queries [R, d], or raw queries [R, Hq, D]: regroup fused in)
//   lsa::sparse_read(q, k, v, ids, lengths, scale) -> out     sparse_read_auto, read_kernel_tiled.py:147
//   lsa::shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths, scale) -> out
//   lsa::shared_prefix_attention_lse(the same) -> (out, lse)
//   lsa::scored_attention(q, k, v, lengths, scores, scale, k_prefix, v_prefix) -> (out, scores)
//   lsa::evict(k, v, scores, lengths, budget, window, sink, capacity)
//                     -> (k, v, scores, lengths, ids)            no reference counterpart
//   lsa::workspace_counters() -> Tensor[]                      the cached counter buffers and status words (checks)
// Meta implementations give FX / torch.compile the output shapes. Workspaces: scratch (any
// content) and int32 counters (zero at rest: the kernels that use them leave them zero) cached
// per (device, stream), grown on demand - the same contract as the C ABI's callers keep.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <cmath>
#include <map>
#include <mutex>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/lsa_b200.h"

namespace {

struct Workspace {
    at::Tensor scratch, counters;
};

std::mutex g_ws_mutex;
std::map<std::pair<int, cudaStream_t>, Workspace> g_ws;

Workspace& workspace(const at::Device& dev, cudaStream_t stream, int64_t scratch_bytes, int64_t n_counters) {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    Workspace& w = g_ws[{dev.index(), stream}];
    if (!w.scratch.defined() || w.scratch.numel() < scratch_bytes)
        w.scratch = at::empty({std::max<int64_t>(scratch_bytes, 256)}, at::TensorOptions().dtype(at::kByte).device(dev));
    if (!w.counters.defined() || w.counters.numel() < n_counters) {
        // a new buffer starts at zero; the old one (if any) is at rest (zero) by contract
        w.counters = at::zeros({std::max<int64_t>(n_counters, 64)}, at::TensorOptions().dtype(at::kInt).device(dev));
    }
    return w;
}

std::map<int, at::Tensor> g_status;  // under g_ws_mutex

// The word that the shared-prefix operators' bounded waits report to, one a device (kernels only ever set it,
// and it is read with the device idle). It is no ticket of another operator, and it neither moves nor is
// zeroed again, since captured calls keep its address: memory of its own, made and zeroed beside a
// capture that may be under way on the current stream (relaxed mode is for this).
int32_t* status_word(const at::Device& dev) {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    at::Tensor& word = g_status[dev.index()];
    if (!word.defined()) {
        void* p = nullptr;
        cudaStream_t aside = nullptr;
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
        cudaError_t rc = cudaMalloc(&p, sizeof(int32_t));
        if (rc == cudaSuccess) rc = cudaStreamCreateWithFlags(&aside, cudaStreamNonBlocking);
        if (rc == cudaSuccess) rc = cudaMemsetAsync(p, 0, sizeof(int32_t), aside);
        if (rc == cudaSuccess) rc = cudaStreamSynchronize(aside);
        if (aside != nullptr) cudaStreamDestroy(aside);
        if (rc != cudaSuccess && p != nullptr) cudaFree(p);
        C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
        C10_CUDA_CHECK(rc);
        word = at::from_blob(p, {1}, at::TensorOptions().dtype(at::kInt).device(dev));
    }
    return word.data_ptr<int32_t>();
}

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return 0;
        case at::kHalf: return 1;
        case at::kBFloat16: return 2;
        default: TORCH_CHECK(false, "lsa: expected fp32 / fp16 / bf16, got ", t);
    }
    return -1;
}

void check_rc(int rc, const char* what) {
    TORCH_CHECK(rc == 0, what, ": the C-ABI entry point returned status ", rc,
                rc == -1 ? " (arguments rejected)" : (rc == -2 ? " (CUDA launch failed)" : ""));
}

std::tuple<at::Tensor, at::Tensor> regroup_cuda(const at::Tensor& q_in, const at::Tensor& k_in) {
    TORCH_CHECK(q_in.is_cuda() && k_in.is_cuda(), "lsa::regroup is a CUDA kernel");
    TORCH_CHECK(q_in.dim() == 3 && k_in.dim() == 3 && q_in.size(0) == k_in.size(0) && q_in.size(2) == k_in.size(2),
                "lsa::regroup: q [T, Hq, D], k [T, Hkv, D]");
    TORCH_CHECK(q_in.scalar_type() == k_in.scalar_type(), "lsa::regroup: q and k share a dtype");
    c10::cuda::CUDAGuard guard(q_in.device());
    auto q = q_in.contiguous(), k = k_in.contiguous();
    const int64_t T = q.size(0), Hq = q.size(1), Hkv = k.size(1), D = q.size(2);
    TORCH_CHECK(Hq % Hkv == 0, "lsa::regroup: query heads must group evenly onto KV heads");
    auto opts = q.options().dtype(at::kFloat);
    auto iq = at::empty({T, Hkv * D}, opts), ik = at::empty({T, Hkv * D}, opts);
    if (T)
        check_rc(lsa_regroup(q.data_ptr(), k.data_ptr(), dtype_code(q.scalar_type()), T, Hq, Hkv, D,
                             iq.data_ptr<float>(), ik.data_ptr<float>(), at::cuda::getCurrentCUDAStream()),
                 "lsa::regroup");
    return {iq, ik};
}

std::tuple<at::Tensor, at::Tensor> select_fused_cuda(const at::Tensor& iq_arg, const at::Tensor& positions_in,
                                                     const at::Tensor& centroids_in, const at::Tensor& members_in,
                                                     int64_t block, int64_t bpb, int64_t top_p, int64_t window,
                                                     int64_t sink, int64_t top_k) {
    TORCH_CHECK(iq_arg.is_cuda() && positions_in.is_cuda() && centroids_in.is_cuda() && members_in.is_cuda(),
                "lsa::select_fused is a CUDA kernel");
    TORCH_CHECK(centroids_in.dim() == 2, "lsa::select_fused: centroids [N, d]");
    c10::cuda::CUDAGuard guard(iq_arg.device());
    const auto cdt = centroids_in.scalar_type();
    TORCH_CHECK(cdt == at::kBFloat16 || cdt == at::kFloat, "lsa::select_fused: bf16 or fp32 centroids");
    at::Tensor iq_in = iq_arg;
    if (iq_arg.dim() == 3) {
        // raw queries [R, Hq, D]: the index queries are built inside the decode select (one
        // launch); rows it does not take are regrouped first and go the two-dimensional way
        auto qr = iq_arg.contiguous();
        const int64_t R = qr.size(0), Hq = qr.size(1), D = qr.size(2), d = centroids_in.size(1);
        TORCH_CHECK(D > 0 && d % D == 0 && Hq % (d / D) == 0,
                    "lsa::select_fused: raw queries [R, Hq, D] need centroids of Hkv * D dims with Hq % Hkv == 0");
        TORCH_CHECK(positions_in.numel() == R, "lsa::select_fused: a position a query");
        const int64_t Hkv = d / D;
        auto c = centroids_in.contiguous();
        auto members = members_in.to(at::kInt).contiguous();
        auto pos = positions_in.to(at::kInt).contiguous();
        const int64_t width = top_k + window + sink;
        auto lists = at::empty({R, width}, qr.options().dtype(at::kInt));
        auto lengths = at::empty({R}, qr.options().dtype(at::kInt));
        if (R == 0) return {lists, lengths};
        auto stream = at::cuda::getCurrentCUDAStream();
        const int rc = lsa_select_fused_grouped(qr.data_ptr(), dtype_code(qr.scalar_type()), R, Hq, Hkv, D,
                                                c.data_ptr(), cdt == at::kFloat ? 0 : 2, c.size(0),
                                                pos.data_ptr<int32_t>(), block, bpb, members.data_ptr<int32_t>(),
                                                members.size(1), top_p, window, sink, top_k,
                                                lists.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(), stream);
        if (rc == LSA_OK) return {lists, lengths};
        TORCH_CHECK(rc == LSA_ERR_ARG, "lsa::select_fused: the C-ABI entry point returned status ", rc);
        iq_in = at::empty({R, d}, qr.options().dtype(at::kFloat));
        check_rc(lsa_regroup(qr.data_ptr(), nullptr, dtype_code(qr.scalar_type()), R, Hq, Hkv, D,
                             iq_in.data_ptr<float>(), nullptr, stream),
                 "lsa::select_fused");
    }
    TORCH_CHECK(iq_in.dim() == 2 && iq_in.size(1) == centroids_in.size(1),
                "lsa::select_fused: index_queries [R, d] (or raw queries [R, Hq, D]), centroids [N, d]");
    TORCH_CHECK(positions_in.numel() == iq_in.size(0), "lsa::select_fused: a position a query");
    at::Tensor q;
    int q_code;
    if (cdt == at::kFloat) {  // fp32 scoring
        q = iq_in.to(at::kFloat).contiguous();
        q_code = 0;
    } else if (iq_in.scalar_type() == at::kFloat) {  // bf16 scoring of fp32 queries, rounded in-kernel
        q = iq_in.contiguous();
        q_code = 3;
    } else {
        q = iq_in.to(at::kBFloat16).contiguous();
        q_code = 2;
    }
    auto c = centroids_in.contiguous();
    auto members = members_in.to(at::kInt).contiguous();
    auto pos = positions_in.to(at::kInt).contiguous();
    const int64_t R = q.size(0), d = q.size(1), N = c.size(0);
    const int64_t width = top_k + window + sink;
    auto lists = at::empty({R, width}, q.options().dtype(at::kInt));
    auto lengths = at::empty({R}, q.options().dtype(at::kInt));
    if (R == 0) return {lists, lengths};
    auto stream = at::cuda::getCurrentCUDAStream();
    Workspace& w = workspace(q.device(), stream, lsa_select_fused_scratch(R, N), R + 1);
    check_rc(lsa_select_fused(q.data_ptr(), q_code, R, d, c.data_ptr(), cdt == at::kFloat ? 0 : 2, N, d,
                              pos.data_ptr<int32_t>(), block, bpb, members.data_ptr<int32_t>(), members.size(1), top_p,
                              window, sink, top_k, lists.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(),
                              w.scratch.data_ptr(), w.scratch.numel(), w.counters.data_ptr<int32_t>(),
                              w.counters.numel(), -1, stream),
             "lsa::select_fused");
    return {lists, lengths};
}

at::Tensor sparse_read_cuda(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                            const at::Tensor& ids_in, const at::Tensor& lengths_in, double scale) {
    TORCH_CHECK(q_in.is_cuda() && k_in.is_cuda() && v_in.is_cuda(), "lsa::sparse_read is a CUDA kernel");
    TORCH_CHECK(q_in.dim() == 4 && k_in.dim() == 4 && v_in.sizes() == k_in.sizes(),
                "lsa::sparse_read: q [B, Tq, Hq, D], k / v [B, Tk, Hkv, D]");
    TORCH_CHECK(q_in.scalar_type() == k_in.scalar_type() && q_in.scalar_type() == v_in.scalar_type(),
                "lsa::sparse_read: q, k, v share a dtype");
    c10::cuda::CUDAGuard guard(q_in.device());
    auto q = q_in.contiguous(), k = k_in.contiguous(), v = v_in.contiguous();
    const int64_t B = q.size(0), Tq = q.size(1), Hq = q.size(2), D = q.size(3), Tk = k.size(1), Hkv = k.size(2);
    TORCH_CHECK(Hq % Hkv == 0, "lsa::sparse_read: query heads must group evenly onto KV heads");
    const int64_t width = ids_in.size(-1);
    auto ids = ids_in.reshape({-1, width}).to(at::kInt).contiguous();
    auto lens = lengths_in.reshape({-1}).to(at::kInt).contiguous();
    auto out = at::empty_like(q);
    if (B * Tq == 0) return out;
    int64_t splits = 0, scratch_bytes = 0, n_counters = 0;
    check_rc(lsa_sparse_read_plan(B, Tq, Hq, Hkv, D, width, 0, &splits, &scratch_bytes, &n_counters),
             "lsa::sparse_read");
    auto stream = at::cuda::getCurrentCUDAStream();
    Workspace& w = workspace(q.device(), stream, scratch_bytes, n_counters);
    check_rc(lsa_sparse_read(q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype_code(q.scalar_type()),
                             ids.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), B, Tq, Tk, Hq, Hkv, D, width,
                             (float)scale, out.data_ptr(), w.scratch.data_ptr(), w.scratch.numel(),
                             w.counters.data_ptr<int32_t>(), w.counters.numel(), 0, stream),
             "lsa::sparse_read");
    return out;
}

// a tensor whose last dimension is contiguous and whose rows start on 16-byte boundaries, a
// stride apart: as it is when it already is one (a cache's view is not copied), else a copy
at::Tensor rows16(const at::Tensor& t) {
    const int64_t unit = 16 / t.element_size();
    bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % unit == 0));
    if (ok) return t;
    auto c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

// stride of a dimension; 0 where the dimension has one entry and any stride would do
int64_t stride_of(const at::Tensor& t, int64_t i) { return t.size(i) == 1 ? 0 : t.stride(i); }

// an uninitialised tensor on a CUDA device, past the dispatcher (half a microsecond each)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const at::Device& dev) {
    return at::Tensor(at::detail::empty_cuda(sizes, dtype, dev, std::nullopt));
}

at::Tensor as_lengths(const at::Tensor& t) {
    return t.scalar_type() == at::kInt && t.is_contiguous() ? t : t.to(at::kInt).contiguous();
}

struct PrefixOut {
    at::Tensor out, lse, scores;
};

PrefixOut prefix_attention(const at::Tensor& q_in, const at::Tensor* kp_in, const at::Tensor* vp_in,
                           const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& lengths_in,
                           const at::Tensor* scores_in, double scale, bool want_lse, const char* what) {
    TORCH_CHECK_VALUE((kp_in == nullptr) == (vp_in == nullptr), what, ": a prefix has keys and values");
    for (const at::Tensor* t : {&q_in, kp_in, vp_in, &k_in, &v_in, &lengths_in})
        TORCH_CHECK_VALUE(t == nullptr || (t->is_cuda() && t->device() == q_in.device()), what,
                          " is a CUDA kernel (B200, sm_100a): every tensor on one CUDA device");
    TORCH_CHECK_VALUE(q_in.dim() == 4 && k_in.dim() == 4 && v_in.sizes() == k_in.sizes(), what,
                      ": q [B, Tq, Hq, D], k / v [B, T, Hkv, D]");
    TORCH_CHECK_VALUE(kp_in == nullptr || (kp_in->dim() == 3 && vp_in->sizes() == kp_in->sizes()), what,
                      ": k_prefix / v_prefix [P, Hkv, D]");
    const int64_t B = q_in.size(0), Tq = q_in.size(1), Hq = q_in.size(2), D = q_in.size(3);
    const int64_t T = k_in.size(1), Hkv = k_in.size(2), P = kp_in ? kp_in->size(0) : 0;
    TORCH_CHECK_VALUE(k_in.size(0) == B && k_in.size(3) == D &&
                          (kp_in == nullptr || (kp_in->size(1) == Hkv && kp_in->size(2) == D)),
                      what,
                      ": batch, KV heads and head dim of q, the prefix and the own caches differ");
    TORCH_CHECK_VALUE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 64, what,
                      ": query heads must group evenly onto KV heads, at most 64 to one");
    TORCH_CHECK_VALUE(D == 64 || D == 128, what, ": head dim 64 or 128, got ", D);
    for (const at::Tensor* t : {kp_in, vp_in, &k_in, &v_in})
        TORCH_CHECK_VALUE(t == nullptr || t->scalar_type() == q_in.scalar_type(), what, ": q, the prefix and the caches share a dtype");
    TORCH_CHECK_VALUE(q_in.scalar_type() == at::kFloat || q_in.scalar_type() == at::kHalf ||
                          q_in.scalar_type() == at::kBFloat16,
                      what, ": fp32, fp16 or bf16, got ", q_in.scalar_type());
    TORCH_CHECK_VALUE(lengths_in.numel() == B && !lengths_in.is_floating_point(), what, ": one whole length a sequence");
    const float scale_log2 = (float)scale * 1.4426950408889634f;  // as the entry point takes it
    TORCH_CHECK_VALUE(std::isfinite(scale_log2) && scale_log2 > 0, what, ": the scale must be positive, and with log2(e) within fp32, got ", scale);
    c10::cuda::CUDAGuard guard(q_in.device());
    auto q = rows16(q_in), k = rows16(k_in), v = rows16(v_in);
    at::Tensor kp, vp;
    if (P > 0) kp = rows16(*kp_in), vp = rows16(*vp_in);
    if (B > 1 && Tq > 1 && q.stride(0) != Tq * q.stride(1)) q = q.contiguous();  // tokens one stride apart
    auto lengths = as_lengths(lengths_in);
    PrefixOut r;
    r.out = fresh({B, Tq, Hq, D}, q.scalar_type(), q.device());
    if (want_lse) r.lse = fresh({B, Tq, Hq}, at::kFloat, q.device());
    at::Tensor scores;
    if (scores_in) {
        TORCH_CHECK_VALUE(scores_in->device() == q_in.device() && scores_in->scalar_type() == at::kFloat &&
                              scores_in->dim() == 3 && scores_in->size(0) == B && scores_in->size(1) == Hkv &&
                              scores_in->size(2) == T,
                          what, ": scores [B, Hkv, T] fp32");
        scores = scores_in->contiguous();
        r.scores = B * Tq == 0 ? scores.clone() : fresh({B, Hkv, T}, at::kFloat, q.device());
    }
    if (B * Tq == 0) return r;
    const int code = dtype_code(q.scalar_type());
    const int64_t bytes = lsa_shared_prefix_scratch(code, B, Tq, Hq, Hkv, D, P, T, scores_in != nullptr);
    TORCH_CHECK_VALUE(bytes >= 0, what, ": sizes out of range");
    auto stream = at::cuda::getCurrentCUDAStream();
    // The parts' scratch is the call's own: one kept for the stream would have to move when a larger call
    // comes, under the feet of a captured graph.
    auto scratch = fresh({bytes}, at::kByte, q.device());
    const int64_t strides[13] = {stride_of(q, 0), stride_of(q, 1), stride_of(q, 2), P ? stride_of(kp, 0) : 0,
                                 P ? stride_of(kp, 1) : 0, P ? stride_of(vp, 0) : 0, P ? stride_of(vp, 1) : 0,
                                 stride_of(k, 0), stride_of(k, 1),
                                 stride_of(k, 2), stride_of(v, 0), stride_of(v, 1), stride_of(v, 2)};
    check_rc(lsa_shared_prefix_attention(q.data_ptr(), P ? kp.data_ptr() : nullptr, P ? vp.data_ptr() : nullptr,
                                         k.data_ptr(), v.data_ptr(), code,
                                         strides, lengths.data_ptr<int32_t>(), B, Tq, Hq, Hkv, D, P, T, (float)scale,
                                         r.out.data_ptr(), want_lse ? r.lse.data_ptr<float>() : nullptr,
                                         scores_in ? scores.data_ptr<float>() : nullptr,
                                         scores_in ? r.scores.data_ptr<float>() : nullptr, scratch.data_ptr(), bytes,
                                         status_word(q.device()), stream),
             what);
    return r;
}

at::Tensor shared_prefix_cuda(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& k,
                              const at::Tensor& v, const at::Tensor& lengths, double scale) {
    return prefix_attention(q, &kp, &vp, k, v, lengths, nullptr, scale, false, "shared_prefix_attention").out;
}

std::tuple<at::Tensor, at::Tensor> shared_prefix_lse_cuda(const at::Tensor& q, const at::Tensor& kp,
                                                          const at::Tensor& vp, const at::Tensor& k,
                                                          const at::Tensor& v, const at::Tensor& lengths,
                                                          double scale) {
    auto r = prefix_attention(q, &kp, &vp, k, v, lengths, nullptr, scale, true, "shared_prefix_attention");
    return {r.out, r.lse};
}

std::tuple<at::Tensor, at::Tensor> scored_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                               const at::Tensor& lengths, const at::Tensor& scores, double scale,
                                               const std::optional<at::Tensor>& kp,
                                               const std::optional<at::Tensor>& vp) {
    auto r = prefix_attention(q, kp ? &*kp : nullptr, vp ? &*vp : nullptr, k, v, lengths, &scores, scale, false,
                              "scored_attention");
    return {r.out, r.scores};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> evict_cuda(
    const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& scores_in, const at::Tensor& lengths_in,
    int64_t budget, int64_t window, int64_t sink, int64_t capacity) {
    for (const at::Tensor* t : {&k_in, &v_in, &scores_in, &lengths_in})
        TORCH_CHECK_VALUE(t->is_cuda() && t->device() == k_in.device(),
                          "evict is a CUDA kernel (B200, sm_100a): every tensor on one CUDA device");
    TORCH_CHECK_VALUE(k_in.dim() == 4 && v_in.sizes() == k_in.sizes() && v_in.scalar_type() == k_in.scalar_type(),
                      "evict: k / v [B, T, Hkv, D] of one dtype");
    const int64_t B = k_in.size(0), T = k_in.size(1), Hkv = k_in.size(2), D = k_in.size(3), es = k_in.element_size();
    TORCH_CHECK_VALUE(Hkv > 0 && D > 0 && D * es % 16 == 0, "evict: rows of a multiple of 16 bytes, got ", D * es);
    TORCH_CHECK_VALUE(scores_in.scalar_type() == at::kFloat && scores_in.dim() == 3 && scores_in.size(0) == B &&
                          scores_in.size(1) == Hkv && scores_in.size(2) == T,
                      "evict: scores [B, Hkv, T] fp32");
    TORCH_CHECK_VALUE(lengths_in.numel() == B && !lengths_in.is_floating_point(), "evict: one whole length a sequence");
    TORCH_CHECK_VALUE(budget >= 0 && window >= 0 && sink >= 0 && window + sink <= budget && capacity >= budget,
                      "evict: window + sink (", window, " + ", sink, ") must fit the budget (", budget,
                      "), and the budget the capacity (", capacity, ")");
    c10::cuda::CUDAGuard guard(k_in.device());
    auto k = rows16(k_in), v = rows16(v_in);
    auto scores = scores_in.contiguous();
    auto lengths = as_lengths(lengths_in);
    const auto dev = k.device();
    auto ko = fresh({B, capacity, Hkv, D}, k.scalar_type(), dev), vo = fresh({B, capacity, Hkv, D}, k.scalar_type(), dev);
    auto so = fresh({B, Hkv, capacity}, at::kFloat, dev);
    auto lo = fresh({B}, at::kInt, dev), ids = fresh({B, Hkv, capacity}, at::kInt, dev);
    if (B == 0) return {ko, vo, so, lo, ids};
    const int64_t strides[6] = {stride_of(k, 0) * es, stride_of(k, 1) * es, stride_of(k, 2) * es,
                                stride_of(v, 0) * es, stride_of(v, 1) * es, stride_of(v, 2) * es};
    check_rc(lsa_evict(k.data_ptr(), v.data_ptr(), D * es, strides, scores.data_ptr<float>(),
                       lengths.data_ptr<int32_t>(), B, T, Hkv, budget, window, sink, capacity, ko.data_ptr(),
                       vo.data_ptr(), so.data_ptr<float>(), lo.data_ptr<int32_t>(), ids.data_ptr<int32_t>(),
                       at::cuda::getCurrentCUDAStream()),
             "evict");
    return {ko, vo, so, lo, ids};
}

std::vector<at::Tensor> workspace_counters() {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    std::vector<at::Tensor> out;
    for (auto& kv : g_ws)
        if (kv.second.counters.defined()) out.push_back(kv.second.counters);
    for (auto& kv : g_status)
        if (kv.second.defined()) out.push_back(kv.second);
    return out;
}

// ------------------------------------------------------------------ shapes (Meta)

std::tuple<at::Tensor, at::Tensor> regroup_meta(const at::Tensor& q, const at::Tensor& k) {
    auto opts = q.options().dtype(at::kFloat);
    return {at::empty({q.size(0), k.size(1) * k.size(2)}, opts), at::empty({q.size(0), k.size(1) * k.size(2)}, opts)};
}

std::tuple<at::Tensor, at::Tensor> select_fused_meta(const at::Tensor& iq, const at::Tensor&, const at::Tensor&,
                                                     const at::Tensor&, int64_t, int64_t, int64_t, int64_t window,
                                                     int64_t sink, int64_t top_k) {
    auto opts = iq.options().dtype(at::kInt);
    return {at::empty({iq.size(0), top_k + window + sink}, opts), at::empty({iq.size(0)}, opts)};
}

at::Tensor sparse_read_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            const at::Tensor&, double) {
    return at::empty_like(q);
}

at::Tensor shared_prefix_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                              const at::Tensor&, const at::Tensor&, double) {
    return at::empty(q.sizes(), q.options());
}

std::tuple<at::Tensor, at::Tensor> shared_prefix_lse_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&,
                                                          const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                          double) {
    return {at::empty(q.sizes(), q.options()),
            at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat))};
}

std::tuple<at::Tensor, at::Tensor> scored_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&,
                                               const at::Tensor&, const at::Tensor& scores, double,
                                               const std::optional<at::Tensor>&, const std::optional<at::Tensor>&) {
    return {at::empty(q.sizes(), q.options()), at::empty(scores.sizes(), scores.options())};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> evict_meta(
    const at::Tensor& k, const at::Tensor&, const at::Tensor& scores, const at::Tensor& lengths, int64_t, int64_t,
    int64_t, int64_t capacity) {
    auto i32 = lengths.options().dtype(at::kInt);
    const int64_t B = k.size(0), Hkv = k.size(2);
    auto ko = at::empty({B, capacity, Hkv, k.size(3)}, k.options());
    return {ko, at::empty_like(ko), at::empty({B, Hkv, capacity}, scores.options()), at::empty({B}, i32),
            at::empty({B, Hkv, capacity}, i32)};
}

}  // namespace

TORCH_LIBRARY(lsa, m) {
    m.def("regroup(Tensor q, Tensor k) -> (Tensor, Tensor)");
    m.def("select_fused(Tensor index_queries, Tensor positions, Tensor centroids, Tensor members, int block, int bpb, "
          "int top_p, int window, int sink, int top_k) -> (Tensor, Tensor)");
    m.def("sparse_read(Tensor q, Tensor k, Tensor v, Tensor ids, Tensor lengths, float scale) -> Tensor");
    m.def("shared_prefix_attention(Tensor q, Tensor k_prefix, Tensor v_prefix, Tensor k, Tensor v, Tensor lengths, "
          "float scale) -> Tensor");
    m.def("shared_prefix_attention_lse(Tensor q, Tensor k_prefix, Tensor v_prefix, Tensor k, Tensor v, "
          "Tensor lengths, float scale) -> (Tensor, Tensor)");
    m.def("scored_attention(Tensor q, Tensor k, Tensor v, Tensor lengths, Tensor scores, float scale, "
          "Tensor? k_prefix=None, Tensor? v_prefix=None) -> (Tensor, Tensor)");
    m.def("evict(Tensor k, Tensor v, Tensor scores, Tensor lengths, int budget, int window, int sink, int capacity) "
          "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("workspace_counters() -> Tensor[]", &workspace_counters);
}

TORCH_LIBRARY_IMPL(lsa, CUDA, m) {
    m.impl("regroup", &regroup_cuda);
    m.impl("select_fused", &select_fused_cuda);
    m.impl("sparse_read", &sparse_read_cuda);
    m.impl("shared_prefix_attention", &shared_prefix_cuda);
    m.impl("shared_prefix_attention_lse", &shared_prefix_lse_cuda);
    m.impl("scored_attention", &scored_cuda);
    m.impl("evict", &evict_cuda);
}

// CPU tensors: the operators' own refusal (a ValueError) in place of the dispatcher's
TORCH_LIBRARY_IMPL(lsa, CPU, m) {
    m.impl("shared_prefix_attention", &shared_prefix_cuda);
    m.impl("shared_prefix_attention_lse", &shared_prefix_lse_cuda);
    m.impl("scored_attention", &scored_cuda);
    m.impl("evict", &evict_cuda);
}

TORCH_LIBRARY_IMPL(lsa, Meta, m) {
    m.impl("regroup", &regroup_meta);
    m.impl("select_fused", &select_fused_meta);
    m.impl("sparse_read", &sparse_read_meta);
    m.impl("shared_prefix_attention", &shared_prefix_meta);
    m.impl("shared_prefix_attention_lse", &shared_prefix_lse_meta);
    m.impl("scored_attention", &scored_meta);
    m.impl("evict", &evict_meta);
}
