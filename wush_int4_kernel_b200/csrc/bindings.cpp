// Python operator surface `my_int4._C`: the same 16 callables, argument names, shapes,
// dtypes and error type (RuntimeError) as the reference's csrc/bindings.cpp:28-68, each a
// thin wrapper over the C ABI of include/wush_int4.h.  The wrappers validate, allocate the
// outputs (and scratch) through torch's caching allocator, pick the current stream and
// launch -- no host synchronisation, so every op can be captured in a CUDA Graph.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <vector>

#include "../../include/wush_int4.h"

namespace {

void check_status(int status, const char* op)
{
    TORCH_CHECK(status == WUSH_OK, op, ": ", wush_last_error(), " (status ", status, ")");
}

cudaStream_t stream_of(const torch::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

void check_bf16_cuda(const torch::Tensor& t, const char* name)
{
    TORCH_CHECK(t.is_cuda() && t.is_contiguous(), name, " must be a contiguous CUDA tensor");
    TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bf16");
}

std::vector<int64_t> with_last(const torch::Tensor& t, int64_t last)
{
    std::vector<int64_t> s = t.sizes().vec();
    s.back() = last;
    return s;
}

// ---- a1 -------------------------------------------------------------------------------
std::vector<torch::Tensor> quant_int4(torch::Tensor x)
{
    check_bf16_cuda(x, "x");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) % 32 == 0, "last dim must be multiple of 32");
    const at::cuda::OptionalCUDAGuard guard(x.device());
    const int64_t K = x.size(-1);
    auto q = torch::empty(with_last(x, K / 2), x.options().dtype(torch::kUInt8));
    auto s = torch::empty(with_last(x, K / 32), x.options());
    check_status(wush_quant_int4(x.data_ptr(), x.numel() / 32, q.data_ptr<uint8_t>(), s.data_ptr(), stream_of(x)),
                 "quant_int4");
    return {q, s};
}

// ---- a4..a7 ---------------------------------------------------------------------------
std::vector<torch::Tensor> fused_tq(torch::Tensor x, torch::Tensor t, int variant, const char* op)
{
    TORCH_CHECK(x.is_cuda() && x.is_contiguous() && t.is_cuda() && t.is_contiguous(),
                "x/t must be contiguous CUDA tensors");
    TORCH_CHECK(x.scalar_type() == torch::kBFloat16 && t.scalar_type() == torch::kBFloat16, "x/t must be bf16");
    TORCH_CHECK(x.dim() >= 1 && t.dim() == 3, "T must be (K/32, 32, 32)");
    const int64_t K = x.size(-1), C = K / 32;
    TORCH_CHECK(K % 32 == 0 && t.size(0) == C && t.size(1) == 32 && t.size(2) == 32, "T must be (K/32, 32, 32)");
    TORCH_CHECK(x.device() == t.device(), "x and t must be on the same device");
    const at::cuda::OptionalCUDAGuard guard(x.device());
    const int64_t rows = K ? x.numel() / K : 0;
    auto q = torch::empty(with_last(x, K / 2), x.options().dtype(torch::kUInt8));
    auto s = torch::empty(with_last(x, C), x.options());
    check_status(wush_fused_transform_quant_int4(x.data_ptr(), t.data_ptr(), rows, K, variant, q.data_ptr<uint8_t>(),
                                                 s.data_ptr(), stream_of(x)),
                 op);
    return {q, s};
}
std::vector<torch::Tensor> fused_transform_quant_int4(torch::Tensor x, torch::Tensor t)
{
    return fused_tq(x, t, WUSH_TQ_EXACT, "fused_transform_quant_int4");
}
// Addition to the reference surface: SiLU(gate) * up -> bf16 -> transform -> quantise in one pass
// over the fp16 output of a fused gate+up projection (gate half first).
std::vector<torch::Tensor> fused_silu_mul_transform_quant_int4(torch::Tensor gate_up, torch::Tensor t)
{
    TORCH_CHECK(gate_up.is_cuda() && gate_up.is_contiguous() && t.is_cuda() && t.is_contiguous(),
                "gate_up/t must be contiguous CUDA tensors");
    TORCH_CHECK(gate_up.scalar_type() == torch::kHalf && t.scalar_type() == torch::kBFloat16,
                "gate_up must be fp16, t bf16");
    TORCH_CHECK(gate_up.dim() >= 1 && t.dim() == 3 && gate_up.size(-1) % 64 == 0, "gate_up must be (..., 2K), K % 32 == 0");
    const int64_t K = gate_up.size(-1) / 2, C = K / 32;
    TORCH_CHECK(t.size(0) == C && t.size(1) == 32 && t.size(2) == 32, "T must be (K/32, 32, 32)");
    TORCH_CHECK(gate_up.device() == t.device(), "gate_up and t must be on the same device");
    const at::cuda::OptionalCUDAGuard guard(gate_up.device());
    const int64_t rows = gate_up.numel() / (2 * K);
    auto q = torch::empty(with_last(gate_up, K / 2), gate_up.options().dtype(torch::kUInt8));
    auto s = torch::empty(with_last(gate_up, C), gate_up.options().dtype(torch::kBFloat16));
    check_status(wush_fused_silu_mul_transform_quant_int4(gate_up.data_ptr(), t.data_ptr(), rows, K, q.data_ptr<uint8_t>(),
                                                          s.data_ptr(), stream_of(gate_up)),
                 "fused_silu_mul_transform_quant_int4");
    return {q, s};
}
std::vector<torch::Tensor> fused_transform_quant_int4_wmma(torch::Tensor x, torch::Tensor t)
{
    return fused_tq(x, t, WUSH_TQ_FAST, "fused_transform_quant_int4_wmma");
}
std::vector<torch::Tensor> fused_transform_quant_int4_v3(torch::Tensor x, torch::Tensor t)
{
    return fused_tq(x, t, WUSH_TQ_FAST, "fused_transform_quant_int4_v3");
}
std::vector<torch::Tensor> fused_transform_quant_int4_smallm(torch::Tensor x, torch::Tensor t)
{
    TORCH_CHECK(x.numel() >= 1, "rows must be >= 1");
    return fused_tq(x, t, WUSH_TQ_FAST, "fused_transform_quant_int4_smallm");
}

// ---- a8..a10 --------------------------------------------------------------------------
struct GemmArgs {
    int64_t M, N, K;
};

GemmArgs check_gemm(const torch::Tensor& xq, const torch::Tensor& xs, const torch::Tensor& wq, const torch::Tensor& ws)
{
    TORCH_CHECK(xq.is_cuda() && wq.is_cuda() && xs.is_cuda() && ws.is_cuda(), "tensors must be CUDA");
    TORCH_CHECK(xq.scalar_type() == torch::kUInt8 && wq.scalar_type() == torch::kUInt8, "packed tensors must be uint8");
    TORCH_CHECK(xs.scalar_type() == torch::kBFloat16 && ws.scalar_type() == torch::kBFloat16, "scales must be bf16");
    TORCH_CHECK(xq.is_contiguous() && xs.is_contiguous() && wq.is_contiguous() && ws.is_contiguous(),
                "tensors must be contiguous");
    TORCH_CHECK(wq.dim() == 2, "w must be 2D (N, K/2)");
    TORCH_CHECK(xq.dim() >= 1 && xs.dim() >= 1 && ws.dim() >= 1, "tensors must have at least one dimension");
    const int64_t K2 = xq.size(-1), K = K2 * 2, G = K / 32;
    TORCH_CHECK(K % 32 == 0, "K must be a multiple of 32");
    TORCH_CHECK(wq.size(1) == K2 && ws.size(-1) == G && xs.size(-1) == G, "K mismatch between x/w tensors");
    const int64_t M = K2 ? xq.numel() / K2 : 0, N = wq.size(0);
    TORCH_CHECK(xs.numel() == M * G && ws.numel() == N * G, "scale tensors do not match the packed tensors");
    TORCH_CHECK(xq.device() == wq.device() && xq.device() == xs.device() && xq.device() == ws.device(),
                "tensors must be on the same device");
    return {M, N, K};
}

torch::Tensor run_gemm(const torch::Tensor& xq, const torch::Tensor& xs, const torch::Tensor& wq,
                       const torch::Tensor& ws, const GemmArgs& a, std::vector<int64_t> yshape, int variant,
                       const char* op)
{
    const at::cuda::OptionalCUDAGuard guard(xq.device());
    auto y = torch::empty(yshape, xq.options().dtype(torch::kHalf));
    const size_t wbytes = wush_w4a4_gemm_workspace_bytes(a.M, a.N, a.K, variant);
    torch::Tensor work;
    if (wbytes) work = torch::empty({(int64_t)wbytes}, xq.options().dtype(torch::kUInt8));
    check_status(wush_w4a4_gemm(xq.data_ptr<uint8_t>(), xs.data_ptr(), wq.data_ptr<uint8_t>(), ws.data_ptr(), a.M, a.N,
                                a.K, y.data_ptr(), variant, wbytes ? work.data_ptr() : nullptr, wbytes, stream_of(xq)),
                 op);
    return y;
}

// v0 keeps the leading dimensions of x (reference csrc/gemm_int4.cu:128-129).
torch::Tensor w4a4_gemm(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws)
{
    auto a = check_gemm(xq, xs, wq, ws);
    return run_gemm(xq, xs, wq, ws, a, with_last(xq, a.N), WUSH_GEMM_AUTO, "w4a4_gemm");
}
// v1 / v2 / s4 return a 2-D (M, N) tensor (reference csrc/gemm_wmma.cu:171, csrc/gemm_s4.cu:378).
torch::Tensor w4a4_gemm_v1(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws)
{
    auto a = check_gemm(xq, xs, wq, ws);
    return run_gemm(xq, xs, wq, ws, a, {a.M, a.N}, WUSH_GEMM_AUTO, "w4a4_gemm_v1");
}
torch::Tensor w4a4_gemm_v2(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws)
{
    auto a = check_gemm(xq, xs, wq, ws);
    TORCH_CHECK(a.K % 64 == 0, "K must be multiple of 64");
    return run_gemm(xq, xs, wq, ws, a, {a.M, a.N}, WUSH_GEMM_AUTO, "w4a4_gemm_v2");
}
torch::Tensor w4a4_gemm_s4(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws)
{
    auto a = check_gemm(xq, xs, wq, ws);
    TORCH_CHECK(a.K % 64 == 0, "K must be multiple of 64");
    return run_gemm(xq, xs, wq, ws, a, {a.M, a.N}, WUSH_GEMM_AUTO, "w4a4_gemm_s4");
}

// ---- a9 -------------------------------------------------------------------------------
torch::Tensor w4a4_gemv(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws)
{
    TORCH_CHECK(xq.dim() >= 1 && xq.dim() <= 2 && xq.numel() == xq.size(-1), "gemv expects a single row");
    auto a = check_gemm(xq, xs, wq, ws);
    return run_gemm(xq, xs, wq, ws, a, {a.N}, WUSH_GEMM_AUTO, "w4a4_gemv");
}
// The reference accepts 1 <= M <= 8 (csrc/gemv_int4.cu:160); this build takes up to 32 rows.
torch::Tensor w4a4_gemv_multi(torch::Tensor xq, torch::Tensor xs, torch::Tensor wq, torch::Tensor ws)
{
    auto a = check_gemm(xq, xs, wq, ws);
    TORCH_CHECK(a.M >= 1 && a.M <= 32, "gemv_multi expects 1<=M<=32");
    return run_gemm(xq, xs, wq, ws, a, {a.M, a.N}, WUSH_GEMM_AUTO, "w4a4_gemv_multi");
}

// ---- a11 ------------------------------------------------------------------------------
torch::Tensor s4_atom_selftest(torch::Tensor a, torch::Tensor b)
{
    TORCH_CHECK(a.is_cuda() && b.is_cuda() && a.is_contiguous() && b.is_contiguous(), "a/b must be contiguous CUDA tensors");
    TORCH_CHECK(a.scalar_type() == torch::kInt8 && b.scalar_type() == torch::kInt8, "a/b must be int8");
    TORCH_CHECK(a.numel() == 8 * 32 && b.numel() == 32 * 8, "a must be (8,32) and b (32,8)");
    const at::cuda::OptionalCUDAGuard guard(a.device());
    auto c = torch::zeros({8, 8}, a.options().dtype(torch::kInt32));
    check_status(wush_i8_atom_selftest(a.data_ptr<int8_t>(), b.data_ptr<int8_t>(), c.data_ptr<int32_t>(), stream_of(a)),
                 "s4_atom_selftest");
    return c;
}

// Exact per-group partial sums P[m][n][g] from the tensor-core path (test-only addition).
torch::Tensor w4a4_group_partials(torch::Tensor xq, torch::Tensor wq)
{
    TORCH_CHECK(xq.is_cuda() && wq.is_cuda() && xq.is_contiguous() && wq.is_contiguous(), "tensors must be contiguous CUDA");
    TORCH_CHECK(xq.scalar_type() == torch::kUInt8 && wq.scalar_type() == torch::kUInt8, "packed tensors must be uint8");
    TORCH_CHECK(wq.dim() == 2 && xq.dim() >= 1 && xq.size(-1) == wq.size(1), "K mismatch");
    const int64_t K2 = wq.size(1), K = K2 * 2, M = xq.numel() / K2, N = wq.size(0);
    TORCH_CHECK(K % 32 == 0, "K must be a multiple of 32");
    const at::cuda::OptionalCUDAGuard guard(xq.device());
    auto P = torch::empty({M, N, K / 32}, xq.options().dtype(torch::kInt32));
    check_status(wush_group_partials(xq.data_ptr<uint8_t>(), wq.data_ptr<uint8_t>(), M, N, K, P.data_ptr<int32_t>(),
                                     stream_of(xq)),
                 "w4a4_group_partials");
    return P;
}

// ---- per-tensor route -----------------------------------------------------------------
torch::Tensor quant_int4_tensor_scale(torch::Tensor x, double scale)
{
    TORCH_CHECK(x.is_cuda() && x.is_contiguous() && x.scalar_type() == torch::kBFloat16, "x must be contiguous CUDA bf16");
    TORCH_CHECK(x.numel() % 32 == 0, "numel must be multiple of 32");
    const at::cuda::OptionalCUDAGuard guard(x.device());
    auto q = torch::empty({x.numel() / 2}, x.options().dtype(torch::kUInt8));
    const float inv = (float)(1.0 / scale);              // same rounding as the reference host code
    check_status(wush_quant_int4_tensor_scale(x.data_ptr(), x.numel(), inv, nullptr, q.data_ptr<uint8_t>(), stream_of(x)),
                 "quant_int4_tensor_scale");
    return q;
}
torch::Tensor quant_int4_tensor_scale_dev(torch::Tensor x, torch::Tensor inv_scale)
{
    TORCH_CHECK(x.is_cuda() && x.is_contiguous() && x.scalar_type() == torch::kBFloat16, "x must be contiguous CUDA bf16");
    TORCH_CHECK(x.numel() % 32 == 0, "numel must be multiple of 32");
    TORCH_CHECK(inv_scale.is_cuda() && inv_scale.scalar_type() == torch::kFloat32 && inv_scale.is_contiguous() &&
                    inv_scale.numel() == 1,
                "inv_scale must be 1-elem contiguous fp32 CUDA tensor");
    const at::cuda::OptionalCUDAGuard guard(x.device());
    auto q = torch::empty({x.numel() / 2}, x.options().dtype(torch::kUInt8));
    check_status(wush_quant_int4_tensor_scale(x.data_ptr(), x.numel(), 0.f, inv_scale.data_ptr<float>(),
                                              q.data_ptr<uint8_t>(), stream_of(x)),
                 "quant_int4_tensor_scale_dev");
    return q;
}

torch::Tensor gemm_ts(torch::Tensor xq, torch::Tensor wq, float alpha, const float* alpha_dev, const char* op)
{
    TORCH_CHECK(xq.is_cuda() && wq.is_cuda(), "tensors must be CUDA");
    TORCH_CHECK(xq.scalar_type() == torch::kUInt8 && wq.scalar_type() == torch::kUInt8, "packed tensors must be uint8");
    TORCH_CHECK(xq.is_contiguous() && wq.is_contiguous(), "tensors must be contiguous");
    TORCH_CHECK(wq.dim() == 2, "w must be 2D (N, K/2)");
    const int64_t K2 = wq.size(1);                       // K comes from wq; xq may be flat
    TORCH_CHECK(K2 > 0 && (K2 * 2) % 32 == 0, "K must be a multiple of 32");
    const int64_t M = xq.numel() / K2, N = wq.size(0);
    TORCH_CHECK(M * K2 == xq.numel(), "xq numel must equal M*K/2 (K from wq)");
    const at::cuda::OptionalCUDAGuard guard(xq.device());
    auto y = torch::empty({M, N}, xq.options().dtype(torch::kHalf));
    const size_t nbytes = wush_w4a4_gemm_tensor_scale_workspace_bytes(M, N, K2 * 2);
    torch::Tensor work;
    if (nbytes) work = torch::empty({(int64_t)nbytes}, xq.options());
    check_status(wush_w4a4_gemm_tensor_scale_ws(xq.data_ptr<uint8_t>(), wq.data_ptr<uint8_t>(), M, N, K2 * 2, alpha, alpha_dev,
                                                y.data_ptr(), nbytes ? work.data_ptr() : nullptr, nbytes, stream_of(xq)),
                 op);
    return y;
}
torch::Tensor w4a4_gemm_cutlass(torch::Tensor xq, torch::Tensor wq, double alpha)
{
    return gemm_ts(xq, wq, (float)alpha, nullptr, "w4a4_gemm_cutlass");
}
torch::Tensor w4a4_gemm_cutlass_dev(torch::Tensor xq, torch::Tensor wq, torch::Tensor alpha)
{
    TORCH_CHECK(alpha.is_cuda() && alpha.scalar_type() == torch::kFloat32 && alpha.is_contiguous() && alpha.numel() == 1,
                "alpha must be 1-elem contiguous fp32 CUDA tensor");
    return gemm_ts(xq, wq, 0.f, alpha.data_ptr<float>(), "w4a4_gemm_cutlass_dev");
}

// ---- 8-bit layers ---------------------------------------------------------------------
// An uninitialised tensor on the device of `like`, straight from the allocator: these operators take a few microseconds, of
// which a dispatched torch::empty would be one and a half.
torch::Tensor new_like(at::IntArrayRef sizes, torch::ScalarType dtype, const torch::Tensor& like)
{
    return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

int dtype_code(const torch::Tensor& t, const char* op, const char* name, bool with_f32)
{
    const auto d = t.scalar_type();
    if (d == torch::kBFloat16) return WUSH_BF16;
    if (d == torch::kHalf) return WUSH_F16;
    TORCH_CHECK(with_f32 && d == torch::kFloat32, op, ": ", name, with_f32 ? " must be bf16, fp16 or fp32" : " must be bf16 or fp16");
    return WUSH_F32;
}

// A contiguous CUDA tensor on the device of `like`.
void check_on(const torch::Tensor& t, const torch::Tensor& like, const char* op, const char* name)
{
    TORCH_CHECK(t.is_cuda() && t.is_contiguous(), op, ": ", name, " must be a contiguous CUDA tensor");
    TORCH_CHECK(t.device() == like.device(), op, ": tensors must be on the same device");
}

void check_type(const torch::Tensor& t, torch::ScalarType d, const char* op, const char* name)
{
    TORCH_CHECK(t.scalar_type() == d, op, ": ", name, " must be ", d);
}

int64_t rows_of(const torch::Tensor& t) { return t.size(-1) ? t.numel() / t.size(-1) : 0; }

std::vector<int64_t> without_last(const torch::Tensor& t)
{
    std::vector<int64_t> s = t.sizes().vec();
    s.pop_back();
    return s;
}

std::vector<torch::Tensor> quant_int8(const torch::Tensor& x)
{
    check_on(x, x, "quant_int8", "x");
    const int dt = dtype_code(x, "quant_int8", "x", true);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) % 16 == 0, "quant_int8: last dim must be a multiple of 16");
    const at::cuda::OptionalCUDAGuard guard(x.device());
    auto q = new_like(x.sizes(), torch::kInt8, x);
    auto s = new_like(without_last(x), torch::kFloat32, x);
    check_status(wush_quant_int8(x.data_ptr(), dt, rows_of(x), x.size(-1), q.data_ptr<int8_t>(), s.data_ptr<float>(), stream_of(x)),
                 "quant_int8");
    return {q, s};
}

// Codes (..., K) with their scales (...).
void check_codes(const torch::Tensor& q, const torch::Tensor& s, const torch::Tensor& like, const char* op, const char* qn, const char* sn)
{
    check_on(q, like, op, qn);
    check_on(s, like, op, sn);
    check_type(q, torch::kInt8, op, qn);
    check_type(s, torch::kFloat32, op, sn);
    TORCH_CHECK(q.dim() >= 1 && q.sizes().slice(0, q.dim() - 1) == s.sizes(), op, ": ", sn, " must have the shape of ", qn,
                " without its last dimension");
}

const float* check_bias(const c10::optional<torch::Tensor>& bias, const torch::Tensor& like, int64_t N, const char* op)
{
    if (!bias.has_value()) return nullptr;
    check_on(*bias, like, op, "bias");
    check_type(*bias, torch::kFloat32, op, "bias");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N, op, ": bias must be (N)");
    return bias->data_ptr<float>();
}

// Scratch of a product of 8-bit codes; undefined where none is needed.
torch::Tensor product_scratch(int64_t rows, int64_t experts, const torch::Tensor& like, size_t* nbytes)
{
    *nbytes = wush_w8a8_gemm_workspace_bytes(rows, experts);
    return *nbytes ? new_like({(int64_t)*nbytes}, torch::kUInt8, like) : torch::Tensor();
}
void* ptr_or_null(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

int out_code(torch::ScalarType d, const char* op)
{
    TORCH_CHECK(d == torch::kHalf || d == torch::kBFloat16 || d == torch::kFloat32, op,
                ": out_dtype must be torch.float16, torch.bfloat16 or torch.float32");
    return d == torch::kHalf ? WUSH_F16 : d == torch::kBFloat16 ? WUSH_BF16 : WUSH_F32;
}

torch::Tensor w8a8_gemm(const torch::Tensor& xq, const torch::Tensor& xs, const torch::Tensor& wq, const torch::Tensor& ws, const c10::optional<torch::Tensor>& bias,
                        torch::ScalarType out_dtype)
{
    const char* op = "w8a8_gemm";
    check_codes(xq, xs, xq, op, "xq", "xs");
    check_codes(wq, ws, xq, op, "wq", "ws");
    TORCH_CHECK(wq.dim() == 2, op, ": wq must be (N, K)");
    const int64_t N = wq.size(0), K = wq.size(1);
    TORCH_CHECK(K > 0 && xq.size(-1) == K, op, ": K mismatch between xq and wq");
    const int code = out_code(out_dtype, op);
    const at::cuda::OptionalCUDAGuard guard(xq.device());
    auto y = new_like(with_last(xq, N), out_dtype, xq);
    size_t nbytes;
    auto work = product_scratch(xq.numel() / K, 1, xq, &nbytes);
    check_status(wush_w8a8_gemm(xq.data_ptr<int8_t>(), xs.data_ptr<float>(), wq.data_ptr<int8_t>(), ws.data_ptr<float>(),
                                check_bias(bias, xq, N, op), xq.numel() / K, N, K, y.data_ptr(), code, ptr_or_null(work), nbytes,
                                stream_of(xq)),
                 op);
    return y;
}

torch::Tensor w8a8_linear(const torch::Tensor& x, const torch::Tensor& wq, const torch::Tensor& ws, const c10::optional<torch::Tensor>& bias)
{
    const char* op = "w8a8_linear";
    check_on(x, x, op, "x");
    const int dt = dtype_code(x, op, "x", false);
    check_codes(wq, ws, x, op, "wq", "ws");
    TORCH_CHECK(wq.dim() == 2 && x.dim() >= 1, op, ": wq must be (N, K)");
    const int64_t N = wq.size(0), K = wq.size(1);
    TORCH_CHECK(K > 0 && x.size(-1) == K, op, ": K mismatch between x and wq");
    const int64_t M = x.numel() / K;
    const at::cuda::OptionalCUDAGuard guard(x.device());
    auto y = new_like(with_last(x, N), x.scalar_type(), x);
    const size_t nbytes = wush_w8a8_linear_workspace_bytes(M, K);
    auto work = new_like({(int64_t)nbytes}, torch::kUInt8, x);
    check_status(wush_w8a8_linear(x.data_ptr(), dt, wq.data_ptr<int8_t>(), ws.data_ptr<float>(), check_bias(bias, x, N, op), M, N, K,
                                  y.data_ptr(), work.data_ptr(), nbytes, stream_of(x)),
                 op);
    return y;
}

// ---- tokens ordered by expert -----------------------------------------------------------
int id_bytes_of(const torch::Tensor& ids, const char* op)
{
    TORCH_CHECK(ids.scalar_type() == torch::kInt32 || ids.scalar_type() == torch::kInt64, op, ": ids must be int32 or int64");
    return ids.scalar_type() == torch::kInt64 ? 8 : 4;
}

struct Route {
    int64_t tokens, k, experts;
};

Route check_route(const torch::Tensor& pos, const torch::Tensor& offsets, const torch::Tensor& like, const char* op)
{
    check_on(pos, like, op, "pos");
    check_on(offsets, like, op, "offsets");
    check_type(pos, torch::kInt32, op, "pos");
    check_type(offsets, torch::kInt32, op, "offsets");
    TORCH_CHECK(pos.dim() == 2 && pos.size(1) >= 1, op, ": pos must be (tokens, k)");
    TORCH_CHECK(offsets.dim() == 1 && offsets.size(0) >= 2, op, ": offsets must be (experts + 1)");
    return {pos.size(0), pos.size(1), offsets.size(0) - 1};
}

std::vector<torch::Tensor> expert_sort(const torch::Tensor& ids, int64_t n_experts)
{
    const char* op = "expert_sort";
    check_on(ids, ids, op, "ids");
    const int bytes = id_bytes_of(ids, op);
    TORCH_CHECK(ids.dim() == 2, op, ": ids must be (tokens, k)");
    TORCH_CHECK(n_experts >= 1 && n_experts <= WUSH_EXPERT_MAX, op, ": takes 1..", WUSH_EXPERT_MAX, " experts (got ", n_experts, ")");
    const at::cuda::OptionalCUDAGuard guard(ids.device());
    auto pos = new_like(ids.sizes(), torch::kInt32, ids);
    auto offsets = new_like({n_experts + 1}, torch::kInt32, ids);
    check_status(wush_expert_sort(ids.data_ptr(), bytes, ids.size(0), ids.size(1), n_experts, pos.data_ptr<int32_t>(),
                                  offsets.data_ptr<int32_t>(), stream_of(ids)),
                 op);
    return {pos, offsets};
}

torch::Tensor expert_gather(const torch::Tensor& x, const torch::Tensor& pos, const torch::Tensor& offsets)
{
    const char* op = "expert_gather";
    check_on(x, x, op, "x");
    const int dt = dtype_code(x, op, "x", true);
    const Route r = check_route(pos, offsets, x, op);
    TORCH_CHECK(x.dim() == 2 && x.size(0) == r.tokens && x.size(1) >= 1, op, ": x must be (tokens, H) with the tokens of pos");
    const at::cuda::OptionalCUDAGuard guard(x.device());
    auto rows = new_like({r.tokens * r.k, x.size(1)}, x.scalar_type(), x);
    check_status(wush_expert_gather(x.data_ptr(), dt, r.tokens, x.size(1), pos.data_ptr<int32_t>(), r.k, offsets.data_ptr<int32_t>(),
                                    r.experts, rows.data_ptr(), stream_of(x)),
                 op);
    return rows;
}

std::vector<torch::Tensor> expert_gather_quant_int8(const torch::Tensor& x, const torch::Tensor& pos, const torch::Tensor& offsets)
{
    const char* op = "expert_gather_quant_int8";
    check_on(x, x, op, "x");
    const int dt = dtype_code(x, op, "x", true);
    const Route r = check_route(pos, offsets, x, op);
    TORCH_CHECK(x.dim() == 2 && x.size(0) == r.tokens && x.size(1) > 0 && x.size(1) % 16 == 0, op,
                ": x must be (tokens, K) with the tokens of pos, K a multiple of 16");
    const at::cuda::OptionalCUDAGuard guard(x.device());
    auto q = new_like({r.tokens * r.k, x.size(1)}, torch::kInt8, x);
    auto s = new_like({r.tokens * r.k}, torch::kFloat32, x);
    check_status(wush_expert_gather_quant_int8(x.data_ptr(), dt, r.tokens, x.size(1), pos.data_ptr<int32_t>(), r.k,
                                               offsets.data_ptr<int32_t>(), r.experts, q.data_ptr<int8_t>(), s.data_ptr<float>(),
                                               stream_of(x)),
                 op);
    return {q, s};
}

void check_weights(const torch::Tensor& w, const torch::Tensor& pos, const torch::Tensor& like, const char* op)
{
    check_on(w, like, op, "weights");
    check_type(w, torch::kFloat32, op, "weights");
    TORCH_CHECK(w.sizes() == pos.sizes(), op, ": weights must be (tokens, k)");
}

torch::Tensor expert_combine(const torch::Tensor& rows, const torch::Tensor& pos, const c10::optional<torch::Tensor>& weights,
                             c10::optional<torch::ScalarType> out_dtype)
{
    const char* op = "expert_combine";
    check_on(rows, rows, op, "rows");
    const int dt = dtype_code(rows, op, "rows", true);
    check_on(pos, rows, op, "pos");
    check_type(pos, torch::kInt32, op, "pos");
    TORCH_CHECK(pos.dim() == 2 && pos.size(1) >= 1, op, ": pos must be (tokens, k)");
    TORCH_CHECK(rows.dim() == 2 && rows.size(0) == pos.numel() && rows.size(1) >= 1, op, ": rows must be (tokens * k, H)");
    if (weights.has_value()) check_weights(*weights, pos, rows, op);
    const torch::ScalarType out = out_dtype.value_or(rows.scalar_type());
    TORCH_CHECK(out == rows.scalar_type() || dt == WUSH_F32, op, ": out_dtype must be the type of rows unless that is fp32");
    const int code = out_code(out, op);
    const at::cuda::OptionalCUDAGuard guard(rows.device());
    auto y = new_like({pos.size(0), rows.size(1)}, out, rows);
    check_status(wush_expert_combine(rows.data_ptr(), dt, code, pos.size(0), rows.size(1), pos.data_ptr<int32_t>(), pos.size(1),
                                     weights.has_value() ? weights->data_ptr<float>() : nullptr, y.data_ptr(), stream_of(rows)),
                 op);
    return y;
}

std::vector<torch::Tensor> expert_combine_grad(const torch::Tensor& dy, const torch::Tensor& rows, const torch::Tensor& pos, const torch::Tensor& offsets,
                                               const torch::Tensor& weights)
{
    const char* op = "expert_combine_grad";
    check_on(rows, rows, op, "rows");
    const int dt = dtype_code(rows, op, "rows", true);
    check_on(dy, rows, op, "dy");
    check_type(dy, rows.scalar_type(), op, "dy");
    const Route r = check_route(pos, offsets, rows, op);
    TORCH_CHECK(rows.dim() == 2 && rows.size(0) == r.tokens * r.k && rows.size(1) >= 1, op, ": rows must be (tokens * k, H)");
    TORCH_CHECK(dy.dim() == 2 && dy.size(0) == r.tokens && dy.size(1) == rows.size(1), op, ": dy must be (tokens, H)");
    check_weights(weights, pos, rows, op);
    const at::cuda::OptionalCUDAGuard guard(rows.device());
    auto d_rows = new_like(rows.sizes(), rows.scalar_type(), rows);
    auto d_weights = new_like(weights.sizes(), weights.scalar_type(), weights);
    check_status(wush_expert_combine_grad(dy.data_ptr(), rows.data_ptr(), dt, r.tokens, rows.size(1), pos.data_ptr<int32_t>(), r.k,
                                          offsets.data_ptr<int32_t>(), r.experts, weights.data_ptr<float>(), d_rows.data_ptr(),
                                          d_weights.data_ptr<float>(), stream_of(rows)),
                 op);
    return {d_rows, d_weights};
}

struct Grouped {
    int64_t rows, experts, N, K;
};

Grouped check_grouped(const torch::Tensor& xq, const torch::Tensor& xs, const torch::Tensor& wq, const torch::Tensor& ws,
                      const torch::Tensor& offsets, const char* op)
{
    check_codes(xq, xs, xq, op, "xq", "xs");
    check_codes(wq, ws, xq, op, "wq", "ws");
    check_on(offsets, xq, op, "offsets");
    check_type(offsets, torch::kInt32, op, "offsets");
    TORCH_CHECK(xq.dim() == 2 && wq.dim() == 3 && xq.size(1) > 0 && xq.size(1) == wq.size(2), op, ": xq must be (rows, K), wq (experts, N, K)");
    TORCH_CHECK(offsets.dim() == 1 && offsets.size(0) == wq.size(0) + 1, op, ": offsets must be (experts + 1)");
    return {xq.size(0), wq.size(0), wq.size(1), xq.size(1)};
}

torch::Tensor w8a8_grouped_gemm(const torch::Tensor& xq, const torch::Tensor& xs, const torch::Tensor& wq, const torch::Tensor& ws, const torch::Tensor& offsets,
                                torch::ScalarType out_dtype)
{
    const char* op = "w8a8_grouped_gemm";
    const Grouped g = check_grouped(xq, xs, wq, ws, offsets, op);
    const int code = out_code(out_dtype, op);
    const at::cuda::OptionalCUDAGuard guard(xq.device());
    auto y = new_like({g.rows, g.N}, out_dtype, xq);
    size_t nbytes;
    auto work = product_scratch(g.rows, g.experts, xq, &nbytes);
    check_status(wush_w8a8_grouped_gemm(xq.data_ptr<int8_t>(), xs.data_ptr<float>(), wq.data_ptr<int8_t>(), ws.data_ptr<float>(),
                                        offsets.data_ptr<int32_t>(), g.rows, g.experts, g.N, g.K, y.data_ptr(), code,
                                        ptr_or_null(work), nbytes, stream_of(xq)),
                 op);
    return y;
}

torch::Tensor w8a8_grouped_gated(const torch::Tensor& xq, const torch::Tensor& xs, const torch::Tensor& wq, const torch::Tensor& ws, const torch::Tensor& offsets)
{
    const char* op = "w8a8_grouped_gated";
    const Grouped g = check_grouped(xq, xs, wq, ws, offsets, op);
    TORCH_CHECK(g.N % 2 == 0, op, ": wq must be (experts, 2 * I, K), the gate channels first");
    const at::cuda::OptionalCUDAGuard guard(xq.device());
    auto h = new_like({g.rows, g.N / 2}, torch::kFloat32, xq);
    size_t nbytes;
    auto work = product_scratch(g.rows, g.experts, xq, &nbytes);
    check_status(wush_w8a8_grouped_gated(xq.data_ptr<int8_t>(), xs.data_ptr<float>(), wq.data_ptr<int8_t>(), ws.data_ptr<float>(),
                                         offsets.data_ptr<int32_t>(), g.rows, g.experts, g.N / 2, g.K, h.data_ptr<float>(),
                                         ptr_or_null(work), nbytes, stream_of(xq)),
                 op);
    return h;
}

torch::Tensor w8a8_expert_ffn(const torch::Tensor& x, const torch::Tensor& ids, const torch::Tensor& weights, const torch::Tensor& w13q, const torch::Tensor& w13s,
                              const torch::Tensor& w2q, const torch::Tensor& w2s)
{
    const char* op = "w8a8_expert_ffn";
    check_on(x, x, op, "x");
    const int dt = dtype_code(x, op, "x", false);
    check_on(ids, x, op, "ids");
    const int bytes = id_bytes_of(ids, op);
    TORCH_CHECK(x.dim() == 2 && ids.dim() == 2 && ids.size(0) == x.size(0) && ids.size(1) >= 1, op,
                ": x must be (tokens, H) and ids (tokens, k)");
    check_weights(weights, ids, x, op);
    check_codes(w13q, w13s, x, op, "w13q", "w13s");
    check_codes(w2q, w2s, x, op, "w2q", "w2s");
    const int64_t T = x.size(0), H = x.size(1), k = ids.size(1);
    TORCH_CHECK(w13q.dim() == 3 && w13q.size(2) == H && w13q.size(1) % 2 == 0, op, ": w13q must be (experts, 2 * I, H)");
    const int64_t E = w13q.size(0), I = w13q.size(1) / 2;
    TORCH_CHECK(w2q.dim() == 3 && w2q.size(0) == E && w2q.size(1) == H && w2q.size(2) == I, op, ": w2q must be (experts, H, I)");
    const at::cuda::OptionalCUDAGuard guard(x.device());
    auto y = new_like(x.sizes(), x.scalar_type(), x);
    const size_t nbytes = wush_w8a8_expert_ffn_workspace_bytes(T, H, I, E, k);
    auto work = new_like({(int64_t)nbytes}, torch::kUInt8, x);
    check_status(wush_w8a8_expert_ffn(x.data_ptr(), dt, ids.data_ptr(), bytes, weights.data_ptr<float>(), w13q.data_ptr<int8_t>(),
                                      w13s.data_ptr<float>(), w2q.data_ptr<int8_t>(), w2s.data_ptr<float>(), T, H, I, E, k, y.data_ptr(),
                                      work.data_ptr(), nbytes, stream_of(x)),
                 op);
    return y;
}

void init() { check_status(wush_init(), "init"); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("quant_int4_tensor_scale", &quant_int4_tensor_scale, "Per-tensor INT4 quantise, host scale", py::arg("x"),
          py::arg("scale"));
    m.def("quant_int4_tensor_scale_dev", &quant_int4_tensor_scale_dev,
          "Per-tensor INT4 quantise, inv_scale read from a 1-element fp32 device tensor (graph-safe)", py::arg("x"),
          py::arg("inv_scale"));
    m.def("quant_int4", &quant_int4, "sigma-clip INT4 group quantise (G=32, bf16 scales)", py::arg("x"));
    m.def("w4a4_gemm", &w4a4_gemm, "W4A4 group-scaled product, keeps leading dims", py::arg("xq"), py::arg("xs"),
          py::arg("wq"), py::arg("ws"));
    m.def("w4a4_gemm_v1", &w4a4_gemm_v1, "W4A4 group-scaled product (alias of the current kernels)", py::arg("xq"),
          py::arg("xs"), py::arg("wq"), py::arg("ws"));
    m.def("w4a4_gemm_cutlass", &w4a4_gemm_cutlass, "W4A4 product with one scalar scale", py::arg("xq"), py::arg("wq"),
          py::arg("alpha"));
    m.def("w4a4_gemm_cutlass_dev", &w4a4_gemm_cutlass_dev,
          "W4A4 product with one scalar scale read from a 1-element fp32 device tensor (graph-safe)", py::arg("xq"),
          py::arg("wq"), py::arg("alpha"));
    m.def("w4a4_gemm_s4", &w4a4_gemm_s4, "W4A4 group-scaled product (main entry)", py::arg("xq"), py::arg("xs"),
          py::arg("wq"), py::arg("ws"));
    m.def("s4_atom_selftest", &s4_atom_selftest, "(8,32)x(32,8) int8 -> int32 through one tensor-core atom");
    m.def("w4a4_gemv", &w4a4_gemv, "W4A4 GEMV (one activation row)", py::arg("xq"), py::arg("xs"), py::arg("wq"),
          py::arg("ws"));
    m.def("w4a4_gemv_multi", &w4a4_gemv_multi, "W4A4 GEMV, 1<=M<=32", py::arg("xq"), py::arg("xs"), py::arg("wq"),
          py::arg("ws"));
    m.def("fused_transform_quant_int4_v3", &fused_transform_quant_int4_v3, "Fused WUSH transform + INT4 quantise (fast)",
          py::arg("x"), py::arg("t"));
    m.def("fused_transform_quant_int4_smallm", &fused_transform_quant_int4_smallm,
          "Fused WUSH transform + INT4 quantise (decode shapes)", py::arg("x"), py::arg("t"));
    m.def("fused_silu_mul_transform_quant_int4", &fused_silu_mul_transform_quant_int4,
          "SiLU(gate) * up -> bf16 -> WUSH transform + INT4 quantise, from the fp16 (..., 2K) gate+up output",
          py::arg("gate_up"), py::arg("t"));
    m.def("fused_transform_quant_int4", &fused_transform_quant_int4,
          "Fused WUSH transform + INT4 quantise (bit-exact serial arithmetic)", py::arg("x"), py::arg("t"));
    m.def("w4a4_gemm_v2", &w4a4_gemm_v2, "W4A4 group-scaled product (alias of the current kernels)", py::arg("xq"),
          py::arg("xs"), py::arg("wq"), py::arg("ws"));
    m.def("fused_transform_quant_int4_wmma", &fused_transform_quant_int4_wmma,
          "Fused WUSH transform + INT4 quantise (tensor-core transform)", py::arg("x"), py::arg("t"));
    // 8-bit layers and experts
    m.def("quant_int8", &quant_int8, "rows to int8 codes with one fp32 scale per row (bf16 / fp16 / fp32 input)", py::arg("x"));
    m.def("w8a8_gemm", &w8a8_gemm, "W8A8 product with scales per token and channel, keeps leading dims", py::arg("xq"), py::arg("xs"),
          py::arg("wq"), py::arg("ws"), py::arg("bias") = py::none(), py::arg("out_dtype") = torch::kHalf);
    m.def("w8a8_linear", &w8a8_linear, "quant_int8 of x, then w8a8_gemm; the result has the type of x", py::arg("x"), py::arg("wq"),
          py::arg("ws"), py::arg("bias") = py::none());
    m.def("expert_sort", &expert_sort, "(tokens, k) expert ids -> row of each entry sorted by expert, first row of each expert",
          py::arg("ids"), py::arg("n_experts"));
    m.def("expert_gather", &expert_gather, "rows[pos[t, j]] = x[t]; rows behind the last entry are zero", py::arg("x"), py::arg("pos"),
          py::arg("offsets"));
    m.def("expert_gather_quant_int8", &expert_gather_quant_int8, "quant_int8 of x, then expert_gather of codes and scales", py::arg("x"),
          py::arg("pos"), py::arg("offsets"));
    m.def("expert_combine", &expert_combine, "y[t] = sum_j weights[t, j] * rows[pos[t, j]] (weights None: ones)", py::arg("rows"),
          py::arg("pos"), py::arg("weights") = py::none(), py::arg("out_dtype") = py::none());
    m.def("expert_combine_grad", &expert_combine_grad, "gradients of expert_combine: (d_rows, d_weights)", py::arg("dy"),
          py::arg("rows"), py::arg("pos"), py::arg("offsets"), py::arg("weights"));
    m.def("w8a8_grouped_gemm", &w8a8_grouped_gemm, "w8a8_gemm of each expert's rows with its weights", py::arg("xq"), py::arg("xs"),
          py::arg("wq"), py::arg("ws"), py::arg("offsets"), py::arg("out_dtype") = torch::kHalf);
    m.def("w8a8_grouped_gated", &w8a8_grouped_gated, "silu(gate) * up of each expert's rows in fp32, gate channels first", py::arg("xq"),
          py::arg("xs"), py::arg("wq"), py::arg("ws"), py::arg("offsets"));
    m.def("w8a8_expert_ffn", &w8a8_expert_ffn, "mixture-of-experts feed-forward block on 8-bit weights", py::arg("x"), py::arg("ids"),
          py::arg("weights"), py::arg("w13q"), py::arg("w13s"), py::arg("w2q"), py::arg("w2s"));
    // additions of this build
    m.def("w4a4_group_partials", &w4a4_group_partials, "exact int32 partial sums per group (test op)", py::arg("xq"),
          py::arg("wq"));
    m.def("init", &init, "one-time per-device set-up; call before CUDA Graph capture");
}
