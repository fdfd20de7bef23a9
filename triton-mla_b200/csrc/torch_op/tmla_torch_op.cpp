// The decode registered as a PyTorch operator, torch.ops.triton_mla.decode, on top of the C ABI
// (include/triton_mla_b200.h, tmla_decode), and the int8 projections (quantize_int8, rms_norm_int8,
// linear_int8) beside it.
//
// The reference runs its decode as Python code around two Triton launches
// (src/triton_mla/kernel.py:204-323), which torch.compile treats as opaque Python.  Here the
// whole call is one operator with a CUDA kernel and a Meta kernel: torch.compile traces a
// function that calls mla_decode (with an explicit num_splits) into one graph without a
// break, and CUDA-graph capture records the launches.  The Python wrapper (triton_mla.kernel)
// keeps the reference's argument checks and calls this operator.
//
// Schema: decode(q [B, H, D], kv_cache [N, P, D], cache_seqlens int32 [B], block_table int32
// [B, W] or None, out [B, H, Dv] (written), lse fp32 [B, H] (written), num_splits, softmax_scale,
// kernel (TMLA_KERNEL_*), q_len, status int32 [1], or None for the library's own word) -> ().  The
// split workspace comes from the caching allocator on the current stream; the launches go on the
// current stream.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "triton_mla_b200.h"

namespace {

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return TMLA_DTYPE_BF16;
    case at::kHalf: return TMLA_DTYPE_FP16;
    case at::kFloat: return TMLA_DTYPE_FP32;
    default: TORCH_CHECK(false, "triton_mla.decode: q must be bfloat16, float16 or float32, got ", t);
  }
  return -1;
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == TMLA_OK, what, " failed: ", tmla_error_string(rc), " ",
              rc == TMLA_ERR_CUDA ? tmla_last_cuda_error() : "");
}

// The caller's status word, or the library's on the current device (what read_status reads: a call without one, as
// torch.compile makes them, must not lose a timed-out wait).
int32_t* status_word(const std::optional<at::Tensor>& status) {
  if (status.has_value()) return status->data_ptr<int32_t>();
  int32_t* word = nullptr;
  check_rc(tmla_status_word(&word), "tmla_status_word");
  return word;
}

void decode_cuda(const at::Tensor& q, const at::Tensor& kv, const at::Tensor& lens,
                 const std::optional<at::Tensor>& block_table, const at::Tensor& out, const at::Tensor& lse,
                 int64_t num_splits, double softmax_scale, int64_t kernel, int64_t q_len,
                 const std::optional<at::Tensor>& status) {
  TORCH_CHECK(q.dim() == 3 && kv.dim() == 3, "triton_mla.decode: q [B, H, D] and kv_cache [N, P, D]");
  TORCH_CHECK(q.is_cuda() && kv.is_cuda() && lens.is_cuda() && out.is_cuda() && lse.is_cuda(),
              "triton_mla.decode: CUDA tensors only (there is no CPU implementation)");
  TORCH_CHECK(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.stride(0) == 1,
              "triton_mla.decode: cache_seqlens must be a contiguous int32 vector");
  TORCH_CHECK(lse.scalar_type() == at::kFloat && out.scalar_type() == q.scalar_type(),
              "triton_mla.decode: out in q's dtype, lse float32");
  const int64_t B = q.size(0), H = q.size(1), D = q.size(2), DV = out.size(2);
  TORCH_CHECK(out.dim() == 3 && out.size(0) == B && out.size(1) == H && out.stride(2) == 1,
              "triton_mla.decode: out must be [B, H, head_dim_v] with unit inner stride");
  TORCH_CHECK(lse.dim() == 2 && lse.size(0) == B && lse.size(1) == H && lse.stride(1) == 1,
              "triton_mla.decode: lse must be [B, H]");
  const bool fp8 = kv.scalar_type() == at::kByte;
  TmlaDecodeParams p = {};
  p.q = q.data_ptr();
  p.q_stride_b = q.stride(0);
  p.q_stride_h = q.stride(1);
  p.kv = kv.data_ptr();
  p.kv_stride_page = kv.stride(0);
  p.kv_stride_tok = kv.stride(1);
  p.page_size = (int32_t)kv.size(1);
  p.seqlens = lens.data_ptr<int32_t>();
  if (block_table.has_value()) {
    const at::Tensor& bt = *block_table;
    TORCH_CHECK(bt.scalar_type() == at::kInt && bt.dim() == 2 && bt.stride(1) == 1 && bt.is_cuda(),
                "triton_mla.decode: block_table must be int32 [B, W] with unit inner stride");
    p.block_table = bt.data_ptr<int32_t>();
    p.bt_stride = bt.stride(0);
    p.bt_width = (int32_t)bt.size(1);
    p.num_pages = kv.size(0);
  } else {
    p.num_pages = B;
  }
  p.out = out.data_ptr();
  p.out_stride_b = out.stride(0);
  p.out_stride_h = out.stride(1);
  p.lse = lse.data_ptr<float>();
  p.lse_stride_b = lse.stride(0);
  p.batch = (int32_t)B;
  p.num_heads = (int32_t)H;
  p.d_qk = (int32_t)D;
  p.d_v = (int32_t)DV;
  p.num_splits = (int32_t)num_splits;
  p.dtype = dtype_code(q.scalar_type());
  p.kernel = (int32_t)kernel;
  p.softmax_scale = (float)softmax_scale;
  p.q_len = (int32_t)q_len;
  p.kv_format = fp8 ? TMLA_KV_FP8_E4M3 : TMLA_KV_SAME;
  if (B == 0) return;
  const c10::cuda::CUDAGuard guard(q.device());
  p.status = status_word(status);
  const size_t ws_bytes = tmla_workspace_bytes(p.batch, p.num_heads, p.num_splits, p.d_v);
  at::Tensor ws;
  if (ws_bytes) {
    ws = at::empty({(int64_t)ws_bytes}, q.options().dtype(at::kByte));
    const size_t o_bytes = ((size_t)B * H * num_splits * DV * 4 + 255) & ~(size_t)255;
    p.ws_o = reinterpret_cast<float*>(ws.data_ptr());
    p.ws_lse = reinterpret_cast<float*>(static_cast<char*>(ws.data_ptr()) + o_bytes);
  }
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  const int rc = tmla_decode(&p, stream);
  TORCH_CHECK(rc == TMLA_OK, "triton_mla.decode: ", tmla_error_string(rc), " ",
              rc == TMLA_ERR_CUDA ? tmla_last_cuda_error() : "");
}

// ---------------------------------------------------------------- int8 projections
// quantize_int8(x [m, k]) -> (q int8 [m, k], scale fp32 [m]); rms_norm_int8 -> (q, scale, h): h is a
// new tensor when there is a residual and no residual_out, else empty; linear_int8(x_q [m, k],
// x_scale [m], w_q [n, k], w_scale [n]) -> y [m, n] in out_dtype.  Rows of q, h and y start on 16-byte
// boundaries (a row stride of k or n rounded up), as the kernels' vector accesses and TMA want them.  Outputs come
// from the caching allocator, the launches go on the current stream of the inputs' device.

// An [m, n] tensor whose rows start on 16-byte boundaries.  Its storage holds the last row's padding too, which the
// product's TMA stores fill (an [m, n] tensor of these strides alone would end with the last row's values).
at::Tensor aligned_rows(int64_t m, int64_t n, const at::TensorOptions& options, at::ScalarType dtype) {
  const int64_t per = 16 / (int64_t)at::elementSize(dtype);
  const int64_t stride = std::max<int64_t>(1, (n + per - 1) / per * per);
  at::Tensor t = at::empty({m, stride}, options.dtype(dtype));
  t.unsafeGetTensorImpl()->set_sizes_and_strides(c10::IntArrayRef{m, n}, c10::IntArrayRef{stride, 1});
  return t;
}
at::Tensor int8_rows(const at::Tensor& x) { return aligned_rows(x.size(0), x.size(1), x.options(), at::kChar); }

void check_rows(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), "triton_mla: CUDA tensors only (there is no CPU implementation), got ", what, " on ",
              t.device());
  TORCH_CHECK(t.dim() == 2 && (t.size(1) == 0 || t.stride(1) == 1), "triton_mla: ", what,
              " must be a matrix with unit inner stride");
}
// A one-row matrix may carry any row stride, which nothing reads: one that breaks no alignment.
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 15) / 16 * 16; }

TmlaInt8RowsParams rows_params(const at::Tensor& x, const at::Tensor& q, const at::Tensor& scale, bool overlap) {
  TmlaInt8RowsParams p = {};
  TORCH_CHECK(x.size(1) <= INT32_MAX, "triton_mla: rows of at most 2^31 - 1 values");
  p.x = x.data_ptr();
  p.x_stride = row_stride(x);
  p.q = q.data_ptr();
  p.q_stride = row_stride(q);
  p.scale = scale.data_ptr<float>();
  p.m = x.size(0);
  p.k = (int32_t)x.size(1);
  p.dtype = dtype_code(x.scalar_type());
  p.flags = overlap ? TMLA_LAYER_FLAG_PDL : 0;
  return p;
}

std::tuple<at::Tensor, at::Tensor> quantize_int8_cuda(const at::Tensor& x, bool overlap) {
  check_rows(x, "x");
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor q = int8_rows(x), scale = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
  const TmlaInt8RowsParams p = rows_params(x, q, scale, overlap);
  check_rc(tmla_quantize_int8(&p, c10::cuda::getCurrentCUDAStream(x.device().index()).stream()),
           "tmla_quantize_int8");
  return {q, scale};
}
std::tuple<at::Tensor, at::Tensor> quantize_int8_meta(const at::Tensor& x, bool) {
  return {int8_rows(x), at::empty({x.size(0)}, x.options().dtype(at::kFloat))};
}

void check_like(const at::Tensor& t, const at::Tensor& x, const char* what) {
  check_rows(t, what);
  TORCH_CHECK(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.device() == x.device(),
              "triton_mla.rms_norm_int8: ", what, " must have x's shape, dtype and device");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_int8_cuda(const at::Tensor& x, const at::Tensor& weight,
                                                                  double eps,
                                                                  const std::optional<at::Tensor>& residual,
                                                                  const std::optional<at::Tensor>& residual_out,
                                                                  bool overlap) {
  check_rows(x, "x");
  TORCH_CHECK(weight.is_cuda(), "triton_mla: CUDA tensors only (there is no CPU implementation), got weight on ",
              weight.device());
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(1) && weight.is_contiguous() &&
                  weight.scalar_type() == x.scalar_type() && weight.device() == x.device(),
              "triton_mla.rms_norm_int8: weight must be a contiguous [k] vector of x's dtype and device");
  TORCH_CHECK(!residual_out.has_value() || residual.has_value(),
              "triton_mla.rms_norm_int8: residual_out without residual");
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor q = int8_rows(x), scale = at::empty({x.size(0)}, x.options().dtype(at::kFloat)), h;
  TmlaInt8RowsParams p = rows_params(x, q, scale, overlap);
  p.weight = weight.data_ptr();
  p.eps = (float)eps;
  if (residual.has_value()) {
    check_like(*residual, x, "residual");
    if (residual_out.has_value()) {
      check_like(*residual_out, x, "residual_out");
      TORCH_CHECK(!(c10::GradMode::is_enabled() && residual_out->requires_grad()),
                  "triton_mla.rms_norm_int8: residual_out requires a gradient, which does not pass through this "
                  "operator; call it under torch.no_grad()");
    } else {
      h = aligned_rows(x.size(0), x.size(1), x.options(), x.scalar_type());
    }
    const at::Tensor& out = residual_out.has_value() ? *residual_out : h;
    p.residual = residual->data_ptr();
    p.residual_stride = row_stride(*residual);
    p.h = out.data_ptr();
    p.h_stride = row_stride(out);
    // Autograd must see that a caller's tensor has been written.
    if (residual_out.has_value() && !residual_out->is_inference())
      residual_out->unsafeGetTensorImpl()->bump_version();
  }
  if (!h.defined()) h = at::empty({0}, x.options());
  check_rc(tmla_rms_norm_int8(&p, c10::cuda::getCurrentCUDAStream(x.device().index()).stream()),
           "tmla_rms_norm_int8");
  return {q, scale, h};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_int8_meta(const at::Tensor& x, const at::Tensor&, double,
                                                                  const std::optional<at::Tensor>& residual,
                                                                  const std::optional<at::Tensor>& residual_out,
                                                                  bool) {
  at::Tensor h = residual.has_value() && !residual_out.has_value()
                     ? aligned_rows(x.size(0), x.size(1), x.options(), x.scalar_type())
                     : at::empty({0}, x.options());
  return {int8_rows(x), at::empty({x.size(0)}, x.options().dtype(at::kFloat)), h};
}

at::Tensor linear_int8_cuda(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& w,
                            const at::Tensor& w_scale, at::ScalarType out_dtype, bool overlap,
                            const std::optional<at::Tensor>& status) {
  check_rows(x, "x_q");
  check_rows(w, "w_q");
  TORCH_CHECK(x.scalar_type() == at::kChar && w.scalar_type() == at::kChar && x.size(1) == w.size(1) &&
                  x.device() == w.device(),
              "triton_mla.linear_int8: x_q [m, k] and w_q [n, k] must be int8 on one device");
  TORCH_CHECK(x_scale.dim() == 1 && x_scale.size(0) == x.size(0) && w_scale.dim() == 1 &&
                  w_scale.size(0) == w.size(0) && x_scale.scalar_type() == at::kFloat &&
                  w_scale.scalar_type() == at::kFloat && x_scale.is_contiguous() && w_scale.is_contiguous() &&
                  x_scale.device() == x.device() && w_scale.device() == x.device(),
              "triton_mla.linear_int8: x_scale [m] and w_scale [n] must be contiguous fp32 vectors on x_q's device");
  TORCH_CHECK(x.size(0) <= INT32_MAX && w.size(0) <= INT32_MAX && x.size(1) <= INT32_MAX,
              "triton_mla.linear_int8: sizes beyond 2^31 - 1");
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = aligned_rows(x.size(0), w.size(0), x.options(), out_dtype);
  TmlaLinearInt8Params p = {};
  p.x = x.data_ptr();
  p.x_stride = row_stride(x);
  p.x_scale = x_scale.data_ptr<float>();
  p.w = w.data_ptr();
  p.w_stride = row_stride(w);
  p.w_scale = w_scale.data_ptr<float>();
  p.y = y.data_ptr();
  p.y_stride = y.stride(0);
  p.m = (int32_t)x.size(0);
  p.n = (int32_t)w.size(0);
  p.k = (int32_t)x.size(1);
  p.dtype = dtype_code(out_dtype);
  p.status = status_word(status);
  p.flags = (overlap ? TMLA_LAYER_FLAG_PDL : 0) | TMLA_LINEAR_FLAG_PAD_Y;
  check_rc(tmla_linear_int8(&p, c10::cuda::getCurrentCUDAStream(x.device().index()).stream()), "tmla_linear_int8");
  return y;
}
at::Tensor linear_int8_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor& w, const at::Tensor&,
                            at::ScalarType out_dtype, bool, const std::optional<at::Tensor>&) {
  return aligned_rows(x.size(0), w.size(0), x.options(), out_dtype);
}

// Shapes only: out and lse are written in place, so there is nothing to return.
void decode_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const std::optional<at::Tensor>&,
                 const at::Tensor&, const at::Tensor&, int64_t, double, int64_t, int64_t,
                 const std::optional<at::Tensor>&) {}

}  // namespace

TORCH_LIBRARY(triton_mla, m) {
  m.def(
      "decode(Tensor q, Tensor kv_cache, Tensor cache_seqlens, Tensor? block_table, Tensor(a!) out, "
      "Tensor(b!) lse, int num_splits, float softmax_scale, int kernel, int q_len, Tensor? status) -> ()");
  m.def("quantize_int8(Tensor x, bool overlap) -> (Tensor, Tensor)");
  m.def(
      "rms_norm_int8(Tensor x, Tensor weight, float eps, Tensor? residual, Tensor(a!)? residual_out, bool overlap) "
      "-> (Tensor, Tensor, Tensor)");
  m.def(
      "linear_int8(Tensor x_q, Tensor x_scale, Tensor w_q, Tensor w_scale, ScalarType out_dtype, bool overlap, "
      "Tensor? status) -> Tensor");
}

TORCH_LIBRARY_IMPL(triton_mla, CUDA, m) {
  m.impl("decode", &decode_cuda);
  m.impl("quantize_int8", &quantize_int8_cuda);
  m.impl("rms_norm_int8", &rms_norm_int8_cuda);
  m.impl("linear_int8", &linear_int8_cuda);
}

TORCH_LIBRARY_IMPL(triton_mla, Meta, m) {
  m.impl("decode", &decode_meta);
  m.impl("quantize_int8", &quantize_int8_meta);
  m.impl("rms_norm_int8", &rms_norm_int8_meta);
  m.impl("linear_int8", &linear_int8_meta);
}

// Serving operators: no gradient passes through them (their outputs require none).
TORCH_LIBRARY_IMPL(triton_mla, Autograd, m) {
  m.impl("quantize_int8", torch::CppFunction::makeFallthrough());
  m.impl("rms_norm_int8", torch::CppFunction::makeFallthrough());
  m.impl("linear_int8", torch::CppFunction::makeFallthrough());
}
