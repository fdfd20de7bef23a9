// int8 rows with one scale per row, the operands of tmla_linear_int8:
//
//   tmla_quantize_int8   s = max(max_j |x_j| / 127, 2^-126),  q_j = rint(x_j / s)
//   tmla_rms_norm_int8   h = T(x + r) (h = x without a residual), y_j = h_j w_j rstd with
//                        rstd = 1 / sqrt(mean_j h_j^2 + eps), then y quantised as above
//
// The scale needs max |y| and the norm needs sum h^2, but rstd is one positive factor of the whole
// row: max_j |h_j w_j rstd| = rstd max_j |h_j w_j| (rounding is monotone).  So both reductions
// run at once over the row, which stays in registers, and every input is read and every
// output written exactly once.  Arithmetic is fp32 whatever T is; h is rounded to T first (the
// norm is of the residual stream as stored), the int8 values are rounded once, to nearest even.
//
// A row that holds a NaN or an infinity has no scale: its scale is NaN and its integers are 0,
// so every product with it is NaN.  The maximum is taken over the bit patterns of |y| as
// unsigned integers, in which NaN > inf > finite.
#include "tmla_common.cuh"
#include "tmla_ptx.cuh"

namespace tmla {
namespace int8_rows {

constexpr float kTiny = 1.17549435e-38f;  // 2^-126, the smallest scale (1 / s stays finite)
constexpr int kMaxK = 1 << 30;  // element indices of a row stay in int
constexpr int kMaxThreads = 1024;

struct Args {
  const void* x;
  int64_t x_stride;
  const void* r;
  int64_t r_stride;
  const void* w;
  void* h;
  int64_t h_stride;
  int8_t* q;
  int64_t q_stride;
  float* scale;
  int64_t m;
  int k;
  float eps;
  // Whether each tensor's rows are aligned for whole-vector accesses.
  bool x_vec, r_vec, w_vec, h_vec, q_vec;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(float v, __half& o) { o = __float2half_rn(v); }

// 16 bytes of T.
template <typename T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T e[N];
};

// Elements [at, at + N) of a row of k, zeros past its end.
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* row, int at, int k, bool aligned) {
  Vec<T> v;
  if (aligned && at + Vec<T>::N <= k) {
    v = *reinterpret_cast<const Vec<T>*>(row + at);
  } else {
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j) {
      if (at + j < k)
        v.e[j] = row[at + j];
      else
        from_float(0.f, v.e[j]);
    }
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* row, int at, int k, bool aligned, const Vec<T>& v) {
  if (aligned && at + Vec<T>::N <= k) {
    *reinterpret_cast<Vec<T>*>(row + at) = v;
  } else {
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j)
      if (at + j < k) row[at + j] = v.e[j];
  }
}

// rint(v * inv) as the low byte of the result, for |v * inv| < 2^21: adding 1.5 * 2^23 leaves the
// nearest integer (ties to even) in the low mantissa bits, in two's complement.
__device__ __forceinline__ uint32_t round_bits(float v, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f));
}
// The integers of N = 4 or 8 values.  |v * inv| <= 127 (1 + 2^-22) by the choice of the scale, so no
// value rounds beyond 127.
template <int N>
__device__ __forceinline__ void store_q(int8_t* row, int at, int k, bool aligned, const float (&v)[N], float inv) {
  uint32_t w[N / 4];
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    const uint32_t lo = __byte_perm(round_bits(v[4 * j], inv), round_bits(v[4 * j + 1], inv), 0x0040);
    const uint32_t hi = __byte_perm(round_bits(v[4 * j + 2], inv), round_bits(v[4 * j + 3], inv), 0x0040);
    w[j] = __byte_perm(lo, hi, 0x5410);
  }
  if (aligned && at + N <= k) {
    if constexpr (N == 8)
      *reinterpret_cast<uint2*>(row + at) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(row + at) = w[0];
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (at + j < k) row[at + j] = (int8_t)(w[j / 4] >> (8 * (j % 4)));
  }
}

// Maximum of `mx` and, with the norm, sum of `sum` over the threads of a row (whole warps).
template <bool kNorm>
__device__ __forceinline__ void reduce_row(uint32_t& mx, float& sum, uint32_t (*s_mx)[32], float (*s_sum)[32]) {
  mx = __reduce_max_sync(0xffffffffu, mx);
  if constexpr (kNorm) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  const int warps = blockDim.x >> 5;
  if (warps == 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    s_mx[threadIdx.y][warp] = mx;
    if constexpr (kNorm) s_sum[threadIdx.y][warp] = sum;
  }
  __syncthreads();
  mx = __reduce_max_sync(0xffffffffu, lane < warps ? s_mx[threadIdx.y][lane] : 0u);
  if constexpr (kNorm) {
    sum = lane < warps ? s_sum[threadIdx.y][lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
}

// From the row's max |h w| (bits) and sum of squares: the scale, and the factors of h w.
template <bool kNorm>
__device__ __forceinline__ void row_scale(uint32_t mx, float sum, int k, float eps, float& scale, float& rstd,
                                          float& inv) {
  rstd = kNorm ? rsqrtf(sum / (float)k + eps) : 1.f;
  const float top = __uint_as_float(mx) * rstd;
  if (!(top < INFINITY)) {  // a NaN or an infinity in the row (or y beyond fp32)
    scale = __uint_as_float(0x7fc00000u);
    inv = 0.f;
    return;
  }
  scale = fmaxf(top / 127.f, kTiny);
  inv = 1.f / scale;
}

// h = T(x + r) of one vector, as floats; written to h when there is a residual.
template <typename T>
__device__ __forceinline__ void add_residual(Vec<T>& x, const Vec<T>& r) {
#pragma unroll
  for (int j = 0; j < Vec<T>::N; ++j) from_float(to_float(x.e[j]) + to_float(r.e[j]), x.e[j]);
}

// blockDim = (threads per row, rows per block).  Each thread holds kVecs vectors of its row:
// vector i of thread t is number i * threads + t.
template <typename T, int kVecs, bool kNorm>
__global__ void __launch_bounds__(kMaxThreads) rows_kernel(const Args a) {
  __shared__ uint32_t s_mx[32][32];
  __shared__ float s_sum[kNorm ? 32 : 1][32];
  constexpr int N = Vec<T>::N;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < a.m;
  const int threads = blockDim.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  Vec<T> w[kNorm ? kVecs : 1];
  if constexpr (kNorm) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      w[i] = load_vec(static_cast<const T*>(a.w), (i * threads + (int)threadIdx.x) * N, a.k, a.w_vec);
  }
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  float v[kVecs][N];
  uint32_t mx = 0;
  float sum = 0.f;
  if (live) {
    Vec<T> xv[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) xv[i] = load_vec(x, (i * threads + (int)threadIdx.x) * N, a.k, a.x_vec);
    if (kNorm && a.r != nullptr) {
      const T* r = static_cast<const T*>(a.r) + row * a.r_stride;
      T* h = static_cast<T*>(a.h) + row * a.h_stride;
      Vec<T> rv[kVecs];
#pragma unroll
      for (int i = 0; i < kVecs; ++i) rv[i] = load_vec(r, (i * threads + (int)threadIdx.x) * N, a.k, a.r_vec);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        add_residual(xv[i], rv[i]);
        store_vec(h, (i * threads + (int)threadIdx.x) * N, a.k, a.h_vec, xv[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float f = to_float(xv[i].e[j]);
        if constexpr (kNorm) {
          sum += f * f;
          f *= to_float(w[i].e[j]);
        }
        v[i][j] = f;
        mx = max(mx, __float_as_uint(f) & 0x7fffffffu);
      }
    }
  }
  reduce_row<kNorm>(mx, sum, s_mx, s_sum);
  if (!live) return;
  float scale, rstd, inv;
  row_scale<kNorm>(mx, sum, a.k, a.eps, scale, rstd, inv);
  if (threadIdx.x == 0) a.scale[row] = scale;
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int at = (i * threads + (int)threadIdx.x) * N;
    if (at >= a.k) break;
#pragma unroll
    for (int j = 0; j < N; ++j) v[i][j] = inv == 0.f ? 0.f : (kNorm ? v[i][j] * rstd : v[i][j]);
    store_q(q, at, a.k, a.q_vec, v[i], inv);
  }
}

// Rows too long for the registers of a block: the row is read a second time (from L2) for its
// integers.  With a residual the second pass reads h, which the same thread has written.
template <typename T, bool kNorm>
__global__ void __launch_bounds__(kMaxThreads) long_rows_kernel(const Args a) {
  __shared__ uint32_t s_mx[1][32];
  __shared__ float s_sum[1][32];
  constexpr int N = Vec<T>::N;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = static_cast<const T*>(a.r) + row * a.r_stride;
  T* h = static_cast<T*>(a.h) + row * a.h_stride;
  const T* w = static_cast<const T*>(a.w);
  const bool res = kNorm && a.r != nullptr;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int step = (int)blockDim.x * N;
  uint32_t mx = 0;
  float sum = 0.f;
  for (int64_t at = (int64_t)threadIdx.x * N; at < a.k; at += step) {
    Vec<T> xv = load_vec(x, (int)at, a.k, a.x_vec);
    if (res) {
      add_residual(xv, load_vec(r, (int)at, a.k, a.r_vec));
      store_vec(h, (int)at, a.k, a.h_vec, xv);
    }
    Vec<T> wv;
    if constexpr (kNorm) wv = load_vec(w, (int)at, a.k, a.w_vec);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float f = to_float(xv.e[j]);
      if constexpr (kNorm) {
        sum += f * f;
        f *= to_float(wv.e[j]);
      }
      mx = max(mx, __float_as_uint(f) & 0x7fffffffu);
    }
  }
  reduce_row<kNorm>(mx, sum, s_mx, s_sum);
  float scale, rstd, inv;
  row_scale<kNorm>(mx, sum, a.k, a.eps, scale, rstd, inv);
  if (threadIdx.x == 0) a.scale[row] = scale;
  int8_t* q = a.q + row * a.q_stride;
  for (int64_t at = (int64_t)threadIdx.x * N; at < a.k; at += step) {
    const Vec<T> xv = res ? load_vec<T>(h, (int)at, a.k, a.h_vec) : load_vec(x, (int)at, a.k, a.x_vec);
    Vec<T> wv;
    if constexpr (kNorm) wv = load_vec(w, (int)at, a.k, a.w_vec);
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v[j] = to_float(xv.e[j]);
      if constexpr (kNorm) v[j] = v[j] * to_float(wv.e[j]) * rstd;
      if (inv == 0.f) v[j] = 0.f;
    }
    store_q(q, (int)at, a.k, a.q_vec, v, inv);
  }
}

// ---------------------------------------------------------------------------- host side

template <typename K>
cudaError_t launch(K kernel, dim3 grid, dim3 block, const Args& a, bool pdl, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, bool kNorm>
cudaError_t run(const Args& a, bool pdl, cudaStream_t stream) {
  constexpr int N = Vec<T>::N;
  constexpr int kMaxVecs = 4;
  const int64_t vecs = ((int64_t)a.k + N - 1) / N;
  if (vecs > (int64_t)kMaxVecs * kMaxThreads)
    return launch(long_rows_kernel<T, kNorm>, dim3((unsigned)a.m), dim3(kMaxThreads), a, pdl, stream);
  const int per = vecs <= kMaxThreads ? 1 : kMaxVecs;
  const int threads = (int)((vecs + 32 * per - 1) / (32 * per) * 32);
  const dim3 grid((unsigned)a.m), block(threads, 1);
  return per == 1 ? launch(rows_kernel<T, 1, kNorm>, grid, block, a, pdl, stream)
                  : launch(rows_kernel<T, kMaxVecs, kNorm>, grid, block, a, pdl, stream);
}

bool rows_aligned(const void* p, int64_t stride, int size, int bytes) {
  return ((uintptr_t)p | (uintptr_t)(stride * size)) % bytes == 0;
}

int start(const TmlaInt8RowsParams& p, bool norm, void* stream) {
  if (p.m < 0 || p.k < 1) return TMLA_ERR_INVALID_ARG;
  if (p.dtype != TMLA_DTYPE_BF16 && p.dtype != TMLA_DTYPE_FP16 && p.dtype != TMLA_DTYPE_FP32)
    return TMLA_ERR_INVALID_ARG;
  if (p.m == 0) return TMLA_OK;
  if (p.m > 0x7fffffff || p.k > kMaxK) return TMLA_ERR_UNSUPPORTED;  // a grid dimension, an int index
  if (!p.x || !p.q || !p.scale || p.x_stride < p.k || p.q_stride < p.k) return TMLA_ERR_INVALID_ARG;
  const bool res = norm && p.residual != nullptr;
  if (norm && !p.weight) return TMLA_ERR_INVALID_ARG;
  if (!norm && (p.weight || p.residual)) return TMLA_ERR_INVALID_ARG;
  if (res && (!p.h || p.residual_stride < p.k || p.h_stride < p.k)) return TMLA_ERR_INVALID_ARG;
  const int size = p.dtype == TMLA_DTYPE_FP32 ? 4 : 2;
  Args a;
  a.x = p.x;
  a.x_stride = p.x_stride;
  a.r = res ? p.residual : nullptr;
  a.r_stride = p.residual_stride;
  a.w = p.weight;
  a.h = p.h;
  a.h_stride = p.h_stride;
  a.q = static_cast<int8_t*>(p.q);
  a.q_stride = p.q_stride;
  a.scale = p.scale;
  a.m = p.m;
  a.k = p.k;
  a.eps = p.eps;
  a.x_vec = rows_aligned(p.x, p.x_stride, size, 16);
  a.r_vec = rows_aligned(p.residual, p.residual_stride, size, 16);
  a.w_vec = (uintptr_t)p.weight % 16 == 0;
  a.h_vec = rows_aligned(p.h, p.h_stride, size, 16);
  a.q_vec = rows_aligned(p.q, p.q_stride, 1, 16 / size);
  const bool pdl = (p.flags & TMLA_LAYER_FLAG_PDL) != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (p.dtype) {
    case TMLA_DTYPE_BF16:
      e = norm ? run<__nv_bfloat16, true>(a, pdl, s) : run<__nv_bfloat16, false>(a, pdl, s);
      break;
    case TMLA_DTYPE_FP16:
      e = norm ? run<__half, true>(a, pdl, s) : run<__half, false>(a, pdl, s);
      break;
    default:
      e = norm ? run<float, true>(a, pdl, s) : run<float, false>(a, pdl, s);
      break;
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? TMLA_OK : record_cuda_error(e);
}

}  // namespace int8_rows
}  // namespace tmla

extern "C" {

int tmla_quantize_int8(const TmlaInt8RowsParams* p, void* stream) {
  if (!p) return TMLA_ERR_INVALID_ARG;
  return tmla::int8_rows::start(*p, false, stream);
}

int tmla_rms_norm_int8(const TmlaInt8RowsParams* p, void* stream) {
  if (!p) return TMLA_ERR_INVALID_ARG;
  return tmla::int8_rows::start(*p, true, stream);
}

}  // extern "C"
