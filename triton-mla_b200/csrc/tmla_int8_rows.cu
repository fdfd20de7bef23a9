// int8 rows with one scale per row, the operands of tmla_linear_int8:
//
//   tmla_quantize_int8   s = max(max_j |x_j| / 127, 2^-126),  q_j = rint(x_j (1 / s))
//   tmla_rms_norm_int8   h = T(x + r) (h = x without a residual), y_j = h_j w_j rstd with
//                        rstd = 1 / sqrt(mean_j h_j^2 + eps), then y quantised as above
//
// The scale needs max |y| and the norm needs sum h^2, but rstd is one positive factor of the whole
// row: max_j |h_j w_j rstd| = rstd max_j |h_j w_j| (rounding is monotone).  So both reductions
// run at once over the row, which stays in registers, and every input is read and every
// output written exactly once (rows too long for a block's registers are read twice, see loop_kernel).
// Arithmetic is fp32 whatever T is; h is rounded to T first (the norm is of the residual stream as
// stored), the integers are rounded to nearest even.
//
// Bound: HBM bandwidth.  Measured on B200 (inputs beyond L2, back to back): quantise 8192 x 7168 bf16
// 28.3 us (6.2 TB/s, 95% of a copy), norm with residual 70 us (5.9 TB/s, 90%), norm without
// 41.7 us; one token 2.0-2.7 us, which is launch and one trip to memory.
//
// A row that holds a NaN or an infinity has no scale: its scale is NaN and its integers are 0,
// so every product with it is NaN.  The maximum keeps a NaN.  Products h w beyond fp32 alone are not that (far_row).
#include "tmla_common.cuh"
#include "tmla_ptx.cuh"

namespace tmla {
namespace int8_rows {

constexpr float kTiny = 1.17549435e-38f;  // 2^-126, the smallest scale (1 / s stays finite)
constexpr int kMaxK = 1 << 30;  // element indices of a row stay in int
constexpr int kMaxThreads = 1024;
constexpr int kValues = 8;  // values per thread of a row off 16-byte boundaries

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
  bool early_w;  // the preceding kernel does not write w
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(float v, __half& o) { o = __float2half_rn(v); }

// The values of a 16-byte vector of T, and back with one rounding each.
template <typename T>
constexpr int kPer = 16 / (int)sizeof(T);

__device__ __forceinline__ void unpack2(uint32_t w, const __nv_bfloat16*, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, const __half*, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x, b = f.y;
}
template <typename T>
__device__ __forceinline__ void unpack(uint4 u, float (&v)[kPer<T>]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  } else {
    const T* t = nullptr;
    unpack2(u.x, t, v[0], v[1]);
    unpack2(u.y, t, v[2], v[3]);
    unpack2(u.z, t, v[4], v[5]);
    unpack2(u.w, t, v[6], v[7]);
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// T(x + r), element by element.
template <typename T>
__device__ __forceinline__ uint4 add(uint4 x, uint4 r) {
  float a[kPer<T>], b[kPer<T>];
  unpack<T>(x, a);
  unpack<T>(r, b);
#pragma unroll
  for (int j = 0; j < kPer<T>; ++j) a[j] += b[j];
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
  } else {
    const T* t = nullptr;
    return make_uint4(pack2(a[0], a[1], t), pack2(a[2], a[3], t), pack2(a[4], a[5], t), pack2(a[6], a[7], t));
  }
}

// rint(v * inv) as the low byte of the result, for |v * inv| < 2^21: adding 1.5 * 2^23 leaves the
// nearest integer (ties to even) in the low mantissa bits, in two's complement.  inv and the product are rounded
// (2^-17 and 2^-18 at 127), so this is rint(v / s) unless v / s lies within 2^-16 of half an integer.  16-bit values
// lie there about once in 3,000 (4.6875 of a row whose largest is 9.375 is 63.5 / 127).  Deciding those too, by a
// division or by the remainder v - n s of the values next to a border, took 30 to 48% more (8192 x 7168 quantise
// 28.3 us to 37-42, fp32 44.5 to 58-61, the norm 71 to 75-83).
__device__ __forceinline__ uint32_t round_bits(float v, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f));
}
// The integers of N = 4 or 8 values.  |v * inv| <= 127 (1 + 2^-22) by the choice of the scale, so no
// value rounds beyond 127.
template <int N>
__device__ __forceinline__ void store_q(int8_t* q, const float (&v)[N], float inv) {
  uint32_t w[N / 4];
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    const uint32_t lo = __byte_perm(round_bits(v[4 * j], inv), round_bits(v[4 * j + 1], inv), 0x0040);
    const uint32_t hi = __byte_perm(round_bits(v[4 * j + 2], inv), round_bits(v[4 * j + 3], inv), 0x0040);
    w[j] = __byte_perm(lo, hi, 0x5410);
  }
  if constexpr (N == 8)
    *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(q) = w[0];
}

// The larger of two values that are not negative; NaN if one of them is NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Maximum of `top` (not negative, or NaN: bit patterns order them, NaN > inf > finite) and, with the
// norm, sum of `sum` over the threads of a row (whole warps).
template <bool kNorm>
__device__ __forceinline__ void reduce_row(float& top, float& sum, uint32_t (*s_mx)[32], float (*s_sum)[32]) {
  uint32_t mx = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  top = __uint_as_float(mx);
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
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < warps ? s_mx[threadIdx.y][lane] : 0u));
  if constexpr (kNorm) {
    sum = lane < warps ? s_sum[threadIdx.y][lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
}

// From the row's max |h w| (bits) and sum of squares: the scale, and the factors of h w.
template <bool kNorm>
__device__ __forceinline__ void row_scale(float mx, float sum, int k, float eps, float& scale, float& rstd,
                                          float& inv) {
  rstd = kNorm ? rsqrtf(sum / (float)k + eps) : 1.f;
  const float top = mx * rstd;
  if (!(top < INFINITY)) {  // a NaN or an infinity in the row (or y beyond fp32)
    scale = __uint_as_float(0x7fc00000u);
    inv = 0.f;
    return;
  }
  scale = fmaxf(top / 127.f, kTiny);
  inv = 1.f / scale;
}

// A row whose largest |h w| is infinite.  That is a row without a scale if h or w holds an infinity, but finite h and w
// may only have a product past fp32: y is then formed as (h rstd) w, which is finite unless y itself is not (and 0 where
// the squares sum past fp32 too, rstd being 0).  Rare, so value by value: each warp looks for the maximum over the whole
// row, without a barrier (rows of a block may differ), then every thread writes its values.  h is the row as stored.
template <typename T>
__device__ __forceinline__ void far_row(const T* h, const T* w, int8_t* q, float* scale_out, int k, float sum,
                                        float eps) {
  __syncwarp();  // h may have been written by this row's other threads (of other warps: a barrier came since)
  const float rstd = rsqrtf(sum / (float)k + eps);
  float top = 0.f;
  for (int j = threadIdx.x & 31; j < k; j += 32) top = max_nan(top, fabsf(to_float(h[j]) * rstd * to_float(w[j])));
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
  float scale, one, inv;
  row_scale<false>(top, 0.f, k, eps, scale, one, inv);
  if (threadIdx.x == 0) *scale_out = scale;
  for (int j = threadIdx.x; j < k; j += blockDim.x)
    q[j] = (int8_t)round_bits(inv == 0.f ? 0.f : to_float(h[j]) * rstd * to_float(w[j]), inv);
}

// For rows_kernel as a call: within it the kernel of 4 vectors a thread takes 42.2 us for 8192 x 7168 instead of 41.6.
template <typename T>
__device__ __noinline__ void far_row_call(const T* h, const T* w, int8_t* q, float* scale, int k, float sum, float eps) {
  far_row(h, w, q, scale, k, sum, eps);
}

// The row's running maximum of |y| (up to rstd) and sum of squares over one value.
template <bool kNorm>
__device__ __forceinline__ float visit(float h, float w, float& mx, float& sum) {
  if constexpr (kNorm) {
    sum += h * h;
    h *= w;
  }
  mx = max_nan(mx, fabsf(h));
  return h;
}

// Rows on 16-byte boundaries.  blockDim = (threads per row, rows per block); each thread holds up
// to kVecs vectors of its row, vector i of thread t being number i * threads + t, and the first
// k % N threads one value each of the row's end.  Loads are predicated, not branched around, so
// that all of a thread's are in flight at once.  The row stays packed in T across the reduction (4
// registers per vector); h w is formed again after it.  One or two vectors a thread are rows of 64 threads at most, in
// blocks of 128, of which an SM's registers are to hold 12 and 9 (65536 x 256, norm with residual: 22.4 us, else 24.6).
template <typename T, int kVecs, bool kNorm>
__global__ void __launch_bounds__(kVecs >= 4 ? 512 : 128, kVecs >= 8 ? 1 : kVecs == 4 ? 2 : kVecs == 2 ? 9 : 12)
    rows_kernel(const Args a) {
  __shared__ uint32_t s_mx[32][32];
  __shared__ float s_sum[kNorm ? 32 : 1][32];
  constexpr int N = kPer<T>;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int threads = blockDim.x, t = threadIdx.x;
  const int vecs = row < a.m ? a.k / N : 0;
  const int last = row < a.m && t < a.k % N ? a.k - a.k % N + t : -1;  // this thread's value of the row's end
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 w[kNorm ? kVecs : 1];
  float w_last = 0.f;
  auto load_weight = [&]() {
    const T* wp = static_cast<const T*>(a.w);
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      w[i] = i * threads + t < vecs ? reinterpret_cast<const uint4*>(wp)[i * threads + t] : zero;
    if (last >= 0) w_last = to_float(wp[last]);
  };
  if constexpr (kNorm)
    if (a.early_w) load_weight();
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  if constexpr (kNorm)
    if (!a.early_w) load_weight();
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  uint4 h[kVecs];
  float h_last = 0.f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
    h[i] = i * threads + t < vecs ? reinterpret_cast<const uint4*>(x)[i * threads + t] : zero;
  if (last >= 0) h_last = to_float(x[last]);
  if (kNorm && a.r != nullptr) {
    const T* r = static_cast<const T*>(a.r) + row * a.r_stride;
    T* out = static_cast<T*>(a.h) + row * a.h_stride;
    uint4 rv[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      rv[i] = i * threads + t < vecs ? reinterpret_cast<const uint4*>(r)[i * threads + t] : zero;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      h[i] = add<T>(h[i], rv[i]);
      if (i * threads + t < vecs) reinterpret_cast<uint4*>(out)[i * threads + t] = h[i];
    }
    if (last >= 0) {
      T v;
      from_float(h_last + to_float(r[last]), v);
      out[last] = v;
      h_last = to_float(v);
    }
  }
  float mx = 0.f, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    float hv[N], wv[N];
    unpack<T>(h[i], hv);
    if constexpr (kNorm) unpack<T>(w[i], wv);
#pragma unroll
    for (int j = 0; j < N; ++j) visit<kNorm>(hv[j], kNorm ? wv[j] : 1.f, mx, sum);
  }
  h_last = visit<kNorm>(h_last, w_last, mx, sum);
  reduce_row<kNorm>(mx, sum, s_mx, s_sum);
  if (row >= a.m) return;
  if (kNorm && mx == INFINITY) {
    far_row_call(a.r != nullptr ? static_cast<const T*>(a.h) + row * a.h_stride : x, static_cast<const T*>(a.w),
                 a.q + row * a.q_stride, a.scale + row, a.k, sum, a.eps);
    return;
  }
  float scale, rstd, inv;
  row_scale<kNorm>(mx, sum, a.k, a.eps, scale, rstd, inv);
  if (t == 0) a.scale[row] = scale;
  int8_t* q = a.q + row * a.q_stride;
  const bool bad = inv == 0.f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    if (i * threads + t >= vecs) break;
    float hv[N], wv[N];
    unpack<T>(h[i], hv);
    if constexpr (kNorm) unpack<T>(w[i], wv);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (kNorm) hv[j] = hv[j] * wv[j] * rstd;
      if (bad) hv[j] = 0.f;
    }
    store_q(q + (i * threads + t) * N, hv, inv);
  }
  if (last >= 0) q[last] = (int8_t)round_bits(bad ? 0.f : (kNorm ? h_last * rstd : h_last), inv);
}

// Rows that do not start on 16-byte boundaries: the same value by value, value i of thread t being number
// i * threads + t.
template <typename T, bool kNorm>
__global__ void __launch_bounds__(kMaxThreads) values_kernel(const Args a) {
  __shared__ uint32_t s_mx[32][32];
  __shared__ float s_sum[kNorm ? 32 : 1][32];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int threads = blockDim.x, t = threadIdx.x;
  const int k = row < a.m ? a.k : 0;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* w = static_cast<const T*>(a.w);
  float h[kValues], wv[kValues];
#pragma unroll
  for (int i = 0; i < kValues; ++i) {
    const int at = i * threads + t;
    h[i] = at < k ? to_float(x[at]) : 0.f;
    wv[i] = kNorm && at < k ? to_float(w[at]) : 0.f;
  }
  if (kNorm && a.r != nullptr) {
    const T* r = static_cast<const T*>(a.r) + row * a.r_stride;
    T* out = static_cast<T*>(a.h) + row * a.h_stride;
    float rv[kValues];
#pragma unroll
    for (int i = 0; i < kValues; ++i) rv[i] = i * threads + t < k ? to_float(r[i * threads + t]) : 0.f;
#pragma unroll
    for (int i = 0; i < kValues; ++i) {
      T v;
      from_float(h[i] + rv[i], v);
      h[i] = to_float(v);
      if (i * threads + t < k) out[i * threads + t] = v;
    }
  }
  float mx = 0.f, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kValues; ++i) h[i] = visit<kNorm>(h[i], wv[i], mx, sum);
  reduce_row<kNorm>(mx, sum, s_mx, s_sum);
  if (row >= a.m) return;
  if (kNorm && mx == INFINITY) {
    far_row(a.r != nullptr ? static_cast<const T*>(a.h) + row * a.h_stride : x, static_cast<const T*>(a.w),
            a.q + row * a.q_stride, a.scale + row, a.k, sum, a.eps);
    return;
  }
  float scale, rstd, inv;
  row_scale<kNorm>(mx, sum, a.k, a.eps, scale, rstd, inv);
  if (t == 0) a.scale[row] = scale;
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int i = 0; i < kValues; ++i) {
    const float v = inv == 0.f ? 0.f : (kNorm ? h[i] * rstd : h[i]);
    if (i * threads + t < k) q[i * threads + t] = (int8_t)round_bits(v, inv);
  }
}

// Rows too long for the registers of a block, by vectors or value by value: the row is read a second
// time (from L1 / L2) for its integers.  With a residual the second pass reads h, which the same thread
// has written.
template <typename T, bool kNorm, bool kAligned>
__global__ void __launch_bounds__(kMaxThreads) loop_kernel(const Args a) {
  __shared__ uint32_t s_mx[1][32];
  __shared__ float s_sum[1][32];
  constexpr int N = kPer<T>;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = static_cast<const T*>(a.r) + row * a.r_stride;
  T* h = static_cast<T*>(a.h) + row * a.h_stride;
  const T* w = static_cast<const T*>(a.w);
  const bool res = kNorm && a.r != nullptr;
  const int vecs = kAligned ? a.k / N : 0;  // the first values as whole vectors, the others one by one
  const int step = blockDim.x;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  float mx = 0.f, sum = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < vecs; i += step) {
    uint4 u = reinterpret_cast<const uint4*>(x)[i];
    if (res) {
      u = add<T>(u, reinterpret_cast<const uint4*>(r)[i]);
      reinterpret_cast<uint4*>(h)[i] = u;
    }
    float hv[N], wv[N];
    unpack<T>(u, hv);
    if constexpr (kNorm) unpack<T>(reinterpret_cast<const uint4*>(w)[i], wv);
#pragma unroll
    for (int j = 0; j < N; ++j) visit<kNorm>(hv[j], kNorm ? wv[j] : 1.f, mx, sum);
  }
#pragma unroll 4
  for (int j = vecs * N + (int)threadIdx.x; j < a.k; j += step) {
    T v = x[j];
    if (res) {
      from_float(to_float(v) + to_float(r[j]), v);
      h[j] = v;
    }
    visit<kNorm>(to_float(v), kNorm ? to_float(w[j]) : 1.f, mx, sum);
  }
  reduce_row<kNorm>(mx, sum, s_mx, s_sum);
  if (kNorm && mx == INFINITY) {
    far_row(res ? h : x, w, a.q + row * a.q_stride, a.scale + row, a.k, sum, a.eps);
    return;
  }
  float scale, rstd, inv;
  row_scale<kNorm>(mx, sum, a.k, a.eps, scale, rstd, inv);
  if (threadIdx.x == 0) a.scale[row] = scale;
  int8_t* q = a.q + row * a.q_stride;
  const T* src = res ? h : x;
  const bool bad = inv == 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < vecs; i += step) {
    float hv[N], wv[N];
    unpack<T>(reinterpret_cast<const uint4*>(src)[i], hv);
    if constexpr (kNorm) unpack<T>(reinterpret_cast<const uint4*>(w)[i], wv);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (kNorm) hv[j] = hv[j] * wv[j] * rstd;
      if (bad) hv[j] = 0.f;
    }
    store_q(q + i * N, hv, inv);
  }
#pragma unroll 4
  for (int j = vecs * N + (int)threadIdx.x; j < a.k; j += step) {
    float v = to_float(src[j]);
    if constexpr (kNorm) v = v * to_float(w[j]) * rstd;
    q[j] = (int8_t)round_bits(bad ? 0.f : v, inv);
  }
}

// ---------------------------------------------------------------------------- host side

// A programmatic launch: the kernel may be scheduled while the one before it in the stream finishes, and
// waits for it (griddepcontrol.wait) before it touches memory.
template <typename K>
cudaError_t launch(K kernel, dim3 grid, dim3 block, const Args& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, bool kNorm>
cudaError_t run(const Args& a, bool aligned, cudaStream_t stream) {
  const int vecs = a.k / kPer<T> > 0 ? a.k / kPer<T> : 1;
  if (!aligned && a.k <= kValues * kMaxThreads) {
    // 333 x 1003 fp32 (norm with residual): 2.6 us, against 6.6 with the loop kernel below.
    const int threads = (a.k + 32 * kValues - 1) / (32 * kValues) * 32, rows = threads >= 128 ? 1 : 128 / threads;
    return launch(values_kernel<T, kNorm>, dim3((unsigned)((a.m + rows - 1) / rows)), dim3(threads, rows), a, stream);
  }
  if (!aligned || vecs > 8 * 512) {
    const int threads = a.k < kMaxThreads ? (a.k + 31) / 32 * 32 : kMaxThreads;
    return aligned ? launch(loop_kernel<T, kNorm, true>, dim3((unsigned)a.m), dim3(threads), a, stream)
                   : launch(loop_kernel<T, kNorm, false>, dim3((unsigned)a.m), dim3(threads), a, stream);
  }
  // Vectors per thread (bf16 on B200, us per call): 4 keep more loads in flight than 1 or 2 (norm with
  // residual of 8192 x 7168: 72.7 against 98.3 and 96.1; 4096 x 16384: 84.7 against 115), and 8
  // leave registers for half the warps (105.5).  Below 128 vectors a row is one warp or less
  // with 4 per thread, so 2 (65536 x 512, quantise: 19.0 against 22.1) or 1 fill it.  Rows of
  // less than 128 threads share a block (24576 x 1536: 20.0 with 128 threads, 22.2 with 256,
  // 25.9 with 64).
  const int per = vecs > 4 * 512 ? 8 : vecs >= 128 ? 4 : vecs >= 64 ? 2 : 1;
  const int threads = (vecs + 32 * per - 1) / (32 * per) * 32;
  const int rows = threads >= 128 ? 1 : 128 / threads;
  const dim3 grid((unsigned)((a.m + rows - 1) / rows)), block(threads, rows);
  switch (per) {
    case 1: return launch(rows_kernel<T, 1, kNorm>, grid, block, a, stream);
    case 2: return launch(rows_kernel<T, 2, kNorm>, grid, block, a, stream);
    case 4: return launch(rows_kernel<T, 4, kNorm>, grid, block, a, stream);
    default: return launch(rows_kernel<T, 8, kNorm>, grid, block, a, stream);
  }
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
  // Every tensor's rows start on whole vectors (16 bytes; one byte a value of q).
  const bool aligned = rows_aligned(p.x, p.x_stride, size, 16) && rows_aligned(p.q, p.q_stride, 1, 16 / size) &&
              (!norm || (uintptr_t)p.weight % 16 == 0) &&
              (!res || (rows_aligned(p.residual, p.residual_stride, size, 16) &&
                        rows_aligned(p.h, p.h_stride, size, 16)));
  a.early_w = (p.flags & TMLA_LAYER_FLAG_PDL) != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (p.dtype) {
    case TMLA_DTYPE_BF16:
      e = norm ? run<__nv_bfloat16, true>(a, aligned, s) : run<__nv_bfloat16, false>(a, aligned, s);
      break;
    case TMLA_DTYPE_FP16:
      e = norm ? run<__half, true>(a, aligned, s) : run<__half, false>(a, aligned, s);
      break;
    default:
      e = norm ? run<float, true>(a, aligned, s) : run<float, false>(a, aligned, s);
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
