// int8 projections: y[i, j] = x_scale[i] w_scale[j] sum_c x[i, c] w[j, c], both operands int8 with
// unit stride along c.  The sum is exact in int32 for k <= 131071 (|sum| <= k 2^14 < 2^31), so
// neither the order of the terms nor the way k is cut changes the result.
//
// tcgen05 kernel (int8_kernel).  The weight rows (output channels) are the MMA's M and the tokens its
// N, whatever their numbers: a tile is 128 channels (one TMEM lane each) x 16 to 256 tokens, so that one
// token wastes no more than 15, and D[channel][token] leaves TMEM with neighbouring channels in
// neighbouring lanes, as y's rows want them.  One instantiation per type serves all sizes; the
// tile's tokens N are an argument.
//   kGroup = 1: one CTA per tile of 128 channels.
//   kGroup = 2: a CTA pair per tile of 256 channels (cta_group::2): each CTA holds its 128 weight
//     rows and half of the tokens, which halves what an MMA reads of the token operand.
//   splits > 1: the CTAs (or pairs) of a cluster each take a part of k for the same tile.  Each
//     accumulates in its own TMEM; then CTA s of the cluster adds up the token columns s of all
//     through distributed shared memory and writes them.  No workspace, no counters, no atomics.
// Per CTA (352 threads): warp 0 loads k-steps of 128 columns (128-byte swizzled boxes of w and x) by
// TMA into a ring of stages; warp 1 issues the MMAs (the pair's even CTA for both); warps 2-9
// are the epilogue; warp 10 stores what they stage.  Unsplit CTAs are persistent, with two
// accumulators, so that a tile's epilogue runs under the next tile's MMAs.
//
// What bounds it, and what it reaches on B200 (weights not in L2, calls back to back).  Few tokens: the weight's
// stream from HBM.  wo (7168 x 16384) 16 tokens 21.3 us (85% of a copy's bandwidth), wq_b (24576 x 1536) 8.6 us,
// [wq_a; wkv_a] (2112 x 7168) 6.6 us, of which a launch with nothing to do is 2.3.  Many tokens: the MMAs; wo 8192
// tokens 600 us = 3.2e15 operations a second at the clock that 1000 W allow, the tensor pipe active for
// 87% of the cycles of a full wave.  Small k: the epilogue; 4096 x 32768 x 512 80 us, 3.4 TB/s of y.
//   An issuing thread alone in its branch took 66 cycles for each MMA and 100 for each TMA load (every operand
//   moved to a uniform register), 560 a k-step whatever its size, above the MMAs' 512.  With the warp converged
//   and one elected thread wo 8192 tokens in tiles of 128 went from 1106 to 832 us.
//   Four epilogue warps with stores of single columns took 13 us for a pair's tile of 256 tokens; eight, with y staged
//   and stored by TMA, 2.3.  Sixteen took as long.
//
// Every wait is bounded (2 s by default): on expiry the kernel sets TMLA_STATUS_TIMEOUT, stops,
// drains the copies and MMAs that it issued, leaves the tiles that it could not finish unwritten,
// waits for what others are still sending it, frees TMEM and returns.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>

#include <atomic>

#include "tmla_common.cuh"
#include "tmla_ptx.cuh"

namespace tmla {
namespace sm100 {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();
}
namespace linear_int8 {

using namespace ptx;

constexpr int kRows = 128;                 // weight rows per CTA (TMEM lanes)
constexpr int kBoxK = 128;                 // columns per k-step: one swizzled 128-byte row
constexpr int kWBytes = kRows * kBoxK;     // weight bytes of a stage
constexpr int kMaxTok = 256;               // tokens per tile (MMA N)
constexpr int kMaxSplits = 8;              // CTAs of a portable cluster
constexpr int kMaxStages = 12;
// Stages whose weights are requested into L2 before the kernel before has ended.  Four, all, none (us on
// B200): wo 16 tokens 22.5, 22.3, 23.1 (single CTAs in 2 parts); rms_norm_int8 and [wq_a; wkv_a] in a row 8.6, 9.3, 9.1.
constexpr int kPrefetch = 4;
constexpr int kEpiWarps = 8, kEpiThreads = 32 * kEpiWarps;
constexpr int kStoreWarp = 2 + kEpiWarps;
constexpr int kThreads = 32 * (kStoreWarp + 1);
// y leaves in chunks of 128 channels x 2 kBoxTok<T> tokens, staged in shared memory as boxes of
// kBoxChannels<T> channels (128 bytes of 16-bit values, swizzled; all 128 of fp32) x kBoxTok<T> tokens.
constexpr uint32_t kChunkBytes = 16384;
constexpr int kChunkBufs = 3;
constexpr uint32_t kStagingBytes = kChunkBufs * kChunkBytes;
template <typename T>
constexpr int kBoxTok = (int)(kChunkBytes / (2 * kRows * sizeof(T)));  // 32 of 16 bits, 16 of fp32
template <typename T>
constexpr int kBoxChannels = sizeof(T) == 2 ? 64 : kRows;
constexpr int kMaxRows = 1 << 30;          // tokens and channels: row numbers past a tile's end stay in int
constexpr uint32_t kSmemMax = 227 * 1024;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr uint64_t kInFlightNs = 100000ull;  // how long a CTA that gave up keeps its memory, far above a transfer's latency

// After the ring and the staged chunks: barriers full / empty per stage, accumulator full / empty (two),
// "MMAs done", chunk full / empty, the parts of a split tile; the TMEM address, the abort flag.
constexpr int kBarFull = 0, kBarEmpty = kMaxStages, kBarAccFull = 2 * kMaxStages, kBarAccEmpty = kBarAccFull + 2,
              kBarMmaDone = kBarAccEmpty + 2, kBarChunkFull = kBarMmaDone + 1, kBarChunkEmpty = kBarChunkFull + kChunkBufs,
              kBarParts = kBarChunkEmpty + kChunkBufs, kNumBars = kBarParts + 1;
constexpr uint32_t kOffTmem = 8 * kNumBars, kOffAbort = kOffTmem + 4, kTailBytes = kOffAbort + 4;

struct Args {
  int m, n;
  int tok, splits;          // tokens per tile, parts of k
  int n_tiles, t_tiles;     // tiles of channels and of tokens
  int k_steps;
  int stages, stage_bytes, x_bytes;  // x_bytes: this CTA's token rows of a stage
  int staging_bytes;        // staged chunks of y, or the parts sent by the cluster's other CTAs
  int acc_cols, tmem_cols;  // TMEM columns of an accumulator, and allocated
  int tma_store;            // y's rows start on 16-byte boundaries: TMA stores (else copied by the epilogue)
  int band;                 // token tiles walked together (see tile_of)
  const float* x_scale;
  const float* w_scale;
  void* y;
  int64_t y_stride;
  int* status;
  unsigned long long wait_ns;
  int early_w;              // the preceding kernel does not write w
  int stall;                // test only: the first CTA never loads its first stage
};

struct Waiter {
  volatile int* abort_flag;
  int* status;
  uint64_t limit_ns;
  // kCluster: the arrivals come from threads of another CTA.
  template <bool kCluster = false>
  __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) const {
    uint64_t t0 = 0;
    for (uint32_t i = 0;; ++i) {
      if (kCluster ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
      if ((i & 63) == 63) {
        if (*abort_flag) return false;
        const uint64_t now = globaltimer();
        if (t0 == 0) {
          t0 = now;
        } else if (now - t0 > limit_ns) {
          *abort_flag = 1;
          if (status) atomicOr(status, TMLA_STATUS_TIMEOUT);
          return false;
        }
      }
    }
  }
  // The same for a converged warp, with one verdict.
  template <bool kCluster = false>
  __device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity) const {
    return __all_sync(0xffffffffu, wait<kCluster>(bar, parity));
  }
};
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity) && globaltimer() - t0 < limit_ns) {
  }
}

// Tile number i as (channel tile, token tile).  Tiles that run at the same time are neighbours in bands
// of `band` token tiles x all channel tiles, so that both operands are re-read from L2.
__device__ __forceinline__ void tile_of(const Args& a, int i, int& tn, int& tt) {
  const int per = a.band * a.n_tiles;
  const int b = i / per, r = i - b * per;
  const int rest = a.t_tiles - b * a.band, width = rest < a.band ? rest : a.band;
  tn = r / width;
  tt = b * a.band + (r - tn * width);
}

__device__ __forceinline__ void put(float v, float* y) { *y = v; }
__device__ __forceinline__ void put(float v, __nv_bfloat16* y) { *y = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(float v, __half* y) { *y = __float2half_rn(v); }

// The scale of a token (of the last one for a row past the end, whose products are never written).
__device__ __forceinline__ float token_scale(const Args& a, int token) { return a.x_scale[min(token, a.m - 1)]; }

__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// (a0 b0 c, a1 b1 c) as two packed products.
__device__ __forceinline__ float2 scale2(float a0, float a1, float2 b, float c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %6};\n\t"
      "mul.rn.f32x2 a, a, b;\n\tmul.rn.f32x2 a, a, c;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a0), "f"(a1), "f"(b.x), "f"(b.y), "f"(c));
  return r;
}

// Past a wait for TMEM loads: their registers are read after it.
template <int N>
__device__ __forceinline__ void loaded(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// A warp's share of a box of tokens: its 32 channels x half of the tokens.
// 16-bit y: 16 tokens.  The 16x256b loads leave the accumulator in the registers as 8 x 8 matrices of
// channels x tokens, which stmatrix writes transposed into 128-byte swizzled rows of 64 channels.
// fp32 y: 8 tokens, a thread's channel straight into rows of 128 channels.
// `scales` holds the scale of box token i in thread i.
template <typename T>
struct Share {
  uint32_t r[16];
  __device__ __forceinline__ void load(uint32_t acc) {
    tmem_ld16x256_x2(acc, *reinterpret_cast<uint32_t(*)[8]>(r));
    tmem_ld16x256_x2(acc + (16u << 16), *reinterpret_cast<uint32_t(*)[8]>(r + 8));
  }
  __device__ __forceinline__ void loaded() { linear_int8::loaded(r); }
  // The channels whose scales a thread needs (of its warp's 32), and how many.
  static constexpr int kScales = 4;
  static __device__ __forceinline__ int channel(int j, int lane) { return 8 * j + (lane >> 2); }
  __device__ __forceinline__ void put(uint32_t stage, float scales, const float (&ws)[kScales], int quarter, int sub,
                                      int lane) const {
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      s[j] = __shfl_sync(0xffffffffu, scales, 16 * sub + 8 * (j >> 1) + 2 * (lane & 3) + (j & 1));
    const T* t = nullptr;
    const int mat = lane >> 3, mrow = lane & 7;
    const uint32_t row =
        stage + (uint32_t)((quarter >> 1) * kBoxTok<T> + 16 * sub + 8 * (mat >> 1) + mrow) * 128;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t* q = r + 8 * h + 4 * j;
        const float2 st = make_float2(s[2 * j], s[2 * j + 1]);
        const float2 lo = scale2((float)(int)q[0], (float)(int)q[1], st, ws[2 * h]);
        const float2 hi = scale2((float)(int)q[2], (float)(int)q[3], st, ws[2 * h + 1]);
        v[2 * j] = pack2(lo.x, lo.y, t);
        v[2 * j + 1] = pack2(hi.x, hi.y, t);
      }
      const uint32_t chunk16 = (uint32_t)((quarter & 1) * 4 + h * 2 + (mat & 1));
      stmatrix_x4_trans(row + ((chunk16 ^ (uint32_t)mrow) << 4), v[0], v[1], v[2], v[3]);
    }
  }
};
template <>
struct Share<float> {
  uint32_t r[8];
  __device__ __forceinline__ void load(uint32_t acc) { tmem_ld8(acc, r); }
  __device__ __forceinline__ void loaded() { linear_int8::loaded(r); }
  static constexpr int kScales = 1;
  static __device__ __forceinline__ int channel(int, int lane) { return lane; }
  __device__ __forceinline__ void put(uint32_t stage, float scales, const float (&ws)[kScales], int quarter, int sub,
                                      int lane) const {
    const uint32_t at = stage + (uint32_t)(8 * sub * kRows + quarter * 32 + lane) * 4;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 s = make_float2(__shfl_sync(0xffffffffu, scales, 8 * sub + j),
                                   __shfl_sync(0xffffffffu, scales, 8 * sub + j + 1));
      const float2 v = scale2((float)(int)r[j], (float)(int)r[j + 1], s, ws[0]);
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + (uint32_t)(j * kRows * 4)), "f"(v.x) : "memory");
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + (uint32_t)((j + 1) * kRows * 4)), "f"(v.y) : "memory");
    }
  }
};

// Row `i` of a staged chunk (128 channels) to y, of which `left` channels exist: for rows of y that TMA
// cannot store to.  All 32 threads of a warp.
template <typename T>
__device__ __forceinline__ void copy_row(const uint8_t* chunk, int i, T* y, int left, int lane) {
  if constexpr (sizeof(T) == 4) {
    const float* row = reinterpret_cast<const float*>(chunk) + i * kRows;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (32 * b + lane < left) y[32 * b + lane] = row[32 * b + lane];
  } else {
    constexpr int kBoxBytes = kBoxTok<T> * 128;
    const uint8_t* box = chunk + (i / kBoxTok<T>) * (kChunkBytes / 2) + (i % kBoxTok<T>) * 128;
    // Word `lane` of each box holds channels 2 lane, 2 lane + 1 (and 64 on).
    const int at = (((lane >> 2) ^ (i & 7)) << 4) + (lane & 3) * 4;
    uint32_t w[2];
    w[0] = *reinterpret_cast<const uint32_t*>(box + at);
    w[1] = *reinterpret_cast<const uint32_t*>(box + kBoxBytes + at);
    const int odd = (int)(((uintptr_t)y >> 1) & 1);
    uint16_t* out = reinterpret_cast<uint16_t*>(y);
    if (odd) {
      // Whole words of y hold channels 2 j + 1, 2 j + 2; the first channel is written alone.
      const uint32_t next0 = __shfl_sync(0xffffffffu, lane == 0 ? w[1] : w[0], (lane + 1) & 31);
      const uint32_t next1 = __shfl_sync(0xffffffffu, w[1], (lane + 1) & 31);
      if (lane == 0 && left > 0) out[0] = (uint16_t)w[0];
      w[0] = __byte_perm(w[0], next0, 0x5432);
      w[1] = __byte_perm(w[1], next1, 0x5432);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int ch = 64 * b + 2 * lane + odd;
      if (ch + 1 < left && ch + 1 < kRows)
        *reinterpret_cast<uint32_t*>(out + ch) = w[b];
      else if (ch < left && ch < kRows)
        out[ch] = (uint16_t)w[b];
    }
  }
}

template <typename T, int kGroup>
__global__ void __launch_bounds__(kThreads, 1) int8_kernel(const __grid_constant__ CUtensorMap tm_w,
                                                        const __grid_constant__ CUtensorMap tm_x,
                                                        const __grid_constant__ CUtensorMap tm_y, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t staging = base + (uint32_t)(a.stages * a.stage_bytes);
  const uint32_t tail = staging + (uint32_t)a.staging_bytes;
  uint8_t* tail_ptr = smem_raw + (tail - raw);
  auto bar = [&](int i) { return tail + 8u * (uint32_t)i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail_ptr + kOffAbort);

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int cluster_size = kGroup * a.splits;
  const int rank = cluster_size > 1 ? (int)cluster_ctarank() : 0;
  const int half = rank % kGroup, split = rank / kGroup;
  const bool leader = half == 0;
  const int cluster = (int)blockIdx.x / cluster_size, clusters = (int)gridDim.x / cluster_size;
  const int tiles = a.n_tiles * a.t_tiles;
  // The token columns of a split tile in groups of 4: `per` for each part, of which this part adds up parts_here.
  const int per = (a.tok / 4 + a.splits - 1) / a.splits;
  const int parts_here = a.splits > 1 ? max(0, min(per, a.tok / 4 - split * per)) : 0;
  const int ks0 = (int)((long long)split * a.k_steps / a.splits);
  const int ks1 = (int)((long long)(split + 1) * a.k_steps / a.splits);

  // Warp 0's part before the roles start: the barriers, and the loads of the first round of the ring.
  const uint32_t elected = elect_one();
  const bool stalled = a.stall && blockIdx.x == 0;
  // A weight row is used by one token tile only, or again by the next ones.
  const uint64_t pol_w = a.t_tiles == 1 ? policy_evict_first() : policy_evict_normal();
  const uint64_t pol_x = policy_evict_last();  // every channel tile re-reads it (2000 x 12000 x 6000: 132 us, else 150)
  const uint32_t pair_bar = kGroup == 2 ? map_to_rank(bar(0), (uint32_t)(rank - half)) : bar(0);
  auto load_w = [&](int s, int ks, int row) {
    if (leader) mbar_arrive_expect_tx(bar(kBarFull + s), (uint32_t)(kGroup * (kWBytes + a.x_bytes)), elected);
    tma_load_2d<kGroup>(base + (uint32_t)(s * a.stage_bytes), &tm_w, pair_bar + 8u * (uint32_t)(kBarFull + s),
                        ks * kBoxK, row, pol_w, elected);
  };
  auto load_x = [&](int s, int ks, int row) {
    tma_load_2d<kGroup>(base + (uint32_t)(s * a.stage_bytes + kWBytes), &tm_x,
                        pair_bar + 8u * (uint32_t)(kBarFull + s), ks * kBoxK, row, pol_x, elected);
  };
  const int pre = ks1 - ks0 < a.stages ? ks1 - ks0 : a.stages;
  auto first_round = [&]() {
    int tn, tt;
    tile_of(a, cluster, tn, tt);
    const int w_row = (tn * kGroup + half) * kRows, x_row = tt * a.tok + half * (a.tok / kGroup);
    // With the caller's word that the kernel before does not write w, the weight boxes of two stages are
    // requested before it has completed; more of them would delay its own loads.
    const int early = !a.early_w ? 0 : pre < 2 ? pre : 2;
    for (int s = 0; s < early; ++s)
      if (!stalled || s > 0) load_w(s, ks0 + s, w_row);
    // Into L2 the weights may come at any time (a write by the kernel before would update them there).
    for (int s = early; s < pre && s < kPrefetch; ++s) tma_prefetch_2d(&tm_w, (ks0 + s) * kBoxK, w_row, elected);
    griddep_wait();
    // Only now may the next kernel be scheduled: its loads ahead of its own wait count on every kernel before this one
    // having completed.  A single CTA holds its TMEM first, so that the next one cannot keep it out.
    if (kGroup == 2) griddep_launch_dependents();
    for (int s = 0; s < pre; ++s) {
      if (s >= early && (!stalled || s > 0)) load_w(s, ks0 + s, w_row);
      if (!stalled || s > 0) load_x(s, ks0 + s, x_row);
    }
  };
  if (warp == 0) {
    for (int i = lane; i < kNumBars; i += 32) {
      const int count = i >= kBarAccEmpty && i < kBarMmaDone       ? kGroup * kEpiWarps
                        : i >= kBarChunkFull && i < kBarChunkEmpty ? kEpiWarps
                        : i >= kBarChunkEmpty && i < kBarParts     ? (a.tma_store ? 1 : kEpiWarps)
                                                                   : 1;
      mbar_init(bar(i), (uint32_t)count);
    }
    if (lane == 0) *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    __syncwarp();
    if (parts_here > 0)
      mbar_arrive_expect_tx(bar(kBarParts), (uint32_t)((a.splits - 1) * parts_here * kRows * 16), elected);
    if (kGroup == 1) first_round();  // a single CTA's loads concern nobody else
  } else if (warp == 1) {
    tmem_alloc_g<kGroup>(tail + kOffTmem, (uint32_t)a.tmem_cols);
    tmem_relinquish_g<kGroup>();
  }
  tc_fence_before();
  __syncthreads();
  // The cluster's CTAs have set up their barriers when this completes: a pair needs that at once, the parts
  // of a split tile before they are sent.
  if (cluster_size > 1) cluster_arrive();
  if (kGroup == 2) cluster_wait();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tail_ptr + kOffTmem);
  const Waiter waiter{abort_flag, a.status, a.wait_ns};

  if (warp == 0) {
    // The whole warp runs this (its operands stay warp-uniform); one thread issues.
    if (kGroup == 1)
      griddep_launch_dependents();  // first_round has waited
    else
      first_round();
    int s = pre == a.stages ? 0 : pre;               // ring position, and how often the ring has wrapped
    uint32_t round = pre == a.stages ? 1 : 0;
    bool ok = true;
    for (int t = cluster; t < tiles && ok; t += clusters) {
      int tn, tt;
      tile_of(a, t, tn, tt);
      const int w_row = (tn * kGroup + half) * kRows, x_row = tt * a.tok + half * (a.tok / kGroup);
      for (int ks = t == cluster ? ks0 + pre : ks0; ks < ks1; ++ks) {
        if (round > 0) ok = waiter.wait_warp(bar(kBarEmpty + s), (round - 1) & 1);
        if (!ok) break;
        load_w(s, ks, w_row);
        load_x(s, ks, x_row);
        if (++s == a.stages) s = 0, ++round;
      }
    }
    if (!ok && leader) {
      // Let the copies in flight land before the CTA can exit.  (A wait gives up in a later round than
      // the first, so every stage has been loaded.)
      for (int j = 0; j < a.stages; ++j)
        drain_wait(bar(kBarFull + j), (j < s ? round : round - 1) & 1, a.wait_ns);
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp runs this (its operands stay warp-uniform); one thread issues.
    if (leader) {
      griddep_wait();  // a bounded wait below must not count the time of the kernel before
      const uint32_t idesc = idesc_i8(kRows * kGroup, (uint32_t)a.tok);
      const uint16_t mask = (uint16_t)(3u << (rank - half));
      int iter = 0, s = 0;
      uint32_t phase = 0;  // parity of the ring's current round
      bool ok = true, issued = false;
      for (int t = cluster; t < tiles && ok; t += clusters, ++iter) {
        const int buf = iter & 1;
        if (iter >= 2) ok = waiter.wait_warp<(kGroup == 2)>(bar(kBarAccEmpty + buf), (uint32_t)((iter >> 1) - 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf * a.acc_cols);
        for (int ks = ks0; ks < ks1; ++ks) {
          ok = waiter.wait_warp(bar(kBarFull + s), phase);
          if (!ok) break;
          tc_fence_after();
          const uint32_t st = base + (uint32_t)(s * a.stage_bytes);
          mma_i8_k128<kGroup>(d, smem_desc(st, 16, 1024, kSwizzle128B),
                              smem_desc(st + kWBytes, 16, 1024, kSwizzle128B),
                              idesc, ks > ks0 ? 1u : 0u, elected);
          issued = true;
          mma_commit_g<kGroup>(bar(kBarEmpty + s), mask, elected);
          if (++s == a.stages) s = 0, phase ^= 1;
        }
        if (!ok) break;
        mma_commit_g<kGroup>(bar(kBarAccFull + buf), mask, elected);
      }
      if (!ok && issued) {
        mma_commit_g<kGroup>(bar(kBarMmaDone), (uint16_t)(1u << rank), elected);
        drain_wait(bar(kBarMmaDone), 0, a.wait_ns);
      }
    }
    __syncwarp();
  } else if (warp < kStoreWarp) {
    // Epilogue: two warps per 32 channels (TMEM lanes), which share the token columns.
    const int sub = (warp - 2) >> 2, quarter = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    griddep_wait();
    int iter = 0, buf_at = 0;
    uint32_t buf_round = 0;
    bool ok = true;
    // This thread's channel scales, a tile ahead, and its tokens' (one of each box) a chunk ahead.
    float ws_next[Share<T>::kScales], s_next[2];
    int tn, tt;
    auto request_tokens = [&](int token) {
      s_next[0] = token_scale(a, token + lane % kBoxTok<T>);
      s_next[1] = token_scale(a, token + kBoxTok<T> + lane % kBoxTok<T>);
    };
    auto request = [&](int t) {
      tile_of(a, t, tn, tt);
#pragma unroll
      for (int j = 0; j < Share<T>::kScales; ++j) {
        const int ch = (tn * kGroup + half) * kRows + quarter * 32 + Share<T>::channel(j, lane);
        ws_next[j] = ch < a.n ? a.w_scale[ch] : 0.f;
      }
    };
    request(cluster);
    for (int t = cluster; t < tiles && ok; t += clusters, ++iter) {
      const int buf = iter & 1;
      const int tn_now = tn, token0 = tt * a.tok;
      float ws[Share<T>::kScales];
#pragma unroll
      for (int j = 0; j < Share<T>::kScales; ++j) ws[j] = ws_next[j];
      if (t + clusters < tiles) request(t + clusters);
      request_tokens(token0);
      ok = waiter.wait_warp(bar(kBarAccFull + buf), (uint32_t)(iter >> 1) & 1);
      if (!ok || a.splits > 1) break;
      tc_fence_after();
      const uint32_t acc = lanes + (uint32_t)(buf * a.acc_cols);
      constexpr int kTok = kBoxTok<T>;
      for (int c = 0; c < a.tok; c += 2 * kTok) {
        const int at = c + sub * (kTok / 2);
        const bool second = c + kTok < a.tok;
        Share<T> part[2];
        part[0].load(acc + (uint32_t)at);
        if (second) part[1].load(acc + (uint32_t)(at + kTok));
        const float s0 = s_next[0], s1 = s_next[1];
        if (c + 2 * kTok < a.tok) request_tokens(token0 + c + 2 * kTok);
        tc_wait_ld();
        part[0].loaded();
        part[1].loaded();
        if (c + 2 * kTok >= a.tok) {  // the accumulator has been read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (kGroup == 2)
              mbar_arrive_cluster(map_to_rank(bar(kBarAccEmpty + buf), (uint32_t)(rank - half)));
            else
              mbar_arrive(bar(kBarAccEmpty + buf));
          }
        }
        if (buf_round > 0) ok = waiter.wait_warp(bar(kBarChunkEmpty + buf_at), (buf_round - 1) & 1);
        if (!ok) break;
        const uint32_t stage = staging + (uint32_t)buf_at * kChunkBytes;
        part[0].put(stage, s0, ws, quarter, sub, lane);
        if (second) part[1].put(stage + kChunkBytes / 2, s1, ws, quarter, sub, lane);
        if (a.tma_store) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBarChunkFull + buf_at));
        if (!a.tma_store) {
          ok = waiter.wait_warp(bar(kBarChunkFull + buf_at), buf_round & 1);
          if (!ok) break;
          const int tokens = min(min(2 * kTok, a.tok - c), a.m - token0 - c);
          const uint8_t* rows = smem_raw + (stage - raw);
          const int ch = (tn_now * kGroup + half) * kRows, left = a.n - ch;
          for (int i = warp - 2; i < tokens; i += kEpiWarps)
            copy_row<T>(rows, i, static_cast<T*>(a.y) + (int64_t)(token0 + c + i) * a.y_stride + ch, left, lane);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kBarChunkEmpty + buf_at));
        }
        if (++buf_at == kChunkBufs) buf_at = 0, ++buf_round;
      }
    }
    if (a.splits > 1) {
      // One tile per cluster: this part's columns to the CTAs that add them up, in groups of 4 token
      // columns, [part][group][channel] x 16 bytes, which complete on their barrier.
      const int row = quarter * 32 + lane, channel = (tn * kGroup + half) * kRows + row, token0 = tt * a.tok;
      const bool live = channel < a.n;
      const float w_scale = live ? a.w_scale[channel] : 0.f;
      // The scales of the columns that this part adds up (at most 128: thread i has those of i, i + 32, ...).
      const int first = 4 * split * per, cols = 4 * parts_here;
      float s_own[kMaxTok / 64];
#pragma unroll
      for (int i = 0; i < kMaxTok / 64; ++i) s_own[i] = token_scale(a, token0 + first + 32 * i + lane);
      if (kGroup == 1) cluster_wait();
      if (ok) {
        const uint32_t per_inv = (65536u + (uint32_t)per - 1) / (uint32_t)per;  // g / per = g per_inv >> 16 for g < 64
        tc_fence_after();
        for (int c = sub * 16; c < a.tok; c += 32) {
          uint32_t r[16];
          tmem_ld16(lanes + (uint32_t)c, r);
          tc_wait_ld();
          loaded(r);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int g = c / 4 + j, owner = (int)(((uint32_t)g * per_inv) >> 16);
            if (owner == split) continue;
            const int part = split < owner ? split : split - 1;
            const uint32_t to = (uint32_t)(owner * kGroup + half);
            st_async_u4(map_to_rank(staging + (uint32_t)(((part * per + g - owner * per) * kRows + row) * 16), to),
                        make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]),
                        map_to_rank(bar(kBarParts), to));
          }
        }
      }
      __syncwarp();
      cluster_arrive();  // everything sent; completed at the end, before any CTA exits
      if (parts_here > 0 && ok && waiter.wait_warp<true>(bar(kBarParts), 0)) {
        T* y = static_cast<T*>(a.y) + (int64_t)(token0 + first) * a.y_stride + channel;
        const uint8_t* parts = smem_raw + (staging - raw) + (size_t)row * 16;
        const int tokens = min(cols, a.m - token0 - first);
#pragma unroll
        for (int i = 0; i < kMaxTok / 64; ++i) {
          const int c = 32 * i + 16 * sub;  // 16 columns, all of their loads in flight at once
          if (c >= cols) break;
          uint32_t r[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + 4 * j < cols) tmem_ld4(lanes + (uint32_t)(first + c + 4 * j), r[j]);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 4; ++j) loaded(r[j]);
          for (int p = 0; p < a.splits - 1; ++p) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (c + 4 * j >= cols) break;
              const uint4 v = *reinterpret_cast<const uint4*>(parts + (size_t)(p * per + c / 4 + j) * kRows * 16);
              r[j][0] += v.x, r[j][1] += v.y, r[j][2] += v.z, r[j][3] += v.w;
            }
          }
          // All values first, then the stores: a store under a condition between two shuffles costs 100 cycles.
          T v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j)
            put((float)(int)r[j / 4][j % 4] * __shfl_sync(0xffffffffu, s_own[i], 16 * sub + j) * w_scale, v + j);
          if (live) {
            T* yc = y + c * a.y_stride;
            if (c + 16 <= tokens) {
#pragma unroll
              for (int j = 0; j < 16; ++j) yc[j * a.y_stride] = v[j];
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (c + j < tokens) yc[j * a.y_stride] = v[j];
            }
          }
          __syncwarp();
        }
      }
    }
    __syncwarp();
  } else if (a.tma_store) {
    // The store warp: a staged chunk to y by TMA, and the buffer of the chunk before back, which has been read.
    constexpr int kTok = kBoxTok<T>;
    griddep_wait();
    int at = 0, before = -1;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = cluster; t < tiles && ok; t += clusters) {
      int tn, tt;
      tile_of(a, t, tn, tt);
      const int channel0 = (tn * kGroup + half) * kRows, token0 = tt * a.tok;
      for (int c = 0; c < a.tok; c += 2 * kTok) {
        ok = waiter.wait_warp(bar(kBarChunkFull + at), phase);
        if (!ok) break;
        const uint32_t stage = staging + (uint32_t)at * kChunkBytes;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int token = c + i * kTok;
          if (token >= a.tok || token0 + token >= a.m) break;
#pragma unroll
          for (int b = 0; b < kRows / kBoxChannels<T>; ++b) {
            const int ch = channel0 + b * kBoxChannels<T>;
            if (ch < a.n)
              tma_store_2d(&tm_y, stage + i * (kChunkBytes / 2) + b * kTok * 128, ch, token0 + token, elected);
          }
        }
        if (elected) {
          bulk_commit_group();
          bulk_wait_group_read<1>();
          if (before >= 0) mbar_arrive(bar(kBarChunkEmpty + before));
        }
        __syncwarp();
        before = at;
        if (++at == kChunkBufs) at = 0, phase ^= 1;
      }
    }
    if (elected) bulk_wait_group0();
    __syncwarp();
  }

  __syncwarp();
  if (cluster_size > 1) {
    // No CTA exits while another may still write to its shared memory or use its half of a pair's operands.
    if (a.splits == 1 || warp < 2 || warp == kStoreWarp) {
      if (kGroup == 1) cluster_wait();
      cluster_arrive();
    }
    cluster_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    // A CTA that gave up has not waited for all that is on its way to it: the parts of a split tile (the cluster barrier
    // orders their sending, not their landing), a pair's arrivals, copies past a short limit.  It keeps its shared memory
    // and TMEM for as long as they can take: a CTA that exits under a landing transfer loses the context.
    if (*abort_flag) {
      const uint64_t t0 = globaltimer();
      while (globaltimer() - t0 < kInFlightNs) {
      }
      __syncwarp();
    }
    tc_fence_after();
    tmem_dealloc_g<kGroup>(tmem, (uint32_t)a.tmem_cols);
  }
}

// ---------------------------------------------------------------------------- CUDA-core kernel
// Rows of any alignment.  A block computes 64 tokens x 64 channels, 4 x 4 per thread, from 64
// columns at a time in shared memory, four products per dp4a.
constexpr int kTile = 64, kStep = 64, kWords = kStep / 4;

struct GenericArgs {
  const int8_t* x;
  int64_t x_stride;
  const float* x_scale;
  const int8_t* w;
  int64_t w_stride;
  const float* w_scale;
  void* y;
  int64_t y_stride;
  int m, n, k;
};

// Columns [k0, k0 + 64) of rows [r0, r0 + 64), zeros outside the matrix.
__device__ __forceinline__ void stage(int (&dst)[kTile][kWords + 1], const int8_t* src, int64_t stride, int r0,
                                      int rows, int k0, int k) {
  for (int i = threadIdx.x; i < kTile * kStep; i += blockDim.x) {
    const int r = i / kStep, c = i % kStep;
    const int8_t v = r0 + r < rows && k0 + c < k ? src[(int64_t)(r0 + r) * stride + k0 + c] : (int8_t)0;
    reinterpret_cast<int8_t*>(dst[r])[c] = v;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) generic_kernel(const GenericArgs a) {
  __shared__ int xs[kTile][kWords + 1], ws[kTile][kWords + 1];
  const int j0 = blockIdx.x * kTile;
  const int tj = threadIdx.x % 16, ti = threadIdx.x / 16;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  for (int i0 = blockIdx.y * kTile; i0 < a.m; i0 += gridDim.y * kTile) {
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.k; k0 += kStep) {
      __syncthreads();
      stage(xs, a.x, a.x_stride, i0, a.m, k0, a.k);
      stage(ws, a.w, a.w_stride, j0, a.n, k0, a.k);
      __syncthreads();
#pragma unroll 4
      for (int c = 0; c < kWords; ++c) {
        int xv[4], wv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[i] = xs[ti + 16 * i][c], wv[i] = ws[tj + 16 * i][c];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(xv[i], wv[j], acc[i][j]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i0 + ti + 16 * i;
      if (row >= a.m) continue;
      const float sx = a.x_scale[row];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = j0 + tj + 16 * j;
        if (col < a.n)
          put((float)acc[i][j] * sx * a.w_scale[col], static_cast<T*>(a.y) + (int64_t)row * a.y_stride + col);
      }
    }
  }
}

template <typename T>
cudaError_t launch_generic(const GenericArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  const int rows = (a.m + kTile - 1) / kTile;
  cfg.gridDim = dim3((unsigned)((a.n + kTile - 1) / kTile), (unsigned)(rows < 65535 ? rows : 65535));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, generic_kernel<T>, a);
}

// ---------------------------------------------------------------------------- host side
struct Plan {
  int group, tok, splits, stages;
};

// The parts of a split tile's columns that a CTA receives, or the staged chunks of y.
int staging_bytes(const Plan& p) {
  return p.splits == 1 ? (int)kStagingBytes : (p.splits - 1) * ((p.tok / 4 + p.splits - 1) / p.splits) * kRows * 16;
}

// Clusters of 1 to 8 CTAs that run at once on 148 SMs with one CTA each (the occupancy calculator's).
constexpr int kClusters[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};

// Estimated microseconds of a call, up to a constant.  The tiles run in waves; a k-step of a tile takes the
// longer of its MMAs and the fill of a CTA's shared memory, an unsplit tile at least the epilogue of the tile
// before it.  HBM's time for the operands and y overlaps in part; further token tiles read the weight again, from
// L2.  The constants are fitted to 5,700 calls measured on B200 (1 to 8000 tokens, n x k from 300 x 300 to
// 512 x 16384 and 24576 x 1536, every variant, bf16 out): the variant with the least estimate is on average
// 1.3% slower than the fastest measured, 7% or less in 95% of the sizes, 18% at worst.
double estimate(int m, int n, int k, int size, int group, int tok, int splits, int sms) {
  const double k_steps = (k + kBoxK - 1) / kBoxK, n_tiles = (n + kRows * group - 1) / (kRows * group),
               t_tiles = (m + tok - 1) / tok;
  const double slots = kClusters[group * splits] * (sms / 148.0);
  const double step = fmax(0.85 * tok, 6.8 * (16 + tok / 8.0 / group)) * 1e-3;
  const double epilogue = (4.06 * tok + 519.) * 1e-3, steps = ceil(k_steps / splits) * step;
  const double tiles_us = ceil(n_tiles * t_tiles / slots) * (splits == 1 ? fmax(steps, epilogue) : steps);
  const double hbm_us = ((double)n * k * (1 + 0.28 * (t_tiles - 1)) + (double)m * k + 0.34 * size * m * n) / 5.38e6;
  const double last = splits == 1 ? epilogue + (group == 2 ? 0.64 : 0.)
                                  : 0.985 + 0.0247 * tok + 0.082 * splits - (group == 2 ? 0.805 : 0.);
  return fmax(tiles_us, hbm_us) + 0.28 * fmin(tiles_us, hbm_us) + last;
}

// The variant with the least estimate.  Examples (us measured, the chosen one first):
//   wo (7168 x 16384), 16 tokens: pairs in 2 parts 21.3, single CTAs in 2 parts 22.5, unsplit 25.1;
//   64 tokens: pairs in 2 parts 21.8, single CTAs in 2 parts 24.1, unsplit 26.6;  256 tokens: pairs of 256 in 2
//   parts 30.4, pairs of 128 33.4, single CTAs of 128 37.3;
//   [wq_a; wkv_a] (2112 x 7168), 16 tokens: pairs in 4 parts 6.6, single CTAs in 6 parts 6.7, unsplit 10.3;
//   wq_b (24576 x 1536), 4096 tokens: pairs of 256 105, single CTAs 130;
//   20000 x 128, 4096 tokens: single CTAs 45, pairs 54;  32768 x 512, 4096 tokens: single CTAs 81, pairs 92;
//   4001 x 2001, 77 tokens: single CTAs of 64 tokens 5.9, pairs of 96 in 2 parts 6.3, pairs of 64 in 2 parts 7.0.
Plan make_plan(int m, int n, int k, int size, int sms) {
  constexpr int kTokens[] = {64, 96, 128, 160, 192, 224, 256}, kSplits[] = {1, 2, 3, 4, 6};
  Plan best{};
  double least = 0;
  const int k_steps = (k + kBoxK - 1) / kBoxK;
  for (int group = 1; group <= 2; ++group) {
    for (int i = 0; i < 7; ++i) {
      // Up to 64 tokens one tile holds them all, in steps of the MMA's N.
      const int step = 16 * group, tok = m <= 64 ? (m + step - 1) / step * step : kTokens[i];
      if (i > 0 && (m <= 64 || kTokens[i - 1] >= m)) break;
      for (const int splits : kSplits) {
        if (splits * group > kMaxSplits || splits > k_steps) break;
        // Split tiles run once each, so all at once or not at all (wq_b, 192 tiles: unsplit 8.6 us, two parts 18.6).
        const long long tiles = (long long)((n + kRows * group - 1) / (kRows * group)) * ((m + tok - 1) / tok);
        if (splits > 1 && tiles * 148 > (long long)kClusters[group * splits] * sms) break;
        const double t = estimate(m, n, k, size, group, tok, splits, sms);
        if (best.group == 0 || t < least) best = Plan{group, tok, splits, 0}, least = t;
      }
    }
  }
  const int stage = (kRows + best.tok / best.group) * kBoxK;
  best.stages = ((int)(kSmemMax - 1024 - kTailBytes) - staging_bytes(best)) / stage;
  if (best.stages > kMaxStages) best.stages = kMaxStages;
  return best;
}

// A matrix of int8 rows as a map of boxes of `rows` rows x 128 swizzled bytes; outside it reads zeros.
int encode(CUtensorMap* map, const void* base, int k, int rows, int64_t stride, int box_rows) {
  auto fn = sm100::encode_fn();
  if (!fn) return TMLA_ERR_CUDA;
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)stride};
  cuuint32_t box[2] = {kBoxK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : TMLA_ERR_MISALIGNED;
}

// The output as a map of its staged boxes.
template <typename T>
int encode_y(CUtensorMap* map, const TmlaLinearInt8Params& p) {
  auto fn = sm100::encode_fn();
  if (!fn) return TMLA_ERR_CUDA;
  const CUtensorMapDataType dt = p.dtype == TMLA_DTYPE_FP32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : p.dtype == TMLA_DTYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  cuuint64_t dims[2] = {(cuuint64_t)p.n, (cuuint64_t)p.m};
  cuuint64_t strides[1] = {(cuuint64_t)p.y_stride * sizeof(T)};
  cuuint32_t box[2] = {kBoxChannels<T>, kBoxTok<T>};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, dt, 2, p.y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  sizeof(T) == 2 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : TMLA_ERR_MISALIGNED;
}

template <typename T, int kGroup>
cudaError_t launch_tc(const CUtensorMap& tw, const CUtensorMap& tx, const CUtensorMap& ty, const Args& a, int clusters,
                      size_t smem, int device, cudaStream_t stream) {
  // The kernel's shared-memory limit is raised once on each device.
  static std::atomic<uint64_t> raised{0};
  const uint64_t bit = 1ull << (device & 63);
  if (!(raised.load(std::memory_order_relaxed) & bit)) {
    cudaError_t e =
        cudaFuncSetAttribute(int8_kernel<T, kGroup>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax);
    if (e != cudaSuccess) return e;
    if (device < 64) raised.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  const int size = kGroup * a.splits;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)size;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(clusters * size));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = size > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, int8_kernel<T, kGroup>, tw, tx, ty, a);
}

template <typename T>
cudaError_t launch(const TmlaLinearInt8Params& p, const Plan& pl, const CUtensorMap& tw, const CUtensorMap& tx, int sms,
                   int device, cudaStream_t stream) {
  Args a;
  a.m = p.m;
  a.n = p.n;
  a.tok = pl.tok;
  a.splits = pl.splits;
  a.n_tiles = (p.n + kRows * pl.group - 1) / (kRows * pl.group);
  a.t_tiles = (p.m + pl.tok - 1) / pl.tok;
  a.k_steps = (p.k + kBoxK - 1) / kBoxK;
  a.x_bytes = pl.tok / pl.group * kBoxK;
  a.stages = pl.stages;
  a.stage_bytes = kRows * kBoxK + a.x_bytes;
  a.staging_bytes = staging_bytes(pl);
  if ((long long)a.n_tiles * a.t_tiles > kMaxRows) return cudaErrorInvalidValue;  // a y beyond any memory
  const int tiles = a.n_tiles * a.t_tiles;
  const int resident = sms / pl.group;
  const int clusters = pl.splits > 1 || tiles < resident ? tiles : resident;
  a.acc_cols = (pl.tok + 31) / 32 * 32;
  const int cols = a.acc_cols * (tiles > clusters ? 2 : 1);
  for (a.tmem_cols = 32; a.tmem_cols < cols;) a.tmem_cols *= 2;
  a.band = a.t_tiles < 8 ? a.t_tiles : 8;
  a.x_scale = p.x_scale;
  a.w_scale = p.w_scale;
  a.y = p.y;
  a.y_stride = p.y_stride;
  a.status = p.status;
  a.wait_ns = p.wait_ns > 0 ? (unsigned long long)p.wait_ns : kWaitNs;
  a.early_w = (p.flags & TMLA_LAYER_FLAG_PDL) != 0;
  a.stall = (p.flags & TMLA_LINEAR_FLAG_TEST_STALL) ? 1 : 0;
  // What the kernel takes for granted.
  if (a.stages < 1 || pl.splits > a.k_steps || pl.splits * pl.group > kMaxSplits || pl.tok > kMaxTok ||
      pl.tok % (16 * pl.group))
    return cudaErrorInvalidValue;
  // TMA stores need rows of y on 16-byte boundaries and write them in 16-byte units, past column n too
  // (clipping is not by the element there), and they write whole boxes of tokens: past a tile's end
  // only where that is past y's end.
  CUtensorMap ty = tx;
  const int64_t size = sizeof(T);
  a.tma_store = pl.splits == 1 && (p.n * size % 16 == 0 || (p.flags & TMLA_LINEAR_FLAG_PAD_Y)) &&
                (pl.tok % kBoxTok<T> == 0 || a.t_tiles == 1) && (uintptr_t)p.y % 16 == 0 && p.y_stride * size % 16 == 0 &&
                encode_y<T>(&ty, p) == 0;
  const size_t smem = 1024 + (size_t)a.stages * a.stage_bytes + a.staging_bytes + kTailBytes;
  return pl.group == 1 ? launch_tc<T, 1>(tw, tx, ty, a, clusters, smem, device, stream)
                       : launch_tc<T, 2>(tw, tx, ty, a, clusters, smem, device, stream);
}

int start(const TmlaLinearInt8Params& p, cudaStream_t stream) {
  if (p.m < 0 || p.n < 0 || p.k < 1) return TMLA_ERR_INVALID_ARG;
  if (p.dtype != TMLA_DTYPE_BF16 && p.dtype != TMLA_DTYPE_FP16 && p.dtype != TMLA_DTYPE_FP32)
    return TMLA_ERR_INVALID_ARG;
  if (p.k > TMLA_LINEAR_INT8_MAX_K || p.m > kMaxRows || p.n > kMaxRows) return TMLA_ERR_UNSUPPORTED;
  if (p.m == 0 || p.n == 0) return TMLA_OK;
  if (!p.x || !p.x_scale || !p.w || !p.w_scale || !p.y) return TMLA_ERR_INVALID_ARG;
  if (p.x_stride < p.k || p.w_stride < p.k || p.y_stride < p.n) return TMLA_ERR_INVALID_ARG;
  cudaError_t e;
  if ((((uintptr_t)p.x | (uintptr_t)p.w) % 16 || p.x_stride % 16 || p.w_stride % 16)) {
    const GenericArgs a{static_cast<const int8_t*>(p.x), p.x_stride, p.x_scale, static_cast<const int8_t*>(p.w),
                        p.w_stride, p.w_scale, p.y, p.y_stride, p.m, p.n, p.k};
    switch (p.dtype) {
      case TMLA_DTYPE_BF16: e = launch_generic<__nv_bfloat16>(a, stream); break;
      case TMLA_DTYPE_FP16: e = launch_generic<__half>(a, stream); break;
      default: e = launch_generic<float>(a, stream); break;
    }
  } else {
    int device = 0, sms = 0;
    e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return record_cuda_error(e);
    const Plan pl = make_plan(p.m, p.n, p.k, p.dtype == TMLA_DTYPE_FP32 ? 4 : 2, sms);
    CUtensorMap tw, tx;
    int rc = encode(&tw, p.w, p.k, p.n, p.w_stride, kRows);
    if (!rc) rc = encode(&tx, p.x, p.k, p.m, p.x_stride, pl.tok / pl.group);
    if (rc) return rc;
    switch (p.dtype) {
      case TMLA_DTYPE_BF16: e = launch<__nv_bfloat16>(p, pl, tw, tx, sms, device, stream); break;
      case TMLA_DTYPE_FP16: e = launch<__half>(p, pl, tw, tx, sms, device, stream); break;
      default: e = launch<float>(p, pl, tw, tx, sms, device, stream); break;
    }
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? TMLA_OK : record_cuda_error(e);
}

}  // namespace linear_int8
}  // namespace tmla

extern "C" int tmla_linear_int8_plan(int32_t m, int32_t n, int32_t k, int32_t dtype, int32_t num_sms, int32_t* plan) {
  using namespace tmla::linear_int8;
  if (m < 1 || n < 1 || k < 1 || num_sms < 1 || !plan) return TMLA_ERR_INVALID_ARG;
  if (dtype != TMLA_DTYPE_BF16 && dtype != TMLA_DTYPE_FP16 && dtype != TMLA_DTYPE_FP32) return TMLA_ERR_INVALID_ARG;
  if (k > TMLA_LINEAR_INT8_MAX_K || m > kMaxRows || n > kMaxRows) return TMLA_ERR_UNSUPPORTED;
  const Plan p = make_plan(m, n, k, dtype == TMLA_DTYPE_FP32 ? 4 : 2, num_sms);
  const long long tiles = (long long)((n + kRows * p.group - 1) / (kRows * p.group)) * ((m + p.tok - 1) / p.tok);
  const long long slots = num_sms / p.group;
  plan[0] = p.group;
  plan[1] = p.tok;
  plan[2] = p.splits;
  plan[3] = p.splits > 1 ? 1 : (int)((tiles + slots - 1) / slots);
  return TMLA_OK;
}

extern "C" int tmla_linear_int8(const TmlaLinearInt8Params* p, void* stream) {
  if (!p) return TMLA_ERR_INVALID_ARG;
  return tmla::linear_int8::start(*p, static_cast<cudaStream_t>(stream));
}
