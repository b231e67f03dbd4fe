// The 8-bit latent cache: sparse-MLA decode over it, the append that writes it, the
// accumulation of attention weights and the compaction that follows an eviction.
//
// Cache layout.  A slot's latent row is 512 e4m3 values (1 sign, 4 exponent, 3 mantissa bits;
// no infinities); every `block` consecutive slots of a page (a power of two that divides the
// page size) share one fp32 scale, so that
//     ckv[slot][d] = float(ckv_q8[slot][d]) * ckv_scale[slot / block].
// The 64 rope key values of a slot stay bf16: they are an eighth of the values, take no part in the
// output, and carry the positions' phases, which 3 mantissa bits would blur.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <utility>

#include "dsa_b200.h"
#include "dsa_common.cuh"
#include "dsa_host.cuh"
#include "sm100_ptx.cuh"

namespace dsa {
namespace q8 {

// A cache as the kernels see it.
struct Cache {
  uint8_t* ckv;
  int64_t ckv_ss;  // bytes between slots
  float* scale;    // one per block, consecutive
  __nv_bfloat16* kpe;
  int64_t kpe_ss;  // elements between slots
  int64_t num_slots;
  int32_t block_shift;  // log2(tokens per scale)
};

// A row-major int32 table of pool pages.
struct PageTable {
  const int32_t* pt;
  int64_t sb;
  int32_t cols;
  int32_t shift;  // log2(page size)
};

// The slot of token position `pos` of a row; -1 when the table has none for it or it lies
// outside the pool.
__device__ __forceinline__ int slot_at(const PageTable& t, int64_t row, int pos,
                                       int64_t num_slots) {
  const int pg = pos >> t.shift;
  if (pos < 0 || pg >= t.cols) return -1;
  const int32_t page = __ldg(t.pt + row * t.sb + pg);
  if (page < 0) return -1;
  const int64_t slot = ((int64_t)page << t.shift) | (int64_t)(pos & ((1 << t.shift) - 1));
  return slot < num_slots ? (int)slot : -1;
}

// Two floats rounded to e4m3 (nearest, ties to even; past 448 to 448; NaN stays NaN).
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two e4m3 values (exact in fp16).
__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// Eight bf16 values (16 bytes) as floats.
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// Sixteen e4m3 values times `ratio`, rounded to e4m3 again.
__device__ __forceinline__ uint4 rescale16(uint4 v, float ratio) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = from_e4m3x2(w[i] & 0xFFFFu), b = from_e4m3x2(w[i] >> 16);
    w[i] = to_e4m3x2(a.x * ratio, a.y * ratio) | (to_e4m3x2(b.x * ratio, b.y * ratio) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The smallest power of two s with amax <= 448 s, at least 2^-126 (so that 1 / s is finite).
// 448 = 1.75 * 2^8: with amax = m 2^e (1 <= m < 2), s = 2^(e - 8) when m <= 1.75, else 2^(e - 7).
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);  // biased
  return __uint_as_float((uint32_t)(e < 1 ? 1 : e) << 23);
}

}  // namespace q8
}  // namespace dsa

#include "dsa_q8_attend.cuh"

namespace dsa {
namespace q8 {

// ------------------------------------------------------------------------------- append
//
// Row r's new tokens [offsets[r], offsets[r + 1]) take the positions starts[r], starts[r] + 1,
// ... of its sequence.  The unit of work is one block of the cache that the call writes to
// (a job): its scale becomes the smallest power of two that holds every new token of the
// block, or the block's earlier scale if that is larger and the block has earlier tokens; if
// the scale grew, the earlier tokens are re-expressed in it (times old / new, an exact shift
// of the exponent for powers of two, except where a value becomes subnormal).  One CTA owns a
// job, so that the amax, the earlier tokens and the scale need no other CTA; a warp moves one
// token at a time, a lane 16 of its values.
//
// A row of n tokens touches at most n / block + 2 blocks, so the CTAs from offset / block + 2 r on
// are enough for row r (in a call of few tokens: the CTAs from its offset on); a CTA finds its row
// by a search with as many branches as it has threads.  The tokens are then fetched once, while
// the page is looked up, and stay in registers until the scale is known (blocks up to 64
// tokens).  A call is a chain of four dependent loads, so this order is what counts.  Measured: 13.3k tokens of 12 prompts, blocks of 16: 8.2 us, 2.9 TB/s (floor 3.7 us;
// 8.8 us with CTAs of eight warps, which do not all fit on the GPU at once, and 11.0 us with the
// tokens read twice, behind the page); one token for each of 64 rows: 3.2 us, of which an empty
// launch is about 2.

struct AppendParams {
  const __nv_bfloat16* ckv;
  int64_t ckv_sb;
  const __nv_bfloat16* kpe;
  int64_t kpe_sb;
  const int32_t* offsets;
  const int32_t* starts;
  int32_t rows;
  int32_t tokens;
  bool by_token;  // a row's CTAs begin at its offset
  PageTable table;
  Cache cache;
  uint32_t* err;
};

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;  // infinities and NaN take no part in the scale
}

__device__ __forceinline__ float amax16(const uint4 (&v)[2]) {
  float a = 0.f, f[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unpack8(v[h], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) a = fmaxf(a, finite_abs(f[j]));
  }
  return a;
}

// kPer: tokens a warp keeps in registers (kPer * kWarps >= block); 0: read again (larger blocks).
template <int kWarps, int kPer>
__global__ void __launch_bounds__(32 * kWarps) append_kernel(const AppendParams p) {
  constexpr int kThreads = 32 * kWarps;
  __shared__ uint32_t amax_s;
  __shared__ int job_s[4];  // row, first token, its position, tokens (0: no such job)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int shift = p.cache.block_shift, block = 1 << shift;
  if (threadIdx.x == 0) {
    amax_s = 0u;
    job_s[3] = 0;
  }
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  // ---- the job: the last row whose places begin at or before this CTA's
  for (int64_t lo = 0, hi = p.rows;;) {
    const int64_t step = (hi - lo + kThreads - 1) / kThreads;
    const int64_t r = lo + threadIdx.x * step;
    int first = 0, count = 0, start = 0;
    if (r < hi) {
      first = min(max(__ldg(p.offsets + r), 0), p.tokens);
      count = min(max(__ldg(p.offsets + r + 1), 0), p.tokens) - first;
      start = __ldg(p.starts + r);
    }
    const int64_t place = p.by_token ? first : (first >> shift) + 2 * r;
    const int at_or_before = __syncthreads_count(r < hi && place <= (int64_t)blockIdx.x);
    if (at_or_before == 0) return;
    if (step > 1) {
      lo += (at_or_before - 1) * step;
      hi = min(lo + step, hi);
      continue;
    }
    const int64_t j = (int64_t)blockIdx.x - place;  // which of the row's jobs
    if ((int)threadIdx.x == at_or_before - 1 && count > 0 && j >= 0) {
      if (start < 0 || start > INT32_MAX - block - count) {  // the row has no such positions
        if (j == 0) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
      } else if (j <= ((start + count - 1) >> shift) - (start >> shift)) {
        const int pos = j == 0 ? start : ((start >> shift) + (int)j) << shift;
        job_s[0] = (int)r;
        job_s[1] = first + (pos - start);
        job_s[2] = pos;
        job_s[3] = min(block - (pos & (block - 1)), start + count - pos);
      }
    }
    break;
  }
  __syncthreads();
  const int row = job_s[0], t = job_s[1], pos = job_s[2], n = job_s[3];
  if (n == 0) return;
  const int in_block = pos & (block - 1);
  // ---- the new tokens, on the way while their slots are looked up
  constexpr int kRegs = kPer > 0 ? kPer : 1;
  uint4 raw[kRegs][2];
  auto token = [&](int i) {
    return reinterpret_cast<const uint4*>(p.ckv + (int64_t)(t + i) * p.ckv_sb) + 2 * lane;
  };
  if (kPer > 0) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = warp + k * kWarps;
      if (i < n) {
        raw[k][0] = __ldg(token(i));
        raw[k][1] = __ldg(token(i) + 1);
      }
    }
  }
  const int slot0 = slot_at(p.table, row, pos, p.cache.num_slots);
  if (slot0 < 0) {
    if (threadIdx.x == 0) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
    return;
  }
  const float old = in_block != 0 ? p.cache.scale[slot0 >> shift] : 0.f;
  float a = 0.f;
  if (kPer > 0) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (warp + k * kWarps < n) a = fmaxf(a, amax16(raw[k]));
  } else {
    for (int i = warp; i < n; i += kWarps) {
      raw[0][0] = __ldg(token(i));
      raw[0][1] = __ldg(token(i) + 1);
      a = fmaxf(a, amax16(raw[0]));
    }
  }
  a = ptx::warp_max(a);
  if (lane == 0) atomicMax(&amax_s, __float_as_uint(a));  // non-negative floats order as bits
  __syncthreads();
  const float scale = fmaxf(scale_for(__uint_as_float(amax_s)), old);
  if (scale != old) {
    const float ratio = old / scale;
    for (int i = warp; i < in_block; i += kWarps) {
      uint4* q = reinterpret_cast<uint4*>(p.cache.ckv + (int64_t)(slot0 - in_block + i) * p.cache.ckv_ss) + lane;
      *q = rescale16(*q, ratio);
    }
    if (threadIdx.x == 0) p.cache.scale[slot0 >> shift] = scale;
  }
  // 1 / scale is exact for a power of two; a caller's other scales take the division
  const bool pow2 = (__float_as_uint(scale) & 0x7FFFFFu) == 0u;
  const float inv = 1.f / scale;
  auto put = [&](int i, const uint4 (&v)[2]) {
    uint32_t w[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
      unpack8(v[h], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (isinf(f[j])) f[j] = NAN;  // e4m3 has no infinities
        f[j] = pow2 ? f[j] * inv : f[j] / scale;
      }
      w[2 * h] = to_e4m3x2(f[0], f[1]) | (to_e4m3x2(f[2], f[3]) << 16);
      w[2 * h + 1] = to_e4m3x2(f[4], f[5]) | (to_e4m3x2(f[6], f[7]) << 16);
    }
    const int64_t slot = slot0 + i;
    reinterpret_cast<uint4*>(p.cache.ckv + slot * p.cache.ckv_ss)[lane] = make_uint4(w[0], w[1], w[2], w[3]);
  };
  // the rope keys: four tokens at a time, eight lanes each
  for (int i = 4 * warp + (lane >> 3); i < n; i += 4 * kWarps)
    reinterpret_cast<uint4*>(p.cache.kpe + (int64_t)(slot0 + i) * p.cache.kpe_ss)[lane & 7] =
        __ldg(reinterpret_cast<const uint4*>(p.kpe + (int64_t)(t + i) * p.kpe_sb) + (lane & 7));
  if (kPer > 0) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (warp + k * kWarps < n) put(warp + k * kWarps, raw[k]);
  } else {
    for (int i = warp; i < n; i += kWarps) {
      raw[0][0] = __ldg(token(i));
      raw[0][1] = __ldg(token(i) + 1);
      put(i, raw[0]);
    }
  }
}

// --------------------------------------------------------------------------- accumulate
//
// acc[r][positions[t][k]] += weights[t][k] for the tokens t of row r.  Tokens of one row may
// name the same position, so a CTA adds them in a fixed order, a barrier between them, with the
// entries of eight tokens fetched ahead.  An SM passes on about one scattered reduction per
// clock, so a row is dealt out to up to eight CTAs by position: each reads all entries and adds
// those of its own 32-byte sectors, which keeps every position's order.  With one token per row
// the entries are independent and spread over CTAs of 256.  The adds are fire-and-forget
// reductions, also right when a token names a position twice.  Measured: 16 rows of 8 x 1500
// entries 4.6 us with eight CTAs a row (floor 0.4; the chain offsets -> entries -> eight barriers;
// 7.1 us with one CTA a row); 64 rows of 2048 entries 1.9 us, an empty launch's time.  A row of
// many tokens is serial: 512 tokens of 2048 entries in one row 201 us, 4096 1.68 ms, 64 in each
// of 16 rows 29 us.

struct AccumulateParams {
  const float* weights;
  int64_t w_sb;
  const int32_t* positions;
  int64_t pos_sb;
  float* acc;
  int64_t acc_sb;
  const int32_t* offsets;  // nullptr: token r is row r
  int32_t tokens;
  int32_t topk;
  int32_t acc_cols;
  uint32_t* err;
};

// share of shares: the CTA's part of the row's positions, by sectors of eight
__device__ __forceinline__ void accumulate_entry(const AccumulateParams& p, float* row, int pos,
                                                 float w, uint32_t share, uint32_t shares) {
  if (pos >= 0 && pos < p.acc_cols) {
    if ((((uint32_t)pos >> 3) & (shares - 1)) == share) atomicAdd(row + pos, w);
  } else if (pos != -1) {
    atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
  }
}

__global__ void __launch_bounds__(256) accumulate_kernel(const AccumulateParams p) {
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  const int64_t t = blockIdx.x;
  const int k = (int)(blockIdx.y * 256 + threadIdx.x);
  if (k < p.topk)
    accumulate_entry(p, p.acc + t * p.acc_sb, __ldg(p.positions + t * p.pos_sb + k),
                     __ldg(p.weights + t * p.w_sb + k), 0u, 1u);
}

__global__ void __launch_bounds__(1024) accumulate_tokens_kernel(const AccumulateParams p) {
  constexpr int kAhead = 8, kPer = 2;  // tokens, and entries of each, that a thread fetches at once
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  const int64_t r = blockIdx.x;
  const int lo = max(0, __ldg(p.offsets + r)), hi = min(p.tokens, __ldg(p.offsets + r + 1));
  float* row = p.acc + r * p.acc_sb;
  for (int k0 = 0; k0 < p.topk; k0 += 1024 * kPer) {
    for (int t0 = lo; t0 < hi; t0 += kAhead) {
      int pos[kAhead][kPer];
      float w[kAhead][kPer];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
          const int k = k0 + c * 1024 + (int)threadIdx.x;
          const bool has = k < p.topk && t0 + j < hi;
          pos[j][c] = has ? __ldg(p.positions + (int64_t)(t0 + j) * p.pos_sb + k) : -1;
          w[j][c] = has ? __ldg(p.weights + (int64_t)(t0 + j) * p.w_sb + k) : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
#pragma unroll
        for (int c = 0; c < kPer; ++c)
          accumulate_entry(p, row, pos[j][c], w[j][c], blockIdx.y, gridDim.y);
        __syncthreads();
      }
    }
  }
}

// ------------------------------------------------------------------------------ compact
//
// Entry j of row r (keep[r][j], a position of the row's sequence; -1: none) moves from the
// slot of that position in the row's pages to slot j of its new pages.  The scale of a new
// block is the largest scale among the tokens that move into it, and every token is
// re-expressed in it, as in the append.  A CTA owns 64 consecutive entries of a row (or one
// block, if that is larger), which are whole blocks of the new pages, and a warp eight of them:
// it looks their slots up and has all eight tokens on the way before the scales are compared,
// so that the chain keep -> page -> token is all that a CTA waits for, and an SM holds 32 warps
// of 5 kB in flight.  Measured: 126k tokens of 32 rows 29.8 us, 5.4 TB/s (floor 24.6 us; 39.2 us
// with a warp's tokens one after another); 2048 tokens of one row 3.8 us.

constexpr int kCompactSpan = 64;
constexpr int kWarpEntries = 8;
constexpr int kMaxBlock = 256;  // tokens per scale

struct CompactParams {
  const int32_t* keep;
  int64_t keep_sb;
  int32_t cols;
  PageTable from, to;
  Cache cache;
  uint32_t* err;
};

__global__ void __launch_bounds__(kMaxBlock / kWarpEntries * 32) compact_kernel(const CompactParams p) {
  __shared__ uint32_t scale_s[kMaxBlock];  // by new block: its scale's bits
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int span = (int)blockDim.x / 32 * kWarpEntries;  // entries per CTA
  if ((int)threadIdx.x < span) scale_s[threadIdx.x] = 0u;
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  const int64_t row = blockIdx.x;
  const int first = warp * kWarpEntries;  // of the CTA's entries
  const int j0 = (int)blockIdx.y * span + first;
  // ---- lane e: entry e
  int src = -1, dst = -1;
  if (lane < kWarpEntries && j0 + lane < p.cols) {
    const int pos = __ldg(p.keep + row * p.keep_sb + j0 + lane);
    if (pos != -1) {
      src = slot_at(p.from, row, pos, p.cache.num_slots);
      dst = slot_at(p.to, row, j0 + lane, p.cache.num_slots);
      if (src < 0 || dst < 0) {
        atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
        src = -1;
      }
    }
  }
  const float old = src >= 0 ? __ldg(p.cache.scale + (src >> p.cache.block_shift)) : 0.f;
  // ---- the tokens: a lane 16 bytes of each latent row, and of one of four rope rows at a time
  uint4 v[kWarpEntries], pe[kWarpEntries / 4];
#pragma unroll
  for (int e = 0; e < kWarpEntries; ++e) {
    const int from = __shfl_sync(0xffffffffu, src, e);
    if (from >= 0)
      v[e] = __ldcs(reinterpret_cast<const uint4*>(p.cache.ckv + (int64_t)from * p.cache.ckv_ss) + lane);
  }
#pragma unroll
  for (int e = 0; e < kWarpEntries / 4; ++e) {
    const int from = __shfl_sync(0xffffffffu, src, 4 * e + (lane >> 3));
    if (from >= 0)
      pe[e] = __ldcs(reinterpret_cast<const uint4*>(p.cache.kpe + (int64_t)from * p.cache.kpe_ss) + (lane & 7));
  }
  // ---- the new blocks' scales (non-negative floats order as bits; fabsf: a scale may be -0)
  __syncthreads();
  uint32_t* const block_s = scale_s + ((first + (lane & (kWarpEntries - 1))) >> p.cache.block_shift);
  if (src >= 0) atomicMax(block_s, __float_as_uint(fabsf(old)));
  __syncthreads();
  const float big = __uint_as_float(*block_s);
  const float ratio = big > 0.f ? old / big : 0.f;
  // every entry that moves into a block writes the same scale
  if (src >= 0) p.cache.scale[dst >> p.cache.block_shift] = big;
#pragma unroll
  for (int e = 0; e < kWarpEntries; ++e) {
    const int from = __shfl_sync(0xffffffffu, src, e), to = __shfl_sync(0xffffffffu, dst, e);
    const float r = __shfl_sync(0xffffffffu, ratio, e);
    if (from >= 0)
      reinterpret_cast<uint4*>(p.cache.ckv + (int64_t)to * p.cache.ckv_ss)[lane] =
          r == 1.f ? v[e] : rescale16(v[e], r);
  }
#pragma unroll
  for (int e = 0; e < kWarpEntries / 4; ++e) {
    const int from = __shfl_sync(0xffffffffu, src, 4 * e + (lane >> 3));
    const int to = __shfl_sync(0xffffffffu, dst, 4 * e + (lane >> 3));
    if (from >= 0)
      reinterpret_cast<uint4*>(p.cache.kpe + (int64_t)to * p.cache.kpe_ss)[lane & 7] = pe[e];
  }
}

// ====================================================================== host side
namespace {

cudaLaunchAttribute pdl_attr() {
  cudaLaunchAttribute a;
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}

// Launched so that the grid may be scheduled while the stream's previous one drains; every
// kernel here waits for it (griddepcontrol.wait) before it touches global memory.
template <typename P>
int launch(void (*kern)(P), dim3 grid, unsigned threads, cudaStream_t st, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1] = {pdl_attr()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? DSA_OK : DSA_ERR_CUDA;
}

bool power_of_two(int32_t v) { return v > 0 && (v & (v - 1)) == 0; }
int32_t log2_of(int32_t v) {
  int32_t s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

int check_cache(const void* ckv, int64_t ckv_ss, const float* scale, const void* kpe,
                int64_t kpe_ss, int64_t num_slots, int32_t block) {
  if (!ckv || !scale || !kpe || ckv_ss < kDCkv || kpe_ss < kDKpe || num_slots < 1 ||
      num_slots > INT32_MAX || !power_of_two(block) || block > kMaxBlock)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(ckv) || !aligned16(kpe) || ckv_ss % 16 || (kpe_ss * 2) % 16)
    return DSA_ERR_MISALIGNED;
  return DSA_OK;
}

int check_table(const int32_t* pt, int64_t sb, int32_t cols, int32_t page_size, int32_t block) {
  if (!pt || cols < 1 || sb < 0 || !power_of_two(page_size) || page_size > (1 << 20) ||
      page_size < block || (int64_t)cols * page_size > INT32_MAX)
    return DSA_ERR_INVALID_ARGUMENT;
  return DSA_OK;
}

Cache cache_of(void* ckv, int64_t ckv_ss, float* scale, void* kpe, int64_t kpe_ss,
               int64_t num_slots, int32_t block) {
  return Cache{static_cast<uint8_t*>(ckv), ckv_ss, scale, static_cast<__nv_bfloat16*>(kpe),
               kpe_ss, num_slots, log2_of(block)};
}

}  // namespace
}  // namespace q8
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_append_q8(const void* ckv, int64_t ckv_stride_t, const void* kpe,
                             int64_t kpe_stride_t, int64_t num_tokens,
                             const int32_t* row_offsets, const int32_t* starts, int32_t num_rows,
                             const int32_t* page_table, int64_t page_table_stride_b,
                             int32_t page_table_cols, int32_t page_size, void* ckv_q8,
                             int64_t ckv_slot_stride, float* ckv_scale, int32_t block,
                             void* kpe_cache, int64_t kpe_slot_stride, int64_t num_slots,
                             void* workspace, void* stream) {
  if (num_tokens < 0 || num_tokens > INT32_MAX || num_rows < 0) return DSA_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0 || num_rows == 0) return DSA_OK;
  if (!ckv || !kpe || !row_offsets || !starts || ckv_stride_t < 0 || kpe_stride_t < 0)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!workspace) return DSA_ERR_WORKSPACE;
  int rc = q8::check_cache(ckv_q8, ckv_slot_stride, ckv_scale, kpe_cache, kpe_slot_stride,
                           num_slots, block);
  if (rc == DSA_OK)
    rc = q8::check_table(page_table, page_table_stride_b, page_table_cols, page_size, block);
  if (rc != DSA_OK) return rc;
  if (!aligned16(ckv) || !aligned16(kpe) || (ckv_stride_t * 2) % 16 || (kpe_stride_t * 2) % 16)
    return DSA_ERR_MISALIGNED;
  q8::AppendParams p;
  p.ckv = static_cast<const __nv_bfloat16*>(ckv);
  p.ckv_sb = ckv_stride_t;
  p.kpe = static_cast<const __nv_bfloat16*>(kpe);
  p.kpe_sb = kpe_stride_t;
  p.offsets = row_offsets;
  p.starts = starts;
  p.rows = num_rows;
  p.tokens = (int32_t)num_tokens;
  p.table = q8::PageTable{page_table, page_table_stride_b, page_table_cols, q8::log2_of(page_size)};
  p.cache = q8::cache_of(ckv_q8, ckv_slot_stride, ckv_scale, kpe_cache, kpe_slot_stride, num_slots,
                         block);
  p.err = static_cast<uint32_t*>(workspace);
  const int64_t bound = num_tokens / block + 2 * (int64_t)num_rows;
  p.by_token = num_tokens <= bound;
  if (!p.by_token && bound > INT32_MAX) return DSA_ERR_INVALID_ARGUMENT;
  const dim3 grid((unsigned)(p.by_token ? num_tokens : bound));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (block <= 16) return q8::launch(q8::append_kernel<4, 4>, grid, 128, st, p);
  if (block <= 64) return q8::launch(q8::append_kernel<8, 8>, grid, 256, st, p);
  return q8::launch(q8::append_kernel<8, 0>, grid, 256, st, p);
}

extern "C" int dsa_accumulate_weights(const float* weights, int64_t weights_stride_t,
                                      const int32_t* positions, int64_t positions_stride_t,
                                      int64_t num_tokens, int32_t topk, float* acc,
                                      int64_t acc_stride_r, int32_t acc_cols, int32_t num_rows,
                                      const int32_t* row_offsets, void* workspace, void* stream) {
  if (num_tokens < 0 || num_tokens > INT32_MAX || num_rows < 0 || topk < 1 || acc_cols < 0)
    return DSA_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0 || num_rows == 0) return DSA_OK;
  if (!weights || !positions || !acc || weights_stride_t < 0 || positions_stride_t < 0 ||
      (num_rows > 1 && acc_stride_r < acc_cols) || (!row_offsets && num_rows != num_tokens) || topk > 65535 * 256)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!workspace) return DSA_ERR_WORKSPACE;
  const q8::AccumulateParams p{weights,  weights_stride_t, positions,           positions_stride_t,
                               acc,      acc_stride_r,     row_offsets,         (int32_t)num_tokens,
                               topk,     acc_cols,         static_cast<uint32_t*>(workspace)};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (row_offsets) {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return DSA_ERR_CUDA;
    unsigned shares = 1;
    while (shares < 8 && 2 * shares * (int64_t)num_rows <= sms) shares *= 2;
    return q8::launch(q8::accumulate_tokens_kernel, dim3((unsigned)num_rows, shares), 1024, st, p);
  }
  return q8::launch(q8::accumulate_kernel,
                    dim3((unsigned)num_tokens, (unsigned)((topk + 255) / 256)), 256, st, p);
}

extern "C" int dsa_compact_q8(const int32_t* keep, int64_t keep_stride_b, int32_t num_rows,
                              int32_t keep_cols, const int32_t* page_table,
                              int64_t page_table_stride_b, int32_t page_table_cols,
                              const int32_t* new_page_table, int64_t new_page_table_stride_b,
                              int32_t new_page_table_cols, int32_t page_size, void* ckv_q8,
                              int64_t ckv_slot_stride, float* ckv_scale, int32_t block,
                              void* kpe_cache, int64_t kpe_slot_stride, int64_t num_slots,
                              void* workspace, void* stream) {
  if (num_rows < 0 || keep_cols < 0) return DSA_ERR_INVALID_ARGUMENT;
  if (num_rows == 0 || keep_cols == 0) return DSA_OK;
  if (!keep || keep_stride_b < 0) return DSA_ERR_INVALID_ARGUMENT;
  if (!workspace) return DSA_ERR_WORKSPACE;
  int rc = q8::check_cache(ckv_q8, ckv_slot_stride, ckv_scale, kpe_cache, kpe_slot_stride,
                           num_slots, block);
  if (rc == DSA_OK)
    rc = q8::check_table(page_table, page_table_stride_b, page_table_cols, page_size, block);
  if (rc == DSA_OK)
    rc = q8::check_table(new_page_table, new_page_table_stride_b, new_page_table_cols, page_size,
                         block);
  if (rc != DSA_OK) return rc;
  q8::CompactParams p;
  p.keep = keep;
  p.keep_sb = keep_stride_b;
  p.cols = keep_cols;
  const int span = block > q8::kCompactSpan ? block : q8::kCompactSpan;
  const int shift = q8::log2_of(page_size);
  p.from = q8::PageTable{page_table, page_table_stride_b, page_table_cols, shift};
  p.to = q8::PageTable{new_page_table, new_page_table_stride_b, new_page_table_cols, shift};
  p.cache = q8::cache_of(ckv_q8, ckv_slot_stride, ckv_scale, kpe_cache, kpe_slot_stride, num_slots,
                         block);
  p.err = static_cast<uint32_t*>(workspace);
  const int64_t spans = ((int64_t)keep_cols + span - 1) / span;
  if (spans > 65535) return DSA_ERR_INVALID_ARGUMENT;
  return q8::launch(q8::compact_kernel, dim3((unsigned)num_rows, (unsigned)spans),
                    (unsigned)(span / q8::kWarpEntries * 32), static_cast<cudaStream_t>(stream), p);
}

namespace dsa {
namespace q8 {
namespace {

using AttendFn = void (*)(CUtensorMap, CUtensorMap, AttendParams);

int group_heads(int heads) { return heads == 16 ? 16 : 32; }
int tile_slots(int nh) { return nh == 16 ? Cfg<16>::kTS : Cfg<32>::kTS; }

// SMs of the current device, with the attend kernels' shared-memory limit raised on it.
int prepare_device() {
  static std::atomic<int> sms[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = sms[dev].load(std::memory_order_acquire);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaFuncSetAttribute(attend_kernel<16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Cfg<16>::SMEM_BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(attend_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Cfg<32>::SMEM_BYTES) != cudaSuccess)
      return 0;
    sms[dev].store(n, std::memory_order_release);
  }
  return n;
}

// CTAs per (row, head group).  Per CTA about 7 us are counted outside the tiles (first gather, end;
// 8 with the merge) and 1.4 us (16 heads) or 1.75 us (32; measured 2.35 to 2.71) per tile; a
// call whose units do not fill the SMs splits them while that shortens the longest CTA.  The rule
// counts SMs, but a cluster must fit into a GPC, so where S G > 2 the last SMs of a wave can stay
// idle and the call takes a second one: 16 rows of 16 heads and 2048 slots take 28.0 us in
// splits of eight, 20 rows 18.0 in splits of four; 36 rows 34.0, 40 rows 24.5 (splits of
// two); 16 rows of 128 heads 58.5, 19 rows 45.6 (unsplit).  Measured, us for S = 1, 2, 4, 8
// (* chosen; -: a cluster of more than eight, or not measured):
//     1 row, 16 heads, 2048 slots          35.4   21.9   15.5   12.1*
//     64 rows, 16 heads, 2048 slots        37.9   26.4*  36.8     -
//     256 ragged rows, 16 heads            77.8*  82.7  125.9     -
//     256 full rows, 16 heads              78.2*  99.6  139.1     -
//     7 rows, 64 heads, 1001 slots         28.9   21.2   16.6*    -
//     32 rows, 128 heads, 2048 slots       50.1*  94.2     -      -
int choose_splits(int64_t units, int nh, int groups, int ntiles, int sms) {
  const double tile = nh == 16 ? 1.4 : 1.75;
  int best = 1;
  double best_cost = 0;
  for (int s = 1; s * groups <= kMaxCluster; s *= 2) {
    const int64_t waves = (units * s + sms - 1) / sms;
    const double cost = (double)waves * ((s > 1 ? 8.0 : 7.0) + tile * ((ntiles + s - 1) / s));
    if (s == 1 || cost < best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}

}  // namespace
}  // namespace q8
}  // namespace dsa

// A decode with weights keeps the scores of at most this many rows at a time: 256 CTAs that take
// row after row, or launches of 256 rows where a row is a cluster's.
constexpr int64_t kScoreRows = 256;

extern "C" size_t dsa_q8_scratch_size(int64_t num_tokens, int32_t num_heads, int32_t topk) {
  if (num_tokens < 0 || topk < 1 || !heads_supported(num_heads)) return 0;
  if (num_tokens > kScoreRows) num_tokens = kScoreRows;
  const int nh = q8::group_heads(num_heads);
  const size_t ts = (size_t)q8::tile_slots(nh), tiles = ((size_t)topk + ts - 1) / ts;
  return (size_t)num_tokens * tiles * ((size_t)num_heads * ts + (size_t)(num_heads / nh)) * 4;
}

extern "C" int dsa_sparse_mla_decode_q8(
    const void* q_nope, int64_t q_nope_stride_b, int64_t q_nope_stride_h, const void* q_pe,
    int64_t q_pe_stride_b, int64_t q_pe_stride_h, const void* ckv_q8, int64_t ckv_slot_stride,
    const float* ckv_scale, int32_t block, const void* kpe_cache, int64_t kpe_slot_stride,
    int64_t num_slots, const int32_t* page_table, int64_t page_table_stride_b,
    int32_t page_table_cols, int32_t page_size, const int32_t* indices, int64_t indices_stride_b,
    float sm_scale, void* output, int64_t output_stride_b, int64_t output_stride_h, float* lse,
    int64_t lse_stride_b, int64_t lse_stride_h, float* weights, int64_t weights_stride_b,
    int64_t num_tokens, int32_t num_heads, int32_t topk, void* scratch, size_t scratch_bytes,
    void* workspace, void* stream) {
  if (num_tokens < 0 || num_tokens > INT32_MAX || topk < 1) return DSA_ERR_INVALID_ARGUMENT;
  if (!heads_supported(num_heads)) return DSA_ERR_UNSUPPORTED;
  if (num_tokens == 0) return DSA_OK;
  if (!q_nope || !q_pe || !indices || !output || !lse || q_nope_stride_h < 0 ||
      q_pe_stride_h < 0 || q_nope_stride_b < 0 || q_pe_stride_b < 0 || indices_stride_b < 0)
    return DSA_ERR_INVALID_ARGUMENT;
  int rc = q8::check_cache(ckv_q8, ckv_slot_stride, ckv_scale, kpe_cache, kpe_slot_stride,
                           num_slots, block);
  if (rc == DSA_OK && page_table != nullptr)
    rc = q8::check_table(page_table, page_table_stride_b, page_table_cols, page_size, block);
  if (rc != DSA_OK) return rc;
  if (!aligned16(q_nope) || !aligned16(q_pe) || (q_nope_stride_b * 2) % 16 ||
      (q_nope_stride_h * 2) % 16 || (q_pe_stride_b * 2) % 16 || (q_pe_stride_h * 2) % 16)
    return DSA_ERR_MISALIGNED;
  if (!workspace) return DSA_ERR_WORKSPACE;
  if (weights != nullptr) {
    if (num_tokens > 1 && weights_stride_b < topk) return DSA_ERR_INVALID_ARGUMENT;
    if (!scratch || scratch_bytes < dsa_q8_scratch_size(num_tokens, num_heads, topk))
      return DSA_ERR_WORKSPACE;
  }
  q8::AttendParams p;
  p.qn = static_cast<const __nv_bfloat16*>(q_nope);
  p.qn_sb = q_nope_stride_b;
  p.qn_sh = q_nope_stride_h;
  p.qp = static_cast<const __nv_bfloat16*>(q_pe);
  p.qp_sb = q_pe_stride_b;
  p.qp_sh = q_pe_stride_h;
  p.cache = q8::cache_of(const_cast<void*>(ckv_q8), ckv_slot_stride, const_cast<float*>(ckv_scale),
                         const_cast<void*>(kpe_cache), kpe_slot_stride, num_slots, block);
  p.idx = indices;
  p.idx_sb = indices_stride_b;
  p.table = q8::PageTable{page_table, page_table_stride_b, page_table_cols,
                          page_table != nullptr ? q8::log2_of(page_size) : 0};
  p.out = static_cast<__nv_bfloat16*>(output);
  p.out_sb = output_stride_b;
  p.out_sh = output_stride_h;
  p.out8 = (reinterpret_cast<uintptr_t>(output) & 7u) == 0 && output_stride_b % 4 == 0 &&
           output_stride_h % 4 == 0;
  p.lse = lse;
  p.lse_sb = lse_stride_b;
  p.lse_sh = lse_stride_h;
  p.weights = weights;
  p.w_sb = weights_stride_b;
  const int nh = q8::group_heads(num_heads);
  p.topk = topk;
  const int ts = q8::tile_slots(nh);
  p.ntiles = (int32_t)(((int64_t)topk + ts - 1) / ts);
  p.groups = num_heads / nh;
  p.scores = static_cast<float*>(scratch);
  p.tiles = weights == nullptr ? nullptr
                               : reinterpret_cast<int32_t*>(
                                     p.scores + std::min(num_tokens, kScoreRows) * p.ntiles * num_heads * ts);
  p.scale_log2 = sm_scale * kLog2e;
  p.wait_cycles = wait_limit_cycles();
  p.err = static_cast<uint32_t*>(workspace);
  const int sms = q8::prepare_device();
  if (sms <= 0) return DSA_ERR_CUDA;
  p.units = num_tokens * p.groups;
  p.splits = q8::choose_splits(p.units, nh, p.groups, p.ntiles, sms);
  // The CTAs of a row form a cluster where they have something to add up: a unit's splits, or
  // the groups' weights.  Otherwise at most one CTA per SM takes unit after unit.
  p.clustered = p.splits > 1 || (weights != nullptr && p.groups > 1);
  const int cluster = p.clustered ? p.splits * p.groups : 1;
  const int64_t rows = weights != nullptr && p.clustered ? std::min(num_tokens, kScoreRows) : num_tokens;
  const int64_t ctas = std::min<int64_t>(sms, kScoreRows);
  if (p.clustered && p.units * p.splits > INT32_MAX) return DSA_ERR_INVALID_ARGUMENT;
  // gathers of single slots: 128-byte boxes of one row
  CUtensorMap m_ckv, m_kpe;
  {
    cuuint64_t dims[2] = {(cuuint64_t)kDCkv, (cuuint64_t)num_slots};
    cuuint64_t str[1] = {(cuuint64_t)ckv_slot_stride};
    cuuint32_t box[2] = {128, 1};
    rc = encode(&m_ckv, ckv_q8, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_DATA_TYPE_UINT8);
  }
  if (rc == DSA_OK) {
    cuuint64_t dims[2] = {(cuuint64_t)kDKpe, (cuuint64_t)num_slots};
    cuuint64_t str[1] = {(cuuint64_t)kpe_slot_stride * 2};
    cuuint32_t box[2] = {64, 1};
    rc = encode(&m_kpe, kpe_cache, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (rc != DSA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(q8::kThreads);
  cfg.dynamicSmemBytes = (size_t)(nh == 16 ? q8::Cfg<16>::SMEM_BYTES : q8::Cfg<32>::SMEM_BYTES);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2] = {q8::pdl_attr(), {}};
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const q8::AttendFn fn = nh == 16 ? q8::attend_kernel<16> : q8::attend_kernel<32>;
  // one launch, or (clusters with weights) launches of `rows` rows that use the scratch in turn
  for (int64_t left = num_tokens; left > 0; left -= rows) {
    p.units = std::min(rows, left) * p.groups;
    cfg.gridDim = dim3((unsigned)(p.clustered ? p.units * p.splits : std::min(p.units, ctas)));
    if (cudaLaunchKernelEx(&cfg, fn, m_ckv, m_kpe, p) != cudaSuccess) return DSA_ERR_CUDA;
    p.qn += rows * p.qn_sb;
    p.qp += rows * p.qp_sb;
    p.idx += rows * p.idx_sb;
    if (p.table.pt != nullptr) p.table.pt += rows * page_table_stride_b;
    p.out += rows * p.out_sb;
    p.lse += rows * p.lse_sb;
    if (p.weights != nullptr) p.weights += rows * p.w_sb;
  }
  return DSA_OK;
}
