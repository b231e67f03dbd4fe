// Dense attention over the bf16 latent cache: a sliding window with sinks, rows behind a shared
// prefix, and the join of attention results over separate sets of positions.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "dsa_b200.h"
#include "dsa_common.cuh"
#include "dsa_host.cuh"
#include "sm100_ptx.cuh"

namespace dsa {
namespace dense {

constexpr int kAll = 0x3fffffff;  // a window that leaves nothing out

// Pages of sequences, row-major int32.
struct Table {
  const int32_t* pt;
  int64_t sb;
  int32_t cols;
};

struct Params {
  Table own, pre;                  // pre.pt == nullptr: no prefixes
  int64_t num_slots;
  int32_t page_shift;
  const int32_t *lengths, *row_offsets;     // row_offsets nullptr: a token a row
  const int32_t *pre_lengths, *group_offsets;  // group_offsets nullptr: one group of all rows
  int32_t rows, groups, tokens, heads;
  int32_t head_shift, tpu;         // log2 heads; tokens of a unit
  int32_t window, sinks;
  int32_t unit_tiles;              // tiles of a unit, at most
  int32_t whole;                   // a pair for each unit
  float scale_log2;
  __nv_bfloat16* out;
  int64_t out_sb, out_sh;
  float* lse;
  int64_t lse_sb, lse_sh;
  uint32_t* err;
  uint64_t wait_cycles;
  // scratch: where units are cut; partial results and their (maximum, sum)
  int4* cuts;  // window: each pair's first unit; shared: each token's units, the prefix's and its own
  int32_t pairs;
  float2* sums;
  float* part;
};

}  // namespace dense
}  // namespace dsa

#include "dsa_dense_attend.cuh"

namespace dsa {
namespace dense {

// ------------------------------------------------------------------------------- the join

constexpr int kMaxParts = 8;

struct MergeParams {
  const __nv_bfloat16* o[kMaxParts];
  const float* z[kMaxParts];
  int64_t o_sb[kMaxParts], o_sh[kMaxParts], z_sb[kMaxParts], z_sh[kMaxParts];
  __nv_bfloat16* out;
  float* lse;
  int64_t out_sb, out_sh, lse_sb, lse_sh;
  int64_t rows;  // tokens x heads
  int32_t heads;
};

// out = sum_i w_i out_i / sum_i w_i with w_i = 2^(lse_i - M), M the largest lse;
// lse = M + log2 sum_i w_i.  A warp is one head of one token, 16 values a lane: all of a row's
// reads come before its writes, so the result may take a part's place.
template <int kParts>
__global__ void __launch_bounds__(256) merge_kernel(const MergeParams p) {
  const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  if (r >= p.rows) return;
  const int64_t t = r / p.heads, h = r % p.heads;
  uint4 v[kParts][2];
  float z[kParts], w[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    z[i] = p.z[i][t * p.z_sb[i] + h * p.z_sh[i]];
    const uint4* src = reinterpret_cast<const uint4*>(p.o[i] + t * p.o_sb[i] + h * p.o_sh[i]);
    v[i][0] = src[lane];
    v[i][1] = src[lane + 32];
  }
  float m = -INFINITY, total = 0.f;
#pragma unroll
  for (int i = 0; i < kParts; ++i) m = fmaxf(m, z[i]);
  // every part empty (or NaN): M plays no part
  const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    w[i] = exp2f(z[i] - base);
    total += w[i];
  }
  const float inv = 1.f / total;
  uint4 res[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float a[8] = {};
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const uint32_t x[4] = {v[i][half].x, v[i][half].y, v[i][half].z, v[i][half].w};
      // a part without weight is left out, whatever its values are
      if (z[i] != -INFINITY) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[2 * j] += w[i] * __uint_as_float(x[j] << 16);
          a[2 * j + 1] += w[i] * __uint_as_float(x[j] & 0xFFFF0000u);
        }
      }
    }
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool some = total != 0.f;  // NaN stays NaN
      const __nv_bfloat162 b = __floats2bfloat162_rn(some ? a[2 * j] * inv : 0.f,
                                                     some ? a[2 * j + 1] * inv : 0.f);
      y[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
    res[half] = make_uint4(y[0], y[1], y[2], y[3]);
  }
  uint4* dst = reinterpret_cast<uint4*>(p.out + t * p.out_sb + h * p.out_sh);
  __syncwarp();
  dst[lane] = res[0];
  dst[lane + 32] = res[1];
  if (lane == 0) p.lse[t * p.lse_sb + h * p.lse_sh] = base + log2f(total);
}

// The rows of a [tokens, heads] tensor (bytes throughout).
struct Rows2 {
  const void* p;
  int64_t sb, sh, width;
};

// Whether rows of a and b meet, for any (t, h) of either; strides are those of a.
bool same_grid_meets(const Rows2& a, const Rows2& b, int64_t tokens, int64_t heads) {
  const int64_t d = (int64_t) reinterpret_cast<intptr_t>(a.p) - (int64_t) reinterpret_cast<intptr_t>(b.p);
  for (int64_t dh = -(heads - 1); dh < heads; ++dh) {
    const int64_t rest = d + dh * a.sh;
    // the tokens' distance that brings them closest, and its neighbours
    const int64_t q = a.sb == 0 ? 0 : std::clamp(-rest / a.sb, -(tokens - 1), tokens - 1);
    for (int64_t dt = q - 1; dt <= q + 1; ++dt) {
      const int64_t x = rest + dt * a.sb;
      if (std::abs(dt) < tokens && x < b.width && -x < a.width) return true;
    }
  }
  return false;
}

// Whether a and b share memory.  Exact where they have the same strides; otherwise all that lies
// between a token's first and last row counts (between the first and last of all, where the tokens'
// strides differ too).
bool overlaps(Rows2 a, Rows2 b, int64_t tokens, int64_t heads) {
  if (tokens == 1) a.sb = b.sb = 0;
  if (heads == 1) a.sh = b.sh = 0;
  auto whole = [](Rows2& r, int64_t n, int64_t stride) {
    const int64_t span = (n - 1) * stride;
    if (span < 0) r.p = static_cast<const char*>(r.p) + span;
    r.width += std::abs(span);
  };
  Rows2 ta = a, tb = b;  // a row for each token
  whole(ta, heads, a.sh);
  whole(tb, heads, b.sh);
  ta.sh = tb.sh = 0;
  Rows2 all_a = ta, all_b = tb;
  whole(all_a, tokens, a.sb);
  whole(all_b, tokens, b.sb);
  all_a.sb = all_b.sb = 0;
  if (!same_grid_meets(all_a, all_b, 1, 1)) return false;  // apart, as most are
  if (a.sb != b.sb) return true;
  return a.sh == b.sh ? same_grid_meets(a, b, tokens, heads) : same_grid_meets(ta, tb, tokens, 1);
}

// Whether they are the same rows.
bool same_rows(const Rows2& a, const Rows2& b, int64_t tokens, int64_t heads) {
  return a.p == b.p && (a.sb == b.sb || tokens == 1) && (a.sh == b.sh || heads == 1);
}

bool aligned_rows(const void* p, int64_t sb, int64_t sh) {
  return aligned16(p) && sb % 8 == 0 && sh % 8 == 0;
}

// What window and shared have in common; `pre` fields are zero for a window call.
struct Call {
  Params p;
  const void *qn, *qp, *ckv, *kpe;
  int64_t qn_sb, qn_sh, qp_sb, qp_sh, ckv_ss, kpe_ss;
  int32_t page_size;
  void* scratch;
  size_t scratch_bytes;
  void* workspace;
  void* stream;
};

constexpr int kMaxDevices = 64;

// CTA pairs that the current device runs at once; 0 on an error.
int max_pairs() {
  static std::atomic<int> known[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  int n = known[dev].load(std::memory_order_acquire);
  if (n > 0) return n;
  if (cudaFuncSetAttribute(attend_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           SMEM_BYTES) != cudaSuccess)
    return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, attend_kernel, &cfg) != cudaSuccess || n < 1) return 0;
  known[dev].store(n, std::memory_order_release);
  return n;
}

// Where scratch holds what.
struct Layout {
  size_t sums, part, total;
  Layout(int64_t tokens, int32_t heads, bool shared, int pairs) {
    const int64_t rows = shared ? 2 * tokens * heads + 128 * (int64_t)pairs : 256 * (int64_t)pairs;
    sums = (size_t)(16 * (shared ? tokens : (int64_t)pairs) + 255) / 256 * 256;
    part = sums + (size_t)(rows * 8 + 255) / 256 * 256;
    total = part + (size_t)rows * kDCkv * 4;
  }
};

int box_map(CUtensorMap* m, const void* base, int64_t stride, int width, int64_t rows, int box) {
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t b[2] = {64, (cuuint32_t)box};
  return encode(m, base, 2, dims, strides, b, CU_TENSOR_MAP_SWIZZLE_128B);
}
int query_map(CUtensorMap* m, const void* base, int64_t sb, int64_t sh, int width, int heads,
              int64_t tokens) {
  const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)sh * 2, (cuuint64_t)sb * 2};
  const cuuint32_t h = (cuuint32_t)std::min(heads, 64);
  const cuuint32_t b[3] = {64, h, 64 / h};
  return encode(m, base, 3, dims, strides, b, CU_TENSOR_MAP_SWIZZLE_128B);
}

int check_table(const Table& t, int32_t page_size) {
  // a stride of 0: all rows share one list of pages
  if (t.pt == nullptr || t.cols < 1 || (t.sb < t.cols && t.sb != 0)) return DSA_ERR_INVALID_ARGUMENT;
  return (int64_t)t.cols * page_size > INT32_MAX / 2 ? DSA_ERR_INVALID_ARGUMENT : DSA_OK;
}

template <typename... A>
int launch_pdl(void (*kern)(A...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st,
               A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? DSA_OK : DSA_ERR_CUDA;
}

int attend(Call& c) {
  Params& p = c.p;
  if (p.tokens < 0 || p.rows < 0) return DSA_ERR_INVALID_ARGUMENT;
  if (!heads_supported(p.heads)) return DSA_ERR_UNSUPPORTED;
  if (p.tokens == 0 || p.rows == 0) return DSA_OK;
  if (p.row_offsets == nullptr && p.rows != p.tokens) return DSA_ERR_INVALID_ARGUMENT;
  if (!c.qn || !c.qp || !c.ckv || !c.kpe || !p.lengths || !p.out || !p.lse || p.num_slots < 1 ||
      p.num_slots > INT32_MAX - 64 || c.ckv_ss < kDCkv || c.kpe_ss < kDKpe || p.window < 0 ||
      p.sinks < 0 || c.page_size < 1 || (c.page_size & (c.page_size - 1)))
    return DSA_ERR_INVALID_ARGUMENT;
  int rc = check_table(p.own, c.page_size);
  if (rc == DSA_OK && p.pre.pt != nullptr) rc = check_table(p.pre, c.page_size);
  if (rc != DSA_OK) return rc;
  if (!aligned_rows(c.qn, c.qn_sb, c.qn_sh) || !aligned_rows(c.qp, c.qp_sb, c.qp_sh) ||
      !aligned_rows(c.ckv, c.ckv_ss, 0) || !aligned_rows(c.kpe, c.kpe_ss, 0) ||
      !aligned_rows(p.out, p.out_sb, p.out_sh))
    return DSA_ERR_MISALIGNED;
  if (c.workspace == nullptr || c.scratch == nullptr) return DSA_ERR_WORKSPACE;
  if (!aligned16(c.scratch)) return DSA_ERR_MISALIGNED;
  const bool shared = p.pre.pt != nullptr, single = p.row_offsets == nullptr;
  if (shared && 2 * (int64_t)p.tokens * p.heads > INT32_MAX / 2) return DSA_ERR_INVALID_ARGUMENT;

  p.page_shift = 0;
  while ((1 << p.page_shift) < c.page_size) ++p.page_shift;
  p.head_shift = 0;
  while ((1 << p.head_shift) < p.heads) ++p.head_shift;
  p.tpu = 128 / p.heads;
  p.window = std::min(p.window, kAll);
  p.sinks = std::min(p.sinks, kAll);
  // The chunks that T tokens' sinks and windows can touch.
  const int64_t span = (int64_t)p.window + p.tpu - 1;
  const int64_t chunks = ((int64_t)p.sinks + kChunk - 1) / kChunk + (span + 30) / kChunk + 1;
  p.unit_tiles = (int32_t)((chunks + kTileChunks - 1) / kTileChunks);
  // The most places that the line can have, which the kernel counts in 32 bits.
  auto places = [&](int64_t units, int64_t most, const Table& t) {
    return units * (std::min<int64_t>(most, ((int64_t)t.cols * c.page_size + kTile - 1) / kTile) + kExtra);
  };
  int64_t line = places(single ? p.rows : p.tokens / p.tpu + p.rows, p.unit_tiles, p.own);
  if (shared) line += places(p.tokens / p.tpu + p.groups, INT32_MAX, p.pre);
  if (line > INT32_MAX / 2) return DSA_ERR_INVALID_ARGUMENT;

  int pairs = max_pairs();
  if (pairs < 1) return DSA_ERR_CUDA;
  const Layout at(p.tokens, p.heads, shared, pairs);
  if (c.scratch_bytes < at.total) return DSA_ERR_WORKSPACE;
  p.err = static_cast<uint32_t*>(c.workspace);
  p.wait_cycles = wait_limit_cycles();
  uint8_t* scratch = static_cast<uint8_t*>(c.scratch);
  p.cuts = reinterpret_cast<int4*>(scratch);
  p.sums = reinterpret_cast<float2*>(scratch + at.sums);
  p.part = reinterpret_cast<float*>(scratch + at.part);

  CUtensorMap ckv, kpe, ckv1, kpe1, qn, qp;
  const int box = std::min(c.page_size, kChunk);
  if ((rc = box_map(&ckv, c.ckv, c.ckv_ss, kDCkv, p.num_slots, box)) != DSA_OK ||
      (rc = box_map(&kpe, c.kpe, c.kpe_ss, kDKpe, p.num_slots, box)) != DSA_OK ||
      (rc = box_map(&ckv1, c.ckv, c.ckv_ss, kDCkv, p.num_slots, 1)) != DSA_OK ||
      (rc = box_map(&kpe1, c.kpe, c.kpe_ss, kDKpe, p.num_slots, 1)) != DSA_OK ||
      (rc = query_map(&qn, c.qn, c.qn_sb, c.qn_sh, kDCkv, p.heads, p.tokens)) != DSA_OK ||
      (rc = query_map(&qp, c.qp, c.qp_sb, c.qp_sh, kDKpe, p.heads, p.tokens)) != DSA_OK)
    return rc;

  const cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  // One unit a row: where two would not fit side by side, each has a pair of its own and is cut
  // nowhere.  That saves the join, 4.1 us, where the rows see about as many positions each (64 rows
  // with a window of 1024: 38.9 us, cut 43.0; all of 8192 positions: 141.3 and 143.5).  Rows that
  // differ wait for the longest (64 rows of 4096 to 32768 positions: 432 us, cut 299; one of 131072
  // among 63 of 1024: 1583 and 111): lengths are on the device, so the call's form decides, and
  // row_offsets ask for the cut.
  p.whole = !shared && single && p.rows <= pairs && 2 * p.rows > pairs;
  if (p.whole) pairs = p.rows;
  pairs = (int)std::min<int64_t>(pairs, line);  // no more than there can be places
  p.pairs = pairs;
  if ((rc = launch_pdl(attend_kernel, dim3(2 * (unsigned)pairs), kThreads, SMEM_BYTES, st, ckv, kpe,
                       ckv1, kpe1, qn, qp, p)) != DSA_OK)
    return rc;
  if (shared)
    return launch_pdl(join_tokens_kernel, dim3((unsigned)((int64_t)p.tokens * p.heads / 16), 4), 128,
                      0, st, p);
  if (!p.whole && pairs > 1)
    return launch_pdl(join_cuts_kernel, dim3((unsigned)(pairs - 1), single ? p.heads / 16 : 8), 256,
                      0, st, p);
  return DSA_OK;
}

}  // namespace dense
}  // namespace dsa

using namespace dsa;

namespace {

int64_t clamp32(int64_t n) { return n < 0 ? -1 : (n > INT32_MAX / 256 ? -1 : n); }

dense::Call common(const void* q_nope, int64_t q_nope_stride_b, int64_t q_nope_stride_h,
                   const void* q_pe, int64_t q_pe_stride_b, int64_t q_pe_stride_h,
                   const void* ckv_cache, int64_t ckv_slot_stride, const void* kpe_cache,
                   int64_t kpe_slot_stride, int64_t num_slots, int32_t page_size,
                   const int32_t* page_table, int64_t page_table_stride_b, int32_t page_table_cols,
                   const int32_t* lengths, const int32_t* row_offsets, int32_t num_rows,
                   float sm_scale, void* output, int64_t output_stride_b, int64_t output_stride_h,
                   float* lse, int64_t lse_stride_b, int64_t lse_stride_h, int64_t num_tokens,
                   int32_t num_heads, void* scratch, size_t scratch_bytes, void* workspace,
                   void* stream) {
  dense::Call c = {};
  dense::Params& p = c.p;
  c.qn = q_nope;
  c.qn_sb = q_nope_stride_b;
  c.qn_sh = q_nope_stride_h;
  c.qp = q_pe;
  c.qp_sb = q_pe_stride_b;
  c.qp_sh = q_pe_stride_h;
  c.ckv = ckv_cache;
  c.ckv_ss = ckv_slot_stride;
  c.kpe = kpe_cache;
  c.kpe_ss = kpe_slot_stride;
  p.num_slots = num_slots;
  p.own = {page_table, page_table_stride_b, page_table_cols};
  p.lengths = lengths;
  p.row_offsets = row_offsets;
  p.rows = num_rows;
  p.tokens = (int32_t)clamp32(num_tokens);
  p.heads = num_heads;
  p.window = dense::kAll;
  p.scale_log2 = sm_scale * kLog2e;
  p.out = static_cast<__nv_bfloat16*>(output);
  p.out_sb = output_stride_b;
  p.out_sh = output_stride_h;
  p.lse = lse;
  p.lse_sb = lse_stride_b;
  p.lse_sh = lse_stride_h;
  c.page_size = page_size;
  c.scratch = scratch;
  c.scratch_bytes = scratch_bytes;
  c.workspace = workspace;
  c.stream = stream;
  return c;
}

}  // namespace

extern "C" {

size_t dsa_dense_scratch_size(int64_t num_tokens, int32_t num_heads, int32_t shared) {
  if (!heads_supported(num_heads) || clamp32(num_tokens) < 1) return 0;
  const int pairs = dense::max_pairs();
  return pairs < 1 ? 0 : dense::Layout(num_tokens, num_heads, shared != 0, pairs).total;
}

int dsa_mla_decode_window(
    const void* q_nope, int64_t q_nope_stride_b, int64_t q_nope_stride_h, const void* q_pe,
    int64_t q_pe_stride_b, int64_t q_pe_stride_h, const void* ckv_cache, int64_t ckv_slot_stride,
    const void* kpe_cache, int64_t kpe_slot_stride, int64_t num_slots, int32_t page_size,
    const int32_t* page_table, int64_t page_table_stride_b, int32_t page_table_cols,
    const int32_t* lengths, const int32_t* row_offsets, int32_t num_rows, int32_t window,
    int32_t sinks, float sm_scale, void* output, int64_t output_stride_b, int64_t output_stride_h,
    float* lse, int64_t lse_stride_b, int64_t lse_stride_h, int64_t num_tokens, int32_t num_heads,
    void* scratch, size_t scratch_bytes, void* workspace, void* stream) {
  dense::Call c = common(q_nope, q_nope_stride_b, q_nope_stride_h, q_pe, q_pe_stride_b,
                         q_pe_stride_h, ckv_cache, ckv_slot_stride, kpe_cache, kpe_slot_stride,
                         num_slots, page_size, page_table, page_table_stride_b, page_table_cols,
                         lengths, row_offsets, num_rows, sm_scale, output, output_stride_b,
                         output_stride_h, lse, lse_stride_b, lse_stride_h, num_tokens, num_heads,
                         scratch, scratch_bytes, workspace, stream);
  c.p.window = window;
  c.p.sinks = sinks;
  return dense::attend(c);
}

int dsa_mla_decode_shared(
    const void* q_nope, int64_t q_nope_stride_b, int64_t q_nope_stride_h, const void* q_pe,
    int64_t q_pe_stride_b, int64_t q_pe_stride_h, const void* ckv_cache, int64_t ckv_slot_stride,
    const void* kpe_cache, int64_t kpe_slot_stride, int64_t num_slots, int32_t page_size,
    const int32_t* prefix_table, int64_t prefix_table_stride_g, int32_t prefix_table_cols,
    const int32_t* prefix_lengths, const int32_t* group_offsets, int32_t num_groups,
    const int32_t* page_table, int64_t page_table_stride_b, int32_t page_table_cols,
    const int32_t* lengths, const int32_t* row_offsets, int32_t num_rows, float sm_scale,
    void* output, int64_t output_stride_b, int64_t output_stride_h, float* lse,
    int64_t lse_stride_b, int64_t lse_stride_h, int64_t num_tokens, int32_t num_heads,
    void* scratch, size_t scratch_bytes, void* workspace, void* stream) {
  dense::Call c = common(q_nope, q_nope_stride_b, q_nope_stride_h, q_pe, q_pe_stride_b,
                         q_pe_stride_h, ckv_cache, ckv_slot_stride, kpe_cache, kpe_slot_stride,
                         num_slots, page_size, page_table, page_table_stride_b, page_table_cols,
                         lengths, row_offsets, num_rows, sm_scale, output, output_stride_b,
                         output_stride_h, lse, lse_stride_b, lse_stride_h, num_tokens, num_heads,
                         scratch, scratch_bytes, workspace, stream);
  c.p.pre = {prefix_table, prefix_table_stride_g, prefix_table_cols};
  c.p.pre_lengths = prefix_lengths;
  c.p.group_offsets = group_offsets;
  c.p.groups = num_groups;
  if (num_groups < 1 || (group_offsets == nullptr && num_groups != 1) ||
      (num_tokens > 0 && (prefix_table == nullptr || prefix_lengths == nullptr)))
    return DSA_ERR_INVALID_ARGUMENT;
  return dense::attend(c);
}

int dsa_merge_states(int32_t num_parts, const void* const* outputs,
                     const int64_t* output_strides, const float* const* lses,
                     const int64_t* lse_strides, void* output, int64_t output_stride_b,
                     int64_t output_stride_h, float* lse, int64_t lse_stride_b,
                     int64_t lse_stride_h, int64_t num_tokens, int32_t num_heads, void* stream) {
  using namespace dense;
  if (num_parts < 1 || num_parts > kMaxParts || num_tokens < 0 || num_heads < 1)
    return DSA_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return DSA_OK;
  if (!outputs || !output_strides || !lses || !lse_strides || !output || !lse ||
      num_tokens > INT64_MAX / num_heads || num_tokens * num_heads > (int64_t)INT32_MAX * 8)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned_rows(output, output_stride_b, output_stride_h)) return DSA_ERR_MISALIGNED;
  const Rows2 out_rows = {output, 2 * output_stride_b, 2 * output_stride_h, 2 * kDCkv},
              lse_rows = {lse, 4 * lse_stride_b, 4 * lse_stride_h, 4};
  MergeParams p = {};
  for (int i = 0; i < num_parts; ++i) {
    if (!outputs[i] || !lses[i]) return DSA_ERR_INVALID_ARGUMENT;
    p.o[i] = static_cast<const __nv_bfloat16*>(outputs[i]);
    p.z[i] = lses[i];
    p.o_sb[i] = output_strides[2 * i];
    p.o_sh[i] = output_strides[2 * i + 1];
    p.z_sb[i] = lse_strides[2 * i];
    p.z_sh[i] = lse_strides[2 * i + 1];
    if (!aligned_rows(p.o[i], p.o_sb[i], p.o_sh[i])) return DSA_ERR_MISALIGNED;
    const Rows2 o = {p.o[i], 2 * p.o_sb[i], 2 * p.o_sh[i], 2 * kDCkv},
                z = {p.z[i], 4 * p.z_sb[i], 4 * p.z_sh[i], 4};
    // a warp reads its own rows of all parts before it writes them, and no others
    auto spoils = [&](const Rows2& to, const Rows2& own, const Rows2& other) {
      return overlaps(to, other, num_tokens, num_heads) ||
             (!same_rows(to, own, num_tokens, num_heads) && overlaps(to, own, num_tokens, num_heads));
    };
    if (spoils(out_rows, o, z) || spoils(lse_rows, z, o))
      return DSA_ERR_INVALID_ARGUMENT;
  }
  p.out = static_cast<__nv_bfloat16*>(output);
  p.lse = lse;
  p.out_sb = output_stride_b;
  p.out_sh = output_stride_h;
  p.lse_sb = lse_stride_b;
  p.lse_sh = lse_stride_h;
  p.rows = num_tokens * num_heads;
  p.heads = num_heads;
  void (*const kern[kMaxParts])(MergeParams) = {
      merge_kernel<1>, merge_kernel<2>, merge_kernel<3>, merge_kernel<4>,
      merge_kernel<5>, merge_kernel<6>, merge_kernel<7>, merge_kernel<8>};
  const dim3 grid((unsigned)((p.rows + 7) / 8));
  return launch_pdl(kern[num_parts - 1], grid, 256, 0, static_cast<cudaStream_t>(stream), p);
}

}  // extern "C"
