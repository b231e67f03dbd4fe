// Dense attention over the bf16 latent cache: a sliding window with sinks, rows behind a shared
// prefix, and the join of attention results over separate sets of positions.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

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
  const __nv_bfloat16 *qn, *qp, *ckv, *kpe;
  int64_t qn_sb, qn_sh, qp_sb, qp_sh, ckv_ss, kpe_ss, num_slots;
  Table own, pre;                  // pre.pt == nullptr: no prefixes
  int32_t page_shift;
  const int32_t *lengths, *row_offsets;     // row_offsets nullptr: a token a row
  const int32_t *pre_lengths, *group_offsets;  // group_offsets nullptr: one group of all rows
  int32_t rows, groups, tokens, heads;
  int32_t window, sinks;
  float scale_log2;
  __nv_bfloat16* out;
  int64_t out_sb, out_sh;
  float* lse;
  int64_t lse_sb, lse_sh;
  uint32_t* err;
};

// The last i in [0, n) with offsets[i] <= x, -1 if there is none (ascending offsets).
__device__ __forceinline__ int owner(const int32_t* offsets, int n, int x) {
  int lo = -1, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(offsets + mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A warp is one head of one token: lane l holds 16 + 2 of the query's values and of the output's
// 512; positions one after another with the running maximum and sum.
__global__ void __launch_bounds__(256) attend_kernel(const Params p) {
  const int t = blockIdx.x, h = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  int row = t, n = 1, j = 0;
  if (p.row_offsets != nullptr) {
    row = owner(p.row_offsets, p.rows + 1, t);
    if (row < 0 || row >= p.rows) return;  // a token of no row: left as it is
    j = t - p.row_offsets[row];
    n = p.row_offsets[row + 1] - p.row_offsets[row];
  }
  float q[18], o[16];
  for (int i = 0; i < 16; ++i) {
    q[i] = __bfloat162float(p.qn[t * p.qn_sb + h * p.qn_sh + lane * 16 + i]);
    o[i] = 0.f;
  }
  for (int i = 0; i < 2; ++i)
    q[16 + i] = __bfloat162float(p.qp[t * p.qp_sb + h * p.qp_sh + lane * 2 + i]);
  float m = -INFINITY, l = 0.f;
  bool bad = false, any = false;
  auto key = [&](const Table& tab, int r, int pos) {
    const int pg = pos >> p.page_shift;
    const int page = pg < tab.cols ? __ldg(tab.pt + r * tab.sb + pg) : -1;
    const int64_t slot = ((int64_t)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
    if (page < 0 || slot >= p.num_slots) {
      bad = true;
      return;
    }
    const __nv_bfloat16* k = p.ckv + slot * p.ckv_ss + lane * 16;
    const __nv_bfloat16* e = p.kpe + slot * p.kpe_ss + lane * 2;
    float v[16], s = 0.f;
    for (int i = 0; i < 16; ++i) {
      v[i] = __bfloat162float(k[i]);
      s += q[i] * v[i];
    }
    for (int i = 0; i < 2; ++i) s += q[16 + i] * __bfloat162float(e[i]);
    for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    s *= p.scale_log2;
    any = true;
    const float mn = fmaxf(m, s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float a = exp2f(m - base), w = exp2f(s - base);
    l = l * a + w;
    for (int i = 0; i < 16; ++i) o[i] = o[i] * a + w * v[i];
    m = mn;
  };
  if (p.pre.pt != nullptr) {
    int g = 0;
    if (p.group_offsets != nullptr) g = owner(p.group_offsets, p.groups + 1, row);
    if (g >= 0 && g < p.groups) {
      const int len = p.pre_lengths[g];
      const int cap = p.pre.cols << p.page_shift;
      bad |= len > cap;
      for (int i = 0; i < min(len, cap); ++i) key(p.pre, g, i);
    }
  }
  const int pos = p.lengths[row] - n + j, cap = p.own.cols << p.page_shift;
  bad |= pos >= cap;
  const int last = min(pos, cap - 1), first = max(0, p.window >= pos + 1 ? 0 : pos - p.window + 1);
  for (int i = 0; i <= min(last, min(p.sinks, first) - 1); ++i) key(p.own, row, i);
  for (int i = first; i <= last; ++i) key(p.own, row, i);
  if (bad && lane == 0) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
  for (int i = 0; i < 16; ++i)
    p.out[t * p.out_sb + h * p.out_sh + lane * 16 + i] = __float2bfloat16(any ? o[i] / l : 0.f);
  if (lane == 0) p.lse[t * p.lse_sb + h * p.lse_sh] = any ? m + log2f(l) : -INFINITY;
}

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

template <typename P>
int launch(void (*kern)(P), dim3 grid, unsigned threads, cudaStream_t st, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? DSA_OK : DSA_ERR_CUDA;
}

// Whether rows of `width` elements at a + t sb + h sh and at b + t sb + h sh meet, for any
// (t, h) of either (bytes throughout).
bool same_grid_meets(int64_t d, int64_t sb, int64_t sh, int64_t tokens, int64_t heads,
                     int64_t width) {
  for (int64_t dh = -(heads - 1); dh < heads; ++dh) {
    const int64_t rest = d - dh * sh;
    if (sb == 0 || tokens == 1) {
      if (std::abs(rest) < width) return true;
      continue;
    }
    const int64_t q = rest / sb;
    for (int64_t dt = q - 1; dt <= q + 1; ++dt)
      if (std::abs(dt) < tokens && std::abs(rest - dt * sb) < width) return true;
  }
  return false;
}

struct Rows2 {
  const void* p;
  int64_t sb, sh;  // bytes
};

// Whether writing `out` may change what is still to be read of `part`: they overlap without
// being the same rows.
bool overlaps(const Rows2& out, const Rows2& part, int64_t tokens, int64_t heads, int64_t width) {
  if (out.p == part.p && out.sb == part.sb && out.sh == part.sh) return false;
  auto range = [&](const Rows2& r, int64_t& lo, int64_t& hi) {
    const int64_t b = (tokens - 1) * r.sb, h = (heads - 1) * r.sh;
    lo = (int64_t) reinterpret_cast<intptr_t>(r.p) + std::min<int64_t>(b, 0) + std::min<int64_t>(h, 0);
    hi = (int64_t) reinterpret_cast<intptr_t>(r.p) + std::max<int64_t>(b, 0) +
         std::max<int64_t>(h, 0) + width;
  };
  int64_t a0, a1, b0, b1;
  range(out, a0, a1);
  range(part, b0, b1);
  if (a1 <= b0 || b1 <= a0) return false;
  if (out.sb != part.sb || out.sh != part.sh) return true;
  return same_grid_meets((int64_t) reinterpret_cast<intptr_t>(out.p) -
                             (int64_t) reinterpret_cast<intptr_t>(part.p),
                         out.sb, out.sh, tokens, heads, width);
}

bool aligned_rows(const void* p, int64_t sb, int64_t sh) {
  return aligned16(p) && sb % 8 == 0 && sh % 8 == 0;
}

// What window and shared have in common; `pre` fields are zero for a window call.
struct Call {
  Params p;
  int32_t page_size;
  void* scratch;
  size_t scratch_bytes;
  void* workspace;
  void* stream;
};

int check_table(const Table& t, int32_t page_size) {
  if (t.pt == nullptr || t.cols < 1 || (t.sb < t.cols)) return DSA_ERR_INVALID_ARGUMENT;
  return (int64_t)t.cols * page_size > INT32_MAX / 2 ? DSA_ERR_INVALID_ARGUMENT : DSA_OK;
}

int attend(Call& c) {
  Params& p = c.p;
  if (p.tokens < 0 || p.rows < 0) return DSA_ERR_INVALID_ARGUMENT;
  if (!heads_supported(p.heads)) return DSA_ERR_UNSUPPORTED;
  if (p.tokens == 0 || p.rows == 0) return DSA_OK;
  if (p.row_offsets == nullptr && p.rows != p.tokens) return DSA_ERR_INVALID_ARGUMENT;
  if (!p.qn || !p.qp || !p.ckv || !p.kpe || !p.lengths || !p.out || !p.lse ||
      p.num_slots < 1 || p.num_slots > INT32_MAX - 64 || p.ckv_ss < kDCkv || p.kpe_ss < kDKpe ||
      p.window < 0 || p.sinks < 0 || c.page_size < 1 || (c.page_size & (c.page_size - 1)))
    return DSA_ERR_INVALID_ARGUMENT;
  int rc = check_table(p.own, c.page_size);
  if (rc == DSA_OK && p.pre.pt != nullptr) rc = check_table(p.pre, c.page_size);
  if (rc != DSA_OK) return rc;
  if (!aligned_rows(p.qn, p.qn_sb, p.qn_sh) || !aligned_rows(p.qp, p.qp_sb, p.qp_sh) ||
      !aligned_rows(p.ckv, p.ckv_ss, 0) || !aligned_rows(p.kpe, p.kpe_ss, 0) ||
      !aligned_rows(p.out, p.out_sb, p.out_sh))
    return DSA_ERR_MISALIGNED;
  if (c.workspace == nullptr) return DSA_ERR_WORKSPACE;
  p.page_shift = 0;
  while ((1 << p.page_shift) < c.page_size) ++p.page_shift;
  p.window = std::min(p.window, kAll);
  p.sinks = std::min(p.sinks, kAll);
  p.err = static_cast<uint32_t*>(c.workspace);
  attend_kernel<<<dim3((unsigned)p.tokens, (unsigned)(p.heads / 8)), 256, 0,
                  static_cast<cudaStream_t>(c.stream)>>>(p);
  return cudaGetLastError() == cudaSuccess ? DSA_OK : DSA_ERR_CUDA;
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
  p.qn = static_cast<const __nv_bfloat16*>(q_nope);
  p.qn_sb = q_nope_stride_b;
  p.qn_sh = q_nope_stride_h;
  p.qp = static_cast<const __nv_bfloat16*>(q_pe);
  p.qp_sb = q_pe_stride_b;
  p.qp_sh = q_pe_stride_h;
  p.ckv = static_cast<const __nv_bfloat16*>(ckv_cache);
  p.ckv_ss = ckv_slot_stride;
  p.kpe = static_cast<const __nv_bfloat16*>(kpe_cache);
  p.kpe_ss = kpe_slot_stride;
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
  (void)shared;
  return 16;
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
    if (overlaps({output, 2 * output_stride_b, 2 * output_stride_h},
                 {p.o[i], 2 * p.o_sb[i], 2 * p.o_sh[i]}, num_tokens, num_heads, 2 * kDCkv) ||
        overlaps({lse, 4 * lse_stride_b, 4 * lse_stride_h}, {p.z[i], 4 * p.z_sb[i], 4 * p.z_sh[i]},
                 num_tokens, num_heads, 4))
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
  return launch(kern[num_parts - 1], grid, 256, static_cast<cudaStream_t>(stream), p);
}

}  // extern "C"
