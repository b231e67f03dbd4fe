// Sparse-MLA decode over the 8-bit latent cache.  For row b, head h and the selected slots k:
//     v[k]     = float(ckv_q8[k]) * ckv_scale[k / block]
//     z[h,k]   = sm_scale * (q_nope[b,h] . v[k] + q_pe[b,h] . kpe[k])
//     lse[b,h] = log2(sum_k exp(z[h,k]))
//     out[b,h] = bf16(sum_k softmax(z)[h,k] v[k])
//     weights[b,k] = sum_h softmax(z)[h,k]          (optional)
//
// One CTA per row, one head at a time, one warp per slot: the plain arrangement that the
// tests pin down first.
#pragma once

namespace dsa {
namespace q8 {

struct AttendParams {
  const __nv_bfloat16* qn;
  int64_t qn_sb, qn_sh;
  const __nv_bfloat16* qp;
  int64_t qp_sb, qp_sh;
  Cache cache;
  const int32_t* idx;
  int64_t idx_sb;
  PageTable table;  // pt == nullptr: idx holds slot ids
  __nv_bfloat16* out;
  int64_t out_sb, out_sh;
  float* lse;
  int64_t lse_sb, lse_sh;
  float* weights;
  int64_t w_sb;
  float* scratch;
  int32_t heads;
  int32_t topk;
  float scale_log2;
  uint32_t* err;
};

// The slot of entry k of row b; -1 for padding and, flagged, for what names no slot.
__device__ __forceinline__ int entry_slot(const AttendParams& p, int64_t b, int k) {
  const int e = __ldg(p.idx + b * p.idx_sb + k);
  if (e == -1) return -1;
  const int slot = p.table.pt != nullptr ? slot_at(p.table, b, e, p.cache.num_slots)
                   : (e >= 0 && e < p.cache.num_slots) ? e : -1;
  if (slot < 0) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
  return slot;
}

__global__ void __launch_bounds__(256) attend_kernel(const AttendParams p) {
  __shared__ float o_s[8][kDCkv];
  __shared__ float m_s[8], l_s[8];
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.weights != nullptr)
    for (int k = threadIdx.x; k < p.topk; k += 256) p.weights[b * p.w_sb + k] = 0.f;
  for (int h = 0; h < p.heads; ++h) {
    float q[16], o[16];
    const __nv_bfloat16* qn = p.qn + b * p.qn_sb + h * p.qn_sh + 16 * lane;
    const __nv_bfloat16* qp = p.qp + b * p.qp_sb + h * p.qp_sh + 2 * lane;
    const float qp0 = __bfloat162float(qp[0]), qp1 = __bfloat162float(qp[1]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      q[i] = __bfloat162float(qn[i]);
      o[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int k = warp; k < p.topk; k += 8) {
      const int slot = entry_slot(p, b, k);
      float z = -INFINITY;
      if (slot >= 0) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(p.cache.ckv + (int64_t)slot * p.cache.ckv_ss) + lane);
        const float scale = __ldg(p.cache.scale + (slot >> p.cache.block_shift));
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
        float v[16], dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 f = from_e4m3x2((ws[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
          v[2 * i] = f.x * scale;
          v[2 * i + 1] = f.y * scale;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) dot += q[i] * v[i];
        const __nv_bfloat16* kp = p.cache.kpe + (int64_t)slot * p.cache.kpe_ss + 2 * lane;
        dot += qp0 * __bfloat162float(kp[0]) + qp1 * __bfloat162float(kp[1]);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
        z = dot * p.scale_log2;
        const float mn = fmaxf(m, z);
        const float keep = m == -INFINITY ? 0.f : exp2f(m - mn), e = exp2f(z - mn);
        l = l * keep + e;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = o[i] * keep + e * v[i];
        m = mn;
      }
      if (p.weights != nullptr && lane == 0) p.scratch[b * p.topk + k] = z;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) o_s[warp][16 * lane + i] = o[i];
    if (lane == 0) {
      m_s[warp] = m;
      l_s[warp] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < 8; ++w) M = fmaxf(M, m_s[w]);
    // a warp without a score has l = 0; scores that are NaN leave its maximum at -inf, and l NaN
    for (int w = 0; w < 8; ++w) L += l_s[w] == 0.f ? 0.f : l_s[w] * exp2f(m_s[w] - M);
    const bool any = L != 0.f;
    const float lse = any ? M + log2f(L) : -INFINITY;
    for (int d = threadIdx.x; d < kDCkv; d += 256) {
      float a = 0.f;
      for (int w = 0; w < 8; ++w) a += l_s[w] == 0.f ? 0.f : o_s[w][d] * exp2f(m_s[w] - M);
      p.out[b * p.out_sb + h * p.out_sh + d] = __float2bfloat16_rn(any ? a / L : 0.f);
    }
    if (threadIdx.x == 0) p.lse[b * p.lse_sb + h * p.lse_sh] = lse;
    if (p.weights != nullptr)
      for (int k = threadIdx.x; k < p.topk; k += 256) {
        const float z = p.scratch[b * p.topk + k];
        if (z != -INFINITY) p.weights[b * p.w_sb + k] += exp2f(z - lse);
      }
    __syncthreads();
  }
}

}  // namespace q8
}  // namespace dsa
