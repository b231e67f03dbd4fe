// Python binding of the C ABI (include/dsa_b200.h) for torch tensors.  It reads the tensors'
// metadata in C++, so one decode call costs a few microseconds of host time instead of the
// tens that ctypes spends on 26 marshalled arguments and Python attribute reads.
//
// Every function returns the native status, or -1 when an argument is not in the plain form
// handled here (a CPU tensor, a dtype or shape mismatch, a non-unit inner stride, a pool
// that is not a uniform slot table); the Python caller then takes its general path, which
// validates, raises the precise error or copies to a supported layout.
#include <torch/extension.h>

#include <vector>

#include "dsa_b200.h"

namespace {

constexpr int64_t kNotHandled = -1;

// Slot stride of a [..., page, width] pool whose pages are uniformly spaced, else -1.
int64_t slot_stride(const at::Tensor& t, int64_t width) {
  if (t.size(-1) != width || t.stride(-1) != 1) return -1;
  if (t.dim() == 2) return t.stride(0);
  if (t.dim() == 3 && t.stride(0) == t.stride(1) * t.size(1)) return t.stride(1);
  return -1;
}

int64_t decode(const at::Tensor& q_nope, const at::Tensor& q_pe, const at::Tensor& ckv,
               const at::Tensor& kpe, const at::Tensor& idx, double sm_scale,
               const at::Tensor& out, const at::Tensor& lse, const at::Tensor& ws,
               int64_t stream) {
  const auto bf16 = at::kBFloat16;
  if (!q_nope.is_cuda() || q_nope.dim() != 3 || q_nope.size(2) != 512) return kNotHandled;
  const int64_t B = q_nope.size(0), H = q_nope.size(1);
  const auto dev = q_nope.device();
  for (const at::Tensor* t : {&q_pe, &ckv, &kpe, &idx, &out, &lse, &ws})
    if (t->device() != dev) return kNotHandled;
  if (q_nope.scalar_type() != bf16 || q_pe.scalar_type() != bf16 || ckv.scalar_type() != bf16 ||
      kpe.scalar_type() != bf16 || out.scalar_type() != bf16 ||
      idx.scalar_type() != at::kInt || lse.scalar_type() != at::kFloat)
    return kNotHandled;
  if (q_pe.dim() != 3 || q_pe.size(0) != B || q_pe.size(1) != H || q_pe.size(2) != 64 ||
      idx.dim() != 2 || idx.size(0) != B || out.dim() != 3 || out.size(0) != B ||
      out.size(1) != H || out.size(2) != 512 || lse.dim() != 2 || lse.size(0) != B ||
      lse.size(1) != H)
    return kNotHandled;
  if (q_nope.stride(2) != 1 || q_pe.stride(2) != 1 || idx.stride(1) != 1 || out.stride(2) != 1)
    return kNotHandled;
  const int64_t ckv_ss = slot_stride(ckv, 512), kpe_ss = slot_stride(kpe, 64);
  if (ckv_ss < 0 || kpe_ss < 0) return kNotHandled;
  const int64_t ckv_slots = ckv.numel() / 512, kpe_slots = kpe.numel() / 64;
  if (ckv_slots != kpe_slots) return kNotHandled;
  return dsa_sparse_mla_decode(
      q_nope.data_ptr(), q_nope.stride(0), q_nope.stride(1), q_pe.data_ptr(), q_pe.stride(0),
      q_pe.stride(1), ckv.data_ptr(), ckv_ss, kpe.data_ptr(), kpe_ss, ckv_slots,
      static_cast<const int32_t*>(idx.data_ptr()), idx.stride(0), (float)sm_scale,
      out.data_ptr(), out.stride(0), out.stride(1), static_cast<float*>(lse.data_ptr()),
      lse.stride(0), lse.stride(1), B, (int32_t)H, (int32_t)idx.size(1), ws.data_ptr(),
      (size_t)ws.numel(), reinterpret_cast<void*>(stream));
}

using OptTensor = c10::optional<at::Tensor>;

// An int32 tensor of `dim` dimensions with a unit inner stride on `dev`.
bool plain_i32(const at::Tensor& t, const at::Device& dev, int64_t dim) {
  return t.device() == dev && t.scalar_type() == at::kInt && t.dim() == dim && t.stride(-1) == 1;
}
bool plain_f32(const at::Tensor& t, const at::Device& dev, int64_t dim) {
  return t.device() == dev && t.scalar_type() == at::kFloat && t.dim() == dim && t.stride(-1) == 1;
}
int32_t* i32(const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
float* f32(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }

// The 8-bit cache's three pools: [pages, page, 512] e4m3, [pages, page / block] fp32 and
// [pages, page, 64] bf16.
struct Q8Cache {
  int64_t ckv_ss = -1, kpe_ss = -1, slots = 0;
  int32_t page = 0, block = 0;
  Q8Cache(const at::Tensor& ckv, const at::Tensor& scale, const at::Tensor& kpe,
          const at::Device& dev) {
    if (ckv.device() != dev || scale.device() != dev || kpe.device() != dev ||
        ckv.scalar_type() != at::kFloat8_e4m3fn || scale.scalar_type() != at::kFloat ||
        kpe.scalar_type() != at::kBFloat16 || ckv.dim() != 3 || kpe.dim() != 3 ||
        scale.dim() != 2 || !scale.is_contiguous())
      return;
    const int64_t P = ckv.size(0), n = ckv.size(1), nb = scale.size(1);
    if (kpe.size(0) != P || kpe.size(1) != n || scale.size(0) != P || nb < 1 || n % nb != 0 ||
        n > (1 << 20))
      return;
    ckv_ss = slot_stride(ckv, 512);
    kpe_ss = slot_stride(kpe, 64);
    slots = P * n;
    page = (int32_t)n;
    block = (int32_t)(n / nb);
  }
  bool ok() const { return ckv_ss >= 0 && kpe_ss >= 0; }
};

int64_t decode_q8(const at::Tensor& q_nope, const at::Tensor& q_pe, const at::Tensor& ckv,
                  const at::Tensor& scale, const at::Tensor& kpe, const OptTensor& page_table,
                  const at::Tensor& idx, double sm_scale, const at::Tensor& out,
                  const at::Tensor& lse, const OptTensor& weights, const at::Tensor& ws,
                  int64_t stream) {
  const auto bf16 = at::kBFloat16;
  if (!q_nope.is_cuda() || q_nope.dim() != 3 || q_nope.size(2) != 512) return kNotHandled;
  const int64_t B = q_nope.size(0), H = q_nope.size(1);
  const auto dev = q_nope.device();
  if (q_pe.device() != dev || out.device() != dev || lse.device() != dev || ws.device() != dev ||
      q_nope.scalar_type() != bf16 || q_pe.scalar_type() != bf16 || out.scalar_type() != bf16 ||
      lse.scalar_type() != at::kFloat || !plain_i32(idx, dev, 2))
    return kNotHandled;
  if (q_pe.dim() != 3 || q_pe.size(0) != B || q_pe.size(1) != H || q_pe.size(2) != 64 ||
      idx.size(0) != B || out.dim() != 3 || out.size(0) != B || out.size(1) != H ||
      out.size(2) != 512 || lse.dim() != 2 || lse.size(0) != B || lse.size(1) != H)
    return kNotHandled;
  if (q_nope.stride(2) != 1 || q_pe.stride(2) != 1 || out.stride(2) != 1) return kNotHandled;
  const Q8Cache c(ckv, scale, kpe, dev);
  if (!c.ok()) return kNotHandled;
  const bool paged = page_table.has_value();
  if (paged && (!plain_i32(*page_table, dev, 2) || page_table->size(0) != B)) return kNotHandled;
  const int64_t topk = idx.size(1);
  at::Tensor scratch;
  if (weights.has_value()) {
    if (!plain_f32(*weights, dev, 2) || weights->size(0) != B || weights->size(1) != topk)
      return kNotHandled;
    scratch = at::empty({(int64_t)dsa_q8_scratch_size(B, (int32_t)H, (int32_t)topk)},
                        at::TensorOptions().dtype(at::kByte).device(dev));
  }
  return dsa_sparse_mla_decode_q8(
      q_nope.data_ptr(), q_nope.stride(0), q_nope.stride(1), q_pe.data_ptr(), q_pe.stride(0),
      q_pe.stride(1), ckv.data_ptr(), c.ckv_ss, f32(scale), c.block, kpe.data_ptr(), c.kpe_ss,
      c.slots, paged ? i32(*page_table) : nullptr, paged ? page_table->stride(0) : 0,
      paged ? (int32_t)page_table->size(1) : 0, c.page, i32(idx), idx.stride(0), (float)sm_scale,
      out.data_ptr(), out.stride(0), out.stride(1), f32(lse), lse.stride(0), lse.stride(1),
      weights.has_value() ? f32(*weights) : nullptr, weights.has_value() ? weights->stride(0) : 0,
      B, (int32_t)H, (int32_t)topk, scratch.defined() ? scratch.data_ptr() : nullptr,
      scratch.defined() ? (size_t)scratch.numel() : 0, ws.data_ptr(),
      reinterpret_cast<void*>(stream));
}

int64_t append_q8(const at::Tensor& ckv, const at::Tensor& kpe, const at::Tensor& offsets,
                  const at::Tensor& starts, const at::Tensor& page_table, const at::Tensor& ckv_q8,
                  const at::Tensor& scale, const at::Tensor& kpe_cache, const at::Tensor& ws,
                  int64_t stream) {
  const auto dev = ckv_q8.device();
  const int64_t R = starts.dim() == 1 ? starts.size(0) : -1;
  if (ckv.device() != dev || kpe.device() != dev || ckv.scalar_type() != at::kBFloat16 ||
      kpe.scalar_type() != at::kBFloat16 || ckv.dim() != 2 || kpe.dim() != 2 ||
      ckv.size(1) != 512 || kpe.size(1) != 64 || kpe.size(0) != ckv.size(0) ||
      ckv.stride(1) != 1 || kpe.stride(1) != 1 || R < 1 || !plain_i32(starts, dev, 1) ||
      !plain_i32(offsets, dev, 1) || offsets.size(0) != R + 1 || !plain_i32(page_table, dev, 2) ||
      page_table.size(0) != R || ws.device() != dev)
    return kNotHandled;
  const Q8Cache c(ckv_q8, scale, kpe_cache, dev);
  if (!c.ok()) return kNotHandled;
  return dsa_append_q8(ckv.data_ptr(), ckv.stride(0), kpe.data_ptr(), kpe.stride(0), ckv.size(0),
                       i32(offsets), i32(starts), (int32_t)R, i32(page_table),
                       page_table.stride(0), (int32_t)page_table.size(1), c.page,
                       ckv_q8.data_ptr(), c.ckv_ss, f32(scale), c.block, kpe_cache.data_ptr(),
                       c.kpe_ss, c.slots, ws.data_ptr(), reinterpret_cast<void*>(stream));
}

int64_t accumulate_weights(const at::Tensor& weights, const at::Tensor& positions,
                           const at::Tensor& acc, const OptTensor& offsets, const at::Tensor& ws,
                           int64_t stream) {
  const auto dev = acc.device();
  if (!plain_f32(weights, dev, 2) || !plain_i32(positions, dev, 2) || !plain_f32(acc, dev, 2) ||
      positions.sizes() != weights.sizes() || ws.device() != dev || acc.size(1) > INT32_MAX ||
      weights.size(1) > INT32_MAX)
    return kNotHandled;
  const int64_t T = weights.size(0), R = acc.size(0);
  if (offsets.has_value() ? !plain_i32(*offsets, dev, 1) || offsets->size(0) != R + 1 : R != T)
    return kNotHandled;
  return dsa_accumulate_weights(f32(weights), weights.stride(0), i32(positions),
                                positions.stride(0), T, (int32_t)weights.size(1), f32(acc),
                                acc.stride(0), (int32_t)acc.size(1), (int32_t)R,
                                offsets.has_value() ? i32(*offsets) : nullptr, ws.data_ptr(),
                                reinterpret_cast<void*>(stream));
}

int64_t evict_positions(const at::Tensor& acc, const at::Tensor& lengths, int64_t budget,
                        int64_t sinks, int64_t recent, const at::Tensor& keep,
                        const at::Tensor& new_lengths, const OptTensor& new_acc, int64_t stream) {
  const auto dev = acc.device();
  if (!plain_f32(acc, dev, 2) || !plain_i32(lengths, dev, 1) || lengths.size(0) != acc.size(0))
    return kNotHandled;
  if (new_acc.has_value() && (!plain_f32(*new_acc, dev, 2) || new_acc->size(0) != acc.size(0)))
    return kNotHandled;
  return dsa_evict_positions(f32(acc), acc.stride(0), i32(lengths), acc.size(0),
                             (int32_t)acc.size(1), (int32_t)budget, (int32_t)sinks,
                             (int32_t)recent, i32(keep), keep.stride(0), i32(new_lengths),
                             new_acc.has_value() ? f32(*new_acc) : nullptr,
                             new_acc.has_value() ? new_acc->stride(0) : 0,
                             new_acc.has_value() ? (int32_t)new_acc->size(1) : 0,
                             reinterpret_cast<void*>(stream));
}

int64_t compact_q8(const at::Tensor& keep, const at::Tensor& page_table,
                   const at::Tensor& new_page_table, const at::Tensor& ckv_q8,
                   const at::Tensor& scale, const at::Tensor& kpe_cache, const at::Tensor& ws,
                   int64_t stream) {
  const auto dev = ckv_q8.device();
  if (!plain_i32(keep, dev, 2) || !plain_i32(page_table, dev, 2) ||
      !plain_i32(new_page_table, dev, 2) || page_table.size(0) != keep.size(0) ||
      new_page_table.size(0) != keep.size(0) || ws.device() != dev)
    return kNotHandled;
  const Q8Cache c(ckv_q8, scale, kpe_cache, dev);
  if (!c.ok()) return kNotHandled;
  return dsa_compact_q8(i32(keep), keep.stride(0), (int32_t)keep.size(0), (int32_t)keep.size(1),
                        i32(page_table), page_table.stride(0), (int32_t)page_table.size(1),
                        i32(new_page_table), new_page_table.stride(0),
                        (int32_t)new_page_table.size(1), c.page, ckv_q8.data_ptr(), c.ckv_ss,
                        f32(scale), c.block, kpe_cache.data_ptr(), c.kpe_ss, c.slots,
                        ws.data_ptr(), reinterpret_cast<void*>(stream));
}

// Queries, pools and outputs of a dense call; page_size -1: the pools' page dimension.
struct DenseArgs {
  int64_t B = 0, H = 0, ckv_ss = -1, kpe_ss = -1, slots = 0, page = 0;
  bool ok = false;
  DenseArgs(const at::Tensor& q_nope, const at::Tensor& q_pe, const at::Tensor& ckv,
            const at::Tensor& kpe, int64_t page_size, const at::Tensor& out,
            const at::Tensor& lse, const at::Tensor& ws) {
    const auto bf16 = at::kBFloat16;
    if (!q_nope.is_cuda() || q_nope.dim() != 3 || q_nope.size(2) != 512) return;
    B = q_nope.size(0);
    H = q_nope.size(1);
    const auto dev = q_nope.device();
    for (const at::Tensor* t : {&q_pe, &ckv, &kpe, &out, &lse, &ws})
      if (t->device() != dev) return;
    for (const at::Tensor* t : {&q_nope, &q_pe, &ckv, &kpe, &out})
      if (t->scalar_type() != bf16) return;
    if (lse.scalar_type() != at::kFloat || q_pe.dim() != 3 || q_pe.size(0) != B ||
        q_pe.size(1) != H || q_pe.size(2) != 64 || out.dim() != 3 || out.size(0) != B ||
        out.size(1) != H || out.size(2) != 512 || lse.dim() != 2 || lse.size(0) != B ||
        lse.size(1) != H || q_nope.stride(2) != 1 || q_pe.stride(2) != 1 || out.stride(2) != 1 ||
        ckv.dim() < 2 || kpe.dim() < 2 || ckv.numel() == 0)
      return;
    ckv_ss = slot_stride(ckv, 512);
    kpe_ss = slot_stride(kpe, 64);
    if (ckv_ss < 0 || kpe_ss < 0) return;
    slots = ckv.numel() / 512;
    page = page_size;
    if (page < 0 && ckv.dim() == 3) page = ckv.size(1);
    ok = slots == kpe.numel() / 64 && page >= 1 && page <= (1 << 30);
  }
};

// The rows of a dense call: page tables, lengths, and offsets or none (a token a row).
bool plain_rows(const at::Tensor& table, const at::Tensor& lengths, const OptTensor& offsets,
                int64_t tokens, const at::Device& dev) {
  if (!plain_i32(table, dev, 2) || !plain_i32(lengths, dev, 1) ||
      table.size(0) != lengths.size(0) || table.size(1) < 1)
    return false;
  if (!offsets.has_value()) return lengths.size(0) == tokens;
  return plain_i32(*offsets, dev, 1) && offsets->size(0) == lengths.size(0) + 1;
}

at::Tensor dense_scratch(int64_t B, int64_t H, bool shared, const at::Device& dev) {
  return at::empty({(int64_t)dsa_dense_scratch_size(B, (int32_t)H, shared ? 1 : 0)},
                   at::TensorOptions().dtype(at::kByte).device(dev));
}

int64_t decode_window(const at::Tensor& q_nope, const at::Tensor& q_pe, const at::Tensor& ckv,
                      const at::Tensor& kpe, int64_t page_size, const at::Tensor& page_table,
                      const at::Tensor& lengths, const OptTensor& row_offsets, int64_t window,
                      int64_t sinks, double sm_scale, const at::Tensor& out,
                      const at::Tensor& lse, const at::Tensor& ws, int64_t stream) {
  const DenseArgs a(q_nope, q_pe, ckv, kpe, page_size, out, lse, ws);
  const auto dev = q_nope.device();
  if (!a.ok || !plain_rows(page_table, lengths, row_offsets, a.B, dev)) return kNotHandled;
  const at::Tensor scratch = dense_scratch(a.B, a.H, false, dev);
  return dsa_mla_decode_window(
      q_nope.data_ptr(), q_nope.stride(0), q_nope.stride(1), q_pe.data_ptr(), q_pe.stride(0),
      q_pe.stride(1), ckv.data_ptr(), a.ckv_ss, kpe.data_ptr(), a.kpe_ss, a.slots,
      (int32_t)a.page, i32(page_table), page_table.stride(0), (int32_t)page_table.size(1),
      i32(lengths), row_offsets.has_value() ? i32(*row_offsets) : nullptr,
      (int32_t)lengths.size(0), (int32_t)window, (int32_t)sinks, (float)sm_scale, out.data_ptr(),
      out.stride(0), out.stride(1), f32(lse), lse.stride(0), lse.stride(1), a.B, (int32_t)a.H,
      scratch.data_ptr(), (size_t)scratch.numel(), ws.data_ptr(), reinterpret_cast<void*>(stream));
}

int64_t decode_shared(const at::Tensor& q_nope, const at::Tensor& q_pe, const at::Tensor& ckv,
                      const at::Tensor& kpe, int64_t page_size, const at::Tensor& prefix_table,
                      const at::Tensor& prefix_lengths, const OptTensor& group_offsets,
                      const at::Tensor& page_table, const at::Tensor& lengths,
                      const OptTensor& row_offsets, double sm_scale, const at::Tensor& out,
                      const at::Tensor& lse, const at::Tensor& ws, int64_t stream) {
  const DenseArgs a(q_nope, q_pe, ckv, kpe, page_size, out, lse, ws);
  const auto dev = q_nope.device();
  if (!a.ok || !plain_rows(page_table, lengths, row_offsets, a.B, dev)) return kNotHandled;
  const int64_t groups = prefix_lengths.numel();
  if (!plain_i32(prefix_table, dev, 2) || !plain_i32(prefix_lengths, dev, 1) || groups < 1 ||
      prefix_table.size(0) != groups || prefix_table.size(1) < 1)
    return kNotHandled;
  if (group_offsets.has_value()
          ? !plain_i32(*group_offsets, dev, 1) || group_offsets->size(0) != groups + 1
          : groups != 1)
    return kNotHandled;
  const at::Tensor scratch = dense_scratch(a.B, a.H, true, dev);
  return dsa_mla_decode_shared(
      q_nope.data_ptr(), q_nope.stride(0), q_nope.stride(1), q_pe.data_ptr(), q_pe.stride(0),
      q_pe.stride(1), ckv.data_ptr(), a.ckv_ss, kpe.data_ptr(), a.kpe_ss, a.slots,
      (int32_t)a.page, i32(prefix_table), prefix_table.stride(0), (int32_t)prefix_table.size(1),
      i32(prefix_lengths), group_offsets.has_value() ? i32(*group_offsets) : nullptr,
      (int32_t)groups, i32(page_table), page_table.stride(0), (int32_t)page_table.size(1),
      i32(lengths), row_offsets.has_value() ? i32(*row_offsets) : nullptr,
      (int32_t)lengths.size(0), (float)sm_scale, out.data_ptr(), out.stride(0), out.stride(1),
      f32(lse), lse.stride(0), lse.stride(1), a.B, (int32_t)a.H, scratch.data_ptr(),
      (size_t)scratch.numel(), ws.data_ptr(), reinterpret_cast<void*>(stream));
}

int64_t merge_states(const std::vector<at::Tensor>& outs, const std::vector<at::Tensor>& lses,
                     const at::Tensor& out, const at::Tensor& lse, int64_t stream) {
  constexpr size_t kMost = 8;
  const size_t n = outs.size();
  if (n < 1 || n > kMost || lses.size() != n || !out.is_cuda() || out.dim() != 3 ||
      out.size(2) != 512 || out.scalar_type() != at::kBFloat16 || out.stride(2) != 1)
    return kNotHandled;
  const auto dev = out.device();
  if (lse.device() != dev || lse.scalar_type() != at::kFloat || lse.dim() != 2 ||
      lse.size(0) != out.size(0) || lse.size(1) != out.size(1))
    return kNotHandled;
  const void* o[kMost];
  const float* z[kMost];
  int64_t os[2 * kMost], zs[2 * kMost];
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &a = outs[i], &b = lses[i];
    if (a.device() != dev || a.scalar_type() != at::kBFloat16 || a.sizes() != out.sizes() ||
        a.stride(2) != 1 || b.device() != dev || b.scalar_type() != at::kFloat ||
        b.sizes() != lse.sizes())
      return kNotHandled;
    o[i] = a.data_ptr();
    z[i] = f32(b);
    os[2 * i] = a.stride(0);
    os[2 * i + 1] = a.stride(1);
    zs[2 * i] = b.stride(0);
    zs[2 * i + 1] = b.stride(1);
  }
  return dsa_merge_states((int32_t)n, o, os, z, zs, out.data_ptr(), out.stride(0), out.stride(1),
                          f32(lse), lse.stride(0), lse.stride(1), out.size(0),
                          (int32_t)out.size(1), reinterpret_cast<void*>(stream));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("decode", &decode, "DSA sparse-MLA decode through the C ABI (status, -1: not handled)");
  m.def("decode_q8", &decode_q8, "decode over the 8-bit cache");
  m.def("append_q8", &append_q8, "tokens into the 8-bit cache");
  m.def("accumulate_weights", &accumulate_weights, "attention weights into running totals");
  m.def("evict_positions", &evict_positions, "the positions an eviction keeps");
  m.def("decode_window", &decode_window, "attention over a window and sinks");
  m.def("decode_shared", &decode_shared, "attention of rows that share prefixes");
  m.def("merge_states", &merge_states, "attention results joined");
  m.def("compact_q8", &compact_q8, "kept tokens of the 8-bit cache to new pages");
}
