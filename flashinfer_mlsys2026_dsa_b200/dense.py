"""Dense attention over the bf16 latent cache, and the join of attention results.

:func:`kernel_window` attends over a sliding window and the sequence's first positions (sinks),
:func:`kernel_shared` over a prefix that many rows share and the rows' own positions;
:func:`merge_states` joins results over separate sets of positions, such as a sparse selection's
(:func:`ops.kernel`) and a window's.

Caches, queries, ``output`` and ``lse`` are those of :func:`ops.kernel_paged`.  A row is a
sequence; its tokens stand at its last positions.  With ``row_offsets`` (int32 [rows + 1],
ascending) row r has the tokens ``[row_offsets[r], row_offsets[r + 1])`` (none, one or many:
decode, drafted tokens, prompt chunks); without it each row has one token.  Tokens outside the
offsets are left as they are, so a batch may be padded.  A token that sees nothing gets output 0
and lse -inf.  Lengths and offsets are read on the device, so captured graphs follow them.

All calls launch on the current CUDA stream and do not synchronise; there is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native, ops
from .ops import D_CKV, D_KPE, SUPPORTED_HEADS, _check, _slot_view
from .q8 import _done, _fast, _finish, _launch_on, _need, _row_offsets, _unit

_BF16 = torch.bfloat16
ALL_POSITIONS = 0x3FFFFFFF
MAX_PARTS = 8


def _common(q_nope, q_pe, ckv_cache, kpe_cache, output, lse, page_size):
    """Checks queries, pools and outputs; returns (ckv, kpe, page_size) with the pools as slots."""
    _need("q_nope", q_nope, _BF16, 3)
    dev = q_nope.device
    B, H, width = q_nope.shape
    if width != D_CKV:
        raise ValueError(f"q_nope must be [num_tokens, num_heads, {D_CKV}], got {tuple(q_nope.shape)}")
    if H not in SUPPORTED_HEADS:
        raise ValueError(f"num_heads={H} is not supported (supported: {SUPPORTED_HEADS})")
    for name, t, dtype, shape in (("q_pe", q_pe, _BF16, (B, H, D_KPE)),
                                  ("output", output, _BF16, (B, H, D_CKV)),
                                  ("lse", lse, torch.float32, (B, H))):
        _need(name, t, dtype, len(shape), dev)
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    for name, t, width in (("ckv_cache", ckv_cache, D_CKV), ("kpe_cache", kpe_cache, D_KPE)):
        _need(name, t, _BF16, t.dim() if isinstance(t, torch.Tensor) else 0, dev)
        if t.dim() < 2 or t.shape[-1] != width:
            raise ValueError(f"{name} must be [pages, page, {width}], got {tuple(t.shape)}")
    if page_size is None:
        if ckv_cache.dim() != 3:
            raise ValueError("page_size is required for a pool that is not [pages, page_size, 512]")
        page_size = ckv_cache.shape[-2]
    page_size = int(page_size)
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two, got {page_size}")
    ckv = _slot_view(ckv_cache, D_CKV, "ckv_cache")
    kpe = _slot_view(kpe_cache, D_KPE, "kpe_cache")
    if ckv.shape[0] != kpe.shape[0]:
        raise ValueError("ckv_cache and kpe_cache hold different slot counts")
    return ckv, kpe, page_size


def _sequences(names, table, lengths, dev):
    """Checks a page table and its lengths; returns them with unit inner strides."""
    _need(names[0], table, torch.int32, 2, dev)
    _need(names[1], lengths, torch.int32, 1, dev)
    if table.shape[0] != lengths.shape[0] or table.shape[1] < 1:
        raise ValueError(f"{names[0]} must be [{lengths.shape[0]}, max_pages], as {names[1]} has "
                         f"{lengths.shape[0]} entries, got {tuple(table.shape)}")
    return _unit(table), lengths.contiguous()


def _rows(row_offsets, rows, tokens, dev):
    if row_offsets is not None:
        return _row_offsets(row_offsets, rows, dev)
    if rows != tokens:
        raise ValueError(f"without row_offsets each of the {tokens} tokens is a row, got {rows} lengths")
    return None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _attend(what, prefix, tail, q_nope, q_pe, ckv, kpe, page, table, lengths, row_offsets, sm_scale,
            output, lse):
    """The general route: lays out what the binding does not take and calls the C ABI."""
    B, H, _ = q_nope.shape
    if B == 0 or lengths.shape[0] == 0:
        return
    q_nope, q_pe = _unit(q_nope), _unit(q_pe)
    # tokens of no row keep what they hold, so a laid-out copy starts with it
    out_t = output if output.stride(-1) == 1 else output.contiguous()
    lib = _native._lib or _native.load()
    guard, stream = _launch_on(q_nope)
    with guard:
        ws = ops.workspace_for(q_nope.device, stream, B, H, 1)
        scratch = torch.empty(lib.dsa_dense_scratch_size(B, H, int(bool(prefix))),
                              dtype=torch.uint8, device=q_nope.device)
        rc = getattr(lib, what)(
            q_nope.data_ptr(), q_nope.stride(0), q_nope.stride(1),
            q_pe.data_ptr(), q_pe.stride(0), q_pe.stride(1),
            ckv.data_ptr(), ckv.stride(0), kpe.data_ptr(), kpe.stride(0), ckv.shape[0], page,
            *prefix, table.data_ptr(), table.stride(0), table.shape[1], lengths.data_ptr(),
            _ptr(row_offsets), lengths.shape[0], *tail, float(sm_scale),
            out_t.data_ptr(), out_t.stride(0), out_t.stride(1),
            lse.data_ptr(), lse.stride(0), lse.stride(1), B, H,
            scratch.data_ptr(), scratch.numel(), ws.data_ptr(), stream)
        _check(rc, what)
        if out_t is not output:
            output.copy_(out_t)
        _finish(rc, q_nope, what)


def kernel_window(q_nope, q_pe, ckv_cache, kpe_cache, page_table, lengths, sm_scale, output, lse,
                  window=None, sinks=0, row_offsets=None, page_size=None) -> None:
    """Attention over a sliding window and the first positions (writes ``output`` and ``lse``).

    The token at position p sees the positions q <= p with ``q < sinks`` or ``q > p - window``;
    ``window`` None: all q <= p.  ``page_table`` [rows, max_pages] int32 lists each row's pool
    pages, ``lengths`` [rows] int32 counts its positions, its own tokens' among them.
    ``page_size`` defaults to the pools' page dimension.  A position past the row's table or on a
    negative page is left out and flagged in :func:`ops.read_device_errors`.

    What a token must not see may hold anything, with one exception: where a row has several
    tokens, a NaN or infinity at a position that one of them sees may reach the others.

    Without ``row_offsets``, 38 to 74 rows get one CTA pair each on a B200: best where they see
    about as many positions each.  For rows of very unequal length pass ``row_offsets``
    0, 1, 2, .. rows, which spread each row over several pairs.
    """
    what = "dsa_mla_decode_window"
    reach = ALL_POSITIONS if window is None else int(window)
    sinks = int(sinks)
    if reach < 0 or sinks < 0:
        raise ValueError(f"window and sinks must be >= 0, got {window} and {sinks}")
    reach, sinks = min(reach, ALL_POSITIONS), min(sinks, ALL_POSITIONS)
    fast = _fast(q_nope)
    if fast is not None and q_nope.shape[0] > 0:
        ext, ws, stream = fast
        try:
            rc = ext.decode_window(q_nope, q_pe, ckv_cache, kpe_cache,
                                   -1 if page_size is None else max(0, int(page_size)), page_table,
                                   lengths, row_offsets, reach, sinks, float(sm_scale), output,
                                   lse, ws, stream)
        except TypeError:
            rc = -1  # an argument that is no tensor: named below
        if _done(rc, q_nope, what):
            return
    ckv, kpe, page = _common(q_nope, q_pe, ckv_cache, kpe_cache, output, lse, page_size)
    dev = q_nope.device
    table, lengths = _sequences(("page_table", "lengths"), page_table, lengths, dev)
    row_offsets = _rows(row_offsets, lengths.shape[0], q_nope.shape[0], dev)
    _attend(what, (), (reach, sinks), q_nope, q_pe, ckv, kpe, page, table, lengths, row_offsets,
            sm_scale, output, lse)


def kernel_shared(q_nope, q_pe, ckv_cache, kpe_cache, prefix_table, prefix_lengths, page_table,
                  lengths, sm_scale, output, lse, row_offsets=None, group_offsets=None,
                  page_size=None) -> None:
    """Attention of rows that share prefixes (writes ``output`` and ``lse``).

    ``prefix_table`` [groups, max_pages] int32 and ``prefix_lengths`` [groups] int32 name the
    prefixes, stored once.  Group g's rows are ``[group_offsets[g], group_offsets[g + 1])`` (int32
    [groups + 1], ascending; None: one group of all rows; rows outside have no prefix).
    ``page_table`` and ``lengths`` describe what follows the prefix, from position 0 of the row's
    own pages (a row of one token and length 0 sees the prefix alone).  A token sees its group's
    prefix and its row's own positions up to its own.  The prefix is read once for up to
    128 / heads tokens at a time.  Otherwise as :func:`kernel_window`.

    A call takes about 4 KB of scratch for each token and head from PyTorch's allocator (8,192
    tokens of 128 heads: 4.3 GB): split long prompts into chunks.
    """
    what = "dsa_mla_decode_shared"
    fast = _fast(q_nope)
    if fast is not None and q_nope.shape[0] > 0:
        ext, ws, stream = fast
        try:
            rc = ext.decode_shared(q_nope, q_pe, ckv_cache, kpe_cache,
                                   -1 if page_size is None else max(0, int(page_size)), prefix_table,
                                   prefix_lengths, group_offsets, page_table, lengths,
                                   row_offsets, float(sm_scale), output, lse, ws, stream)
        except TypeError:
            rc = -1
        if _done(rc, q_nope, what):
            return
    ckv, kpe, page = _common(q_nope, q_pe, ckv_cache, kpe_cache, output, lse, page_size)
    dev = q_nope.device
    table, lengths = _sequences(("page_table", "lengths"), page_table, lengths, dev)
    pre, pre_lengths = _sequences(("prefix_table", "prefix_lengths"), prefix_table, prefix_lengths, dev)
    row_offsets = _rows(row_offsets, lengths.shape[0], q_nope.shape[0], dev)
    groups = pre_lengths.shape[0]
    if groups < 1:
        raise ValueError("prefix_lengths must name at least one prefix")
    if group_offsets is None:
        if groups != 1:
            raise ValueError(f"{groups} prefixes need group_offsets")
    else:
        _need("group_offsets", group_offsets, torch.int32, 1, dev)
        if group_offsets.shape[0] != groups + 1:
            raise ValueError(f"group_offsets must be [{groups + 1}], got {tuple(group_offsets.shape)}")
        group_offsets = group_offsets.contiguous()
    prefix = (pre.data_ptr(), pre.stride(0), pre.shape[1], pre_lengths.data_ptr(),
              _ptr(group_offsets), groups)
    _attend(what, prefix, (), q_nope, q_pe, ckv, kpe, page, table, lengths, row_offsets, sm_scale,
            output, lse)


def merge_states(outputs, lses, output, lse) -> None:
    """Joins attention results over separate sets of positions (writes ``output`` and ``lse``).

    ``outputs``: 1 to 8 tensors [tokens, heads, 512] bfloat16, ``lses`` their base-2 log-sum-exps
    [tokens, heads] float32 (any head count).  The result is that of one softmax over all the
    positions: with M the largest lse and ``w_i = 2 ** (lse_i - M)``, ``output = sum w_i outputs_i /
    sum w_i`` (summed in fp32) and ``lse = M + log2(sum w_i)``.  A part of lse -inf is left out
    whatever its output holds; where all are, output is 0 and lse -inf.  ``output`` and ``lse`` may
    each be one of the parts themselves; another overlap with a part's output or lse is refused.
    """
    what = "dsa_merge_states"
    outputs, lses = list(outputs), list(lses)
    if not 1 <= len(outputs) <= MAX_PARTS or len(lses) != len(outputs):
        raise ValueError(f"merge_states takes 1 to {MAX_PARTS} parts, got {len(outputs)} outputs "
                         f"and {len(lses)} lses")
    ext = _native._ext if _native._ext_tried else _native.ext()
    if (ext is not None and type(output) is torch.Tensor and output.is_cuda
            and torch._C._cuda_getDevice() == output.get_device()):
        try:
            rc = ext.merge_states(outputs, lses, output, lse,
                                  torch._C._cuda_getCurrentRawStream(output.get_device()))
        except TypeError:
            rc = -1
        if rc == _native.DSA_OK:
            return
        if rc not in ops._REVALIDATE:
            _check(rc, what)
    _need("output", output, _BF16, 3)
    dev, shape = output.device, tuple(output.shape)
    if shape[2] != D_CKV:
        raise ValueError(f"output must be [num_tokens, num_heads, {D_CKV}], got {shape}")
    _need("lse", lse, torch.float32, 2, dev)
    if tuple(lse.shape) != shape[:2]:
        raise ValueError(f"lse must be {list(shape[:2])}, got {tuple(lse.shape)}")
    for i, (o, z) in enumerate(zip(outputs, lses)):
        _need(f"outputs[{i}]", o, _BF16, 3, dev)
        _need(f"lses[{i}]", z, torch.float32, 2, dev)
        if tuple(o.shape) != shape or tuple(z.shape) != shape[:2]:
            raise ValueError(f"part {i} must be {list(shape)} and {list(shape[:2])}, got "
                             f"{tuple(o.shape)} and {tuple(z.shape)}")
    if shape[0] == 0 or shape[1] == 0:
        return
    outs = [_unit(o) for o in outputs]
    out_t = output if output.stride(-1) == 1 else torch.empty_like(output, memory_format=torch.contiguous_format)
    n = len(outs)
    lib = _native._lib or _native.load()
    guard, stream = _launch_on(output)
    with guard:
        rc = lib.dsa_merge_states(
            n, (ctypes.c_void_p * n)(*(o.data_ptr() for o in outs)),
            (ctypes.c_int64 * (2 * n))(*(s for o in outs for s in o.stride()[:2])),
            (ctypes.c_void_p * n)(*(z.data_ptr() for z in lses)),
            (ctypes.c_int64 * (2 * n))(*(s for z in lses for s in z.stride())),
            out_t.data_ptr(), out_t.stride(0), out_t.stride(1),
            lse.data_ptr(), lse.stride(0), lse.stride(1), shape[0], shape[1], stream)
        if rc == 1:
            raise ValueError("output or lse overlaps a part without being that part")
        _check(rc, what)
        if out_t is not output:
            output.copy_(out_t)
