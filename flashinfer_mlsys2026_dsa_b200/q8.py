"""The 8-bit latent cache: its append, the decode that reads it, and its eviction.

A cache is three pools: ``ckv_q8`` [pages, page, 512] float8_e4m3fn, ``ckv_scale``
[pages, page // block] float32 and ``kpe_cache`` [pages, page, 64] bfloat16.  Every ``block``
consecutive tokens of a page share one scale (``block`` is the page size divided by
``ckv_scale``'s second dimension, a power of two up to 256); the latent value of a token is
``ckv_q8.float() * ckv_scale``.  The rope keys stay bfloat16.

A serving loop appends each step's tokens (:func:`append_q8`), decodes over the selected slots
or positions (:func:`kernel_q8`, :func:`kernel_q8_paged`, the forms of :func:`ops.kernel` and
:func:`ops.kernel_paged`), adds the attention weights of the step to running totals
(:func:`accumulate_weights`), and, when a sequence outgrows its budget, keeps its heaviest
positions (:func:`evict_positions`) and moves them to new pages (:func:`compact_q8`).

All calls launch on the current CUDA stream and do not synchronise; there is no CPU path.
"""
from __future__ import annotations

import contextlib

import torch

from . import _native, ops
from .ops import D_CKV, D_KPE, SUPPORTED_HEADS, _REVALIDATE, _check, _slot_view, _workspaces

MAX_BLOCK = 256
_E4M3 = torch.float8_e4m3fn
_BF16 = torch.bfloat16


def _need(name, t, dtype, dim, dev=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")
    if dev is not None and t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {str(dtype)[6:]}, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, got {tuple(t.shape)}")


def _cache(ckv_q8, ckv_scale, kpe_cache, dev=None):
    """Checks the three pools; returns the arguments the C ABI takes for them, and the page size."""
    _need("ckv_q8", ckv_q8, _E4M3, 3, dev)
    dev = ckv_q8.device
    _need("ckv_scale", ckv_scale, torch.float32, 2, dev)
    _need("kpe_cache", kpe_cache, _BF16, 3, dev)
    pages, page, width = ckv_q8.shape
    if width != D_CKV or tuple(kpe_cache.shape) != (pages, page, D_KPE):
        raise ValueError(f"ckv_q8 / kpe_cache must be [pages, page, {D_CKV}] / [pages, page, {D_KPE}], "
                         f"got {tuple(ckv_q8.shape)} / {tuple(kpe_cache.shape)}")
    blocks = ckv_scale.shape[1]
    if ckv_scale.shape[0] != pages or blocks < 1 or page % blocks:
        raise ValueError(f"ckv_scale must be [{pages}, page // block], got {tuple(ckv_scale.shape)}")
    block = page // blocks
    if block & (block - 1) or block > MAX_BLOCK:
        raise ValueError(f"a scale must cover a power of two of tokens, at most {MAX_BLOCK}, got {block}")
    if not ckv_scale.is_contiguous():
        raise ValueError("ckv_scale must be contiguous")
    ckv = _slot_view(ckv_q8, D_CKV, "ckv_q8")
    kpe = _slot_view(kpe_cache, D_KPE, "kpe_cache")
    return (ckv.data_ptr(), ckv.stride(0), ckv_scale.data_ptr(), block, kpe.data_ptr(),
            kpe.stride(0), ckv.shape[0]), page


def _table(name, t, rows, page, dev):
    _need(name, t, torch.int32, 2, dev)
    if t.shape[0] != rows or t.shape[1] < 1:
        raise ValueError(f"{name} must be [{rows}, max_pages], got {tuple(t.shape)}")
    if page & (page - 1):
        raise ValueError(f"the page size must be a power of two, got {page}")
    return t if t.stride(1) == 1 else t.contiguous()


def _unit(t):
    """t with a unit inner stride (a copy where it has none)."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _rows_meet(a, b):
    """Whether the rows of two 2-D tensors of one type share memory (columns beside each other do not)."""
    size = a.element_size()
    i = j = 0
    while i < a.shape[0] and j < b.shape[0] and a.shape[1] and b.shape[1]:
        at, bt = a.data_ptr() + i * a.stride(0) * size, b.data_ptr() + j * b.stride(0) * size
        ae, be = at + a.shape[1] * size, bt + b.shape[1] * size
        if at < be and bt < ae:
            return True
        if ae <= bt:
            i += 1
        else:
            j += 1
    return False


def _row_offsets(t, rows, dev):
    _need("row_offsets", t, torch.int32, 1, dev)
    if t.shape[0] != rows + 1:
        raise ValueError(f"row_offsets must be [{rows + 1}], got {tuple(t.shape)}")
    return t.contiguous()


def _launch_on(t):
    """The raw current stream of t's device, that device made current while it is used."""
    dev = t.get_device()
    here = torch._C._cuda_getDevice()
    guard = contextlib.nullcontext() if here == dev else torch.cuda.device(dev)
    return guard, torch._C._cuda_getCurrentRawStream(dev)


def _fast(t):
    """(binding, workspace, stream) for the direct route of a call on t's device, or None."""
    ext = _native._ext if _native._ext_tried else _native.ext()
    if ext is None or type(t) is not torch.Tensor or not t.is_cuda:
        return None
    dev = t.get_device()
    if torch._C._cuda_getDevice() != dev:
        return None
    stream = torch._C._cuda_getCurrentRawStream(dev)
    ws = _workspaces.get((dev, stream))
    return None if ws is None else (ext, ws, stream)


def _done(rc, t, what) -> bool:
    """Whether the direct route ran the call; raises what it could not."""
    if rc == _native.DSA_OK:
        if ops._strict:
            ops._strict_check(t.device, what)
        return True
    if rc not in _REVALIDATE:
        _check(rc, what)
    return False


def _finish(rc, t, what) -> None:
    _check(rc, what)
    if ops._strict:
        ops._strict_check(t.device, what)


def _attend(q_nope, q_pe, ckv_q8, ckv_scale, kpe_cache, page_table, indices, index_name, sm_scale,
            output, lse, weights):
    what = "dsa_sparse_mla_decode_q8"
    fast = _fast(q_nope)
    if fast is not None and q_nope.shape[0] > 0:
        ext, ws, stream = fast
        try:
            rc = ext.decode_q8(q_nope, q_pe, ckv_q8, ckv_scale, kpe_cache, page_table, indices,
                               float(sm_scale), output, lse, weights, ws, stream)
        except TypeError:
            rc = -1  # an argument that is no tensor: named below
        if _done(rc, q_nope, what):
            return
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
    cache, page = _cache(ckv_q8, ckv_scale, kpe_cache, dev)
    _need(index_name, indices, torch.int32, 2, dev)
    topk = indices.shape[1]
    if indices.shape[0] != B or topk < 1:
        raise ValueError(f"{index_name} must be [{B}, topk >= 1], got {tuple(indices.shape)}")
    table = (None, 0, 0)
    if page_table is not None:
        page_table = _table("page_table", page_table, B, page, dev)
        table = (page_table.data_ptr(), page_table.stride(0), page_table.shape[1])
    if weights is not None:
        _need("weights", weights, torch.float32, 2, dev)
        if tuple(weights.shape) != (B, topk):
            raise ValueError(f"weights must be [{B}, {topk}], got {tuple(weights.shape)}")
    if B == 0:
        return
    q_nope, q_pe, indices = _unit(q_nope), _unit(q_pe), _unit(indices)
    out_t = output if output.stride(-1) == 1 else torch.empty_like(output, memory_format=torch.contiguous_format)
    w_t = weights if weights is None or weights.stride(1) == 1 else torch.empty_like(weights, memory_format=torch.contiguous_format)
    lib = _native._lib or _native.load()
    guard, stream = _launch_on(q_nope)
    with guard:
        ws = ops.workspace_for(dev, stream, B, H, topk)
        scratch = None
        if w_t is not None:
            scratch = torch.empty(lib.dsa_q8_scratch_size(B, H, topk), dtype=torch.uint8, device=dev)
        rc = lib.dsa_sparse_mla_decode_q8(
            q_nope.data_ptr(), q_nope.stride(0), q_nope.stride(1),
            q_pe.data_ptr(), q_pe.stride(0), q_pe.stride(1), *cache, *table, page,
            indices.data_ptr(), indices.stride(0), float(sm_scale),
            out_t.data_ptr(), out_t.stride(0), out_t.stride(1),
            lse.data_ptr(), lse.stride(0), lse.stride(1),
            *((None, 0) if w_t is None else (w_t.data_ptr(), w_t.stride(0))), B, H, topk,
            *((None, 0) if scratch is None else (scratch.data_ptr(), scratch.numel())),
            ws.data_ptr(), stream)
        _check(rc, what)
        if out_t is not output:
            output.copy_(out_t)
        if w_t is not weights:
            weights.copy_(w_t)
        _finish(rc, q_nope, what)


def kernel_q8(q_nope, q_pe, ckv_q8, ckv_scale, kpe_cache, sparse_indices, sm_scale, output, lse,
              weights=None) -> None:
    """:func:`ops.kernel` over the 8-bit cache (writes ``output``, ``lse`` and ``weights``).

    ``weights`` (optional) [B, topk] float32 receives each entry's attention probability summed
    over the heads, 0 for padding: what :func:`accumulate_weights` adds up.  Head counts,
    strides, padding and error bits are those of :func:`ops.kernel`.  The scales of a selection
    may differ, up to 2^88-fold without any loss (beyond, a value may be off by 2^-106 of the
    largest scale).
    """
    _attend(q_nope, q_pe, ckv_q8, ckv_scale, kpe_cache, None, sparse_indices, "sparse_indices",
            sm_scale, output, lse, weights)


def kernel_q8_paged(q_nope, q_pe, ckv_q8, ckv_scale, kpe_cache, page_table, positions, sm_scale,
                    output, lse, weights=None) -> None:
    """:func:`kernel_q8` with the slots formed from token positions, as :func:`ops.kernel_paged`.

    ``positions`` [B, topk] int32 (-1 = padding), ``page_table`` [B, max_pages] int32; the page
    size is the pools'.
    """
    if page_table is None:
        raise TypeError("page_table must be a torch.Tensor")
    _attend(q_nope, q_pe, ckv_q8, ckv_scale, kpe_cache, page_table, positions, "positions",
            sm_scale, output, lse, weights)


def append_q8(ckv, kpe, row_offsets, starts, page_table, ckv_q8, ckv_scale, kpe_cache) -> None:
    """Writes new tokens into the 8-bit cache.

    ``ckv`` [tokens, 512] and ``kpe`` [tokens, 64] bfloat16.  Row r's new tokens are
    ``[row_offsets[r], row_offsets[r + 1])`` (int32 [rows + 1], ascending; tokens outside are
    not read, so a batch may be padded) and take the positions ``starts[r], starts[r] + 1, ...``
    (int32 [rows]) of the sequence whose pages are ``page_table[r]`` (int32).

    The scale of a block becomes the smallest power of two that holds its new tokens within
    +-448, unless the block has earlier tokens (positions before ``starts[r]``) with a larger
    one; when it grows, the earlier tokens are re-expressed in it.  Infinities are stored as
    NaN and take no part in the scale.  A position without a page is skipped and flagged in
    :func:`ops.read_device_errors`.  Rows must not share the blocks they write.
    """
    what = "dsa_append_q8"
    fast = _fast(ckv_q8)
    if fast is not None:
        ext, ws, stream = fast
        try:
            rc = ext.append_q8(ckv, kpe, row_offsets, starts, page_table, ckv_q8, ckv_scale,
                               kpe_cache, ws, stream)
        except TypeError:
            rc = -1
        if _done(rc, ckv_q8, what):
            return
    cache, page = _cache(ckv_q8, ckv_scale, kpe_cache)
    dev = ckv_q8.device
    _need("ckv", ckv, _BF16, 2, dev)
    _need("kpe", kpe, _BF16, 2, dev)
    tokens = ckv.shape[0]
    if ckv.shape[1] != D_CKV or tuple(kpe.shape) != (tokens, D_KPE):
        raise ValueError(f"ckv / kpe must be [tokens, {D_CKV}] / [tokens, {D_KPE}], "
                         f"got {tuple(ckv.shape)} / {tuple(kpe.shape)}")
    _need("starts", starts, torch.int32, 1, dev)
    rows = starts.shape[0]
    row_offsets = _row_offsets(row_offsets, rows, dev)
    page_table = _table("page_table", page_table, rows, page, dev)
    if tokens == 0 or rows == 0:
        return
    ckv, kpe, starts = _unit(ckv), _unit(kpe), starts.contiguous()
    lib = _native._lib or _native.load()
    guard, stream = _launch_on(ckv_q8)
    with guard:
        ws = ops.workspace_for(dev, stream, 1, 16, 1)
        rc = lib.dsa_append_q8(
            ckv.data_ptr(), ckv.stride(0), kpe.data_ptr(), kpe.stride(0), tokens,
            row_offsets.data_ptr(), starts.data_ptr(), rows, page_table.data_ptr(),
            page_table.stride(0), page_table.shape[1], page, *cache, ws.data_ptr(), stream)
        _finish(rc, ckv_q8, what)


def accumulate_weights(weights, positions, acc, row_offsets=None) -> None:
    """Adds a step's attention weights to running totals: ``acc[r, positions[t, k]] += weights[t, k]``.

    ``weights`` [tokens, topk] float32 (from :func:`kernel_q8`), ``positions`` [tokens, topk]
    int32 (-1 entries are left out), ``acc`` [rows, max_len] float32.  ``row_offsets`` (int32
    [rows + 1], ascending) gives each row's tokens; None: one token per row.  The sums have the
    same bits in every run as long as no token names a position twice (then both count, in no
    fixed order).  A row's tokens are added one after another (about 0.4 us each): meant for a
    step's few.  A position outside ``acc`` is skipped and flagged.
    """
    what = "dsa_accumulate_weights"
    fast = _fast(acc)
    if fast is not None:
        ext, ws, stream = fast
        try:
            rc = ext.accumulate_weights(weights, positions, acc, row_offsets, ws, stream)
        except TypeError:
            rc = -1
        if _done(rc, acc, what):
            return
    _need("acc", acc, torch.float32, 2)
    dev = acc.device
    _need("weights", weights, torch.float32, 2, dev)
    _need("positions", positions, torch.int32, 2, dev)
    if positions.shape != weights.shape:
        raise ValueError(f"positions must be {list(weights.shape)}, got {tuple(positions.shape)}")
    tokens, topk = weights.shape
    rows, cols = acc.shape
    if cols >= 2 ** 31:
        raise ValueError(f"acc must have less than 2**31 columns, got {cols}")
    if acc.stride(1) != 1 or (rows > 1 and acc.stride(0) < cols):
        raise ValueError(f"acc must have a unit inner stride and rows apart, got strides {acc.stride()}")
    if row_offsets is not None:
        row_offsets = _row_offsets(row_offsets, rows, dev)
    elif rows != tokens:
        raise ValueError(f"acc must have {tokens} rows (one per token), got {rows}")
    if tokens == 0 or rows == 0 or topk == 0:
        return
    weights, positions = _unit(weights), _unit(positions)
    lib = _native._lib or _native.load()
    guard, stream = _launch_on(acc)
    with guard:
        ws = ops.workspace_for(dev, stream, 1, 16, 1)
        rc = lib.dsa_accumulate_weights(
            weights.data_ptr(), weights.stride(0), positions.data_ptr(),
            positions.stride(0), tokens, topk, acc.data_ptr(), acc.stride(0), cols, rows,
            None if row_offsets is None else row_offsets.data_ptr(), ws.data_ptr(), stream)
        _finish(rc, acc, what)


def evict_positions(acc, lengths, budget, sinks=0, recent=0, new_acc=None):
    """Which positions of each row an eviction keeps: ``(keep, new_lengths)``.

    ``acc`` [rows, max_len] float32 totals (:func:`accumulate_weights`), ``lengths`` [rows]
    int32.  A row longer than ``budget`` keeps its first ``sinks`` and last ``recent`` positions
    and those with the largest totals (ties to the smaller positions), ``budget`` in all; a
    shorter row keeps every position.  ``keep`` [rows, budget] int32 lists them ascending, -1
    after the last; ``new_lengths`` [rows] int32 counts them.  ``new_acc`` (optional, [rows, at
    least budget] float32, not overlapping ``acc``) receives their totals, then zeros.
    """
    _need("acc", acc, torch.float32, 2)
    dev = acc.device
    rows, max_len = acc.shape
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if not 1 <= budget < 2 ** 31 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"budget must be >= 1 and hold sinks + recent, got {budget}, {sinks}, {recent}")
    if max_len >= 2 ** 31:
        raise ValueError(f"acc must have less than 2**31 columns, got {max_len}")
    keep = torch.empty(rows, budget, dtype=torch.int32, device=dev)
    new_lengths = torch.empty(rows, dtype=torch.int32, device=dev)
    if rows == 0:
        return keep, new_lengths
    what = "dsa_evict_positions"
    guard, stream = _launch_on(acc)
    ext = _native._ext if _native._ext_tried else _native.ext()
    if ext is not None and type(guard) is contextlib.nullcontext:
        try:
            rc = ext.evict_positions(acc, lengths, budget, sinks, recent, keep, new_lengths,
                                     new_acc, stream)
        except TypeError:
            rc = -1
        if rc == _native.DSA_OK:
            return keep, new_lengths
        if rc not in _REVALIDATE:
            _check(rc, what)
    _need("lengths", lengths, torch.int32, 1, dev)
    if lengths.shape[0] != rows:
        raise ValueError(f"lengths must be [{rows}], got {tuple(lengths.shape)}")
    acc, lengths = _unit(acc), lengths.contiguous()
    out = (None, 0, 0)
    if new_acc is not None:
        _need("new_acc", new_acc, torch.float32, 2, dev)
        if new_acc.shape[0] != rows or new_acc.shape[1] < budget or new_acc.stride(1) != 1:
            raise ValueError(f"new_acc must be [{rows}, >= {budget}] with a unit inner stride, "
                             f"got {tuple(new_acc.shape)}, strides {new_acc.stride()}")
        if _rows_meet(new_acc, acc):
            raise ValueError("new_acc must not overlap acc")
        out = (new_acc.data_ptr(), new_acc.stride(0), new_acc.shape[1])
    lib = _native._lib or _native.load()
    with guard:
        _check(lib.dsa_evict_positions(acc.data_ptr(), acc.stride(0),
                                       lengths.data_ptr(), rows, max_len, budget, sinks, recent,
                                       keep.data_ptr(), budget, new_lengths.data_ptr(), *out,
                                       stream), what)
    return keep, new_lengths


def compact_q8(keep, page_table, new_page_table, ckv_q8, ckv_scale, kpe_cache) -> None:
    """Moves kept tokens of the 8-bit cache to new pages.

    Position ``keep[r, j]`` of row r (``page_table[r]``) becomes position j of
    ``new_page_table[r]``; -1 entries are left out.  A new block takes the largest scale among
    the tokens that move into it.  The new pages must be distinct and none of those that are
    read (so a prefix that other sequences share stays theirs); the old pages can be freed
    afterwards.  A position without a page is skipped and flagged.
    """
    what = "dsa_compact_q8"
    fast = _fast(ckv_q8)
    if fast is not None:
        ext, ws, stream = fast
        try:
            rc = ext.compact_q8(keep, page_table, new_page_table, ckv_q8, ckv_scale, kpe_cache, ws,
                                stream)
        except TypeError:
            rc = -1
        if _done(rc, ckv_q8, what):
            return
    cache, page = _cache(ckv_q8, ckv_scale, kpe_cache)
    dev = ckv_q8.device
    _need("keep", keep, torch.int32, 2, dev)
    rows, cols = keep.shape
    page_table = _table("page_table", page_table, rows, page, dev)
    new_page_table = _table("new_page_table", new_page_table, rows, page, dev)
    if rows == 0 or cols == 0:
        return
    keep = _unit(keep)
    lib = _native._lib or _native.load()
    guard, stream = _launch_on(ckv_q8)
    with guard:
        ws = ops.workspace_for(dev, stream, 1, 16, 1)
        rc = lib.dsa_compact_q8(
            keep.data_ptr(), keep.stride(0), rows, cols,
            page_table.data_ptr(), page_table.stride(0), page_table.shape[1],
            new_page_table.data_ptr(), new_page_table.stride(0),
            new_page_table.shape[1], page, *cache, ws.data_ptr(), stream)
        _finish(rc, ckv_q8, what)
