"""Timed cases of the dense attention operators of a bf16 latent cache, and their plain forms.

``listed()`` gives the cases, ``prepare`` a step's inputs on the GPU, ``run`` one pass through an
operator: with ``own`` false as elementary torch operations in 32 bits, otherwise through
flashinfer_mlsys2026_dsa_b200.  Three operators:

  window  attention over the last `window` positions of a sequence and its first `sinks`
  shared  attention of rows whose sequences begin with one prefix, stored once, over that prefix
          and the rows' own positions
  merge   attention results over separate sets of positions joined into that over all of them
"""
import math

import torch

own = False

D_CKV, D_KPE = 512, 64
SM_SCALE = 1.0 / math.sqrt(192.0)
LOG2E = math.log2(math.e)


# ------------------------------------------------------------------------------- the cases


def _window(name, rows, heads, min_len, max_len, window, sinks, max_new=1, page=64):
    return dict(name=name, op="window", rows=rows, heads=heads, min_len=min_len, max_len=max_len,
                window=window, sinks=sinks, max_new=max_new, page=page)


def _shared(name, rows, heads, min_prefix, max_prefix, min_own, max_own, groups=1, max_new=1,
            page=64):
    return dict(name=name, op="shared", rows=rows, heads=heads, min_prefix=min_prefix,
                max_prefix=max_prefix, min_own=min_own, max_own=max_own, groups=groups,
                max_new=max_new, page=page)


def _merge(name, tokens, heads, parts):
    return dict(name=name, op="merge", tokens=tokens, heads=heads, parts=parts)


def listed():
    return [
        # one user's chat: the smallest decode step, where latency is all
        _window("window_1x16", 1, 16, 1500, 1500, 512, 4),
        # a full decode batch over long sequences
        _window("window_b64_h16", 64, 16, 4096, 32768, 1024, 4),
        # a batch of an unsharded model (all 128 heads on the GPU), a wide window
        _window("window_b32_h128", 32, 128, 65536, 65536, 4096, 64),
        # drafted tokens checked in one step: 1 to 7 for each row, new and old sequences, odd sizes
        _window("window_draft_h64", 37, 64, 1, 5000, 333, 3, max_new=7, page=16),
        # chunks of four prompts
        _window("window_prompts", 4, 16, 1500, 9000, 1024, 4, max_new=1500),
        # two users of one short system prompt
        _shared("shared_2x16", 2, 16, 700, 700, 1, 50),
        # a decode batch behind one system prompt
        _shared("shared_b64_h16", 64, 16, 8192, 8192, 1, 1024),
        # all 128 heads behind a long document
        _shared("shared_b32_h128", 32, 128, 16384, 16384, 100, 3000),
        # requests of five tenants with a prompt each, up to 4 drafted tokens a row
        _shared("shared_5_tenants", 61, 32, 1000, 30000, 10, 2000, groups=5, max_new=4, page=16),
        # many questions about one long document: the largest
        _shared("shared_b256_h16", 256, 16, 32768, 32768, 128, 2048),
        # sparse and window attention of a decode batch joined
        _merge("merge_b64_h16", 64, 16, 2),
        # a prompt chunk's three parts
        _merge("merge_b2048_h16", 2048, 16, 3),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm where the range spans more than ten."""
    if hi > 10 * lo:
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return rng.randint(lo, hi)


def draw(rng):
    op = rng.choice(["window", "window", "shared", "shared", "merge"])
    heads = rng.choice([16, 16, 32, 64, 128])
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "merge":
        return dict(op=op, tokens=_spread(rng, 1, 32768 // heads), heads=heads,
                    parts=rng.randint(2, 4))
    if op == "window":
        new = rng.choice([1, 1, 1, _spread(rng, 2, 8), _spread(rng, 9, 1500 * 16 // heads)])
        rows = _spread(rng, 1, max(1, min(64, 6000 * 16 // heads // new)))
        longest = 65536 if rows <= 32 else 32768
        top = _spread(rng, max(1, new), longest)
        window = _spread(rng, 1, 4096 if new <= 8 else 1024)
        return dict(op=op, rows=rows, heads=heads, min_len=_spread(rng, 1, top), max_len=top,
                    window=window, sinks=rng.choice([0, 1, 4, _spread(rng, 5, 128)]), max_new=new,
                    page=page)
    rows = _spread(rng, 1, 256 * 16 // heads)
    new = rng.choice([1, 1, _spread(rng, 2, 8)]) if rows <= 64 * 16 // heads else 1
    top = _spread(rng, max(1, new), 2048)
    prefix = _spread(rng, 1, 32768)
    return dict(op=op, rows=rows, heads=heads, min_prefix=_spread(rng, 1, prefix),
                max_prefix=prefix, min_own=_spread(rng, 1, top), max_own=top,
                groups=min(rows, rng.choice([1, 1, _spread(rng, 2, 8)])), max_new=new, page=page)


def _lengths(n, lo, hi):
    """n lengths from lo to hi, evenly spaced (over their logarithm past a factor of ten)."""
    if n == 1 or lo == hi:
        return [hi] * n
    if hi > 10 * lo:
        return [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _new_tokens(c, lens):
    """Each row's new tokens: 1 to max_new in turn (all of max_new from 9 on: prompts)."""
    top = c["max_new"]
    return [min(n, top if top > 8 else 1 + (5 * r) % top) for r, n in enumerate(lens)]


def _group_sizes(rows, groups):
    """Rows of each group: larger and smaller ones, at least one row each."""
    free = rows - groups
    cuts = [free * g * g // (groups * groups) for g in range(groups + 1)]
    return [1 + cuts[g + 1] - cuts[g] for g in range(groups)]


# ------------------------------------------------------------------------------- the work


def _seen(length, new, window, sinks):
    """(keys read for a row, pairs of a token and a position that it sees)."""
    pairs = 0
    for p in range(length - new, length):
        recent = min(window, p + 1)
        pairs += recent + min(sinks, p + 1 - recent)
    first = max(0, length - new - window + 1)  # the first position in any token's window
    return length - first + min(sinks, first), pairs


def work(case):
    c = case
    if c["op"] == "merge":
        rh = c["tokens"] * c["heads"]
        return {"bytes": rh * (c["parts"] + 1) * (2 * D_CKV + 4),
                "flops": rh * c["parts"] * 2 * D_CKV}
    key = 2 * (D_CKV + D_KPE)
    keys = pairs = tokens = 0
    if c["op"] == "window":
        lens = _lengths(c["rows"], c["min_len"], c["max_len"])
        for n, m in zip(lens, _new_tokens(c, lens)):
            k, p = _seen(n, m, c["window"], c["sinks"])
            keys, pairs, tokens = keys + k, pairs + p, tokens + m
    else:
        lens = _lengths(c["rows"], c["min_own"], c["max_own"])
        new = _new_tokens(c, lens)
        for n, m in zip(lens, new):
            k, p = _seen(n, m, n, 0)
            keys, pairs, tokens = keys + k, pairs + p, tokens + m
        row = 0
        for size, n in zip(_group_sizes(c["rows"], c["groups"]),
                           _lengths(c["groups"], c["min_prefix"], c["max_prefix"])):
            keys, pairs = keys + n, pairs + n * sum(new[row:row + size])
            row += size
    return {"bytes": keys * key + tokens * c["heads"] * (key + 2 * D_CKV + 4),
            "flops": 2 * c["heads"] * pairs * (2 * D_CKV + D_KPE)}


# ------------------------------------------------------------------------------ the inputs


def _pools(pages, page, g):
    """The latent and rope key pools: rows of varying size, as a model's tokens have them."""
    ckv = torch.empty(pages, page, D_CKV, dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 27) // (page * D_CKV))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        size = torch.exp(torch.randn(n, page, 1, generator=g, device="cuda") * 0.5 - 0.7)
        x = torch.randn(n, page, D_CKV, generator=g, device="cuda", dtype=torch.bfloat16)
        ckv[a:a + n] = x * size.to(torch.bfloat16)
    kpe = torch.randn(pages, page, D_KPE, generator=g, device="cuda", dtype=torch.bfloat16)
    return ckv, kpe.mul_(0.5)


def _tables(lens, page, order):
    """A page table of the sequences, from the pages in `order`; -1 past a sequence's pages."""
    counts = torch.tensor([-(-n // page) for n in lens], device="cuda")
    j = torch.arange(max(1, int(counts.max())), device="cuda")
    at = (counts.cumsum(0) - counts)[:, None] + j
    table = torch.where(j < counts[:, None], order[at.clamp(max=len(order) - 1)], -1)
    return table.to(torch.int32).contiguous(), int(counts.sum())


def _int32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _offsets(counts):
    return torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()


def _shuffled(values, seed):
    p = torch.randperm(len(values), generator=torch.Generator().manual_seed(seed)).tolist()
    return [values[i] for i in p]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "merge":
        shape = (c["tokens"], c["heads"])
        # parts of unequal weight; a token in sixteen has nothing in its last part
        outs = [torch.randn(*shape, D_CKV, generator=g, device="cuda", dtype=torch.bfloat16)
                for _ in range(c["parts"])]
        lses = [torch.randn(*shape, generator=g, device="cuda") * 3 + 10 for _ in range(c["parts"])]
        gone = torch.rand(c["tokens"], generator=g, device="cuda") < 1 / 16
        outs[-1][gone] = 0
        lses[-1][gone] = -math.inf
        return dict(case=c, outputs=outs, lses=lses, output=torch.empty_like(outs[0]),
                    lse=torch.empty_like(lses[0]))
    s = dict(case=c)
    if c["op"] == "window":
        lens = _lengths(c["rows"], c["min_len"], c["max_len"])
    else:
        lens = _lengths(c["rows"], c["min_own"], c["max_own"])
    both = list(zip(lens, _new_tokens(c, lens)))
    if c["op"] == "window":
        both = _shuffled(both, seed)
    s["lens"], s["new"] = [n for n, _ in both], [m for _, m in both]
    prefix = []
    if c["op"] == "shared":
        prefix = _lengths(c["groups"], c["min_prefix"], c["max_prefix"])
        s["sizes"], s["prefix"] = _group_sizes(c["rows"], c["groups"]), prefix
        s["prefix_lengths"] = _int32(prefix)
        s["group_offsets"] = _offsets(s["sizes"]) if c["groups"] > 1 else None
    page = c["page"]
    pages = sum(-(-n // page) for n in s["lens"] + prefix)
    order = torch.randperm(pages, generator=g, device="cuda")
    s["page_table"], used = _tables(s["lens"], page, order)
    if prefix:
        s["prefix_table"], _ = _tables(prefix, page, order[used:])
    s["lengths"] = _int32(s["lens"])
    s["ckv"], s["kpe"] = _pools(pages, page, g)
    s["row_offsets"] = _offsets(s["new"]) if c["max_new"] > 1 else None
    shape = (sum(s["new"]), c["heads"])
    s["q_nope"] = torch.randn(*shape, D_CKV, generator=g, device="cuda", dtype=torch.bfloat16)
    s["q_pe"] = torch.randn(*shape, D_KPE, generator=g, device="cuda", dtype=torch.bfloat16)
    s["output"] = torch.empty(*shape, D_CKV, dtype=torch.bfloat16, device="cuda")
    s["lse"] = torch.empty(*shape, dtype=torch.float32, device="cuda")
    return s


# ------------------------------------------------------------------------- the plain forms


def _keys(s, table, at):
    """[rows, n, 576] keys (float) at the positions `at` [rows, n] of the sequences of `table`."""
    page = s["case"]["page"]
    slot = table.long().gather(1, at // page).clamp(min=0) * page + at % page
    return torch.cat([s["ckv"].view(-1, D_CKV)[slot], s["kpe"].view(-1, D_KPE)[slot]], 2).float()


def _queries(s):
    """[rows, most new tokens, heads, 576] scaled queries (float), zeros behind a row's tokens, their
    positions [rows, most new tokens] and where each row's token stands in the packed inputs."""
    new, lens = _int64(s["new"]), s["lengths"].long()
    j = torch.arange(max(s["new"]), device="cuda")
    first = new.cumsum(0) - new
    live = j < new[:, None]
    at = torch.where(live, first[:, None] + j, 0)
    q = torch.cat([s["q_nope"][at], s["q_pe"][at]], 3).float() * (SM_SCALE * LOG2E)
    return q, (lens - new)[:, None] + j, live


def _int64(values):
    return torch.tensor(values, device="cuda")


def _part(q, k, seen):
    """Scores of q [b, m, 576] against k [b, n, 576] where `seen`: their maximum, the sum of the
    probabilities' numerators and the values weighted by them."""
    z = torch.matmul(q, k.transpose(1, 2))
    z.masked_fill_(~seen, -math.inf)
    m = z.amax(2, keepdim=True).clamp(min=-3e38)
    p = torch.exp2(z.sub_(m))
    return m, p.sum(2, keepdim=True), torch.matmul(p, k[..., :D_CKV])


def _run_window(s):
    c = s["case"]
    q, pos, live = _queries(s)
    rows, new, heads, width = q.shape
    lens = s["lengths"].long()
    # the positions that any token of the row may see: sinks, then from the first window's begin
    first = (lens - _int64(s["new"]) - c["window"] + 1).clamp(min=0)
    span = min(c["window"] + new - 1, max(s["lens"]))
    recent = first[:, None] + torch.arange(span, device="cuda")
    sink = torch.arange(c["sinks"], device="cuda").expand(rows, -1)
    at = torch.cat([sink, recent], 1)
    fresh = torch.cat([sink < first[:, None], recent < lens[:, None]], 1)  # each position once
    k = _keys(s, s["page_table"], torch.where(fresh, at, 0))
    seen = (fresh[:, None] & (at[:, None] <= pos[..., None])
            & ((at[:, None] > pos[..., None] - c["window"]) | (at[:, None] < c["sinks"])))
    seen = seen[:, :, None].expand(-1, -1, heads, -1).reshape(rows, new * heads, -1)
    m, total, o = _part(q.view(rows, new * heads, width), k, seen)
    o = (o / total.clamp(min=1e-30)).view(rows, new, heads, D_CKV)
    s["output"].copy_(o[live])
    s["lse"].copy_((m + torch.log2(total)).view(rows, new, heads)[live])


def _run_shared(s):
    c = s["case"]
    q, pos, live = _queries(s)
    rows, new, heads, width = q.shape
    at = torch.arange(max(s["lens"]), device="cuda").expand(rows, -1)
    fresh = at < s["lengths"].long()[:, None]
    k = _keys(s, s["page_table"], torch.where(fresh, at, 0))
    seen = (at[:, None] <= pos[..., None])[:, :, None].expand(-1, -1, heads, -1)
    m1, l1, o1 = _part(q.view(rows, new * heads, width), k, seen.reshape(rows, new * heads, -1))
    # the prefix: each group's rows (padded to the largest group) against its keys
    groups, most = c["groups"], max(s["sizes"])
    size = _int64(s["sizes"])
    j = torch.arange(most, device="cuda")
    member = j < size[:, None]
    row = torch.where(member, (size.cumsum(0) - size)[:, None] + j, 0)
    at = torch.arange(max(s["prefix"]), device="cuda").expand(groups, -1)
    fresh = at < s["prefix_lengths"].long()[:, None]
    k = _keys(s, s["prefix_table"], torch.where(fresh, at, 0))
    part = _part(q[row].view(groups, most * new * heads, width), k, fresh[:, None])
    m2, l2, o2 = (x.view(groups, most, new * heads, -1)[member] for x in part)
    m = torch.maximum(m1, m2)
    w1, w2 = torch.exp2(m1 - m), torch.exp2(m2 - m)
    total = w1 * l1 + w2 * l2
    o = ((w1 * o1 + w2 * o2) / total).view(rows, new, heads, D_CKV)
    s["output"].copy_(o[live])
    s["lse"].copy_((m + torch.log2(total)).view(rows, new, heads)[live])


def _run_merge(s):
    lse = torch.stack(s["lses"])
    m = lse.amax(0).clamp(min=-3e38)
    w = torch.exp2(lse - m)
    total = w.sum(0)
    o = sum(x.float() * y[..., None] for x, y in zip(s["outputs"], w))
    s["output"].copy_(o / total.clamp(min=1e-30)[..., None])
    s["lse"].copy_(m + torch.log2(total))


def run(state):
    s = state
    c = s["case"]
    if not own:
        {"window": _run_window, "shared": _run_shared, "merge": _run_merge}[c["op"]](s)
        return {"output": s["output"], "lse": s["lse"]}
    import flashinfer_mlsys2026_dsa_b200 as dsa

    if c["op"] == "window":
        dsa.kernel_window(s["q_nope"], s["q_pe"], s["ckv"], s["kpe"], s["page_table"],
                          s["lengths"], SM_SCALE, s["output"], s["lse"], c["window"], c["sinks"],
                          row_offsets=s["row_offsets"])
    elif c["op"] == "shared":
        dsa.kernel_shared(s["q_nope"], s["q_pe"], s["ckv"], s["kpe"], s["prefix_table"],
                          s["prefix_lengths"], s["page_table"], s["lengths"], SM_SCALE,
                          s["output"], s["lse"], row_offsets=s["row_offsets"],
                          group_offsets=s["group_offsets"])
    else:
        dsa.merge_states(s["outputs"], s["lses"], s["output"], s["lse"])
    return {"output": s["output"], "lse": s["lse"]}


# ---------------------------------------------------------------------- the definition, 64 bits


def _sequence(s, table_row, n):
    """The first n positions' keys [n, 576] of one sequence, in 64 bits."""
    page = s["case"]["page"]
    pages = table_row[:-(-n // page)].tolist()
    if not pages:
        return torch.empty(0, D_CKV + D_KPE, dtype=torch.float64, device="cuda")
    ckv, kpe = (torch.cat([pool[i] for i in pages])[:n] for pool in (s["ckv"], s["kpe"]))
    return torch.cat([ckv, kpe], 1).double()


def _softmax_rows(x, values):
    """softmax over the last axis of natural scores x [..., n] times values, and log2 of its sum."""
    lse = torch.logsumexp(x, -1)
    return torch.exp(x - lse[..., None]) @ values, lse * LOG2E


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "merge":
        weight = torch.stack([x.double() * math.log(2.0) for x in s["lses"]], -1)  # [t, h, parts]
        share = torch.softmax(weight, -1)
        o = torch.zeros(s["output"].shape, dtype=torch.float64, device="cuda")
        for i, x in enumerate(s["outputs"]):
            o += x.double() * share[..., i:i + 1]
        return {"output": o, "lse": torch.logsumexp(weight, -1) * LOG2E}
    out = torch.empty(s["output"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["lse"].shape, dtype=torch.float64, device="cuda")
    owner = [g for g, n in enumerate(s.get("sizes", [])) for _ in range(n)]
    prefixes = [_sequence(s, s["prefix_table"][g], n) for g, n in enumerate(s.get("prefix", []))]
    token = 0
    for r, (n, m) in enumerate(zip(s["lens"], s["new"])):
        keys = _sequence(s, s["page_table"][r], n)
        before = len(prefixes[owner[r]]) if prefixes else 0
        if before:
            keys = torch.cat([prefixes[owner[r]], keys])
        place = torch.arange(len(keys), device="cuda") - before  # below 0: the prefix
        for a in range(0, m, 64):
            b = min(m, a + 64)
            mine = torch.arange(n - m + a, n - m + b, device="cuda")[:, None]
            allowed = place <= mine
            if c["op"] == "window":
                allowed &= (place < c["sinks"]) | (mine - place < c["window"])
            some = allowed.any(0)
            q = torch.cat([s["q_nope"][token + a:token + b], s["q_pe"][token + a:token + b]], 2)
            x = q.double() @ keys[some].T * SM_SCALE
            x = x.masked_fill(~allowed[:, None, some], -math.inf)
            o, z = _softmax_rows(x, keys[some][:, :D_CKV])
            out[token + a:token + b], lse[token + a:token + b] = o, z
        token += m
    return {"output": out, "lse": lse}
