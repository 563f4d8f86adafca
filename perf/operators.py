"""The operators of the 4-bit paged KV cache as cases that can be timed and compared.

    append    rows of K and V are quantized into the pages of a cache and read back
    attend    attention of a packed batch of query rows over such a cache
    beams     a batch forks onto its parents, then every sequence makes room for more tokens (shared last pages are copied)
    compact   the used pages of a pool move to its front

``run`` computes a case in elementary torch operations, or, where ``own`` is true, with ``ctransformers_amd.ops``.

Layout of a cache (both sides): ``pages`` is uint8 [n_pages, page_bytes]; a page is [kv head][page_tokens / 32] blocks, a block holds 32 tokens of
one head as [K codes | V codes | K scales | V scales].  A head's dims fall into groups of 32 (`groups_of`; dims past the head's are zeros), a value is
f16(d) * (code - 8) with d = (the value of largest magnitude) / -8.
    K dword (token t, dim c): (4 t + (c mod 32) / 8) * G + c / 32, element c mod 8
    V dword (token t, dim c): ((t mod 16) / 4) * 32 G + c, element t mod 4 + 4 (t / 16)
    element e of a dword is its nibble e / 2 + 4 (e mod 2)
    K scales [t / 16][(t mod 16) / 4][group][t mod 4], V scales [(t mod 16) / 4][group][element of t]
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one generated token for each of 64 conversations, heads of Llama-2-70B
        {"name": "append_step", "op": "append", "seqs": 64, "new": 1, "past": 4096, "heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # prompts of different lengths behind different pasts, heads of 112 (MPT-30B), float32 rows
        {"name": "append_ragged", "op": "append", "seqs": 16, "new": 1500, "past": 700, "heads": 64, "dim": 112, "page": 32, "dtype": "f32"},
        # a single conversation's token step near the start of its context, heads of Llama-2-7B: latency is all there is
        {"name": "decode_one", "op": "attend", "seqs": 1, "new": 1, "past": 140, "heads": 32, "kv": 32, "dim": 128, "page": 64, "dtype": "f16"},
        # one long document, heads of Llama-2-70B: few rows, a long axis
        {"name": "decode_long", "op": "attend", "seqs": 1, "new": 1, "past": 130000, "heads": 64, "kv": 8, "dim": 128, "page": 256, "dtype": "bf16"},
        # a server's batch of conversations of all lengths, heads of Llama-2-70B
        {"name": "decode_batch", "op": "attend", "seqs": 64, "new": 1, "past": 8192, "heads": 64, "kv": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one KV head for 71 query heads of 64 (Falcon-7B)
        {"name": "decode_mqa", "op": "attend", "seqs": 16, "new": 1, "past": 2000, "heads": 71, "kv": 1, "dim": 64, "page": 128, "dtype": "f16"},
        # a whole prompt of 2048 tokens, heads of Llama-2-7B
        {"name": "prompt", "op": "attend", "seqs": 1, "new": 2048, "past": 0, "heads": 32, "kv": 32, "dim": 128, "page": 64, "dtype": "f16"},
        # prompt chunks of different lengths behind long pasts, heads of Llama-2-70B
        {"name": "chunk_ragged", "op": "attend", "seqs": 4, "new": 512, "past": 8000, "heads": 64, "kv": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one step of a beam search with four beams, cache of a 32-layer model
        {"name": "beams_four", "op": "beams", "seqs": 4, "past": 300, "add": 1, "page": 64, "heads": 8, "dim": 128, "layers": 32},
        # a server forks a batch of long conversations and makes room for the next chunk
        {"name": "beams_many", "op": "beams", "seqs": 256, "past": 8192, "add": 16, "page": 64, "heads": 8, "dim": 64, "layers": 2},
        # a small pool with a few holes
        {"name": "compact_small", "op": "compact", "seqs": 8, "past": 500, "page": 32, "heads": 8, "dim": 64, "layers": 4, "freed": 0.25},
        # most of a large pool was freed; what is left moves to the front
        {"name": "compact_large", "op": "compact", "seqs": 48, "past": 2000, "page": 64, "heads": 8, "dim": 128, "layers": 16, "freed": 0.5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "beams", "compact"])
    page = rng.choice([32, 64, 128, 256])
    dim = rng.choice([64, 80, 96, 112, 128])
    dtype = rng.choice(["f16", "bf16"])
    if op == "append":
        dtype = rng.choice(["f16", "bf16", "f32"])
        seqs, heads = _log(rng, 1, 64), _log(rng, 1, 64)
        new = _log(rng, 1, max(1, min(2048, 100_000_000 // (seqs * heads * dim))))
        return {"op": op, "seqs": seqs, "new": new, "past": _log(rng, 1, 4096), "heads": heads, "dim": dim, "page": page, "dtype": dtype}
    if op == "attend":
        kv = rng.choice([1, 2, 4, 8, 32])
        heads = kv * (rng.randint(1, 71) if kv == 1 else rng.choice([1, 2, 4, 5, 7, 8, 16]) if kv < 32 else 1)
        if rng.random() < 0.6:
            new, seqs = rng.choice([1, 1, 1, 2, 5]), _log(rng, 1, 64)
            past = _log(rng, 1, max(1, min(130000, 400_000_000 // (seqs * kv * dim))))
        else:
            seqs, new = _log(rng, 1, 8), _log(rng, 6, 2048)
            past = _log(rng, 1, 8000)
            new = max(2, min(new, 300_000_000 // (seqs * heads * (past + new))))
        return {"op": op, "seqs": seqs, "new": new, "past": past, "heads": heads, "kv": kv, "dim": dim, "page": page, "dtype": dtype}
    heads, layers = rng.choice([1, 2, 8, 32]), rng.choice([1, 2, 16])
    seqs = _log(rng, 1, 200)
    past = _log(rng, 1, max(2, min(8192, 500_000_000 // (seqs * heads * layers * dim))))
    if op == "beams":
        return {"op": op, "seqs": seqs, "past": past, "add": _log(rng, 1, 64), "page": page, "heads": heads, "dim": dim, "layers": layers}
    return {"op": op, "seqs": seqs, "past": past, "page": page, "heads": heads, "dim": dim, "layers": layers, "freed": rng.choice([0.1, 0.5, 0.9])}


# ---- the cache's layout ------------------------------------------------------------------------------------------------------------------------
def groups_of(dim):
    """Groups of 32 dims that a head of `dim` takes; five and seven take the room of six and eight."""
    g = (dim + 31) // 32
    return {5: 6, 7: 8}.get(g, g)


def page_bytes(heads, dim, page):
    return heads * (page // 32) * groups_of(dim) * 32 * 36


def _maps(groups, device):
    """For [token of a block][dim]: the nibble of its code within the K (V) codes; for [token][group]: the place of its scale."""
    t = torch.arange(32, device=device)[:, None]
    c = torch.arange(32 * groups, device=device)[None, :]
    nib = lambda e: e // 2 + 4 * (e % 2)  # noqa: E731
    kn = ((4 * t + (c % 32) // 8) * groups + c // 32) * 8 + nib(c % 8)
    vn = (((t % 16) // 4) * (32 * groups) + c) * 8 + nib(t % 4 + 4 * (t // 16))
    g = torch.arange(groups, device=device)[None, :]
    ks = (((t // 16) * 4 + (t % 16) // 4) * groups + g) * 4 + t % 4
    vs = (((t % 16) // 4) * groups + g) * 8 + t % 4 + 4 * (t // 16)
    return kn, vn, ks, vs


def _quantize(x, groups, wide=torch.float32):
    """x [.., dim] -> codes uint8 [.., 32 groups], scales f16 [.., groups]."""
    x = torch.nn.functional.pad(x.to(wide), (0, 32 * groups - x.shape[-1])).unflatten(-1, (groups, 32)).clamp(-65504, 65504)
    top = torch.take_along_dim(x, x.abs().argmax(-1, keepdim=True), -1)
    d = top / -8
    h = d.to(torch.float16)
    inv = torch.where((h != 0) & ~torch.isnan(h), 1 / d, 0)
    q = (x * inv + 8.5).floor().clamp(0, 15)
    q = torch.where(torch.isnan(d), 8, q).to(torch.uint8)
    return q.flatten(-2), h.squeeze(-1)


def _store_blocks(pages, where, heads, dim, kc, ks, vc, vs):
    """Whole blocks of codes [n, heads, 32, 32 G] and scales [n, heads, 32, G] into the places `where` ([n]: page * blocks a page + block)."""
    G = groups_of(dim)
    kn, vn, km, vm = (m.flatten() for m in _maps(G, pages.device))
    blocks = pages.view(pages.shape[0], heads, -1, G * 1152)
    out = []
    for codes, at in ((kc, kn), (vc, vn)):
        n = codes.flatten(2)[..., torch.argsort(at)]
        out.append(n[..., 0::2] | (n[..., 1::2] << 4))
    for scale, at in ((ks, km), (vs, vm)):
        out.append(scale.flatten(2)[..., torch.argsort(at)].contiguous().view(torch.uint8))
    nb = blocks.shape[2]
    blocks[where // nb, :, where % nb] = torch.cat(out, -1)


def _load_blocks(pages, where, heads, dim, half):
    """Codes uint8 [n, heads, 32, 32 G] and scales f16 [n, heads, 32, G] of K (half 0) or V (half 1) of the blocks `where`."""
    G = groups_of(dim)
    maps = _maps(G, pages.device)
    blocks = pages.view(pages.shape[0], heads, -1, G * 1152)
    nb = blocks.shape[2]
    b = blocks[where // nb, :, where % nb]
    c = b[..., half * 512 * G:(half + 1) * 512 * G]
    nibbles = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    s = b[..., (16 + half) * 64 * G:(17 + half) * 64 * G].contiguous().view(torch.float16)
    return nibbles[..., maps[half]], s[..., maps[2 + half]]


def _load(pages, where, heads, dim, half, wide=torch.float32):
    """Values [n, heads, 32, dim] of the blocks `where`."""
    codes, scales = _load_blocks(pages, where, heads, dim, half)
    x = (codes.to(wide) - 8).unflatten(-1, (-1, 32)) * scales.to(wide).unsqueeze(-1)
    return x.flatten(-2)[..., :dim]


# ---- the cases' inputs -------------------------------------------------------------------------------------------------------------------------
def _lengths(n, most, least=0, turn=0.618034):
    """n lengths from `least` to `most`, spread evenly over the range, the last one the longest: the same for every seed."""
    x = (least + (most - least) * ((torch.arange(1, n + 1) * turn) % 1)).long()
    x[-1] = most
    return x


def _new_and_past(case):
    """Of each sequence: its new rows and the tokens before them."""
    return _lengths(case["seqs"], case["new"], 1 if case["new"] == 1 else 0), _lengths(case["seqs"], case["past"], 0, 0.754878)


def _tables(g, lens, page, spare=0):
    """A table [n, widest + spare pages] of pages in random order for sequences of these lengths, and the pages in use."""
    need = (lens + page - 1) // page
    table = torch.full((len(lens), int(need.max()) + spare), -1, dtype=torch.int32)
    total = int(need.sum())
    table[torch.arange(table.shape[1])[None, :] < need[:, None]] = torch.randperm(total, generator=g).int()
    return table, total


def _rows(gen, shape, dtype, dev):
    """Rows as a layer gives them: normal values, some channels larger than the rest and off zero, as K's are."""
    x = torch.randn(shape, generator=gen, device=dev)
    wide = torch.rand(shape[-2:], generator=gen, device=dev)
    return (x * (1 + 3 * (wide > 0.95)) + 2 * (wide < 0.04)).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    page = case["page"]
    if case["op"] in ("append", "attend"):
        heads = s["kv"] = case.get("kv", case["heads"])
        new, past = (x[torch.randperm(case["seqs"], generator=torch.Generator().manual_seed(seed))] for x in _new_and_past(case))
        lens = past + new
        table, total = _tables(g, lens, page)
        s["total"] = int(new.sum())
        s["max_new"] = case["new"]
        s["cu"] = torch.nn.functional.pad(new.cumsum(0), (1, 0)).int().to(dev)
        s["lens"] = lens.int().to(dev)
        s["table"] = table.to(dev)
        s["pages"] = torch.zeros(total, page_bytes(heads, case["dim"], page), dtype=torch.uint8, device=dev)
        dtype = DTYPES[case["dtype"]]
        if case["op"] == "append":
            s["k"] = _rows(gen, (s["total"], heads, case["dim"]), dtype, dev)
            s["v"] = _rows(gen, (s["total"], heads, case["dim"]), dtype, dev)
        else:
            s["q"] = _rows(gen, (s["total"], case["heads"], case["dim"]), dtype, dev)
            G, step = groups_of(case["dim"]), max(1, (1 << 27) // (heads * 32 * case["dim"]))
            places = torch.arange(total * (page // 32), device=dev)
            for i in range(0, len(places), step):
                w = places[i:i + step]
                kc, ks = _quantize(_rows(gen, (len(w) * 32, heads, case["dim"]), torch.float32, dev).unflatten(0, (-1, 32)).transpose(1, 2), G)
                vc, vs = _quantize(torch.randn((len(w), heads, 32, case["dim"]), generator=gen, device=dev), G)
                _store_blocks(s["pages"], w, heads, case["dim"], kc, ks, vc, vs)
        return s
    lens = _lengths(case["seqs"], case["past"], 1)[torch.randperm(case["seqs"], generator=g)]
    width = page_bytes(case["heads"], case["dim"], page)
    if case["op"] == "beams":
        spare = (case["add"] + page - 1) // page + 1
        table, total = _tables(g, lens, page, spare)
        s["parents"] = torch.randint(case["seqs"], (case["seqs"],), generator=g).int().to(dev)
        s["add"] = torch.full((case["seqs"],), case["add"], dtype=torch.int32, device=dev)
        n_pages = total + case["seqs"] * (spare + 1)
        place = torch.randperm(n_pages, generator=g)[:total].int()
    else:
        table, total = _tables(g, lens, page)
        n_pages = max(total + 1, int(total / (1 - case["freed"])))
        place = torch.randperm(n_pages, generator=g)[:total].int()
    table = torch.where(table >= 0, place[table.long().clamp(min=0)], table)
    refs = torch.zeros(n_pages, dtype=torch.int32)
    refs[place.long()] = 1
    s["table"], s["lens"], s["refs"] = table.to(dev), lens.int().to(dev), refs.to(dev)
    s["pages"] = torch.randint(0, 256, (case["layers"], n_pages, width), generator=gen, device=dev, dtype=torch.uint8)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------------
def _row_places(s):
    """Of each packed row: its sequence and its position."""
    row = torch.arange(s["total"], device=s["cu"].device)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    return seq, s["lens"].long()[seq] - s["cu"].long()[seq + 1] + row


def _plain_append(s):
    dim, page, heads, G = s["dim"], s["page"], s["kv"], groups_of(s["dim"])
    seq, pos = _row_places(s)
    pid = s["table"].long()[seq, pos // page]
    pages = s["pages"].view(-1, heads, page // 32, G * 1152)
    (kc, ks), (vc, vs) = _quantize(s["k"], G), _quantize(s["v"], G)
    bad = (torch.isnan(ks).any(-1) | torch.isnan(vs).any(-1))[..., None]
    ks, vs = torch.where(bad, float("nan"), ks), torch.where(bad, 0, vs)
    # the blocks that the rows fall into, read, changed and written back
    block, which = torch.unique(pid * (page // 32) + (pos % page) // 32, return_inverse=True)
    old = [_load_blocks(s["pages"], block, heads, dim, half) for half in (0, 1)]
    for (codes, scales), c, x in zip(old, (kc, vc), (ks, vs)):
        codes[which, :, pos % 32] = c
        scales[which, :, pos % 32] = x
    _store_blocks(s["pages"], block, heads, dim, *old[0], *old[1])
    return [_load(s["pages"], block, heads, dim, half)[which, :, pos % 32].to(torch.float16) for half in (0, 1)]


def _attend(s, wide):
    """The whole batch at once: padded to its longest sequence and its most rows."""
    dim, page, kv, G = s["dim"], s["page"], s["kv"], s["heads"] // s["kv"]
    most = s["table"].shape[1] * page
    per = page // 32
    where = (s["table"].long().clamp(min=0)[:, :, None] * per + torch.arange(per, device=s["table"].device)).flatten()
    k = _load(s["pages"], where, kv, dim, 0, wide).unflatten(0, (s["seqs"], -1)).transpose(1, 2).flatten(2, 3)   # [seq][kv][position][dim]
    seq, pos = _row_places(s)
    row = torch.arange(s["total"], device=seq.device) - s["cu"].long()[seq]
    q = torch.zeros(s["seqs"], s["max_new"], kv, G, dim, dtype=wide, device=seq.device)
    q[seq, row] = s["q"].to(wide).unflatten(1, (kv, G))
    at = torch.full((s["seqs"], s["max_new"]), -1, device=seq.device)
    at[seq, row] = pos
    q = q.permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dim)                                               # [seq][kv][row, head][position]
    del k
    seen = torch.arange(most, device=seq.device) <= at.repeat_interleave(G, 1)[:, None, :, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0, top))
    del scores
    v = _load(s["pages"], where, kv, dim, 1, wide).unflatten(0, (s["seqs"], -1)).transpose(1, 2).flatten(2, 3)
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=torch.finfo(wide).tiny)
    return out.unflatten(2, (-1, G)).permute(0, 2, 1, 3, 4)[seq, row].flatten(1, 2)


def _counts(table, lens, page, n_pages):
    """How many entries of the table name each page."""
    used = (torch.arange(table.shape[1], device=table.device) < ((lens + page - 1) // page)[:, None]) & (table >= 0)
    return torch.zeros(n_pages + 1, dtype=torch.int32, device=table.device).index_add_(
        0, torch.where(used, table, n_pages).flatten().long(), torch.ones(table.numel(), dtype=torch.int32, device=table.device))[:n_pages], used


def _plain_beams(s):
    page, n_pages, par = s["page"], s["refs"].shape[0], s["parents"].long()
    before, used = _counts(s["table"], s["lens"], page, n_pages)
    table, lens = torch.where(used, s["table"], -1)[par], s["lens"][par]
    refs = s["refs"] - before + _counts(table, lens, page, n_pages)[0]
    # room for `add` more tokens each: the pages behind the last one, and a page of its own where the last one is shared at the sequence's turn
    first, last = lens // page, (lens + s["add"] + page - 1) // page
    partly = lens % page != 0
    tail = torch.where(partly, torch.take_along_dim(table, first[:, None].long(), 1)[:, 0], -1)
    n = torch.arange(len(par), device=par.device)
    earlier = ((tail[:, None] == tail[None, :]) & (n[None, :] < n[:, None]) & (s["add"] > 0)[None, :]).sum(1)
    copied = partly & (s["add"] > 0) & (refs[tail.long().clamp(min=0)] - earlier > 1)
    start = first + (partly & ~copied)
    need = torch.where(s["add"] > 0, last - start, 0)
    free = torch.argsort(refs != 0, stable=True)
    short = (need.sum() - (refs == 0).sum()).clamp(min=0).int()
    entry = torch.arange(table.shape[1], device=par.device)
    fresh = (entry >= start[:, None]) & (entry < (start + need)[:, None])
    new = free[((need.cumsum(0) - need)[:, None] + entry - start[:, None]).clamp(0, n_pages - 1)].int()
    grown = torch.where(fresh, new, table)
    src, dst = tail[copied].long(), torch.take_along_dim(grown, first[:, None].long(), 1)[:, 0][copied].long()
    s["pages"][:, dst] = s["pages"][:, src]
    refs = refs - torch.zeros_like(refs).index_add_(0, tail.long().clamp(min=0), copied.int())
    refs[grown[fresh].long()] = 1
    return [grown, lens + s["add"], refs, short, s["pages"]]


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    n_pages = refs.shape[0]
    used = refs > 0
    count = used.sum()
    at = torch.arange(n_pages, device=refs.device)
    src, dst = at[used & (at >= count)], at[~used & (at < count)]
    to = at.clone()
    to[src] = dst
    s["pages"][:, dst] = s["pages"][:, src]
    new = torch.zeros_like(refs)
    new[to[used]] = refs[used]
    return [torch.where(table >= 0, to[table.long().clamp(min=0)].int(), table), new, count.int(), s["pages"]]


def run(s):
    if own:
        from ctransformers_amd import ops
        if s["op"] == "append":
            ops.kv4_append(s["k"], s["v"], s["pages"], s["table"], s["lens"], s["cu"], s["max_new"], page_tokens=s["page"])
            return ops.kv4_read(s["pages"], s["table"], s["lens"], s["cu"], s["max_new"], s["total"], n_head_kv=s["kv"], head_dim=s["dim"], page_tokens=s["page"])
        if s["op"] == "attend":
            return ops.kv4_attention(s["q"], s["pages"], s["table"], s["lens"], s["cu"], s["max_new"], n_head_kv=s["kv"], page_tokens=s["page"])
        if s["op"] == "beams":
            table, lens, refs = ops.kv_fork(s["table"], s["lens"], s["refs"], s["parents"], page_tokens=s["page"])
            table, lens, refs, short = ops.kv_reserve(s["pages"], table, lens, refs, s["add"], page_tokens=s["page"])
            return [table, lens, refs, short, s["pages"]]
        table, refs, used = ops.kv_compact(s["pages"], s["table"], s["refs"])
        return [table, refs, used, s["pages"]]
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "attend":
        return _attend(s, torch.float32).to(s["q"].dtype)
    return _plain_beams(s) if s["op"] == "beams" else _plain_compact(s)


def work(case):
    if case["op"] in ("append", "attend"):
        new, past = _new_and_past(case)
    if case["op"] == "append":
        rows = int(new.sum()) * case["heads"] * 2
        # the rows in, their 4.5 bits out and in again, the halves out
        return {"bytes": rows * (case["dim"] * (DTYPES[case["dtype"]].itemsize + 2) + 2 * groups_of(case["dim"]) * 18), "flops": rows * case["dim"] * 4}
    if case["op"] == "attend":
        rows, keys = int(new.sum()), int((past + new)[new > 0].sum())
        seen = int((new * past + new * (new + 1) // 2).sum())
        return {"bytes": keys * case["kv"] * groups_of(case["dim"]) * 36 + rows * case["heads"] * case["dim"] * 2 * DTYPES[case["dtype"]].itemsize,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    g = torch.Generator().manual_seed(0)
    lens = _lengths(case["seqs"], case["past"], 1)
    page, width = case["page"], page_bytes(case["heads"], case["dim"], case["page"]) * case["layers"]
    table, total = _tables(g, lens, page, (case["add"] + page - 1) // page + 1 if case["op"] == "beams" else 0)
    if case["op"] == "beams":
        par = torch.randint(case["seqs"], (case["seqs"],), generator=g)
        sharing = torch.bincount(par, minlength=case["seqs"])
        copies = int(torch.where((lens % page != 0) & (sharing > 1), sharing - 1, 0).sum())
        return {"bytes": 2 * copies * width + 8 * table.numel() + 8 * (total + 3 * case["seqs"]), "flops": 0}
    n_pages = max(total + 1, int(total / (1 - case["freed"])))
    place = torch.randperm(n_pages, generator=g)[:total]
    return {"bytes": 2 * int((place >= total).sum()) * width + 8 * table.numel() + 8 * n_pages, "flops": 0}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------------------
def _exact_values(rows, dim):
    """What rows [n, heads, dim] stand for once stored."""
    out = torch.zeros_like(rows, dtype=torch.float64)
    for c in range(0, dim, 32):
        x = rows[..., c:c + 32].double()
        hi, lo = x.max(-1).values, x.min(-1).values
        tie = torch.where((x == hi[..., None]).int().argmax(-1) <= (x == lo[..., None]).int().argmax(-1), hi, lo)
        d = torch.where(hi > -lo, hi, torch.where(hi < -lo, lo, tie)) / -8
        code = torch.trunc(x / torch.where(d == 0, 1, d)[..., None] + 8.5).clamp(max=15)
        out[..., c:c + 32] = d.half().double()[..., None] * (code - 8)
    return out


def exact(case, seed):
    if case["op"] not in ("append", "attend"):
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        return [_exact_values(s["k"], case["dim"]), _exact_values(s["v"], case["dim"])]
    page, per, kv, dim = case["page"], case["page"] // 32, s["kv"], case["dim"]
    G = case["heads"] // kv
    out = torch.zeros(s["total"], case["heads"], dim, dtype=torch.float64, device="cuda")
    for b in range(case["seqs"]):
        lo, hi, n = int(s["cu"][b]), int(s["cu"][b + 1]), int(s["lens"][b])
        if hi == lo or n == 0:
            continue
        spot = torch.arange(n, device="cuda")
        where = s["table"][b, : (n + page - 1) // page].long()[:, None] * per + torch.arange(per, device="cuda")[None, :]
        where = where.flatten()[: (n + 31) // 32]
        hidden = spot[None, :] > torch.arange(n - (hi - lo), n, device="cuda")[:, None]
        for half in range(kv):   # one KV head at a time: the others' blocks are not touched
            alone = s["pages"].view(s["pages"].shape[0], kv, -1)[:, half].contiguous()
            k = _load(alone, where, 1, dim, 0, torch.float64)[:, 0].flatten(0, 1)[:n]
            v = _load(alone, where, 1, dim, 1, torch.float64)[:, 0].flatten(0, 1)[:n]
            for h in range(half * G, half * G + G):
                x = (s["q"][lo:hi, h].double() @ k.T) * dim ** -0.5
                x[hidden] = -math.inf
                out[lo:hi, h] = torch.softmax(x, -1) @ v
    return out
