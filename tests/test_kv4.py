"""The 4-bit paged KV cache (ctransformers_amd/ops.py): rows in and out, attention over it, the pages' bookkeeping — each against a plain implementation in 64 bits
(the stored bits against the format's definition in the arithmetic it names), on the CPU emulation of the kernels and on the GPU.

Tolerances, from the roundings that the kernels make (ops.kv4_attention): p and V's values are halves, off by 2^-11 each, relative; a result row is a mean of values
v with weights p, so an element is off by at most (2^-11 + 2^-11) A with A = sum p |v| / sum p.  An error of e in a score (natural units) changes every weight by a
factor within exp(+-e): 2 e A.  A score's error: f32 sums, (D + 8) 2^-24 scale sum |q| |k|; the exponent's argument, (4 |s| + 8) 2^-23; queries that are not
halves already, 2^-11 scale sum |q| |k| (float32) or the part below f16's range after the row's power of two, 2^-25 max |q| scale sum |k| (bf16); and in the
many-row kernel K's values as halves, 2^-11 scale sum |q| |k|.  The result's own rounding is half a step of its type.

Halves below 2^-14 are multiples of 2^-24, so there a rounding is off by up to 2^-25 absolutely.  That happens to p (the largest weight is at least 1: weights are
relative to a running maximum, which no final maximum is below), 2^-25 sum |v| / sum p <= 2^-25 sum |v| in the result; in the few-row kernel the second half of p has
the same spacing, so it does not help there.  And it happens to float16 results, 2^-25.  (V's values are exempt: d is a multiple of 2^-24 and so is d (code - 8).)
attention64 adds both to A, divided by the 2^-10 that A is multiplied with.  A row whose largest weight belongs to a value of 0 shows it: A is then 1e-9 of its
neighbours' values, and the bound without these terms is smaller than the spacing of the type that the result has."""
import math
import os
import re

import numpy as np
import pytest
import torch

from conftest import EMU_LIB, HIP_LIB, ROOT, has_gpu
from ctransformers_amd import ops

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(params=["emu", pytest.param("hip", marks=pytest.mark.gpu)])
def dev(request):
    if request.param == "emu":
        if has_gpu():
            pytest.skip("the emulation is for hosts without a GPU")
        request.getfixturevalue("emu_lib")
        ops.load(EMU_LIB)
        yield torch.device("cpu")
    else:
        request.getfixturevalue("hip_lib")
        ops.load(HIP_LIB)
        yield torch.device("cuda:0")
    ops._lib = None
    ops._on_gpu = True


# ---- the format, from its definition ------------------------------------------------------------------------------------------------------------
def groups(dim):
    g = -(-dim // 32)
    return {5: 6, 7: 8}.get(g, g)


def nib(e):
    return e // 2 + 4 * (e % 2)


def quantize(x):
    """codes and scales of float32 rows [.., dim] -> uint8 [.., 32 G], float16 [.., G]; float32 arithmetic, as the format says"""
    G = groups(x.shape[-1])
    y = np.zeros(x.shape[:-1] + (32 * G,), np.float32)
    y[..., :x.shape[-1]] = np.clip(x, -65504, 65504)
    y = y.reshape(y.shape[:-1] + (G, 32))
    top = np.take_along_axis(y, np.argmax(np.abs(y), -1)[..., None], -1)
    d = top / np.float32(-8)
    with np.errstate(all="ignore"):
        h = d.astype(np.float16)
        inv = np.where((h != 0) & ~np.isnan(d), np.float32(1) / d, np.float32(0)).astype(np.float32)
        q = np.minimum(np.floor(y * inv + np.float32(8.5)), 15)
    q = np.where(np.isnan(d), 8, q)
    return q.reshape(x.shape[:-1] + (32 * G,)).astype(np.uint8), h[..., 0]


class Cache:
    """One layer's pages with their contents kept beside them as codes and scales per token."""

    def __init__(self, seed, lens, heads, dim, page, extra_pages=2, extra_width=1):
        rng = np.random.default_rng(seed)
        self.lens, self.heads, self.dim, self.page, self.G = list(lens), heads, dim, page, groups(dim)
        need = [-(-n // page) for n in lens]
        self.n_pages = max(1, sum(need) + extra_pages)
        order = rng.permutation(self.n_pages)[:sum(need)]
        self.table = np.full((len(lens), max(need + [0]) + extra_width), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.bytes = heads * (page // 32) * self.G * 1152
        self.pages = rng.integers(0, 256, (self.n_pages, self.bytes), dtype=np.uint8)   # what nobody has written is anything: scales that are NaN among it

    def block(self, b, pos, h):
        base = (h * (self.page // 32) + pos % self.page // 32) * self.G * 1152
        return self.table[b, pos // self.page], base

    def put(self, b, pos, h, half, codes, scales):
        """one token's codes [32 G] and scales [G] at their places"""
        p, base = self.block(b, pos, h)
        t, G, row = pos % 32, self.G, self.pages[self.table[b, pos // self.page]]
        for c in range(32 * G):
            if half == 0:
                n = ((4 * t + (c % 32) // 8) * G + c // 32) * 8 + nib(c % 8)
            else:
                n = 1024 * G + ((t % 16 // 4) * 32 * G + c) * 8 + nib(t % 4 + 4 * (t // 16))
            o = base + n // 2
            row[o] = (row[o] & (0xF0 if n % 2 == 0 else 0x0F)) | (codes[c] << (4 * (n % 2)))
        s = scales.view(np.uint8).reshape(G, 2)
        for g in range(G):
            at = (((t // 16) * 4 + t % 16 // 4) * G + g) * 4 + t % 4 if half == 0 else ((t % 16 // 4) * G + g) * 8 + t % 4 + 4 * (t // 16)
            o = base + (16 + half) * 64 * G + 2 * at
            row[o:o + 2] = s[g]

    def fill(self, seed, scale=1.0):
        """every token of every sequence: random codes and scales; their values in float64 [b][half] -> [len, heads, dim]"""
        rng = np.random.default_rng(seed)
        self.values = []
        for b, n in enumerate(self.lens):
            both = []
            for half in (0, 1):
                x = (rng.standard_normal((n, self.heads, self.dim)) * scale).astype(np.float32)
                x[..., rng.integers(0, self.dim)] += 3 * scale
                codes, scales = quantize(x)
                for pos in range(n):
                    for h in range(self.heads):
                        self.put(b, pos, h, half, codes[pos, h], scales[pos, h])
                both.append(((codes.astype(np.float64) - 8).reshape(n, self.heads, self.G, 32) * scales.astype(np.float64)[..., None])
                            .reshape(n, self.heads, 32 * self.G)[..., :self.dim])
            self.values.append(both)

    def on(self, dev):
        return (torch.from_numpy(self.pages.copy()).to(dev), torch.from_numpy(self.table).to(dev), torch.tensor(self.lens, dtype=torch.int32, device=dev))


def attention64(q, values, heads_kv, scale, extra):
    """rows q [n, H, D] of one sequence (float64) -> result, A and the error allowed in a score, all [n, H, ..]"""
    k, v = values
    n, H, D = q.shape
    L, rep = k.shape[0], H // heads_kv
    out, mag, err = np.zeros((n, H, D)), np.zeros((n, H, D)), np.zeros((n, H))
    for i in range(n):
        see = L - n + i + 1
        if see <= 0:
            continue
        for h in range(H):
            kk, vv = k[:see, h // rep], v[:see, h // rep]
            s = kk @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], mag[i, h] = p @ vv, p @ np.abs(vv) + 2.0**-15 * np.abs(vv).sum(0) + 2.0**-15
            dots = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
            err[i, h] = ((D + 8) * 2.0**-24 + extra[0]) * dots + extra[1] * np.abs(q[i, h]).max() * np.abs(kk).sum(-1).max() * abs(scale) + (4 * np.abs(s).max() + 8) * 2.0**-23
    return out, mag, err


def check_attention(dev, lens, news, H, heads_kv, dim, page, dtype, seed=0, out_dtype=None, table_edit=None, scale=None, width=1, strided=False):
    c = Cache(seed, lens, heads_kv, dim, page, extra_width=width)
    c.fill(seed + 1)
    g = torch.Generator().manual_seed(seed + 2)
    total = sum(news)
    q = torch.randn((total, H, dim), generator=g).to(dtype)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=dev)
    pages, table, n = c.on(dev)
    qd = q.to(dev)
    if strided:   # rows of a wider tensor, heads before rows
        wide = torch.full((H, total, dim + 16), float("nan"), dtype=dtype, device=dev)
        wide[..., 8:8 + dim] = qd.transpose(0, 1)
        qd = wide[..., 8:8 + dim].transpose(0, 1)
    out = torch.full((total + 3, H, dim), 7.0, dtype=out_dtype or dtype, device=dev)
    got = ops.kv4_attention(qd, pages, table, n, cu, max(news + [0]), n_head_kv=heads_kv, page_tokens=page, scale=scale, out=out[:total])
    assert got.data_ptr() == out.data_ptr() or total == 0
    assert (out[total:] == 7).all()
    sc = 1 / math.sqrt(dim) if scale is None else scale
    rows = max(news + [0]) * (H // heads_kv)
    many = rows > (192 if groups(dim) <= 2 else 96 if groups(dim) <= 4 else 16)
    extra = ((2.0**-11 if many else 0) + (2.0**-11 if dtype == F32 else 0), 2.0**-25 if dtype != F16 else 0)
    eps = torch.finfo(out.dtype).eps / 2
    res = out.double().cpu().numpy()
    at = 0
    for b, k in enumerate(news):
        want, mag, err = attention64(q[at:at + k].double().numpy(), c.values[b], heads_kv, sc, extra)
        tol = mag * (2 * 2.0**-11 + 2 * np.expm1(err)[..., None]) * 1.01 + np.abs(want) * eps * 1.01 + 1e-12
        bad = np.abs(res[at:at + k] - want) > tol
        assert not bad.any(), (b, int(bad.sum()), float(np.abs(res[at:at + k] - want).max()), float(tol.max()))
        at += k


# ---- attention ----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [8, 32, 64, 80, 96, 112, 128, 160, 192, 256])
def test_token_step_every_head_size(dev, dim):
    check_attention(dev, [37], [1], 4, 2, dim, 32, F16, seed=dim)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rep", [1, 3, 16])
def test_token_step_grouped_heads(dev, rep, dtype):
    check_attention(dev, [1, 33, 64], [1, 1, 1], 2 * rep, 2, 64, 64, dtype, seed=rep)


@pytest.mark.parametrize("lens,news", [([0], [1]), ([5], [7]), ([32, 0, 31], [1, 0, 2]), ([70, 3], [3, 3]), ([100, 33], [0, 4])])
def test_lengths_that_leave_rows_empty_or_end_inside_a_block(dev, lens, news):
    """a sequence without tokens, more rows than tokens (the first see nothing), sequences without rows, rows that end inside blocks and pages"""
    check_attention(dev, lens, news, 4, 2, 64, 32, F16, seed=3)


@pytest.mark.parametrize("dim,lens,news,H,kv", [(64, [40], [40], 2, 1), (128, [75], [33], 2, 2), (80, [65, 20, 0, 9], [9, 20, 3, 9], 8, 2), (32, [130], [5], 7, 1),
                                                (64, [60], [50], 8, 2), (128, [75], [33], 8, 2), (80, [65, 20, 0, 9], [30, 20, 3, 9], 8, 2), (32, [130, 1], [30, 1], 7, 1), (192, [40], [18], 1, 1), (256, [33], [17], 1, 1)])
def test_many_rows(dev, dim, lens, news, H, kv):
    check_attention(dev, lens, news, H, kv, dim, 64, BF16 if dim == 80 else F16, seed=dim)


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_two_row_tiles(dev, dim):
    check_attention(dev, [50, 35], [2, 1], 12, 1, dim, 32, F16, seed=5)


def test_keys_split_over_workgroups(dev):
    """a table wide enough that the keys of a tile are divided, with sequences that fill one part, a few and none of them"""
    check_attention(dev, [600, 3, 257], [1, 1, 2], 2, 1, 32, 32, F16, seed=7, width=40)
    check_attention(dev, [700, 40], [20, 40], 2, 1, 32, 32, F16, seed=8, width=40)
    check_attention(dev, [700, 40], [20, 40], 5, 1, 32, 32, F16, seed=8, width=40)


def test_queries_of_any_stride_and_results_of_another_type(dev):
    check_attention(dev, [40], [3], 4, 2, 64, 32, F16, strided=True)
    check_attention(dev, [40], [20], 4, 2, 64, 32, BF16, strided=True, out_dtype=F32)
    check_attention(dev, [140], [98], 4, 2, 64, 32, F32, strided=True, out_dtype=BF16)
    check_attention(dev, [40], [1], 4, 2, 72, 32, F32, out_dtype=F16)


@pytest.mark.parametrize("news", [1, 20, 100])
def test_queries_far_outside_of_halves(dev, news):
    """bf16 rows of 1e30 and of 1e-30: the scale brings the scores back"""
    for big in (2.0**100, 2.0**-100):
        c = Cache(1, [40 + news], 1, 64, 32)
        c.fill(2)
        q = (torch.randn((news, 2, 64), generator=torch.Generator().manual_seed(4)) * big).to(BF16)
        pages, table, n = c.on(dev)
        got = ops.kv4_attention(q.to(dev), pages, table, n, None, news, n_head_kv=1, page_tokens=32, scale=0.125 / big).double().cpu().numpy()
        want, mag, err = attention64(q.double().numpy(), c.values[0], 1, 0.125 / big, (2.0**-11, 2.0**-25))
        assert (np.abs(got - want) <= mag * (2.0**-10 + 2 * np.expm1(err)[..., None]) * 1.01 + np.abs(want) * 2.0**-8 * 1.01).all()


@pytest.mark.parametrize("news,H", [(1, 2), (36, 2), (36, 6)])
def test_absent_pages_are_not_attended_to(dev, news, H):
    c = Cache(3, [100], 1, 64, 32)
    c.fill(4)
    pages, table, n = c.on(dev)
    for bad in (-1, c.n_pages, 2**31 - 1, -2**31):
        table[0, 1] = bad
        q = torch.randn((news, H, 64), generator=torch.Generator().manual_seed(5)).to(F16)
        got = ops.kv4_attention(q.to(dev), pages, table, n, None, news, n_head_kv=1, page_tokens=32).double().cpu().numpy()
        k, v = (np.concatenate([x[:32], x[64:]]) for x in c.values[0])
        # (every row's own position lies behind the hole)
        want, mag, err = attention64(q.double().numpy(), (k, v), 1, 0.125, (2.0**-11, 0))
        assert (np.abs(got - want) <= mag * (2.0**-10 + 2 * np.expm1(err)[..., None]) * 1.01 + np.abs(want) * 2.0**-11 * 1.01).all()
    table[0] = -1
    assert (ops.kv4_attention(q.to(dev), pages, table, n, None, news, n_head_kv=1, page_tokens=32) == 0).all()


def test_a_nan_reaches_the_rows_that_see_it_and_no_others(dev):
    for rows in (2, 40, 100):
        for where in ("k", "v"):
            k, v = (torch.randn((rows, 2, 64), generator=torch.Generator().manual_seed(i)).to(F16) for i in (1, 2))
            {"k": k, "v": v}[where][rows // 2, 1, 5] = float("nan")
            c = Cache(1, [rows], 2, 64, 32)
            pages, table, n = c.on(dev)
            ops.kv4_append(k.to(dev), v.to(dev), pages, table, n, None, rows, page_tokens=32)
            q = torch.randn((rows, 4, 64), generator=torch.Generator().manual_seed(3)).to(F16).to(dev)
            out = ops.kv4_attention(q, pages, table, n, None, rows, n_head_kv=2, page_tokens=32).isnan().cpu()
            want = torch.zeros_like(out)
            want[rows // 2:, 2:] = True
            assert torch.equal(out, want)
            kr, vr = ops.kv4_read(pages, table, n, None, rows, rows, n_head_kv=2, head_dim=64, page_tokens=32)
            assert kr[rows // 2, 1].isnan().all() and (vr[rows // 2, 1] == 0).all() and int(kr.isnan().sum()) == 64 and not vr.isnan().any()
    q[1, 0, 0] = float("nan")
    q[2, 1, 0] = float("inf")
    c.fill(1)
    out = ops.kv4_attention(q[:3], torch.from_numpy(c.pages).to(dev), table, n, None, 3, n_head_kv=2, page_tokens=32).isnan().all(-1).cpu()
    assert out.nonzero().tolist() == [[1, 0], [2, 1]]


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales_of_any_sign(dev, scale):
    check_attention(dev, [45], [1], 4, 2, 64, 32, F16, scale=scale)
    check_attention(dev, [140], [98], 4, 2, 32, 32, BF16, scale=scale)


# ---- rows in and out ----------------------------------------------------------------------------------------------------------------------------
def rows_like(shape, seed, dtype):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed))
    flat = x.view(-1)
    flat[::53] = 0
    flat[7::101] *= 300
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim,page,lens,news", [(64, 32, [1], [1]), (128, 64, [100, 31, 0, 33], [3, 31, 0, 1]), (80, 128, [40, 40], [40, 39]), (8, 32, [33], [2]),
                                                (112, 32, [65], [34]), (256, 32, [3], [3]), (160, 256, [20], [9])])
def test_append_stores_the_format_and_nothing_else(dev, dim, page, lens, news, dtype):
    heads = 2
    c = Cache(dim, lens, heads, dim, page)
    total = sum(news)
    k, v = rows_like((total, heads, dim), 1, dtype), rows_like((total, heads, dim), 2, dtype)
    pages, table, n = c.on(dev)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=dev)
    ops.kv4_append(k.to(dev), v.to(dev), pages, table, n, cu, max(news), page_tokens=page)
    at, values = 0, []
    for b, m in enumerate(news):
        for i in range(m):
            for half, x in ((0, k), (1, v)):
                codes, scales = quantize(x[at].float().numpy())
                for h in range(heads):
                    c.put(b, lens[b] - m + i, h, half, codes[h], scales[h])
                val = (codes.reshape(heads, -1, 32).astype(np.float64) - 8) * scales.astype(np.float64)[..., None]
                values.append(val.reshape(heads, -1)[:, :dim])
            at += 1
    assert np.array_equal(pages.cpu().numpy(), c.pages)   # every other byte of every page as it was
    for out in (F32, F16, BF16):
        kr, vr = ops.kv4_read(pages, table, n, cu, max(news), total, n_head_kv=heads, head_dim=dim, page_tokens=page, dtype=out)
        want = torch.from_numpy(np.array(values)).to(out)   # f16(d) * (code - 8) is exact in f32
        assert torch.equal(kr.cpu(), want[0::2]) and torch.equal(vr.cpu(), want[1::2])
    # against the rows themselves: half a step of the group, a whole one where the code was cut at 15; plus d's rounding
    err = (torch.from_numpy(np.array(values)[0::2]) - k.double()).abs()
    step = torch.nn.functional.pad(k.double(), (0, 32 * groups(dim) - dim)).unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)[..., :dim] / 8
    assert (err <= step * (1 + 8 * 2.0**-11) + 8 * 2.0**-25).all()


def test_append_of_strided_rows_and_of_rows_before_the_start(dev):
    big = rows_like((6, 64, 5), 1, F16)
    k = big.permute(2, 0, 1)[:, 1:3]                     # [5, 2, 64], no stride of 1 but one
    v = rows_like((5, 2, 128), 2, F32)[..., ::2]
    pages = {}
    for name, (kk, vv) in {"views": (k, v), "copies": (k.contiguous(), v.contiguous())}.items():
        c = Cache(9, [40], 2, 64, 32)
        p, table, n = c.on(dev)
        kd = big.to(dev).permute(2, 0, 1)[:, 1:3] if name == "views" else kk.to(dev)
        vd = rows_like((5, 2, 128), 2, F32).to(dev)[..., ::2] if name == "views" else vv.to(dev)
        ops.kv4_append(kd, vd, p, table, n, None, 5, page_tokens=32)
        pages[name] = p
    assert torch.equal(pages["views"], pages["copies"])
    # five rows, two tokens: the last two rows are theirs
    c = Cache(9, [2], 2, 64, 32)
    p, table, n = c.on(dev)
    ops.kv4_append(k.contiguous().to(dev), v.contiguous().to(dev), p, table, n, None, 5, page_tokens=32)
    kr, vr = ops.kv4_read(p, table, n, None, 5, 5, n_head_kv=2, head_dim=64, page_tokens=32)
    full, tf, nf = Cache(9, [40], 2, 64, 32).on(dev)
    ops.kv4_append(k.contiguous().to(dev), v.contiguous().to(dev), full, tf, nf, None, 5, page_tokens=32)
    kf, vf = ops.kv4_read(full, tf, nf, None, 5, 5, n_head_kv=2, head_dim=64, page_tokens=32)
    assert (kr[:3] == 0).all() and (vr[:3] == 0).all() and torch.equal(kr[3:], kf[3:]) and torch.equal(vr[3:], vf[3:])


def test_append_skips_pages_that_are_absent(dev):
    c = Cache(9, [70], 1, 64, 32)
    p, table, n = c.on(dev)
    old = p.clone()
    for bad in (-1, c.n_pages, 2**31 - 1):
        table[0, 1] = bad
        k = rows_like((40, 1, 64), 1, F16).to(dev)
        ops.kv4_append(k, k, p, table, n, None, 40, page_tokens=32)
        kr, vr = ops.kv4_read(p, table, n, None, 40, 40, n_head_kv=1, head_dim=64, page_tokens=32)
        # positions 30, 31 | 32 .. 63 absent | 64 .. 69
        assert (kr[2:34] == 0).all() and (vr[2:34] == 0).all() and not (kr[:2] == 0).all() and not (kr[34:] == 0).all()
    untouched = [i for i in range(c.n_pages) if i not in (int(table[0, 0]), int(table[0, 2]))]
    assert torch.equal(p[untouched], old[untouched])
    n[0] = 200   # past the table's width: nothing to write there
    before = p.clone()
    ops.kv4_append(k, k, p, table, n, None, 40, page_tokens=32)
    assert torch.equal(before, p)


def test_extremes_of_the_format(dev):
    """zeros, values too small for the scale, ties for the largest magnitude, values beyond f16, infinities"""
    x = torch.zeros((6, 1, 32))
    x[1, 0, 3] = 1e-9
    x[2, 0, 2], x[2, 0, 5] = 4.0, -4.0
    x[3, 0, 2], x[3, 0, 5] = -4.0, 4.0
    x[4, 0, 0], x[4, 0, 1] = 1e30, -7e4
    x[5, 0, 0], x[5, 0, 1] = float("-inf"), 1.0
    c = Cache(1, [6], 1, 32, 32)
    p, table, n = c.on(dev)
    ops.kv4_append(x.to(dev), x.to(dev), p, table, n, None, 6, page_tokens=32)
    for got in ops.kv4_read(p, table, n, None, 6, 6, n_head_kv=1, head_dim=32, page_tokens=32, dtype=F32):
        got = got.cpu()[:, 0]
        assert (got[0] == 0).all() and (got[1] == 0).all()
        assert got[2, 2] == 4 and got[2, 5] == -3.5 and got[3, 2] == -4 and got[3, 5] == 3.5
        assert got[4, 0] == 65504 and got[4, 1] == -65504 * 7 / 8 and got[5, 0] == -65504 and got[5, 1] == 0


# ---- pages --------------------------------------------------------------------------------------------------------------------------------------
class Book:
    """The bookkeeping, one page at a time."""

    def __init__(self, table, lens, refs, page):
        self.table, self.lens, self.refs, self.page = [list(r) for r in table], list(lens), list(refs), page

    def entries(self, s):
        return min(-(-max(self.lens[s], 0) // self.page), len(self.table[s]))

    def drop(self, s):
        for e in range(self.entries(s)):
            if 0 <= self.table[s][e] < len(self.refs):
                self.refs[self.table[s][e]] -= 1

    def fork(self, parents, keep=None):
        width = len(self.table[0]) if self.table else 0
        rows = []
        lens = [max(self.lens[p], 0) if 0 <= p < len(self.lens) else 0 for p in parents]
        lens = lens if keep is None else [max(min(n, k), 0) for n, k in zip(lens, keep)]
        for p, m in zip(parents, lens):
            ok = 0 <= p < len(self.lens)
            n = min(-(-m // self.page), width) if ok else 0
            rows.append((self.table[p][:n] if ok else []) + [-1] * (width - n))
            for e in rows[-1]:
                if 0 <= e < len(self.refs):
                    self.refs[e] += 1
        for s in range(len(self.lens)):
            self.drop(s)
        self.lens = lens
        self.table = rows

    def reserve(self, add, pool):
        table, lens, refs = [list(r) for r in self.table], list(self.lens), list(self.refs)
        want, copies, over = 0, [], False
        free = [i for i, r in enumerate(refs) if r == 0]
        wanted = []
        for s, a in enumerate(add):
            if a <= 0:
                continue
            n = max(lens[s], 0)
            first, last = n // self.page, -(-(n + a) // self.page)
            if last > len(table[s]):
                over = True
                continue
            if n % self.page:
                tail = table[s][first]
                if not 0 <= tail < len(refs):
                    wanted.append((s, first, -1))
                elif refs[tail] > 1:
                    refs[tail] -= 1
                    wanted.append((s, first, tail))
                first += 1
            wanted += [(s, e, -1) for e in range(first, last)]
            lens[s] = n + a
        if over:
            return -1
        if len(wanted) > len(free):
            return len(wanted) - len(free)
        for (s, e, src), p in zip(wanted, free):
            table[s][e] = p
            refs[p] = 1
            if src >= 0:
                copies.append((src, p))
        for src, p in copies:
            pool[:, p] = pool[:, src]
        self.table, self.lens, self.refs = table, lens, refs
        return 0

    def compact(self, pool):
        used = [i for i, r in enumerate(self.refs) if r > 0]
        mark = len(used)
        holes = [i for i in range(mark) if self.refs[i] <= 0]
        to = {p: p for p in used}
        to.update(zip([p for p in used if p >= mark], holes))
        old = pool.copy()
        refs = [0] * len(self.refs)
        for p, q in to.items():
            pool[:, q] = old[:, p]
            refs[q] = self.refs[p]
        self.table = [[to.get(e, -1) if 0 <= e < len(self.refs) else e for e in r] for r in self.table]
        self.refs = refs
        return mark


def a_batch(seed, n_seq, most, page, n_pages, width, shared=True):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, most + 1, n_seq)
    table, refs, free = np.full((n_seq, width), -1, np.int32), np.zeros(n_pages, np.int32), list(rng.permutation(n_pages))
    for s in range(n_seq):
        if shared and s and rng.random() < 0.5:
            o = int(rng.integers(0, s))
            lens[s] = lens[o]
            table[s] = table[o]
            refs[table[o][table[o] >= 0]] += 1
            continue
        for e in range(-(-int(lens[s]) // page)):
            table[s, e] = free.pop()
            refs[table[s, e]] = 1
    return table, lens.astype(np.int32), refs


def same(got, book, short=None):
    table, lens, refs = got[:3]
    assert table.cpu().tolist() == book.table and lens.cpu().tolist() == book.lens and refs.cpu().tolist() == book.refs


@pytest.mark.parametrize("seed", range(8))
def test_a_run_of_forks_reservations_and_compactions(dev, seed):
    """as a batch of beams lives: fork, make room, free, compact — the tables and every byte of the pool against the book, page for page"""
    rng = np.random.default_rng(100 + seed)
    page, n_seq = [32, 48, 1, 64][seed % 4], [3, 9, 1, 17][seed % 4]
    width = 6 if page > 1 else 40
    n_pages = n_seq * width + 3
    table, lens, refs = a_batch(seed, n_seq, page * width // 2, page, n_pages, width)
    pool = rng.integers(0, 256, (2, n_pages, 48), dtype=np.uint8)
    book = Book(table.tolist(), lens.tolist(), refs.tolist(), page)
    t, n, r, p = (torch.from_numpy(x.copy()).to(dev) for x in (table, lens, refs, pool))
    for step in range(5):
        parents = rng.integers(-1, len(book.lens) + 1, n_seq).astype(np.int32)
        keep = rng.integers(-1, 2 * max(book.lens) + 2, n_seq).astype(np.int32) if step % 2 else None
        book.fork(parents.tolist(), None if keep is None else keep.tolist())
        t, n, r = ops.kv_fork(t, n, r, torch.from_numpy(parents).to(dev), page_tokens=page, keep=None if keep is None else torch.from_numpy(keep).to(dev))
        same((t, n, r), book)
        add = rng.integers(-1, page + 2, n_seq).astype(np.int32)
        before = (t, n, r)
        want = book.reserve(add.tolist(), pool)
        t, n, r, short = ops.kv_reserve(p, t, n, r, torch.from_numpy(add).to(dev), page_tokens=page)
        assert int(short) == want
        same((t, n, r), book)
        if want:
            assert all(torch.equal(x, y) for x, y in zip((t, n, r), before))
        if step % 2:
            used = book.compact(pool)
            t, r, mark = ops.kv_compact(p, t, r)
            assert int(mark) == used
            same((t, n, r), book)
            # what lies behind the mark is nobody's
            assert np.array_equal(p.cpu().numpy()[:, :used], pool[:, :used])
            pool = p.cpu().numpy().copy()
        else:
            assert np.array_equal(p.cpu().numpy(), pool)


def test_reserve_says_what_is_missing(dev):
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    pages = torch.zeros((3, 16), dtype=torch.uint8, device=dev)
    table, lens, refs = i([0, -1, -1], [1, -1, -1]), i(4, 4), i(1, 1, 0)
    for add, want in (((1, 0), 0), ((1, 1), 1), ((8, 8), 3), ((0, 9), -1), ((0, 0), 0), ((-5, -1), 0)):
        t, n, r, short = ops.kv_reserve(pages, table, lens, refs, i(*add), page_tokens=4)
        assert int(short) == want
        if want:
            assert torch.equal(t, table) and torch.equal(n, lens) and torch.equal(r, refs)
    # all the holders of a shared last page write: the last of them keeps it
    t, n, r, short = ops.kv_reserve(pages, i([0, -1], [0, -1]), i(2, 2), i(2, 0, 0), i(1, 1), page_tokens=4)
    assert int(short) == 0 and t.tolist() == [[1, -1], [0, -1]] and r.tolist() == [1, 1, 0]


def test_many_sequences_and_pages(dev):
    """more than one round of the planning workgroup, for the sequences as for the pages"""
    rng = np.random.default_rng(5)
    n_seq, page = (2500, 8) if dev.type == "cuda" else (1100, 8)
    n_pages = 4 * n_seq + 5000
    table, lens, refs = a_batch(5, n_seq, 20, page, n_pages, 5)
    pool = rng.integers(0, 256, (1, n_pages, 16), dtype=np.uint8)
    book = Book(table.tolist(), lens.tolist(), refs.tolist(), page)
    t, n, r, p = (torch.from_numpy(x.copy()).to(dev) for x in (table, lens, refs, pool))
    parents = np.sort(rng.integers(0, n_seq, n_seq)).astype(np.int32)
    book.fork(parents.tolist())
    t, n, r = ops.kv_fork(t, n, r, torch.from_numpy(parents).to(dev), page_tokens=page)
    add = rng.integers(0, 12, n_seq).astype(np.int32)
    want = book.reserve(add.tolist(), pool)
    t, n, r, short = ops.kv_reserve(p, t, n, r, torch.from_numpy(add).to(dev), page_tokens=page)
    assert int(short) == want == 0
    same((t, n, r), book)
    assert np.array_equal(p.cpu().numpy(), pool)
    used = book.compact(pool)
    t, r, mark = ops.kv_compact(p, t, r)
    same((t, n, r), book)
    assert int(mark) == used and np.array_equal(p.cpu().numpy()[:, :used], pool[:, :used])


def test_fork_of_nothing_and_into_nothing(dev):
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    t, n, r = ops.kv_fork(i([0, 1]), i(5), i(1, 1, 0), torch.zeros(0, dtype=torch.int32, device=dev), page_tokens=4)
    assert t.shape == (0, 2) and n.shape == (0,) and r.tolist() == [0, 0, 0]
    t, n, r = ops.kv_fork(i([0, 1]), i(5), i(1, 1, 0), i(-1, 7, -2**31), page_tokens=4)
    assert t.tolist() == [[-1, -1]] * 3 and n.tolist() == [0, 0, 0] and r.tolist() == [0, 0, 0]


# ---- the operators together ---------------------------------------------------------------------------------------------------------------------
def test_a_conversation_forks_and_its_branches_go_their_own_ways(dev):
    """a prompt is stored, the sequence forks in three, each branch gets tokens of its own: every branch attends to the prompt and to its own tokens only"""
    heads, H, dim, page, width = 2, 4, 64, 32, 6
    n_pages = 14
    pages = torch.zeros((n_pages, ops.kv4_page_bytes(heads, dim, page)), dtype=torch.uint8, device=dev)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table, lens, refs = i([[-1] * width]), i([0]), i([0] * n_pages)
    history = [[]]
    rng = torch.Generator().manual_seed(0)

    def step(news):
        nonlocal table, lens, refs
        table, lens, refs, short = ops.kv_reserve(pages, table, lens, refs, i(news), page_tokens=page)
        assert int(short) == 0
        total = sum(news)
        k, v = (torch.randn((total, heads, dim), generator=rng).to(F16) for _ in range(2))
        q = torch.randn((total, H, dim), generator=rng).to(F16)
        cu = i([0] + np.cumsum(news).tolist())
        ops.kv4_append(k.to(dev), v.to(dev), pages, table, lens, cu, max(news), page_tokens=page)
        out = ops.kv4_attention(q.to(dev), pages, table, lens, cu, max(news), n_head_kv=heads, page_tokens=page).double().cpu().numpy()
        at = 0
        for b, m in enumerate(news):
            for j in range(at, at + m):
                history[b] = history[b] + [(k[j].float().numpy(), v[j].float().numpy())]
            kv = []
            for half in (0, 1):
                codes, scales = quantize(np.array([x[half] for x in history[b]]))
                n = len(history[b])
                kv.append(((codes.astype(np.float64) - 8).reshape(n, heads, 2, 32) * scales.astype(np.float64)[..., None]).reshape(n, heads, 64))
            want, mag, err = attention64(q[at:at + m].double().numpy(), kv, heads, dim**-0.5, (2.0**-11, 0))
            assert (np.abs(out[at:at + m] - want) <= mag * (2.0**-10 + 2 * np.expm1(err)[..., None]) * 1.01 + np.abs(want) * 2.0**-11 * 1.01).all()
            at += m

    step([41])
    table, lens, refs = ops.kv_fork(table, lens, refs, i([0, 0, 0]), page_tokens=page)
    history = [history[0]] * 3
    for news in ([1, 1, 1], [1, 2, 30], [3, 1, 1]):
        step(news)
    table, lens, refs = ops.kv_fork(table, lens, refs, i([2, 2, -1]), page_tokens=page)   # the last branch twice, one free place
    history = [history[2], history[2], []]
    table, refs, used = ops.kv_compact(pages, table, refs)
    assert int(used) == int((refs > 0).sum()) and bool((refs[:int(used)] > 0).all())
    for news in ([1, 1, 9], [2, 33, 1]):
        step(news)


# ---- refusals -----------------------------------------------------------------------------------------------------------------------------------
def test_refusals(dev):
    c = Cache(1, [40, 9], 2, 64, 32)
    p, table, n = c.on(dev)
    cu = torch.tensor([0, 2, 3], dtype=torch.int32, device=dev)
    q = torch.zeros((3, 4, 64), dtype=F16, device=dev)
    k = torch.zeros((3, 2, 64), dtype=F16, device=dev)
    old = p.clone()
    att = lambda **x: ops.kv4_attention(**{**dict(q=q, pages=p, table=table, lens=n, cu=cu, max_rows=2, n_head_kv=2, page_tokens=32), **x})  # noqa: E731
    app = lambda **x: ops.kv4_append(**{**dict(k=k, v=k, pages=p, table=table, lens=n, cu=cu, max_rows=2, page_tokens=32), **x})  # noqa: E731
    for call, bad in [(att, dict(page_tokens=48)), (att, dict(page_tokens=0)), (att, dict(n_head_kv=3)), (att, dict(n_head_kv=0)), (att, dict(cu=None)),
                      (att, dict(cu=cu[:2])), (att, dict(lens=n[:1])), (att, dict(pages=p[:, :-16])), (att, dict(pages=p.view(-1))), (att, dict(max_rows=-1)),
                      (att, dict(table=table[:, ::2])), (att, dict(q=q[..., :60])), (att, dict(q=q[0])), (att, dict(out=q[:2])), (att, dict(table=table[0])),
                      (app, dict(v=k[:2])), (app, dict(k=k[..., :32])), (app, dict(page_tokens=64)), (app, dict(cu=None))]:
        with pytest.raises(ValueError):
            call(**bad)
    for call, bad in [(att, dict(q=q.double())), (att, dict(q=q.int())), (att, dict(table=table.long())), (att, dict(lens=n.float())), (att, dict(pages=p.short())),
                      (att, dict(out=q.double())), (app, dict(k=k.int())), (app, dict(pages=None)), (app, dict(table=None))]:
        with pytest.raises(TypeError):
            call(**bad)
    shifted = torch.zeros(p.numel() + 16, dtype=torch.uint8, device=dev)[8:8 + p.numel()].view(p.shape)
    with pytest.raises(ValueError, match="aligned"):
        att(pages=shifted)
    for bad in (0, 4, 12, 264, -8):
        with pytest.raises(ValueError):
            ops.kv4_page_bytes(2, bad, 32)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    t, l, r, a = i([0, 1]), i(5), i(1, 1, 0), i(1)
    pool = torch.zeros((3, 16), dtype=torch.uint8, device=dev)
    for call in (lambda: ops.kv_fork(t, l, r, i(0), page_tokens=0), lambda: ops.kv_fork(t, i(5, 5), r, i(0), page_tokens=4), lambda: ops.kv_fork(t, l, r, i(0), page_tokens=4, keep=i(1, 2)), lambda: ops.kv_reserve(pool[:2], t, l, r, a, page_tokens=4),
                 lambda: ops.kv_reserve(pool, t, l, r, i(1, 1), page_tokens=4), lambda: ops.kv_reserve(torch.zeros((3, 8), dtype=torch.uint8, device=dev), t, l, r, a, page_tokens=4),
                 lambda: ops.kv_reserve(pool.t(), t, l, r, a, page_tokens=4), lambda: ops.kv_compact(pool, t[0], r), lambda: ops.kv_compact(pool, t, i([1, 1, 0]))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.kv_fork(t.long(), l, r, i(0), page_tokens=4), lambda: ops.kv_fork(t, l, r, None, page_tokens=4), lambda: ops.kv_compact(pool, t, r.float())):
        with pytest.raises(TypeError):
            call()
    assert torch.equal(p, old)
    # nothing to do is not an error
    none = torch.zeros((0, 2, 64), dtype=F16, device=dev)
    zero = torch.zeros(3, dtype=torch.int32, device=dev)
    app(k=none, v=none, cu=zero, max_rows=0)
    assert att(q=q[:0], cu=zero, max_rows=0).shape == (0, 4, 64)


def test_no_host_tensors(hip_lib):
    ops.load(hip_lib)
    try:
        x = torch.zeros((1, 2, 64), dtype=F16)
        i = torch.zeros((1, 1), dtype=torch.int32)
        with pytest.raises(ValueError, match="GPU memory"):
            ops.kv4_append(x, x, torch.zeros((1, ops.kv4_page_bytes(2, 64, 32)), dtype=torch.uint8), i, i[0], None, 1, page_tokens=32)
        with pytest.raises(ValueError, match="GPU memory"):
            ops.kv_compact(x, i, i[0])
    finally:
        ops._lib = None


def test_c_interface(hip_lib):
    """the header, the Python table and the library agree; null pointers and overlapping outputs come back as errors (nothing is launched)"""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ctransformers_amd_ops.h")).read(), flags=re.S)
    assert sorted(set(re.findall(r"\b(ctamd_\w+)\s*\(", text))) == sorted(ops.ABI)
    lib = ops.load(hip_lib)
    try:
        assert lib.ctamd_kv4_append(None, None, None, None) == -1 and b"null cache" in lib.ctamd_ops_error()
        c = ops.CACHE.pack(0, 0, 0, 0, 36864, 0, 1, 1, 1, 1, 2, 64, 32, 1)
        assert lib.ctamd_kv4_append(c, None, None, None) == -1 and b"null rows" in lib.ctamd_ops_error()
        assert lib.ctamd_kv_fork(None, None, None, 0, None) == -1 and lib.ctamd_kv_reserve(None, None, None, 0, 0, 0, None, None, None) == -1
        t = ops.TABLES.pack(4096, 8192, 12288, 4096, 16384, 20480, 1, 2, 3, 4)
        assert lib.ctamd_kv_fork(t, 24576, None, 1, None) == -1 and b"overlaps an input" in lib.ctamd_ops_error()
        assert lib.ctamd_kv_compact(ops.TABLES.pack(4096, 0, 12288, 32768, 0, 20480, 1, 2, 3, 1), 16, 1, 48, 16, None, None, None) == -1
    finally:
        ops._lib = None


# ---- more sequences than a wave has lanes, large pools, graphs, streams ----------------------------------------------------------------------------
def test_more_sequences_than_lanes_share_the_line(dev):
    """70 sequences, some without rows or tokens, in a table wide enough that the work is divided"""
    rng = np.random.default_rng(3)
    lens = [int(x) for x in rng.integers(0, 70, 70)]
    lens[65] = 300
    news = [int(min(x, n)) if n else int(x == 1) for x, n in zip(rng.integers(0, 3, 70), lens)]
    check_attention(dev, lens, news, 2, 1, 32, 32, F16, seed=9, width=12)


@pytest.mark.gpu
def test_pages_beyond_4_gib(hip_lib):
    """a pool of 5 GB: rows stored, read, attended to and copied in its last pages equal those in a small pool"""
    ops.load(hip_lib)
    dev = torch.device("cuda:0")
    width = ops.kv4_page_bytes(8, 128, 256)
    n_pages = 5 * 2**30 // width
    big, small = torch.zeros((n_pages, width), dtype=torch.uint8, device=dev), torch.zeros((4, width), dtype=torch.uint8, device=dev)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    k, v = (torch.randn((500, 8, 128), device=dev).half() for _ in range(2))
    q = torch.randn((500, 16, 128), device=dev).half()
    outs = []
    for pages, table in ((big, i([n_pages - 1, n_pages - 3])), (small, i([1, 0]))):
        ops.kv4_append(k, v, pages, table, i(500), None, 500, page_tokens=256)
        rows = ops.kv4_read(pages, table, i(500), None, 500, 500, n_head_kv=8, head_dim=128, page_tokens=256)
        one = ops.kv4_attention(q[-1:], pages, table, i(500), None, 1, n_head_kv=8, page_tokens=256)
        outs.append(rows + (ops.kv4_attention(q, pages, table, i(500), None, 500, n_head_kv=8, page_tokens=256), one))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    # the partly filled last page is shared: making room copies it, from the pool's end to its start
    refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
    refs[n_pages - 1], refs[n_pages - 3] = 1, 2
    t, n, r, short = ops.kv_reserve(big, i([n_pages - 1, n_pages - 3]), i(500), refs, i(3), page_tokens=256)
    assert int(short) == 0 and t.tolist() == [[n_pages - 1, 0]] and torch.equal(big[0], big[n_pages - 3])
    used = ops.kv_compact(big, t, r)
    assert int(used[2]) == 3 and used[0].tolist() == [[2, 0]] and torch.equal(big[1], big[0])   # pages n - 3 and n - 1 go to the holes 1 and 2


@pytest.mark.gpu
@pytest.mark.parametrize("news,width", [(1, 2), (1, 40), (70, 8)])
def test_captured_and_replayed(hip_lib, news, width):
    """append, attention, fork and room in one graph, two graphs at once, on a stream of their own: every replay equals the eager run on its inputs"""
    ops.load(hip_lib)
    dev = torch.device("cuda:0")
    heads, H, dim, page, B = 2, 8, 64, 32, 3
    n_pages = B * width + 4

    def state(seed):
        g = torch.Generator().manual_seed(seed)
        table = torch.randperm(n_pages, generator=g)[:B * width].view(B, width).int().to(dev)
        lens = torch.randint(news, width * page - 10, (B,), generator=g).int().clamp(min=news).to(dev)
        refs = torch.zeros(n_pages, dtype=torch.int32)
        refs[table.cpu().flatten().long()] = 1
        x = [torch.randn((B * news, h, dim), generator=g).half().to(dev) for h in (H, heads, heads)]
        return [torch.randint(0, 2, (n_pages, ops.kv4_page_bytes(heads, dim, page)), generator=g, dtype=torch.uint8).to(dev), table, lens, refs.to(dev),
                torch.randint(-1, B, (B,), generator=g).int().to(dev)] + x

    cu = (torch.arange(B + 1) * news).int().to(dev)

    def run(pages, table, lens, refs, parents, q, k, v):
        ops.kv4_append(k, v, pages, table, lens, cu, news, page_tokens=page)
        out = ops.kv4_attention(q, pages, table, lens, cu, news, n_head_kv=heads, page_tokens=page)
        t, n, r = ops.kv_fork(table, lens, refs, parents, page_tokens=page)
        t, n, r, short = ops.kv_reserve(pages, t, n, r, torch.ones_like(n), page_tokens=page)
        return [out, t, n, r, short, pages]

    stream = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        s = state(0)
        with torch.cuda.stream(stream):
            run(*[x.clone() for x in s])
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = run(*s)
        graphs.append((graph, s, outs, torch.cuda.Stream()))
    for seed in range(1, 7):
        wants = []
        for k, (graph, s, outs, _) in enumerate(graphs):
            new = state(10 * seed + k)
            for x, y in zip(s, new):
                x.copy_(y)
            wants.append([x.clone() for x in run(*new)])
        torch.cuda.synchronize()
        for graph, s, outs, mine in graphs:
            with torch.cuda.stream(mine):
                graph.replay()
        torch.cuda.synchronize()
        for (graph, s, outs, _), want in zip(graphs, wants):
            assert all(torch.equal(x, y) for x, y in zip(outs, want))


@pytest.mark.gpu
def test_same_bits_every_time(hip_lib):
    ops.load(hip_lib)
    dev = torch.device("cuda:0")
    for news, width in ((1, 60), (40, 30)):
        c = Cache(4, [900, 30, 511], 2, 64, 32, extra_width=width)
        c.fill(5)
        pages, table, n = c.on(dev)
        q = torch.randn((3 * news, 16, 64), device=dev).half()
        cu = torch.tensor([0, news, 2 * news, 3 * news], dtype=torch.int32, device=dev)
        first = ops.kv4_attention(q, pages, table, n, cu, news, n_head_kv=2, page_tokens=32)
        for _ in range(5):
            assert torch.equal(first, ops.kv4_attention(q, pages, table, n, cu, news, n_head_kv=2, page_tokens=32))
