"""The 4-bit paged KV cache (ctransformers_amd/ops.py, csrc/engine_kv4.h) at the edges of what its calls accept."""
import ctypes
import math
import time

import numpy as np
import pytest
import torch

from ctransformers_amd import ops
from test_kv4 import Cache, attention64, dev  # noqa: F401  (the fixture)


def ints(dev, *x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def c_attention(dev, q, pages, table, lens, cu, rows, heads_kv, page, out, width, stride):
    """ctamd_kv4_attention with a table of `width` entries that lie where `table` begins, and what it returns"""
    total, H, dim = q.shape
    types = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
    c = ops.CACHE.pack(pages.data_ptr(), table.data_ptr(), lens.data_ptr(), cu.data_ptr(), pages.stride(0), pages.shape[0], stride, width, lens.shape[0], total, heads_kv, dim, page, rows)
    row = lambda x: ops.ROWS.pack(x.data_ptr(), *x.stride(), types[x.dtype])  # noqa: E731
    n = ops._lib.ctamd_kv4_attention_ws(c, H)
    ws = torch.empty(max(n, 1), dtype=torch.float32, device=dev)
    code = ops._lib.ctamd_kv4_attention(c, H, row(q), row(out), dim**-0.5, ws.data_ptr(), n, ops._stream(dev.index) if dev.type == "cuda" else None)
    if dev.type == "cuda":
        torch.cuda.synchronize()
    return code


# ---- attention ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("news", [1, 20, 100])
def test_a_table_without_entries(dev, news):
    """the memory behind it names a page: it is no entry of the table, and no row sees anything"""
    c = Cache(1, [40], 1, 64, 32, extra_width=3)
    c.fill(2)
    pages, table, lens = c.on(dev)
    q = torch.ones((news, 2, 64), dtype=torch.float16, device=dev)
    out = torch.full_like(q, 7)
    assert c_attention(dev, q, pages, table, lens, ints(dev, 0, news), news, 1, 32, out, 0, 4) == 0
    assert (out == 0).all()


@pytest.mark.parametrize("n_pages", [0, 3])
def test_sequences_that_have_no_pages_yet(dev, n_pages):
    """a table of no columns is an empty tensor, whose address is null: rows are not stored, read back as zeros and see nothing"""
    pages = torch.full((n_pages, ops.kv4_page_bytes(2, 64, 32)), 5, dtype=torch.uint8, device=dev)
    table, lens, cu = torch.empty((2, 0), dtype=torch.int32, device=dev), ints(dev, 0, 3), ints(dev, 0, 0, 3)
    x = torch.ones((3, 2, 64), dtype=torch.float16, device=dev)
    old = pages.clone()
    ops.kv4_append(x, x, pages, table, lens, cu, 3, page_tokens=32)
    assert torch.equal(pages, old)
    for rows in ops.kv4_read(pages, table, lens, cu, 3, 3, n_head_kv=2, head_dim=64, page_tokens=32):
        assert (rows == 0).all()
    assert (ops.kv4_attention(x, pages, table, lens, cu, 3, n_head_kv=2, page_tokens=32) == 0).all()


def test_a_pool_of_no_pages_still_needs_lengths(dev):
    """the C interface: no page is touched, but the sequences' lengths are read all the same; null ones are an error, not an access"""
    x = torch.ones((1, 2, 64), dtype=torch.float16, device=dev)
    row, table = ops.ROWS.pack(x.data_ptr(), *x.stride(), 0), ints(dev, 0)
    for t, lens in ((table.data_ptr(), 0), (0, table.data_ptr())):
        c = ops.CACHE.pack(0, t, lens, 0, 36864, 0, 1, 1, 1, 1, 2, 64, 32, 1)
        assert ops._lib.ctamd_kv4_read(c, row, row, None) == -1 and b"null cache pointer" in ops._lib.ctamd_ops_error()
        assert ops._lib.ctamd_kv4_attention(c, 2, row, row, 1.0, None, 0, None) == -1 and b"null cache pointer" in ops._lib.ctamd_ops_error()
        assert ops._lib.ctamd_kv4_append(c, row, row, None) == 0   # (nothing to do)


def test_rows_between_sequences_are_left_as_they_are(dev):
    """cu that does not ascend (whose own rows are undefined): a row that no sequence holds is not joined from memory in front of another row's parts"""
    c = Cache(1, [600, 40, 600], 1, 32, 32, extra_width=8)
    c.fill(2)
    pages, table, lens = c.on(dev)
    q = torch.ones((9, 2, 32), dtype=torch.float16, device=dev)
    out = torch.full_like(q, 7)
    ops.kv4_attention(q, pages, table, lens, ints(dev, 7, 9, 2, 3), 2, n_head_kv=1, page_tokens=32, out=out)
    assert (out[[0, 1, 3, 4, 5, 6]] == 7).all()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 1e39])
def test_scales_that_are_no_numbers(dev, scale):
    """refused (a NaN used to give the mean of V); 1e39 is infinite as the float that it is passed as"""
    c = Cache(1, [40], 1, 32, 32)
    c.fill(2)
    pages, table, lens = c.on(dev)
    for news in (1, 40, 200):
        q = torch.ones((news, 1, 32), dtype=torch.float16, device=dev)
        out = torch.full_like(q, 7)
        with pytest.raises(ValueError, match="scale"):
            ops.kv4_attention(q, pages, table, lens, None, news, n_head_kv=1, page_tokens=32, scale=scale, out=out)
        assert (out == 7).all()


def far_rows(dev, news, big, scale, dtype, k_scale):
    """rows of magnitude `big` (times 1 .. 4), keys of k_scale: kv4_attention against the 64-bit formula, with the bound that test_kv4.py derives; the queries are exact
    as halves (few bits), but bf16's and float32's roundings to halves are allowed for all the same"""
    c = Cache(1, [40 + news], 1, 64, 32)
    c.fill(2, k_scale)
    q = (torch.randint(-3, 4, (news, 2, 64), generator=torch.Generator().manual_seed(4)).double() * big).to(dtype)
    assert q.isfinite().all() and (q.double().abs().max() >= 2 * big)
    pages, table, n = c.on(dev)
    got = ops.kv4_attention(q.to(dev), pages, table, n, None, news, n_head_kv=1, page_tokens=32, scale=scale, out=torch.empty(q.shape, dtype=torch.float32, device=dev)).double().cpu().numpy()
    want, mag, err = attention64(q.double().numpy(), c.values[0], 1, float(np.float32(scale)), (2.0**-11, 2.0**-25))
    assert err.max() < 0.1   # (the bound says something)
    assert (np.abs(got - want) <= mag * (2.0**-10 + 2 * np.expm1(err)[..., None]) * 1.01 + np.abs(want) * 2.0**-24 * 1.01).all()


@pytest.mark.parametrize("news", [1, 20, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_queries_at_the_ends_of_their_type(dev, dtype, news):
    """the largest values (beyond 2^127) with a small scale, subnormal ones with a large scale and large keys"""
    far_rows(dev, news, 2.0**126, 2.0**-129, dtype, 1.0)
    far_rows(dev, news, 2.0**-133, 2.0**120, dtype, 1024.0)
    if dtype == torch.float32:
        far_rows(dev, news, 2.0**-147, 1.5 * 2.0**127, dtype, 8192.0)


@pytest.mark.parametrize("scale", [1.0, -1.0, 3e38])
@pytest.mark.parametrize("news", [1, 20, 200])
@pytest.mark.parametrize("big", [2.0**12, 2.0**60, 2.0**126])
def test_scores_of_any_size(dev, big, news, scale, dtype=torch.float32, key=4096.0):
    """scores beyond 2^30, where a float's steps are larger than the range that exp2 has: the largest takes all, several that are equal share it"""
    width = 10                                       # (in parts too)
    c = Cache(1, [330 + news], 1, 32, 32, extra_width=width)
    pages, table, n = c.on(dev)
    total = 330 + news
    k = torch.zeros((total, 1, 32))
    k[:, 0, 0] = key
    k[:, 0, 1] = key * torch.randint(-7, 5, (total,), generator=torch.Generator().manual_seed(5)) / 8   # (exact: a group's largest is `key`, its step an eighth of it)
    k[[3, 77, 300], 0, 1] = -key if scale < 0 else key * 6 / 8
    k[[3, 77, 300], 0, 0] = -key if scale < 0 else key
    v = torch.randn((total, 1, 32), generator=torch.Generator().manual_seed(6))
    ops.kv4_append(k.to(dev), v.to(dev), pages, table, n, None, total, page_tokens=32)
    kr, vr = (x.double().cpu().numpy()[:, 0] for x in ops.kv4_read(pages, table, n, None, total, total, n_head_kv=1, head_dim=32, page_tokens=32, dtype=torch.float32))
    q = torch.zeros((news, 2, 32), dtype=dtype)
    q[..., 1] = big
    q[..., 0] = big / 4
    got = ops.kv4_attention(q.to(dev), pages, table, n, None, news, n_head_kv=1, page_tokens=32, scale=scale, out=torch.empty(q.shape, dtype=torch.float32, device=dev)).double().cpu().numpy()
    score = (0.25 * kr[:, 0] + kr[:, 1]) * (1 if scale > 0 else -1)   # times big |scale|: neighbours are 2^20 and more apart
    for i in range(news):
        see = total - news + i + 1
        top = score[:see] == score[:see].max()
        want, mag = vr[:see][top].mean(0), np.abs(vr[:see][top]).mean(0)
        assert (np.abs(got[i] - want) <= mag * 2.0**-10 * 1.01 + np.abs(want) * 2.0**-22).all(), i


@pytest.mark.parametrize("scale", [1e37, -3e38])
@pytest.mark.parametrize("news", [1, 20, 200])
def test_scores_of_any_size_from_halves(dev, news, scale):
    """float16 queries go into the products as they are"""
    test_scores_of_any_size(dev, 2.0**15, news, scale, torch.float16, 32768.0)


@pytest.mark.parametrize("news", [1, 20, 200])
@pytest.mark.parametrize("tail", [24.4, 25.2, 29.0, 35.5])
@pytest.mark.parametrize("total,parts", [(1024, 0), (1024, 1), pytest.param(60000, 0, marks=pytest.mark.gpu), pytest.param(60000, 1, marks=pytest.mark.gpu)])
def test_a_peak_and_a_long_flat_tail(dev, total, parts, tail, news):
    """One token takes all but 2^-tail a token of the weight, and its value is 0: the result is the tail.  Weights are halves, 2^11 times as large as beside a
    maximum of 1, so the smallest are rounded by 2^-25 2^-11 of the largest at most: sum |v| 2^-36 in the result, beside test_kv4.py's relative roundings (p and v as halves) and its
    error of a score.  parts: whether the table is wide enough for keys to be divided."""
    if total > 1024 and dev.type == "cpu":
        pytest.skip("GPU only (60 000 tokens)")
    x = torch.tensor(-tail * math.log(2)).half().float()             # (a row with one value has it exactly)
    for peak in (0, total // 2 + 5, total - news):                   # (every row sees it)
        pages = torch.zeros((-(-total // 64), ops.kv4_page_bytes(1, 32, 64)), dtype=torch.uint8, device=dev)
        table = torch.full((1, pages.shape[0] if parts or total > 1024 else 16), -1, dtype=torch.int32, device=dev)
        table[0, :pages.shape[0]] = torch.arange(pages.shape[0])
        if parts:
            table = torch.cat([table, torch.full((1, 200), -1, dtype=torch.int32, device=dev)], 1)
        k, v = torch.zeros((total, 1, 32)), torch.ones((total, 1, 32))
        k[:, 0, 0] = x
        k[peak, 0, 0] = v[peak] = 0
        n = ints(dev, total)
        ops.kv4_append(k.to(dev), v.to(dev), pages, table, n, None, total, page_tokens=64)
        q = torch.zeros((news, 1, 32), dtype=torch.float16)
        q[..., 0] = 1
        got = ops.kv4_attention(q.to(dev), pages, table, n, None, news, n_head_kv=1, page_tokens=64, scale=1.0, out=torch.empty(q.shape, dtype=torch.float32, device=dev)).double().cpu()
        see = torch.arange(total - news + 1, total + 1).double()[:, None, None]
        w = (see - 1) * math.exp(float(x))
        want = w / (1 + w)
        err = (32 + 8) * 2.0**-24 * abs(float(x)) + (4 * abs(float(x)) + 8) * 2.0**-23
        tol = want * (2 * 2.0**-11 + 2 * math.expm1(err)) * 1.01 + see * 2.0**-36 + want * 2.0**-24 * 1.01
        assert ((got - want).abs() <= tol).all(), (peak, float(((got - want).abs() / tol).max()))


@pytest.mark.parametrize("news", [1, 20, 200])
def test_results_in_the_queries_place(dev, news):
    c = Cache(1, [300 + news, 20], 2, 32, 32, extra_width=12)
    c.fill(2)
    pages, table, lens = c.on(dev)
    q = torch.randn((news + 3, 10, 32), generator=torch.Generator().manual_seed(1)).half().to(dev)
    att = lambda out: ops.kv4_attention(q, pages, table, lens, ints(dev, 0, news, news + 3), max(news, 3), n_head_kv=2, page_tokens=32, out=out)  # noqa: E731
    want = att(None)
    assert torch.equal(att(q), want)


def test_results_whose_rows_share_memory(dev):
    """refused, rows that lie between others are not"""
    c = Cache(1, [40], 1, 32, 32)
    c.fill(2)
    pages, table, lens = c.on(dev)
    q = torch.randn((5, 4, 32), generator=torch.Generator().manual_seed(1)).half().to(dev)
    att = lambda out: ops.kv4_attention(q, pages, table, lens, None, 5, n_head_kv=1, page_tokens=32, out=out)  # noqa: E731
    want = att(None)
    flat = torch.full((4000,), 7.0, dtype=torch.float16, device=dev)
    for size, stride in (((5, 4, 32), (0, 32, 1)), ((5, 4, 32), (128, 0, 1)), ((5, 4, 32), (64, 32, 1)), ((5, 4, 32), (128, 24, 1)), ((5, 4, 32), (16, 160, 1))):
        with pytest.raises(ValueError, match="share memory"):
            att(flat.as_strided(size, stride))
    assert (flat == 7).all()
    for stride in ((128, 32, 1), (40, 208, 1), (160, 40, 1), (700, 33, 1)):
        flat.fill_(7)
        assert torch.equal(att(flat.as_strided((5, 4, 32), stride)), want)
        assert int((flat != 7).sum()) <= 640
    row = lambda *s: ops.ROWS.pack(flat.data_ptr(), *s, 0)  # noqa: E731
    cache = ops.CACHE.pack(pages.data_ptr(), table.data_ptr(), lens.data_ptr(), 0, pages.stride(0), pages.shape[0], table.shape[1], table.shape[1], 1, 5, 1, 32, 32, 5)
    for k, v in ((row(0, 32, 1), row(32, 32, 1)), (row(32, 32, 1), row(16, 32, 1))):
        assert ops._lib.ctamd_kv4_read(cache, k, v, None) == -1 and b"share memory" in ops._lib.ctamd_ops_error()


def test_an_error_that_another_call_left(dev):
    """it is not this call's, and stays there for its owner"""
    pages, table, lens, refs = torch.zeros((2, ops.kv4_page_bytes(1, 32, 32)), dtype=torch.uint8, device=dev), ints(dev, [0, -1]), ints(dev, 1), ints(dev, 1, 0)
    x = torch.ones((1, 1, 32), device=dev)
    if dev.type == "cpu":
        word = ctypes.c_int.in_dll(ops._lib, "emu_last_error")
        leave, take = lambda: setattr(word, "value", 101), ops._lib.emu_get_last_error
    else:
        hip = ctypes.CDLL(next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line))
        leave, take = lambda: hip.hipSetDevice(10**6), hip.hipGetLastError
    parents = ints(dev, 0)
    for _ in range(2):   # (kernels are loaded, memory has been taken)
        ops.kv4_append(x, x, pages, table, lens, None, 1, page_tokens=32)
        out = ops.kv4_attention(x, pages, table, lens, None, 1, n_head_kv=1, page_tokens=32)
        ops.kv_fork(table, lens, refs, parents, page_tokens=32)
    take()
    leave()
    try:
        ops.kv4_append(x, x, pages, table, lens, None, 1, page_tokens=32)
        assert take() == 101
        leave()
        out = ops.kv4_attention(x, pages, table, lens, None, 1, n_head_kv=1, page_tokens=32)
        ops.kv_fork(table, lens, refs, parents, page_tokens=32)
    finally:
        take()
    assert (out == 1).all()


def test_a_gradient_is_not_lost_in_silence(dev):
    c = Cache(1, [40], 1, 32, 32)
    c.fill(2)
    pages, table, lens = c.on(dev)
    old = pages.clone()
    x = torch.ones((1, 1, 32), device=dev)
    g = torch.ones((1, 1, 32), device=dev, requires_grad=True)
    att = lambda q, out=None: ops.kv4_attention(q, pages, table, lens, None, 1, n_head_kv=1, page_tokens=32, out=out)  # noqa: E731
    app = lambda k, v: ops.kv4_append(k, v, pages, table, lens, None, 1, page_tokens=32)  # noqa: E731
    for call in (lambda: att(g), lambda: att(x, g), lambda: att(g * 2), lambda: app(g, x), lambda: app(x, g)):
        with pytest.raises(ValueError, match="gradient"):
            call()
    assert torch.equal(pages, old)
    want = att(x)
    assert torch.equal(att(g.detach()), want)
    with torch.no_grad():
        assert torch.equal(att(g), want)
        app(g, x)


@pytest.mark.parametrize("news,most", [(7, 3), (40, 1), (40, 33), (300, 130), (200, 50)])
def test_rows_beyond_max_rows_are_not_processed(dev, news, most):
    """a sequence with more rows than the call allows: the first of them are those of the whole, the others' places are left as they are"""
    for width in (1, 10):
        c = Cache(1, [320 + news, 5], 1, 32, 32, extra_width=width)
        c.fill(2)
        cu = ints(dev, 0, news, news + 2)
        k, v = (torch.randn((news + 2, 1, 32), generator=torch.Generator().manual_seed(i)).half().to(dev) for i in (3, 4))
        whole, table, lens = c.on(dev)
        part, old = whole.clone(), whole.clone()
        ops.kv4_append(k, v, whole, table, lens, cu, news, page_tokens=32)
        ops.kv4_append(k, v, part, table, lens, cu, most, page_tokens=32)
        read = lambda p, n: ops.kv4_read(p, table, lens, cu, n, news + 2, n_head_kv=1, head_dim=32, page_tokens=32, dtype=torch.float32)  # noqa: E731
        new, was = read(whole, news), read(old, news)
        take = [i < most or i >= news for i in range(news)] + [True, most > 1]
        here = torch.tensor(take, device=dev)
        for got, n, w in zip(read(part, news), new, was):
            assert torch.equal(got[here], n[here]) and torch.equal(got[~here], w[~here])
        q = torch.randn((news + 2, 3, 32), generator=torch.Generator().manual_seed(5)).half().to(dev)
        att = lambda n, out: ops.kv4_attention(q, whole, table, lens, cu, n, n_head_kv=1, page_tokens=32, out=out)  # noqa: E731
        want, got = att(news, None), att(most, torch.full_like(q, 7))
        assert (got[~here] == 7).all()
        assert (got[here].float() - want[here].float()).abs().max() < 2.0**-7   # (another kernel may have taken them: values of 1, halves)


def test_no_rows_of_any_stride(dev):
    """an empty tensor is contiguous whatever its strides are; there is nothing to do"""
    c = Cache(1, [40, 3], 2, 64, 32)
    pages, table, lens = c.on(dev)
    q = torch.empty((64, 0, 4), dtype=torch.float16, device=dev).permute(1, 2, 0)
    cu = ints(dev, 0, 0, 0)
    assert ops.kv4_attention(q, pages, table, lens, cu, 0, n_head_kv=2, page_tokens=32).shape == (0, 4, 64)
    out = torch.empty((64, 0, 4), dtype=torch.float32, device=dev).permute(1, 2, 0)
    assert ops.kv4_attention(q, pages, table, lens, cu, 5, n_head_kv=2, page_tokens=32, out=out) is out
    old = pages.clone()
    ops.kv4_append(q[:, :2], q[:, 2:], pages, table, lens, cu, 5, page_tokens=32)
    assert torch.equal(pages, old)


# ---- pages --------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("length,add", [(2**31 - 1, 2**31 - 1), (1, 2**31 - 1), (2**31 - 1, 1), (2**30, 2**30)])
def test_room_behind_lengths_near_2_31(dev, length, add):
    """pages of one token: the end of what is asked for lies at 2^31 and beyond, far outside of the table.  Refused, nothing has changed, its neighbours included."""
    pages = torch.zeros((8, 16), dtype=torch.uint8, device=dev)
    table, lens, refs = ints(dev, [0, 1, -1, -1], [2, -1, -1, -1]), ints(dev, length, 1), ints(dev, 1, 1, 1, 0, 0, 0, 0, 0)
    t, n, r, short = ops.kv_reserve(pages, table, lens, refs, ints(dev, add, 1), page_tokens=1)
    assert int(short) == -1
    assert torch.equal(t, table) and torch.equal(n, lens) and torch.equal(r, refs)


def test_no_length_beyond_2_31(dev):
    """a table with room for it, but no int32 that could hold the length: refused; the largest length that fits is not"""
    pages = torch.zeros((4, 16), dtype=torch.uint8, device=dev)
    table, refs = ints(dev, [0, 1, -1, -1]), ints(dev, 1, 1, 0, 0)
    for length, add, want in ((2**31 - 1, 10, -1), (2**31 - 10, 10, -1), (2**31 - 10, 9, 0), (2**30, 2**30, -1)):
        lens = ints(dev, length)
        t, n, r, short = ops.kv_reserve(pages, table, lens, refs, ints(dev, add), page_tokens=2**30)
        assert int(short) == want and n.tolist() == [length + (0 if want else add)]
        assert torch.equal(t, table) and torch.equal(r, refs)


def shared_by_all(dev, n):
    """n sequences of five tokens in two pages of four, forks of one another; room for one more each"""
    table = torch.tensor([[0, 1, -1]], dtype=torch.int32).repeat(n, 1).to(dev)
    refs = torch.zeros(n + 1, dtype=torch.int32, device=dev)
    refs[:2] = n
    pages = torch.zeros((n + 1, 16), dtype=torch.uint8, device=dev)
    lens, add = torch.full((n,), 5, dtype=torch.int32, device=dev), torch.ones(n, dtype=torch.int32, device=dev)
    t0 = time.perf_counter()
    t, m, r, short = ops.kv_reserve(pages, table, lens, refs, add, page_tokens=4)
    assert int(short) == 0
    took = time.perf_counter() - t0
    # pages 2, 3, .. in order; the last sequence keeps the shared one
    assert t[:, 0].tolist() == [0] * n and t[:, 1].tolist() == list(range(2, n + 1)) + [1] and m.tolist() == [6] * n
    assert r.tolist() == [n] + [1] * n
    return took


def test_room_for_very_many_sequences_of_one_last_page(dev):
    """in time that grows with their number, not with its square"""
    shared_by_all(dev, 3000)
    if dev.type == "cuda":
        assert shared_by_all(dev, 1 << 20) < 1.0
        return
    few, many = (min(shared_by_all(dev, n) for _ in range(2)) for n in (1 << 15, 1 << 17))
    assert many < 5 * few   # (linear: less than 4; quadratic: towards 16)


@pytest.mark.parametrize("n_new", [4096, 4097])
def test_forks_into_very_many(dev, n_new):
    """either way of counting references: parents with many children, one, and none, children of nobody"""
    n, width = 40, 3
    g = torch.Generator().manual_seed(n_new)
    table = torch.randperm(n * width, generator=g)[:n * width].view(n, width).int()
    lens = torch.randint(0, 4 * width + 1, (n,), generator=g).int()
    used = (lens[:, None] + 3) // 4 > torch.arange(width)
    table[~used] = -1
    refs = torch.zeros(n * width + 1, dtype=torch.int32)
    refs[table[used].long()] = 1
    parents = torch.cat([torch.tensor([n, -1, 3, 5]), torch.randint(6, n, (n_new - 4,), generator=g)]).int()
    t, m, r = (x.cpu() for x in ops.kv_fork(table.to(dev), lens.to(dev), refs.to(dev), parents.to(dev), page_tokens=4))
    ok = (parents >= 0) & (parents < n)
    at = parents.clamp(0, n - 1).long()
    want = torch.where(ok[:, None], table[at], -1)
    counts = torch.zeros_like(refs).index_add_(0, want[want >= 0].long(), torch.ones(int((want >= 0).sum()), dtype=torch.int32))
    assert torch.equal(t, want) and torch.equal(m, torch.where(ok, lens[at], 0)) and torch.equal(r, counts)


# ---- graphs ---------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dim", [96, 128, 256])
@pytest.mark.parametrize("news", [1, 6, 150])
def test_every_attention_kernel_in_a_graph(hip_lib, dim, news):
    """head sizes whose kernels take more LDS than a launch may without asking, the asking within the capture: replays equal eager calls, with eager work between them"""
    ops.load(hip_lib)
    dev = torch.device("cuda:0")  # noqa: F811
    heads, H, page, B, width = 2, 8, 64, 2, 24

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        lens = torch.randint(news, width * page + 1, (B,), generator=g).int()
        pages = torch.zeros((B * width, ops.kv4_page_bytes(heads, dim, page)), dtype=torch.uint8, device=dev)
        table = torch.randperm(B * width, generator=g).view(B, width).int().to(dev)
        total = int(lens.sum())
        k, v = (torch.randn((total, heads, dim), generator=g).half().to(dev) for _ in range(2))
        ops.kv4_append(k, v, pages, table, lens.to(dev), ints(dev, 0, int(lens[0]), total), int(lens.max()), page_tokens=page)
        return [torch.randn((B * news, H, dim), generator=g).half().to(dev), pages, table, lens.to(dev)]

    cu = ints(dev, 0, news, 2 * news)
    run = lambda x: ops.kv4_attention(*x, cu, news, n_head_kv=heads, page_tokens=page)  # noqa: E731
    held = inputs(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(held)
    for seed in range(1, 5):
        new = inputs(seed)
        for x, y in zip(held, new):
            x.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, run(new))
        graph.replay()
        assert torch.equal(out, got)
