"""CT_AMD_KV=q4: a handle's attention over the 4-bit paged cache (csrc/engine_kv4.h), and its contexts.

The attention of a one-layer model is checked against the formula: K and V rows are the default handle's (the same launches write them), quantized as the format says;
Q is read from the 4-bit handle.  Contexts are checked against a handle that evaluated the same tokens in the same requests: bit for bit, a page is read by the same
kernels wherever it lies and whoever shares it."""
import ctypes
import os

import numpy as np
import pytest

from conftest import HIP_LIB, ROOT, has_gpu
from ctransformers_amd.llm import LLM, Config
from ctransformers_amd.measure import LaunchStat
from test_kv4 import attention64, quantize
from tools import synth

GOLDEN = os.path.join(ROOT, "tests", "golden")


@pytest.fixture(params=["emu", pytest.param("hip", marks=pytest.mark.gpu)])
def lib(request):
    if request.param == "emu":
        if has_gpu():
            pytest.skip("the emulation is for hosts without a GPU")
        return request.getfixturevalue("emu_lib")
    return request.getfixturevalue("hip_lib")


def open_model(path, lib, monkeypatch, kv="q4", contexts=1, ctx=256, **env):
    for name, value in dict(CT_AMD_KV=kv, CT_AMD_CONTEXTS=contexts, **env).items():
        monkeypatch.setenv(name, str(value))
    return LLM(path, config=Config(context_length=ctx, batch_size=512, threads=1), lib=lib)


def read(m, name, dtype, shape, *args):
    f = getattr(m._lib, name)
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int]
    buf = np.zeros(shape, dtype)
    assert f(m._llm, buf.ctypes.data, *args) > 0
    return buf


def kv_rows(m, heads, n_ctx, hd):
    f = m._lib.ctamd_debug_read_kv
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    k, v = np.zeros((heads, n_ctx, hd), np.float16), np.zeros(heads * hd * (n_ctx + 512), np.float16)
    stride = f(m._llm, 0, k.ctypes.data, v.ctypes.data)
    assert stride > 0
    return k, v[:heads * hd * stride].reshape(heads, hd, stride)


def values(rows):
    codes, scales = quantize(rows.astype(np.float32))
    return ((codes.astype(np.float64) - 8).reshape(scales.shape + (32,)) * scales.astype(np.float64)[..., None]).reshape(rows.shape)


def launches(m):
    m._lib.ctamd_kv4_launches.restype, m._lib.ctamd_kv4_launches.argtypes = ctypes.c_longlong, [ctypes.c_void_p]
    return int(m._lib.ctamd_kv4_launches(m._llm))


@pytest.mark.parametrize("n_prompt", [1, 33, 70])
def test_attention_of_a_handle_is_the_formula(lib, n_prompt, tmp_path, monkeypatch):
    """a prompt chunk, then a token step, pages of 32: the rows pass pages' ends.  (The emulation takes a second a token: not 70 of them.)"""
    if lib != HIP_LIB and n_prompt > 33:
        pytest.skip("GPU only")
    monkeypatch.setenv("CT_AMD_KV_PAGE", "32")
    shape = dict(synth.LLAMA_SHAPES["llama-tiny"], n_layer=1)
    path = str(tmp_path / "one.gguf")
    synth.write_llama_gguf(path, shape, "Q4_K_M", seed=5)
    heads, kv, E = shape["n_head"], shape["n_head_kv"], shape["n_embd"]
    hd, ctx = E // heads, 128
    toks = synth.prompt_tokens(n_prompt + 1, shape["n_vocab"])
    plain = open_model(path, lib, monkeypatch, kv="f16", ctx=ctx)
    four = open_model(path, lib, monkeypatch, ctx=ctx)
    for m in (plain, four):
        m.eval(toks[:n_prompt])
    for step in (0, 1):
        if step:
            for m in (plain, four):
                m.eval(toks[n_prompt:])
        n, rows = n_prompt + step, 1 if step or n_prompt == 1 else n_prompt
        k, v = kv_rows(plain, kv, ctx, hd)
        kk, vv = values(k[:, :n].transpose(1, 0, 2)), values(v[:, :, :n].transpose(2, 0, 1))
        q = read(four, "ctamd_debug_read_q", np.float16, (rows, heads, hd), 0 if rows == 1 else rows).astype(np.float64)
        out = read(four, "ctamd_debug_read_attn_out", np.float32, (rows, heads, hd), 0 if rows == 1 else rows).astype(np.float64)
        want, mag, err = attention64(q, (kk, vv), kv, float(np.float32(1) / np.sqrt(np.float32(hd))), (2.0**-11, 0))
        tol = mag * (2 * 2.0**-11 + 2 * np.expm1(err)[..., None]) * 1.01 + np.abs(want) * 2.0**-23   # (test_kv4.py; the result is float32)
        assert (np.abs(out - want) <= tol).all(), float((np.abs(out - want) / tol).max())
    assert launches(plain) == 0 and launches(four) > 0
    assert np.isfinite(four.logits.to_numpy()).all()


@pytest.mark.parametrize("name", ["tiny-q4km.gguf", "falcon-tiny-q4km.gguf", "tiny-q80.gguf"])
def test_models_run_on_the_4bit_cache(lib, name, monkeypatch):
    """every graph that serves it: prompt and token steps run, from position to position the same handle gives the same logits again"""
    path = os.path.join(GOLDEN, name)
    m = open_model(path, lib, monkeypatch, ctx=96)
    n, steps = (20, 4) if lib == HIP_LIB else (3, 2)
    toks = [int(t) for t in np.random.default_rng(0).integers(3, m.vocab_size, n + steps)]
    runs = []
    for _ in range(2):
        m._context.clear()
        m.eval(toks[:n])
        rows = [m.logits.to_numpy().copy()]
        for t in toks[n:]:
            m.eval([t])
            rows.append(m.logits.to_numpy().copy())
        runs.append(np.array(rows))
    assert np.isfinite(runs[0]).all() and np.array_equal(runs[0], runs[1]) and launches(m) > 0
    assert len({r.tobytes() for r in runs[0]}) == 1 + steps


def logits_after(m, *requests):
    for r in requests:
        m.eval(list(r))
    return m.logits.to_numpy().copy()


def test_contexts_fork_share_and_go_their_own_ways(lib, tmp_path, monkeypatch):
    """a prompt that ends inside a page, forked twice; the branches write on, one is rolled back into the shared pages, one freed and used anew.  `alone` is one
    context that is rolled back to where the branches part."""
    gpu = lib == HIP_LIB
    page, n, cut = (64, 70, 40) if gpu else (32, 34, 31)
    path = os.path.join(GOLDEN, "tiny-q4km.gguf")
    if not gpu:
        path = str(tmp_path / "one.gguf")
        synth.write_llama_gguf(path, dict(synth.LLAMA_SHAPES["llama-tiny"], n_layer=1), "Q4_K_M", seed=5)
    monkeypatch.setenv("CT_AMD_KV_PAGE", str(page))
    m = open_model(path, lib, monkeypatch, contexts=3, ctx=3 * page)
    alone = open_model(path, lib, monkeypatch, contexts=1, ctx=3 * page)
    assert m.n_contexts == 3 and alone.n_contexts == 1
    toks = [int(t) for t in np.random.default_rng(1).integers(3, m.vocab_size, 2 * page + 20)]
    prompt, a, b, c = toks[:n], toks[n:n + 3], toks[n:n + (page if gpu else 2)], toks[n + 5:n + 7]

    def expect(prefix, *requests):   # `alone` holds the prefix: what follows is written over what is there
        alone._context[:] = prefix
        return logits_after(alone, *requests)

    m.eval(prompt)
    alone.eval(prompt)
    m.fork_context(0, 1)
    m.fork_context(0, 2)
    assert [m._extension("ctamd_context_length", i) for i in range(3)] == [n] * 3
    assert m.compact_contexts() == 2                                       # two pages, shared by three
    m.use_context(1)
    assert m._context == prompt
    assert np.array_equal(logits_after(m, a[:1], a[1:]), expect(prompt, a[:1], a[1:]))
    assert m.compact_contexts() == 3                                       # its own copy of the partly filled page
    m.use_context(2)
    assert np.array_equal(logits_after(m, b), expect(prompt, b))
    m.use_context(0)
    assert np.array_equal(logits_after(m, c), expect(prompt, c))           # the original, untouched by its branches
    m.use_context(1)
    assert np.array_equal(logits_after(m, [9]), expect(prompt, a[:1], a[1:], [9]))
    # back to the middle of the shared prompt: its pages stay what they are for the others
    del m._context[cut:]
    got = logits_after(m, a, [7])
    m.use_context(0)
    assert np.array_equal(logits_after(m, [11]), expect(prompt, c, [11]))
    # freed and used anew, and forked over while it is in use
    m.free_context(2)
    m.use_context(2)
    assert m._context == [] and m._extension("ctamd_context_length", 2) == 0
    m.eval(b[:2])
    m.fork_context(1, 2)
    assert m._context == prompt[:cut] + a + [7]
    last = logits_after(m, [5])
    m.compact_contexts()
    m.use_context(0)
    assert np.array_equal(logits_after(m, [12]), expect(prompt, c, [11], [12]))
    assert np.array_equal(got, expect(prompt[:cut], a, [7])) and np.array_equal(last, logits_after(alone, [5]))


def test_contexts_filled_to_the_end(lib, monkeypatch):
    """every context takes its whole length: the pool has room for all of them"""
    if lib != HIP_LIB:
        pytest.skip("GPU only (140 tokens)")
    m = open_model(os.path.join(GOLDEN, "tiny-q4km.gguf"), lib, monkeypatch, contexts=2, ctx=70)
    toks = [int(t) for t in np.random.default_rng(2).integers(3, m.vocab_size, 70)]
    m.eval(toks[:66])
    m.fork_context(0, 1)
    for i in (1, 0):
        m.use_context(i)
        m.eval(toks[66:69])
        m.eval(toks[69:])
    assert m._extension("ctamd_context_length", 0) == m._extension("ctamd_context_length", 1) == 70
    assert m.compact_contexts() == 3                                                        # 64 tokens in common, two ends


def test_refusals(lib, monkeypatch, capfd):
    path = os.path.join(GOLDEN, "tiny-q4km.gguf")
    for env in (dict(kv="q5"), dict(kv="f16", contexts=2), dict(kv="q4", contexts=1000)):
        with pytest.raises(RuntimeError):
            open_model(path, lib, monkeypatch, **env)
    with pytest.raises(RuntimeError):
        monkeypatch.setenv("CT_AMD_KV", "q4")
        monkeypatch.setenv("CT_AMD_CONTEXTS", "1")
        LLM(os.path.join(GOLDEN, "gpt2-tiny-q40.bin"), "gpt2", config=Config(context_length=64), lib=lib)
    m = open_model(path, lib, monkeypatch, contexts=2)
    for call in (lambda: m.use_context(2), lambda: m.use_context(-1), lambda: m.fork_context(0, 0), lambda: m.fork_context(0, 5), lambda: m.free_context(2)):
        with pytest.raises(ValueError):
            call()
    plain = open_model(path, lib, monkeypatch, kv="f16")
    assert plain.n_contexts == 1
    with pytest.raises(ValueError):
        plain.use_context(0)
    with pytest.raises(RuntimeError):
        plain.compact_contexts()


@pytest.mark.parametrize("nth", [1, 3, 5, 7, 9, 12])
def test_a_refused_attention_launch_fails_every_eval_that_would_lack_it(lib, nth, monkeypatch):
    """The nth attention launch of the handle is refused (two layers; on the GPU: the load's warm-up, the captures of the token steps, an eager chunk, a chunk's capture, ..).
    The load or the eval that issues it fails; whatever succeeds afterwards has all its launches: no graph without the launch stays behind."""
    path = os.path.join(GOLDEN, "tiny-q4km.gguf")
    toks = [int(t) for t in np.random.default_rng(3).integers(3, 200, 12)]
    plain = open_model(path, lib, monkeypatch, ctx=64)
    failed = 0
    try:
        m = open_model(path, lib, monkeypatch, ctx=64, CT_AMD_DBG_KV4_FAIL=nth)
    except RuntimeError:
        assert lib == HIP_LIB
        return
    steps = [toks[:3], toks[3:6], toks[6:9], toks[9:10], toks[10:11]] if lib == HIP_LIB else [toks[:2], toks[2:3]]
    for step in steps:
        for _ in range(2):
            plain._context[:] = m._context
            try:
                m.eval(step)
            except RuntimeError:
                failed += 1
                continue
            plain.eval(step)
            assert np.array_equal(m.logits.to_numpy(), plain.logits.to_numpy())
            break
    assert failed == (nth <= (10 if lib == HIP_LIB else 4))


@pytest.mark.gpu
@pytest.mark.parametrize("active", [0, 1])
def test_measurements_do_not_write_into_pages_that_a_fork_shares(hip_lib, active, monkeypatch):
    """a measurement replays the last token of the active context; after a fork that position lies in the other context's pages too (or was dropped): there is nothing to replay"""
    path = os.path.join(GOLDEN, "tiny-q4km.gguf")
    m = open_model(path, hip_lib, monkeypatch, contexts=2, ctx=128)
    alone = open_model(path, hip_lib, monkeypatch, ctx=128)
    lib = m._lib
    lib.ctamd_profile_decode.restype, lib.ctamd_profile_decode.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_int]
    lib.ctamd_trace_site.restype, lib.ctamd_trace_site.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p, ctypes.c_int]
    buf, stamps = (LaunchStat * 32)(), (ctypes.c_uint64 * 512)()
    toks = [int(t) for t in np.random.default_rng(4).integers(3, m.vocab_size, 24)]
    for h in (m, alone):
        h.eval(toks[:20])
    if active == 1:
        m.use_context(1)
        m.eval(toks[20:21])                  # (its position 0 becomes context 0's)
    m.fork_context(0, 1)
    assert lib.ctamd_profile_decode(m._llm, 2, buf, 32) <= 0 and lib.ctamd_trace_site(m._llm, b"qkv", stamps, 8) < 0
    m.use_context(0)
    got = logits_after(m, toks[21:22], toks[22:23])
    assert np.array_equal(got, logits_after(alone, toks[21:22], toks[22:23]))
    assert lib.ctamd_profile_decode(m._llm, 1, buf, 32) > 0              # an eval's last token is there again
    m.free_context(0)
    assert lib.ctamd_profile_decode(m._llm, 1, buf, 32) <= 0


@pytest.mark.gpu
def test_a_burst_is_no_part_of_the_context(hip_lib, monkeypatch):
    path = os.path.join(GOLDEN, "tiny-q4km.gguf")
    m = open_model(path, hip_lib, monkeypatch, contexts=2, ctx=256)
    alone = open_model(path, hip_lib, monkeypatch, ctx=256)
    m._lib.ctamd_decode_burst.restype, m._lib.ctamd_decode_burst.argtypes = ctypes.c_double, [ctypes.c_void_p, ctypes.c_int]
    toks = [int(t) for t in np.random.default_rng(5).integers(3, m.vocab_size, 70)]
    for h in (m, alone):
        h.eval(toks[:60])
    assert m._lib.ctamd_decode_burst(m._llm, 100) > 0                     # (through two pages' ends)
    assert m._extension("ctamd_context_length", 0) == 60
    m.fork_context(0, 1)
    assert m._extension("ctamd_context_length", 1) == 60 and m.compact_contexts() == 3   # what the burst has taken stays the first context's until it is written over
    m.use_context(1)
    assert np.array_equal(logits_after(m, toks[60:61], toks[61:62]), logits_after(alone, toks[60:61], toks[61:62]))


def test_the_dump_of_a_handle_with_one_layers_rows(lib, tmp_path, monkeypatch):
    """CT_AMD_DUMP writes a layer's K / V rows after its attention: with the 4-bit cache they lie in one layer's buffer, which all layers use in turn"""
    if lib == HIP_LIB:
        pytest.skip("the emulation alone: the copy is the host's")
    path = os.path.join(GOLDEN, "tiny-q4km.gguf")
    rows = {}
    for kv in ("f16", "q4"):
        out = tmp_path / kv
        out.mkdir()
        m = open_model(path, lib, monkeypatch, kv=kv, ctx=32, CT_AMD_DUMP=out)
        m.eval([5])
        for il in (0, 1):
            name = sorted(f for f in os.listdir(out) if f.endswith("_l%02d_kv.bin" % il))[-1]
            rows[kv, il] = np.fromfile(out / name, np.float16).astype(np.float32)
        del m
    monkeypatch.delenv("CT_AMD_DUMP")
    assert np.array_equal(rows["f16", 0], rows["q4", 0])
    a, b = rows["f16", 1], rows["q4", 1]
    assert a.any() and np.array_equal(a != 0, b != 0)                     # one position's rows, and zeros everywhere else
    assert np.linalg.norm(a - b) < 0.3 * np.linalg.norm(a)                 # layer 0 attended to V in 4 bits: half a step of 1/8 of a group's largest, 1/16, at worst in every value
