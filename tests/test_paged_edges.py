"""Operators over a paged cache at the edges of what their arguments may be.

Tolerances are those of tests/test_paged.py, or derived where they stand.
"""
import math
import os
import subprocess

import pytest
import torch

import megacute_b200 as mc
from megacute_b200 import _lib, paged
from oracle import paged_oracle as ref
from tests.test_paged import BF, HALF, W, attention_tolerance, check_attention, close, half_step, make_attention, on, smallest


# -- the hint of the largest number of new tokens ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("max_new", [0, -3, -2 ** 31])
@pytest.mark.parametrize("H,KVH,D", [(32, 1, 64), (40, 1, 128), (34, 2, 64), (3, 3, 128)])
def test_hint_below_one_with_many_heads(cuda, H, KVH, D, max_new, binding, monkeypatch):
    """A hint below one is taken as one by the query of the workspace too, where a token's heads are more than an item for few rows holds."""
    if not binding:
        monkeypatch.setattr(paged, "_direct", lambda: None)
    args, kw = make_attention([33, 0], [2, 1], H, KVH, D, 16, BF, seed=8)
    check_attention(cuda, args, dict(kw, max_new=max_new))


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [-5, 0, 1, 2, 4, 5, 16, 17, 4096])
@pytest.mark.parametrize("H,KVH,D", [(4, 4, 64), (8, 2, 128), (16, 1, 64), (17, 1, 64), (40, 1, 128)])
def test_workspace_query_suffices(cuda, H, KVH, D, max_new):
    """What the query returns is enough for the call with the same hint, whatever the scale; one byte is refused as an argument."""
    lib = _lib.load()
    nbytes = lib.mk_paged_attention_workspace(0, H, KVH, D, max_new)
    assert nbytes > 0
    work = torch.empty(nbytes, dtype=torch.uint8, device=cuda)
    cache = torch.zeros(32, 2 * KVH * D, dtype=BF, device=cuda)
    q, out = torch.zeros(2, H * D, dtype=BF, device=cuda), torch.ones(2, H * D, dtype=BF, device=cuda)
    pos, table = torch.tensor([[3], [20]], dtype=torch.int32, device=cuda), torch.tensor([[0, 1], [1, 0]], dtype=torch.int32, device=cuda)
    b = _lib.Batch(pos.data_ptr(), None, 1, 2, 2)
    c = _lib.PagedCache(cache.data_ptr(), cache[:, KVH * D:].data_ptr(), table.data_ptr(), 2 * KVH * D, 2 * KVH * D, 2, 2, 16, 2, KVH, D, 0)
    stream = torch.cuda.current_stream().cuda_stream
    for scale in (0.125, 0.0, -1.0):
        call = lambda size: lib.mk_paged_attention(0, b, c, q.data_ptr(), H * D, out.data_ptr(), H * D, H, scale, 0, max_new, work.data_ptr(), size, stream)
        assert call(1) == -2 and b"workspace smaller" in lib.mk_last_cuda_error()
        out.fill_(1.0)
        assert call(nbytes) == 0, lib.mk_last_cuda_error()
        assert (out == 0).all()


# -- scalings of the frequencies --------------------------------------------------------------------------------------------
YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


def yarn(rotary_dim, theta, factor, orig, fast=32.0, slow=1.0, rounded=True):
    """Pair by pair: 1 / factor of the angle for pairs of at most `slow` turns over the original length, all of it from `fast` on, linear between."""
    def pair(turns):
        return rotary_dim * math.log(orig / (2 * math.pi * turns)) / (2 * math.log(theta))
    a, b = pair(fast), pair(slow)
    a, b = (math.floor(a), math.ceil(b)) if rounded else (a, b)
    a, b = max(a, 0), min(b, rotary_dim - 1)
    out = []
    for i in range(rotary_dim // 2):
        stretched = min(max((i - a) / (b - a), 0.0), 1.0)
        w = theta ** (-2.0 * i / rotary_dim)
        out.append(w * (stretched / factor + 1.0 - stretched))
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("mscale,all_dim", [(1.0, 1.0), (0.707, 0.707), (0.707, 1.0), (1.0, 0.8), (2.0, 0.5), (None, None), (1.0, None), (1.0, 0.0), (1, 0)])
def test_yarn_mscale(mscale, all_dim):
    inv, f = mc.rotary_frequencies(64, 10000.0, dict(YARN, mscale=mscale, mscale_all_dim=all_dim))
    term = lambda s: 0.1 * s * math.log(40.0) + 1.0
    want = term(mscale) / term(all_dim) if mscale and all_dim else term(1.0)
    assert abs(f - want) < 1e-12
    assert torch.allclose(inv, yarn(64, 10000.0, 40.0, 4096.0), rtol=1e-12, atol=0)
    cos, _ = mc.rotary_tables(2, 64, 10000.0, dict(YARN, mscale=mscale, mscale_all_dim=all_dim))
    assert abs(float(cos[0, 0]) - want) < 1e-6
    assert mc.rotary_frequencies(64, 10000.0, dict(YARN, mscale=mscale, mscale_all_dim=all_dim, attention_factor=1.25))[1] == 1.25


@pytest.mark.parametrize("rotary_dim,theta,factor,orig,fast,slow", [(64, 150000.0, 32.0, 4096, 32.0, 1.0), (128, 10000.0, 16.0, 4096, 32.0, 1.0),
                                                                    (48, 1e6, 4.0, 32768, 20.0, 2.0)])
def test_yarn_corners(rotary_dim, theta, factor, orig, fast, slow):
    sc = {"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": orig, "beta_fast": fast, "beta_slow": slow}
    for more, rounded in (({}, True), ({"truncate": True}, True), ({"truncate": None}, True), ({"truncate": False}, False)):
        got, _ = mc.rotary_frequencies(rotary_dim, theta, dict(sc, **more))
        assert torch.allclose(got, yarn(rotary_dim, theta, factor, float(orig), fast, slow, rounded), rtol=1e-12, atol=0)
    assert not torch.allclose(got, mc.rotary_frequencies(rotary_dim, theta, sc)[0], rtol=1e-6, atol=0)


def test_scaling_lengths_of_the_config():
    """What a dict leaves to the config's own length."""
    full = {"type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048}
    part = {"type": "dynamic", "factor": 2.0}
    for n in (None, 100, 8192):
        a, b = mc.rotary_frequencies(64, 1e4, full, n), mc.rotary_frequencies(64, 1e4, part, n, max_position_embeddings=2048)
        assert torch.equal(a[0], b[0]) and a[1] == b[1] == 1.0
    assert torch.equal(mc.rotary_tables(8192, 64, 1e4, full)[0], mc.rotary_tables(8192, 64, 1e4, part, max_position_embeddings=2048)[0])
    want = mc.rotary_frequencies(64, 1e4, YARN)
    for sc, n in (({"rope_type": "yarn", "factor": 40.0}, 4096), ({"rope_type": "yarn", "factor": None, "original_max_position_embeddings": 4096}, 163840),
                  ({"rope_type": "yarn", "original_max_position_embeddings": 4096}, 163840), (YARN, 7)):
        got = mc.rotary_frequencies(64, 1e4, sc, max_position_embeddings=n)
        assert torch.equal(got[0], want[0]) and got[1] == want[1]
    got = mc.rotary_frequencies(64, 1e4, {"rope_type": "yarn"}, max_position_embeddings=4096)      # as long as it was: as it is
    assert torch.allclose(got[0], mc.rotary_frequencies(64, 1e4)[0], rtol=1e-12, atol=0) and got[1] == 1.0


@pytest.mark.parametrize("kind", ["default", "linear", "dynamic", "llama3", "yarn"])
def test_scaling_keys_without_effect(kind):
    """Keys that repeat an argument or say how the config was made, and keys that hold None."""
    sc = {"rope_type": kind, "original_max_position_embeddings": 4096}
    if kind != "default":
        sc["factor"] = 8.0
    if kind == "llama3":
        sc.update(low_freq_factor=1.0, high_freq_factor=4.0)
    want = mc.rotary_frequencies(64, 5e5, sc)
    got = mc.rotary_frequencies(64, 500000, dict(sc, type=kind, rope_theta=500000.0, partial_rotary_factor=0.5, finetuned=True, mscale=None, long_factor=None))
    assert torch.equal(got[0], want[0]) and got[1] == want[1]


@pytest.mark.parametrize("scaling,words", [
    ({"rope_type": "yarn", "factor": 4.0}, "needs original_max_position_embeddings"),
    ({"rope_type": "yarn", "factor": None, "original_max_position_embeddings": 4096}, "needs factor"),
    ({"rope_type": "yarn", "original_max_position_embeddings": 4096}, "needs factor"),
    ({"type": "dynamic", "factor": 2.0}, "needs original_max_position_embeddings"),
    ({"type": "dynamic", "original_max_position_embeddings": 4096}, "needs factor"),
    ({"type": "linear"}, "needs factor"),
    ({"type": "linear", "factor": 0.0}, "positive"),
    ({"type": "linear", "factor": float("nan")}, "positive"),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "original_max_position_embeddings": 8192}, "needs high_freq_factor"),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0}, "needs original_max_position_embeddings"),
    (dict(YARN, mscale=0.707), "for each other"),
    (dict(YARN, mscale_all_dim=1.0), "for each other"),
    (dict(YARN, mscale=0.707, mscale_all_dim=0.0), "for each other"),
    (dict(YARN, mscale=0.0, mscale_all_dim=0.0), "for each other"),
    (dict(YARN, low_freq_factor=1.0), "does not take low_freq_factor"),
    (dict(YARN, attn_factor=2.0), "does not take attn_factor"),
    ({"type": "linear", "factor": 2.0, "mscale": 1.0, "beta_fast": 32}, "does not take beta_fast, mscale"),
    ({"rope_type": "default", "mrope_section": [16, 24, 24]}, "does not take mrope_section"),
    ({"rope_type": "linear", "factor": 2.0, "rope_theta": 500000.0}, "rope_theta"),
    ({"rope_type": "default", "rope_theta": 500000.0}, "rope_theta"),
])
def test_scalings_refused(scaling, words):
    with pytest.raises(ValueError, match=words):
        mc.rotary_frequencies(64, 10000.0, scaling)
    with pytest.raises(ValueError, match=words):
        mc.rotary_tables(4, 64, 10000.0, scaling)


# -- waits that gave up -------------------------------------------------------------------------------------------------------
class Failing:
    """The library with a count of failed waits of its own (no wait is made to fail): one more of `counts` each time it is asked."""

    def __init__(self, lib, counts):
        self.lib, self.counts = lib, list(counts)

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def mk_paged_attention_failures(self, device, stream, count):
        count.value = self.counts.pop(0)
        return 0


def test_failed_waits_raise(monkeypatch):
    """Every caller learns of a failure, however often and by whom the count was read before."""
    lib = Failing(_lib.load(), [0, 3, 3, 3, 3, 5])
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(paged, "_stream", lambda what, device: 0)
    dev = torch.device("cuda", 0)
    assert mc.paged_attention_check(dev) == 0
    for _ in range(2):
        with pytest.raises(_lib.MegakernelTimeout, match="timed out"):
            mc.paged_attention_check(dev)
    assert mc.paged_attention_check("cuda:0", None) == 3
    assert mc.paged_attention_check(dev, seen=3) == 3
    with pytest.raises(_lib.MegakernelTimeout):
        mc.paged_attention_check(dev, seen=3)
    with pytest.raises(ValueError, match="no CUDA device"):
        mc.paged_attention_check("cpu")


def test_failures_needs_a_place():
    assert _lib.load().mk_paged_attention_failures(0, None, None) == -2


@pytest.mark.gpu
def test_no_failures(cuda):
    args, kw = make_attention([33, 0], [40, 1], 4, 2, 64, 16, BF, seed=8)
    check_attention(cuda, args, kw)
    assert mc.paged_attention_check() == mc.paged_attention_check(cuda) == mc.paged_attention_check("cuda", None) == 0
    with torch.cuda.stream(torch.cuda.Stream()):
        assert mc.paged_attention_check(cuda) == 0
    assert _lib.load().mk_paged_attention_status(0, torch.cuda.current_stream().cuda_stream) == 0


@pytest.mark.gpu
def test_generator_tells_of_failed_waits(cuda, monkeypatch):
    """A prompt in chunks behind which a wait is known to have failed, in an attention call or in one of its launches (a wait target that
    nothing reaches, with a limit of 50 ms), is an error and not a sequence of tokens."""
    from megacute_b200.checkpoint import LlamaGenerator
    from tests.test_checkpoint import CFG, hf_state_dict
    gen = LlamaGenerator(CFG, hf_state_dict(CFG, seed=5), max_seq=128, device=cuda, prompt_chunk=16)
    assert gen.generate(list(range(1, 20)), 2).shape == (1, 2)
    real = _lib.load()
    lib = Failing(real, [2, 2, 2, 3])
    with monkeypatch.context() as m:
        m.setattr(_lib, "load", lambda: lib)
        assert gen.prefill(list(range(16))) == 16                             # (what failed before it began is not its own)
        with pytest.raises(_lib.MegakernelTimeout):
            gen.generate(list(range(1, 20)), 2)
    prog = gen._between[1]
    s = prog.sched
    prog.set_timeout(0.05)
    _lib.check(real.mk_program_poke_wait(prog._handle, 0, int(s.wait_cnt[0]), int(s.wait_tgt[0]) + 1000))
    with pytest.raises(_lib.MegakernelTimeout):
        gen.prefill(list(range(16)))


# -- building the binding -----------------------------------------------------------------------------------------------------
@pytest.fixture
def own_binding(tmp_path, monkeypatch):
    """A place for the module of this test's own, and a compiler that only makes the file; the list of its runs."""
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        (tmp_path / "_binding.so").write_text("module")
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(_lib, "BINDING_PATH", tmp_path / "_binding.so")
    monkeypatch.setattr(_lib.subprocess, "run", run)
    return runs


def test_library_without_a_compiler_for_the_binding(own_binding, monkeypatch):
    """Where the Python module cannot be compiled the library is there all the same, with a warning, and no module of other sources is loaded."""
    monkeypatch.setattr(_lib, "needs_build_of", lambda path: False)
    assert _lib.build() == _lib.LIB_PATH and _lib.BINDING_PATH.exists()
    for error in (lambda cmd, **kw: subprocess.CompletedProcess(cmd, 1, "", "Python.h: No such file"), None):
        def missing(cmd, **kw):
            raise FileNotFoundError("g++")
        monkeypatch.setattr(_lib.subprocess, "run", error or missing)
        _lib.BINDING_PATH.write_text("of older sources")
        os.utime(_lib.BINDING_PATH, (0, 0))
        with pytest.warns(RuntimeWarning, match="ctypes"):
            assert _lib.build() == _lib.LIB_PATH
        assert not _lib.BINDING_PATH.exists()
        with pytest.raises((RuntimeError, FileNotFoundError)):
            _lib.build_binding()


def test_binding_is_built_again_for_another_torch(own_binding, monkeypatch):
    """A module that was built against another torch, or of which that is not known, would be left aside at run time."""
    _lib.build_binding()
    assert len(own_binding) == 1 and any(torch.__version__ in word for word in own_binding[0])
    _lib.build_binding()
    assert len(own_binding) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    _lib.build_binding()
    assert len(own_binding) == 2 and any("0.0.1+other" in word for word in own_binding[1])
    _lib.build_binding()
    assert len(own_binding) == 2
    _lib.BINDING_PATH.with_suffix(".built_for").unlink()
    _lib.build_binding()
    assert len(own_binding) == 3
    _lib.build_binding(force=True)
    assert len(own_binding) == 4


# -- probabilities of single tokens -----------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("scale", [None, 0.02])
@pytest.mark.parametrize("D,H,KVH,new,dtype", [(64, 4, 2, 1, BF), (128, 8, 1, 1, BF), (128, 8, 2, 2, BF), (64, 7, 1, 1, BF), (64, 32, 8, 1, BF),
                                               (128, 6, 3, 3, HALF), (64, 8, 1, 1, HALF)])
def test_probabilities_of_few_rows_in_two_halves(cuda, D, H, KVH, new, dtype, scale):
    """Up to 8 rows an item: a probability is handed on as a rounded value and its rounded rest, off by u^2 of it; with the error of a score (2 (D + 6) w S),
    of the sum (w for each of n + 64 additions) and of an exponential (2^-22, in the weight and in the sum), and no 2^-13 for a polynomial, which this
    kernel has not.  Little more than the result's own rounding is left."""
    args, kw = make_attention([700, 0, 1023, 16, 300], [new] * 5, H, KVH, D, 32, dtype, seed=H + new)
    got = mc.paged_attention(**on(cuda, args), **kw, scale=scale, max_new=new)
    want, mag, size = ref.paged_attention(**args, **kw, scale=scale)
    u, keys = half_step(dtype), 1024 + new
    under = keys * 2.0 ** -25 * float(args["v_cache"].double().abs().max()) if dtype == HALF else 0.0
    per = u ** 2 + 2 * (D + 6) * W * size + (keys + 64) * W + 2.0 ** -21
    close(got, want, u * want.abs() + (1 + u) * (per * mag + under) + smallest(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,KVH,new,dtype", [(64, 4, 2, 1, BF), (128, 4, 1, 2, HALF), (64, 4, 1, 2, BF), (128, 16, 1, 1, BF)])
def test_infinite_values_of_few_rows(cuda, D, H, KVH, new, dtype):
    """An infinite value gives the tokens that see it an infinite result, not none, whatever the sign of a probability's rounding."""
    args, kw = make_attention([300, 40], [new, new], H, KVH, D, 16, dtype, seed=D + new, qstd=0.3)
    n = args["k_cache"].shape[0] // 16
    for s, p in ((0, 7), (0, 300 + new - 1), (1, 33)):
        args["v_cache"][ref.cache_row(args["pages"], s, p, 16, n), s::5] = float("inf") if s else float("-inf")
    got = mc.paged_attention(**on(cuda, args), **kw, max_new=new).cpu().double()
    want = ref.paged_attention(**args, **kw)[0]
    for f in (torch.isposinf, torch.isneginf, torch.isnan):
        assert torch.equal(f(got), f(want))
    assert torch.isinf(want).any() and torch.isfinite(want).any()


# -- messages of the C entries --------------------------------------------------------------------------------------------------
def test_messages_of_the_c_entries():
    """Each refusal leaves its own message (addresses here are never followed; the one before is of another kind each time)."""
    lib = _lib.load()
    batch = lambda **k: _lib.Batch(**{**dict(pos=4096, starts=None, pos_ld=1, rows=4, seqs=2), **k})
    rot = lambda **k: _lib.Rotation(**{**dict(cos=4096, sin=4096, ld_cos=32, ld_sin=32, rows=8, columns=32, dtype=1, interleaved=0), **k})
    cache = lambda **k: _lib.PagedCache(**{**dict(k=4096, v=4096, table=4096, ld_k=128, ld_v=128, table_ld=4, pages=4, page_size=16, table_cols=4,
                                                  kv_heads=2, head_dim=64, dtype=0), **k})
    rotary = lambda b=batch(), r=rot(), x=4096, ld=256, dim=64: lib.mk_rotary(0, b, r, x, ld, 8192, 256, 0, 4, dim, None)
    append = lambda c=cache(), r=rot(), q=8192, heads=4: lib.mk_paged_append(0, batch(), r, c, 4096, 512, q, 256, heads, None)
    attend = lambda c=cache(), ws=4096, window=0, heads=4, q=4096: lib.mk_paged_attention(0, batch(), c, q, 256, 8192, 256, heads, 1.0, window, 1, ws, 1 << 40, None)
    for call, words in ((lambda: rotary(x=4104), b"16-byte"), (lambda: rotary(batch(rows=5)), b"same number of rows"), (lambda: rotary(ld=128), b"hold all heads"),
                        (lambda: rotary(dim=60), b"multiple of 16"), (lambda: rotary(r=rot(columns=12)), b"are rotated"), (lambda: rotary(r=rot(rows=0)), b"no tables"),
                        (lambda: rotary(r=rot(dtype=3)), b"tables are"), (lambda: append(q=8200), b"16-byte"), (lambda: append(cache(page_size=24)), b"power of two"),
                        (lambda: append(heads=0), b"multiple of 16"), (lambda: append(cache(k=4098)), b"16-byte"), (lambda: append(cache(k=None)), b"no memory"),
                        (lambda: append(cache(dtype=1)), b"bf16 or fp16"), (lambda: attend(cache(pages=2 ** 30)), b"2^31 - 1 rows"),
                        (lambda: attend(ws=None), b"256-byte"), (lambda: attend(cache(table_cols=2 ** 30)), b"65536"), (lambda: attend(ws=4100), b"256-byte"),
                        (lambda: attend(window=-1), b"window"), (lambda: attend(heads=3), b"multiple of kv_heads"), (lambda: attend(q=None), b"16-byte"),
                        (lambda: attend(cache(head_dim=32)), b"64 or 128"), (lambda: attend(cache(ld_k=120)), b"kv_heads heads"),
                        (lambda: lib.mk_paged_attention_workspace(0, 3, 2, 64, 1), b"multiple of kv_heads"),
                        (lambda: lib.mk_paged_attention_workspace(0, 4, 2, 96, 1), b"64 or 128")):
        assert call() == -2 and words in lib.mk_last_cuda_error(), (words, lib.mk_last_cuda_error())


# -- chunks: windows over values that are no numbers, far contexts -----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("D,H,KVH,dtype,page", [(64, 4, 2, BF, 16), (128, 4, 1, HALF, 128), (64, 3, 3, HALF, 64), (128, 2, 2, BF, 256)])
@pytest.mark.parametrize("window", [1, 30, 100, 128, 200, 300])
@pytest.mark.parametrize("new", [3, 140, 256, 300])
def test_window_over_values_not_finite(cuda, D, H, KVH, dtype, page, window, new):
    """Infinite values and ones that are no numbers anywhere in a chunk and the window in front of it: for the tokens whose window holds them what the definition
    gives, for those in front of them and those whose window has passed them nothing."""
    pos = [300, 77]
    args, kw = make_attention(pos, [new, new], H, KVH, D, page, dtype, seed=new + window)
    n, g, v = args["k_cache"].shape[0] // page, torch.Generator().manual_seed(window), args["v_cache"]
    for s, p in enumerate(pos):
        for i, at in enumerate(torch.randint(max(0, p - window), p + new, (9,), generator=g).tolist()):
            v[ref.cache_row(args["pages"], s, at, page, n), i::11] = (float("inf"), float("-inf"), float("nan"))[i % 3]
    got = mc.paged_attention(**on(cuda, args), **kw, window=window).cpu().double()
    want = ref.paged_attention(**args, **kw, window=window)[0]
    finite = torch.isfinite(want)
    clean = dict(args, v_cache=torch.where(torch.isfinite(v), v, torch.zeros((), dtype=dtype)))
    _, mag, size = ref.paged_attention(**clean, **kw, window=window)
    tol = attention_tolerance(want, mag, size, dtype, D, args["pages"].shape[1] * page, float(clean["v_cache"].double().abs().max()))
    close(got[finite], want[finite], tol[finite])
    for f in (torch.isposinf, torch.isneginf, torch.isnan):
        assert torch.equal(f(got), f(want))


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,KVH,new,window", [(64, 8, 2, 509, 0), (128, 4, 1, 300, 0), (64, 8, 2, 130, 5000), (128, 16, 2, 1, 0), (64, 4, 4, 17, 0)])
def test_far_context(cuda, D, H, KVH, new, window):
    """Tokens behind 16001 others, against 64 bits on the GPU."""
    page, ctx = 128, 16001
    args, kw = make_attention([ctx], [new], H, KVH, D, page, BF, seed=new)
    a = on(cuda, args)
    got = mc.paged_attention(**a, **kw, window=window)
    idx = torch.arange(ctx + new, device=cuda)
    rows = a["pages"][0].long()[idx // page] * page + idx % page
    at = torch.arange(ctx, ctx + new, device=cuda)[:, None]
    hidden = (idx[None] > at) | (idx[None] <= at - (window or 2 ** 40))
    for h in range(H):
        j = h // (H // KVH)
        k, v = (a[x][rows][:, j * D:(j + 1) * D].double() for x in ("k_cache", "v_cache"))
        x = a["q"][:, h * D:(h + 1) * D].double()
        w = torch.softmax((x @ k.T * D ** -0.5).masked_fill(hidden, float("-inf")), -1)
        want, mag = (w @ v).cpu(), (w @ v.abs()).cpu()
        size = torch.full_like(want, float((x.abs() @ k.abs().T).max()) * D ** -0.5)
        # (the sum of more than a thousand probabilities: w each)
        close(got[:, h * D:(h + 1) * D], want, attention_tolerance(want, mag, size, BF, D, ctx + new, 6.0) + ((ctx + new) * W) * mag)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk,steps", [(0, 9), (4, 5), (6, 3), (100, 9)])
def test_command_counts_its_steps(cuda, monkeypatch, capsys, chunk, steps):
    """The command's time of a step is over the steps it takes: the tokens that go in chunks are none of them."""
    from megacute_b200 import checkpoint
    from tests.test_checkpoint import CFG, hf_state_dict
    monkeypatch.setattr(checkpoint, "load_local", lambda path: (CFG, hf_state_dict(CFG, seed=5)))
    checkpoint.main(["--model", "here", "--prompt-ids", "1,2,3,4,5,6,7", "--tokens", "3", "--max-seq", "128", "--prompt-chunk", str(chunk)])
    lines = capsys.readouterr().out.splitlines()
    want = [f"{9 - steps} prompt tokens x batch 1 in chunks"] * (steps < 9) + [f"{steps} steps x batch 1"]
    assert [s.split(":")[0] for s in lines[:-1]] == want and len(eval(lines[-1])) == 3
