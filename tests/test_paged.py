"""Rotation, paged append and paged attention against their definitions in 64 bits (oracle/paged_oracle.py).

Tolerances, from the arithmetic.  u is half a step of the type (finfo.eps / 2), w = 2^-24 that of fp32.
  rotation: two products and a sum in fp32, each off by at most w of the products' magnitudes: 3 w (|a c| + |b s|) in all; then one rounding, u
    of the result; a result below the type's normal range is off by half of its smallest step.
  attention: one rounding of the result, u |y|.  A probability is rounded to the type (u of it).  A score of D products summed in fp32 is off by at
    most (D + 4) w times the sum of the products' magnitudes, in every order; it goes through 2^(s log2(e)), whose argument is off by two further
    roundings (of the scaled score and of the difference, 2 w of its size, itself at most the scaled magnitudes) and whose value by 2^-18.5 (the
    polynomial that replaces some of the hardware's approximations, which are closer).  The sum of probabilities has these errors too, and those of at
    most n + 64 additions, w each, taken here as 2^-14 for all n up to a thousand; 2^-14 + 2 * 2^-18.5 is below 2^-13: so every weight is off by
    u + 2 (D + 6) w S + 2^-13, S the largest sum of magnitudes, and the result by that times sum_j w_j |v_j|.  fp16 probabilities below the normal range: half a smallest step (2^-25) each, of a largest probability of at least one.
"""
import ctypes

import pytest
import torch

import megacute_b200 as mc
from megacute_b200 import _lib, paged
from oracle import paged_oracle as ref

BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32
W = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half of the smallest step of a type (below its normal range)."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def close(got, want, tol):
    got = got.detach().cpu().double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off; worst {((got - want).abs() / tol.clamp_min(1e-300))[bad].max():.2f} tolerances"


def rotation_tolerance(want, mag, dtype):
    return half_step(dtype) * (want.abs() + 3 * W * mag) + 3 * W * mag + smallest(dtype)


def attention_tolerance(want, mag, size, dtype, head_dim, keys, vmax):
    per = half_step(dtype) + 2 * (head_dim + 6) * W * size + 2.0 ** -13
    under = keys * 2.0 ** -25 * vmax if dtype == HALF else 0.0
    return half_step(dtype) * want.abs() + (1 + half_step(dtype)) * (per * mag + under) + smallest(dtype)


def tables(rows, n, dtype=F32, theta=10000.0):
    return mc.rotary_tables(rows, 2 * n, theta, dtype=dtype)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make_pages(need, width, page_size, g, spare=3):
    """A page table of `need` rows of each sequence in pages that lie anywhere; the number of pages."""
    counts = [-(-n // page_size) for n in need]
    order = torch.randperm(sum(counts) + spare, generator=g).int()
    pages = torch.full((len(need), width), -1, dtype=torch.int32)
    used = 0
    for s, c in enumerate(counts):
        pages[s, :c] = order[used:used + c]
        used += c
    return pages, sum(counts) + spare


def make_attention(pos, new, H, KVH, D, page_size, dtype, seed=0, starts=True, head_rows=0, tail_rows=0, qstd=1.3, width=None):
    """Arguments of paged_attention on the CPU: packed batch with `head_rows` rows in front and `tail_rows` behind."""
    g = gen(seed)
    b = [head_rows]
    for n in new:
        b.append(b[-1] + n)
    need = [max(0, p + n) for p, n in zip(pos, new)]
    width = width or max(1, max(-(-n // page_size) for n in need))
    pages, n_pages = make_pages(need, width, page_size, g)
    rows = n_pages * page_size
    r = lambda m, c, std: (torch.randn(m, c, generator=g) * std).to(dtype)
    args = dict(q=r(b[-1] + tail_rows, H * D, qstd), k_cache=r(rows, KVH * D, 1.3), v_cache=r(rows, KVH * D, 1.0),
                pos=torch.tensor(pos, dtype=torch.int32).reshape(-1, 1), pages=pages,
                starts=torch.tensor(b, dtype=torch.int32) if starts else None)
    return args, dict(heads=H, kv_heads=KVH, head_dim=D, page_size=page_size)


def on(dev, d):
    return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in d.items()}


def check_attention(dev, args, kw, out=None, got=None):
    a = on(dev, args)
    if got is None:
        o = None if out is None else out.to(dev)
        got = mc.paged_attention(**a, **kw, out=o)
    want, mag, size = ref.paged_attention(**args, **kw, out=out)
    v = args["v_cache"].double()
    vmax = float(v[torch.isfinite(v)].abs().max()) if v.numel() else 0.0
    covered = torch.zeros(want.shape[0], dtype=torch.bool)
    for r, _, _ in ref.batch_rows(want.shape[0], args["pos"], args["starts"]):
        covered[r] = True
    tol = attention_tolerance(want, mag, size, args["q"].dtype, kw["head_dim"], args["pages"].shape[1] * kw["page_size"], vmax)
    close(got.cpu()[covered], want[covered], tol[covered])
    if out is not None:
        assert torch.equal(got.cpu()[~covered], out[~covered])                # rows without a sequence: as they were
    empty = covered & (mag.sum(1) == 0)
    assert (got.cpu()[empty] == 0).all()                                       # rows that see nothing: zeros exactly
    return got


# -- rotary -------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,tdtype,H,D,n", [(BF, BF, 4, 64, 32), (BF, F32, 3, 128, 48), (HALF, F32, 5, 64, 16), (F32, F32, 2, 128, 64),
                                                (F32, BF, 1, 16, 8), (BF, HALF, 33, 80, 24), (HALF, HALF, 7, 256, 128)])
def test_rotary(cuda, dtype, tdtype, H, D, n, interleaved):
    g = gen(H * 100 + D)
    pos, bounds = torch.tensor([[0], [517], [3], [1021], [-2]], dtype=torch.int32), torch.tensor([1, 2, 2, 40, 45, 48], dtype=torch.int32)
    cos, sin = tables(1024, n, tdtype)                                         # (row 4 of sequence 3 is behind the tables, two rows in front of them)
    x = torch.randn(50, H * D, generator=g).to(dtype)
    out = torch.full_like(x, 7.0)
    kw = dict(heads=H, head_dim=D, interleaved=interleaved)
    want = ref.rotary(x, cos, sin, pos, bounds, out=out, **kw)
    mag = ref.rotary(x.double().abs(), cos.abs(), -sin.abs(), pos, bounds, **kw).abs() + ref.rotary(x.double().abs(), cos.abs(), sin.abs(), pos, bounds, **kw).abs()
    d = [t.to(cuda) for t in (x, cos, sin, pos, bounds)]
    got = mc.rotary(*d, out=out.to(cuda), **kw)
    close(got, want, rotation_tolerance(want, mag, dtype))
    assert torch.equal(got.cpu()[[0, 48, 49]], out[[0, 48, 49]])               # rows without a sequence: as they were
    assert (got.cpu()[[44, 45, 46]] == 0).all()                                # position 1024, -2 and -1
    rest = got.cpu()[1:40].view(-1, H, D)[..., 2 * n:]
    assert torch.equal(rest, x[1:40].view(-1, H, D)[..., 2 * n:])              # the rest of the head: copied
    again = mc.rotary(d[0].clone(), *d[1:], **kw)
    assert torch.equal(again[1:48], got[1:48])
    inplace = d[0].clone()
    assert mc.rotary(inplace, *d[1:], out=inplace, **kw) is inplace
    assert torch.equal(inplace[1:48], got[1:48]) and torch.equal(inplace[48:], d[0][48:])


@pytest.mark.gpu
def test_rotary_matches_graph_rope(cuda):
    """The same rotation as Graph.rope with the graph's own tables (their first half of columns)."""
    from megacute_b200 import workloads as Wl
    H, D, S = 4, 64, 37
    cos, sin = Wl.rope_tables(S, D, device=cuda)
    x = torch.randn(S, H * D, generator=gen(3)).to(BF).to(cuda)
    g = mc.Graph()
    g.output(g.rope(g.input("x", (S, H * D)), g.input("cos", (S, D)), g.input("sin", (S, D)), H, D, S))
    want = mc.compile(g)(x=x, cos=cos, sin=sin)
    got = mc.rotary(x, cos[:, :D // 2], sin[:, :D // 2], torch.zeros(1, 1, dtype=torch.int32, device=cuda), heads=H, head_dim=D)
    step = torch.maximum(got.float().abs(), want.float().abs()) * 2 ** -7      # one rounding each: at most a whole step apart
    assert ((got.float() - want.float()).abs() <= step + 1e-6).all()


def test_rotary_tables_scalings():
    """Angles of far positions from fp64, and each scaling at the frequencies where its definition is plain."""
    cos, sin = mc.rotary_tables(200_001, 64, 500000.0)
    p = 200_000.0
    import math
    for i in (0, 5, 31):
        a = p * 500000.0 ** (-2 * i / 64)
        assert abs(float(cos[200_000, i]) - math.cos(a)) < 1e-7 and abs(float(sin[200_000, i]) - math.sin(a)) < 1e-7
    inv, one = mc.rotary_frequencies(64, 10000.0)
    assert one == 1.0 and float(inv[0]) == 1.0
    lin, _ = mc.rotary_frequencies(64, 10000.0, {"type": "linear", "factor": 4.0})
    assert torch.allclose(lin * 4, inv)
    dyn, _ = mc.rotary_frequencies(64, 10000.0, {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048}, max_pos=2048)
    assert torch.allclose(dyn, inv)                                            # not longer than the original: as it is
    dyn, _ = mc.rotary_frequencies(64, 10000.0, {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048}, max_pos=8192)
    assert torch.allclose(dyn[-1], inv[-1] / 7.0) and float(dyn[0]) == 1.0     # 2 * 4 - 1 times slower at the slow end
    ll = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}
    got, _ = mc.rotary_frequencies(128, 500000.0, ll)
    from megacute_b200.checkpoint import rope_inverse_frequencies
    want = rope_inverse_frequencies(dict(hidden_size=128, num_attention_heads=1, rope_theta=500000.0, rope_scaling=ll))
    assert torch.allclose(got, want, rtol=1e-12)
    y, f = mc.rotary_frequencies(128, 10000.0, {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096})
    base, _ = mc.rotary_frequencies(128, 10000.0)
    assert abs(f - (0.1 * math.log(16.0) + 1.0)) < 1e-12
    turns = 4096 * base / (2 * math.pi)
    assert torch.allclose(y[turns > 33], base[turns > 33]) and torch.allclose(y[turns < 0.9], base[turns < 0.9] / 16)
    assert ((y <= base * (1 + 1e-12)) & (y >= base / 16 * (1 - 1e-12))).all()
    c, _ = mc.rotary_tables(4, 128, 10000.0, {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096})
    assert abs(float(c[0, 0]) - f) < 1e-6
    with pytest.raises(ValueError):
        mc.rotary_frequencies(64, 1e4, {"rope_type": "spiral", "factor": 2.0})
    with pytest.raises(ValueError):
        mc.rotary_frequencies(63)
    with pytest.raises(TypeError):
        mc.rotary_tables(8, 64, dtype=torch.int32)


# -- append -------------------------------------------------------------------------------------------------------------------
def make_append(pos, new, H, KVH, D, n, page_size, dtype, tdtype, seed, trows=None):
    args, kw = make_attention(pos, new, H, KVH, D, page_size, dtype, seed, head_rows=1, tail_rows=2)
    qkv = torch.randn(args["q"].shape[0], (H + 2 * KVH) * D, generator=gen(seed + 1)).to(dtype)
    cos, sin = tables(trows or max(p + m for p, m in zip(pos, new)) + 1, n, tdtype)
    del args["q"]
    return dict(qkv=qkv, cos=cos, sin=sin, **args), kw


def check_append(dev, args, kw, interleaved):
    a = on(dev, args)
    H, D = kw["heads"], kw["head_dim"]
    out = torch.full((args["qkv"].shape[0], H * D), 7.0, dtype=args["qkv"].dtype)
    q = mc.paged_append(**a, **kw, interleaved=interleaved, out=out.to(dev))
    want = ref.paged_append(**args, **kw, interleaved=interleaved, out=out)
    big = dict(args, qkv=args["qkv"].double().abs(), cos=args["cos"].abs(), sin=args["sin"].abs(), k_cache=args["k_cache"].abs() * 0, v_cache=args["v_cache"].abs() * 0)
    mag = ref.paged_append(**big, **kw, interleaved=interleaved)
    neg = ref.paged_append(**dict(big, sin=-big["sin"]), **kw, interleaved=interleaved)
    for got, w, m1, m2, before in zip((q, a["k_cache"], a["v_cache"]), want, mag, neg, (out, args["k_cache"], args["v_cache"])):
        close(got, w, rotation_tolerance(w, m1.abs() + m2.abs(), args["qkv"].dtype))
        same = (m1.abs().sum(1) == 0) & (w == before.double()).all(1)          # rows that nothing is written to: bit for bit
        assert torch.equal(got.cpu()[same], before[same])
    return q, a


APPENDS = [  # pos, new, H, KVH, D, n, page, dtype, table dtype
    ([5], [1], 4, 2, 64, 32, 16, BF, BF),
    ([0, 31, 100, 7, 200], [1, 1, 1, 1, 1], 8, 1, 128, 64, 32, BF, F32),
    ([0, 3, 250, 16], [70, 0, 33, 16], 6, 3, 64, 16, 64, HALF, F32),
    ([127], [130], 12, 12, 128, 48, 128, BF, F32),
    ([0, 0, 0], [0, 300, 0], 3, 1, 80, 40, 256, HALF, HALF),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", APPENDS)
def test_paged_append(cuda, case, interleaved):
    args, kw = make_append(*case, seed=len(case[0]))
    check_append(cuda, args, kw, interleaved)


@pytest.mark.gpu
def test_paged_append_skips(cuda):
    """Positions outside the tables and the page table, absent pages of every kind: nothing is written, and nothing beside them."""
    args, kw = make_append([0, 20, 60, 0, 40], [5, 20, 10, 40, 4], 4, 2, 64, 32, 16, BF, F32, 11, trows=64)
    n = args["k_cache"].shape[0] // 16
    args["pos"][0, 0], args["pos"][4, 0] = -3, 2 ** 31 - 3
    args["pages"][1, 1], args["pages"][3, 0], args["pages"][3, 2] = -1, n, 2 ** 31 - 1
    args["pages"] = args["pages"][:, :4].contiguous()                          # 64 rows: what is behind has no page
    check_append(cuda, args, kw, False)


@pytest.mark.gpu
def test_paged_append_strided(cuda):
    """Caches that are column ranges of one tensor, qkv and out with a pitch, one position column with a stride."""
    args, kw = make_append([3, 40], [30, 9], 4, 2, 64, 32, 16, BF, BF, 5)
    a = on(cuda, args)
    kv = torch.zeros(a["k_cache"].shape[0], 3 * 128 + 64, dtype=BF, device=cuda)
    kv[:, :128], kv[:, 192:320] = a["k_cache"], a["v_cache"]
    wide = torch.zeros(a["qkv"].shape[0], a["qkv"].shape[1] + 8, dtype=BF, device=cuda)
    wide[:, 8:] = a["qkv"]
    pos = torch.zeros(2, 3, dtype=torch.int32, device=cuda)
    pos[:, 1:2] = a["pos"]
    pages = torch.full((2, a["pages"].shape[1] + 5), -1, dtype=torch.int32, device=cuda)
    pages[:, :a["pages"].shape[1]] = a["pages"]
    q = torch.zeros(a["qkv"].shape[0], 304, dtype=BF, device=cuda)[:, 8:264]
    mc.paged_append(wide[:, 8:], a["cos"], a["sin"], pos[:, 1:2], kv[:, :128], kv[:, 192:320], pages[:, :a["pages"].shape[1]], a["starts"], **kw, out=q)
    b = on(cuda, args)
    want = mc.paged_append(**b, **kw)
    assert torch.equal(q[1:-2], want[1:-2]) and torch.equal(kv[:, :128], b["k_cache"]) and torch.equal(kv[:, 192:320], b["v_cache"])
    assert (kv[:, 128:192] == 0).all() and (kv[:, 320:] == 0).all()


# -- attention ----------------------------------------------------------------------------------------------------------------
SHAPES = [  # pos, new, H, KVH, D, page, dtype, window
    ([0], [1], 4, 2, 64, 16, BF, 0),                                           # one token, the first of all
    ([1023], [1], 8, 2, 64, 16, BF, 0),
    ([700, 0, 15, 16, 127, 128, 500], [1] * 7, 8, 2, 128, 16, BF, 0),          # ends of pages and tiles
    ([300, 77, 511], [1] * 3, 7, 1, 64, 64, HALF, 0),
    ([300, 77, 511], [1] * 3, 14, 2, 128, 32, BF, 100),
    ([600, 3], [1] * 2, 12, 12, 64, 128, HALF, 16),                            # one kv head per head
    ([260, 9, 70], [1] * 3, 16, 1, 128, 32, BF, 0),                            # 16 heads, one kv head
    ([260, 9], [1] * 2, 32, 1, 64, 16, BF, 0),                                 # 32 heads, one kv head
    ([260, 9], [2, 1], 40, 1, 64, 16, HALF, 64),
    ([200, 1, 400, 33], [4] * 4, 8, 2, 128, 32, HALF, 0),                      # speculative tokens
    ([200, 1, 400, 33], [5, 0, 3, 1], 6, 2, 64, 16, BF, 30),
    ([0, 0], [3, 17], 4, 4, 64, 16, BF, 1),                                    # window of one: V itself
    ([0], [300], 4, 2, 64, 64, BF, 0),                                         # a prompt from its start
    ([0, 0, 0, 0], [127, 128, 129, 257], 4, 1, 128, 128, BF, 0),
    ([333], [200], 8, 2, 64, 32, BF, 0),                                       # a chunk in the middle
    ([333, 50], [70, 131], 6, 2, 128, 16, HALF, 0),
    ([400, 0, 37], [90, 140, 1], 4, 1, 64, 256, BF, 64),                       # window over a chunk
    ([500, 0, 400, 60], [100, 1, 1, 33], 7, 1, 128, 64, BF, 200),              # chunks and single tokens
    ([100, 600], [66, 45], 3, 1, 64, 16, HALF, 0),
    ([150], [40], 9, 3, 128, 32, BF, 0),
    ([20, 300], [129, 64], 16, 16, 64, 64, HALF, 0),
    ([40], [50], 32, 1, 128, 16, BF, 0),
    ([0, 0, 0], [0, 0, 0], 4, 2, 64, 16, BF, 0),                               # no rows of any sequence
]


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [True, False])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_paged_attention(cuda, i, hint):
    """Every shape with and without the hint of how many rows a sequence has: with it, and a row per sequence or a few, the form for few rows."""
    pos, new, H, KVH, D, page, dtype, window = SHAPES[i]
    args, kw = make_attention(pos, new, H, KVH, D, page, dtype, seed=i, head_rows=2, tail_rows=3)
    out = torch.randn(args["q"].shape, generator=gen(1)).to(dtype)
    check_attention(cuda, args, dict(kw, window=window, max_new=max(new) if hint else None), out=out)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 1000])
@pytest.mark.parametrize("D,H,KVH,new", [(64, 4, 2, 1), (128, 8, 1, 3), (64, 32, 8, 70), (128, 4, 2, 200)])
def test_paged_attention_any_form(cuda, D, H, KVH, new, max_new):
    """A hint that is far off is right all the same; equal sequences without starts."""
    args, kw = make_attention([90, 5, 260], [new] * 3, H, KVH, D, 32, BF, seed=new)
    check_attention(cuda, args, dict(kw, max_new=max_new))
    check_attention(cuda, dict(args, starts=None), kw)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [0, -3])
@pytest.mark.parametrize("H,KVH", [(12, 1), (32, 2), (3, 3)])
def test_paged_attention_hint_below_one(cuda, H, KVH, max_new):
    """... is taken as one token, also where a group has more heads than half of an item has rows."""
    args, kw = make_attention([33, 0], [2, 1], H, KVH, 64, 16, BF, seed=8)
    check_attention(cuda, args, dict(kw, max_new=max_new))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 4, 150])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HALF)])
def test_paged_attention_absent_pages(cuda, D, dtype, new):
    """Pages that are not there: at the front (a window that has passed them), in the middle, all; positions in front of the sequence and behind
    the table.  What they would name must not be read: a page number outside the cache, and NaN in every row nobody owns."""
    pos = [300, 200, 64, -2, 400, 250]
    args, kw = make_attention(pos, [new] * 6, 8, 2, D, 16, dtype, seed=new)
    n = args["k_cache"].shape[0] // 16
    args["pages"][0, :9] = -1
    args["pages"][1, 3] = n
    args["pages"][1, 7:10] = 2 ** 31 - 1
    args["pages"][2] = -2 ** 31
    args["pages"] = args["pages"][:, :20].contiguous()                         # 320 rows: sequence 4 lies behind
    free = torch.ones(n * 16, dtype=torch.bool)
    for s in range(6):
        for p in range(pos[s] + new):
            row = ref.cache_row(args["pages"], s, p, 16, n)
            if row is not None:
                free[row] = False
    assert free.any()
    args["k_cache"][free], args["v_cache"][free] = float("nan"), float("inf")
    check_attention(cuda, args, kw)
    check_attention(cuda, args, dict(kw, window=40))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("rows,width", [(0, 3), (64, 0), (0, 0)])
def test_paged_attention_no_pages(cuda, new, rows, width):
    """A cache without pages, a page table without columns: nobody sees anything, nothing is appended."""
    q = torch.randn(2 * new, 256, generator=gen(1)).to(BF)
    args = dict(q=q, k_cache=torch.ones(rows, 128, dtype=BF), v_cache=torch.ones(rows, 128, dtype=BF), pos=torch.tensor([[5], [0]], dtype=torch.int32),
                pages=torch.zeros(2, width, dtype=torch.int32), starts=None)
    kw = dict(heads=4, kv_heads=2, head_dim=64, page_size=16)
    got = mc.paged_attention(**on(cuda, args), **kw)
    assert (got == 0).all()
    cos, sin = tables(64, 32)
    qkv = torch.randn(2 * new, 512, generator=gen(2)).to(BF)
    a = on(cuda, {k: v for k, v in args.items() if k != "q"})
    out = mc.paged_append(qkv.to(cuda), cos.to(cuda), sin.to(cuda), **a, **kw)
    want = ref.paged_append(qkv, cos, sin, **{k: v for k, v in args.items() if k != "q"}, **kw)[0]
    assert float((out.cpu().double() - want).abs().max()) < 0.02 and (a["k_cache"] == 1).all() and (a["v_cache"] == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [2, 4, 9, 140])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_paged_attention_later_tokens_not_finite(cuda, new, D, bad):
    """A key or value that is no number belongs to the tokens that see it: those in front of it in the same chunk stay as they are."""
    args, kw = make_attention([37, 200], [new, new], 4, 2, D, 16, BF, seed=new)
    k2 = dict(args, k_cache=args["k_cache"].clone(), v_cache=args["v_cache"].clone())
    where = [(0, 37 + new - 1), (1, 200 + new // 2)]
    for s, p in where:
        row = ref.cache_row(args["pages"], s, p, 16, args["k_cache"].shape[0] // 16)
        k2["v_cache"][row, 3::7] = bad
        k2["k_cache"][row, 5] = float("nan")
    got = mc.paged_attention(**on(cuda, k2), **kw).cpu()
    want, mag, size = ref.paged_attention(**args, **kw)
    tol = attention_tolerance(want, mag, size, BF, D, 256, float(args["v_cache"].double().abs().max()))
    clean = torch.tensor([p < where[s][1] for _, s, p in ref.batch_rows(2 * new, args["pos"], args["starts"])])
    close(got[clean], want[clean], tol[clean])
    assert torch.isnan(got[~clean][:, :2 * D]).all()                           # (kv head 0: their scores are no numbers)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 60])
def test_paged_attention_large_scores(cuda, new):
    """Scores up to a few hundred: the maximum is what is subtracted, and rises along the sequence."""
    args, kw = make_attention([500, 90], [new, new], 4, 2, 64, 16, BF, seed=3, qstd=20.0)
    for s in range(2):
        for p in range(0, 400, 7):
            row = ref.cache_row(args["pages"], s, p, 16, args["k_cache"].shape[0] // 16)
            if row is not None:
                args["k_cache"][row] *= 1 + p / 200
    check_attention(cuda, args, kw)
    check_attention(cuda, args, dict(kw, scale=-0.1))
    check_attention(cuda, args, dict(kw, scale=0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
def test_paged_attention_scores_of_minus_infinity(cuda, new, D):
    """A key whose score overflows to -inf has no weight, like one that is masked; a row of such keys alone becomes zeros."""
    args, kw = make_attention([300, 280], [new, new], 4, 2, D, 16, BF, seed=15)
    q, k = args["q"], args["k_cache"]
    q[:, 0] = 2.0 ** 120                                                       # head 0
    k[:, 0] = -2.0 ** 120                                                      # every key of its kv head
    got = mc.paged_attention(**on(cuda, args), **kw).cpu()
    assert (got[:, :D] == 0).all()
    assert torch.isfinite(got[:, 2 * D:]).all()
    rows = args["pages"][0, :4].repeat_interleave(16) * 16 + torch.arange(16).repeat(4)      # the first 64 rows of sequence 0
    k[rows.long(), 0] = 0.0
    got = mc.paged_attention(**on(cuda, args), **kw).cpu()[:new, :D]
    only = dict(args, q=q[:new], pos=torch.full((new, 1), 63, dtype=torch.int32), pages=args["pages"][:1].expand(new, -1).contiguous(), starts=None)
    only["q"] = only["q"].clone()
    only["k_cache"] = k.clone()
    only["k_cache"][:, 0] = 0.0
    want, mag, size = ref.paged_attention(**only, **kw)
    tol = attention_tolerance(want, mag, size, BF, D, 64, float(args["v_cache"].double().abs().max()))
    close(got, want[:, :D], tol[:, :D])


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_paged_attention_strided(cuda, new):
    """q a column range of qkv, caches column ranges of one tensor, a page table and an out with a pitch: the same bits as contiguous ones."""
    args, kw = make_attention([70, 300], [new, new], 8, 2, 64, 32, BF, seed=8)
    a = on(cuda, args)
    want = check_attention(cuda, args, kw)
    kv = torch.full((a["k_cache"].shape[0], 400), float("nan"), dtype=BF, device=cuda)
    kv[:, 8:136], kv[:, 136:264] = a["k_cache"], a["v_cache"]
    qkv = torch.full((a["q"].shape[0], 800), float("nan"), dtype=BF, device=cuda)
    qkv[:, 16:16 + 512] = a["q"]
    pages = torch.full((2, 40), -1, dtype=torch.int32, device=cuda)
    pages[:, 1:1 + a["pages"].shape[1]] = a["pages"]
    out = torch.zeros(a["q"].shape[0], 544, dtype=BF, device=cuda)
    mc.paged_attention(qkv[:, 16:528], kv[:, 8:136], kv[:, 136:264], a["pos"], pages[:, 1:1 + a["pages"].shape[1]], a["starts"], **kw, out=out[:, 8:520])
    assert torch.equal(out[:, 8:520], want) and (out[:, :8] == 0).all() and (out[:, 520:] == 0).all()


@pytest.mark.gpu
def test_paged_attention_far_rows(cuda):
    """Cache rows whose element offsets pass 32 bits, and a sequence whose pages lie at both ends of such a cache."""
    ld, D, KVH, page = 16384, 64, 2, 64
    n_pages = 2 ** 31 // ld // page + 40
    kv = torch.zeros(n_pages * page, ld, dtype=BF, device=cuda)
    k, v = kv[:, :KVH * D], kv[:, ld - KVH * D:]
    few = torch.tensor([n_pages - 1, 0, n_pages - 2, 1, n_pages - 3], dtype=torch.int64)
    rows = (few[:, None] * page + torch.arange(page)).flatten()
    g = gen(5)
    ks, vs = ((torch.randn(rows.numel(), KVH * D, generator=g) * 1.2).to(BF) for _ in range(2))
    k[rows.to(cuda)], v[rows.to(cuda)] = ks.to(cuda), vs.to(cuda)
    for new in (1, 33):
        q = torch.randn(new, 4 * D, generator=g).to(BF)
        pos = torch.tensor([[5 * page - new]], dtype=torch.int32)
        kw = dict(heads=4, kv_heads=KVH, head_dim=D, page_size=page)
        got = mc.paged_attention(q.to(cuda), k, v, pos.to(cuda), few.int()[None].to(cuda), **kw)
        small = dict(q=q, k_cache=ks, v_cache=vs, pos=pos, pages=torch.arange(5, dtype=torch.int32)[None], starts=None)
        check_attention(cuda, small, kw, got=got)
        cos, sin = tables(5 * page, 32)
        qkv = torch.randn(new, 8 * D, generator=g).to(BF)
        sc = dict(small, qkv=qkv, cos=cos, sin=sin)
        del sc["q"]
        want = ref.paged_append(**sc, **kw)
        mc.paged_append(qkv.to(cuda), cos.to(cuda), sin.to(cuda), pos.to(cuda), k, v, few.int()[None].to(cuda), **kw)
        at = rows[5 * page - new:].to(cuda)
        close(v[at], want[2][5 * page - new:], torch.zeros(1, dtype=torch.float64))
        close(k[at], want[1][5 * page - new:], half_step(BF) * want[1][5 * page - new:].abs() + 1e-5)
        ks[5 * page - new:], vs[5 * page - new:] = k[at].cpu(), v[at].cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("new,seqs,ctx", [(1, 1, 5000), (1, 70, 300), (3, 2, 2500), (200, 1, 3000), (33, 40, 100), (16, 16, 1500), (1, 900, 40),
                                          (2, 900, 60)])
@pytest.mark.parametrize("hint", [False, True])
def test_paged_attention_repeats(cuda, new, seqs, ctx, hint):
    """Long and many sequences, against 64-bit torch on the GPU; a second call gives the same bits, on another stream beside other calls too."""
    H, KVH, D, page = 8, 2, 64, 32
    args, kw = make_attention([max(0, ctx - 13 * i) for i in range(seqs)], [new] * seqs, H, KVH, D, page, BF, seed=seqs)
    a = on(cuda, args)
    if hint:
        kw["max_new"] = new
    got = mc.paged_attention(**a, **kw)
    for s in range(0, seqs, max(1, seqs // 7)):
        p, b0 = int(args["pos"][s, 0]), int(args["starts"][s])
        idx = torch.arange(p + new, device=cuda)
        rows = a["pages"][s].long()[idx // page] * page + idx % page
        k = a["k_cache"][rows].double().view(-1, KVH, D).repeat_interleave(H // KVH, 1)
        v = a["v_cache"][rows].double().view(-1, KVH, D).repeat_interleave(H // KVH, 1)
        x = a["q"][b0:b0 + new].double().view(new, H, D)
        sc = torch.einsum("ihd,jhd->hij", x, k) * D ** -0.5
        sc = sc.masked_fill(idx[None] > torch.arange(p, p + new, device=cuda)[:, None], float("-inf"))
        w = torch.softmax(sc, -1)
        want, mag = (torch.einsum("hij,jhd->ihd", w, t).reshape(new, H * D).cpu() for t in (v, v.abs()))
        size = torch.full_like(want, float(torch.einsum("ihd,jhd->hij", x.abs(), k.abs()).max()) * D ** -0.5)
        # (the sum of more than a thousand probabilities: w each)
        tol = attention_tolerance(want, mag, size, BF, D, p + new, 6.0) + ((p + new) * W) * mag
        close(got[b0:b0 + new], want, tol)
    side = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for i in range(9):
        with torch.cuda.stream(side[i % 3]):
            outs.append(mc.paged_attention(**a, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, got) for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,KVH,dtype,window", [(64, 4, 4, BF, 0), (128, 8, 4, HALF, 0), (128, 14, 2, BF, 50), (64, 32, 8, BF, 0)])
def test_paged_attention_many_items(cuda, D, H, KVH, dtype, window):
    """More items than SMs by far, of one and two operand tiles and of one and several key tiles, one behind the other in a block: single tokens
    between chunks, sequences without rows."""
    seqs = 260
    pos = [(37 * i) % 300 for i in range(seqs)]
    new = [(1, 0, 40, 1, 1, 2, 90, 1, 1, 1, 1, 1, 9)[i % 13] for i in range(seqs)]
    new[17] = 200
    args, kw = make_attention(pos, new, H, KVH, D, 16, dtype, seed=D + H)
    for hint in (1, 200):
        got = mc.paged_attention(**on(cuda, args), **kw, window=window, max_new=hint).cpu()
        assert _lib.load().mk_paged_attention_status(0, torch.cuda.current_stream().cuda_stream) == 0
        for s in list(range(0, seqs, 23)) + [17, 18, 19]:
            r0, r1 = int(args["starts"][s]), int(args["starts"][s + 1])
            one = dict(args, q=args["q"][r0:r1], pos=args["pos"][s:s + 1], pages=args["pages"][s:s + 1], starts=None)
            if r1 > r0:
                check_attention(cuda, one, dict(kw, window=window), got=got[r0:r1])


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 33])
@pytest.mark.parametrize("H,max_new", [(128, 1000), (64, 1000), (16, 1)])
@pytest.mark.parametrize("pos,new", [([0], [150]), ([0, 500, 3, 40, 7], [100, 70, 0, 131, 1]), ([0] * 17, [3, 140] + [1] * 15)])
def test_paged_attention_many_items_of_a_sequence(cuda, pos, new, H, max_new, window):
    """Sequences of more items than a warp has lanes: an item is 2 or 4 tokens of one kv head, or (few rows) one."""
    args, kw = make_attention(pos, new, H, 1, 64, 16, BF, seed=len(pos) + H)
    check_attention(cuda, args, dict(kw, window=window, max_new=max_new))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 24])
def test_captured_steps_follow_their_arguments(cuda, new):
    """A captured append and attention: each replay works with the positions, pages and rows of its own time; two graphs beside each other."""
    H, KVH, D, page = 8, 2, 64, 16
    args, kw = make_append([30, 0, 90], [new] * 3, H, KVH, D, 32, page, BF, F32, 21, trows=256)
    args["starts"], args["qkv"] = None, args["qkv"][:3 * new].contiguous()
    width = 16
    args["pages"] = torch.cat([args["pages"], torch.full((3, width - args["pages"].shape[1]), -1, dtype=torch.int32)], 1)
    order = torch.randperm(3 * width, generator=gen(2)).int().view(3, width)
    rows = 3 * width * page
    a = on(cuda, dict(args, pages=order, k_cache=torch.zeros(rows, KVH * D, dtype=BF), v_cache=torch.zeros(rows, KVH * D, dtype=BF)))

    def step():
        q = mc.paged_append(**a, **kw)
        return mc.paged_attention(q, a["k_cache"], a["v_cache"], a["pos"], a["pages"], **kw)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step()
        graphs.append((g, y))
    k0 = a["k_cache"].clone()
    for turn, (g, y) in enumerate(graphs * 2):
        a["pos"].copy_(torch.tensor([[3 + turn], [100 - turn], [77]], dtype=torch.int32))
        a["pages"].copy_(torch.randperm(3 * width, generator=gen(turn)).int().view(3, width))
        a["qkv"].copy_(torch.randn(a["qkv"].shape, generator=gen(50 + turn)).to(BF))
        a["k_cache"].copy_(k0 + turn)
        keep = a["k_cache"].clone(), a["v_cache"].clone()
        g.replay()
        got = y.clone()
        a["k_cache"].copy_(keep[0])
        a["v_cache"].copy_(keep[1])
        assert torch.equal(got, step())
        cpu = {k: v.cpu() for k, v in a.items() if isinstance(v, torch.Tensor)}
        q = mc.rotary(a["qkv"][:, :H * D], a["cos"], a["sin"], a["pos"], heads=H, head_dim=D).cpu()
        check_attention(cuda, dict(q=q, k_cache=cpu["k_cache"], v_cache=cpu["v_cache"], pos=cpu["pos"], pages=cpu["pages"], starts=None), kw, got=got)


@pytest.mark.gpu
def test_generation_over_pages(cuda):
    """The operators as a server uses them: prompts in chunks of unlike lengths, then single tokens, sequences that share the pages of a common
    beginning; the cache stays what one append of everything gives, and each step's result that of the definition."""
    H, KVH, D, page, n = 8, 2, 64, 16, 32
    kw = dict(heads=H, kv_heads=KVH, head_dim=D, page_size=page)
    cos, sin = mc.rotary_tables(256, D, 10000.0, device=cuda)
    g = gen(77)
    k, v = (torch.zeros(40 * page, KVH * D, dtype=BF, device=cuda) for _ in range(2))
    pages = torch.full((3, 16), -1, dtype=torch.int32)
    pages[0, :10], pages[1, :10] = torch.arange(0, 10), torch.arange(10, 20)
    pages[2, :2], pages[2, 2:10] = pages[0, :2], torch.arange(20, 28)          # 32 tokens of sequence 0 begin sequence 2
    have, free = [0, 0, 32], 28
    steps = [[40, 17, 0], [33, 1, 20], [1, 1, 1], [0, 1, 1], [1, 50, 4], [1, 1, 1]]
    seen = [[], [], []]
    for new in steps:
        rows = sum(new)
        qkv = torch.randn(rows, (H + 2 * KVH) * D, generator=g).to(BF)
        b = [0]
        for m in new:
            b.append(b[-1] + m)
        pos, starts = torch.tensor(have, dtype=torch.int32).reshape(-1, 1), torch.tensor(b, dtype=torch.int32)
        d = dict(pos=pos.to(cuda), pages=pages.to(cuda), starts=starts.to(cuda))
        q = mc.paged_append(qkv.to(cuda), cos, sin, d["pos"], k, v, d["pages"], d["starts"], **kw)
        y = mc.paged_attention(q, k, v, d["pos"], d["pages"], d["starts"], max_new=max(new), **kw)
        check_attention(cuda, dict(q=q.cpu(), k_cache=k.cpu(), v_cache=v.cpu(), pos=pos, pages=pages, starts=starts), kw, got=y)
        for s in range(3):
            seen[s].append(qkv[b[s]:b[s + 1], H * D:])
            have[s] += new[s]
    seen[2].insert(0, torch.cat(seen[0])[:32])
    for s in range(3):
        kv = torch.cat(seen[s])
        kk = mc.rotary(kv[:, :KVH * D].contiguous().to(cuda), cos, sin, torch.zeros(1, 1, dtype=torch.int32, device=cuda), heads=KVH, head_dim=D)
        rows = torch.tensor([ref.cache_row(pages, s, p, page, 40) for p in range(have[s])], device=cuda)
        assert torch.equal(k[rows], kk) and torch.equal(v[rows].cpu(), kv[:, KVH * D:])


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 50])
def test_matches_the_graph_decode_ops(cuda, window):
    """One token per sequence: what Graph.rope_append and Graph.decode_attention give over a contiguous cache, which is a paged one whose pages
    lie one behind the other."""
    B, H, KVH, D, S = 3, 8, 2, 64, 256
    from megacute_b200 import workloads as Wl
    cos, sin = Wl.rope_tables(S, D, device=cuda)
    g = mc.Graph()
    qkv, c, s = g.input("qkv", (B, (H + 2 * KVH) * D)), g.input("cos", (S, D)), g.input("sin", (S, D))
    pos, kc, vc = g.state("pos", (B, 1), torch.int32), g.state("k_cache", (B * S, KVH * D)), g.state("v_cache", (B * S, KVH * D))
    kw = dict(heads=H, kv_heads=KVH, head_dim=D)
    g.output(g.decode_attention(g.rope_append(qkv, c, s, pos, kc, vc, max_seq=S, **kw), kc, vc, pos, max_seq=S, window=window, **kw))
    r = lambda m, n, seed: torch.randn(m, n, generator=gen(seed)).to(BF).to(cuda)
    x, k0, v0 = r(B, (H + 2 * KVH) * D, 1), r(B * S, KVH * D, 2), r(B * S, KVH * D, 3)
    p = torch.tensor([[5], [100], [255]], dtype=torch.int32, device=cuda)
    k1, v1 = k0.clone(), v0.clone()
    want = mc.compile(g)(qkv=x, cos=cos, sin=sin, pos=p, k_cache=k1, v_cache=v1).clone()
    pages = torch.arange(B * 2, dtype=torch.int32, device=cuda).view(B, 2)
    k2, v2 = k0.clone(), v0.clone()
    q = mc.paged_append(x, cos[:, :D // 2], sin[:, :D // 2], p, k2, v2, pages, page_size=128, **kw)
    got = mc.paged_attention(q, k2, v2, p, pages, page_size=128, window=window, **kw)
    assert torch.equal(v1, v2) and ((k1.float() - k2.float()).abs() <= k1.float().abs() * 2 ** -7 + 1e-6).all()
    assert float((got.float() - want.float()).norm() / want.float().norm()) < 1e-2


# -- refusals -----------------------------------------------------------------------------------------------------------------
def cpu_calls():
    a, kw = make_append([3, 40], [2, 3], 4, 2, 64, 32, 16, BF, F32, 1)
    b, _ = make_attention([3, 40], [2, 3], 4, 2, 64, 16, BF, 1)
    r = dict(x=b["q"], cos=a["cos"], sin=a["sin"], pos=b["pos"], starts=b["starts"])
    return {"rotary": (mc.rotary, r, dict(heads=4, head_dim=64)), "append": (mc.paged_append, a, kw), "attention": (mc.paged_attention, b, kw)}


REFUSED = [  # call, what is changed, exception, words of the message
    ("rotary", dict(x=lambda t: t[0]), ValueError, "2-D"),
    ("rotary", dict(x=lambda t: t.int()), TypeError, "dtype"),
    ("rotary", dict(x=lambda t: t[:, 64:]), ValueError, "columns"),
    ("rotary", dict(heads=0), ValueError, "heads"),
    ("rotary", dict(head_dim=60), ValueError, "head_dim"),
    ("rotary", dict(x=lambda t: t.t().contiguous().t()), ValueError, "stride"),
    ("rotary", dict(x=lambda t: torch.zeros(t.numel() + 8, dtype=BF)[1:1 + t.numel()].view(t.shape)), ValueError, "16-byte"),
    ("rotary", dict(cos=lambda t: t[:, :20], sin=lambda t: t[:, :20]), ValueError, "multiple of 8"),
    ("rotary", dict(cos=lambda t: torch.cat([t, t], 1), sin=lambda t: torch.cat([t, t], 1)), ValueError, "half the rotated part"),
    ("rotary", dict(cos=lambda t: t[:3]), ValueError, "one shape"),
    ("rotary", dict(cos=lambda t: t[:0], sin=lambda t: t[:0]), ValueError, "empty"),
    ("rotary", dict(pos=lambda t: t.long()), TypeError, "int32"),
    ("rotary", dict(pos=lambda t: t.flatten()), ValueError, "pos"),
    ("rotary", dict(pos=lambda t: t.t()), ValueError, "one column"),
    ("rotary", dict(starts=lambda t: t[:2]), ValueError, "one entry more"),
    ("rotary", dict(starts=lambda t: None), ValueError, "same number"),
    ("rotary", dict(out=lambda a: torch.zeros(4, 256, dtype=BF)), ValueError, "rows"),
    ("rotary", dict(out=lambda a: torch.zeros(a["x"].shape, dtype=F32)), TypeError, "dtype"),
    ("rotary", dict(out=lambda a: a["x"].flatten()[:16].expand(5, 16)), ValueError, "columns"),
    ("rotary", {}, ValueError, "CUDA"),
    ("append", dict(qkv=lambda t: t.float()), TypeError, "dtype"),
    ("append", dict(qkv=lambda t: t.half()), TypeError, "activations"),
    ("append", dict(k_cache=lambda t: t[:, :64]), ValueError, "columns"),
    ("append", dict(v_cache=lambda t: t[:32]), ValueError, "one shape"),
    ("append", dict(page_size=24), ValueError, "power of two"),
    ("append", dict(page_size=8), ValueError, "power of two"),
    ("append", dict(page_size=1024), ValueError, "whole pages"),
    ("append", dict(pages=lambda t: t.long()), TypeError, "int32"),
    ("append", dict(pages=lambda t: t[:1]), ValueError, "rows"),
    ("append", dict(k_cache=lambda t: None, v_cache=lambda t: None), ValueError, "shares memory"),
    ("append", {}, ValueError, "CUDA"),
    ("attention", dict(head_dim=32), ValueError, "head_dim"),
    ("attention", dict(heads=3), ValueError, "multiple"),
    ("attention", dict(window=-1), ValueError, "window"),
    ("attention", dict(q=lambda t: t.float()), TypeError, "dtype"),
    ("attention", dict(q=lambda t: t.half()), TypeError, "activations"),
    ("attention", dict(k_cache=lambda t: t[:1].expand(t.shape)), ValueError, "stride"),
    ("attention", dict(out=lambda a: a["q"]), ValueError, "shares memory"),
    ("attention", {}, ValueError, "CUDA"),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refusals(i):
    """Wrong arguments are refused before anything reaches the device: here CPU tensors, which are refused last."""
    call, change, exc, words = REFUSED[i]
    fn, args, kw = cpu_calls()[call]
    args, kw = dict(args), dict(kw)
    for k, f in change.items():
        if k == "out":
            kw["out"] = f(args)
        elif k in args:
            args[k] = f(args[k])
        else:
            kw[k] = f
    if "shares memory" in words and call == "append":
        kv = torch.zeros(64, 192, dtype=BF)
        args["k_cache"], args["v_cache"] = kv[:, :128], kv[:, 64:]
    with pytest.raises(exc, match=words):
        fn(**args, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("i", [i for i, r in enumerate(REFUSED) if r[3] != "CUDA"])
def test_refusals_of_device_tensors(cuda, i):
    """The same of tensors on the device, which the binding looks at first."""
    call, change, exc, words = REFUSED[i]
    fn, args, kw = cpu_calls()[call]
    args, kw = on(cuda, args), dict(kw)
    for k, f in change.items():
        if k == "out":
            kw["out"] = f(args).to(cuda)
        elif k in args:
            args[k] = f(args[k])
            if words == "16-byte":
                args[k] = torch.zeros(5 * 256 + 8, dtype=BF, device=cuda)[1:1 + 5 * 256].view(5, 256)
        else:
            kw[k] = f
    if "shares memory" in words and call == "append":
        kv = torch.zeros(64, 192, dtype=BF, device=cuda)
        args["k_cache"], args["v_cache"] = kv[:, :128], kv[:, 64:]
    with pytest.raises(exc, match=words):
        fn(**args, **kw)


def test_binding_refuses_other_objects():
    """None, no exception, for what is no tensor on a device; the callers' checks go on from there."""
    direct = paged._direct()
    assert direct is not None
    t = torch.zeros(4, 64, dtype=BF)
    for call, n in ((direct.rotary, 8), (direct.paged_append, 13), (direct.paged_attention, 13)):
        for args in ((), (None,) * n, (t,) * n, (1,) * n, ("x",) * n, (t, *[10 ** 30] * (n - 1)), (t,) * (n + 1)):
            assert call(*args) is None
    with pytest.raises(ValueError):
        direct.bind(1, 2, 3)


@pytest.mark.gpu
def test_binding_and_ctypes_agree(cuda, monkeypatch):
    """The calls that the binding takes, and the same through the checks in Python."""
    def calls():
        for dtype in (BF, HALF):
            for starts in (True, False):
                a, kw = make_append([3, 40, 7], [4, 4, 4], 4, 2, 64, 16, 16, dtype, F32, 3)
                kc, vc = a["k_cache"], a["v_cache"]
                a = on(cuda, dict(a, starts=a["starts"] if starts else None, k_cache=kc.clone(), v_cache=vc.clone()))
                for inter in (False, True):
                    yield mc.paged_append, a, dict(kw, interleaved=inter), ("k_cache", "v_cache")
                b, kw = make_attention([3, 40, 70], [4, 4, 4], 4, 2, 64, 16, dtype, 3, starts=starts)
                b = on(cuda, b)
                for more in ({}, dict(window=9, scale=0.3), dict(max_new=4), dict(scale=2, window=None), dict(max_new=0)):
                    yield mc.paged_attention, b, dict(kw, **more), ()
        x = torch.randn(6, 3 * 64, generator=gen(5)).to(cuda)[:, 64:]                             # (strided, fp32)
        cos, sin = (t.to(cuda) for t in tables(64, 24))
        yield mc.rotary, dict(x=x, cos=cos, sin=sin, pos=torch.tensor([[2], [9]], dtype=torch.int32, device=cuda)), dict(heads=2, head_dim=64), ()

    def results():
        got = []
        for fn, args, kw, state in calls():
            args = dict(args, **{k: args[k].clone() for k in state})
            y = fn(**args, **kw)
            got.append([y[1:13] if state else y, *[args[k] for k in state]])         # (appended rows 1 .. 12 have a sequence)
        return got

    used = []
    real = paged._direct()
    monkeypatch.setattr(paged, "_direct", lambda: type("D", (), {n: staticmethod(lambda *a, f=getattr(real, n): (used.append(f(*a)), used[-1])[1])
                                                                 for n in ("rotary", "paged_append", "paged_attention")}))
    first = results()
    assert len(used) == len(first) and all(y is not None for y in used)       # the binding took them all
    monkeypatch.setattr(paged, "_direct", lambda: None)
    for a, b in zip(first, results()):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_column_ranges_of_one_tensor_are_apart():
    """k and v side by side in one tensor are no overlap; the call gets as far as the device."""
    fn, args, kw = cpu_calls()["append"]
    kv = torch.zeros(args["k_cache"].shape[0], 256, dtype=BF)
    with pytest.raises(ValueError, match="CUDA"):
        fn(**dict(args, k_cache=kv[:, :128], v_cache=kv[:, 128:]), **kw)
    with pytest.raises(ValueError, match="CUDA"):
        fn(**dict(args, k_cache=kv[:, 128:], v_cache=kv[:, :128]), **kw)


def test_abi_refusals():
    """The C entries check what they are given by themselves (addresses here are never followed)."""
    lib = _lib.load()
    B = lambda **k: _lib.Batch(**{**dict(pos=4096, starts=None, pos_ld=1, rows=4, seqs=2), **k})
    R = lambda **k: _lib.Rotation(**{**dict(cos=4096, sin=4096, ld_cos=32, ld_sin=32, rows=8, columns=32, dtype=1, interleaved=0), **k})
    C = lambda **k: _lib.PagedCache(**{**dict(k=4096, v=4096, table=4096, ld_k=128, ld_v=128, table_ld=4, pages=4, page_size=16, table_cols=4,
                                              kv_heads=2, head_dim=64, dtype=0), **k})
    E = -2

    def attention(b=B(), c=C(), q=4096, ld_q=256, out=8192, ld_out=256, heads=4, window=0, ws=4096, nbytes=1 << 40):
        return lib.mk_paged_attention(0, b, c, q, ld_q, out, ld_out, heads, 1.0, window, 1, ws, nbytes, None)

    def append(b=B(), r=R(), c=C(), qkv=4096, ld=512, q=8192, ld_q=256, heads=4):
        return lib.mk_paged_append(0, b, r, c, qkv, ld, q, ld_q, heads, None)

    def rotary(b=B(), r=R(), x=4096, ld=256, out=8192, ld_out=256, dtype=0, heads=4, head_dim=64):
        return lib.mk_rotary(0, b, r, x, ld, out, ld_out, dtype, heads, head_dim, None)

    for bad in (B(rows=-1), B(seqs=-1), B(pos=None), B(pos_ld=-1), B(rows=5)):
        assert attention(bad) == append(bad) == rotary(bad) == E
    for bad in (C(k=None), C(table=None), C(page_size=24), C(page_size=8), C(pages=2 ** 30), C(table_cols=2 ** 30), C(table_ld=-1), C(kv_heads=0),
                C(ld_k=120), C(ld_v=130), C(k=4098), C(dtype=1)):
        assert attention(c=bad) == append(c=bad) == E, bad
    for bad in (R(cos=None), R(rows=0), R(columns=12), R(columns=40), R(dtype=3), R(ld_sin=30), R(sin=4100)):
        assert append(r=bad) == rotary(r=bad) == E
    assert attention(c=C(head_dim=32)) == attention(heads=3) == attention(window=-1) == attention(q=None) == attention(ld_q=252) == attention(out=8200) == E
    assert attention(ws=None) == attention(ws=4100) == E and attention(nbytes=1) < 0
    assert append(ld=504) == append(ld_q=128) == append(qkv=4104) == append(heads=0) == E
    assert rotary(dtype=3) == rotary(head_dim=60) == rotary(out=None) == rotary(ld=128) == E
    assert b"16-byte" in lib.mk_last_cuda_error() or lib.mk_last_cuda_error()
    assert lib.mk_paged_attention_workspace(0, 3, 2, 64, 1) == lib.mk_paged_attention_workspace(0, 4, 2, 96, 1) == E
    # nothing to do: nothing is launched
    none = B(rows=0)
    assert attention(none) == append(none) == rotary(none) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("batch,chunk", [(2, 16), (1, 3), (3, 64)])
def test_generator_prompt_in_chunks(cuda, batch, chunk):
    """LlamaGenerator feeding its prompt in chunks: the cache afterwards is that of the token-by-token prompt (both bf16, from
    activations rounded at other places), and the logits behind it are those of the plain forward pass."""
    from megacute_b200.checkpoint import LlamaGenerator, rope_tables_from_config
    from tests.helpers import TOL, rel_l2
    from tests.test_checkpoint import CFG, hf_forward, hf_state_dict
    sd = hf_state_dict(CFG, seed=5)
    prompt = torch.randint(0, CFG["vocab_size"], (71,), generator=gen(4)).tolist()
    one = LlamaGenerator(CFG, sd, batch=batch, max_seq=128, device=cuda)
    many = LlamaGenerator(CFG, sd, batch=batch, max_seq=128, device=cuda, prompt_chunk=chunk)
    fed = many.prefill(prompt[:-1])
    assert fed == 70 // chunk * chunk == int(many.state["pos"])
    for g, start in ((one, 0), (many, fed)):
        for tok in prompt[start:]:
            g.state["ids"].fill_(tok)
            logits = g.step()
        g.logits = logits.float().cpu()
    for name in ("k_cache", "v_cache"):
        a, b = (g.state[name].view(CFG["num_hidden_layers"], batch, 128, -1) for g in (one, many))
        assert rel_l2(b[:, :, :71].float().cpu(), a[:, :, :71].float().cpu()) < TOL and (b[:, :, 71:] == 0).all()
    cos, sin = rope_tables_from_config(CFG, 128)
    want = hf_forward(CFG, sd, prompt, cos, sin)[-1]
    for g in (one, many):
        assert rel_l2(g.logits[0], want) < TOL
    again = LlamaGenerator(CFG, sd, batch=batch, max_seq=128, device=cuda, prompt_chunk=chunk)
    assert again.generate(prompt, 5).shape == (batch, 5) and int(again.state["pos"]) == 75
    with pytest.raises(ValueError):
        again.prefill(prompt[:64])
