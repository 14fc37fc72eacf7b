"""The operators of a paged key/value cache, each one pass through its public entry point.

* ``rotary``     rotation of heads by their positions: both pair layouts, all or part of the head
* ``append``     rotation of q and k of new tokens, k and v written into the pages of their sequences (``paged_append``)
* ``attention``  new tokens against the cached rows of their sequences (``paged_attention``): single tokens, a few speculative
                 ones, chunks of prompts, whole prompts, and batches that mix them

A cache row holds the kv heads of one token side by side; a page is ``page`` rows one behind the other; a sequence's pages lie
anywhere in the cache.  Sequence ``s`` has ``pos[s]`` tokens in the cache before the call and brings ``starts[s + 1] - starts[s]``
new ones, which are rows of the packed batch.  Caches are filled with N(0, 1) rows, stale ones behind the sequences' ends among
them; queries and keys are scaled so that scores spread over a few units, as a trained model's do.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# (heads, kv heads): the repository's own two, one kv head per head, one kv head, groups that no power of two divides
HEADS = [(32, 8), (16, 4), (12, 12), (8, 1), (28, 4), (18, 6)]
THETA = 500000.0

# Largest amounts of work, which draw() keeps to.
MAX_TOKENS = 16384
MAX_CACHE_ROWS = 64 * 4096
MAX_ATTENTION_FLOPS = 280e9


def listed() -> list[dict]:
    return [
        # one token of one sequence in front of a contiguous cache: latency
        {"name": "rotary_1", "op": "rotary", "dtype": "bf16", "table": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64, "part": 64,
         "interleaved": False, "seqs": 1, "new": 1, "ctx": 1000, "spread": "even"},
        # the queries of many prompts of unlike lengths; neighbours paired, part of the head rotated, exact tables
        {"name": "rotary_chunks", "op": "rotary", "dtype": "bf16", "table": "fp32", "heads": 32, "kv_heads": 8, "head_dim": 128, "part": 96,
         "interleaved": True, "seqs": 5, "new": 3271, "ctx": 20000, "spread": "ragged"},
        # interactive chat, one user: the new token of one layer goes into its page
        {"name": "append_1", "op": "append", "dtype": "bf16", "table": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64, "part": 64,
         "interleaved": False, "seqs": 1, "new": 1, "ctx": 1000, "spread": "even", "page": 16},
        # a loaded server: one new token of each of 64 sequences, each with a length of its own
        {"name": "append_64", "op": "append", "dtype": "bf16", "table": "fp32", "heads": 16, "kv_heads": 4, "head_dim": 128, "part": 128,
         "interleaved": True, "seqs": 64, "new": 1, "ctx": 2900, "spread": "ragged", "page": 64},
        # four long prompts at once (the benchmark's prefill shape)
        {"name": "append_4x4096", "op": "append", "dtype": "bf16", "table": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64, "part": 64,
         "interleaved": False, "seqs": 4, "new": 4096, "ctx": 0, "spread": "even", "page": 128},
        # interactive chat, one user: latency
        {"name": "decode_1x1k", "op": "attention", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64, "seqs": 1, "new": 1,
         "ctx": 1024, "spread": "even", "page": 16, "window": 0},
        # one user with a long document in context
        {"name": "decode_1x16k", "op": "attention", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64, "seqs": 1, "new": 1,
         "ctx": 16384, "spread": "even", "page": 64, "window": 0},
        # a loaded server, sequences of unlike lengths
        {"name": "decode_64_ragged", "op": "attention", "dtype": "bf16", "heads": 16, "kv_heads": 4, "head_dim": 128, "seqs": 64, "new": 1,
         "ctx": 4096, "spread": "ragged", "page": 16, "window": 0},
        # speculative decoding: four proposed tokens of each sequence checked at once, fp16 activations
        {"name": "verify_9x4", "op": "attention", "dtype": "fp16", "heads": 16, "kv_heads": 4, "head_dim": 128, "seqs": 9, "new": 4,
         "ctx": 5003, "spread": "ragged", "page": 32, "window": 0},
        # the next chunk of a long prompt against what is cached of it
        {"name": "chunk_509_at_16k", "op": "attention", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64, "seqs": 1, "new": 509,
         "ctx": 16001, "spread": "even", "page": 64, "window": 0},
        # continuous batching: prompt chunks and single tokens in one call, layers with a sliding window and 128-wide heads
        {"name": "mixed_24_window", "op": "attention", "dtype": "bf16", "heads": 28, "kv_heads": 4, "head_dim": 128, "seqs": 24, "new": 700,
         "ctx": 6000, "spread": "mixed", "page": 32, "window": 1024},
        # four long prompts at once (the benchmark's prefill shape)
        {"name": "prompts_4x4096", "op": "attention", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64, "seqs": 4, "new": 4096,
         "ctx": 0, "spread": "even", "page": 128, "window": 0},
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], uniform over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(["rotary", "append", "attention", "attention", "attention"])
    heads, kv_heads = rng.choice(HEADS)
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "heads": heads, "kv_heads": kv_heads,
            "head_dim": rng.choice([64, 128]), "spread": rng.choice(["even", "ragged", "mixed"])}
    if op != "attention":
        case["seqs"] = _spread(rng, 1, 64)
        case["new"] = 1 if rng.random() < 0.3 else _spread(rng, 1, min(4096, MAX_TOKENS // case["seqs"]))
        case["ctx"] = _spread(rng, 1, MAX_CACHE_ROWS // 8 // case["seqs"] - case["new"])
        if op == "rotary" and rng.random() < 0.3:
            case["dtype"] = "fp32"
        case.update(table=rng.choice(["bf16", "fp32"]), part=rng.choice([case["head_dim"], case["head_dim"], case["head_dim"] // 4 * 3, 32]),
                    interleaved=rng.random() < 0.5)
        if op == "append":
            case["page"] = rng.choice([16, 32, 64, 128, 256])
        return case
    case.update(page=rng.choice([16, 32, 64, 128, 256]), window=rng.choice([0, 0, _spread(rng, 16, 4096)]))
    case["seqs"] = _spread(rng, 1, 64)
    case["new"] = rng.choice([1, 1, _spread(rng, 2, 8), _spread(rng, 9, 4096)])
    case["new"] = min(case["new"], MAX_CACHE_ROWS // case["seqs"] // 2, MAX_TOKENS // case["seqs"])
    case["ctx"] = _spread(rng, 16, min(32768, MAX_CACHE_ROWS // case["seqs"] - case["new"]))
    while work(case)["flops"] > MAX_ATTENTION_FLOPS:
        case["ctx"], case["new"] = (case["ctx"] // 2, case["new"]) if case["ctx"] > 1024 else (case["ctx"], case["new"] * 3 // 4)
    return case


def _lengths(case) -> tuple[list[int], list[int]]:
    """Tokens in the cache before the call and new tokens of each sequence.  even: all the same; ragged: contexts from a
    sixteenth to all of ``ctx``, new tokens from an eighth to all of ``new``; mixed: such contexts, one sequence in four with a
    chunk and the others with one new token."""
    b, ctx, new = case["seqs"], case["ctx"], case["new"]
    if case["spread"] == "even" or b == 1:
        return [ctx] * b, [new] * b
    pos = [ctx // 16 + (ctx - ctx // 16) * ((i * 5) % b) // (b - 1) for i in range(b)]
    if case["spread"] == "ragged":
        return pos, [max(1, new * (1 + i * 3 % 8) // 8) for i in range(b)]
    return pos, [new if i % 4 == 0 else 1 for i in range(b)]


def _tables(rows: int, part: int, dtype: torch.dtype, dev):
    inv = THETA ** -(torch.arange(0, part, 2, dtype=torch.float64, device=dev) / part)
    ang = torch.arange(rows, dtype=torch.float64, device=dev)[:, None] * inv
    return ang.cos().to(dtype), ang.sin().to(dtype)


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(rows, cols, std):
        return (torch.randn(rows, cols, generator=gen, device=dev) * std).to(dtype)

    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    pos, new = _lengths(case)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st = {"case": case, "op": case["op"], "host_pos": pos, "host_starts": starts,
          "pos": torch.tensor(pos, dtype=torch.int32, device=dev).reshape(-1, 1),
          "starts": torch.tensor(starts, dtype=torch.int32, device=dev), "even": len(set(new)) == 1, "max_new": max(new)}
    if case["op"] != "attention":
        st["cos"], st["sin"] = _tables(max(p + n for p, n in zip(pos, new)) + 1, case["part"], DTYPES[case["table"]], dev)
    if case["op"] == "rotary":
        st["x"] = randn(starts[-1], h * d, 1.0)
        return st
    page = case["page"]
    need = [-(-(p + n) // page) for p, n in zip(pos, new)]
    width = max(need)
    order = torch.randperm(sum(need) + 3, generator=gen, device=dev).to(torch.int32)     # (three pages belong to nobody)
    pages = torch.zeros(case["seqs"], width, dtype=torch.int32, device=dev)
    used = 0
    for s, n in enumerate(need):
        pages[s, :n] = order[used:used + n]
        used += n
    st["pages"] = pages
    rows = (sum(need) + 3) * page
    st["k_cache"], st["v_cache"] = randn(rows, kvh * d, 1.3), randn(rows, kvh * d, 1.0)
    if case["op"] == "append":
        st["qkv"] = randn(starts[-1], (h + 2 * kvh) * d, 1.0)
    else:
        st["q"] = randn(starts[-1], h * d, 1.3)
    return st


def run(state: dict):
    return _RUN[state["op"]](state)


# -- the framework's entry points
def _own_args(st):
    c = st["case"]
    return (None if st["even"] else st["starts"]), c["heads"], c["kv_heads"], c["head_dim"]


def _rotary(st):
    if not own:
        return _plain_rotary(st)
    import megacute_b200 as mc
    starts, h, _, d = _own_args(st)
    return mc.rotary(st["x"], st["cos"], st["sin"], st["pos"], starts, heads=h, head_dim=d, interleaved=st["case"]["interleaved"])


def _append(st):
    if not own:
        return _plain_append(st)
    import megacute_b200 as mc
    starts, h, kvh, d = _own_args(st)
    q = mc.paged_append(st["qkv"], st["cos"], st["sin"], st["pos"], st["k_cache"], st["v_cache"], st["pages"], starts, heads=h,
                        kv_heads=kvh, head_dim=d, page_size=st["case"]["page"], interleaved=st["case"]["interleaved"])
    return [q, st["k_cache"], st["v_cache"]]


def _attention(st):
    if not own:
        return _plain_attention(st)
    import megacute_b200 as mc
    starts, h, kvh, d = _own_args(st)
    return mc.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["pos"], st["pages"], starts, heads=h, kv_heads=kvh, head_dim=d,
                              page_size=st["case"]["page"], window=st["case"]["window"], max_new=st["max_new"])


_RUN = {"rotary": _rotary, "append": _append, "attention": _attention}


# -- plain forms, 32 bits
def _plain_positions(st) -> torch.Tensor:
    """Position of every row of the packed batch."""
    starts = st["starts"].long()
    row = torch.arange(st["host_starts"][-1], device=starts.device)
    seq = torch.repeat_interleave(torch.arange(len(st["host_pos"]), device=starts.device), starts[1:] - starts[:-1],
                                  output_size=st["host_starts"][-1])
    return seq, st["pos"].long()[seq, 0] + row - starts[seq]


def _plain_rotate(x, cos, sin, interleaved):
    """x (tokens, heads, head_dim) in 32 bits; cos and sin (tokens, 1, pairs)."""
    n = cos.shape[-1]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_rotary(st):
    c = st["case"]
    x = st["x"]
    _, p = _plain_positions(st)
    y = _plain_rotate(x.float().view(-1, c["heads"], c["head_dim"]), st["cos"][p].float()[:, None], st["sin"][p].float()[:, None],
                      c["interleaved"])
    return y.view_as(x).to(x.dtype)


def _plain_append(st):
    c = st["case"]
    h, kvh, d = c["heads"], c["kv_heads"], c["head_dim"]
    qkv = st["qkv"]
    seq, p = _plain_positions(st)
    qk = _plain_rotate(qkv[:, :(h + kvh) * d].float().view(-1, h + kvh, d), st["cos"][p].float()[:, None], st["sin"][p].float()[:, None],
                       c["interleaved"]).to(qkv.dtype)
    row = st["pages"].long()[seq, p // c["page"]] * c["page"] + p % c["page"]
    st["k_cache"][row] = qk[:, h:].reshape(-1, kvh * d)
    st["v_cache"][row] = qkv[:, (h + kvh) * d:]
    return [qk[:, :h].reshape(-1, h * d), st["k_cache"], st["v_cache"]]


def _plain_attention(st):
    c = st["case"]
    h, kvh, d, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    g, q = h // kvh, st["q"]
    out = torch.empty_like(q)
    for s, first in enumerate(st["host_pos"]):
        r0, r1 = st["host_starts"][s], st["host_starts"][s + 1]
        for a in range(r0, r1, 1024):
            b = min(r1, a + 1024)
            last = first + b - r0
            lo = max(0, first + a - r0 + 1 - c["window"]) if c["window"] else 0
            key = torch.arange(lo, last, device=q.device)
            row = st["pages"][s].long()[key // page] * page + key % page
            k = st["k_cache"][row].float().view(-1, kvh, d).permute(1, 2, 0)
            v = st["v_cache"][row].float().view(-1, kvh, d).permute(1, 0, 2)
            x = q[a:b].float().view(b - a, kvh, g, d).permute(1, 2, 0, 3).reshape(kvh, g * (b - a), d)
            score = (torch.matmul(x, k) * d ** -0.5).view(kvh, g, b - a, -1)
            p = torch.arange(first + a - r0, last, device=q.device)[:, None]
            hidden = key > p
            if c["window"]:
                hidden = hidden | (key <= p - c["window"])
            score = score.masked_fill(hidden, float("-inf"))
            e = torch.exp(score - score.amax(-1, keepdim=True))
            y = torch.matmul(e.view(kvh, g * (b - a), -1), v).view(kvh, g, b - a, d) / e.sum(-1, keepdim=True)
            out[a:b] = y.permute(2, 0, 1, 3).reshape(b - a, h * d).to(q.dtype)
    return out


# -- definitions in 64 bits, token by token of the packed batch or kv head by kv head
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    token_pos, token_seq = [], []
    for s, p in enumerate(st["host_pos"]):
        for i in range(st["host_starts"][s + 1] - st["host_starts"][s]):
            token_pos.append(p + i)
            token_seq.append(s)
    at = torch.tensor(token_pos, device=st["pos"].device)

    def turned(x):
        """The complex product (a + ib)(cos + i sin) of every pair."""
        n = case["part"] // 2
        first = torch.arange(n, device=x.device) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else n)
        y = x.double().clone()
        z = torch.complex(y[..., first], y[..., second]) * torch.complex(st["cos"].double()[at], st["sin"].double()[at])[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    if case["op"] == "rotary":
        return turned(st["x"].view(-1, h, d)).view(-1, h * d)
    page = case["page"]
    table = st["pages"].cpu().tolist()
    if case["op"] == "append":
        parts = st["qkv"].view(-1, h + 2 * kvh, d)
        qk = turned(parts[:, :h + kvh])
        rows = torch.tensor([table[s][p // page] * page + p % page for s, p in zip(token_seq, token_pos)], device=at.device)
        k, v = st["k_cache"].double(), st["v_cache"].double()
        k[rows], v[rows] = qk[:, h:].flatten(1), parts[:, h + kvh:].double().flatten(1)
        return [qk[:, :h].flatten(1), k, v]
    g, q = h // kvh, st["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for s, first in enumerate(st["host_pos"]):
        r0, r1 = st["host_starts"][s], st["host_starts"][s + 1]
        n, total = r1 - r0, first + r1 - r0
        rows = torch.tensor([table[s][i // page] * page + i % page for i in range(total)], device=q.device)
        for kv in range(kvh):
            k, v = (st[x][rows, kv * d:(kv + 1) * d].double() for x in ("k_cache", "v_cache"))
            for a in range(0, n, 2048):
                m = min(n, a + 2048) - a
                lo = max(0, first + a + 1 - case["window"]) if case["window"] else 0
                hi = first + a + m
                who = torch.arange(first + a, hi, device=q.device)
                what = torch.arange(lo, hi, device=q.device)
                seen = what[None] <= who[:, None]
                if case["window"]:
                    seen &= what[None] > who[:, None] - case["window"]
                for head in range(kv * g, (kv + 1) * g):
                    cols = slice(head * d, (head + 1) * d)
                    logit = q[r0 + a:r0 + a + m, cols].double() @ k[lo:hi].T / math.sqrt(d)
                    logit[~seen] = -math.inf
                    out[r0 + a:r0 + a + m, cols] = torch.exp(logit - torch.logsumexp(logit, 1, keepdim=True)) @ v[lo:hi]
    return out


def work(case: dict) -> dict:
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    size = DTYPES[case["dtype"]].itemsize
    pos, new = _lengths(case)
    tokens = sum(new)
    if case["op"] != "attention":
        # a table row of cosines and one of sines for each token
        tables = tokens * case["part"] * DTYPES[case["table"]].itemsize
        cols, turned = (h, h) if case["op"] == "rotary" else (h + 2 * kvh, h + kvh)
        return {"bytes": 2 * tokens * cols * d * size + tables + 4 * len(pos), "flops": 3 * tokens * turned * case["part"]}
    rows = pairs = 0
    for p, n in zip(pos, new):
        w = case["window"] or p + n
        rows += p + n - max(0, p + 1 - w)
        full = max(0, min(n, w - p - 1))                # tokens that see all rows up to their own
        pairs += full * p + full * (full + 1) // 2 + (n - full) * w
    return {"bytes": size * d * (2 * tokens * h + 2 * rows * kvh) + 4 * (rows // case["page"] + 2 * len(pos)), "flops": 4 * d * h * pairs}
