"""Operators over a paged key/value cache, each one call on the current stream of its tensors' device.

    cos, sin = mc.rotary_tables(max_pos, head_dim, theta=500000.0, scaling=config.get("rope_scaling"))
    q = mc.paged_append(qkv, cos, sin, pos, k_cache, v_cache, pages, starts, heads=H, kv_heads=KVH, head_dim=D, page_size=P)
    y = mc.paged_attention(q, k_cache, v_cache, pos, pages, starts, heads=H, kv_heads=KVH, head_dim=D, page_size=P)

``Graph.rope_append`` and ``Graph.decode_attention`` keep one contiguous cache and add one token per sequence inside a launch; these
take any number of new tokens of each sequence and find its rows through a page table, so that sequences grow, end and share pages
without a copy.  (The reference has no counterpart: its README.md:225-228 lists what its decode ops leave out.)

The conventions are the graph's: activations are (rows, features) with heads side by side, a cache row holds the kv heads of one
token, ``pos`` counts the tokens a sequence has before the call.

* ``k_cache``, ``v_cache``: (pages * page_size, kv_heads * head_dim) bf16 or fp16, rows ``[i * page_size, (i + 1) * page_size)`` are page
  ``i``; they may be column ranges of one tensor.  ``page_size`` is a power of two, at least 16.
* ``pages``: (sequences, n) int32; row ``p`` of sequence ``s`` is row ``p % page_size`` of page ``pages[s, p // page_size]``.  An entry outside
  the cache (-1, say) is an absent page: it is not written to, and its rows are not attended.
* ``pos``: (sequences, 1) int32.  ``starts``: None, every sequence has the same number of rows of the packed batch; or (sequences + 1,)
  int32, never decreasing, sequence ``s`` has rows ``[starts[s], starts[s + 1])``, possibly none.  Rows in front of the first sequence or behind the
  last one are left as they are (in a new ``out``: undefined).

Positions, starts and page tables are read on the device when the call runs: nothing synchronises, and a captured call replays with
what they hold then.  The contents are the caller's: a position or page outside its range is never followed out of memory, but gives zeros
or is skipped, as each function says.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .graph import DTYPE_CODE

_HALVES = (torch.bfloat16, torch.float16)
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None, max_pos: int | None = None):
    """Inverse frequencies of the ``rotary_dim / 2`` pairs, fp64, and the factor on cosines and sines.

    ``scaling`` is a ``rope_scaling`` dict of a Hugging Face config: type ``linear`` (angles divided by ``factor``), ``dynamic`` (theta raised
    so that the slowest pair covers ``max_pos`` positions), ``llama3`` (slow pairs stretched by ``factor``, a linear blend between the two
    corner wavelengths) or ``yarn`` (pairs below ``beta_slow`` turns over the original length stretched, those above ``beta_fast`` kept, a ramp over
    the pairs between; cosines and sines times ``attention_factor``, 0.1 ln(factor) + 1 by default)."""
    if rotary_dim < 4 or rotary_dim % 2:
        raise ValueError("rotary_frequencies: rotary_dim is even and at least 4")
    expo = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    inv = float(theta) ** -expo
    sc = scaling or {}
    kind = sc.get("rope_type", sc.get("type", "default"))
    if kind == "default":
        return inv, 1.0
    if kind not in ("linear", "dynamic", "llama3", "yarn"):
        raise ValueError(f"rotary_frequencies: unknown scaling {kind!r}")
    factor = float(sc["factor"])
    if kind == "linear":
        return inv / factor, 1.0
    orig = float(sc["original_max_position_embeddings"])
    if kind == "dynamic":
        length = max(float(max_pos or orig), orig)
        base = float(theta) * (factor * length / orig - (factor - 1.0)) ** (rotary_dim / (rotary_dim - 2))
        return base ** -expo, 1.0
    if kind == "llama3":
        lo, hi = float(sc["low_freq_factor"]), float(sc["high_freq_factor"])
        blend = ((orig * inv / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)          # 0: stretched, 1: as it is
        return (1.0 - blend) * inv / factor + blend * inv, 1.0
    def pair_with(turns):                        # the pair that turns so often over the original length
        return rotary_dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(float(theta)))
    first = max(math.floor(pair_with(float(sc.get("beta_fast", 32.0)))), 0)
    last = min(math.ceil(pair_with(float(sc.get("beta_slow", 1.0)))), rotary_dim - 1)
    ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
    attention = sc.get("attention_factor")
    if attention is None:
        attention = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return inv / factor * ramp + inv * (1.0 - ramp), float(attention)


def rotary_tables(max_pos: int, rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None, dtype: torch.dtype = torch.float32,
                  device=None):
    """cos and sin, (max_pos, rotary_dim / 2), of positions 0 .. max_pos - 1: angles in fp64, rounded once to ``dtype``.  ``scaling`` as in
    ``rotary_frequencies``.  (``checkpoint.rope_tables_from_config`` makes the graph's tables, which hold each column twice; their
    first half of columns serves here too.)"""
    if dtype not in _FLOATS:
        raise TypeError(f"rotary_tables: unsupported dtype {dtype}")
    inv, factor = rotary_frequencies(rotary_dim, theta, scaling, max_pos)
    ang = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv.to(device)[None]
    return (ang.cos() * factor).to(dtype), (ang.sin() * factor).to(dtype)


# -- arguments
def _rows(what, name, t, dtypes, device=None, cols=None):
    """A (rows, cols) tensor whose rows start on 16-byte boundaries."""
    if t.dim() != 2:
        raise ValueError(f"{what}: {name} is 2-D")
    if t.dtype not in dtypes:
        raise TypeError(f"{what}: {name} has unsupported dtype {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{what}: {name} is on {t.device}, the others on {device}")
    if cols is not None and t.shape[1] != cols:
        raise ValueError(f"{what}: {name} has {t.shape[1]} columns, expected {cols}")
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]) or \
            t.stride(0) * t.element_size() % 16 or t.data_ptr() % 16:
        raise ValueError(f"{what}: {name} needs unit inner stride and rows that start on 16-byte boundaries")
    return t


def _row_stride(t) -> int:
    """Elements between rows; a single row's stride says nothing."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _ints(what, name, t, device, dim):
    if t.dtype != torch.int32:
        raise TypeError(f"{what}: {name} is int32")
    if t.device != device or t.dim() != dim or t.stride(0) < 0 or (t.shape[dim - 1] > 1 and t.stride(dim - 1) != 1):
        raise ValueError(f"{what}: {name} is a {dim}-D tensor on {device} with unit inner stride")


def _batch(what, rows, pos, starts, device) -> _lib.Batch:
    _ints(what, "pos", pos, device, 2)
    seqs = pos.shape[0]
    if pos.shape[1] != 1:
        raise ValueError(f"{what}: pos has one column, one row per sequence")
    if starts is not None:
        _ints(what, "starts", starts, device, 1)
        if starts.shape[0] != seqs + 1:
            raise ValueError(f"{what}: starts has one entry more than there are sequences")
    elif (rows % seqs if seqs else rows):
        raise ValueError(f"{what}: {rows} rows for {seqs} sequences: without starts every sequence has the same number")
    return _lib.Batch(pos.data_ptr(), None if starts is None else starts.data_ptr(), pos.stride(0), rows, seqs)


def _rotation(what, cos, sin, interleaved, head_dim, device) -> _lib.Rotation:
    for name, t in (("cos", cos), ("sin", sin)):
        _rows(what, name, t, _FLOATS, device)
    if cos.shape != sin.shape or cos.dtype != sin.dtype:
        raise ValueError(f"{what}: cos and sin have one shape and dtype")
    n = cos.shape[1]
    if n % 8 or n == 0 or 2 * n > head_dim:
        raise ValueError(f"{what}: cos has {n} columns: half the rotated part of a head of {head_dim}, a multiple of 8")
    if cos.shape[0] == 0:
        raise ValueError(f"{what}: empty tables")
    return _lib.Rotation(cos.data_ptr(), sin.data_ptr(), _row_stride(cos), _row_stride(sin), cos.shape[0], n, DTYPE_CODE[cos.dtype],
                         1 if interleaved else 0)


def _cache(what, k_cache, v_cache, pages, seqs, kv_heads, head_dim, page_size, dtype, device) -> _lib.PagedCache:
    if kv_heads <= 0:
        raise ValueError(f"{what}: kv_heads is positive")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _rows(what, name, t, _HALVES, device, kv_heads * head_dim)
        if t.dtype != dtype:
            raise TypeError(f"{what}: {name} is {t.dtype}, the activations {dtype}")
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"{what}: page_size is a power of two from 16 up")
    if k_cache.shape != v_cache.shape or k_cache.shape[0] % page_size:
        raise ValueError(f"{what}: k_cache and v_cache have one shape, whole pages of {page_size} rows")
    _ints(what, "pages", pages, device, 2)
    if pages.shape[0] != seqs:
        raise ValueError(f"{what}: pages has {pages.shape[0]} rows, pos {seqs}")
    if max(k_cache.shape[0], pages.shape[1] * page_size) > 2 ** 31 - 1:
        raise ValueError(f"{what}: at most 2^31 - 1 rows in the cache and of a sequence")
    return _lib.PagedCache(k_cache.data_ptr(), v_cache.data_ptr(), pages.data_ptr(), _row_stride(k_cache), _row_stride(v_cache),
                           pages.stride(0), k_cache.shape[0] // page_size, page_size, pages.shape[1], kv_heads, head_dim, DTYPE_CODE[dtype])


def _out(what, out, like, cols):
    if out is None:
        return torch.empty(like.shape[0], cols, dtype=like.dtype, device=like.device)
    _rows(what, "out", out, (like.dtype,), like.device, cols)
    if out.shape[0] != like.shape[0]:
        raise ValueError(f"{what}: out has {like.shape[0]} rows")
    return out


def _span(t) -> tuple[int, int]:
    """First and last byte address of a (rows, cols) tensor."""
    if t.numel() == 0:
        return (0, -1)
    return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size() - 1


def _apart(what, name, written, *read):
    """Refuse outputs that share memory with what the call reads (column ranges of one tensor are apart)."""
    a0, a1 = _span(written)
    for t in read:
        b0, b1 = _span(t)
        if a0 > b1 or b0 > a1:
            continue
        pitch = written.stride(0) * written.element_size()
        if pitch and pitch == t.stride(0) * t.element_size():        # both in one grid of rows: compare the column ranges
            at, wa, wb = (b0 - a0) % pitch, written.shape[1] * written.element_size(), t.shape[1] * t.element_size()
            if at >= wa and at + wb <= pitch:
                continue
        raise ValueError(f"{what}: {name} shares memory with an operand")


def _stream(what, device):
    if device.type != "cuda":
        raise ValueError(f"{what}: expected CUDA tensors")
    return torch.cuda.current_stream(device).cuda_stream


def _heads(what, heads, head_dim):
    if heads <= 0 or head_dim <= 0 or head_dim % 16:
        raise ValueError(f"{what}: heads is positive and head_dim a multiple of 16")


# -- the operators
def rotary(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, starts: torch.Tensor | None = None, *, heads: int,
           head_dim: int, interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate ``heads`` heads of each row of x (rows, heads * head_dim; bf16, fp16 or fp32) by its position: ``Graph.rope`` outside a
    launch, at any positions, in both pair layouts and for part of the head.

    ``cos`` and ``sin`` are (positions, n), row p the angles of position p (``rotary_tables``); the first ``2 n`` elements of a head are rotated, the rest is
    copied.  Pair i is elements (i, i + n), or (2 i, 2 i + 1) if ``interleaved``.  fp32 arithmetic, rounded once.  A row at a position outside the tables
    becomes zeros.  ``out`` may be x itself."""
    what = "rotary"
    _heads(what, heads, head_dim)
    _rows(what, "x", x, _FLOATS, None, heads * head_dim)
    rot = _rotation(what, cos, sin, interleaved, head_dim, x.device)
    batch = _batch(what, x.shape[0], pos, starts, x.device)
    out = _out(what, out, x, heads * head_dim)
    if out.data_ptr() != x.data_ptr() or _row_stride(out) != _row_stride(x):
        _apart(what, "out", out, x)
    stream = _stream(what, x.device)
    if batch.rows == 0:
        return out
    _lib.check(_lib.load().mk_rotary(x.device.index, batch, rot, x.data_ptr(), _row_stride(x), out.data_ptr(), _row_stride(out),
                                     DTYPE_CODE[x.dtype], heads, head_dim, stream), "mk_rotary")
    return out


def paged_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 pages: torch.Tensor, starts: torch.Tensor | None = None, *, heads: int, kv_heads: int, head_dim: int, page_size: int,
                 interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q and k of each row of qkv (rows, (heads + 2 kv_heads) * head_dim; q, k and v heads side by side), write k and v to the cache
    row of the row's position and return rotated q: ``Graph.rope_append`` for a paged cache and any number of new tokens.

    Rotation as in ``rotary``.  A row at a position outside the tables or the page table (a negative one, say, for the padding of a batch) is not
    appended, and its q becomes zeros; a row whose page is absent is not appended.  ``pos`` is not changed.  Two rows of a call must not have one cache
    row: pages that sequences share lie below their positions."""
    what = "paged_append"
    _heads(what, heads, head_dim)
    _rows(what, "qkv", qkv, _HALVES, None, (heads + 2 * kv_heads) * head_dim)
    rot = _rotation(what, cos, sin, interleaved, head_dim, qkv.device)
    batch = _batch(what, qkv.shape[0], pos, starts, qkv.device)
    cache = _cache(what, k_cache, v_cache, pages, batch.seqs, kv_heads, head_dim, page_size, qkv.dtype, qkv.device)
    out = _out(what, out, qkv, heads * head_dim)
    for name, t, others in (("out", out, (qkv, k_cache, v_cache)), ("k_cache", k_cache, (qkv, v_cache)), ("v_cache", v_cache, (qkv,))):
        _apart(what, name, t, *others)
    stream = _stream(what, qkv.device)
    if batch.rows == 0:
        return out
    _lib.check(_lib.load().mk_paged_append(qkv.device.index, batch, rot, cache, qkv.data_ptr(), _row_stride(qkv), out.data_ptr(),
                                           _row_stride(out), heads, stream), "mk_paged_append")
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor, pages: torch.Tensor,
                    starts: torch.Tensor | None = None, *, heads: int, kv_heads: int, head_dim: int, page_size: int,
                    scale: float | None = None, window: int | None = None, max_new: int | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """New tokens against the cached rows of their sequences, their own among them (append first): ``Graph.decode_attention`` for a paged
    cache and any number of new tokens -- one, a few speculative ones, a chunk of a prompt, a whole prompt, or a batch that mixes them.

    A row at position p attends rows [0, p] of its sequence, or the last ``window`` of these; grouped queries: head h reads kv head
    h // (heads / kv_heads).  Rows of absent pages and rows behind the page table are not there; a row that sees none becomes zeros.  ``scale``
    is head_dim ** -0.5 by default.  head_dim 64 or 128.  Statistics and sums are fp32; the probabilities are rounded to q's type in front of the product
    with V.

    ``max_new``: the largest number of rows a sequence has in this call, where ``starts`` is given (it is on the device): the kernel is chosen by it, and
    a wrong value costs time but changes no more than the order of sums."""
    what = "paged_attention"
    if head_dim not in (64, 128):
        raise ValueError(f"{what}: head_dim must be 64 or 128")
    if kv_heads <= 0 or heads <= 0 or heads % kv_heads:
        raise ValueError(f"{what}: heads must be a multiple of kv_heads")
    window = int(window or 0)
    if window < 0 or window > 2 ** 31 - 1:
        raise ValueError(f"{what}: window is a number of tokens (0 or None: the whole context)")
    _rows(what, "q", q, _HALVES, None, heads * head_dim)
    device = q.device
    batch = _batch(what, q.shape[0], pos, starts, device)
    cache = _cache(what, k_cache, v_cache, pages, batch.seqs, kv_heads, head_dim, page_size, q.dtype, device)
    out = _out(what, out, q, heads * head_dim)
    _apart(what, "out", out, q, k_cache, v_cache)
    if max_new is None or starts is None:
        max_new = batch.rows if starts is not None else batch.rows // max(batch.seqs, 1)
    stream = _stream(what, device)
    if batch.rows == 0:
        return out
    lib = _lib.load()
    nbytes = lib.mk_paged_attention_workspace(device.index, heads, cache, max_new)
    if nbytes < 0:
        _lib.check(int(nbytes), "mk_paged_attention_workspace")
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _lib.check(lib.mk_paged_attention(device.index, batch, cache, q.data_ptr(), _row_stride(q), out.data_ptr(), _row_stride(out), heads,
                                      head_dim ** -0.5 if scale is None else scale, window, max_new, workspace.data_ptr(), nbytes,
                                      stream), "mk_paged_attention")
    return out
