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
what they hold then.  (``paged_attention_check`` synchronises and tells whether a wait inside a kernel gave up.)  The contents are
the caller's: a position or page outside its range is never followed out of memory, but gives zeros or is skipped, as each function says.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib
from .graph import DTYPE_CODE

_HALVES = {torch.bfloat16: 2, torch.float16: 2}      # types and their sizes
_FLOATS = {torch.bfloat16: 2, torch.float16: 2, torch.float32: 4}


# The keys of a scaling dict that each type is defined by.  Those of every type say how it was made, or repeat what is an argument here.
_SCALING_KEYS = {
    "default": (),
    "linear": ("factor",),
    "dynamic": ("factor",),
    "llama3": ("factor", "low_freq_factor", "high_freq_factor"),
    "yarn": ("factor", "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate"),
}
_ANY_SCALING = ("rope_type", "type", "rope_theta", "original_max_position_embeddings", "partial_rotary_factor", "finetuned")


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None, max_pos: int | None = None,
                       max_position_embeddings: int | None = None):
    """Inverse frequencies of the ``rotary_dim / 2`` pairs, fp64, and the factor on cosines and sines.

    ``scaling`` is a ``rope_scaling`` dict of a Hugging Face config: type ``linear`` (angles divided by ``factor``), ``dynamic`` (theta raised
    so that the slowest pair covers ``max_pos`` positions), ``llama3`` (slow pairs stretched by ``factor``, a linear blend between the two
    corner wavelengths) or ``yarn`` (pairs below ``beta_slow`` turns over the original length stretched, those above ``beta_fast`` kept, a ramp over
    the pairs between, whose corners are rounded outwards unless ``truncate`` is false).  Cosines and sines of ``yarn`` are times ``attention_factor``, by default
    m(1) with m(s) = 0.1 s ln(factor) + 1, or m(mscale) / m(mscale_all_dim) where the dict has both.

    ``max_position_embeddings``: the config's.  It is the original length of ``dynamic`` and ``yarn`` dicts that hold none, and over the original
    length the factor of a ``yarn`` dict without one.  A key that holds None counts as absent.  A dict that lacks what its type needs, or holds a key that would be
    ignored, is refused; so is a ``rope_theta`` that is not ``theta``."""
    if rotary_dim < 4 or rotary_dim % 2:
        raise ValueError("rotary_frequencies: rotary_dim is even and at least 4")
    expo = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    inv = float(theta) ** -expo
    sc = {k: v for k, v in (scaling or {}).items() if v is not None}
    kind = sc.get("rope_type", sc.get("type", "default"))
    if kind not in _SCALING_KEYS:
        raise ValueError(f"rotary_frequencies: unknown scaling {kind!r}")
    ignored = sorted(set(sc) - set(_SCALING_KEYS[kind]) - set(_ANY_SCALING))
    if ignored:
        raise ValueError(f"rotary_frequencies: scaling {kind!r} does not take {', '.join(ignored)}")
    if float(sc.get("rope_theta", theta)) != float(theta):
        raise ValueError(f"rotary_frequencies: theta is {theta}, rope_theta of the scaling {sc['rope_theta']}")

    def need(key, instead=None):
        value = sc.get(key, instead)
        if value is None:
            raise ValueError(f"rotary_frequencies: scaling {kind!r} needs {key}")
        if not float(value) > 0:
            raise ValueError(f"rotary_frequencies: {key} of scaling {kind!r} is {value}, expected a positive number")
        return float(value)

    if kind == "default":
        return inv, 1.0
    if kind == "linear":
        return inv / need("factor"), 1.0
    if kind == "dynamic":
        factor, orig = need("factor"), need("original_max_position_embeddings", max_position_embeddings)
        length = max(float(max_pos or orig), orig)
        base = float(theta) * (factor * length / orig - (factor - 1.0)) ** (rotary_dim / (rotary_dim - 2))
        return base ** -expo, 1.0
    if kind == "llama3":
        factor, lo, hi, orig = (need(k) for k in (*_SCALING_KEYS["llama3"], "original_max_position_embeddings"))
        blend = ((orig * inv / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)          # 0: stretched, 1: as it is
        return (1.0 - blend) * inv / factor + blend * inv, 1.0
    orig = need("original_max_position_embeddings", max_position_embeddings)
    factor = need("factor", max_position_embeddings / orig if max_position_embeddings else None)

    def pair_with(turns):                        # the pair that turns so often over the original length
        return rotary_dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(float(theta)))
    first, last = pair_with(need("beta_fast", 32.0)), pair_with(need("beta_slow", 1.0))
    if sc.get("truncate", True):
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rotary_dim - 1)
    ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)

    def m(s):
        return 0.1 * s * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    if "attention_factor" in sc:
        attention = float(sc["attention_factor"])
    elif sc.get("mscale") and sc.get("mscale_all_dim"):
        attention = m(float(sc["mscale"])) / m(float(sc["mscale_all_dim"]))
    elif sc.get("mscale", 1.0) == 1.0 and not sc.get("mscale_all_dim"):
        attention = m(1.0)
    else:                                        # (those who publish such dicts differ in what one of them alone means)
        raise ValueError("rotary_frequencies: mscale and mscale_all_dim are for each other, both not zero")
    return inv / factor * ramp + inv * (1.0 - ramp), attention


def rotary_tables(max_pos: int, rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None, dtype: torch.dtype = torch.float32,
                  device=None, max_position_embeddings: int | None = None):
    """cos and sin, (max_pos, rotary_dim / 2), of positions 0 .. max_pos - 1: angles in fp64, rounded once to ``dtype``.  ``scaling`` and
    ``max_position_embeddings`` as in ``rotary_frequencies``.  (``checkpoint.rope_tables_from_config`` makes the graph's tables, which hold each column twice; their
    first half of columns serves here too.)"""
    if dtype not in _FLOATS:
        raise TypeError(f"rotary_tables: unsupported dtype {dtype}")
    inv, factor = rotary_frequencies(rotary_dim, theta, scaling, max_pos, max_position_embeddings)
    ang = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv.to(device)[None]
    return (ang.cos() * factor).to(dtype), (ang.sin() * factor).to(dtype)


# -- the binding (csrc/binding.cpp) takes calls whose arguments are plainly right and that have no ``out``; it answers None to others, whose
# checks, errors and results are the ones below
@functools.lru_cache(maxsize=1)
def _direct():
    lib = _lib.load()
    try:
        from . import _binding
    except ImportError:                              # not built for this interpreter: every call goes through ctypes
        return None
    if _binding.built_for != torch.__version__:
        return None
    names = ("mk_rotary", "mk_paged_append", "mk_paged_attention", "mk_paged_attention_workspace")
    _binding.bind(*[ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in names])
    return _binding


# -- arguments: each tensor is looked at once, into a tuple of plain numbers
_PTR, _LD, _ROWS, _COLS, _SIZE = range(5)


def _rows(what, name, t, dtypes, device=None, cols=None):
    """(address, elements between rows, rows, columns, element size) of a 2-D tensor whose rows start on 16-byte boundaries."""
    size = dtypes.get(t.dtype)
    if size is None:
        raise TypeError(f"{what}: {name} has unsupported dtype {t.dtype}")
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{what}: {name} is 2-D")
    if device is not None and t.device != device:
        raise ValueError(f"{what}: {name} is on {t.device}, the others on {device}")
    rows, width = shape
    if cols is not None and width != cols:
        raise ValueError(f"{what}: {name} has {width} columns, expected {cols}")
    ld, inner = t.stride()
    ptr = t.data_ptr()
    if (inner != 1 and width > 1) or (ld < width and rows > 1) or ld * size % 16 or ptr % 16:
        raise ValueError(f"{what}: {name} needs unit inner stride and rows that start on 16-byte boundaries")
    return ptr, ld if ld > width else width, rows, width, size          # (a single row's stride says nothing)


def _ints(what, name, t, device, dim):
    if t.dtype != torch.int32:
        raise TypeError(f"{what}: {name} is int32")
    shape, stride = t.shape, t.stride()
    if len(shape) != dim or t.device != device or stride[0] < 0 or (stride[-1] != 1 and shape[-1] > 1):
        raise ValueError(f"{what}: {name} is a {dim}-D tensor on {device} with unit inner stride")
    return t.data_ptr(), stride[0], shape


def _batch(what, rows, pos, starts, device) -> _lib.Batch:
    ptr, ld, shape = _ints(what, "pos", pos, device, 2)
    seqs = shape[0]
    if shape[1] != 1:
        raise ValueError(f"{what}: pos has one column, one row per sequence")
    if rows > 2 ** 31 - 1 or seqs > 2 ** 31 - 2:
        raise ValueError(f"{what}: at most 2^31 - 1 rows and 2^31 - 2 sequences")
    bounds = None
    if starts is not None:
        bounds, _, shape = _ints(what, "starts", starts, device, 1)
        if shape[0] != seqs + 1:
            raise ValueError(f"{what}: starts has one entry more than there are sequences")
    elif (rows % seqs if seqs else rows):
        raise ValueError(f"{what}: {rows} rows for {seqs} sequences: without starts every sequence has the same number")
    return _lib.Batch(ptr, bounds, ld, rows, seqs)


def _rotation(what, cos, sin, interleaved, head_dim, device) -> _lib.Rotation:
    c, s = _rows(what, "cos", cos, _FLOATS, device), _rows(what, "sin", sin, _FLOATS, device)
    if c[_ROWS:] != s[_ROWS:] or cos.dtype != sin.dtype:
        raise ValueError(f"{what}: cos and sin have one shape and dtype")
    rows, n = c[_ROWS], c[_COLS]
    if n % 8 or n == 0 or 2 * n > head_dim:
        raise ValueError(f"{what}: cos has {n} columns: half the rotated part of a head of {head_dim}, a multiple of 8")
    if rows == 0:
        raise ValueError(f"{what}: empty tables")
    return _lib.Rotation(c[_PTR], s[_PTR], c[_LD], s[_LD], rows, n, DTYPE_CODE[cos.dtype], 1 if interleaved else 0)


def _cache(what, k_cache, v_cache, pages, seqs, kv_heads, head_dim, page_size, dtype, device):
    """mk_paged_cache and what _rows says of k_cache and v_cache"""
    if kv_heads <= 0:
        raise ValueError(f"{what}: kv_heads is positive")
    k = _rows(what, "k_cache", k_cache, _HALVES, device, kv_heads * head_dim)
    v = _rows(what, "v_cache", v_cache, _HALVES, device, kv_heads * head_dim)
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise TypeError(f"{what}: k_cache is {k_cache.dtype}, v_cache {v_cache.dtype}, the activations {dtype}")
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"{what}: page_size is a power of two from 16 up")
    rows = k[_ROWS]
    if rows != v[_ROWS] or rows % page_size:
        raise ValueError(f"{what}: k_cache and v_cache have one shape, whole pages of {page_size} rows")
    table, table_ld, shape = _ints(what, "pages", pages, device, 2)
    if shape[0] != seqs:
        raise ValueError(f"{what}: pages has {shape[0]} rows, pos {seqs}")
    if rows > 2 ** 31 - 1 or shape[1] * page_size > 2 ** 31 - 65536:
        raise ValueError(f"{what}: at most 2^31 - 1 rows in the cache, 2^31 - 65536 of a sequence")
    return _lib.PagedCache(k[_PTR], v[_PTR], table, k[_LD], v[_LD], table_ld, rows // page_size, page_size, shape[1], kv_heads, head_dim,
                           DTYPE_CODE[dtype]), k, v


def _out(what, out, like, device, dtype, rows, cols):
    """The result tensor (of the type and on the device of `like`), what _rows says of it, and whether it is the caller's."""
    if out is None:
        out = like.new_empty((rows, cols))
        return out, (out.data_ptr(), cols, rows, cols, _FLOATS[dtype]), False
    o = _rows(what, "out", out, {dtype: _FLOATS[dtype]}, device, cols)
    if o[_ROWS] != rows:
        raise ValueError(f"{what}: out has {rows} rows")
    return out, o, True


def _apart(what, name, a, b):
    """Refuse a result that shares memory with what the call reads (column ranges of one tensor are apart)."""
    a0, b0 = a[_PTR], b[_PTR]
    if a[_ROWS] == 0 or b[_ROWS] == 0 or a0 >= b0 + ((b[_ROWS] - 1) * b[_LD] + b[_COLS]) * b[_SIZE] or \
            b0 >= a0 + ((a[_ROWS] - 1) * a[_LD] + a[_COLS]) * a[_SIZE]:
        return
    pitch = a[_LD] * a[_SIZE]
    if pitch == b[_LD] * b[_SIZE]:                   # both in one grid of rows: compare the column ranges
        at = (b0 - a0) % pitch
        if at >= a[_COLS] * a[_SIZE] and at + b[_COLS] * b[_SIZE] <= pitch:
            return
    raise ValueError(f"{what}: {name} shares memory with an operand")


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device_index, heads, kv_heads, head_dim, max_new) -> int:
    nbytes = _lib.load().mk_paged_attention_workspace(device_index, heads, kv_heads, head_dim, max_new)
    if nbytes < 0:
        _lib.check(int(nbytes), "mk_paged_attention_workspace")
    return nbytes


def _stream(what, device):
    if device.type != "cuda":
        raise ValueError(f"{what}: expected CUDA tensors")
    return torch._C._cuda_getCurrentRawStream(device.index)      # (torch.cuda.current_stream makes an object, 1.2 us)


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
    direct = _direct() if out is None else None
    if direct is not None:
        y = direct.rotary(x, cos, sin, pos, starts, heads, head_dim, interleaved)
        if y is not None:
            return y
    what = "rotary"
    _heads(what, heads, head_dim)
    src = _rows(what, "x", x, _FLOATS, None, heads * head_dim)
    device, dtype, rows = x.device, x.dtype, src[_ROWS]
    rot = _rotation(what, cos, sin, interleaved, head_dim, device)
    batch = _batch(what, rows, pos, starts, device)
    out, dst, given = _out(what, out, x, device, dtype, rows, heads * head_dim)
    if given and dst != src:
        _apart(what, "out", dst, src)
    stream = _stream(what, device)
    if rows:
        _lib.check(_lib.load().mk_rotary(device.index, batch, rot, src[_PTR], src[_LD], dst[_PTR], dst[_LD], DTYPE_CODE[dtype], heads,
                                         head_dim, stream), "mk_rotary")
    return out


def paged_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 pages: torch.Tensor, starts: torch.Tensor | None = None, *, heads: int, kv_heads: int, head_dim: int, page_size: int,
                 interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q and k of each row of qkv (rows, (heads + 2 kv_heads) * head_dim; q, k and v heads side by side), write k and v to the cache
    row of the row's position and return rotated q: ``Graph.rope_append`` for a paged cache and any number of new tokens.

    Rotation as in ``rotary``.  A row at a position outside the tables or the page table (a negative one, say, for the padding of a batch) is not
    appended, and its q becomes zeros; a row whose page is absent is not appended.  ``pos`` is not changed.  Two rows of a call must not have one cache
    row: pages that sequences share lie below their positions."""
    direct = _direct() if out is None else None
    if direct is not None:
        y = direct.paged_append(qkv, cos, sin, pos, k_cache, v_cache, pages, starts, heads, kv_heads, head_dim, page_size, interleaved)
        if y is not None:
            return y
    what = "paged_append"
    _heads(what, heads, head_dim)
    src = _rows(what, "qkv", qkv, _HALVES, None, (heads + 2 * kv_heads) * head_dim)
    device, dtype, rows = qkv.device, qkv.dtype, src[_ROWS]
    rot = _rotation(what, cos, sin, interleaved, head_dim, device)
    batch = _batch(what, rows, pos, starts, device)
    cache, k, v = _cache(what, k_cache, v_cache, pages, batch.seqs, kv_heads, head_dim, page_size, dtype, device)
    out, dst, given = _out(what, out, qkv, device, dtype, rows, heads * head_dim)
    if given:
        for t in (src, k, v):
            _apart(what, "out", dst, t)
    _apart(what, "k_cache", k, src)
    _apart(what, "v_cache", v, src)
    _apart(what, "k_cache", k, v)
    stream = _stream(what, device)
    if rows:
        _lib.check(_lib.load().mk_paged_append(device.index, batch, rot, cache, src[_PTR], src[_LD], dst[_PTR], dst[_LD], heads, stream),
                   "mk_paged_append")
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor, pages: torch.Tensor,
                    starts: torch.Tensor | None = None, *, heads: int, kv_heads: int, head_dim: int, page_size: int,
                    scale: float | None = None, window: int | None = None, max_new: int | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """New tokens against the cached rows of their sequences, their own among them (append first): ``Graph.decode_attention`` for a paged
    cache and any number of new tokens -- one, a few speculative ones, a chunk of a prompt, a whole prompt, or a batch that mixes them.

    A row at position p attends rows [0, p] of its sequence, or the last ``window`` of these; grouped queries: head h reads kv head
    h // (heads / kv_heads).  Rows of absent pages and rows behind the page table are not there; a row that sees none becomes zeros.  (A key whose
    score overflows to -inf has no weight; a row that sees a score of +inf or NaN has no result, NaN.)  ``scale`` is head_dim ** -0.5 by default.
    head_dim 64 or 128.  Statistics and sums are fp32; the probabilities are rounded to q's type in front of the product with V,
    which in calls of at most 8 rows (heads of a kv head times ``max_new``) takes what the rounding left over as well.

    ``max_new``: the largest number of rows a sequence has in this call, where ``starts`` is given (it is on the device): the kernel is chosen by it, and
    a wrong value costs time (single tokens without it 1.3 to 1.5 times as much: all rows could be one sequence's) but changes no more than the order of sums
    and whether the probabilities' rounding counts."""
    direct = _direct() if out is None else None
    if direct is not None:
        y = direct.paged_attention(q, k_cache, v_cache, pos, pages, starts, heads, kv_heads, head_dim, page_size, scale, window, max_new)
        if y is not None:
            return y
    what = "paged_attention"
    if head_dim not in (64, 128):
        raise ValueError(f"{what}: head_dim must be 64 or 128")
    if kv_heads <= 0 or heads <= 0 or heads % kv_heads:
        raise ValueError(f"{what}: heads must be a multiple of kv_heads")
    window = int(window or 0)
    if window < 0 or window > 2 ** 31 - 1:
        raise ValueError(f"{what}: window is a number of tokens (0 or None: the whole context)")
    src = _rows(what, "q", q, _HALVES, None, heads * head_dim)
    device, dtype, rows = q.device, q.dtype, src[_ROWS]
    batch = _batch(what, rows, pos, starts, device)
    seqs = batch.seqs
    cache, k, v = _cache(what, k_cache, v_cache, pages, seqs, kv_heads, head_dim, page_size, dtype, device)
    out, dst, given = _out(what, out, q, device, dtype, rows, heads * head_dim)
    if given:
        for t in (src, k, v):
            _apart(what, "out", dst, t)
    stream = _stream(what, device)
    if rows == 0 or seqs == 0:
        return out
    if starts is None:
        max_new = rows // seqs
    elif max_new is None:
        max_new = rows
    nbytes = _workspace_bytes(device.index, heads, kv_heads, head_dim, max_new)
    workspace = q.new_empty(nbytes // 2)               # (of 2-byte elements)
    _lib.check(_lib.load().mk_paged_attention(device.index, batch, cache, src[_PTR], src[_LD], dst[_PTR], dst[_LD], heads,
                                      head_dim ** -0.5 if scale is None else scale, window, max_new, workspace.data_ptr(), nbytes, stream),
               "mk_paged_attention")
    return out


def paged_attention_check(device=None, seen: int | None = 0) -> int:
    """Synchronise the current stream of ``device`` (the current one by default) and raise ``MegakernelTimeout`` if a call of ``paged_attention`` on that
    device, on whichever stream, gave up a wait (they end after two seconds; what it returned is then not to be used).

    What is returned counts up with each such wait and is never put back.  ``seen`` is the count that the caller knows of already, from an
    earlier call, say, behind which it goes on; None raises nothing."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"paged_attention_check: {device} is no CUDA device")
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    count = ctypes.c_uint32()
    _lib.check(_lib.load().mk_paged_attention_failures(device.index, _stream("paged_attention_check", device), count), "mk_paged_attention_failures")
    if seen is not None and count.value != seen:
        raise _lib.MegakernelTimeout(f"paged_attention: a wait inside a call on {device} timed out (count {count.value}, {seen} seen before)")
    return count.value
