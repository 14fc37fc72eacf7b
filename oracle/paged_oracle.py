"""Plain definitions in 64 bits of the operators over a paged cache (megacute_b200/paged.py), row by row, on the CPU.

Arguments are those of the operators, as CPU tensors; what they return is float64.
"""

from __future__ import annotations

import torch


def batch_rows(rows, pos, starts):
    """(row, sequence, position) of every row of the packed batch that has a sequence."""
    seqs = pos.shape[0]
    if starts is None:
        bounds = [s * (rows // seqs) for s in range(seqs + 1)]
    else:
        bounds = starts.tolist()
    return [(r, s, int(pos[s, 0]) + r - bounds[s]) for s in range(seqs) for r in range(bounds[s], bounds[s + 1])]


def cache_row(pages, s, p, page_size, n_pages):
    """Cache row of position p of sequence s, None if it has none."""
    if p < 0 or p // page_size >= pages.shape[1]:
        return None
    page = int(pages[s, p // page_size])
    return page * page_size + p % page_size if 0 <= page < n_pages else None


def rotate(x, c, s, interleaved):
    """One head: x (head_dim,), c and s (n,)."""
    x, c, s = x.double(), c.double(), s.double()
    n = c.shape[0]
    y = x.clone()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def rotary(x, cos, sin, pos, starts=None, *, heads, head_dim, interleaved=False, out=None):
    y = torch.zeros(x.shape, dtype=torch.float64) if out is None else out.double().clone()
    for r, _, p in batch_rows(x.shape[0], pos, starts):
        inside = 0 <= p < cos.shape[0]
        y[r] = rotate(x[r].view(heads, head_dim), cos[p], sin[p], interleaved).flatten() if inside else 0.0
    return y


def paged_append(qkv, cos, sin, pos, k_cache, v_cache, pages, starts=None, *, heads, kv_heads, head_dim, page_size, interleaved=False, out=None):
    """q, and the caches afterwards."""
    q = torch.zeros(qkv.shape[0], heads * head_dim, dtype=torch.float64) if out is None else out.double().clone()
    k, v = k_cache.double().clone(), v_cache.double().clone()
    n_pages = k_cache.shape[0] // page_size
    for r, s, p in batch_rows(qkv.shape[0], pos, starts):
        if not 0 <= p < min(cos.shape[0], pages.shape[1] * page_size):
            q[r] = 0.0
            continue
        x = qkv[r].view(heads + 2 * kv_heads, head_dim)
        turned = rotate(x[:heads + kv_heads], cos[p], sin[p], interleaved)
        q[r] = turned[:heads].flatten()
        row = cache_row(pages, s, p, page_size, n_pages)
        if row is not None:
            k[row], v[row] = turned[heads:].flatten(), x[heads + kv_heads:].double().flatten()
    return q, k, v


def paged_attention(q, k_cache, v_cache, pos, pages, starts=None, *, heads, kv_heads, head_dim, page_size, scale=None, window=None,
                    max_new=None, out=None):
    """The result, the same sums over the values' magnitudes, and each result's largest sum of magnitudes of a score's products."""
    scale = head_dim ** -0.5 if scale is None else scale
    y = torch.zeros(q.shape, dtype=torch.float64) if out is None else out.double().clone()
    mag, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    n_pages, group = k_cache.shape[0] // page_size, heads // kv_heads
    for r, s, p in batch_rows(q.shape[0], pos, starts):
        first = max(0, p + 1 - window) if window else 0
        rows = [cache_row(pages, s, j, page_size, n_pages) for j in range(first, min(p + 1, pages.shape[1] * page_size))]
        rows = [j for j in rows if j is not None]
        if not rows:
            y[r] = 0.0
            continue
        k = k_cache[rows].double().view(-1, kv_heads, head_dim).repeat_interleave(group, 1)
        v = v_cache[rows].double().view(-1, kv_heads, head_dim).repeat_interleave(group, 1)
        x = q[r].double().view(1, heads, head_dim)
        w = torch.softmax((x * k).sum(-1) * scale, 0)[..., None]
        y[r] = (w * v).sum(0).flatten()
        mag[r] = (w * v.abs()).sum(0).flatten()
        size[r] = ((x * k).abs().sum(-1) * abs(scale)).amax(0).repeat_interleave(head_dim)
    return y, mag, size
