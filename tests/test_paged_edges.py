"""Operators over a paged cache at the edges of what their arguments may be.

Tolerances are those of tests/test_paged.py, or derived where they stand.
"""
import pytest
import torch

import megacute_b200 as mc
from megacute_b200 import _lib, paged
from tests.test_paged import BF, check_attention, make_attention


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
