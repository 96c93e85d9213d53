"""Interleaved rotary positions of heads whose pairs do not start on their own size: odd offsets, odd row and head strides, odd heads."""
import pytest
import torch

from test_gpu_serving_ops import DEV, _check_rotary, clean_status, gen  # noqa: F401  (an autouse fixture)
from turboquant.kernels.rotary import make_rotary_table, rotary_embedding

pytestmark = pytest.mark.gpu


def _views(g, dtype, T, hq, hk, D, first, pad):
    """q and k as views of rows that are `pad` values longer than their heads, beginning `first` values into the storage."""
    row = (hq + hk) * D + pad
    flat = torch.randn(first + T * row, generator=g, device=DEV).to(dtype)
    rows = flat[first:].view(T, row)
    return flat, rows[:, :hq * D].unflatten(1, (hq, D)), rows[:, hq * D:(hq + hk) * D].unflatten(1, (hk, D))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,hq,hk,D,R,first,pad", [(5, 4, 2, 128, 128, 1, 0), (33, 3, 1, 64, 32, 0, 1), (700, 8, 2, 128, 64, 3, 5), (9, 2, 1, 7, 6, 0, 0),
                                                   (40, 5, 3, 81, 20, 0, 0), (1, 1, 1, 3, 2, 1, 1)])
def test_interleaved_pairs_that_start_anywhere(T, hq, hk, D, R, first, pad, dtype):
    g = gen(T)
    flat, q, k = _views(g, dtype, T, hq, hk, D, first, pad)
    table = make_rotary_table(R, 512, device=DEV)
    pos = torch.randint(0, 512, (T,), generator=g, device=DEV)
    for inverse in (False, True):
        a, b = rotary_embedding(q, k, pos, table, interleaved=True, inverse=inverse)
        _check_rotary(a, q, table, pos, True, inverse)
        _check_rotary(b, k, table, pos, True, inverse)
        assert a.is_contiguous() and b.is_contiguous() and a.shape == q.shape and b.shape == k.shape
    a, b = rotary_embedding(q, k, pos, table, interleaved=True)
    alone, none = rotary_embedding(q, None, pos, table, interleaved=True)
    assert none is None and torch.equal(alone, a)
    before = flat.clone()
    res = rotary_embedding(q, k, pos, table, interleaved=True, out=(q, k))          # in place: nothing else of the storage changes
    assert res[0] is q and torch.equal(q, a) and torch.equal(k, b)
    if pad:
        gaps = slice((hq + hk) * D, None)
        assert torch.equal(flat[first:].view(T, -1)[:, gaps], before[first:].view(T, -1)[:, gaps])
    assert torch.equal(flat[:first], before[:first])
    assert torch.equal(torch.ops.tq_b200.rotary(q, None, pos, table, True, True)[0], rotary_embedding(q, None, pos, table, interleaved=True, inverse=True)[0])


def test_outputs_that_start_anywhere():
    g = gen(4)
    q = torch.randn(20, 4, 64, generator=g, device=DEV).half()
    table, pos = make_rotary_table(64, 32, device=DEV), torch.arange(20, device=DEV)
    want = rotary_embedding(q, None, pos, table, interleaved=True)[0]
    flat = torch.full((1 + q.numel() + 1,), 7.0, device=DEV, dtype=torch.float16)
    out = flat[1:-1].view(20, 4, 64)
    assert rotary_embedding(q, None, pos, table, interleaved=True, out=(out, None))[0] is out
    assert torch.equal(out, want) and flat[0] == 7 and flat[-1] == 7
    empty = rotary_embedding(flat[1:1].view(0, 4, 64), None, pos[:0], table, interleaved=True)[0]
    assert empty.shape == (0, 4, 64)
