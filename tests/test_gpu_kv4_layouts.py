"""The 4-bit K/V cache's calls on row tensors whose slots or rows come in another order than the other
tests': the results are those of contiguous tensors, bit for bit, and nothing else is written."""
import pytest

pytestmark = pytest.mark.gpu


def _row_major(x, pad=0):
    """x [slots][rows][w] with the memory order [rows][slots][w + pad]."""
    import torch
    S, T, W = x.shape
    buf = torch.full((T, S, W + pad), 9.0, dtype=x.dtype, device=x.device)
    buf[..., :W] = x.transpose(0, 1)
    return buf, buf[..., :W].transpose(0, 1)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("slots,rows,kv_heads,pad", [(2, 5, 2, 0), (3, 1, 1, 8), (1, 4, 2, 0), (4, 40, 3, 64), (2, 150, 1, 0)])
def test_row_major_rows(madi, slots, rows, kv_heads, pad, dtype):
    import torch
    from madi_b200 import kv4
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    k, v = (torch.randn((slots, rows, kv_heads * 64), generator=g, device="cuda").to(dt) for _ in range(2))
    q = torch.randn((slots, rows, 2 * kv_heads * 64), generator=g, device="cuda").to(dt)
    pos = torch.arange(slots, dtype=torch.int32, device="cuda")
    a, b = (kv4.Cache.empty(slots, kv_heads, rows + slots) for _ in range(2))
    a.data.fill_(0)
    b.data.fill_(0)
    kv4.store(a, k, v, pos=pos)
    kv4.store(b, _row_major(k, pad)[1], _row_major(v, pad)[1], pos=pos)
    assert torch.equal(a.data, b.data)
    want = kv4.load(a, rows, pos=pos, dtype=dt)
    (kb, ko), (vb, vo) = (_row_major(torch.zeros_like(k), pad) for _ in range(2))
    kv4.load(b, rows, pos=pos, k_out=ko, v_out=vo)
    assert torch.equal(ko, want[0]) and torch.equal(vo, want[1])
    assert (kb[..., kv_heads * 64:] == 9.0).all() and (vb[..., kv_heads * 64:] == 9.0).all()
    want = kv4.attn(q, a, 2 * kv_heads, pos=pos)
    ob, out = _row_major(torch.zeros_like(q), pad)
    kv4.attn(_row_major(q, pad)[1], b, 2 * kv_heads, pos=pos, out=out)
    assert torch.equal(out, want) and (ob[..., q.shape[2]:] == 9.0).all()


def test_rows_that_overlap_are_refused(madi):
    import torch
    from madi_b200 import kv4
    from madi_b200._lib import MadiError
    c = kv4.Cache.empty(3, 1, 64)
    x = torch.zeros(4096, device="cuda")
    good = torch.zeros((3, 4, 64), device="cuda")
    kv4.load(c, 4, k_out=x.as_strided((3, 4, 64), (64, 192)+(1,)), v_out=good.transpose(0, 1).contiguous().transpose(0, 1))
    for strides in ((64, 64, 1), (0, 64, 1), (64, 0, 1), (64, 128, 1), (128, 64, 1), (252, 64, 1), (60, 192, 1), (256, 60, 1),
                    (64, 188, 1)):
        bad = x.as_strided((3, 4, 64), strides)
        for call in (lambda: kv4.store(c, bad, bad), lambda: kv4.load(c, 4, k_out=bad, v_out=x[2048:].as_strided((3, 4, 64), strides)),
                     lambda: kv4.attn(bad, c, 1, out=good), lambda: kv4.attn(good, c, 1, out=bad)):
            with pytest.raises((ValueError, MadiError)):
                call()
