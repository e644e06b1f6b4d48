"""Attention over the 4-bit K/V cache where a warp or a CTA takes many blocks of keys (rings that turn over,
sums that are carried and rescaled, clusters that share the keys), held to what the type allows and
not to a bound that grows with the length; and what keeping rows in 4 bits costs."""
import pytest

from tests import test_gpu_kv4 as base
from tests.test_gpu_kv4_precision import F32_SUMS, _gen, _split, _stored

pytestmark = pytest.mark.gpu


def _case(seed, slots, rows, heads, kv_heads, M, grow):
    """Random rows.  grow: keys whose scores rise by 12 nats and values that rise by 2^8 along the cache, so
    that the maximum and the largest step move all the time."""
    import torch
    rn = _gen(seed)
    q = 1.5 * rn(slots, rows, heads * 64)
    K, V = rn(slots, M, kv_heads, 64), 0.5 * rn(slots, M, kv_heads, 64)
    if grow:
        at = (torch.arange(M, device="cuda") / M).view(1, M, 1, 1)
        x = q.view(slots, rows, kv_heads, -1, 64)[:, 0, :, 0].unsqueeze(1)
        K = K + at * 12 * 8 * x / (x * x).sum(-1, keepdim=True)
        V = V * (8 * at).exp2()
    return q, K.reshape(slots, M, -1), V.reshape(slots, M, -1)


def _errors(q, K, V, heads, kv_heads, lens=None):
    """(error, rounding of the exact result to q's type, effect of independent errors of the weights, result), in
    norm and in 64 bits."""
    import torch
    from madi_b200 import kv4
    S, M = K.shape[:2]
    c, k, v, _ = _stored(K, V, kv_heads)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = _split(kv4.attn(q, c, heads, lens=n), kv_heads)
    x = _split(q, kv_heads)
    sums = [0.0] * 4
    for s in range(S):
        L = M if lens is None else lens[s]
        p = torch.softmax(x[s] @ k[s, :, :L].transpose(-1, -2) / 8, -1)
        want = p @ v[s, :, :L]
        each = ((p * p) @ (v[s, :, :L] ** 2)).sqrt()
        for i, e in enumerate((got[s] - want, want.to(q.dtype).double() - want, each, want)):
            sums[i] += (e * e).sum().item()
    assert torch.isfinite(got).all()
    return [e ** 0.5 for e in sums]


STREAM = [(1, 1, 1, 1, 30000), (1, 1, 1, 1, 65003), (8, 1, 20, 20, 1500), (40, 1, 20, 20, 1500), (2, 1, 16, 2, 9000),
          (2, 6, 4, 4, 12000), (8, 16, 20, 20, 1500), (1, 28, 4, 4, 20000), (40, 5, 20, 20, 600)]


@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("slots,rows,heads,kv_heads,M", STREAM)
def test_f32_over_many_blocks(madi, slots, rows, heads, kv_heads, M, grow):
    """1e-6 for the sums, as in test_gpu_kv4.py, and the rounding of scores (q's scaling, the three operations
    of a score, the subtraction) that reach 6 nats, 18 where they grow: 2^-24 each of that in a weight."""
    err, _, _, ref = _errors(*_case(M + slots, slots, rows, heads, kv_heads, M, grow), heads, kv_heads)
    assert err <= (F32_SUMS + 5 * 2.0 ** -24 * (18 if grow else 6)) * ref, f"{err / ref:.2e}"


@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("slots,rows,heads,kv_heads,M", STREAM)
def test_f16_over_many_blocks(madi, slots, rows, heads, kv_heads, M, grow):
    """The streaming form's result, rounded to f16, is that of an exact one but for its scores: a product of
    a query element below 2^-4 of the row's largest is cut at 2^-14 of that largest (times d): 64 such
    cuts spread by 2.3 of them (uniform), 2.3 x 2^-14 x 4.5 x 0.33 / 8 < 2^-14 of a weight here, and with
    keys that grow (d up to 2) < 2^-12."""
    q, K, V = _case(M + slots, slots, rows, heads, kv_heads, M, grow)
    err, rounding, _, ref = _errors(q.half(), K, V, heads, kv_heads)
    assert err <= rounding + 2.0 ** (-12 if grow else -14) * ref, f"{err / ref:.2e}, rounding {rounding / ref:.2e}"


@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("slots,rows,heads,kv_heads,M,lens", [
    (1, 40, 2, 2, 20000, None), (8, 20, 20, 20, 1500, None), (2, 140, 76, 76, 12400, [12400, 300]),
    (2, 140, 76, 76, 12400, None), (2, 1100, 8, 2, 4000, [4000, 3333]), (1, 128, 16, 8, 30000, None)])
def test_f16_tiles_over_many_blocks(madi, slots, rows, heads, kv_heads, M, lens, grow):
    """Many f16 rows: beside the output's rounding that of the weights, 2^-11 of each, independent of one
    another, and the scores' (tensor-core sums of 80 products: 2^-14 of a weight, where they grow 2^-12)."""
    q, K, V = _case(M + slots, slots, rows, heads, kv_heads, M, grow)
    err, rounding, each, ref = _errors(q.half(), K, V, heads, kv_heads, lens)
    assert err <= rounding + 2.0 ** -11 * each + 2.0 ** (-12 if grow else -14) * ref, f"{err / ref:.2e}"


@pytest.mark.parametrize("qscale,spread", [(0.0, 1.0), (1e-6, 1.0), (40.0, 1.0), (1.5, 1e-4), (1.5, 2e4)])
@pytest.mark.parametrize("rows", [1, 12, 40, 140])
def test_f16_scales(madi, rows, qscale, spread):
    """Flat and one-hot softmaxes, small and large values, in f16: both forms."""
    base._attn_case(madi, 2, rows, 4, 2, 500, base.F16, lens=[500, 133], qscale=qscale, spread=spread, seed=3)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_what_four_bits_cost(madi, dtype):
    """Attention over stored rows against attention over the rows themselves: the elements are off by
    up to half a step d, uniformly, so a score is off by |q| d / (8 sqrt 12) and a value by d / sqrt 12,
    independently.  For normal rows (d about a third of their deviation) that makes some 13 % of the result in
    norm; the prediction holds to a fifth."""
    import torch
    from madi_b200 import kv4
    rn = _gen(1)
    S, H, M = 4, 4, 1500
    q, K, V = (rn(S, n, H * 64).to(getattr(torch, dtype)) for n in (3, M, M))
    c = kv4.Cache.empty(S, H, M)
    kv4.store(c, K, V)
    got = _split(kv4.attn(q, c, H), H)
    x = _split(q, H)
    k, v = (t.double().view(S, M, H, 64).transpose(1, 2) for t in (K, V))
    p = torch.softmax(x @ k.transpose(-1, -2) / 8, -1)
    want = p @ v
    d = [c.data[..., at:at + 256].contiguous().view(torch.float16).double().reshape(S, H, -1, 2)[:, :, :M, 1]
         for at in (2048, 2048 + 2304)]
    score = x.norm(dim=-1, keepdim=True) * d[0].unsqueeze(2) / (8 * 12 ** 0.5)
    var = (p * p * score ** 2) @ (v * v) + (p * p) @ (d[1] ** 2 / 12).unsqueeze(-1)
    err, expect = (got - want).norm().item(), var.sum().sqrt().item()
    print(f"4 bits: {err / want.norm().item():.3f} of the result in norm, predicted {expect / want.norm().item():.3f}")
    assert 0.8 * expect <= err <= 1.2 * expect
