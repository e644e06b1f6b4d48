"""How near attention over the 4-bit K/V cache comes to the exact result on inputs that are hard for
it: one key that outweighs all others by many orders while its value is small, values of very
different size.  The exact result is computed in 64 bits from the rows read back (which
test_gpu_kv4.py compares bit for bit).  And the smallest numbers a row to store can hold."""
import math

import numpy as np
import pytest

from tests import kv4_ref as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -23             # a tensor-core sum may cut its last place instead of rounding it
LOG2E = math.log2(math.e)


def _gen(seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *s: torch.randn(s, generator=g, device="cuda")


def _stored(K, V, kv_heads):
    """(cache, k, v [S][H][M][64] f64 as read back, |c| + 16 d of each [S][H][M] f64)."""
    import torch
    from madi_b200 import kv4
    S, M, _ = K.shape
    c = kv4.Cache.empty(S, kv_heads, M)
    kv4.store(c, K, V)
    k, v = (x.double().view(S, M, kv_heads, 64).transpose(1, 2) for x in kv4.load(c, M, dtype=torch.float32))
    mags = []
    for at in (2048, 2048 + 2304):
        cd = c.data[..., at:at + 256].contiguous().view(torch.float16).double().reshape(S, kv_heads, -1, 2)[:, :, :M]
        mags.append(cd[..., 0].abs() + 16 * cd[..., 1])
    return c, k, v, mags


def _split(q, kv_heads):
    """q [S][T][heads * 64] -> [S][kv_heads][T * group][64] f64."""
    S, T, W = q.shape
    return q.double().view(S, T, kv_heads, -1, 64).permute(0, 2, 1, 3, 4).reshape(S, kv_heads, -1, 64)


def _sink(seed, rows, heads, kv_heads, M, gap, noise, value=0.0):
    """Every query row prefers key 0 to the others by about `gap` nats; its value is `value` times theirs."""
    rn = _gen(seed)
    one = rn(1, 1, kv_heads, 1, 64)
    q = one.expand(1, rows, kv_heads, heads // kv_heads, 64).reshape(1, rows, heads * 64).contiguous()
    K = noise * rn(1, M, kv_heads, 64)
    x = one[:, 0, :, 0]
    K[:, 0] = gap * 8 * x / (x * x).sum(-1, keepdim=True)
    V = rn(1, M, kv_heads, 64) + 1.0
    V[:, 0] *= value
    return q, K.reshape(1, M, -1), V.reshape(1, M, -1)


@pytest.mark.parametrize("rows,heads,kv_heads", [(40, 1, 1), (100, 4, 2)])
@pytest.mark.parametrize("M", [448, 1500, 20000])
@pytest.mark.parametrize("gap,noise", [(8, 0.5), (12, 0.0), (15, 0.0), (15, 0.5), (17, 0.0), (17, 0.5)])
def test_f16_weights_behind_a_dominant_key(madi, rows, heads, kv_heads, M, gap, noise):
    """Many f16 rows: a weight is rounded to f16 by at most 2^-11 of itself, and by 2^-38 of the largest
    where it is smaller than 2^-27 of that.  Beside it, as in kv4_ref.attend: the scores' sums (16 u of
    the sum of magnitudes), the subtraction in base 2, exp2, the products' sums (2 M / 16 + 16 steps), and the
    output's rounding."""
    import torch
    from madi_b200 import kv4
    q, K, V = _sink(rows + M + gap, rows, heads, kv_heads, M, gap, noise)
    q = q.half()
    c, k, v, (kmag, vmag) = _stored(K, V, kv_heads)
    got = kv4.attn(q, c, heads).double()
    x = _split(q, kv_heads)
    z = x @ k.transpose(-1, -2) / 8
    z = z - z.amax(-1, keepdim=True)
    p = torch.softmax(z, -1)
    mag = x.abs().sum(-1, keepdim=True) / 8 * (1.5 * kmag).unsqueeze(2)           # |q| (|c| + 24 d) / 8
    ep = (16 * U * mag + U * LOG2E * z.abs() + 4 * U).amax(-1, keepdim=True)
    want, a, b = p @ v, p @ v.abs(), p @ vmag.unsqueeze(-1)
    tol = 2 * ep * a + (2 * M / 16 + 16) * U * b + 2 * 2.0 ** -11 * a + 2 * M * 2.0 ** -38 * v.abs().max()
    tol = tol + torch.clamp(2.0 ** -11 * (want.abs() + tol), min=2.0 ** -25)
    err = (_split(got, kv_heads) - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"error {err.max().item():.3e}, {(err / tol).max().item():.2f} x its bound"


def _norm_error(q, c, k, v, heads, kv_heads):
    import torch
    from madi_b200 import kv4
    got = _split(kv4.attn(q, c, heads), kv_heads)
    want = torch.softmax(_split(q, kv_heads) @ k.transpose(-1, -2) / 8, -1) @ v
    assert torch.isfinite(got).all()
    return ((got - want).norm() / want.norm()).item()


# f32 results in norm: 1e-6 for the sums (a plain f32 form is 2e-7 to 5e-7 off, see test_gpu_kv4.py)
F32_SUMS = 1e-6


@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 1, 1), (1, 12, 3), (6, 1, 1), (20, 2, 1)])
@pytest.mark.parametrize("M", [448, 1500, 20000])
@pytest.mark.parametrize("gap", [0.0, 8.3, 10.0, 13.0, 20.0])
def test_f32_weights_behind_a_dominant_key(madi, rows, heads, kv_heads, M, gap):
    """All keys but the first score 0 and hold the same values, so that a rounding of their weight is not
    averaged out.  The first scores `gap` nats: q's scaling to base 2, the score's three operations and the
    subtraction round at 2^-24 of it each, and the weights behind it carry that."""
    import torch
    rn = _gen(M + rows)
    q = torch.zeros((2, rows, heads * 64), device="cuda")
    q[..., ::64] = 8.0
    K = torch.zeros((2, M, kv_heads, 64), device="cuda")
    K[:, 0, :, 0] = gap
    V = torch.where(rn(1, 1, kv_heads, 64) > 0, 1.0, -1.0) * (0.7 + 0.3 * rn(1, 1, kv_heads, 64).abs())
    V = V.repeat(2, M, 1, 1)
    V[:, 0] = 0.0
    c, k, v, _ = _stored(K.reshape(2, M, -1), V.reshape(2, M, -1), kv_heads)
    err = _norm_error(q, c, k, v, heads, kv_heads)
    assert err <= F32_SUMS + 5 * 2.0 ** -24 * gap, f"{err:.2e}"


@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 1, 1), (6, 1, 1), (20, 2, 1)])
@pytest.mark.parametrize("M", [300, 1000, 20000])
@pytest.mark.parametrize("ratio", [10.0, 1e3, 1e4])
def test_f32_values_beside_a_large_one_of_no_weight(madi, rows, heads, kv_heads, M, ratio):
    """One key some 60 nats below the others holds values `ratio` times as large.  The others' scores, within
    6 nats of one another, differ, so that their weights need all bits; they round as above."""
    import torch
    rn = _gen(M + rows)
    one = rn(1, 1, kv_heads, 1, 64)
    q = one.expand(1, rows, kv_heads, heads // kv_heads, 64).reshape(1, rows, heads * 64).contiguous()
    K = rn(1, M, kv_heads, 64)
    x = one[:, 0, :, 0]
    K[:, 3] = -60 * 8 * x / (x * x).sum(-1, keepdim=True)
    V = rn(1, M, kv_heads, 64)
    V[:, 3] *= ratio
    c, k, v, _ = _stored(K.reshape(1, M, -1), V.reshape(1, M, -1), kv_heads)
    err = _norm_error(q, c, k, v, heads, kv_heads)
    assert err <= F32_SUMS + 5 * 2.0 ** -24 * 6, f"{err:.2e}"


@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 2, 1), (7, 2, 2), (20, 1, 1)])
@pytest.mark.parametrize("scale", [1e-38, 1e-20, 2.0 ** 20, 2.0 ** 60, 2.0 ** 97])
def test_f32_query_magnitudes(madi, rows, heads, kv_heads, scale):
    """From the smallest normal queries (a flat softmax) to nearly the largest the interface takes: there the
    key of the largest score alone counts, if its lead is more than the scores' rounding, 2^-18 of the largest
    magnitudes (a few hundred f32 units), which all rows' is here."""
    import torch
    rn = _gen(rows)
    M = 200
    q = rn(2, rows, heads * 64).clamp(-4, 4) * scale
    c, k, v, _ = _stored(rn(2, M, kv_heads * 64), rn(2, M, kv_heads * 64), kv_heads)
    if scale > 1:
        z = _split(q, kv_heads) @ k.transpose(-1, -2)
        top = z.topk(2, dim=-1).values
        lead = (top[..., 0] - top[..., 1]) / (_split(q, kv_heads).abs().sum(-1) * 4)
        assert lead.min().item() > 2.0 ** -18, "another seed"
    err = _norm_error(q, c, k, v, heads, kv_heads)
    assert err <= F32_SUMS + 5 * 2.0 ** -24 * 6, f"{err:.2e}"


def test_store_of_the_smallest_numbers(madi):
    """Groups of a few 2^-149 on one side or both, whose step has to be 2^-24 and not 0: the same bytes
    as the format's definition gives."""
    import torch
    from madi_b200 import kv4
    tiny = np.float32(2.0 ** -149)
    rows = [np.full(64, a) for a in range(-12, 13)]
    for lo in range(-9, 10):
        for hi in range(lo + 1, 10):
            rows.append(np.where(np.arange(64) % 3 == 0, lo, hi))
    g = np.random.default_rng(2)
    rows += [np.rint(g.uniform(-1, 1, 64) * 2.0 ** b) for b in (4, 10, 20, 30, 60, 120, 122, 124, 125, 126, 127)]
    x = (np.array(rows, dtype=np.float64) * float(tiny)).astype(np.float32)
    c = kv4.Cache.empty(1, 1, len(x))
    X = torch.from_numpy(x[None]).cuda()
    kv4.store(c, X, X)
    z, cc, dd = R.quantise(x)
    assert (dd[np.abs(x).max(-1) > 0] >= 2.0 ** -24).all()
    torch.cuda.synchronize()
    for kv in (0, 1):
        gz, gc, gd = R.unpack(c.data.cpu().numpy(), kv, len(x))
        assert np.array_equal(gc[0, 0], cc) and np.array_equal(gd[0, 0], dd) and np.array_equal(gz[0, 0], z)


def test_store_beside_the_halves_of_a_step(madi):
    """Elements on a half of a step and up to three places beside it, every code, for steps that are
    powers of two and others, around zero and far from it: the definition's bytes."""
    import torch
    from madi_b200 import kv4
    g = np.random.default_rng(11)
    rows = []
    for d in (2.0 ** -24, 3 * 2.0 ** -24, 2.0 ** -20, 0.25, 0.375, 1.0, 129 / 128, 2.0, 1024.0):
        for c in (0.0, -0.0, 1.5 * d, -3 * d, 64 * d, 1000 * d):
            c = float(np.float16(np.clip(c, -20000, 20000)))
            for n in range(-7, 8):
                for off in (None, -2, -1, 0, 1, 2):
                    # on or beside the half below code n: one such element in each lane's sixteen, the others
                    # on their values, or (off None) all of them within three places of one
                    x = (c + g.integers(-8, 8, 64) * d).astype(np.float32)
                    x[1], x[2] = c - 8 * d, c + 7 * d             # the range that gives c and d, nearly
                    half = np.float32(c + (n - 0.5) * d).view(np.int32)
                    if off is None:
                        x[3:] = (half + g.integers(-3, 4, 61).astype(np.int32) * (half != 0)).view(np.float32)
                    else:
                        x[g.integers(3, 16)::16] = (half + np.int32(off)).view(np.float32)
                    rows.append(np.where(np.abs(x) <= 57344, x, 0))
    x = np.array(rows, np.float32)
    for dt in (np.float32, np.float16):
        y = x.astype(dt)
        c4 = kv4.Cache.empty(1, 1, len(y))
        Y = torch.from_numpy(y[None]).cuda()
        kv4.store(c4, Y, Y)
        z, cc, dd = R.quantise(y)
        torch.cuda.synchronize()
        for kv in (0, 1):
            gz, gc, gd = R.unpack(c4.data.cpu().numpy(), kv, len(y))
            assert np.array_equal(gc[0, 0], cc) and np.array_equal(gd[0, 0], dd)
            assert np.array_equal(gz[0, 0], z), f"{(gz[0, 0] != z).sum()} codes differ"
