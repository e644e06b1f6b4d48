"""The 4-bit K/V cache on the GPU against its definition in 64 bits (kv4_ref): the bytes that
store writes, the values that load gives (both bit for bit), attention within the bound that
kv4_ref.attend derives, and a run of them together."""
import numpy as np
import pytest

from tests import kv4_ref as R

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32


def _t(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _u32(v):
    return None if v is None else _t(np.asarray(v, np.uint32).view(np.int32))


def _cache(data, max_tok):
    from madi_b200 import kv4
    return kv4.Cache(_t(data), max_tok)


def _host(t):
    import torch
    torch.cuda.synchronize()
    return t.cpu().numpy()


def _stored(data, kv, x, heads, max_tok, pos, n):
    """data with rows x [slots][rows][heads * 64] written as store has to write them."""
    S, T, _ = x.shape
    for s in range(S):
        for i in range(T if n is None else min(T, n[s])):
            row = (0 if pos is None else pos[s]) + i
            if row >= max_tok:
                continue
            for h in range(heads):
                z, c, d = R.quantise(x[s, i, h * 64:(h + 1) * 64])
                R.pack(data, kv, s, h, row, z, c, d)


STORES = [(1, 1, 20, 448, F32, [0], None), (1, 1, 20, 448, F32, [447], None), (3, 1, 4, 448, F32, [5, 447, 448], None),
          (2, 130, 3, 200, F16, [0, 63], None), (2, 65, 2, 100, F32, [35, 60], [65, 7]), (4, 5, 1, 64, F16, None, [0, 1, 5, 9]),
          (1, 300, 20, 300, F16, None, None), (2, 3, 2, 70, F32, [4294967295, 4294967294], None)]


@pytest.mark.parametrize("slots,rows,heads,max_tok,dt,pos,n", STORES)
def test_store_and_load(madi, slots, rows, heads, max_tok, dt, pos, n):
    import torch
    from madi_b200 import kv4
    g = np.random.default_rng(slots * 1000 + rows)
    k = (g.standard_normal((slots, rows, heads * 64)) + g.standard_normal(heads * 64)).astype(dt)
    v = (g.standard_normal((slots, rows, heads * 64)) * 0.3).astype(dt)
    before = g.integers(0, 256, (slots, heads, (max_tok + 63) // 64, 4608)).astype(np.uint8)
    c = _cache(before, max_tok)
    kv4.store(c, _t(k), _t(v), pos=_u32(pos), n=_u32(n))
    want = before.copy()
    for kv, x in ((0, k), (1, v)):
        _stored(want, kv, x, heads, max_tok, pos, n)
    assert np.array_equal(_host(c.data), want), "stored bytes differ (rows that were not stored included)"

    # read back, f32 and f16, each rounded once; rows that load does not give keep their content
    for out_dt in (F32, F16):
        tdt = torch.float32 if out_dt == F32 else torch.float16
        ko = torch.full((slots, rows, heads * 64), 7.0, dtype=tdt, device="cuda")
        vo = torch.full_like(ko, -7.0)
        kv4.load(c, rows, pos=_u32(pos), n=_u32(n), k_out=ko, v_out=vo)
        for kv, got, keep in ((0, _host(ko), 7.0), (1, _host(vo), -7.0)):
            z, cc, dd = R.unpack(want, kv, max_tok)
            exp = np.full((slots, rows, heads, 64), keep, out_dt)
            for s in range(slots):
                for i in range(rows if n is None else min(rows, n[s])):
                    row = (0 if pos is None else pos[s]) + i
                    if row < max_tok:
                        exp[s, i] = R.values(z[s, :, row], cc[s, :, row], dd[s, :, row]).astype(out_dt)
            assert np.array_equal(got, exp.reshape(got.shape), equal_nan=True), f"load {out_dt.__name__} kv={kv}"


def test_quantiser_edges(madi):
    """Constant groups, zeros, one outlier, exact halves of a step, f16 subnormals, the largest
    magnitudes, and groups that hold NaN, infinities or too large values, in both types."""
    import torch
    from madi_b200 import kv4
    g = np.random.default_rng(7)
    for dt in (F16, F32):
        x = [np.zeros(64), np.full(64, 3.0), np.full(64, -0.1), np.where(np.arange(64) == 9, 100.0, 0.0),
             np.arange(64) % 16 * 0.25 - 2.0, np.arange(64) % 31 * 0.125 - 2.0, g.standard_normal(64) * 2.0 ** -20,
             np.linspace(-57344, 57344, 64), g.integers(-3, 4, 64) * 2.0 ** -24, g.standard_normal(64) * 1e-6 + 1,
             g.standard_normal(64) * 3e4, np.where(np.arange(64) == 3, np.nan, 1.0), np.where(np.arange(64) == 63, np.inf, 1.0),
             np.where(np.arange(64) == 0, -np.inf, 1.0), np.where(np.arange(64) == 5, 60000.0, 1.0),
             g.choice([-1.5, -1.0, -0.5, 0.5, 7.0, 0.0], 64), g.standard_normal(64) * 1000 + 2e4]
        x += [g.standard_normal(64) * 10.0 ** g.uniform(-8, 4) + g.standard_normal() * 10.0 ** g.uniform(-8, 4)
              for _ in range(400)]
        x = np.array(x).astype(dt)
        c = kv4.Cache.empty(1, 1, len(x))
        X = _t(x[None])
        kv4.store(c, X, X)
        z, cc, dd = R.quantise(x)
        for kv in (0, 1):
            gz, gc, gd = R.unpack(_host(c.data), kv, len(x))
            assert np.array_equal(gc[0, 0], cc, equal_nan=True) and np.array_equal(gd[0, 0], dd), "c or d"
            assert np.array_equal(gz[0, 0], z), f"codes {dt.__name__}"
        val = _host(kv4.load(c, len(x), dtype=torch.float32)[0])[0].astype(np.float64)
        ok = ~np.isnan(cc)
        assert np.isnan(val[~ok]).all() and (~ok).sum() >= 4
        # within half a step, and the f32 rounding of the value
        assert (np.abs(val[ok] - x[ok].astype(np.float64)) <= dd[ok][:, None] / 2 + np.abs(val[ok]) * 2.0 ** -24).all()


def _check(got, want, tol, what):
    err = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all(), f"{what}: non-finite output"
    assert (err <= tol).all(), f"{what}: error {err.max():.3e}, {(err / np.maximum(tol, 1e-300)).max():.2f} x its bound"


def _attn_case(madi, slots, rows, heads, kv_heads, max_tok, dt, pos=None, lens=None, n=None, seed=0, qscale=1.5,
               spread=1.0):
    import torch
    from madi_b200 import kv4
    g = np.random.default_rng(seed + slots * 100 + rows * 7 + max_tok)
    L = R.key_counts(slots, rows, max_tok, pos, lens)
    nn = [rows] * slots if n is None else [min(rows, x) for x in n]
    written = [max([int(v) for v in L[s, :nn[s]]], default=0) for s in range(slots)]
    data = R.random_cache(g, slots, kv_heads, max_tok, written, spread)
    q = (g.standard_normal((slots, rows, heads * 64)) * qscale).astype(dt)
    p16 = dt == F16                # the many-row form rounds its weights to f16
    want, tol = R.attend(q, data, max_tok, heads, L, n, f16=dt == F16, p16=p16)
    Q = _t(q)
    out = torch.full(Q.shape, 5.0, dtype=Q.dtype, device="cuda")
    c = _cache(data, max_tok)
    kv4.attn(Q, c, heads, pos=_u32(pos), lens=_u32(lens), n=_u32(n), out=out)
    got = _host(out)
    for s in range(slots):
        assert (got[s, nn[s]:] == 5.0).all(), "padding rows were written"
        _check(got[s, :nn[s]], want[s, :nn[s]], tol[s, :nn[s]], f"slot {s} L {L[s, :4]}")
    again = torch.full_like(out, 5.0)
    kv4.attn(Q, c, heads, pos=_u32(pos), lens=_u32(lens), n=_u32(n), out=again)
    assert np.array_equal(_host(again), got), "the same call gives other bits"


@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("slots,heads,kv_heads,max_tok,lens", [
    (1, 20, 20, 448, None), (2, 20, 20, 1500, None), (3, 4, 4, 1, None), (4, 4, 2, 70, [0, 1, 64, 70]),
    (5, 8, 1, 200, [63, 65, 0, 199, 4294967295]), (2, 6, 2, 5000, [4999, 17]), (1, 3, 1, 30000, None),
    (2, 16, 1, 129, [128, 129]), (1, 40, 1, 640, None)])
def test_attn_one_token(madi, slots, heads, kv_heads, max_tok, lens, dt):
    _attn_case(madi, slots, 1, heads, kv_heads, max_tok, dt, lens=lens)


@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("slots,rows,heads,kv_heads,max_tok,pos,lens,n", [
    (1, 1, 20, 20, 448, [0], None, None), (3, 1, 4, 4, 448, [447, 200, 4294967295], None, None),
    (2, 5, 4, 4, 448, [0, 443], None, None), (2, 5, 4, 2, 100, [98, 60], None, [5, 2]),
    (3, 7, 6, 2, 300, None, [0, 65, 300], [7, 7, 0]), (1, 33, 3, 1, 90, [0], None, None),
    (2, 17, 2, 2, 64, None, None, [16, 17]), (1, 130, 2, 1, 700, [500], None, None),
    (2, 70, 4, 4, 260, [0, 190], None, [70, 41]), (1, 60, 2, 1, 3000, [2900], None, None),
    (2, 33, 2, 2, 4100, None, [4099, 96], [33, 1]), (1, 140, 2, 1, 5000, [4800], None, [137]),
    (2, 129, 1, 1, 97, None, [97, 0], None), (1, 300, 1, 1, 1000, [700], None, None)])
def test_attn_many_tokens(madi, slots, rows, heads, kv_heads, max_tok, pos, lens, n, dt):
    _attn_case(madi, slots, rows, heads, kv_heads, max_tok, dt, pos=pos, lens=lens, n=n)


@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("slots,rows,heads,kv_heads,max_tok,mode", [
    (40, 1, 32, 32, 64, "lens"), (40, 1, 32, 32, 200, "pos"), (20, 5, 32, 32, 100, "pos"), (20, 8, 32, 32, 130, "lens"),
    (10, 50, 16, 16, 52, "pos"), (10, 20, 32, 32, 128, "lens"), (10, 20, 32, 32, 260, "pos"), (5, 10, 64, 32, 500, "lens"),
    (10, 17, 16, 16, 97, "pos"), (5, 9, 64, 32, 300, "lens")])
def test_attn_more_heads_than_the_gpu_holds_at_once(madi, slots, rows, heads, kv_heads, max_tok, mode, dt):
    """Many short caches: smaller CTAs, without a cluster; empty and full ones among them, and padding."""
    g = np.random.default_rng(17)
    length = [0, max_tok, max_tok - 1, 1] + [int(x) for x in g.integers(0, max_tok + 1, slots - 4)]
    n = [int(x) for x in g.integers(0, rows + 1, slots)] if rows > 1 else None
    _attn_case(madi, slots, rows, heads, kv_heads, max_tok, dt, n=n, **{mode: length})


@pytest.mark.parametrize("qscale,spread", [(0.0, 1.0), (1e-6, 1.0), (40.0, 1.0), (1.5, 1e-4), (1.5, 2e4)])
def test_attn_scales(madi, qscale, spread):
    """Flat and one-hot softmaxes, small and large values: the weights' scale follows d."""
    _attn_case(madi, 2, 1, 4, 2, 1000, F32, lens=[1000, 333], qscale=qscale, spread=spread, seed=3)


def test_attn_strided_rows(madi):
    """q as columns of a packed projection, out as columns of a wider buffer."""
    import torch
    from madi_b200 import kv4
    g = np.random.default_rng(5)
    S, T, H, M = 2, 3, 4, 100
    data = R.random_cache(g, S, H, M, [M] * S)
    wide = g.standard_normal((S, T, 3 * H * 64)).astype(F32)
    W = _t(wide)
    out = torch.zeros((S, T, 2 * H * 64), dtype=torch.float32, device="cuda")
    kv4.attn(W[..., H * 64:2 * H * 64], _cache(data, M), H, out=out[..., H * 64:])
    want, tol = R.attend(wide[..., H * 64:2 * H * 64], data, M, H, R.key_counts(S, T, M))
    got = _host(out)
    _check(got[..., H * 64:], want, tol, "strided")
    assert (got[..., :H * 64] == 0).all()


def test_nan_rows_reach_only_the_queries_that_attend_them(madi):
    """A K or V row that reads back as NaN makes the queries that attend it NaN and no other."""
    import torch
    from madi_b200 import kv4
    for dt, T in ((torch.float32, 4), (torch.float16, 4), (torch.float16, 80), (torch.float16, 140)):
        for which in (0, 1):
            M, H, bad = 150, 2, 100
            c = kv4.Cache.empty(1, H, M)
            k = torch.randn((1, M, H * 64), device="cuda")
            v = torch.randn_like(k)
            (k, v)[which][0, bad, 64:] = float("nan")                       # head 1 only
            kv4.store(c, k, v)
            q = torch.randn((1, T, H * 64), device="cuda").to(dt)
            p0 = bad - 2
            o = _host(kv4.attn(q, c, H, pos=_u32([p0])))[0].reshape(T, H, 64)
            assert np.isfinite(o[:, 0]).all() and np.isfinite(o[:2, 1]).all() and np.isnan(o[2:, 1]).all()


def _rand_store(slots, heads, max_tok, seed):
    import torch
    from madi_b200 import kv4
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = kv4.Cache.empty(slots, heads, max_tok)
    k, v = (torch.randn((slots, max_tok, heads * 64), generator=g, device="cuda") for _ in range(2))
    return c, k, v, g


@pytest.mark.parametrize("dt,rows,heads,kv_heads,max_tok", [
    (F32, 1, 4, 4, 320), (F16, 1, 8, 2, 9000), (F32, 6, 4, 4, 700), (F16, 40, 4, 2, 400), (F16, 40, 2, 2, 20000)])
def test_captured_calls_on_another_stream(madi, dt, rows, heads, kv_heads, max_tok):
    """Store, attention and load captured on a side stream, two graphs of them replayed at once on
    two streams with inputs that change between replays, against eager calls on the default stream;
    lengths are read on the device."""
    import torch
    from madi_b200 import kv4
    tdt = torch.float32 if dt == F32 else torch.float16
    S = 2
    jobs = []
    for j in range(2):
        c, k, v, g = _rand_store(S, kv_heads, max_tok, 10 + j)
        q = torch.randn((S, rows, heads * 64), generator=g, device="cuda").to(tdt)
        pos = torch.tensor([max_tok - rows, 5], dtype=torch.int32, device="cuda")
        out = torch.zeros_like(q)
        ko, vo = (torch.zeros((S, 3, kv_heads * 64), device="cuda") for _ in range(2))
        st = torch.cuda.Stream()

        def call(c=c, k=k, v=v, q=q, pos=pos, out=out, ko=ko, vo=vo, stream=None):
            kv4.store(c, k, v, stream=stream)
            kv4.attn(q, c, heads, pos=pos, out=out, stream=stream)
            kv4.load(c, 3, pos=pos, k_out=ko, v_out=vo, stream=stream)
        call()                                              # one-time set-up
        torch.cuda.synchronize()
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2, stream=st):
            call()
        jobs.append((call, g2, st, (k, v, q, pos), (out, ko, vo), c))
    for turn in range(3):
        wants = []
        for call, g2, st, (k, v, q, pos), outs, c in jobs:
            k.normal_()
            v.normal_()
            q.copy_(torch.randn(q.shape, device="cuda"))
            pos.copy_(torch.tensor([(max_tok - rows) // (turn + 1), 7 * turn], dtype=torch.int32))
            for o in outs:                                  # rows that load leaves alone are compared too
                o.fill_(-1.0)
            call()
            torch.cuda.synchronize()
            wants.append([o.clone() for o in outs])
            for o in outs:
                o.fill_(-1.0)
            c.data.fill_(0xFF)
        torch.cuda.synchronize()
        for _, g2, st, _, _, _ in jobs:
            with torch.cuda.stream(st):
                g2.replay()
        torch.cuda.synchronize()
        for (_, _, _, _, outs, _), want in zip(jobs, wants):
            for o, w in zip(outs, want):
                assert torch.equal(o, w)
        # and eagerly on a stream that is not the current one
        call, _, st, _, outs, c = jobs[0]
        for o in outs:
            o.fill_(-1.0)
        st.wait_stream(torch.cuda.current_stream())
        call(stream=st)
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants[0]))


def test_allocations_follow_the_given_stream(madi):
    """Outputs that a call makes itself are made (and zeroed) on the stream it runs on, given as a
    stream object or as a handle, the default stream's 0 among them."""
    import torch
    from madi_b200 import kv4
    c, k, v, _ = _rand_store(2, 2, 100, 8)
    kv4.store(c, k, v)
    n = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    q = torch.randn((2, 4, 128), device="cuda")
    want = kv4.attn(q, c, 2, n=n), kv4.load(c, 4, n=n, dtype=torch.float32)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for s in (side, side.cuda_stream, torch.cuda.default_stream(), 0):
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda._sleep(2_000_000)                    # work that the calls must not wait for or race with
            got = kv4.attn(q, c, 2, n=n, stream=s), kv4.load(c, 4, n=n, dtype=torch.float32, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][0], want[1][0]) and torch.equal(got[1][1], want[1][1])


def test_row_by_row_append_equals_one_store(madi):
    import torch
    from madi_b200 import kv4
    c, k, v, _ = _rand_store(3, 2, 150, 4)
    kv4.store(c, k, v)
    d = kv4.Cache.empty(3, 2, 150)
    for i in range(150):
        kv4.store(d, k[:, i:i + 1], v[:, i:i + 1], pos=torch.full((3,), i, dtype=torch.int32, device="cuda"))
    a, b = kv4.load(c, 150, dtype=torch.float32), kv4.load(d, 150, dtype=torch.float32)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dt", [F32, F16])
def test_rows_give_the_same_as_one_by_one(madi, dt):
    """A causal call of several rows against one call per row: both within the bound of the exact
    result; checked here to the type's rounding of each other."""
    import torch
    from madi_b200 import kv4
    tdt = torch.float32 if dt == F32 else torch.float16
    c, k, v, g = _rand_store(2, 2, 300, 6)
    kv4.store(c, k, v)
    q = torch.randn((2, 20, 4 * 64), generator=g, device="cuda").to(tdt)
    p0 = torch.tensor([250, 0], dtype=torch.int32, device="cuda")
    many = kv4.attn(q, c, 4, pos=p0)
    one = torch.stack([kv4.attn(q[:, i].contiguous(), c, 4, pos=p0 + i) for i in range(20)], 1)
    torch.cuda.synchronize()
    # f32: each call is within 2e-6 of the largest output (its sums in another order); f16: the weights'
    # rounding in one of the two (2^-11 of sum p|v| <= max|v| there), and both outputs' own (2^-11)
    tol = 4e-6 * many.abs().max().item() if dt == F32 else 4 * 2.0 ** -11 * v.abs().max().item()
    assert (many.double() - one.double()).abs().max().item() <= tol


def test_f32_results_are_as_exact_as_f32_arithmetic(madi):
    """In norm: a plain f32 form of these sizes is 2e-7 to 5e-7 off the 64-bit result (its sums of 64
    products and of up to 1500 weights round at 2^-24 each); 1e-6 leaves a factor of two."""
    import torch
    from madi_b200 import kv4
    for slots, rows, heads, kv_heads, max_tok in ((2, 1, 4, 4, 1500), (1, 5, 4, 4, 448), (1, 3, 6, 2, 900)):
        g = np.random.default_rng(max_tok)
        data = R.random_cache(g, slots, kv_heads, max_tok, [max_tok] * slots)
        q = (g.standard_normal((slots, rows, heads * 64)) * 1.5).astype(F32)
        want, _ = R.attend(q, data, max_tok, heads, R.key_counts(slots, rows, max_tok))
        got = _host(kv4.attn(_t(q), _cache(data, max_tok), heads)).astype(np.float64)
        assert np.linalg.norm(got - want) <= 1e-6 * np.linalg.norm(want)


def test_offsets_past_32_bits(madi):
    """A cache of more than 2^32 bytes: rows stored at its end are the ones attended and read."""
    import torch
    from madi_b200 import kv4
    heads, max_tok = 8, 1 << 20
    slots = 8
    c = kv4.Cache.empty(slots, heads, max_tok)
    assert c.data.numel() > 1 << 32
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    k, v = (torch.randn((slots, 64, heads * 64), generator=g, device="cuda") for _ in range(2))
    at = torch.full((slots,), max_tok - 64, dtype=torch.int32, device="cuda")
    kv4.store(c, k, v, pos=at)
    ko, vo = kv4.load(c, 64, pos=at, dtype=torch.float32)
    small = kv4.Cache.empty(slots, heads, 64)
    kv4.store(small, k, v)
    ks, vs = kv4.load(small, 64, dtype=torch.float32)
    assert torch.equal(ko, ks) and torch.equal(vo, vs)
    # attention over the last slot's last block: all other rows hold keys that no query can prefer
    c.data.zero_()                                          # codes 0, c = d = 0: scores 0, values 0
    kv4.store(c, k, v, pos=at)
    big = 50.0 * k[:, 63].reshape(slots, heads, 64)         # each query looks for its own last key
    for dt, rows in ((torch.float32, 1), (torch.float16, 33)):
        q = big.reshape(slots, 1, heads * 64).expand(slots, rows, heads * 64).contiguous().to(dt)
        o = kv4.attn(q, c, heads)
        s = kv4.attn(q, small, heads)
        torch.cuda.synchronize()
        # 2^20 keys of score 0 against scores of some hundreds: their weights vanish
        assert (o.float() - s.float()).abs().max().item() <= 1e-3


def test_refusals_on_the_device(madi):
    import torch
    from madi_b200 import kv4
    from madi_b200._lib import MadiError
    c, k, v, _ = _rand_store(2, 2, 70, 1)
    q = torch.zeros((2, 1, 256), device="cuda")
    before = c.data.clone()
    bad = [lambda: kv4.store(c, k[:, 1:, :].reshape(-1)[1:1 + 2 * 60 * 128].view(2, 60, 128), v[:, :60]),      # strides differ
           lambda: kv4.attn(q, c, 4, out=q),                                        # in place
           lambda: kv4.attn(torch.zeros((2, 1, 3 * 64), device="cuda"), c, 3),      # 3 heads over 2 kv heads
           lambda: kv4.attn(q, c, 4, pos=torch.zeros(2, dtype=torch.int32)),        # a host index
           lambda: kv4.attn(q.cpu(), c, 4),
           lambda: kv4.store(c, k[:1].expand(2, -1, -1), v[:1].expand(2, -1, -1)),  # overlapping slots
           lambda: kv4.load(c, 70, k_out=k, v_out=k)]
    wide = torch.zeros((2, 3, 130), device="cuda")
    bad.append(lambda: kv4.store(c, wide[..., 1:129], wide[..., 1:129]))            # rows not 16-byte aligned
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, MadiError)):
            f()
    torch.cuda.synchronize()
    assert torch.equal(c.data, before)
    # nothing to do
    kv4.store(c, k[:, :0], v[:, :0])
    assert kv4.load(c, 0)[0].shape == (2, 0, 128)
    assert kv4.attn(q[:, :0], c, 4).shape == (2, 0, 256)
