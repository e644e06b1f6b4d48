"""CPU: what the 4-bit K/V cache's entry points refuse before any launch, and the format's own
promises (64-bit definition in kv4_ref)."""
import numpy as np
import pytest
import torch

from madi_b200 import kv4
from tests import kv4_ref as R


def _cache(slots=2, heads=3, max_tok=100):
    return kv4.Cache.empty(slots, heads, max_tok, device="cpu")


def test_cache_shapes():
    c = _cache()
    assert c.data.shape == (2, 3, 2, 4608) and (c.slots, c.kv_heads, c.max_tok) == (2, 3, 100)
    assert kv4.Cache.empty(1, 1, 64, device="cpu").data.shape[2] == 1
    assert kv4.Cache.empty(1, 1, 65, device="cpu").data.shape[2] == 2
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError):
            kv4.Cache.empty(*bad, device="cpu")
    d = c.data
    for data, m in ((d, 64), (d, 129), (d, 0), (d[..., :4000], 100), (d.float(), 100), (d[0], 100),
                    (d.transpose(0, 1), 100)):
        with pytest.raises(ValueError):
            kv4.Cache(data, m)


def test_bytes():
    from madi_b200 import _lib, build
    build.build()
    f = _lib.load().madi_kv4_bytes
    assert f(2, 3, 100) == 2 * 3 * 2 * 4608 == _cache().data.numel()
    assert f(16, 8, 1 << 20) == 16 * 8 * (1 << 14) * 4608                 # past 32 bits
    for bad in ((0, 1, 1), (65536, 1, 1), (1, 0, 1), (1, 1025, 1), (1, 1, 0), (1, 1, (1 << 30) + 1), (-1, 1, 1)):
        assert f(*bad) == 0


def _raises(match, fn, *a, **k):
    with pytest.raises(ValueError, match=match):
        fn(*a, **k)


def test_store_and_load_refusals():
    c, x = _cache(), torch.zeros((2, 5, 192))
    i = torch.zeros(2, dtype=torch.int32)
    _raises("host memory", kv4.store, c, x, x)                             # a cache in host memory
    _raises("k must be", kv4.store, c, x[:1], x[:1])
    _raises("k must be", kv4.store, c, x[..., :128], x[..., :128])
    _raises("k must be", kv4.store, c, x.double(), x.double())
    _raises("k must be", kv4.store, c, x[0], x[0])
    _raises("last dimension", kv4.store, c, x.transpose(1, 2).contiguous().transpose(1, 2), x)
    _raises("v must match", kv4.store, c, x, x.half())
    _raises("v must match", kv4.store, c, x, x[:, :4])
    _raises("v must match", kv4.store, c, x, torch.zeros((2, 5, 384))[..., :192])
    for name in ("pos", "n"):
        for bad in (i.long(), i[:1], torch.zeros((2, 1), dtype=torch.int32), torch.zeros(4, dtype=torch.int32)[::2]):
            _raises(name, kv4.store, c, x, x, **{name: bad})
            _raises(name, kv4.load, c, 5, k_out=x, v_out=x.clone(), **{name: bad})
    _raises("host memory", kv4.load, c, 5, k_out=x, v_out=x.clone())
    _raises("go together", kv4.load, c, 5, k_out=x)
    _raises("holds 5 rows", kv4.load, c, 4, k_out=x, v_out=x.clone())
    _raises("v_out must match", kv4.load, c, 5, k_out=x, v_out=x.half())
    _raises("f32 or f16", kv4.load, c, 5, dtype=torch.bfloat16)
    _raises("rows", kv4.load, c, -1)


def test_attn_refusals():
    c, q = _cache(), torch.zeros((2, 6 * 64))
    i = torch.zeros(2, dtype=torch.int32)
    _raises("host memory", kv4.attn, q, c, 6)
    _raises("q must be", kv4.attn, q, c, 3)
    _raises("q must be", kv4.attn, q.double(), c, 6)
    _raises("q must be", kv4.attn, q[:1], c, 6)
    _raises("last dimension", kv4.attn, q.t().contiguous().t(), c, 6)
    _raises("exclude", kv4.attn, q, c, 6, pos=i, lens=i)
    _raises("out must", kv4.attn, q, c, 6, out=q.half())
    _raises("out must", kv4.attn, q, c, 6, out=q.unsqueeze(1))
    for name in ("pos", "lens", "n"):
        _raises(name, kv4.attn, q, c, 6, **{name: i.float()})


def test_a_cache_on_another_device_is_refused(monkeypatch):
    c = _cache()
    c.device = 1
    monkeypatch.setattr(kv4, "_current_device", lambda: 0)
    _raises("not the current device", kv4._raw_stream, None, c)


def test_calls_before_init_fail_cleanly():
    from madi_b200 import _lib, build
    build.build()
    if torch.cuda.is_available():
        pytest.skip("another test may have initialised the library")
    L = _lib.load()
    h, x = kv4._CACHE(4096, 1, 1, 64), kv4._ROWS(4096, 8192, 0, 0, 64, 64, 0, 1)
    q = kv4._QUERY(4096, 8192, 0, 0, 0, 64, 64, 64, 64, 0, 1, 1, 0)
    for f, a in ((L.madi_kv4_store, x), (L.madi_kv4_load, x), (L.madi_kv4_attn, q)):
        assert f(h, a, None) == _lib.MADI_ENOINIT
        assert f(h, None, None) == _lib.MADI_EINVAL


def test_format_promises():
    """Every element within half a step of its value; codes in range; d n' exact in f16; a step is
    at most 1/15 of the range, the rounding of c and one part in 128 apart."""
    g = np.random.default_rng(1)
    x = (g.standard_normal((3000, 64)) * 10.0 ** g.uniform(-6, 4, (3000, 1)) +
         g.standard_normal((3000, 1)) * 10.0 ** g.uniform(-6, 4, (3000, 1))).astype(np.float16)
    x = np.where(np.abs(x) > 57344, np.float16(0), x)
    z, c, d = R.quantise(x)
    f = x.astype(np.float64)
    assert z.min() >= -8 and z.max() <= 7
    assert (np.abs(R.values(z, c, d) - f) <= d[:, None] / 2).all()
    prod = d[:, None] * z
    assert (prod.astype(np.float16).astype(np.float64) == prod).all()
    rng = f.max(-1) - f.min(-1)
    ulp_c = np.maximum(np.abs(c) * 2.0 ** -10, 2.0 ** -24)
    assert (d <= (rng / 15 + ulp_c / 7) * (1 + 1 / 128) + 2.0 ** -24).all()
    data = np.zeros((1, 1, 1, 4608), np.uint8)
    R.pack(data, 1, 0, 0, 37, z[0], c[0], d[0])
    uz, uc, ud = R.unpack(data, 1, 64)
    assert (uz[0, 0, 37] == z[0]).all() and uc[0, 0, 37] == c[0] and ud[0, 0, 37] == d[0]
