"""The 4-bit K/V cache as the decoder uses it: store and attention in the token step, beside the
f32 attention kernels on the same rows read back; a captured step replayed; the pipeline's
decoders.

Bar of the comparison: the f32 attention kernels are held to 2e-5 x max|out| of the exact result
(test_gpu_attn.py) and so is the 4-bit form here; two results within that of the same exact one
lie within 4e-5 of one another."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _decoder(slots, frames, seed=3, **k):
    import torch
    from madi_b200 import decoder as dec
    d = dec.Decoder(dec.device_weights(seed), slots, kv4_cache=True, **k)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    enc = torch.randn((slots, frames, dec.D), generator=g, device="cuda").half()
    d.set_encoder(enc)
    return d


@pytest.mark.parametrize("slots,act16", [(1, False), (3, True)])
def test_every_attention_of_a_step_matches_the_rows_read_back(madi, monkeypatch, slots, act16):
    import torch
    from madi_b200 import attn, decoder as dec, kv4
    d = _decoder(slots, 700, act16=act16)
    real, seen = kv4.attn, []

    def checked(q, cache, heads, pos=None, out=None, **k):
        real(q, cache, heads, pos=pos, out=out, **k)
        K, V = kv4.load(cache, cache.max_tok, dtype=torch.float32)
        # rows that were not stored yet hold anything; the f32 kernels do not read past pos
        want = attn.cross_attn(q, K, V, heads) if pos is None else attn.self_attn(q, K, V, pos, heads)
        torch.cuda.synchronize()
        err = (out.double() - want.double()).abs().max().item()
        seen.append((pos is None, err / want.abs().max().item()))
        return out

    d.reset()
    with torch.no_grad():
        monkeypatch.setattr(dec.kv4, "attn", checked)
        for _ in range(4):
            d.step()
    assert len(seen) == 4 * 2 * dec.LAYERS
    assert max(e for _, e in seen) <= 4e-5, max(seen, key=lambda s: s[1])


def test_captured_step_gives_the_eager_tokens(madi):
    """Twelve eager steps, and the same from one captured step replayed: equal tokens and
    confidences, bit for bit, also after a second audio chunk and a reset."""
    import torch
    from madi_b200 import decoder as dec
    d = _decoder(2, 300, act16=True)
    d.reset()
    for _ in range(12):
        d.step()
    torch.cuda.synchronize()
    want = d.tokens.clone(), d.conf.clone(), d.x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d.step()
    for chunk in range(2):
        if chunk:
            old = [c.data.data_ptr() for c in d.cross4]
            d.set_encoder(torch.randn((2, 300, dec.D), device="cuda").half())
            assert [c.data.data_ptr() for c in d.cross4] == old, "a captured step must stay valid across chunks"
            d.reset()
            for _ in range(12):
                d.step()
            torch.cuda.synchronize()
            want = d.tokens.clone(), d.conf.clone(), d.x.clone()
        d.reset()
        for _ in range(12):
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, (d.tokens, d.conf, d.x)):
            assert torch.equal(a, b)


def test_cache_bytes_and_step_bytes(madi):
    from madi_b200 import decoder as dec
    d = _decoder(1, 1500)
    per = dec.HEADS * 36 * 2
    assert sum(c.data.numel() for c in d.self4) == dec.LAYERS * dec.MAX_TOK * per
    assert sum(c.data.numel() for c in d.cross4) == dec.LAYERS * 1536 * per       # whole blocks of 64
    full = dec.Decoder(dec.device_weights(3), 1)
    assert full.step_bytes() - d.step_bytes() == dec.LAYERS * 2 * dec.HEADS * (dec.MAX_TOK * 220 + dec.ENC * 92)


def test_pipeline_with_4_bit_caches(madi):
    """Chunks in batches on two decoders: a chunk's tokens do not depend on its batch."""
    import torch
    from madi_b200 import pipeline
    tr = pipeline.Transcriber(slots=2, enc_layers=1, tokens=8, decoders=2, kv4_cache=True)
    mel = torch.from_numpy(pipeline.synthetic_mel(3)).cuda()
    states = tr.encode(mel)
    alone = [tr.decode(states[i:i + 1], 0).clone() for i in range(3)]
    pair = tr.decode(states[1:3], 1).clone()
    torch.cuda.synchronize()
    assert torch.equal(pair, torch.cat(alone[1:3]))
