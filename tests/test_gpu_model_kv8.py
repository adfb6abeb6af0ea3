"""The model over an 8-bit cache: forward against the oracle with its keys and values quantised
block by block, speculative decoding, rollback and graphs."""

import pytest
import torch

from lollm_b200.qwen3_5.config import MICRO, MICRO_WIDE, Qwen3_5Config
from lollm_b200.qwen3_5.weights import load_checkpoint, random_init
from oracle import kv8
from oracle import qwen35 as Q
from tolerance import assert_close_dt

pytestmark = pytest.mark.gpu
SEED = 1234
F8 = torch.float8_e4m3fn


def build(raw, dtype, **kw):
    from lollm_b200 import qwen3_5 as fam
    cfg = Qwen3_5Config.from_hf(raw)
    w = random_init(cfg, SEED, generator="numpy")
    model = fam.load(raw, dict(w), dtype=dtype, **kw)
    return cfg, model, fam.load_mtp(model, dict(w))


def _quantised(x, sb):
    """(B, n_kv, L, hd) -> what an 8-bit cache holds of it."""
    y = x.clone()
    for p in range(0, x.shape[2], sb):
        for b in range(x.shape[0]):
            for g in range(x.shape[1]):
                z = x[b, g, p:p + sb].double()
                e = kv8.scale_exp(float(z.abs().max()))
                y[b, g, p:p + sb] = (kv8.e4m3(z * 2.0 ** -e).double() * 2.0 ** e).to(x.dtype)
    return y


@pytest.mark.parametrize("raw,dt", [(MICRO, torch.float32), (MICRO_WIDE, torch.bfloat16)])
def test_forward_matches_oracle_with_quantised_cache(monkeypatch, raw, dt):
    """A prompt, a verify pass and a decode step. The oracle's attention sees its keys and values
    through the quantisation. Bar 2e-2 in both types: a key that the two compute 1e-6 apart can fall to
    different sides of an e4m3 border, a step of 2^-3 in one element."""
    sb = 16
    cfg, model, _ = build(raw, dt, max_positions=256)
    P = load_checkpoint(cfg, random_init(cfg, SEED, generator="numpy"), dtype=dt)
    attend = Q.offset_causal_attention
    monkeypatch.setattr(Q, "offset_causal_attention", lambda q, k, v, scale=None: attend(q, _quantised(k, sb), _quantised(v, sb), scale))
    g = torch.Generator().manual_seed(2)
    cache, oc = model.new_cache(2, 96, kv_dtype=F8, scale_block=sb), None
    assert cache.kv8 and cache.k_pages.dtype == F8
    for t in (37, 4, 1):
        ids = torch.randint(0, cfg.vocab_size, (2, t), generator=g)
        got, _ = model(ids.cuda(), cache)
        want, oc, _ = Q.model_forward(P, cfg, ids, oc)
        assert_close_dt(got.to(torch.bfloat16), want.to(torch.bfloat16), torch.bfloat16)
    cache.check()
    full = model.new_cache(2, 96)
    ids = torch.randint(0, cfg.vocab_size, (2, 20), generator=g)
    small = model.new_cache(2, 96, kv_dtype=F8, scale_block=sb)
    model(ids.cuda(), full)
    model(ids.cuda(), small)
    layer = cfg.attn_layers[0]      # the first attention layer's inputs are the same in both
    for a, b in zip(full.read_kv(layer), small.read_kv(layer)):
        a, b = a.float(), b.float()
        # half a step of e4m3, of the subnormals of the block's scale (2^-10 of at most amax / 224), and the
        # 16-bit cache's own roundings (three products and sums of bf16, 3 half steps of the pair's size)
        tol = a.abs() * 2.0 ** -4 + a.abs().amax() * (2.0 ** -10 / 224 + (0 if dt == torch.float32 else 3 * 2.0 ** -8) + 2.0 ** -20)
        assert ((a - b).abs() <= tol).all()


def test_speculative_stream_equals_plain_stream():
    """fp32, a scale for each token (so a rejected draft leaves no trace in a scale): the speculative
    decoder's stream, eager and from a captured graph, is the plain generator's, both over 8 bits."""
    from lollm_b200.generate import generate
    from lollm_b200.qwen3_5 import SpecDecoder
    cfg, model, mtp = build(MICRO, torch.float32, max_positions=256)
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, cfg.vocab_size, (9,), generator=g).tolist()
    n = 24
    kw = dict(kv_dtype=F8, scale_block=1)
    text = "".join(generate(model, prompt, lambda toks: "".join(chr(0x1000 + t) for t in toks), [], "cuda", max_new_tokens=n,
                            temperature=0.0, top_k=0, top_p=1.0, repetition_penalty=1.0, **kw))
    want = [ord(c) - 0x1000 for c in text]
    for captured in (False, True):
        dec = SpecDecoder(model, mtp, 2, 3, 9 + n + 12, out_capacity=n + 8, **kw)
        dec.prefill(torch.tensor([prompt, prompt]).cuda())
        if captured:
            dec.capture(warmup=1)
        while int(dec.n_out.min()) - dec.prompt_len < n:
            dec.replay()
        assert [o[:n] for o in dec.outputs()] == [want, want]
        dec.cache.check()


def test_production_shapes_in_a_graph():
    """bf16 with the 2B shape's head sizes (the tensor-core attention), block scales, drafts rejected
    along the way: every committed token is the verify forward's own pick."""
    from lollm_b200.qwen3_5 import SpecDecoder
    cfg, model, mtp = build(MICRO_WIDE, torch.bfloat16, max_positions=512)
    g = torch.Generator().manual_seed(1)
    B, P, k = 5, 130, 3
    dec = SpecDecoder(model, mtp, B, k, P + 60, out_capacity=60, kv_dtype=F8)
    dec.prefill(torch.randint(0, cfg.vocab_size, (B, P), generator=g).cuda(), chunk=48)
    dec.capture(warmup=1)
    for _ in range(8):
        n0 = dec.n_out.clone()
        dec.replay()
        ids, ws = dec.ids.clone(), model.workspace(B, k + 1, dec.cache)
        picks = ws.logits.view(B, k + 1, -1).float().argmax(-1)
        for b, n in enumerate((dec.n_out - n0).tolist()):
            assert 1 <= n <= k + 1 and torch.equal(ids[b, 1:n], picks[b, :n - 1]) and int(dec.next_tok[b]) == int(picks[b, n - 1])
    dec.cache.check()
