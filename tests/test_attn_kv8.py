"""Host side of the 8-bit KV cache, without a GPU: argument checks refuse before any launch, and
the oracle's own rules (scales, rescaling, non-finite tokens) hold."""

import ctypes as C
import math

import pytest
import torch

from lollm_b200 import _lib as L
from lollm_b200 import kernels as K
from oracle import kv8

FAKE = 1 << 20     # an aligned address that no refused call touches


def _layer():
    d = L.AttnKv8Layer()
    d.batch, d.tokens, d.n_heads, d.n_kv_heads, d.head_dim, d.rotary_dim = 2, 4, 16, 2, 256, 64
    d.page_size, d.max_pages, d.num_pages, d.scale_block, d.rope_rows = 64, 8, 16, 16, 512
    d.dtype, d.eps, d.scale = L.QSP_BF16, 1e-6, 1 / 16
    for f in ("qkv", "q_norm_w", "k_norm_w", "rope_cos", "rope_sin", "k_pages", "v_pages", "k_scales", "v_scales", "page_table",
              "seq_lens", "q_buf", "out", "workspace"):
        setattr(d, f, FAKE)
    d.ld_qkv, d.ld_out = 36 * 256, 16 * 256
    d.workspace_bytes = L.load().qsp_attn_kv8_workspace_bytes(2, 4, 16, 2, 256, L.QSP_BF16)
    return d


BAD = [("batch", 0), ("tokens", 0), ("tokens", -1), ("n_kv_heads", 3), ("head_dim", 48), ("page_size", 0), ("max_pages", 0),
       ("max_pages", 1 << 30), ("num_pages", 0), ("scale_block", 0), ("scale_block", 12), ("scale_block", 128), ("page_size", 40),
       ("dtype", 2), ("ld_qkv", 36 * 256 - 1), ("k_pages", 0), ("k_pages", FAKE + 8), ("v_pages", FAKE + 1), ("q_buf", FAKE + 2),
       ("seq_lens", 0), ("page_table", 0), ("v_scales", 0)]


@pytest.mark.parametrize("field,value", BAD)
def test_both_entry_points_refuse(field, value):
    for fn in (L.load().qsp_attn_kv8_prep, L.load().qsp_attn_kv8_verify):
        d = _layer()
        setattr(d, field, value)
        assert fn(C.byref(d), None) == L.QSP_ERR_INVALID
        assert fn(None, None) == L.QSP_ERR_INVALID


@pytest.mark.parametrize("field,value", [("rotary_dim", 63), ("rotary_dim", 258), ("rotary_dim", 72), ("rope_rows", 0), ("rope_cos", 0), ("k_norm_w", 0)])
def test_prep_refuses(field, value):
    d = _layer()
    setattr(d, field, value)
    assert L.load().qsp_attn_kv8_prep(C.byref(d), None) == L.QSP_ERR_INVALID


@pytest.mark.parametrize("field,value", [("out", 0), ("ld_out", 16 * 256 - 1), ("workspace", 0), ("workspace", FAKE + 4),
                                         ("workspace_bytes", 0)])
def test_verify_refuses(field, value):
    d = _layer()
    setattr(d, field, value)
    assert L.load().qsp_attn_kv8_verify(C.byref(d), None) == L.QSP_ERR_INVALID


def test_verify_refuses_a_workspace_one_byte_short():
    d = _layer()
    d.workspace_bytes -= 1
    assert L.load().qsp_attn_kv8_verify(C.byref(d), None) == L.QSP_ERR_INVALID
    assert b"workspace" in L.load().qsp_last_error()


def test_workspace_query():
    q = L.load().qsp_attn_kv8_workspace_bytes
    assert q(0, 1, 16, 2, 256, L.QSP_BF16) == 0 and q(1, 1, 16, 3, 256, L.QSP_BF16) == 0 and q(1, 1, 16, 2, 256, 7) == 0
    # the parts of a call are per CTA, so the batch does not enter
    assert 0 < q(1, 4, 16, 2, 256, L.QSP_BF16) == q(512, 4, 16, 2, 256, L.QSP_BF16) < 64 << 20
    with pytest.raises(RuntimeError):
        K.attn_kv8_workspace_bytes(1, 1, 5, 2, 64, torch.float32)
    with pytest.raises(RuntimeError):
        K.attn_kv8_workspace_bytes(1, 1, 4, 2, 64, torch.float16)


def test_layer_builder_refuses_cpu_tensors():
    z = torch.zeros(8, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.attn_kv8_layer(z, z, z, z, z, z, z, z, z, z, z, z, z, tokens=1, n_heads=1, eps=1e-6)


# ---------------------------------------------------------------- the oracle's rules
@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.0001, 1), (449.0, 1), (224.0, -1), (224.01, 0), (0.0, -40), (1e-30, -40),
                                    (448.0 * 2 ** -40, -40), (2.0, -7), (1.75, -8), (3.4e38, 120)])
def test_scale_rule(amax, e):
    assert kv8.scale_exp(amax) == e


def _case(T, lens, hd=32, nkv=1, nh=1, ps=16, sb=8, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(len(lens) * T, (2 * nh + 2 * nkv) * hd, generator=g)
    z, rows = torch.zeros(hd), max(lens) + 2 * T
    c = kv8.new_cache(8, nkv, ps, hd, sb, [[2 * b, 2 * b + 1] for b in range(len(lens))], lens)
    return c, qkv, z, torch.ones(rows, 8), torch.zeros(rows, 8)


def test_oracle_values_within_half_a_step():
    """e4m3 keeps 4 significant bits: a stored value is within 2^-4 of itself, or half the smallest
    subnormal (2^-10 of the scale), of what was appended."""
    c, qkv, z, cos, sin = _case(11, [0, 3])
    kv8.append(c, qkv, 11, 1, z, z, cos, sin)
    _, _, _, v = kv8.split(qkv, 1, 1, 32)
    for b, n in enumerate(c["lens"]):
        _, got, has = kv8.read(c, b, n + 11)
        want = v[b * 11:(b + 1) * 11, 0].double()
        step = want.abs() * 2.0 ** -4 + 2.0 ** -10 * c["v_scales"].max()
        assert has.all() and ((got[0, n:] - want).abs() <= step).all()


def test_oracle_rescales_earlier_tokens_exactly():
    """A block that starts small and grows: the earlier codes stand for the same values."""
    c, qkv, z, cos, sin = _case(4, [0])
    _, _, _, v = kv8.split(qkv, 1, 1, 32)
    v[:] = torch.randint(8, 15, v.shape).float() / 8      # 4 significant bits: exact in e4m3
    kv8.append(c, qkv, 4, 1, z, z, cos, sin)
    c["lens"] = [4]
    v *= 64
    kv8.append(c, qkv, 4, 1, z, z, cos, sin)
    _, got, _ = kv8.read(c, 0, 8)
    assert torch.equal(got[0, :4] * 64, v[:, 0].double()) and torch.equal(got[0, 4:], v[:, 0].double())


def test_oracle_non_finite_tokens():
    c, qkv, z, cos, sin = _case(3, [0])
    q, gate, k, v = kv8.split(qkv, 1, 1, 32)
    v[1, 0, 5] = math.inf
    kv8.append(c, qkv, 3, 1, z, z, cos, sin)
    kk, vv, _ = kv8.read(c, 0, 3)
    assert torch.isnan(kk[0, 1]).all() and (vv[0, 1] == 0).all() and torch.isfinite(kk[0, [0, 2]]).all()
    out = kv8.attend(c, q, gate, 3, 32 ** -0.5)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:]).all()


# ---------------------------------------------------------------- the family cache
def _cache(**kw):
    from lollm_b200.qwen3_5 import Qwen3_5Cache, Qwen3_5Config
    from lollm_b200.qwen3_5.config import MICRO
    return Qwen3_5Cache(Qwen3_5Config.from_hf(MICRO), 2, 40, dtype=torch.bfloat16, device="cpu", page_size=16, **kw)


def test_cache_refuses():
    for kw in (dict(kv_dtype=torch.float16), dict(kv_dtype=torch.float32), dict(kv_dtype=kv8.F8, scale_block=3),
               dict(kv_dtype=kv8.F8, scale_block=32), dict(kv_dtype=kv8.F8, scale_block=0)):
        with pytest.raises(RuntimeError):
            _cache(**kw)


def test_cache_bytes_and_clone():
    a, b = _cache(), _cache(kv_dtype=kv8.F8, scale_block=8)
    kv = a.k_pages.numel() * 2
    scales = b.k_scales.numel() * 4
    assert a.nbytes() - b.nbytes() == 2 * (kv - kv // 2 - scales)
    c = b.clone()
    c.k_scales.fill_(3.0)
    c.k_pages.view(torch.uint8).fill_(1)
    assert (b.k_scales == 1).all() and (b.k_pages.view(torch.uint8) == 0).all()


def test_cache_append_kv_matches_the_rule():
    """The compatibility path token by token against the oracle's append (values: no norm there)."""
    c = _cache(kv_dtype=kv8.F8, scale_block=8)
    layer, s = c.cfg.attn_layers[1], 1
    nkv, hd = c.cfg.num_key_value_heads, c.cfg.head_dim
    g = torch.Generator().manual_seed(0)
    o = kv8.new_cache(c.num_pages, nkv, 16, hd, 8, c.page_table.tolist(), [0, 0])
    z = torch.zeros(hd)
    for step, t in enumerate([3, 1, 9, 5]):
        x = torch.randn(2, nkv, t, hd, generator=g) * [1.0, 8.0, 0.1, 100.0][step]
        got = c.append_kv(layer, -x, x)
        qkv = torch.zeros(2 * t, 2 * hd + 2 * nkv * hd)
        qkv[:, 2 * hd + nkv * hd:] = x.transpose(1, 2).reshape(2 * t, -1)
        for j in range(t):    # token by token, as the path appends
            rows = qkv.view(2, t, -1)[:, j].contiguous()
            kv8.append(o, rows, 1, 1, z, z, torch.ones(64, 8), torch.zeros(64, 8))
            o["lens"] = [n + 1 for n in o["lens"]]
        for b in range(2):
            want = kv8.read(o, b, o["lens"][b])[1]
            assert torch.equal(got[1][b].double(), want.to(torch.bfloat16).double())
            assert torch.equal(got[0][b], -got[1][b])
    assert c.seen_tokens == 18


def test_cache_append_kv_non_finite():
    """As the kernel stores them: a token whose key or value is not finite in a kv head is a NaN key there, a value
    that is not finite is zero, and neither counts in the block's scale."""
    c, ref = (_cache(kv_dtype=kv8.F8, scale_block=8) for _ in range(2))
    layer = c.cfg.attn_layers[0]
    nkv, hd = c.cfg.num_key_value_heads, c.cfg.head_dim
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(2, 2, nkv, 6, hd, generator=g)
    k0, v0 = k.clone(), v.clone()
    k[0, 1, 2, 3], v[1, 0, 4, 1], v[1, 0, 4, 2] = float("inf"), float("nan"), float("-inf")
    k0[0, 1, 2], k0[1, 0, 4], v0[1, 0, 4] = 0.0, 0.0, 0.0
    c.append_kv(layer, k, v)
    ref.append_kv(layer, k0, v0)
    assert torch.equal(c.k_scales, ref.k_scales) and torch.equal(c.v_scales, ref.v_scales)
    assert torch.equal(c.v_pages.view(torch.uint8), ref.v_pages.view(torch.uint8))
    got = c.read_kv(layer)[0]
    bad = torch.isnan(got)
    assert bad[0, 1, 2].all() and bad[1, 0, 4].all() and int(bad.sum()) == 2 * hd
    assert torch.equal(got[~bad], ref.read_kv(layer)[0][~bad])
