"""Attention over the 8-bit cache where one key draws most of the weight: what the many weak keys add up to has to
be right however long the context is.

Bound, element by element, with p the exact weights (the largest 1), |v| the stored values and S = Σ p·|v| / Σ p:
* a weight is held to 2^-8 of itself, as bf16 would, or to `floor` of the largest where that is more: a floor that lies
  2^-6 under the weakest weights that the cases have. The sum over the keys of the larger of the two, times |v|;
* a score is a sum of hd products in fp32, scaled: off by (hd + 2)·2^-23·A, A = scale·Σ|q·k| of the worst key + 1; a
  weight moves by as much, numerator and denominator: 2·(hd + 2)·2^-23·A·S;
* n weights and products are added 32 at a time in fp32, 2^-22 of the sum so far each time (the 32 are aligned to
  the largest and cut off, two bits allowed for that), numerator and denominator: 2·(n / 32 + 64)·2^-22·S;
* half a step of the output's type.
No term grows with the number of keys beyond 2^-12·S at 32k."""

import math

import pytest
import torch

from oracle import kv8

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
FLOOR = 2.0 ** -28


def _pages(x, ps, sb):
    """[n, nkv, hd] in order -> codes [pages, nkv, ps, hd] and scales [pages, nkv, ps / sb], one scale a block."""
    n, nkv, hd = x.shape
    P = -(-n // ps)
    y = torch.zeros(P * ps, nkv, hd)
    y[:n] = x
    y = y.view(P, ps // sb, sb, nkv, hd)
    amax = y.abs().amax((2, 4))                                        # [P, blocks, nkv]
    e = torch.ceil(torch.log2(amax.double().clamp_min(1e-30) / 448.0)).clamp_min(-40)
    codes = (y.double() * 2.0 ** -e[:, :, None, :, None]).float().to(kv8.F8)
    raw = codes.view(torch.uint8).view(P, ps, nkv, hd).transpose(1, 2).contiguous()
    return raw.view(kv8.F8), (2.0 ** e).float().transpose(1, 2).contiguous()


def _values(codes, scales, n):
    P, nkv, ps, hd = codes.shape
    x = codes.double() * scales.double().repeat_interleave(ps // scales.shape[2], -1)[..., None]
    return x.transpose(0, 1).reshape(nkv, P * ps, hd)[:, :n]


def run_sink(heads, T, n, B, gap, spread, sink_value, dt=BF16, at=5, ps=64, sb=16, seed=0):
    """B sequences of n keys (the T tokens among them) that share their pages; key `at` scores `gap` nats over the mean of
    the others. Returns got [B, T, nh, hd], want and the bound [T, nh, hd]."""
    from lollm_b200 import kernels as K
    nh, nkv, hd = heads
    rep = nh // nkv
    g = torch.Generator().manual_seed(seed)
    # the first dim is the strong key's alone; the others give the weak keys' scores
    q = torch.randn(T, nh, hd, generator=g)
    q[..., 0] = 16.0
    q = q.to(dt)
    k = spread * torch.randn(n, nkv, hd, generator=g)
    k[:, :, 0] = 0.0
    k[at] = 0.0
    k[at, :, 0] = gap * hd ** 0.5 / 16.0
    v = torch.randn(n, nkv, hd, generator=g) + 0.5
    v[at] *= sink_value
    (kc, ks), (vc, vs) = _pages(k, ps, sb), _pages(v, ps, sb)
    kk, vv = _values(kc, ks, n), _values(vc, vs, n)
    qkv = torch.full((B * T, (2 * nh + 2 * nkv) * hd), 30.0, dtype=dt, device=DEV)      # sigmoid(gate) = 1 - 1e-13
    table = torch.arange(kc.shape[0], dtype=torch.int32).repeat(B, 1)
    z = torch.zeros(hd, dtype=dt, device=DEV)
    rope = torch.zeros(1, 0, dtype=dt, device=DEV)
    q_buf = q.view(1, T, nh * hd).expand(B, T, nh * hd).reshape(B * T, nh * hd).to(DEV)
    out = torch.full((B * T, nh * hd), 7.0, dtype=dt, device=DEV)
    d = K.attn_kv8_layer(qkv, z, z, rope, rope, kc.view(torch.uint8).to(DEV).view(kv8.F8), vc.view(torch.uint8).to(DEV).view(kv8.F8), ks.to(DEV),
                         vs.to(DEV), table.to(DEV), torch.full((B,), n - T, dtype=torch.int32, device=DEV), q_buf, out, tokens=T, n_heads=nh, eps=1e-6)
    K.attn_kv8_verify(d)
    torch.cuda.synchronize()
    assert K.device_status() == 0
    want, tol = torch.zeros(2, T, nh, hd, dtype=torch.float64, device=DEV).unbind()
    keys, lim = torch.arange(n, device=DEV), n - T + torch.arange(T, device=DEV)
    kk, vv, qd = kk.to(DEV), vv.to(DEV), q.double().to(DEV)
    for h in range(nh):
        kh, vh = kk[h // rep], vv[h // rep]
        s = qd[:, h] @ kh.T * hd ** -0.5                                  # [T, n]
        # (e4m3 rounds the strong key: 2^-4)
        assert float((s[:, at] - (s.sum(-1) - s[:, at]) / (n - 1) - gap).abs().max()) < 0.08 * gap
        s = s.masked_fill(keys > lim[:, None], -math.inf)
        p = (s - s.amax(-1, keepdim=True)).exp()
        l = p.sum(-1, keepdim=True)
        S = p @ vh.abs() / l
        A = (qd[:, h].abs() @ kh.abs().T).amax(-1, keepdim=True) * hd ** -0.5 + 1
        m = (lim[:, None] + 1).double()
        err = (2 * (hd + 2) * 2.0 ** -23 * A + 2 * (m / 32 + 64) * 2.0 ** -22) * S
        if dt == BF16:
            err = err + torch.clamp(p * 2.0 ** -8, min=FLOOR).masked_fill(keys > lim[:, None], 0.0) @ vh.abs() / l
        want[:, h] = p @ vh / l
        tol[:, h] = err + (want[:, h].abs() + err) * torch.finfo(dt).eps / 2
    return out.double().view(B, T, nh, hd), want, tol


def check(*args, **kw):
    got, want, tol = run_sink(*args, **kw)
    err = (got - want).abs() / tol
    rel = float(((got - want).norm(dim=-1) / want.norm(dim=-1)).max())
    assert float(err.max()) <= 1.0, f"error / bound {float(err.max()):.3g}, relative error of a row {rel:.3g}"


# heads (q, kv, size), tokens, sequences. 148 units of head size 256 are one each for the 148 SMs, so every key of a sequence
# shares one running maximum; 3 sequences are divided.
UNITS = [((4, 2, 32), 1, 148), ((16, 2, 256), 1, 74), ((16, 2, 256), 2, 74), ((16, 2, 256), 4, 74), ((16, 2, 256), 8, 74), ((8, 2, 64), 4, 74), ((3, 3, 128), 3, 49),
         ((16, 2, 256), 16, 74), ((16, 2, 256), 20, 30), ((8, 2, 64), 32, 74), ((3, 3, 128), 100, 49), ((16, 2, 256), 4, 3)]


@pytest.mark.parametrize("heads,T,B", UNITS)
@pytest.mark.parametrize("gap,spread", [(9.0, 0.0), (11.0, 1.0), (12.0, 0.0), (13.0, 1.0), (14.0, 0.0)])
def test_weak_keys_behind_a_strong_one(heads, T, B, gap, spread):
    """32k keys; the strong one has hardly a value of its own."""
    check(heads, T, 32768, B, gap, spread, 0.0)


@pytest.mark.parametrize("heads,T,B", [((16, 2, 256), 4, 74), ((4, 2, 32), 32, 148), ((16, 2, 256), 16, 74)])
def test_lengths_and_places(heads, T, B):
    """The strong key first, in the middle and last; with a value; few keys and very many."""
    for n, at, value in [(200, 0, 0.0), (5000, 4711, 0.0), (5000, 4990 - T, 1.0), (2304, 0, 1.0), (131072, 3, 0.05)]:
        check(heads, T, n, B if n < 10 ** 5 else 10, 12.0, 1.0, value, at=at)
    check(heads, T, 131072, B, 14.0, 1.0, 0.0)


def test_fp32():
    for gap in (9.0, 14.0):
        check((8, 2, 64), 3, 8192, 4, gap, 1.0, 0.0, dt=F32)


def test_two_strong_keys_tiles_apart():
    """Weights that fall and rise along the keys, by many powers of two each way."""
    import test_gpu_attn_kv8 as M
    for T in (4, 20):
        c = M.Case(BF16, M.H2B, T, [3000], 64, 16, seed=4)
        q = c.set_q()
        s = c.c["k_scales"]
        for p in range(0, 3000, 16):
            s[c.table[0, p // 64], :, p % 64 // 16] = 2.0 ** (-7 if p // 16 % 40 == 7 else -12)
        c.d["k_scales"].copy_(s)
        c.check_out(*c.attend(q))


# shapes whose kernels nothing else here reaches: heads, tokens, lengths, page, block
SHAPES = [((4, 2, 32, 8), 8, [0, 130], 16, 8), ((4, 2, 32, 8), 15, [300, 5], 32, 32), ((4, 2, 32, 8), 31, [129], 64, 1), ((3, 3, 128, 128), 9, [40, 250], 64, 16),
          ((3, 3, 128, 128), 16, [500], 16, 2), ((4, 2, 32, 8), 3, [0, 50], 12, 4), ((3, 3, 128, 128), 5, [77, 3], 20, 4), ((16, 2, 256, 64), 3, [90], 36, 4),
          ((16, 2, 256, 64), 17, [200, 0], 12, 2)]


@pytest.mark.parametrize("heads,T,lens,ps,sb", SHAPES)
def test_other_shapes(heads, T, lens, ps, sb):
    import test_gpu_attn_kv8 as M
    c = M.Case(BF16, heads, T, lens, ps, sb, seed=3)
    c.append()
    c.check_stored()
    c.check_out(*c.attend(c.set_q()))
