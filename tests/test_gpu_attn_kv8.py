"""The 8-bit KV cache on the GPU (`qsp_attn_kv8_prep`, `qsp_attn_kv8_verify`) against the oracle in
64 bits.

Tolerances, by arithmetic:
* stored codes and scales: equal. k is computed in 64 bits on both sides and v is not computed at all.
* q: one rounding to the model type, half a step `eps / 2` relative, after fp32 arithmetic: the norm's
  factor comes from a sum of up to 256 squares (a few 2^-24 relative, 2^-20 allowed), the rotation adds
  two products: 2^-19 of the row's largest value covers both.
* attention: see `_attend_bound`.
"""

import math

import pytest
import torch

from oracle import kv8

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def K():
    from lollm_b200 import kernels
    return kernels


class Case:
    """A cache with junk in it, shuffled pages, and its image for the oracle."""

    def __init__(self, dt, heads, T, lens, ps, sb, seed=0, spare=2, junk=True, rows=None, cap=None, q_scale=1.5):
        self.dt, self.T, self.lens = dt, T, list(lens)
        self.nh, self.nkv, self.hd, self.rd = heads
        nh, nkv, hd, rd = heads
        g = torch.Generator().manual_seed(seed)
        self.g = g
        B = len(lens)
        self.B = B
        cap = cap or max(max(lens) + T, 1)
        mp = -(-cap // ps)
        P = B * mp + spare
        self.table = torch.randperm(P, generator=g)[:B * mp].view(B, mp).int()
        rows = rows or mp * ps + 8
        inv = 1.0 / (1e4 ** (torch.arange(0, rd, 2).float() / max(rd, 1)))
        f = torch.arange(rows).float()[:, None] * inv
        f = torch.cat([f, f], -1)
        self.cos, self.sin = f.cos().to(dt), f.sin().to(dt)
        self.qn, self.kn = [(0.2 * torch.randn(hd, generator=g)).to(dt) for _ in range(2)]
        self.c = kv8.new_cache(P, nkv, ps, hd, sb, self.table.tolist(), lens)
        if junk:
            for n in ("k", "v"):
                x = torch.randint(0, 256, (P, nkv, ps, hd), generator=g, dtype=torch.uint8)
                self.c[n + "_pages"] = torch.where((x & 0x7f) == 0x7f, x & 0xf0, x).view(kv8.F8)   # no NaN
                self.c[n + "_scales"] = 2.0 ** torch.randint(-9, -6, (P, nkv, ps // sb), generator=g).float()
        self.new_inputs()
        self.q_scale = q_scale
        self.d = {n: self.c[n].view(torch.uint8).to(DEV).view(kv8.F8) for n in ("k_pages", "v_pages")}
        self.d |= {n: self.c[n].to(DEV) for n in ("k_scales", "v_scales")}
        self.d |= dict(page_table=self.table.to(DEV), seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                       q_norm_w=self.qn.to(DEV), k_norm_w=self.kn.to(DEV), rope_cos=self.cos.to(DEV), rope_sin=self.sin.to(DEV))
        self.bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.q_buf = torch.full((B * T, nh * hd), math.nan, dtype=dt, device=DEV)
        self.out = torch.full((B * T, nh * hd), 7.0, dtype=dt, device=DEV)

    def new_inputs(self):
        self.qkv = torch.randn(self.B * self.T, (2 * self.nh + 2 * self.nkv) * self.hd, generator=self.g).to(self.dt)

    def layer(self, qkv=None, **kw):
        qkv = self.qkv.to(DEV) if qkv is None else qkv
        kw.setdefault("out", self.out)
        return K().attn_kv8_layer(qkv, q_buf=self.q_buf, bad_index=self.bad, tokens=self.T, n_heads=self.nh, eps=1e-6, **self.d, **kw)

    # ---- append
    def append(self, d=None):
        K().attn_kv8_prep(d if d is not None else self.layer())
        return kv8.append(self.c, self.qkv, self.T, self.nh, self.qn, self.kn, self.cos, self.sin)

    def check_stored(self):
        for n in ("k_pages", "v_pages"):
            got, want = self.d[n].view(torch.uint8).cpu().view(kv8.F8).float(), self.c[n].float()
            assert torch.equal(torch.isnan(got), torch.isnan(want)), n
            diff = (got != want) & ~torch.isnan(want)
            assert not diff.any(), f"{n}: {int(diff.sum())} codes differ, first at {diff.nonzero()[0].tolist()}"
        for n in ("k_scales", "v_scales"):
            assert torch.equal(self.d[n].cpu(), self.c[n]), n

    def check_q(self, q):
        got, want = self.q_buf.double().cpu().view(q.shape), q
        tol = want.abs() * torch.finfo(self.dt).eps / 2 + want.abs().amax(-1, keepdim=True) * 2.0 ** -19
        fine = torch.isfinite(want).all(-1)
        assert ((got - want).abs() <= tol)[fine].all()

    # ---- attend
    def set_q(self):
        q = (self.q_scale * torch.randn(self.B * self.T, self.nh * self.hd, generator=self.g)).to(self.dt)
        self.q_buf.copy_(q)
        return q

    def attend(self, q, d=None):
        K().attn_kv8_verify(d if d is not None else self.layer())
        q = q.view(self.B * self.T, self.nh, self.hd)
        gate = kv8.split(self.qkv, self.nh, self.nkv, self.hd)[1]
        want = kv8.attend(self.c, q, gate, self.T, self.hd ** -0.5)
        return want.view(self.B * self.T, -1), _attend_bound(self, q).view(self.B * self.T, -1)

    def check_out(self, want, tol):
        torch.cuda.synchronize()
        got = self.out.double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = ~torch.isnan(want)
        worst = ((got - want).abs() / tol.clamp_min(1e-300))[fine]
        assert not len(worst) or float(worst.max()) <= 1.0, f"error / bound = {float(worst.max()):.3g}"
        assert K().device_status() == 0


def _attend_bound(c, q):
    """How far a right output may be off, element by element.

    A score s = scale·Σ q·k is a sum of hd products in fp32: off by at most hd·2^-23·A, A = scale·Σ|q·k| of
    the row's worst key, and its 2 roundings more (scaling, log2 units: 2^-22·|s| <= 2^-22·A). That moves
    a weight p by the same relative amount, and the output, a mean of values with weights that are all off,
    by at most twice that times V = max|v|. Summing n weights and n products in fp32: n·2^-23·V each. bf16
    models: the weights are held as the sum of two e4m3 values, 2^-8 relative (a half step of a half
    step, 2^-4·2^-4), or 2^-18 of the largest where that is more (the second value's subnormals): a mean
    over n keys moves by at most 2^-8·V + n·2^-18·V·p_max, and p_max·n·2^-18 <= n·2^-18. The output: half a
    step of its type. The gate is at most 1; its own error (2^-22) is within the allowance of A >= 1."""
    tol = torch.zeros(q.shape, dtype=torch.float64)
    rep = c.nh // c.nkv
    for b, n in enumerate(c.lens):
        for t in range(c.T):
            m = n + t + 1
            if m <= 0:
                continue
            k, v, has = kv8.read(c.c, b, m)
            k, v = torch.nan_to_num(k[:, has]), torch.nan_to_num(v[:, has])
            if not has.any():
                continue
            for g in range(c.nkv):
                h = slice(g * rep, (g + 1) * rep)
                A = (torch.nan_to_num(q[b * c.T + t, h].double(), posinf=0, neginf=0).abs() @ k[g].abs().T).amax(-1) * c.hd ** -0.5 + 1
                V = v[g].abs().max()
                rel = 2 * (c.hd + 2) * 2.0 ** -23 * A + 2 * m * 2.0 ** -23
                if c.dt == BF16:
                    rel = rel + 2.0 ** -8 + m * 2.0 ** -18
                tol[b * c.T + t, h] = (rel * V)[:, None]
    gate = torch.sigmoid(kv8.split(c.qkv, c.nh, c.nkv, c.hd)[1].double())
    q0 = torch.nan_to_num(q.double(), posinf=0, neginf=0)
    want = torch.nan_to_num(kv8.attend(c.c, q0, torch.full_like(gate, 100.0), c.T, c.hd ** -0.5)).abs()
    return gate * (tol + (want + tol) * torch.finfo(c.dt).eps / 2)


# heads: (q heads, kv heads, head size, rotated dims)
H2B, HTINY, HMICRO, HMHA, HODD = (16, 2, 256, 64), (8, 2, 64, 16), (4, 2, 32, 8), (3, 3, 128, 128), (6, 2, 64, 0)

APPEND = [
    # heads, T, lens, page, block
    (H2B, 1, [0], 64, 16), (H2B, 1, [15, 16, 63, 64, 100], 64, 16), (H2B, 4, [14, 0, 61, 127], 64, 16), (H2B, 67, [3, 64], 64, 16),
    (HTINY, 5, [90, 201, 7], 32, 8), (HTINY, 9, [1, 30], 16, 1), (HMICRO, 3, [0, 2, 31], 32, 32), (HMHA, 33, [10, 63], 64, 64),
    (HODD, 6, [5, 11], 8, 4), (HODD, 6, [5, 11], 24, 8), (HTINY, 3, [4], 5, 1),
]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("heads,T,lens,ps,sb", APPEND)
def test_append(dt, heads, T, lens, ps, sb):
    c = Case(dt, heads, T, lens, ps, sb)
    q, bad = c.append()
    c.check_stored()          # whole pages: what lies beside the new tokens is as it was
    c.check_q(q)
    assert not bad and int(c.bad) == 0
    c.append()                # once more in the same place: the same again
    c.check_stored()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_append_step_by_step_with_rollback(dt):
    """Steps of 4 with 1 to 4 of them kept; magnitudes that rise and fall make block scales grow, and
    earlier codes be rescaled."""
    c = Case(dt, HTINY, 4, [0, 5, 13], 16, 8, junk=False, cap=64, rows=64)
    d = c.layer()
    keep = [[4, 1, 2], [3, 4, 1], [1, 2, 3], [4, 4, 4], [2, 1, 1]]
    for step, kept in enumerate(keep):
        c.new_inputs()
        c.qkv[:, 2 * c.nh * c.hd:] *= [1e-3, 1.0, 30.0, 0.02, 5.0][step]
        d._keep["qkv"].copy_(c.qkv)
        q, _ = c.append(d)
        c.check_stored()
        c.check_q(q)
        c.lens = c.c["lens"] = [n + k for n, k in zip(c.lens, kept)]
        c.d["seq_lens"].copy_(torch.tensor(c.lens, dtype=torch.int32))


def test_append_extremes():
    """Zeros (the smallest scale), the largest fp32 values, values that only e4m3's subnormals hold."""
    c = Case(F32, HMICRO, 8, [0, 8], 16, 8, junk=False)
    _, _, k, v = kv8.split(c.qkv, c.nh, c.nkv, c.hd)
    k[0], v[0:8] = 0.0, 0.0
    v[8], v[9, :, ::2] = 3.0e38, 1e-38
    v[10] *= 2.0 ** 120
    c.append()
    c.check_stored()


def test_append_non_finite():
    c = Case(BF16, H2B, 6, [3, 10], 16, 8)
    _, _, k, v = kv8.split(c.qkv, c.nh, c.nkv, c.hd)
    k[1, 0, 7], v[2, 1, 0], v[4, 0, 255], k[8, 1, 3], v[8, 1, 9] = math.nan, math.inf, math.nan, -math.inf, math.nan
    q, _ = c.append()
    c.check_stored()
    c.check_q(q)


@pytest.mark.parametrize("what", ["page", "capacity", "table", "negative"])
def test_append_out_of_place(what):
    """Positions without a page (a bad entry, past the capacity), past the RoPE table or below zero are
    left out and flagged; the other sequence is stored."""
    c = Case(F32, HTINY, 4, {"capacity": [30, 2], "negative": [-2, 5]}.get(what, [13, 2]), 16, 8, cap=32,
             rows=14 if what == "table" else None)
    if what == "page":
        c.table[0, 0] = 99
        c.c["table"][0][0] = 99
        c.d["page_table"].copy_(c.table)
    _, bad = c.append()
    c.check_stored()
    assert bad and int(c.bad) == 1


def test_append_strided_rows():
    """qkv as a slice of a wider buffer, at an address and a pitch that are not multiples of 16 bytes."""
    for off, pad in [(0, 8), (3, 5), (8, 8)]:
        c = Case(BF16, H2B, 3, [5, 40], 64, 16)
        wide = torch.zeros(c.qkv.shape[0], c.qkv.shape[1] + off + pad, dtype=BF16, device=DEV)
        view = wide[:, off:off + c.qkv.shape[1]]
        view.copy_(c.qkv)
        q, _ = c.append(c.layer(view))
        c.check_stored()
        c.check_q(q)


ATTEND = [
    (H2B, 1, [0], 64, 16), (H2B, 1, [32, 127, 128, 300], 64, 16), (H2B, 4, [0, 700, 125, 126], 64, 16), (H2B, 2, [1500], 64, 16),
    (H2B, 9, [40, 250], 128, 64), (H2B, 40, [100], 16, 8), (HTINY, 5, [90, 201, 7], 32, 8), (HTINY, 33, [0, 130], 16, 1),
    (HMICRO, 3, [0, 2, 31, 513], 32, 32), (HMHA, 1, [400, 10], 32, 32), (HMHA, 17, [200], 64, 64), (HODD, 6, [5, 300], 8, 4),
    (HODD, 6, [5, 150], 24, 8), (HTINY, 3, [140], 5, 1), (HTINY, 200, [0], 16, 8), (H2B, 131, [0, 70], 64, 16), (HMHA, 70, [0, 33], 256, 64), ((8, 1, 256, 64), 16, [100], 64, 16), ((40, 2, 128, 32), 3, [70, 200], 64, 16),
]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("heads,T,lens,ps,sb", ATTEND)
def test_attend(dt, heads, T, lens, ps, sb):
    c = Case(dt, heads, T, lens, ps, sb)
    c.check_out(*c.attend(c.set_q()))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attend_ignores_what_it_may_not_see(dt):
    """NaN codes in every slot past the sequences (and in pages of nobody): no output changes."""
    c = Case(dt, H2B, 4, [3, 131, 200], 64, 16)
    used = torch.zeros(c.c["k_pages"].shape[0], 64, dtype=torch.bool)
    for b, n in enumerate(c.lens):
        for p in range(n + c.T):
            used[c.table[b, p // 64], p % 64] = True
    for n in ("k_pages", "v_pages"):
        raw = c.c[n].view(torch.uint8)
        raw[~used[:, None].expand(-1, c.nkv, -1)] = 0x7f
        c.d[n].view(torch.uint8).copy_(raw)
    c.check_out(*c.attend(c.set_q()))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attend_rows_that_see_nothing(dt):
    """A negative length leaves the first queries without a key: zeros. Unmapped pages are not seen."""
    c = Case(dt, H2B, 4, [-2, -9, 150], 64, 16, cap=256)
    c.table[2, 1] = -1
    c.c["table"][2][1] = -1
    c.d["page_table"].copy_(c.table)
    c.check_out(*c.attend(c.set_q()))
    c = Case(dt, H2B, 4, [100], 64, 16)
    c.table[:] = 10 ** 6
    c.d["page_table"].copy_(c.table)
    c.c["table"] = c.table.tolist()
    want, _ = c.attend(c.set_q())
    torch.cuda.synchronize()
    assert (want == 0).all() and (c.out == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attend_non_finite(dt):
    """A NaN or infinite query gives a row of NaN; a stored NaN key gives NaN to the rows that see it."""
    c = Case(dt, H2B, 4, [140, 20], 64, 16)
    _, _, k, v = kv8.split(c.qkv, c.nh, c.nkv, c.hd)
    v[2, 1, 5] = math.inf                      # token 2 of sequence 0, kv head 1
    q, _ = c.append()
    q = c.q_buf.cpu()
    q[5, 3], q[6, 256] = math.nan, math.inf
    c.q_buf.copy_(q)
    want, tol = c.attend(q)
    assert torch.isnan(want).any() and torch.isfinite(want).any()
    c.check_out(want, tol)


def _uniform_codes(c, k=0.0, v=None):
    for n, x in (("k", k), ("v", v)):
        if x is not None:
            c.c[n + "_pages"] = torch.full(c.c[n + "_pages"].shape, x).to(kv8.F8)
            c.d[n + "_pages"].view(torch.uint8).copy_(c.c[n + "_pages"].view(torch.uint8))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attend_equal_scores_and_a_sink(dt):
    """All keys alike (a mean of the values), then one strong key and many weak ones whose weights are
    the same: no rounding of weights may add up."""
    c = Case(dt, H2B, 2, [900], 64, 16)
    _uniform_codes(c, 0.0)
    c.check_out(*c.attend(c.set_q()))
    q = torch.zeros(2, c.nh * c.hd, dtype=dt)
    q.view(2, c.nh, c.hd)[..., 0] = 16.0
    c.q_buf.copy_(q)
    page, j = c.table[0, 3], 0
    sc = float(c.c["k_scales"][page, 0, j])
    c.c["k_pages"].view(torch.uint8)[page, :, 5, 0] = torch.tensor(min(9.0 / sc, 448.0)).to(kv8.F8).view(torch.uint8)
    c.d["k_pages"].view(torch.uint8).copy_(c.c["k_pages"].view(torch.uint8))
    c.check_out(*c.attend(q))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attend_scales_far_apart(dt):
    """Blocks whose value scales span many powers of two, and scores that grow along the keys."""
    c = Case(dt, H2B, 4, [700, 260], 64, 16)
    s = c.c["v_scales"]
    s.mul_(2.0 ** torch.randint(-25, 12, s.shape, generator=c.g).float())
    c.d["v_scales"].copy_(s)
    s = c.c["k_scales"]
    for p in range(0, 700, 16):
        s[c.table[0, p // 64], :, p % 64 // 16] = 2.0 ** (-14 + p / 70 // 1)
    c.d["k_scales"].copy_(s)
    c.check_out(*c.attend(c.set_q()))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_append_then_attend(dt):
    """The two as a forward calls them, on a stream of their own, three steps."""
    c = Case(dt, HTINY, 4, [0, 60, 33], 16, 8, junk=False, cap=128)
    for n in ("k", "v"):      # what the sequences hold already
        x = torch.randint(0, 100, c.c[n + "_pages"].shape, generator=c.g, dtype=torch.uint8)
        c.c[n + "_pages"] = x.view(kv8.F8)
        c.d[n + "_pages"].view(torch.uint8).copy_(x)
    d = c.layer()
    st = torch.cuda.Stream()
    for _ in range(3):
        c.new_inputs()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            d._keep["qkv"].copy_(c.qkv)
            c.append(d)
            K().attn_kv8_verify(d)
        st.synchronize()
        c.check_stored()
        c.check_out(*c.attend(c.q_buf.cpu(), d))
        c.lens = c.c["lens"] = [n + 3 for n in c.lens]
        c.d["seq_lens"].copy_(torch.tensor(c.lens, dtype=torch.int32))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_repeated_captured_and_two_at_once(dt):
    """Repeated calls give the same bits; a captured graph replays on new lengths and inputs; two
    layers with workspaces of their own run at once on two streams."""
    a, b = Case(dt, H2B, 4, [700, 90, 300], 64, 16, seed=1), Case(dt, H2B, 4, [10, 1100], 64, 16, seed=2)
    qa, qb = a.set_q(), b.set_q()
    da, db = a.layer(), b.layer()
    want = [a.attend(qa, da), b.attend(qb, db)]
    torch.cuda.synchronize()
    a0, b0 = a.out.clone(), b.out.clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(s1):
            K().attn_kv8_verify(da)
        with torch.cuda.stream(s2):
            K().attn_kv8_verify(db)
    torch.cuda.synchronize()
    assert torch.equal(a.out, a0) and torch.equal(b.out, b0)
    a.check_out(*want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s1):
        K().attn_kv8_prep(da)
        K().attn_kv8_verify(da)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s1):
        K().attn_kv8_prep(da)
        K().attn_kv8_verify(da)
    a.append(da)
    a.new_inputs()
    da._keep["qkv"].copy_(a.qkv)
    a.lens = a.c["lens"] = [690, 3, 299]
    a.d["seq_lens"].copy_(torch.tensor(a.lens, dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    got, stored = a.out.clone(), a.d["k_pages"].view(torch.uint8).clone()
    kv8.append(a.c, a.qkv, a.T, a.nh, a.qn, a.kn, a.cos, a.sin)
    a.check_stored()
    a.check_out(*a.attend(a.q_buf.cpu(), da))
    assert torch.equal(a.out, got) and torch.equal(stored, a.d["k_pages"].view(torch.uint8))


def test_many_sequences():
    """More units than CTAs, most of one tile; and a batch with one long sequence among short ones."""
    c = Case(BF16, HTINY, 1, [(7 * i) % 190 for i in range(300)], 16, 8)
    c.check_out(*c.attend(c.set_q()))
    c = Case(BF16, HTINY, 2, [4000] + [i for i in range(40)], 64, 16)
    c.check_out(*c.attend(c.set_q()))


def test_output_beside_others():
    """out as columns of a wider buffer; rows and columns beside it stay."""
    c = Case(BF16, H2B, 3, [5, 140], 64, 16)
    q = c.set_q()
    wide = torch.full((9, 16 * 256 + 24), 3.0, dtype=BF16, device=DEV)
    d = c.layer(out=wide[:, 5:5 + 16 * 256])
    want, tol = c.attend(q, d)
    torch.cuda.synchronize()
    c.out.copy_(wide[:6, 5:5 + 16 * 256])
    c.check_out(want, tol)
    assert (wide[6:] == 3).all() and (wide[:, :5] == 3).all() and (wide[:, 5 + 16 * 256:] == 3).all()


def test_builder_refuses():
    c = Case(BF16, HTINY, 2, [5], 16, 8)
    ok = dict(c.d)
    for name, t in [("k_pages", c.d["k_pages"].view(torch.uint8)), ("v_scales", c.d["v_scales"].double()), ("v_scales", c.d["v_scales"][:, :, :1].contiguous()),
                    ("page_table", c.d["page_table"].long()), ("seq_lens", c.d["seq_lens"].repeat(2)), ("q_norm_w", c.d["q_norm_w"].float()),
                    ("rope_sin", c.d["rope_sin"][:-1]), ("k_pages", c.d["k_pages"].transpose(1, 2)), ("k_scales", c.d["k_scales"].cpu())]:
        c.d = dict(ok, **{name: t})
        with pytest.raises(RuntimeError):
            c.layer()
    c.d = ok
    with pytest.raises(RuntimeError):
        c.layer(qkv=c.qkv.to(DEV)[:, :-1])
    with pytest.raises(RuntimeError):
        c.layer(out=c.out[:, :-1])
    with pytest.raises(RuntimeError):
        K().attn_kv8_verify(c.layer(workspace=torch.empty(16, dtype=torch.uint8, device=DEV)))


# more than 64 rows of query per kv head: chunks of prompts
CHUNKS = [
    (HMICRO, 40, [0, 100, 7], 32, 32), (HMICRO, 70, [300], 64, 8), (HODD, 30, [5, 300, 0], 24, 8), (HODD, 45, [130], 8, 8),
    (HTINY, 17, [64, 60, 2], 16, 8), (HTINY, 32, [1000], 64, 64), (HMHA, 65, [129, 0], 32, 16), (H2B, 16, [2600], 64, 16),
    (H2B, 17, [3, 900, 127], 128, 32), ((12, 2, 256, 0), 11, [0, 255], 64, 64), ((64, 1, 64, 32), 3, [250, 4], 16, 16),
    (H2B, 20, [40, 250], 16, 4), (HTINY, 40, [70], 16, 2),
]


@pytest.mark.parametrize("heads,T,lens,ps,sb", CHUNKS)
def test_attend_chunk(heads, T, lens, ps, sb):
    c = Case(BF16, heads, T, lens, ps, sb)
    c.check_out(*c.attend(c.set_q()))


@pytest.mark.parametrize("q_scale", [1e-3, 12.0])
def test_attend_chunk_flat_and_peaked(q_scale):
    """Scores that hardly differ, and ones whose maximum keeps rising along the keys (O is rescaled often)."""
    c = Case(BF16, H2B, 18, [700, 30], 64, 16, q_scale=q_scale)
    c.check_out(*c.attend(c.set_q()))
    for n in ("k", "v"):
        s = c.c[n + "_scales"]
        s.mul_(2.0 ** torch.randint(-12, 4, s.shape, generator=c.g).float())
        for p in range(0, 700, 16):
            s[c.table[0, p // 64], :, p % 64 // 16] = 2.0 ** (-13 + p / 90 // 1)
        c.d[n + "_scales"].copy_(s)
    c.check_out(*c.attend(c.set_q()))


def test_attend_chunk_sink():
    """One strong key and many weak ones that weigh the same: no rounding of weights may add up."""
    T = 12
    c = Case(BF16, H2B, T, [900], 64, 16)
    _uniform_codes(c, 0.0)
    q = torch.zeros(T, c.nh * c.hd, dtype=BF16)
    q.view(T, c.nh, c.hd)[..., 0] = 16.0
    c.q_buf.copy_(q)
    page, j = c.table[0, 3], 0
    sc = float(c.c["k_scales"][page, 0, j])
    c.c["k_pages"].view(torch.uint8)[page, :, 5, 0] = torch.tensor(min(9.0 / sc, 448.0)).to(kv8.F8).view(torch.uint8)
    c.d["k_pages"].view(torch.uint8).copy_(c.c["k_pages"].view(torch.uint8))
    c.check_out(*c.attend(q))


def test_attend_chunk_ignores_what_it_may_not_see():
    """NaN codes past the sequences, in pages of nobody and in a page that the table does not name; a
    negative length leaves the first queries without a key; a row of NaN and one of infinities."""
    T = 20
    c = Case(BF16, H2B, T, [3, 230, -7, 107], 64, 16, cap=320)
    c.table[1, 1] = -1
    c.table[3, 0] = 10 ** 6
    c.c["table"] = c.table.tolist()
    c.d["page_table"].copy_(c.table)
    P = c.c["k_pages"].shape[0]
    used = torch.zeros(P, 64, dtype=torch.bool)
    for b, n in enumerate(c.lens):
        for p in range(n + T):
            if 0 <= c.table[b, p // 64] < P:
                used[c.table[b, p // 64], p % 64] = True
    for n in ("k_pages", "v_pages"):
        raw = c.c[n].view(torch.uint8)
        raw[~used[:, None].expand(-1, c.nkv, -1)] = 0x7f
        c.d[n].view(torch.uint8).copy_(raw)
    q = c.set_q()
    c.check_out(*c.attend(q))
    q[5, 3], q[T + 6, 256] = math.nan, math.inf
    c.q_buf.copy_(q)
    want, tol = c.attend(q)
    assert torch.isnan(want).any() and torch.isfinite(want).any()
    c.check_out(want, tol)


def test_attend_chunk_past_the_capacity():
    """Tokens behind the last page are not there: their rows see what there is."""
    c = Case(BF16, H2B, 40, [100, 128, 300], 64, 16, cap=128, rows=400)
    c.check_out(*c.attend(c.set_q()))


def test_append_then_attend_chunk():
    """A prompt in chunks as a forward runs them, rows strided and not aligned, outputs beside others; a stored
    NaN key is seen by the rows at and behind it."""
    T = 33
    c = Case(BF16, H2B, T, [0, 70], 64, 16, cap=256)
    wide = torch.zeros(c.qkv.shape[0], c.qkv.shape[1] + 3, dtype=BF16, device=DEV)
    out = torch.full((2 * T + 2, c.nh * c.hd + 7), 3.0, dtype=BF16, device=DEV)
    d = c.layer(wide[:, 3:], out=out[:, 2:2 + c.nh * c.hd])
    for step in range(3):
        c.new_inputs()
        if step == 2:
            kv8.split(c.qkv, c.nh, c.nkv, c.hd)[2][T + 9, 1, 5] = math.inf
        wide[:, 3:].copy_(c.qkv)
        c.append(d)
        c.check_stored()
        want, tol = c.attend(c.q_buf.cpu(), d)
        c.out.copy_(out[:2 * T, 2:2 + c.nh * c.hd])
        c.check_out(want, tol)
        assert (out[2 * T:] == 3).all() and (out[:, :2] == 3).all() and (out[:, 2 + c.nh * c.hd:] == 3).all()
        c.lens = c.c["lens"] = [n + T for n in c.lens]
        c.d["seq_lens"].copy_(torch.tensor(c.lens, dtype=torch.int32))
    assert torch.isnan(want).any() and torch.isfinite(want).any()


def test_chunk_repeated_captured_and_two_at_once():
    """Repeated calls give the same bits, two layers at once on two streams too; a captured graph replays on
    new lengths and queries."""
    a, b = Case(BF16, H2B, 17, [700, 90, 1300], 64, 16, seed=1), Case(BF16, HMHA, 70, [10, 1100], 64, 16, seed=2)
    qa, qb = a.set_q(), b.set_q()
    da, db = a.layer(), b.layer()
    want = [a.attend(qa, da), b.attend(qb, db)]
    torch.cuda.synchronize()
    a0, b0 = a.out.clone(), b.out.clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(s1):
            K().attn_kv8_verify(da)
        with torch.cuda.stream(s2):
            K().attn_kv8_verify(db)
    torch.cuda.synchronize()
    assert torch.equal(a.out, a0) and torch.equal(b.out, b0)
    a.check_out(*want[0])
    b.check_out(*want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s1):
        K().attn_kv8_verify(da)
    a.lens = a.c["lens"] = [4, 1290, 0]
    a.d["seq_lens"].copy_(torch.tensor(a.lens, dtype=torch.int32))
    qa = a.set_q()
    g.replay()
    torch.cuda.synchronize()
    got = a.out.clone()
    a.check_out(*a.attend(qa, da))
    assert torch.equal(a.out, got)


@pytest.mark.parametrize("heads,T,lens,sb", [(H2B, 1100, [37, 0, 2000], 16), (HMHA, 1500, [0, 900], 64), (HMICRO, 3000, [5], 8)])
def test_attend_long_chunk(heads, T, lens, sb):
    """Many row groups a sequence: some tokens of each against the definition (bound as in `_attend_bound`)."""
    c = Case(BF16, heads, T, lens, 64, sb)
    q = c.set_q().double().view(-1, c.nh, c.hd)
    K().attn_kv8_verify(c.layer())
    got = c.out.double().cpu().view(-1, c.nh, c.hd)
    gate = torch.sigmoid(kv8.split(c.qkv, c.nh, c.nkv, c.hd)[1].double())
    rep = c.nh // c.nkv
    for b, n in enumerate(lens):
        for t in (0, 1, 15, 16, 17, 63, 127, 128, T // 2, T - 2, T - 1):
            m, row = n + t + 1, b * T + t
            k, v, has = kv8.read(c.c, b, m)
            assert has.all()
            for g in range(c.nkv):
                h = slice(g * rep, (g + 1) * rep)
                s = q[row, h] @ k[g].T * c.hd ** -0.5
                want = torch.softmax(s, -1) @ v[g] * gate[row, h]
                A = (q[row, h].abs() @ k[g].abs().T).amax(-1, keepdim=True) * c.hd ** -0.5 + 1
                tol = (2 * (c.hd + 2) * 2.0 ** -23 * A + 2 * m * 2.0 ** -23 + 2.0 ** -8 + m * 2.0 ** -18) * v[g].abs().max() * gate[row, h]
                assert ((got[row, h] - want).abs() <= tol + (want.abs() + tol) * torch.finfo(BF16).eps / 2).all(), (b, t, g)
    assert K().device_status() == 0
