"""The 8-bit KV cache in plain torch on the CPU, token by token in 64 bits: the oracle of
`qsp_attn_kv8_prep` and `qsp_attn_kv8_verify`.

A cache is a dict: k_pages, v_pages [P, n_kv, ps, hd] float8_e4m3fn, k_scales, v_scales
[P, n_kv, ps / sb] fp32, table [B, max_pages] and lens [B] (Python lists of ints)."""

from __future__ import annotations

import math

import torch

F8 = torch.float8_e4m3fn
MIN_EXP = -40


def scale_exp(amax: float) -> int:
    """The least e >= -40 with amax <= 448·2^e."""
    e = MIN_EXP
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def e4m3(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.float32).to(F8)


def new_cache(pages, n_kv, ps, hd, sb, table, lens):
    z = lambda: torch.zeros(pages, n_kv, ps, hd, dtype=torch.uint8).view(F8)
    one = lambda: torch.ones(pages, n_kv, ps // sb)
    return dict(k_pages=z(), v_pages=z(), k_scales=one(), v_scales=one(), table=[list(r) for r in table], lens=list(lens))


def normed_rotated(x, w, cos, sin, eps):
    """x [..., hd] in 64 bits -> RMS-normed, times 1 + w, first rd dims rotated."""
    x, w, cos, sin = (t.double() for t in (x, w, cos, sin))
    y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * (1 + w)
    rd = cos.shape[-1]
    a, b = y[..., :rd // 2], y[..., rd // 2:rd]
    h = rd // 2
    return torch.cat([a * cos[..., :h] - b * sin[..., :h], b * cos[..., h:] + a * sin[..., h:], y[..., rd:]], -1)


def split(qkv, nh, nkv, hd):
    """Rows of [q|gate per head, k, v] -> q, gate [N, nh, hd], k, v [N, nkv, hd]."""
    n = qkv.shape[0]
    qg = qkv[:, :2 * nh * hd].reshape(n, nh, 2, hd)
    k = qkv[:, 2 * nh * hd:(2 * nh + nkv) * hd].reshape(n, nkv, hd)
    v = qkv[:, (2 * nh + nkv) * hd:(2 * nh + 2 * nkv) * hd].reshape(n, nkv, hd)
    return qg[:, :, 0], qg[:, :, 1], k, v


def append(c, qkv, T, nh, qn, kn, cos, sin, eps=1e-6):
    """Stores the T tokens of every sequence after its lens (not moved); returns q [B·T, nh, hd] in
    64 bits and whether a position had no place."""
    P, nkv, ps, hd = c["k_pages"].shape
    sb = ps // c["k_scales"].shape[2]
    q, _, k, v = split(qkv, nh, nkv, hd)
    qs, bad = [], False
    for b, n in enumerate(c["lens"]):
        todo = {}                                    # (page, block) -> [(slot, token row)]
        for t in range(T):
            p, m = n + t, b * T + t
            at = p if 0 <= p < cos.shape[0] else 0
            qs.append(normed_rotated(q[m], qn, cos[at], sin[at], eps))
            page = c["table"][b][p // ps] if 0 <= p < cos.shape[0] and p // ps < len(c["table"][b]) else -1
            if not 0 <= page < P:
                bad = True
                continue
            todo.setdefault((page, p % ps // sb), []).append((p % ps, m, p))
        for (page, j), tokens in todo.items():
            for g in range(nkv):
                ys = {"k": [], "v": []}
                for slot, m, p in tokens:
                    yk = normed_rotated(k[m, g], kn, cos[p], sin[p], eps).float()
                    yv = v[m, g].float()
                    if not (torch.isfinite(yk).all() and torch.isfinite(yv).all()):
                        yk = torch.full_like(yk, math.nan)
                    if not torch.isfinite(yv).all():
                        yv = torch.zeros_like(yv)
                    ys["k"].append(yk)
                    ys["v"].append(yv)
                for name, y in ys.items():
                    pages, scales = c[name + "_pages"], c[name + "_scales"]
                    y = torch.stack(y)
                    fine = y[torch.isfinite(y)]
                    e = scale_exp(float(fine.abs().max()) if fine.numel() else 0.0)
                    first = tokens[0][0]
                    if first % sb:
                        was = round(math.log2(float(scales[page, g, j])))
                        e = max(e, was)
                        old = pages[page, g, j * sb:first].double() * 2.0 ** (was - e)
                        pages.view(torch.uint8)[page, g, j * sb:first] = e4m3(old).view(torch.uint8)
                    pages.view(torch.uint8)[page, g, first:first + len(y)] = e4m3(y.double() * 2.0 ** -e).view(torch.uint8)
                    scales[page, g, j] = 2.0 ** e
    return torch.stack(qs), bad


def read(c, b, n):
    """The first n keys and values of sequence b, [n_kv, n, hd] in 64 bits, and which have a page."""
    P, nkv, ps, hd = c["k_pages"].shape
    sb = ps // c["k_scales"].shape[2]
    k, v = torch.zeros(2, nkv, n, hd, dtype=torch.float64).unbind()
    has = torch.zeros(n, dtype=torch.bool)
    for lp in range(-(-n // ps)):
        page = c["table"][b][lp] if lp < len(c["table"][b]) else -1
        if not 0 <= page < P:
            continue
        m = min(ps, n - lp * ps)
        at = slice(lp * ps, lp * ps + m)
        has[at] = True
        for x, name in ((k, "k"), (v, "v")):
            s = c[name + "_scales"][page].double().repeat_interleave(sb, -1)[:, :m, None]
            x[:, at] = c[name + "_pages"][page, :, :m].double() * s
    return k, v, has


def attend(c, q, gate, T, scale):
    """q, gate [B·T, nh, hd] -> gated attention over lens + t + 1 keys, [B·T, nh, hd] in 64 bits."""
    nkv = c["k_pages"].shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    rep = q.shape[1] // nkv
    for b, n in enumerate(c["lens"]):
        if n + T <= 0:
            continue
        k, v, has = read(c, b, n + T)
        for t in range(T):
            m = n + t + 1
            if m <= 0 or not has[:m].any():
                continue
            at = has[:m]
            for g in range(nkv):
                h = slice(g * rep, (g + 1) * rep)
                s = q[b * T + t, h].double() @ k[g, :m][at].T * scale
                out[b * T + t, h] = torch.softmax(s, -1) @ v[g, :m][at]
    return out * torch.sigmoid(gate.double())
