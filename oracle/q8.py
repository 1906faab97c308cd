"""64-bit restatements (numpy) of the 8-bit K/V cache operators and of the token log
probabilities, from their formulas: test infrastructure, no counterpart in the reference.
"""

from __future__ import annotations

import math

import numpy as np

E4M3_MAX = 448.0
MIN_SCALE_EXP = -100


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 codes: sign, 4 exponent bits (bias 7), 3 fraction bits."""
    c = np.arange(256)
    e, f = (c >> 3) & 15, (c & 7).astype(np.float64)
    v = np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0))
    v = np.where((c & 0x7F) == 0x7F, np.nan, v)
    return np.where(c >= 128, -v, v)


_POS = e4m3_values()[:127]      # 0 .. 448, increasing


def e4m3_round(x) -> np.ndarray:
    """Nearest e4m3 value, ties to the even code; NaN for what is not finite."""
    x = np.asarray(x, dtype=np.float64)
    fine = np.isfinite(x)
    a = np.minimum(np.abs(np.where(fine, x, 0.0)), E4M3_MAX)
    hi = np.clip(np.searchsorted(_POS, a), 1, 126)
    lo = hi - 1
    dl, dh = a - _POS[lo], _POS[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.where(fine, np.copysign(_POS[pick], np.where(fine, x, 0.0)), np.nan)


def scale_for(amax: float) -> float:
    k = MIN_SCALE_EXP
    if amax > E4M3_MAX * 2.0 ** k:
        k = int(math.floor(math.log2(amax / E4M3_MAX))) - 1
        while amax > E4M3_MAX * 2.0 ** k:
            k += 1
    return 2.0 ** max(k, MIN_SCALE_EXP)


def write_kv_slots(x, slots, codes, scale):
    """One of K and V.  x [T,H,D], slots [T], codes [N,bs,H,D] (values of the codes), scale
    [N,H]; returns the new codes and scales (float64)."""
    x = np.asarray(x, dtype=np.float64)
    codes, scale = np.array(codes, dtype=np.float64), np.array(scale, dtype=np.float64)
    n, bs, heads = codes.shape[:3]
    rows = {}
    for t, s in enumerate(np.asarray(slots).tolist()):
        if 0 <= s < n * bs:
            rows.setdefault(s // bs, {})[s % bs] = t      # the last row for a slot stays
    for b, new in rows.items():
        for h in range(heads):
            mine = np.stack([x[t, h] for t in new.values()])
            fine = np.abs(mine[np.isfinite(mine)])
            old = 0.0 if 0 in new else scale[b, h]
            if not (old > 0 and np.isfinite(old)):
                old = 0.0
            now = max(old, scale_for(fine.max() if fine.size else 0.0))
            for o in range(bs):
                if o in new:
                    codes[b, o, h] = e4m3_round(x[new[o], h] / now)
                elif 0 in new:
                    codes[b, o, h] = 0.0
                elif now != old:
                    codes[b, o, h] = e4m3_round(codes[b, o, h] * (old / now))
            scale[b, h] = now
    return codes, scale


def paged_decode(q, k_codes, v_codes, k_scale, v_scale, tables, ctx, max_context_len=None):
    """q [B,1,Hq,D] -> (out, sum_t p_t |v_t|, max_t sum_d |q_d k_td| / sqrt(D), max_d |q_d| max_t sum_d |k_td| / sqrt(D),
    max |v|): the output, and for error bounds per output element, and per head."""
    q = np.asarray(q, dtype=np.float64)
    B, _, hq, d = q.shape
    n, bs, hkv = k_codes.shape[:3]
    g = hq // hkv
    out, mass = np.zeros_like(q), np.zeros_like(q)
    span, wide, vmax = np.zeros((B, hq)), np.zeros((B, hq)), np.zeros((B, hq))
    width = tables.shape[1]
    if max_context_len is not None:
        width = min(width, -(-max_context_len // bs))
    for b in range(B):
        c = min(int(ctx[b]), width * bs)
        if c <= 0:
            continue
        t = np.arange(c)
        blk, off = tables[b][t // bs].astype(np.int64), t % bs
        ok = (blk >= 0) & (blk < n)
        safe = np.where(ok, blk, 0)
        k = np.where(ok[:, None, None], k_codes[safe, off].astype(np.float64) * k_scale[safe][..., None].astype(np.float64), 0.0)
        v = np.where(ok[:, None, None], v_codes[safe, off].astype(np.float64) * v_scale[safe][..., None].astype(np.float64), 0.0)
        for h in range(hq):
            kh, vh = k[:, h // g], v[:, h // g]
            s = kh @ q[b, 0, h] / math.sqrt(d)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[b, 0, h] = p @ vh
            mass[b, 0, h] = p @ np.abs(vh)
            span[b, h] = (np.abs(kh) @ np.abs(q[b, 0, h])).max() / math.sqrt(d)
            wide[b, h] = np.abs(q[b, 0, h]).max() * np.abs(kh).sum(-1).max() / math.sqrt(d)
            vmax[b, h] = np.abs(vh).max()
    return out, mass, span, wide, vmax


def token_logprobs(logits, tokens, top_k):
    """-> (logprobs, entropy, top_logprobs, top_tokens, E|d|, E d^2) with d = x - max under the row's distribution."""
    x = np.asarray(logits, dtype=np.float64)
    rows, vocab = x.shape
    with np.errstate(all="ignore"):
        m = x.max(-1, keepdims=True)
        e = np.exp(x - m)
        s = e.sum(-1, keepdims=True)
        logp = (x - m) - np.log(s)
        p = e / s
        d = np.where(e > 0, x - m, 0.0)
        entropy = np.log(s[:, 0]) - (p * d).sum(-1)
    tok = np.asarray(tokens)
    inside = (tok >= 0) & (tok < vocab)
    lp = np.where(inside, logp[np.arange(rows), np.where(inside, tok, 0)], -np.inf)
    bad = np.isnan(x)
    order = np.lexsort((np.broadcast_to(np.arange(vocab), x.shape), -np.where(bad, 0.0, x) + 0.0, ~bad), axis=-1)[:, :top_k]
    return lp, entropy, np.take_along_axis(logp, order, -1), order.astype(np.int32), -(p * d).sum(-1), (p * d * d).sum(-1)
