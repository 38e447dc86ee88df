"""Plain forms in 64 bits of the operators between the projections and the output projection, for the tests of their kernels."""
import numpy as np


def encode(x, kind):
    """f32 [..., d] as a cache holds it: (quants, scales) or (f16, None). kind: 0 f16, 1 q8, 2 q4."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        if kind == 0:
            return np.where(np.isfinite(x), np.clip(x, -65504, 65504), x).astype(np.float16), None
        b = x.reshape(*x.shape[:-1], -1, 32)
        odd = ~np.isfinite(b).all(-1)
        hi, lo = b.max(-1), b.min(-1)
        top = np.maximum(hi, -lo) if kind == 1 else np.where(hi >= -lo, hi, lo)
        d = np.clip((top / np.float32(127 if kind == 1 else -8)).astype(np.float32), -65504, 65504).astype(np.float16)
        d = np.where(odd, np.float16(np.nan), d)
        q = np.rint(b / d.astype(np.float32)[..., None])
        q = np.where((d == 0)[..., None] | odd[..., None], 0, q)
        if kind == 1:
            return np.clip(q, -127, 127).astype(np.int8).reshape(x.shape), d
        q = (np.clip(q, -8, 7) + 8).astype(np.uint8)
        return (q[..., :16] | q[..., 16:] << 4).reshape(*x.shape[:-1], -1), d


def decode(rows, scale, kind):
    """Rows of a cache in 64 bits."""
    rows = np.asarray(rows)
    if kind == 0:
        return rows.astype(np.float64)
    if kind == 1:
        q = rows.reshape(*rows.shape[:-1], rows.shape[-1] // 32, 32).astype(np.float64)
    else:
        b = rows.reshape(*rows.shape[:-1], rows.shape[-1] // 16, 16)
        q = np.concatenate([b & 15, b >> 4], -1).astype(np.float64) - 8
    return (q * np.asarray(scale, np.float64)[..., None]).reshape(*q.shape[:-2], 32 * q.shape[-2])


def attention(q, k, v, seen, scale, softcap=0.0, sinks=None):
    """One sequence. q [rows, heads, d], k and v [positions, kv heads, d], seen [rows, positions] -> (out, tolerance).

    The tolerance counts, for each output, against sum(w |v|) / sum(w) =: a, with s the scores:
      queries in two f16 terms 2^-22, products summed in f32 in steps of 16 (a rounding of 2^-23 each, truncations included): a score is off by
      at most (2^-22 + (d / 16 + 4) 2^-23) scale sum|q||k|; the score times log2(e), its difference from the maximum (a second time where that rises) and the exponential
      round by 2 2^-24 (|s| + |max|) + 2^-22, tanh by 2^-21 of the softcap; a weight is off by the sum of these, in numerator and denominator;
      weights in two f16 terms 2^-22 each, times 2^14 under a power of two up to twice the values' greatest scale; f16 ends in steps of 2^-24, so a weight
      is off by 2^-25 / 2^14 of twice the greatest value besides, whatever its own size (what is left of a
      sum where the heavy positions' values are zeros); with many rows weights are times 2^11 under a reference that the greatest weight is up to 2^4
      above: 2^-25 / 2^11 of the greatest value, 2^-35 max|v| for each position that is seen covers both; sums over the positions: a step of 16 of each of four warps and the joining of up to 300 parts, 2^-23 each.
    """
    rows, heads, d = q.shape
    group = heads // k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    n = k.shape[0]
    for h in range(heads):
        kk, vv = k[:, h // group].astype(np.float64), v[:, h // group].astype(np.float64)
        qq = q[:, h].astype(np.float64)
        for r in range(rows):
            at = np.flatnonzero(seen[r])
            if not len(at):
                continue
            with np.errstate(all="ignore"):
                s = kk[at] @ qq[r] * scale
                size = np.abs(kk[at]) @ np.abs(qq[r]) * abs(scale)
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                top = max(s.max(), sinks[h]) if sinks is not None else s.max()
                w = np.exp(s - top)
                total = w.sum() + (np.exp(sinks[h] - top) if sinks is not None else 0.0)
                out[r, h] = w @ vv[at] / total
                a = w @ np.abs(vv[at]) / total
                off = (2.0 ** -22 + (d / 16 + 4) * 2.0 ** -23) * size.max() + 2.0 ** -24 * 2 * (np.abs(s).max() + abs(top)) + 2.0 ** -22 + softcap * 2.0 ** -21
                floor = len(at) * 2.0 ** -35 * np.nan_to_num(np.abs(v.astype(np.float64)), nan=0.0, posinf=0.0).max() * np.exp(s.max() - top) / total
                tol[r, h] = a * (2 * off + 2.0 ** -21 + (n / 16 + 300) * 2.0 ** -23) + floor
    return out, tol


def visible(masks, n_q, length, window=0):
    """[n_q, length]: what a sequence's rows see."""
    seen = np.zeros((n_q, max(length, 0)), bool)
    before = length - n_q
    for i in range(n_q):
        m = int(masks[i]) if masks is not None else (2 << i) - 1
        row = before + bin(m).count("1") - 1
        for p in range(max(0, row - window + 1) if window else 0, max(before, 0)):
            seen[i, p] = True
        for j in range(n_q):
            if before + j >= 0 and m >> j & 1:
                seen[i, before + j] = True
    return seen
