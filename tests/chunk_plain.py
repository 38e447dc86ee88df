"""Plain forms in 64 bits of attention of chunks, for the test of its kernels."""
import torch


def decoded(rows, scale, kind):
    """Rows of a cache (torch tensors, 0 f16, 1 q8, 2 q4) in 64 bits."""
    if kind == 0:
        return rows.double()
    if kind == 1:
        q = rows.double()
    else:
        b = rows.unflatten(-1, (-1, 16))
        q = torch.cat([b & 15, b >> 4], -1).flatten(-2).double() - 8
    return q * scale.double().repeat_interleave(32, -1)


def attention(q, k, v, seen, scale, softcap=0.0, sinks=None, half=False, quants=False, q_half=False):
    """One sequence. q [rows, heads, d], k and v [positions, kv heads, d] in 64 bits, seen [rows, positions] -> (out, tolerance).

    The tolerance counts, against a = sum(w |v|) / sum(w), with s the scores and S = scale sum|q||k| of the largest position that a row sees:
      f32: queries in two f16 terms 2^-22 of S; over quants, whose values are two terms exactly, the product of both second terms (2^-11 each) is left out,
      2^-22 of S and of a; half: f32 queries rounded to 11 bits, 2^-11 of S (f16 ones enter as they are), quants' keys and values
      rounded to f16, 2^-11 of S and of a, 2^-25 (f16's last step, halved) sum|q| scale and 2^-25 besides
      products summed in f32 in steps of 16, truncations included: (d / 16 + 4) 2^-23 S (two terms: twice as many, over quants three times)
      half: half of the exponentials are a polynomial's, 7.5e-5 < 2^-13 off, in numerator and denominator
      the score times log2(e), its difference from the reference and the exponential: 2^-23 (|s| + |max|) + 2^-21; tanh by 2^-21 of the softcap
      a weight is off by the sum of these, in numerator and denominator; f32: weights in two f16 terms 2^-22; half: rounded to f16, 2^-11; f16 ends in steps of
      2^-24, and weights are times 2^7 or more under the greatest: 2^-25 / 2^7 max|v| for each position that is seen
      sums over the positions in steps of 16, and the joining of up to 300 parts: 2^-23 each
      half: the result is rounded, 2^-11 of itself and 2^-25.
    """
    group = q.shape[1] // k.shape[1]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    if not k.shape[0]:
        return out, tol
    n = seen.sum(1).double()[:, None]
    vmax = torch.where(torch.isfinite(v), v, 0).abs().amax()
    for h in range(q.shape[1]):
        kk, vv, qq = k[:, h // group], v[:, h // group], q[:, h]
        s = torch.where(seen, qq @ torch.nan_to_num(kk, 0.0, 0.0, 0.0).T, 0) * scale
        size = (torch.where(seen, qq.abs() @ torch.nan_to_num(kk, 0.0, 0.0, 0.0).abs().T, 0) * abs(scale)).amax(1, keepdim=True)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        most = s.abs().amax(1, keepdim=True)
        # a key that is no number: what it does to the rows that see it is theirs alone
        odd = ~torch.isfinite(kk).all(1)
        s = torch.where(odd & seen, torch.nan, s)
        z = torch.where(seen, s, -torch.inf)
        top = z.nan_to_num(nan=0.0, neginf=-torch.inf).amax(1, keepdim=True)
        if sinks is not None:
            top = torch.maximum(top, sinks[h].double())
        top = torch.where(torch.isinf(top) & (top < 0), 0, top)
        w = torch.exp(z - top)
        total = w.sum(1, keepdim=True) + (torch.exp(sinks[h].double() - top) if sinks is not None else 0)
        safe = torch.where(total > 0, total, 1)
        good = torch.where(torch.isfinite(vv), vv, 0)
        o, a = w @ good / safe, w.nan_to_num(nan=0.0) @ good.abs() / safe
        # values that are no numbers reach the rows that see them, in their column
        bad = torch.where(torch.isfinite(vv), 0, vv)
        for p in torch.nonzero((bad != 0).any(1)).flatten().tolist():
            o = torch.where(seen[:, p:p + 1] & (bad[p] != 0), o + bad[p], o)
        out[:, h] = o
        off = (2.0 ** -11 * ((not q_half) + quants) if half else 2.0 ** -22 * (1 + quants)) * size + (d_steps(q) * (1 if half else 3 if quants else 2)) * 2.0 ** -23 * size
        if half and quants:
            off = off + 2.0 ** -25 * qq.abs().sum(1, keepdim=True) * abs(scale)
        off = off + 2.0 ** -23 * (most + top.abs()) + 2.0 ** -21 + softcap * 2.0 ** -21
        t = a * (2 * off + (2.0 ** -11 * (1 + quants) + 2.0 ** -12 if half else 2.0 ** -22 * (2 + quants)) + (n / 16 + 300) * 2.0 ** -23) + n * 2.0 ** -32 * vmax / safe.clamp(min=1.0)
        if half:
            t = t + 2.0 ** -11 * o.abs() + 2.0 ** -25 * (2 + quants)
        tol[:, h] = torch.where(n > 0, t, 0)
    return out, tol


def d_steps(q):
    return q.shape[-1] / 16 + 4


def seen_of(rows, length, window=0, there=None):
    """[rows, length]: what the rows of a sequence see, the last of whose `length` positions are theirs."""
    at = length - rows + torch.arange(rows, device="cuda")[:, None]
    p = torch.arange(max(length, 0), device="cuda")
    seen = p <= at
    if window:
        seen &= p > at - window
    return seen if there is None else seen & there
