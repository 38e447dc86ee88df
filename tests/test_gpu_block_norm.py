"""Norms either side of a block with its gate and residual, against the formula in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def plain(x, weight, residual, post_weight, post, gate, alpha, eps, offset, half):
    """(y, h, tolerance of y, of h). u = 2^-24. A mean of squares: a thread's up to 64 values one after the other, then trees of ten steps, all of one sign: (64 + 10 + 2) u
    relative, half of it after the root; the root, the quotient and the sum with eps 3 u; the factor, offset + weight and each product one u more. h: the
    product with alpha, the sum: u of each term. y's factor changes by h's own error (its 2-norm against h's): no more than the largest relative one
    against the row's root mean square; f16: 2^-11 of the value, 2^-25."""
    u = 2.0 ** -24
    x = x.astype(np.float64)
    n = x.shape[1]
    p, p_off = x, np.zeros_like(x)
    if post:
        f = 1 / np.sqrt((x ** 2).mean(1, keepdims=True) + eps)
        p = x * f * ((offset + post_weight.astype(np.float64)) if post_weight is not None else 1.0)
        p_off = np.abs(x * f) * (np.abs(offset) + np.abs(post_weight) if post_weight is not None else 1.0) * 46 * u
    g = 1.0 if gate is None else gate.astype(np.float64)
    r = 0.0 if residual is None else residual.astype(np.float64)
    h = r + alpha * g * p
    h_off = np.abs(alpha * g) * (p_off + 3 * u * np.abs(p)) + u * (np.abs(h) + np.abs(r))
    f = 1 / np.sqrt((h ** 2).mean(1, keepdims=True) + eps)
    w = offset + weight.astype(np.float64) if weight is not None else 1.0
    w_abs = np.abs(offset) + np.abs(weight) if weight is not None else 1.0
    y = h * f * w
    grows = np.sqrt((h_off ** 2).mean(1, keepdims=True)) * f
    y_off = f * w_abs * (h_off + np.abs(h) * (46 * u + grows)) + 1e-40
    if half:
        y_off = y_off + 2.0 ** -11 * np.abs(y) + 2.0 ** -25
    return y, h, y_off * 1.001, h_off * 1.001 + 1e-40


def check(cuda, rows, n, residual=True, weight=True, post_weight=False, post=None, gate=None, alpha=0.7, eps=1e-5, offset=0.0, half=False, size=1.0, skew=0):
    import torch
    rng = np.random.default_rng(rows * 7 + n)
    f = lambda *s: (size * rng.standard_normal(s)).astype(np.float32)  # noqa: E731
    x, r = f(rows, n), 2 * f(rows, n) if residual else None
    w, pw = f(n) + 1 if weight else None, f(n) if post_weight else None
    g = {None: None, "vector": f(n), "rows": f(rows, n)}[gate]

    def dev(a):
        if a is None:
            return None
        t = torch.from_numpy(a).cuda()
        if skew and a.ndim == 2:   # rows apart, off their 16-byte boundaries
            wide = torch.zeros((a.shape[0], n + 2 * skew), device="cuda")
            wide[:, skew:skew + n] = t
            return wide[:, skew:skew + n]
        return t
    y, h = cuda.block_norm(dev(x), dev(w), dev(r), dev(pw), post, dev(g), alpha, eps, offset, torch.float16 if half else None)
    assert y.dtype == (torch.float16 if half else torch.float32) and h.dtype == torch.float32
    want_y, want_h, y_off, h_off = plain(x, w, r, pw, bool(post or post_weight), g, np.float64(np.float32(alpha)), np.float64(np.float32(eps)), np.float64(np.float32(offset)), half)
    for name, got, want, off in (("h", h, want_h, h_off), ("y", y, want_y, y_off)):
        d = np.abs(got.cpu().numpy().astype(np.float64) - want)
        assert (d <= off).all(), f"{name}: {float((d / off).max()):.3g} of the tolerance"
    return x, r, w, pw, g, y, h


@pytest.mark.parametrize("n", [1, 2, 3, 4, 31, 33, 100, 512, 1000, 2048, 4096, 4097, 5120, 8192, 11008, 16384, 16388, 20001, 65536])
@pytest.mark.parametrize("rows", [1, 5])
def test_widths(cuda, n, rows):
    check(cuda, rows, n, post_weight=True, gate="vector")
    check(cuda, rows, n, half=True)


@pytest.mark.parametrize("n", [64, 4096, 4100, 17000])
def test_parts(cuda, n):
    check(cuda, 3, n, residual=False, weight=False, alpha=1.0)
    check(cuda, 3, n, post=True, weight=False, gate="rows", half=True)
    check(cuda, 3, n, post_weight=True, offset=1.0, gate="rows")
    check(cuda, 3, n, alpha=-2.0, eps=0.0)
    check(cuda, 3, n, residual=False, post=True)
    check(cuda, 3, n, post_weight=True, gate="rows", skew=1)
    check(cuda, 3, n, post_weight=True, gate="vector", skew=3, half=True)


@pytest.mark.parametrize("size", [1e-12, 1e-3, 1e4])
def test_sizes(cuda, size):
    check(cuda, 2, 1000, size=size, post_weight=True)


def test_in_place_and_zeros(cuda):
    import torch
    for n in (256, 4096, 20004):
        x, r, w, pw, g, y, h = check(cuda, 4, n, post_weight=True, gate="vector")
        t = [torch.from_numpy(a).cuda() for a in (x, w, r, pw, g)]
        for at in (0, 2):   # h in the place of x, of the residual
            args = [a.clone() for a in t]
            y2, h2 = cuda.block_norm(args[0], args[1], args[2], args[3], gate=args[4], alpha=0.7, eps=1e-5, h_out=args[at])
            assert h2 is args[at] and torch.equal(y2, y) and torch.equal(h2, h)
        out = torch.full((4, n + 4), 5.0, dtype=torch.float16, device="cuda")
        cuda.block_norm(*t[:4], gate=t[4], alpha=0.7, eps=1e-5, out=out[:, :n])
        assert torch.equal(out[:, :n], y.half()) and (out[:, n:] == 5).all()
    z = torch.zeros((3, 100), device="cuda")
    assert (cuda.block_norm(z, z[0], z, post_norm=True)[0] == 0).all()
    assert cuda.block_norm(z[:0])[0].shape == (0, 100) and cuda.block_norm(z[:, :0])[0].shape == (3, 0)
    bad = z.clone()
    bad[1, 5] = float("nan")
    y, h = cuda.block_norm(bad, residual=z + 1)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2]]).all() and torch.isnan(h[1]).sum() == 1


def test_without_h(cuda):
    """The C call without a place for h, over rows that the registers hold and wider ones."""
    import ctypes as C

    import torch
    for n in (4096, 20000):
        x, r = torch.randn((2, n), device="cuda"), torch.randn((2, n), device="cuda")
        want, _ = cuda.block_norm(x, residual=r, post_norm=True)
        y = torch.zeros_like(x)
        m = cuda.Norm(residual=r.data_ptr(), rows=2, n=n, x_stride=n, residual_stride=n, y_stride=n, post_norm=1, alpha=1.0, eps=1e-6)
        assert cuda.lib.krk_cuda_block_norm(y.data_ptr(), None, x.data_ptr(), C.byref(m), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(y, want)


@pytest.mark.parametrize("n", [1024, 1540, 2052, 4096, 4100])
@pytest.mark.parametrize("rows", [887, 1000, 2500])
def test_many_rows(cuda, n, rows):
    """The same bits as for a few rows at a time, whatever a row's neighbours are; rows in place, rows apart, without h."""
    import ctypes as C

    import torch
    gen = torch.Generator("cuda").manual_seed(n + rows)
    x, r = (torch.randn((rows, n + 4), device="cuda", generator=gen)[:, :n] for _ in range(2))
    x *= torch.exp(2 * torch.randn((rows, 1), device="cuda", generator=gen))
    w, pw, g = (torch.rand(n, device="cuda", generator=gen) + 0.5 for _ in range(3))
    for more in (dict(), dict(residual=r, weight=w), dict(residual=r, weight=w, post_weight=pw, gate=g, alpha=0.7, dtype=torch.float16), dict(post_norm=True, offset=1.0, weight=w),
                 dict(residual=r, post_weight=pw, offset=1.0)):
        y, h = cuda.block_norm(x, **more)
        for a in range(0, rows, 400):
            few = {k: v[a:a + 400] if k == "residual" else v for k, v in more.items()}
            y2, h2 = cuda.block_norm(x[a:a + 400], **few)
            assert torch.equal(y[a:a + 400], y2) and torch.equal(h[a:a + 400], h2)
    y, h = cuda.block_norm(x, w, r, pw)
    for place in (0, 1):
        args = [x.clone(), r.clone()]
        y2, h2 = cuda.block_norm(args[0], w, args[1], pw, h_out=args[place])
        assert torch.equal(y2, y) and torch.equal(args[place], h)
    both = x.clone()
    assert torch.equal(cuda.block_norm(both, w, r, pw, out=both)[0], y)
    y2 = torch.full((rows, n + 4), 3.0, device="cuda")
    m = cuda.Norm(residual=r.data_ptr(), weight=w.data_ptr(), post_weight=pw.data_ptr(), rows=rows, n=n, x_stride=n + 4, residual_stride=n + 4, y_stride=n + 4, post_norm=1, alpha=1.0,
                  eps=1e-6)
    assert cuda.lib.krk_cuda_block_norm(y2.data_ptr(), None, x.data_ptr(), C.byref(m), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(y2[:, :n], y) and (y2[:, n:] == 3).all()
