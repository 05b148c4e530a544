"""The operators around a block from their definitions in 64 bits, each result with the magnitude of what was added up for it
(what fp32 rounding errors are relative to), and dropout's numbers from integers."""
import numpy as np
import torch

EPS = 1e-6


def philox4x32_10(counter, key):
    """Four 32-bit words, from Salmon et al., "Parallel random numbers: as easy as 1, 2, 3" (2011), in Python integers."""
    c, k, low = list(counter), list(key), 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def factor(p, seed, offset, start, count):
    """Dropout's factor of the elements start .. start + count - 1, float64."""
    t = int(p * 65536 + 0.5)
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    seed, offset = seed & (1 << 64) - 1, offset & (1 << 64) - 1
    g = np.arange(start // 8, (start + count + 7) // 8, dtype=np.uint64)
    c = [g & low, g >> sh, np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> sh) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> sh) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    halves = np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], -1).reshape(-1)
    at = start - 8 * (start // 8)
    return torch.from_numpy(np.where(halves[at:at + count] >= t, 65536.0 / (65536.0 - t), 0.0))


def norm(x, w, du=None):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    xh = x * r
    got = {"u": (w * xh, (w * xh).abs())}
    if du is not None:
        t = w * du
        c = (t * xh).mean(-1, keepdim=True)
        ca = (t * xh).abs().mean(-1, keepdim=True)
        got["dx"] = r * (t - xh * c), r * (t.abs() + xh.abs() * ca)
        got["dw"] = (du * xh).sum(0), (du * xh).abs().sum(0)
    return got


def residual(x, y, w=None, gate=None, kind="", scale=1.0, w_next=None, m=1.0, dout=None, du=None, grad=False):
    """float64 [tokens, d] rows; `gate` shaped to broadcast. Gradients in closed form."""
    g = 1.0 if gate is None else gate
    ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) if w is not None else 1.0
    yh = y * ry
    ww = 1.0 if w is None else w
    b = ww * yh * m
    o = x + scale * (g * b)
    oa = x.abs() + (scale * g * b).abs()
    got = {"out": (o, oa)}
    if w_next is not None:
        ro = torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS)
        oh, oha = o * ro, oa * ro
        got["u"] = w_next * oh, (w_next * oha).abs()
    if not grad:
        return got
    D, Da = torch.zeros_like(x), torch.zeros_like(x)
    if dout is not None:
        D, Da = dout.clone(), dout.abs()
    if du is not None:
        t = w_next * du
        D = D + ro * (t - oh * (t * oh).mean(-1, keepdim=True))
        Da = Da + ro * (t.abs() + oha * (t.abs() * oha).mean(-1, keepdim=True))
        got["dw_next"] = (du * oh).sum(0), (du.abs() * oha).sum(0)
    got["dx"] = D, Da
    a, aa = D * m * yh, Da * m * yh.abs()
    got["dscale"] = (g * ww * a).sum().reshape(1), (g * ww * aa).abs().sum().reshape(1)
    dg, dga = scale * ww * a, (scale * ww * aa).abs()
    if kind == "channel":
        got["dgate"] = dg.sum(0), dga.sum(0)
    elif kind == "token":
        got["dgate"] = dg.sum(-1, keepdim=True), dga.sum(-1, keepdim=True)
    elif kind == "full":
        got["dgate"] = dg, dga
    E, Ea = scale * (g * m * D), (scale * (g * m * Da)).abs()
    if w is not None:
        got["dw"] = (E * yh).sum(0), (Ea * yh.abs()).sum(0)
        t, ta = w * E, w.abs() * Ea
        E = ry * (t - yh * (t * yh).mean(-1, keepdim=True))
        Ea = ry * (ta + yh.abs() * (ta * yh.abs()).mean(-1, keepdim=True))
    got["dy"] = E, Ea
    return got


def check(name, got, want, magnitude, steps=64):
    """One rounding to the result's type (half a step), and `steps` fp32 roundings relative to what was added up."""
    half = torch.finfo(got.dtype).eps / 2
    tol = half * want.abs() + steps * 2.0 ** -24 * magnitude + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / tol).max()):.3g} tolerances"


def ffn(x, wg, wu, wd, act, dy=None):
    """float64; each result with (a bound on) how far the kernels' roundings can move it: bf16 roundings of what is kept
    between the products (h, dg, du: 2^-8 relative each; act'(g) u and act(g): cut to 24 bits, 2^-16), and fp32 accumulation, at most one rounding of
    2^-23 (the tensor core may cut off) for every 16 columns of k, relative to the sum of the magnitudes."""
    half, step = 2.0 ** -8, 2.0 ** -23
    acc = lambda k: (k / 16 + 4) * step  # noqa: E731
    d, f, t = x.shape[1], wg.shape[0], x.shape[0]
    g, u = x @ wg.T, x @ wu.T
    eg, eu = acc(d) * (x.abs() @ wg.abs().T), acc(d) * (x.abs() @ wu.abs().T)
    if act == "silu":
        s = torch.sigmoid(g)
        a, slope = g * s, s * (1 + g * (1 - s))
        most, curve = 1.1, 0.5                            # of |act'|, |act''|
    else:
        cdf, pdf = 0.5 * (1 + torch.erf(g / 2 ** 0.5)), torch.exp(-g * g / 2) / (2 * np.pi) ** 0.5
        a, slope = g * cdf, cdf + g * pdf
        most, curve = 1.13, 0.8
    tiny = 16 * 2.0 ** -23                                # exp, erf and the products around them
    h = a * u
    eh = (1 + half) * (most * eg * u.abs() + (a.abs() + most * eg) * eu) + (half + tiny) * h.abs()
    y = h @ wd.T
    got = {"y": (y, eh @ wd.abs().T + acc(f) * (h.abs() @ wd.abs().T))}
    if dy is None:
        return got
    dh = dy @ wd
    edh = acc(d) * (dy.abs() @ wd.abs())
    dg, du = dh * u * slope, dh * a
    cut = 2.0 ** -16 + tiny
    ep = u.abs() * curve * eg + (slope.abs() + curve * eg) * eu + cut * (u * slope).abs()      # of act'(g) u as it is kept
    ea = most * eg + cut * a.abs()
    edg = (1 + half) * (edh * ((u * slope).abs() + ep) + dh.abs() * ep) + half * dg.abs()
    edu = (1 + half) * (edh * (a.abs() + ea) + dh.abs() * ea) + half * du.abs()
    got["dx"] = dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + acc(2 * f) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    got["dw_gate"] = dg.T @ x, edg.T @ x.abs() + acc(t) * (dg.abs().T @ x.abs())
    got["dw_up"] = du.T @ x, edu.T @ x.abs() + acc(t) * (du.abs().T @ x.abs())
    got["dw_down"] = dy.T @ h, dy.abs().T @ eh + acc(t) * (dy.abs().T @ h.abs())
    return got


# independent bf16 roundings on the way to each result, for the norm of its error: h or dg, du, and its own
ROUNDINGS = 2


def check_ffn(name, got, want, bound):
    """Element by element against the bound (plus the result's own rounding), and, over many elements, in norm: a rounding
    is off by at most 2^-8 relative, 2^-8 / sqrt 3 in the mean square, and independent ones add up in squares; the factor
    sqrt 3 that is left is margin."""
    off = (got.double() - want).abs()
    tol = bound + 2.0 ** -8 * (want.abs() + bound) + 1e-30
    assert bool((off <= tol).all()), f"{name}: worst {float((off / tol).max()):.3g} of its bound"
    if want.numel() >= 4096:
        rel = float(off.norm() / want.norm())
        assert rel <= 2.0 ** -8 * ROUNDINGS ** 0.5, f"{name}: {rel:.3g} in norm"
