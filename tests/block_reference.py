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
