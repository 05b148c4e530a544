"""The operators of a looped block between two reads of the update stack, in their plain form and as the framework
offers them: the norms around the block with its gate and residual scale, dropout whose mask is never stored, and the
gated feed-forward product. Each case is one pass of one operator, with or without its gradients.

    norm       u = w n(x),  n(v) = v rsqrt(mean(v^2) + eps)
    residual   b = w n(y) (or y);  out = x + s g m b;  u = w' n(out)      g a gate, s the residual scale, m dropout's factor
    dropout    out = m x
    ffn        y = (act(x Wg^T) * (x Wu^T)) Wd^T

Dropout's factor m: the elements, counted in row-major order, are taken in groups of 8; group i draws eight 16-bit
numbers, the halves (low one first) of the four words of Philox4x32-10 (Salmon et al., 2011) with the counter
(i, offset) and the key seed, 64 bits each. An element is kept where its number is at least t = round(65536 p), and is
then scaled by 65536 / (65536 - t).
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name, op, tokens, d, dtype, grad, f=0, act="", post=False, gate="", learned=False, after=False, p=0.0):
    c = {"op": op, "tokens": tokens, "d": d, "dtype": dtype, "grad": grad}
    if op == "ffn":
        c.update(f=f, act=act)
    if op == "residual":
        c.update(post=post, gate=gate, learned=learned, after=after, p=p)
    if op == "dropout":
        c.update(p=p)
    return {"name": name, **c} if name else c


def listed():
    return [
        # the norm before the block, one decode step of 64 sequences
        _case("norm_decode", "norm", 64, 2048, "bf16", False),
        # the same in training: 8 sequences of 4096 tokens
        _case("norm_train", "norm", 32768, 1024, "bf16", True),
        # the end of a block in a decode step: norm after, gate, residual and the next block's norm
        _case("residual_decode", "residual", 64, 2048, "bf16", False, post=True, gate="channel", after=True),
        # the same in training, with dropout on the branch and a learned residual scale
        _case("residual_train", "residual", 32768, 1024, "bf16", True, post=True, gate="channel", learned=True, after=True, p=0.1),
        # a ragged batch in fp32 with a gate per token, trained without dropout
        _case("residual_ragged", "residual", 4099, 768, "fp32", True, post=True, gate="token", after=True),
        # dropout of a small batch (2 sequences of 256 tokens) in fp32, forward
        _case("dropout_small", "dropout", 512, 768, "fp32", False, p=0.2),
        # dropout in training
        _case("dropout_train", "dropout", 32768, 1024, "bf16", True, p=0.1),
        # the feed-forward block for one sequence's next token, and for a decode step of 64 sequences
        _case("ffn_decode_one", "ffn", 1, 2048, "bf16", False, f=5632, act="silu"),
        _case("ffn_decode", "ffn", 64, 2048, "bf16", False, f=5632, act="silu"),
        # a prompt of odd length
        _case("ffn_prompt", "ffn", 1021, 768, "bf16", False, f=2048, act="gelu"),
        # training: a small batch, and a large ragged one
        _case("ffn_train", "ffn", 8192, 1024, "bf16", True, f=2816, act="silu"),
        _case("ffn_train_large", "ffn", 16411, 1536, "bf16", True, f=4096, act="silu"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "residual", "dropout", "ffn", "ffn"))
    if op == "ffn":
        d, f = 8 * _spread(rng, 32, 256), 8 * _spread(rng, 64, 704)
        grad = rng.random() < 0.5
        most = int((4e12 if grad else 1.2e13) / (18 if grad else 6) / d / f / 2.2)
        tokens = _spread(rng, 16, min(16411, most)) if grad else _spread(rng, 1, min(16411, most))
        return _case("", op, tokens, d, "bf16", grad, f=f, act=rng.choice(("silu", "silu", "gelu")))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    d = 8 * _spread(rng, 8, 256 if dtype == "bf16" else 128)
    tokens = _spread(rng, 1, (1 << 25) // d)
    grad = rng.random() < 0.6
    if op == "norm":
        return _case("", op, tokens, d, dtype, grad)
    if op == "dropout":
        return _case("", op, tokens, d, dtype, grad, p=rng.choice((0.02, 0.1, 0.25, 0.5)))
    return _case("", op, tokens, d, dtype, grad, post=rng.random() < 0.7, gate=rng.choice(("", "channel", "token", "full")),
                 learned=rng.random() < 0.4, after=rng.random() < 0.7, p=rng.choice((0.0, 0.0, 0.1)))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, t, d = _TYPES[case["dtype"]], case["tokens"], case["d"]

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(scale).add_(mean).to(dt)

    s = {"case": dict(case), "x": normal(t, d)}
    op, grad = case["op"], case["grad"]
    if op in ("dropout", "residual"):
        s["rng"] = torch.randint(0, 1 << 40, (2,), device="cuda", generator=gen)
    if op == "norm":
        s["w"] = normal(d, scale=0.1, mean=1.0)
    elif op == "residual":
        s["y"] = normal(t, d, scale=0.5)
        s["w"] = normal(d, scale=0.1, mean=1.0) if case["post"] else None
        shape = {"": None, "channel": (d,), "token": (t, 1), "full": (t, d)}[case["gate"]]
        s["gate"] = None if shape is None else normal(*shape, scale=0.1, mean=0.8)
        s["scale"] = torch.rand(1, device="cuda", generator=gen).add_(0.2) if case["learned"] else 0.25
        s["w_after"] = normal(d, scale=0.1, mean=1.0) if case["after"] else None
    elif op == "ffn":
        f = case["f"]
        s["w_gate"], s["w_up"] = normal(f, d, scale=d ** -0.5), normal(f, d, scale=d ** -0.5)
        s["w_down"] = normal(d, f, scale=f ** -0.5)
    if grad:
        # what comes back is partly along the activations, as gradients of a residual stream are
        s["d_out"] = (torch.randn(t, d, device="cuda", generator=gen) * 0.02 + s["x"].float() * 0.004 +
                      (s["y"].float() * 0.02 if op == "residual" else 0.0)).to(dt)
        if case.get("after"):
            s["d_after"] = normal(t, d, scale=0.02)
        for k in ("x", "y", "w", "gate", "scale", "w_after", "w_gate", "w_up", "w_down"):
            if isinstance(s.get(k), torch.Tensor):
                s[k].requires_grad_()
    return s


def work(case):
    t, d, e = case["tokens"], case["d"], 2 if case["dtype"] == "bf16" else 4
    row, op = t * d * e, case["op"]
    if op == "ffn":
        weights, flops = 3 * d * case["f"] * e, 6 * t * d * case["f"]
        return {"bytes": 2 * row + weights + ((2 * row + weights) if case["grad"] else 0), "flops": flops * (3 if case["grad"] else 1)}
    if op == "residual":
        ins = 2 + (case["gate"] == "full")
        outs = 1 + case["after"]
        return {"bytes": row * (ins + outs + ((outs + ins) if case["grad"] else 0)), "flops": (60 if case["grad"] else 20) * t * d}
    return {"bytes": row * (4 if case["grad"] else 2), "flops": (12 if case["grad"] else 4) * t * d}


# ---------------------------------------------------------------------------------------------------------------
# the plain form: 32-bit arithmetic, one rounding at the end
# ---------------------------------------------------------------------------------------------------------------
def _factor(p, rng, shape):
    """Dropout's factor, fp32."""
    t = int(p * 65536 + 0.5)
    n = math.prod(shape)
    low = 0xFFFFFFFF
    i = torch.arange((n + 7) // 8, device=rng.device)
    c0, c1, c2, c3 = i & low, i >> 32, rng[1] & low, (rng[1] >> 32) & low
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # low 64 bits of the products; what follows masks the sign
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), -1)
    halves = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)[:n].reshape(shape)
    return (halves >= t).float() * (65536.0 / (65536 - t))


def _scale_of(v):
    return torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)


def _norm_back(dv, vh, r):
    """The gradient of n(v) = vh for the gradient dv."""
    return r * (dv - vh * (dv * vh).mean(-1, keepdim=True))


def _plain_norm(s):
    x, w, dt = s["x"].float(), s["w"].float(), s["x"].dtype
    r = _scale_of(x)
    xh = x * r
    u = (w * xh).to(dt)
    if not s["case"]["grad"]:
        return {"u": u}
    g = s["d_out"].float()
    return {"u": u, "dx": _norm_back(w * g, xh, r).to(dt), "dw": (g * xh).sum(0).to(s["w"].dtype)}


def _plain_residual(s):
    case, dt = s["case"], s["x"].dtype
    x, y = s["x"].float(), s["y"].float()
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    scale = s["scale"].float() if isinstance(s["scale"], torch.Tensor) else s["scale"]
    m = _factor(case["p"], s["rng"], x.shape) if case["p"] else 1.0
    if case["post"]:
        w, ry = s["w"].float(), _scale_of(y)
        yh = y * ry
        b = w * yh
    else:
        b = y
    out = x + scale * (gate * m * b)
    got = {"out": out.to(dt)}
    if case["after"]:
        wa, ro = s["w_after"].float(), _scale_of(out)
        oh = out * ro
        got["u"] = (wa * oh).to(dt)
    if not case["grad"]:
        return got
    dx = s["d_out"].float()
    if case["after"]:
        du = s["d_after"].float()
        dx = dx + _norm_back(wa * du, oh, ro)
        got["dw_after"] = (du * oh).sum(0).to(s["w_after"].dtype)
    got["dx"] = dx.to(dt)
    along = dx * m * b                                   # the gradient of scale * gate, element by element
    if isinstance(s["scale"], torch.Tensor):
        got["dscale"] = (gate * along).double().sum().reshape(1).to(s["scale"].dtype)
    if case["gate"]:
        dg = scale * along
        dg = dg.sum(0) if case["gate"] == "channel" else dg.sum(-1, keepdim=True) if case["gate"] == "token" else dg
        got["dgate"] = dg.to(s["gate"].dtype)
    db = scale * (gate * m * dx)
    if case["post"]:
        got["dw"] = (db * yh).sum(0).to(s["w"].dtype)
        db = _norm_back(w * db, yh, ry)
    got["dy"] = db.to(dt)
    return got


def _plain_dropout(s):
    x, dt = s["x"].float(), s["x"].dtype
    m = _factor(s["case"]["p"], s["rng"], x.shape)
    got = {"out": (m * x).to(dt)}
    if s["case"]["grad"]:
        got["dx"] = (m * s["d_out"].float()).to(dt)
    return got


def _plain_ffn(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[k].detach().float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.T, x @ wu.T
    if case["act"] == "silu":
        sig = 1 / (1 + torch.exp(-g))
        a = g * sig
    else:
        cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        a = g * cdf
    h = a * u
    got = {"y": (h @ wd.T).to(dt)}
    if not case["grad"]:
        return got
    dy = s["d_out"].float()
    dh = dy @ wd
    slope = sig * (1 + g * (1 - sig)) if case["act"] == "silu" else cdf + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    dg, du = dh * u * slope, dh * a
    got.update(dx=(dg @ wg + du @ wu).to(dt), dw_gate=(dg.T @ x).to(dt), dw_up=(du.T @ x).to(dt), dw_down=(dy.T @ h).to(dt))
    return got


_PLAIN = {"norm": _plain_norm, "residual": _plain_residual, "dropout": _plain_dropout, "ffn": _plain_ffn}


# ---------------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------------
def _own_forward(s):
    from loopback_b200 import block
    case = s["case"]
    if case["op"] == "norm":
        return {"u": block.block_norm(s["x"], s["w"], eps=EPS)}
    if case["op"] == "dropout":
        return {"out": block.dropout(s["x"], case["p"], s["rng"])}
    if case["op"] == "ffn":
        return {"y": block.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], act=case["act"])}
    got = block.block_residual(s["x"], s["y"], s["w"], gate=s["gate"], scale=s["scale"], next_weight=s["w_after"], eps=EPS,
                               p=case["p"], rng=s["rng"] if case["p"] else None)
    return {"out": got[0], "u": got[1]} if case["after"] else {"out": got}


_GRADS = {"x": "dx", "y": "dy", "w": "dw", "gate": "dgate", "scale": "dscale", "w_after": "dw_after", "w_gate": "dw_gate",
          "w_up": "dw_up", "w_down": "dw_down"}


def _own(s):
    if not s["case"]["grad"]:
        with torch.no_grad():
            return _own_forward(s)
    got = _own_forward(s)
    wanted = [k for k in _GRADS if isinstance(s.get(k), torch.Tensor)]
    up = [s["d_out"], s["d_after"]] if s["case"].get("after") else [s["d_out"]]
    grads = torch.autograd.grad(list(got.values()), [s[k] for k in wanted], up)
    got.update({_GRADS[k]: g for k, g in zip(wanted, grads)})
    return {k: v.detach() for k, v in got.items()}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------
# the same from the definitions in 64 bits, gradients by differentiating the definition
# ---------------------------------------------------------------------------------------------------------------
def _exact_factor(p, rng, n):
    t = round(p * 65536)
    seed, offset = (int(v) for v in rng.cpu())
    i = np.arange((n + 7) // 8, dtype=np.uint64)
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [i & low, i >> shift, np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    for r in range(10):
        k0, k1 = ((seed & 0xFFFFFFFF) + r * 0x9E3779B9) % 2 ** 32, ((seed >> 32) + r * 0xBB67AE85) % 2 ** 32
        m0, m1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(m1 >> shift) ^ c[1] ^ np.uint64(k0), m1 & low, (m0 >> shift) ^ c[3] ^ np.uint64(k1), m0 & low]
    words = np.stack([v.astype(np.uint32) for v in c], -1)
    halves = words.view("<u2").reshape(-1)[:n]
    return torch.from_numpy(np.where(halves >= t, 65536.0 / (65536.0 - t), 0.0)).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    names = [k for k in _GRADS if isinstance(s.get(k), torch.Tensor)]
    v = {k: s[k].detach().double().requires_grad_(case["grad"]) for k in names}

    def unit(a):
        return a / torch.sqrt((a * a).sum(-1, keepdim=True) / a.shape[-1] + EPS)

    with torch.set_grad_enabled(case["grad"]):
        x = v["x"]
        if case["op"] == "norm":
            got = {"u": unit(x) * v["w"]}
        elif case["op"] == "dropout":
            got = {"out": x * _exact_factor(case["p"], s["rng"], x.numel()).view_as(x)}
        elif case["op"] == "ffn":
            act = torch.nn.functional.silu if case["act"] == "silu" else torch.nn.functional.gelu
            h = act(torch.nn.functional.linear(x, v["w_gate"])) * torch.nn.functional.linear(x, v["w_up"])
            got = {"y": torch.nn.functional.linear(h, v["w_down"])}
        else:
            b = unit(v["y"]) * v["w"] if case["post"] else v["y"]
            if case["p"]:
                b = b * _exact_factor(case["p"], s["rng"], x.numel()).view_as(x)
            if case["gate"]:
                b = b * v["gate"]
            out = x + b * v.get("scale", s["scale"])
            got = {"out": out, "u": unit(out) * v["w_after"]} if case["after"] else {"out": out}
        if case["grad"]:
            up = [s["d_out"].double()] + ([s["d_after"].double()] if case.get("after") else [])
            grads = torch.autograd.grad(list(got.values()), [v[k] for k in names], up)
            got.update({_GRADS[k]: g for k, g in zip(names, grads)})
    return {k: a.detach() for k, a in got.items()}
