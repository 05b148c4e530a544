"""The operators around a block (loopback_b200.block) against their definitions in 64 bits.

Tolerances: a result is rounded once to its type (half a step: 2^-8 for bf16, 2^-24 for fp32, relative to the value). Before
that come fp32 operations, each off by 2^-24 relative to what it adds up: a row sum is at most 32 fragment elements, 5 shuffle
steps and 8 warps deep (45 additions; the root halves what it makes of it), two such statistics and about ten products enter a
gradient: 64 steps relative to the magnitudes cover them. A parameter's gradient adds rows in fp32 inside a CTA (at most
ceil(rows / CTAs) + 8 of them) before the fp64 sum: as many steps more."""
import numpy as np
import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu
EPS = ref.EPS
TYPES = {"bf16": (torch.bfloat16, torch.bfloat16), "bf16_w32": (torch.bfloat16, torch.float32), "fp32": (torch.float32, torch.float32)}


def _rows(gen, t, d, dtype, scale=1.0):
    return (torch.randn(t, d, device="cuda", generator=gen) * scale).to(dtype)


def _weight(gen, d, dtype):
    return (1 + 0.2 * torch.randn(d, device="cuda", generator=gen)).to(dtype)


def _steps(t):
    return 64 + 8 + t // 148 + 1


SHAPES = [(1, 64), (3, 8), (2, 72), (64, 768), (37, 1000), (300, 1024), (5, 2048), (129, 4096), (2500, 1536), (40011, 64)]


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("t,d", SHAPES + [(7, 8192)])
def test_norm(types, t, d):
    from loopback_b200 import block
    dt, wt = TYPES[types]
    if d > 4096 and dt == torch.float32:
        d = 4096
    gen = torch.Generator(device="cuda").manual_seed(t * 10007 + d)
    x, w, du = _rows(gen, t, d, dt).requires_grad_(), _weight(gen, d, wt).requires_grad_(), _rows(gen, t, d, dt)
    want = ref.norm(x.detach().double(), w.detach().double(), du.double())
    u = block.block_norm(x, w, EPS)
    dx, dw = torch.autograd.grad(u, (x, w), du)
    with torch.no_grad():
        assert torch.equal(block.block_norm(x, w, EPS), u)
    assert dw.dtype == wt
    ref.check("u", u, *want["u"])
    ref.check("dx", dx, *want["dx"])
    ref.check("dw", dw, *want["dw"], steps=_steps(t))


def _residual_case(types, t, d, post, kind, learned, after, p, seed):
    dt, wt = TYPES[types]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"x": _rows(gen, t, d, dt), "y": _rows(gen, t, d, dt, 0.5), "w": _weight(gen, d, wt) if post else None,
         "w_next": _weight(gen, d, wt) if after else None, "dout": _rows(gen, t, d, dt), "du": _rows(gen, t, d, dt) if after else None}
    shape = {"": None, "channel": (d,), "token": (t, 1), "full": (t, d)}[kind]
    s["gate"] = None if shape is None else (0.8 + 0.3 * torch.randn(*shape, device="cuda", generator=gen)).to(wt if kind == "channel" else dt)
    s["scale"] = torch.tensor([0.37], device="cuda") if learned else 0.37
    s["rng"] = torch.tensor([seed * 1234567891011 + 5, (1 << 33) + seed], device="cuda")
    return s


def _run_residual(s, p):
    from loopback_b200 import block
    names = [k for k in ("x", "y", "w", "gate", "scale", "w_next") if isinstance(s[k], torch.Tensor)]
    for k in names:
        s[k].requires_grad_()
    got = block.block_residual(s["x"], s["y"], s["w"], gate=s["gate"], scale=s["scale"], next_weight=s["w_next"], eps=EPS, p=p,
                               rng=s["rng"] if p else None)
    outs = list(got) if s["w_next"] is not None else [got]
    ups = [s["dout"], s["du"]][:len(outs)]
    res = dict(zip(("out", "u"), outs))
    res.update({"d" + k: g for k, g in zip(names, torch.autograd.grad(outs, [s[k] for k in names], ups))})
    return res


def _want_residual(s, kind, p, t, d):
    f = lambda v: None if v is None else v.detach().double()  # noqa: E731
    m = ref.factor(p, int(s["rng"][0]), int(s["rng"][1]), 0, t * d).view(t, d).cuda() if p else 1.0
    scale = float(s["scale"].detach().double()) if isinstance(s["scale"], torch.Tensor) else s["scale"]
    return ref.residual(f(s["x"]), f(s["y"]), f(s["w"]), f(s["gate"]), kind, scale, f(s["w_next"]), m, f(s["dout"]), f(s["du"]), True)


@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("kind", ["", "channel", "token", "full"])
@pytest.mark.parametrize("post,after,learned", [(True, True, True), (True, False, False), (False, True, False), (False, False, True)])
@pytest.mark.parametrize("types", list(TYPES))
def test_residual_forms(types, post, after, learned, kind, p):
    t, d = 61, 712
    s = _residual_case(types, t, d, post, kind, learned, after, p, 3)
    want = _want_residual(s, kind, p, t, d)
    got = _run_residual(s, p)
    for k, v in got.items():
        v = v.reshape(want[k][0].shape)
        ref.check(k, v, *want[k], steps=_steps(t))


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("t,d,kind", [(*s, "channel") for s in SHAPES] + [(7, 8192, "channel"), (5, 8192, "full"), (700, 1024, "full")])
def test_residual_sizes(types, t, d, kind):
    if types == "fp32" and d > 4096:
        d = 4096
    s = _residual_case(types, t, d, True, kind, True, True, 0.1, t + d)
    want = _want_residual(s, kind, 0.1, t, d)
    got = _run_residual(s, 0.1)
    again = _run_residual(s, 0.1)
    for k, v in got.items():
        ref.check(k, v, *want[k], steps=_steps(t))
        assert torch.equal(v, again[k]), f"{k} differs from run to run"


@pytest.mark.parametrize("types,d,p", [("fp32", 256, 0.0), ("bf16", 520, 0.25), ("bf16_w32", 2048, 0.0)])
def test_residual_single_upstream_and_frozen_parameters(types, d, p):
    """Only one of the two results is used, and parameters without gradients get none."""
    from loopback_b200 import block
    t = 33
    s = _residual_case(types, t, d, True, "channel", True, True, p, 9)
    pair = [int(v) for v in s["rng"]]
    m = ref.factor(p, *pair, 0, t * d).view(t, d).cuda() if p else 1.0
    for which in (0, 1):
        x, y = s["x"].clone().requires_grad_(), s["y"].clone().requires_grad_()
        w, wn, gate = (s[k].clone().requires_grad_() for k in ("w", "w_next", "gate"))
        got = block.block_residual(x, y, w, gate=gate, scale=0.37, next_weight=wn, eps=EPS, p=p, rng=pair)
        up = s["dout"]
        grads = torch.autograd.grad(got[which], (x, y, w, gate, wn), up, allow_unused=True)
        want = ref.residual(*(v.detach().double() for v in (x, y, w, gate)), "channel", 0.37, wn.detach().double(), m,
                            up.double() if which == 0 else None, up.double() if which else None, True)
        for k, g in zip(("dx", "dy", "dw", "dgate"), grads):
            ref.check(k, g, *want[k])
        if which:
            ref.check("dw_next", grads[4], *want["dw_next"])
        else:
            assert grads[4] is None or not grads[4].any()
    x = s["x"].clone().requires_grad_()
    out, u = block.block_residual(x, s["y"], s["w"], gate=s["gate"], next_weight=s["w_next"])
    (out + u).sum().backward()                       # expanded (stride 0) gradients
    assert x.grad is not None and s["w"].grad is None


def test_gradients_against_differences():
    """fp32, central differences of the 64-bit definition along random directions: independent of the closed forms above."""
    t, d = 6, 64
    s = _residual_case("fp32", t, d, True, "full", True, True, 0.25, 4)
    got = _run_residual(s, 0.25)
    m = ref.factor(0.25, int(s["rng"][0]), int(s["rng"][1]), 0, t * d).view(t, d).cuda()
    v = {k: s[k].detach().double() for k in ("x", "y", "w", "gate", "scale", "w_next")}

    def loss(a):
        r = ref.residual(a["x"], a["y"], a["w"], a["gate"], "full", a["scale"], a["w_next"], m)
        return float((r["out"][0] * s["dout"].double()).sum() + (r["u"][0] * s["du"].double()).sum())

    gen = torch.Generator(device="cuda").manual_seed(0)
    for k in v:
        z = torch.randn(v[k].shape, device="cuda", generator=gen).double()
        h = 1e-5
        diff = (loss({**v, k: v[k] + h * z}) - loss({**v, k: v[k] - h * z})) / (2 * h)
        along = (got["d" + k].double() * z)
        # the difference quotient is off by O(h^2) = 1e-10 of the third derivative, the gradient by 64 fp32 steps
        assert abs(diff - float(along.sum())) <= 1e-5 * float(along.abs().sum()) + 1e-6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 3, 8, 9, 12, 1000, 65536, 300007])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999])
def test_dropout(dtype, n, p):
    from loopback_b200 import block
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, device="cuda", generator=gen).to(dtype).requires_grad_()
    g = torch.randn(n, device="cuda", generator=gen).to(dtype)
    seed, offset = (1 << 63) + 12345, (1 << 40) + 7
    m = ref.factor(p, seed, offset, 0, n).cuda()
    out = block.dropout(x, p, (seed, offset))
    (dx,) = torch.autograd.grad(out, x, g)
    # the factor is rounded to fp32 and multiplied in fp32: two steps of 2^-24, then the type's own rounding
    ref.check("out", out, x.detach().double() * m, (x.detach().double() * m).abs(), steps=2)
    ref.check("dx", dx, g.double() * m, (g.double() * m).abs(), steps=2)
    assert torch.equal(out == 0, (m == 0) | (x == 0))
    if p and n > 1000:
        kept = float((m > 0).double().mean())
        assert abs(kept - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5


def test_dropout_clears_what_it_drops():
    """A dropped infinity or NaN leaves 0, not NaN; a kept one stays."""
    from loopback_b200 import block
    m = ref.factor(0.5, 1, 2, 0, 4096).cuda()
    for bad in (float("inf"), float("nan")):
        out = block.dropout(torch.full((4096,), bad, device="cuda"), 0.5, (1, 2))
        assert torch.equal(torch.isfinite(out), m == 0) and not out[m == 0].any()
    x, y = torch.ones(4, 1024, device="cuda"), torch.full((4, 1024), float("inf"), device="cuda")
    out = block.block_residual(x, y, p=0.5, rng=(1, 2))
    assert torch.equal(out == 1, (m == 0).view(4, 1024))


@pytest.mark.parametrize("after", [False, True])
@pytest.mark.parametrize("kind", ["", "channel", "token", "full"])
@pytest.mark.parametrize("types", list(TYPES))
def test_dropped_values_reach_no_gradient(types, kind, after):
    """Without a norm after the block, what y (and a gate per element) holds where it is dropped changes no bit of any result."""
    t, d, p = 37, 264, 0.4
    finite = _residual_case(types, t, d, False, kind, True, after, p, 6)
    dropped = (ref.factor(p, int(finite["rng"][0]), int(finite["rng"][1]), 0, t * d) == 0).view(t, d).cuda()
    clone = lambda v: v.detach().clone() if isinstance(v, torch.Tensor) else v  # noqa: E731
    for bad in (float("inf"), float("nan")):
        s = {k: clone(v) for k, v in finite.items()}
        s["y"][dropped] = bad
        if kind == "full":
            s["gate"][dropped] = bad
        want, got = _run_residual({k: clone(v) for k, v in finite.items()}, p), _run_residual(s, p)
        for k, v in got.items():
            assert torch.isfinite(v).all(), k
            assert torch.equal(v, want[k]), k


@pytest.mark.parametrize("types", list(TYPES))
def test_infinite_branch_without_a_norm_has_a_finite_gradient(types):
    """out = x + s y: dy = s dout whatever y holds."""
    s = _residual_case(types, 9, 136, False, "", False, False, 0.0, 2)
    want = _run_residual(dict(s), 0.0)["dy"]
    y = s["y"].detach().clone()
    y[3, 5], y[8, 135] = float("inf"), float("nan")
    assert torch.equal(_run_residual({**s, "y": y}, 0.0)["dy"], want)


def test_dropout_past_32_bits_of_elements():
    from loopback_b200 import block
    n = (1 << 32) + 1024 + 5
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    out = block.dropout(x, 0.5, (3, 4))
    del x
    for at in (0, (1 << 31) - 64, (1 << 32) - 512, n - 1029):
        m = ref.factor(0.5, 3, 4, at, min(1029, n - at)).cuda()
        assert torch.equal(out[at:at + len(m)].double(), m)


def test_rows_past_32_bits_of_elements():
    """Rows are independent: those behind 2^32 elements have the bits of a small batch of the same rows."""
    from loopback_b200 import block
    d, few = 1024, 4096
    t = (1 << 32) // d + 5
    gen = torch.Generator(device="cuda").manual_seed(8)
    xs, ys = (_rows(gen, few, d, torch.bfloat16) for _ in range(2))
    w, wn = (_weight(gen, d, torch.bfloat16) for _ in range(2))
    up = torch.ones(t, d, device="cuda", dtype=torch.bfloat16)

    def run(x, y):
        x.requires_grad_(), y.requires_grad_()
        out, u = block.block_residual(x, y, w, scale=0.5, next_weight=wn)
        return [out.detach(), u.detach(), *torch.autograd.grad((out, u), (x, y), (up[:len(x)],) * 2)]

    want = run(xs, ys)
    got = run(*(torch.cat((v.detach().repeat(t // few, 1), v.detach()[:t % few])) for v in (xs, ys)))
    for a, b in zip(want, got):
        assert torch.equal(b[:few], a) and torch.equal(b[-(t % few) - few:-(t % few)], a) and torch.equal(b[-(t % few):], a[:t % few])


def test_dropout_same_mask_in_the_residual():
    """block_residual's dropout is dropout() of the branch: without a norm and with x = 0 the two give the same bits."""
    from loopback_b200 import block
    y = torch.randn(50, 520, device="cuda").bfloat16()
    a = block.dropout(y, 0.2, (77, 8))
    b = block.block_residual(torch.zeros_like(y), y, p=0.2, rng=(77, 8))
    assert torch.equal(a, b)


def test_rng_tensor_is_read_by_the_kernel_and_remembered():
    """The pair may move on between a forward and its backward; a replayed graph draws from the pair as it then is."""
    from loopback_b200 import block
    x = torch.randn(256, 512, device="cuda")
    rng = torch.tensor([11, 5], device="cuda")
    xs = x.clone().requires_grad_()
    out = block.dropout(xs, 0.3, rng)
    r = block.block_residual(torch.zeros_like(x), (ys := x.clone().requires_grad_()), p=0.3, rng=rng)
    rng[1] += 1
    (dx,) = torch.autograd.grad(out, xs, torch.ones_like(x))
    (dy,) = torch.autograd.grad(r, ys, torch.ones_like(x))
    want = ref.factor(0.3, 11, 5, 0, x.numel()).view_as(x).cuda().float()
    assert torch.equal(dx, want) and torch.equal(dy, want)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block.dropout(x, 0.3, rng)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    xg = x.clone().requires_grad_()
    with torch.cuda.graph(graph):
        got = block.dropout(xg, 0.3, rng)
        (dg,) = torch.autograd.grad(got, xg, torch.ones_like(x))
        rng[1] += 1
    for offset in (100, 101):
        rng[1] = offset
        graph.replay()
        torch.cuda.synchronize()
        want = block.dropout(x, 0.3, (11, offset))
        assert torch.equal(got, want) and torch.equal(dg != 0, want != 0) and int(rng[1]) == offset + 1


def test_strides_other_shapes_and_empty_batches():
    from loopback_b200 import block
    gen = torch.Generator(device="cuda").manual_seed(0)
    base = torch.randn(4, 6, 2, 96, device="cuda", generator=gen)
    x, y = base[:, ::2, 0].transpose(0, 1), base[:, 1::2, 1].transpose(0, 1)
    assert not x.is_contiguous()
    w = torch.randn(96, device="cuda", generator=gen)
    gate = torch.randn(3, 4, 1, device="cuda", generator=gen)
    out, u = block.block_residual(x, y, w, gate=gate, next_weight=w[torch.randperm(96, device="cuda")])
    assert out.shape == u.shape == x.shape
    want = ref.residual(x.double().reshape(12, 96), y.double().reshape(12, 96), w.double(), gate.double().reshape(12, 1), "token")
    ref.check("out", out.reshape(12, 96), *want["out"])
    odd = torch.randn(12 * 96 + 1, device="cuda", generator=gen)[1:].view(12, 96).requires_grad_()     # not on 16 bytes
    up = torch.randn(12 * 96 + 1, device="cuda", generator=gen)[1:].view(12, 96)
    ow = torch.randn(97, device="cuda", generator=gen)[1:].requires_grad_()
    u = block.block_norm(odd, ow, EPS)
    dx, dw = torch.autograd.grad(u, (odd, ow), up)
    want = ref.norm(odd.detach().double(), ow.detach().double(), up.double())
    for k, v in (("u", u.detach()), ("dx", dx), ("dw", dw)):
        ref.check(k, v, *want[k])
    (dd,) = torch.autograd.grad(block.dropout(odd, 0.5, (1, 2)), odd, up)
    assert torch.equal(dd, block.dropout(up, 0.5, (1, 2)))
    e = torch.zeros(0, 5, 96, device="cuda").requires_grad_()
    we, sc = w.clone().requires_grad_(), torch.tensor(0.5, device="cuda", requires_grad=True)
    out, u = block.block_residual(e, e, we, gate=we, scale=sc, next_weight=we)
    (out.sum() + u.sum() + block.block_norm(e, we).sum() + block.dropout(e, 0.5, (1, 2)).sum()).backward()
    assert e.grad.shape == e.shape and not we.grad.any() and float(sc.grad) == 0


def test_on_another_stream():
    from loopback_b200 import block
    t, d = 2048, 1024
    s = _residual_case("bf16", t, d, True, "channel", True, True, 0.1, 1)
    want = _run_residual(s, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        x = s["x"].detach().clone()
        s2 = {**{k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in s.items()}, "x": x}
        got = _run_residual(s2, 0.1)
    side.synchronize()
    for k in want:
        assert torch.equal(want[k], got[k]), k


def test_zero_rows_and_extremes():
    """A row of zeros has the scale eps^-1/2 and stays zero; rows of large bf16 values keep the definition's value."""
    from loopback_b200 import block
    x = torch.zeros(3, 64, device="cuda")
    x[1] = 1e15
    x[2, 5] = 1e-30
    w = torch.ones(64, device="cuda")
    u = block.block_norm(x, w, EPS)
    want = ref.norm(x.double(), w.double())["u"]
    ref.check("u", u, *want)


def test_refusals():
    from loopback_b200 import block
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    for call in (lambda: block.block_norm(x.half(), w), lambda: block.block_norm(x, w[:32]), lambda: block.block_norm(x[:, :3], w[:3]),
                 lambda: block.block_norm(x, w.cpu()), lambda: block.block_norm(torch.ones((), device="cuda"), w),
                 lambda: block.block_norm(torch.randn(2, 16384, device="cuda"), torch.ones(16384, device="cuda")),
                 lambda: block.block_residual(x, x[:2]), lambda: block.block_residual(x, x.bfloat16()),
                 lambda: block.block_residual(x, x, gate=torch.ones(2, 64, device="cuda")),
                 lambda: block.block_residual(x, x, gate=torch.ones(4, 1, device="cuda", dtype=torch.float64)),
                 lambda: block.block_residual(x, x, scale=torch.ones(2, device="cuda")),
                 lambda: block.block_residual(x, x, scale=torch.ones(1)),
                 lambda: block.dropout(x, 0.5, torch.ones(2, device="cuda")), lambda: block.dropout(x, 0.5, torch.ones(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: block.dropout(x, 1.0, (1, 2)), lambda: block.dropout(x, -0.1, (1, 2)), lambda: block.dropout(x, 0.5, None),
                 lambda: block.dropout(x, float("nan"), (1, 2)), lambda: block.block_residual(x, x, p=0.5)):
        with pytest.raises(ValueError):
            call()


def test_second_derivatives_raise():
    """The operators are differentiable once: under create_graph a second derivative raises instead of being taken for zero."""
    from loopback_b200 import block
    x = torch.randn(4, 64, device="cuda").requires_grad_()
    w = torch.ones(64, device="cuda").requires_grad_()
    for f in (lambda: block.block_norm(x, w), lambda: block.block_residual(x, x, w, next_weight=w)[1], lambda: block.dropout(x, 0.5, (1, 2))):
        (g,) = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.sum().backward()
