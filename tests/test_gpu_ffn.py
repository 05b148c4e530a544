"""The gated feed-forward block (loopback_b200.block.gated_ffn) against its definition in 64 bits. The bounds are worked out
in block_reference.ffn from the roundings the operator documents."""
import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu


def _inputs(t, d, f, seed, grad=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=gen) * scale).bfloat16()  # noqa: E731
    x, wg, wu, wd = rnd(t, d), rnd(f, d, scale=1.3 * d ** -0.5), rnd(f, d, scale=d ** -0.5), rnd(d, f, scale=f ** -0.5)
    dy = rnd(t, d)
    return [v.requires_grad_(grad) for v in (x, wg, wu, wd)], dy


def _check(t, d, f, act="silu", seed=0, grad=True):
    from loopback_b200 import block
    from loopback_b200._lib import device_error
    (x, wg, wu, wd), dy = _inputs(t, d, f, seed, grad)
    want = ref.ffn(*(v.detach().double() for v in (x, wg, wu, wd)), act, dy.double() if grad else None)
    y = block.gated_ffn(x, wg, wu, wd, act=act)
    got = {"y": y}
    if grad:
        got.update(zip(("dx", "dw_gate", "dw_up", "dw_down"), torch.autograd.grad(y, (x, wg, wu, wd), dy)))
    torch.cuda.synchronize()
    assert device_error() == 0, "a kernel gave up a bounded wait"
    for k, v in got.items():
        ref.check_ffn(k, v.detach(), *want[k])
    return got


SIZES = [(128, 64, 128), (128, 128, 256), (256, 256, 512), (1, 8, 8), (1, 64, 64), (7, 72, 120), (64, 512, 264), (127, 136, 1000),
         (129, 768, 2048), (255, 1000, 136), (257, 264, 520), (300, 8, 1032), (300, 1032, 8), (1000, 512, 1408)]


@pytest.mark.parametrize("tile", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("t,d,f", SIZES)
def test_training_sizes(t, d, f, tile):
    import loopback_b200._lib as L
    try:
        L.set_option("ffn_tile", tile)
        _check(t, d, f, seed=t + d + f)
    finally:
        L.reset_options()


@pytest.mark.parametrize("tile,t", [(1, 1400), (2, 1400), (3, 1400), (5, 700)])
@pytest.mark.parametrize("splits", [1, 2, 3, 5, 6, 7, 8])
def test_splits_along_k(tile, t, splits):
    import loopback_b200._lib as L
    try:
        L.set_option("ffn_tile", tile)
        L.set_option("ffn_splits", splits)
        _check(t, 264, 1288, seed=splits)
    finally:
        L.reset_options()


@pytest.mark.parametrize("t,d,f", [(16500, 520, 72), (300, 1544, 4096), (20011, 264, 776)])
def test_several_wide_tiles_per_pair(t, d, f):
    """256 x 512 tiles have one accumulator: more tiles than pairs of CTAs, with a last one of one half or less."""
    import loopback_b200._lib as L
    try:
        L.set_option("ffn_tile", 4)
        _check(t, d, f, seed=t)
    finally:
        L.reset_options()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("t,d,f", [(333, 768, 2048), (4099, 1024, 2816), (16, 2048, 5632)])
def test_chosen_shapes(t, d, f, act):
    _check(t, d, f, act)


@pytest.mark.parametrize("t,d,f", [(1300, 264, 1288), (3000, 1032, 520), (700, 1024, 2816)])
def test_gradients_of_both_weights_and_of_one(t, d, f):
    """Both weight gradients at once (one launch where that is faster) and each alone give the same values up to the order of
    a sum split along the rows."""
    from loopback_b200 import block
    (x, wg, wu, wd), dy = _inputs(t, d, f, 11)
    want = ref.ffn(*(v.detach().double() for v in (x, wg, wu, wd)), "silu", dy.double())
    for need in ((1, 2, 3), (1, 2), (2,), (3,)):
        ins = [v.detach().requires_grad_(i in need) for i, v in enumerate((x, wg, wu, wd))]
        got = torch.autograd.grad(block.gated_ffn(*ins), [ins[i] for i in need], dy)
        for i, g in zip(need, got):
            name = ("dx", "dw_gate", "dw_up", "dw_down")[i]
            ref.check_ffn(name, g, *want[name])


def test_same_bits_every_run():
    a, b = _check(2500, 520, 1416), _check(2500, 520, 1416)
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 33, 64, 65, 100, 128, 129, 200])
@pytest.mark.parametrize("d,f", [(8, 8), (64, 128), (136, 40), (768, 2048), (1000, 1416), (2048, 5632), (4096, 1024)])
def test_few_rows_without_gradients(t, d, f):
    from loopback_b200 import block
    (x, wg, wu, wd), _ = _inputs(t, d, f, t + d, grad=False)
    want = ref.ffn(*(v.double() for v in (x, wg, wu, wd)), "silu")
    y = block.gated_ffn(x, wg, wu, wd)
    ref.check_ffn("y", y, *want["y"])
    with torch.no_grad():
        assert torch.equal(block.gated_ffn(x, wg, wu, wd), y)
    if t > 1:                                             # a batch padded with rows that hold no number
        x[-1] = float("nan")
        assert torch.equal(block.gated_ffn(x, wg, wu, wd)[:-1], y[:-1])


def test_rows_behind_the_last_stay():
    """Written rows end with the batch, and the workspace's old contents (here NaN) reach no result."""
    import loopback_b200._lib as L
    for t in (3, 70, 200):
        (x, wg, wu, wd), _ = _inputs(t, 136, 264, 5, grad=False)
        y = torch.full((t + 40, 136), 7.0, device="cuda", dtype=torch.bfloat16)
        h = torch.full((t + 40, 264), 7.0, device="cuda", dtype=torch.bfloat16)
        kept = torch.empty(L.lib().lb_ffn_kept_bytes(t, 264), device="cuda", dtype=torch.uint8)
        n = L.lib().lb_ffn_workspace_bytes(t, 136, 264, 0)
        ws = torch.full((n // 4 + 1,), float("nan"), device="cuda")
        L.check(L.lib().lb_ffn_fwd(L.ptr(x), L.ptr(wg), L.ptr(wu), L.ptr(wd), L.ptr(y), L.ptr(h), L.ptr(kept), L.ptr(ws), n, t, 136, 264, 0,
                                   L.LB_DTYPE_BF16, L.stream_ptr()), "gated ffn")
        ref.check_ffn("y", y[:t], *ref.ffn(*(v.double() for v in (x, wg, wu, wd)), "silu")["y"])
        assert bool((y[t:] == 7).all()) and bool((h[t:] == 7).all())
        y.fill_(7.0)
        n = L.lib().lb_ffn_workspace_bytes(t, 136, 264, 2)
        ws = torch.full((n // 4 + 1,), float("nan"), device="cuda")
        L.check(L.lib().lb_ffn_fwd(L.ptr(x), L.ptr(wg), L.ptr(wu), L.ptr(wd), L.ptr(y), None, None, L.ptr(ws), n, t, 136, 264, 0,
                                   L.LB_DTYPE_BF16, L.stream_ptr()), "gated ffn")
        ref.check_ffn("y", y[:t], *ref.ffn(*(v.double() for v in (x, wg, wu, wd)), "silu")["y"])
        assert bool((y[t:] == 7).all())


def test_special_values_stay_in_their_rows():
    """An infinity or a NaN in one row reaches that row of y and of dx, no other."""
    from loopback_b200 import block
    (x, wg, wu, wd), dy = _inputs(200, 136, 264, 6)
    clean = block.gated_ffn(x, wg, wu, wd)
    (cdx,) = torch.autograd.grad(clean, x, dy)
    xb = x.detach().clone()
    xb[17, 3], xb[130, 5] = float("nan"), float("inf")
    xb.requires_grad_()
    y = block.gated_ffn(xb, wg, wu, wd)
    (dx,) = torch.autograd.grad(y, xb, dy)
    keep = torch.ones(200, dtype=torch.bool, device="cuda")
    keep[17] = keep[130] = False
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], cdx[keep])
    assert not torch.isfinite(y[17]).any() and not torch.isfinite(y[130]).all()


def test_large_activations():
    """g far from zero on both sides: act saturates without overflow."""
    from loopback_b200 import block
    for act in ("silu", "gelu"):
        x = torch.zeros(130, 64, device="cuda", dtype=torch.bfloat16)
        x[:, 0] = torch.linspace(-300, 300, 130, device="cuda").bfloat16()
        w = torch.zeros(128, 64, device="cuda", dtype=torch.bfloat16)
        w[:, 0] = 1
        wd = torch.eye(128, device="cuda", dtype=torch.bfloat16)[:64].contiguous()
        ins = [v.requires_grad_() for v in (x, w, torch.ones_like(w), wd)]
        y = block.gated_ffn(*ins, act=act)
        dy = torch.ones_like(y)
        grads = torch.autograd.grad(y, ins, dy)
        want = ref.ffn(*(v.detach().double() for v in ins), act, dy.double())
        ref.check_ffn("y", y.detach(), *want["y"])
        for k, g in zip(("dx", "dw_gate", "dw_up", "dw_down"), grads):
            off = (g.double() - want[k][0]).abs()
            assert bool((off <= want[k][1] + 2.0 ** -8 * (want[k][0].abs() + want[k][1]) + 1e-30).all()), (act, k)


def test_hidden_past_32_bits_of_elements():
    """What is kept between the products passes 2^32 elements: the last rows' result and gradient are right."""
    from loopback_b200 import block
    d, f, few = 64, 4096, 300
    t = (1 << 32) // f + few
    (x, wg, wu, wd), dy = _inputs(t, d, f, 3)
    y = block.gated_ffn(x, wg.detach(), wu.detach(), wd.detach())
    (dx,) = torch.autograd.grad(y, x, dy)
    for rows in (slice(0, few), slice(t // 2 - few, t // 2), slice(t - few, t)):
        want = ref.ffn(*(v.detach().double() for v in (x[rows], wg, wu, wd)), "silu", dy[rows].double())
        ref.check_ffn("y", y[rows].detach(), *want["y"])
        ref.check_ffn("dx", dx[rows], *want["dx"])


def test_shapes_frozen_weights_and_empty_batches():
    from loopback_b200 import block
    (x, wg, wu, wd), dy = _inputs(60, 72, 136, 1)
    y = block.gated_ffn(x, wg, wu, wd)
    x3 = x.detach().view(3, 4, 5, 72).transpose(0, 1)
    y3 = block.gated_ffn(x3, wg.detach(), wu.detach(), wd.detach())
    assert torch.equal(y3.transpose(0, 1).reshape(60, 72), y)
    full = torch.autograd.grad(y, (x, wg, wu, wd), dy)
    for i in range(4):
        ins = [v.detach().requires_grad_(i == j) for j, v in enumerate((x, wg, wu, wd))]
        (g,) = torch.autograd.grad(block.gated_ffn(*ins), ins[i], dy)
        assert torch.equal(g, full[i])
    odd = torch.empty(60 * 72 + 3, device="cuda", dtype=torch.bfloat16)[3:].view(60, 72).copy_(x.detach())   # not on 16 bytes
    assert torch.equal(block.gated_ffn(odd, wg.detach(), wu.detach(), wd.detach()), y)
    fused = torch.cat((wg, wu)).detach()                  # one parameter holding both projections
    assert torch.equal(block.gated_ffn(x.detach(), *fused.chunk(2), wd.detach()), y)
    e = torch.zeros(0, 72, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    same = wg.detach().requires_grad_()                   # one tensor as both projections: its two gradients add up
    xs = x.detach()
    (gs,) = torch.autograd.grad(block.gated_ffn(xs, same, same, wd), same, dy)
    w1, w2 = (wg.detach().clone().requires_grad_() for _ in range(2))
    assert torch.equal(gs, sum(torch.autograd.grad(block.gated_ffn(xs, w1, w2, wd), (w1, w2), dy)))
    ge = torch.autograd.grad(block.gated_ffn(e, wg, wu, wd), (e, wg, wu, wd), torch.zeros_like(e))
    assert ge[0].shape == e.shape and not any(g.any() for g in ge[1:])


def test_on_another_stream_and_in_a_graph():
    from loopback_b200 import block
    (x, wg, wu, wd), dy = _inputs(700, 264, 520, 2)
    want = torch.autograd.grad(block.gated_ffn(x, wg, wu, wd), (x, wg, wu, wd), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        xs = x.detach().clone().requires_grad_()
        ws = [w.detach().clone().requires_grad_() for w in (wg, wu, wd)]
        got = torch.autograd.grad(block.gated_ffn(xs, *ws), (xs, *ws), dy)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = torch.zeros_like(x).requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.gated_ffn(static, *ws)
        grads = torch.autograd.grad(y, (static, *ws), dy)
    for _ in range(2):
        with torch.no_grad():
            static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


@pytest.mark.parametrize("t,tile", [(300, 1), (300, 3), (300, 4), (300, 5), (40, 0)])
def test_a_wait_that_runs_out_unwinds_and_reports(t, tile):
    """The products' waits are bounded. With the limit at about a millisecond and the hook that leaves out one tile copy of the
    first CTA, its multiplies give up, everybody unwinds, the kernel returns and the device error word names a wait; the next
    launch is unaffected."""
    import loopback_b200._lib as L
    from loopback_b200 import block
    (x, wg, wu, wd), _ = _inputs(t, 264, 520, 4, grad=False)
    try:
        L.set_option("ffn_tile", tile)
        good = block.gated_ffn(x, wg, wu, wd)
        assert L.device_error() == 0
        L.set_option("wait_cycles", 2_000_000)
        L.set_option("test_skip_item", 2)
        block.gated_ffn(x, wg, wu, wd)
        torch.cuda.synchronize()
        L.set_option("wait_cycles", 0)
        L.set_option("test_skip_item", 0)
        # the first wait to run out: for a tile, a free stage, the producer's last stages (begun as early, with a tile this
        # short), an accumulator
        assert L.device_error(clear=True) in (1, 2, 5, 7)
        assert torch.equal(block.gated_ffn(x, wg, wu, wd), good) and L.device_error() == 0
    finally:
        L.reset_options()


def test_two_calls_at_once():
    """Two streams at the same time: each call has a workspace of its own."""
    from loopback_b200 import block
    (x, wg, wu, wd), _ = _inputs(1500, 520, 1032, 3, grad=False)
    x2 = x.flip(0).contiguous()
    wa, wb = block.gated_ffn(x, wg, wu, wd), block.gated_ffn(x2, wg, wu, wd)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        for s, v in ((s1, x), (s2, x2)):
            with torch.cuda.stream(s):
                outs.append(block.gated_ffn(v, wg, wu, wd))
    torch.cuda.synchronize()
    assert all(torch.equal(o, (wa, wb)[i % 2]) for i, o in enumerate(outs))


def test_refusals():
    from loopback_b200 import block
    (x, wg, wu, wd), _ = _inputs(8, 64, 128, 0, grad=False)
    wide = torch.zeros(1, 1 << 20, device="cuda", dtype=torch.bfloat16)
    for call in (lambda: block.gated_ffn(x.float(), wg, wu, wd), lambda: block.gated_ffn(x, wg.float(), wu, wd),
                 lambda: block.gated_ffn(x, wg, wu, wd.t().contiguous()), lambda: block.gated_ffn(x, wg, wu[:64], wd),
                 lambda: block.gated_ffn(x, wg.t().contiguous().t(), wu, wd), lambda: block.gated_ffn(x, wg.cpu(), wu, wd),
                 lambda: block.gated_ffn(x[:, :36].contiguous(), wg[:, :36].contiguous(), wu[:, :36].contiguous(), wd[:36]),
                 lambda: block.gated_ffn(x, wg.view(-1)[4:4 + 64 * 64].view(64, 64), wu[:64], wd[:, :64].contiguous()),
                 lambda: block.gated_ffn(wide[:, :0], wide[:0], wide[:0], wide[:0])):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        block.gated_ffn(x, wg, wu, wd, act="relu")
