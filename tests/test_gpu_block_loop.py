"""The operators around a block used together, as a looped model uses them: shared feed-forward blocks between the reads of
the update stack (write, combine), trained and decoded."""
import pytest
import torch

import block_reference as ref
from oracle import torch_oracle as TO

pytestmark = pytest.mark.gpu
K, R, D, F, EPS = 3, 2, 256, 520, 1e-6
N = K * R


def _model(seed, p=0.0):
    from loopback_b200.block import FeedForwardBlock
    from loopback_b200.cell import LoopDeltaAttnRes
    torch.manual_seed(seed)
    blocks = torch.nn.ModuleList(FeedForwardBlock(D, F, "silu" if i else "gelu", post_norm=i != 1, gate=i == 2, scale=0.5, learn_scale=i == 0,
                                                  p=p, device="cuda") for i in range(K))
    cell = LoopDeltaAttnRes(D, R, K, beta=0.75, eps=EPS).cuda()
    with torch.no_grad():
        cell.query.normal_(0, 0.05)
        for b in blocks:
            b.norm.add_(0.1 * torch.randn_like(b.norm))
    return blocks, cell


def _run(blocks, cell, h0, rng=None):
    stack = cell.new_stack(h0.shape, h0.dtype, "cuda")
    x, deltas, keys, coeffs, prior, states = h0, [], [], None, None, []
    for s in range(N):
        l, b = divmod(s, K)
        h = blocks[b](x, rng=None if rng is None else (rng, s))
        deltas.append(stack.write(s, h, x))
        x, coeffs, prior = cell.combine(h, h0, deltas, coeffs, prior, l, b, keys=keys, stack=stack)
        states.append(x)
    return states


def _exact(params, h0, t, p=0.0, rng=0):
    """The same pass in 64 bits, nothing rounded."""
    x, sources, scales, tc, c0, states = h0, [], [], None, None, []
    for s in range(N):
        b = s % K
        g = {k[len(f"{b}."):]: v for k, v in params.items() if k.startswith(f"{b}.")}
        unit = lambda a: a * torch.rsqrt(a.square().mean(-1, keepdim=True) + EPS)  # noqa: E731
        u = unit(x) * g["norm"]
        act = torch.nn.functional.silu if b else torch.nn.functional.gelu
        y = (act(u @ g["w_gate"].T) * (u @ g["w_up"].T)) @ g["w_down"].T
        if "norm_after" in g:
            y = unit(y) * g["norm_after"]
        if p:
            y = y * ref.factor(p, rng, s, 0, t * D).view(1, t, D).cuda()
        h = x + g.get("scale", 0.5) * g.get("gate", 1.0) * y
        v = h - x
        sources.append(v)
        scales.append(TO.key_scale(v, EPS))
        base, cbar, c0 = TO.prologue(h, h0, tc, c0, 0.75, b == K - 1)
        if s == 0:
            x, tc = base, cbar
        else:
            x, tc = TO.read(base, sources, params["query"][s - 1], cbar, c0, EPS, scales=scales)
        states.append(x)
    return states


@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("t", [1, 77, 640])
def test_looped_blocks_train(t, p):
    """Every state and every parameter's gradient against the pass in 64 bits, in norm. A step rounds about ten bf16 tensors on
    the way to its state (norm, h, y, the residual's sum, the update, the read's sum) and as many in its backward; a rounding
    is off by at most 2^-8 / sqrt 3 in the mean square, independent ones add in squares: over 6 steps sqrt(60) 2^-8 / sqrt 3 =
    1.8e-2 for the states; twice as many roundings lie on a gradient's way: 2.5e-2. Single tokens average less: twice that. The
    residual scale's gradient is one number, a sum over the elements whose terms cancel: the terms are off by 2.5e-2 of
    themselves in the mean square, so their sum by 2.5e-2 of the root of the sum of their squares (one standard deviation;
    three are allowed), whatever is left of the sum itself. The terms are the gradient of a scale per element."""
    blocks, cell = _model(1, p)
    gen = torch.Generator(device="cuda").manual_seed(t)
    h0 = torch.randn(1, t, D, device="cuda", generator=gen).bfloat16().requires_grad_()
    ups = [torch.randn(1, t, D, device="cuda", generator=gen).bfloat16() for _ in range(N)]
    states = _run(blocks, cell, h0, rng=99)
    names = {n: v for n, v in blocks.named_parameters()} | {"query": cell.query, "h0": h0}
    grads = dict(zip(names, torch.autograd.grad(states, list(names.values()), ups)))
    exact = {n: (v.detach().double().expand(1, t, D).clone() if n.endswith("scale") else v.detach().double()).requires_grad_() for n, v in names.items()}
    want = _exact(exact, exact["h0"], t, p, 99)
    wants = dict(zip(names, torch.autograd.grad(want, list(exact.values()), [u.double() for u in ups])))
    from loopback_b200._lib import device_error
    assert device_error() == 0
    more = 2.0 if t == 1 else 1.0
    for s, (a, b) in enumerate(zip(states, want)):
        rel = float((a.double() - b).detach().norm() / b.detach().norm())
        assert rel <= 1.8e-2 * more, f"state {s}: {rel:.3g}"
    for n in names:
        if n.endswith("scale"):
            off = abs(float(grads[n].double() - wants[n].sum()))
            assert off <= 3 * 2.5e-2 * more * float(wants[n].norm()), f"{n}: {off:.3g} where the terms' norm is {float(wants[n].norm()):.3g}"
            continue
        rel = float((grads[n].double() - wants[n]).norm() / wants[n].norm())
        assert rel <= 2.5e-2 * more, f"{n}: {rel:.3g}"


def test_norm_formed_by_the_previous_block():
    """Without a read in between, a block can be handed the norm the one before it formed."""
    blocks, _ = _model(2)
    x = torch.randn(2, 33, D, device="cuda").bfloat16()
    out, u = blocks[0](x, next_weight=blocks[1].norm)
    a, b = blocks[1](out, normed=u), blocks[1](out)
    # u is the norm of out before its rounding (2^-8 / sqrt 3 in the mean square), and both results are rounded
    assert float(((a - b).detach().float().norm() / b.detach().float().norm())) < 2 * 2.0 ** -8


def test_decode_equals_the_same_rows_of_a_pass():
    """Few rows take kernels of their own in every operator: their states against the same rows in a larger batch, in norm
    (the products are summed in another order, the rest is the same arithmetic): the bound of the states above."""
    blocks, cell = _model(3)
    h0 = torch.randn(1, 512, D, device="cuda").bfloat16()
    with torch.no_grad():
        full = _run(blocks.eval(), cell, h0)
        few = _run(blocks, cell, h0[:, :5].contiguous())
    for a, b in zip(few, full):
        assert float((a.double() - b[:, :5].double()).norm() / b[:, :5].double().norm()) <= 1.8e-2


def test_eval_has_no_dropout_and_training_needs_numbers():
    blocks, _ = _model(4, p=0.5)
    x = torch.randn(1, 8, D, device="cuda").bfloat16()
    with pytest.raises(ValueError):
        blocks[0](x)
    blocks.eval()
    with torch.no_grad():
        assert torch.equal(blocks[0](x), blocks[0](x, rng=(1, 2)))


def test_a_pass_in_a_graph_draws_new_masks():
    """One captured training step of a block, replayed: each replay reads the pair as it then is."""
    blocks, _ = _model(5, p=0.25)
    block = blocks[2]
    x = torch.randn(1, 300, D, device="cuda").bfloat16()
    rng = torch.tensor([5, 0], device="cuda")
    params = [v.detach().clone().requires_grad_() for v in (block.w_gate, block.w_up, block.w_down)]
    from loopback_b200 import block as B

    def step():
        y = B.gated_ffn(B.block_norm(x, block.norm.detach()), *params)
        out = B.block_residual(x, y, block.norm_after.detach(), gate=block.gate.detach(), scale=0.5, p=0.25, rng=rng)
        return (out, *torch.autograd.grad(out, params, torch.ones_like(out)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    seen = []
    for offset in (7, 8):
        rng[1] = offset
        graph.replay()
        torch.cuda.synchronize()
        mine = [v.clone() for v in got]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(mine, want))
        seen.append(mine[0])
    assert not torch.equal(*seen)


def _chain(x, block, rng):
    """Every kind of launch of the operators behind one another, each result from the one before."""
    from loopback_b200 import block as B
    u = B.block_norm(x, block.norm)
    y = B.dropout(B.gated_ffn(u, block.w_gate, block.w_up, block.w_down), 0.25, rng)
    out, n = B.block_residual(x, y, block.norm_after, gate=block.gate, scale=0.5, next_weight=block.norm, p=0.1, rng=rng)
    return out, n


@pytest.mark.parametrize("t", [1, 64, 300, 5000])
@pytest.mark.parametrize("before", ["nothing", "copy", "fill", "memset", "host copy", "other stream", "own kernel"])
def test_launches_wait_for_what_comes_before(t, before):
    """The launches overlap their edges with whatever precedes them on the stream, eager and captured: what an earlier piece of
    work still writes when the operator is launched (weights and rows, behind a long kernel) has to be what it reads."""
    blocks, _ = _model(6)
    block = blocks[2]
    gen = torch.Generator(device="cuda").manual_seed(t)
    x = torch.randn(t, D, device="cuda", generator=gen).bfloat16()
    rng = torch.tensor([5, 6], device="cuda")
    side = torch.cuda.Stream()
    host = x.cpu().pin_memory()
    with torch.no_grad():
        want = _chain(x, block, rng)
        good = {n: v.clone() for n, v in block.named_parameters()}
        wrong, late = torch.zeros_like(x), torch.full_like(x, 9.0)
        names = ("w_gate", "w_up", "w_down", "norm")

        def spoil():
            late.fill_(9.0)
            for n in names:
                getattr(block, n).fill_(3.0)

        def put(v):                                       # a slow kernel, then what the chain reads
            torch.cuda._sleep(200_000)
            for n in names:
                getattr(block, n).copy_(good[n])
            if v == "copy":
                late.copy_(x)
            elif v == "fill":
                late.copy_(x)
                wrong.fill_(1.0)
            elif v == "memset":
                late.copy_(x)
                wrong.zero_()
            elif v == "host copy":
                late.copy_(host, non_blocking=True)
            elif v == "other stream":
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    torch.cuda._sleep(100_000)
                    late.copy_(x)
                torch.cuda.current_stream().wait_stream(side)
            elif v == "own kernel":
                from loopback_b200 import block as B
                late.copy_(x)
                B.block_norm(late, block.norm)
        if before != "nothing":
            for _ in range(3):
                spoil()
                put(before)
                got = _chain(late, block, rng)
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        late.copy_(x)
        with torch.cuda.graph(graph):
            if before != "nothing":
                put(before)
            got = _chain(late, block, rng)
            again = _chain(late, block, rng)              # its own launches precede it
        for _ in range(3):
            if before != "nothing":
                spoil()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(again, want))


_CAPTURE = """
import torch
from loopback_b200 import block as B
x = torch.randn(300, 64, device="cuda").bfloat16().requires_grad_()
w, wg, wu, wd = (torch.randn(*s, device="cuda").bfloat16().requires_grad_() for s in ((64,), (128, 64), (128, 64), (64, 128)))
calls = {"block_norm": (lambda: B.block_norm(x, w), (x, w)), "dropout": (lambda: B.dropout(x, 0.5, (1, 2)), (x,)),
         "block_residual": (lambda: B.block_residual(x, x, w, p=0.5, rng=(1, 2)), (x, w)),
         "gated_ffn": (lambda: B.gated_ffn(x, wg, wu, wd), (x, wg, wu, wd))}
up = torch.ones_like(x)
for name, (call, leaves) in calls.items():
    alive = call()                                       # its graph holds the leaves' nodes, on the default stream
    want = torch.autograd.grad(alive, leaves, up, retain_graph=True)
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            torch.autograd.grad(call(), leaves, up)
        raise SystemExit(name + " was captured")
    except RuntimeError as e:
        assert "is alive" in str(e), e
    again = torch.autograd.grad(alive, leaves, up)       # the eager graph is as it was
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(), leaves, up)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, again, got)), name
print("refused and captured")
"""


def test_capture_of_a_backward_beside_a_live_eager_graph():
    """The backward of leaves whose eager graph is alive cannot be captured: it raises, and works once that graph is gone. In a
    child process, since the error it stands in front of would end this one."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", _CAPTURE], capture_output=True, text=True, timeout=300, cwd=here)
    assert done.returncode == 0 and "refused and captured" in done.stdout, done.stdout[-2000:] + done.stderr[-2000:]
