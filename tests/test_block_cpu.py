"""CPU-side checks of the operators around a block: refusals come before any GPU call, dropout's generator against its
published answers, the closed-form gradients the GPU tests use against automatic differentiation."""
import pytest
import torch

import block_reference as ref


def test_no_cpu_path():
    from loopback_b200 import block
    x, w = torch.zeros(2, 64), torch.ones(64)
    b = torch.zeros(64, 64, dtype=torch.bfloat16)
    for call in (lambda: block.block_norm(x, w), lambda: block.block_residual(x, x, w), lambda: block.dropout(x, 0.5, (1, 2)),
                 lambda: block.gated_ffn(b, b, b, b), lambda: block.FeedForwardBlock(64, 128)(b)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for bad in (lambda: block.FeedForwardBlock(60, 128), lambda: block.FeedForwardBlock(64, 0), lambda: block.FeedForwardBlock(64, 64, "relu"),
                lambda: block.FeedForwardBlock(64, 64, p=1.0), lambda: block.gated_ffn(b, b, b, b, act="tanh")):
        with pytest.raises(ValueError):
            bad()
    m = block.FeedForwardBlock(64, 128, post_norm=True, gate=True, learn_scale=True)
    assert {n: tuple(v.shape) for n, v in m.named_parameters()} == {
        "norm": (64,), "norm_after": (64,), "gate": (64,), "scale": (1,), "w_gate": (128, 64), "w_up": (128, 64), "w_down": (64, 128)}


def test_argument_validation_needs_no_gpu():
    import loopback_b200._lib as L
    lib, bf, f32 = L.lib(), L.LB_DTYPE_BF16, L.LB_DTYPE_F32
    a, odd = 1 << 20, (1 << 20) + 8                       # addresses that are looked at, never used
    assert lib.lb_block_scratch_bytes(1024) >= 2 * 304 * 1024 * 4 and lib.lb_block_scratch_bytes(-1) == 0
    norm = lambda x, w, u, d=64, dt=bf, wt=bf, n=4: lib.lb_norm_fwd(x, w, u, None, n, d, 1e-6, dt, wt, None)  # noqa: E731
    assert norm(None, a, a) == -1 and norm(a, None, a) == -1 and norm(a, a, None) == -1
    assert norm(odd, a, a) == -2 and norm(a, a, a, d=63) == -2 and norm(a, a, a, d=8200) == -3
    assert norm(a, a, a, dt=9) == -1 and norm(a, a, a, dt=f32, wt=bf) == -1 and norm(a, a, a, n=-1) == -1
    bwd = lambda r=a, dw=None, scratch=None: lib.lb_norm_bwd(a, a, r, a, a, dw, scratch, 4, 64, bf, bf, None)  # noqa: E731
    assert bwd(r=None) == -1

    def res(y=a, gate=None, kind=0, nxt=None, u=None, thr=0, rng=None):
        return lib.lb_residual_fwd(a, y, None, gate, kind, None, 1.0, nxt, a, u, None, None, thr, rng, 0, 0, None, 4, 64, 1e-6, bf,
                                   bf, None)
    assert res(y=None) == -1 and res(gate=a) == -1 and res(kind=1) == -1 and res(kind=4, gate=a) == -1 and res(nxt=a) == -1
    assert res(gate=odd, kind=2) == -2 and res(thr=65536) == -1 and res(thr=-1) == -1 and res(thr=5, rng=a + 4) == -2

    def resb(dout=a, du=None, nxt=None, ry=None, w=None, dw=None, dscale=None, dgate=None):
        return lib.lb_residual_bwd(a, a, w, None, 0, None, 1.0, nxt, ry, None, 0, None, 0, 0, dout, du, a, a, dw, dgate, dscale, None,
                                   None, 4, 64, bf, bf, None)
    assert resb(dout=None) == -1 and resb(du=a) == -1 and resb(w=a) == -1 and resb(dw=a) == -1 and resb(dscale=a) == -1
    assert resb(dgate=a) == -1
    ffn = lambda x=a, h=None, kept=None, ws=a, t=4, d=64, f=64, act=0, dt=bf: lib.lb_ffn_fwd(  # noqa: E731
        x, a, a, a, a, h, kept, ws, 1 << 30, t, d, f, act, dt, None)
    assert ffn(x=None) == -1 and ffn(ws=None) == -1 and ffn(kept=a) == -1 and ffn(act=2) == -1 and ffn(t=-1) == -1 and ffn(f=0) == -1
    assert ffn(d=60) == -2 and ffn(f=12) == -2 and ffn(x=odd) == -2 and ffn(dt=f32) == -3 and ffn(f=(1 << 20) + 8) == -3
    assert ffn(t=(1 << 31) - 8) == -3
    ffnb = lambda dy=a, h=a, kept=a, d=64, dt=bf: lib.lb_ffn_bwd(a, a, a, a, h, kept, dy, a, a, a, a, 1 << 30, 4, d, 64, dt, None)  # noqa: E731
    assert ffnb(dy=None) == -1 and ffnb(h=None) == -1 and ffnb(kept=None) == -1 and ffnb(dy=odd) == -2 and ffnb(d=4) == -2 and ffnb(dt=f32) == -3
    assert lib.lb_ffn_kept_bytes(33, 40) >= 2 * 2 * 6144 and lib.lb_ffn_kept_bytes(3, 4) == 0 and lib.lb_ffn_workspace_bytes(4, 64, 64, 7) == 0
    drop = lambda x, o, n=8, thr=1, dt=bf: lib.lb_dropout(x, o, thr, None, 0, 0, None, n, dt, None)  # noqa: E731
    assert drop(None, a) == -1 and drop(a, a) == -1 and drop(odd, a) == -2 and drop(a, a + 16, n=-1) == -1
    assert drop(a, a + 16, thr=70000) == -1 and drop(a, a + 16, dt=3) == -1


def test_generator_against_published_answers():
    """The known answers that Random123 ships for philox4x32 with 10 rounds."""
    assert ref.philox4x32_10((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    top = 0xFFFFFFFF
    assert ref.philox4x32_10((top,) * 4, (top, top)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    m = ref.factor(0.25, (7 << 32) + 9, (3 << 32) + 2, 8 * 5, 8)
    words = ref.philox4x32_10((5, 0, 2, 3), (9, 7))
    halves = [h for w in words for h in (w & 0xFFFF, w >> 16)]
    assert m.tolist() == [65536 / 49152 if h >= 16384 else 0.0 for h in halves]


@pytest.mark.parametrize("kind", ["", "channel", "token", "full"])
def test_closed_form_gradients(kind):
    gen = torch.Generator().manual_seed(0)
    t, d = 5, 24
    rnd = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    v = {"x": rnd(t, d), "y": rnd(t, d), "w": rnd(d), "scale": rnd(1), "w_next": rnd(d)}
    if kind:
        v["gate"] = rnd(*{"channel": (d,), "token": (t, 1), "full": (t, d)}[kind])
    v = {k: a.requires_grad_() for k, a in v.items()}
    m, dout, du = (rnd(t, d) > 0).double() * 2, rnd(t, d), rnd(t, d)
    r = ref.residual(v["x"], v["y"], v["w"], v.get("gate"), kind, v["scale"], v["w_next"], m, dout, du, True)
    grads = torch.autograd.grad([r["out"][0], r["u"][0]], list(v.values()), [dout, du])
    for k, g in zip(v, grads):
        assert torch.allclose(r["d" + k][0].detach(), g, rtol=1e-11, atol=1e-11), k
