"""What refil_amd.blocks does on a device beyond the values (tests/test_gpu_blocks.py): other streams, captured graphs, two calls in flight."""
import pytest
import torch

from refil_amd import blocks

pytestmark = pytest.mark.gpu


def _inputs(seed=0, B=4, T=150, D=96, F=160):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return dict(x=r(B, T, D), ga=r(B, T, D), gi=r(B, T, D), decay=r(D) - 3, h0=r(B, D), dy=r(B, T, D), g=r(B, T, D), w=1 + 0.1 * r(D),
                wg=r(F, D) * D ** -0.5, wu=r(F, D) * D ** -0.5, dh=r(B, T, F))


def _all(s):
    """every explicit call once; a flat list of their outputs"""
    y, hl, saved = blocks.linrec_forward(s["x"], s["ga"], s["gi"], s["decay"], h0=s["h0"], save=True)
    out = [y, hl, *blocks.linrec_backward(s["dy"], s["x"], s["ga"], s["gi"], s["decay"], saved, h0=s["h0"])]
    state = s["h0"].clone()
    out += [blocks.linrec_step(s["x"][:, 0], s["ga"][:, 0], s["gi"][:, 0], s["decay"], state), state]
    out += blocks.norm_gate_forward(s["x"], y, s["g"], post_weight=s["w"], res_scale=s["w"], pre_weight=s["w"])
    out += blocks.norm_gate_backward(s["dy"], s["dy"], s["x"], y, s["g"], post_weight=s["w"], res_scale=s["w"], pre_weight=s["w"])
    h, sv = blocks.gated_ff_forward(s["x"], s["wg"], s["wu"], save=True)
    out += [h, *blocks.gated_ff_backward(s["dh"], s["x"], s["wg"], s["wu"], sv)[:3]]
    few = s["x"][:, :3]
    out += [blocks.gated_ff_forward(few, s["wg"], s["wu"])[0]]
    return out


def test_other_streams_and_calls_in_flight():
    a, b = _inputs(1), _inputs(2)
    want_a, want_b = _all(a), _all(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        got_a = _all(a)
    with torch.cuda.stream(s2):
        got_b = _all(b)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want_a + want_b, got_a + got_b))


def test_captured_graphs_replay_on_new_inputs():
    """forward and backward of every operator in one graph (two of them alive, replayed in turn with eager work between): each replay equals
    the eager calls on the same inputs"""
    bufs, graphs, outs = [_inputs(3), _inputs(4, B=1, T=700)], [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in bufs:
            _all(s)
    torch.cuda.current_stream().wait_stream(side)
    for s in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = _all(s)
        graphs.append(g)
        outs.append(o)
    for seed in (10, 11, 12):
        for s, g, o, shape in zip(bufs, graphs, outs, (dict(), dict(B=1, T=700))):
            for k, v in _inputs(seed, **shape).items():
                s[k].copy_(v)
            g.replay()
            got = [t.clone() for t in o]
            want = _all(s)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_autograd_backward_under_capture_is_refused():
    """a whole step captured while an eager graph of the same leaf lives: the backward raises, the process, the eager graph and later captures live on"""
    s = _inputs(5, B=2, T=20, D=16, F=24)
    x = s["x"].clone().requires_grad_(True)
    calls = [lambda: blocks.linear_recurrence(x, s["ga"], s["gi"], s["decay"])[0], lambda: blocks.norm_gate_residual(x, s["g"])[0], lambda: blocks.gated_ff(x, s["wg"], s["wu"])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        for call in calls:
            call()
    torch.cuda.current_stream().wait_stream(side)
    for call in calls:
        eager = call().sum()
        with pytest.raises(RuntimeError, match="cannot run under graph capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call().sum().backward()
        x.grad = None
        eager.backward()
        assert torch.isfinite(x.grad).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h, _ = blocks.gated_ff_forward(x.detach(), s["wg"], s["wu"])
    g.replay()
    assert torch.equal(h, blocks.gated_ff(x.detach(), s["wg"], s["wu"]))


def test_tensors_of_the_other_device_are_refused():
    s = _inputs(6, B=1, T=4, D=8, F=8)
    with pytest.raises(ValueError, match="decay_gate is on cpu"):
        blocks.linrec_forward(s["x"], s["ga"].cpu(), s["gi"], s["decay"])
    with pytest.raises(ValueError, match="w_gate is on cpu"):
        blocks.gated_ff_forward(s["x"], s["wg"].cpu(), s["wu"])
    with pytest.raises(ValueError, match="o is on cpu"):
        blocks.norm_gate_forward(s["x"], s["g"].cpu())


def test_offsets_past_32_bits():
    """row and batch strides of 2^30 elements: the last rows start past 6 * 2^30 bytes"""
    n = 1 << 30
    pool = torch.empty(3 * n + 64, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(pool, (4, 2, 32), (n, 32, 1))
    g = torch.Generator(device="cuda").manual_seed(1)
    x.copy_(torch.randn(4, 2, 32, generator=g, device="cuda"))
    dense = x.contiguous()
    decay = torch.randn(32, generator=g, device="cuda") - 3

    def rec(t):
        y, h, saved = blocks.linrec_forward(t, t, t, decay, save=True)
        return [y, h, *blocks.linrec_backward(t, t, t, t, decay, saved), blocks.linrec_step(t[:, 0], t[:, 0], t[:, 0], decay, torch.zeros(4, 32, device="cuda"))]

    def norm(t):
        return [*blocks.norm_gate_forward(t, t, t), *blocks.norm_gate_backward(t, t, t, t, t)[:3]]
    w = torch.randn(40, 32, generator=g, device="cuda").to(torch.bfloat16)

    def ff(t):
        h, saved = blocks.gated_ff_forward(t, w, w, save=True)
        return [h, *blocks.gated_ff_backward(h, t, w, w, saved)[:3]]
    for f, a, b in ((rec, x, dense), (norm, x[:, 0], dense[:, 0].contiguous()), (ff, x[:, 0], dense[:, 0].contiguous())):
        assert all(torch.equal(p, q) for p, q in zip(f(a), f(b)))


def test_more_than_two_to_the_31_elements():
    """the last episode / rows of tensors of 2.2e9 elements against calls on them alone (other tile and chunk counts: to rounding)"""
    B, T, D = 33, 8192, 8192
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.empty(B, T, D, dtype=torch.bfloat16, device="cuda")
    for b in range(B):
        x[b] = torch.randn(T, D, generator=g, device="cuda")
    decay = torch.randn(D, generator=g, device="cuda") - 5

    def near(a, b):
        torch.testing.assert_close(a, b, rtol=2 ** -7, atol=1e-3)        # (two roundings to bf16 apart at most)
    y, h, _ = blocks.linrec_forward(x, x, x, decay)
    y1, h1, _ = blocks.linrec_forward(x[-1:], x[-1:], x[-1:], decay)
    near(y[-1], y1[0])
    torch.testing.assert_close(h[-1], h1[0], rtol=1e-4, atol=1e-5)
    rows = x.view(-1, D)
    n = blocks.norm_gate_forward(rows, y.view(-1, D), want_y=False)[1]
    near(n[-300:], blocks.norm_gate_forward(rows[-300:], y.view(-1, D)[-300:], want_y=False)[1])
    del n, y
    w = (torch.randn(D, 64, generator=g, device="cuda") * 0.1).to(torch.bfloat16)
    narrow = rows[:, :64]
    out = blocks.gated_ff(narrow, w, w)
    near(out[-300:], blocks.gated_ff(narrow[-300:], w, w))
