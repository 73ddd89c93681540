"""The residual temporal block (refil_amd.blocks: gated linear recurrence, norms with gate and residual scale, gated feed-forward) against
plain implementations in 64 bits.

Tolerances are majorants of the rounding errors, evaluated in 64 bits beside the value itself: every fp32 operation is off by at most
2^-24 of its result, an output of type t by at most eps(t) / 2 of its value more. U = 2^-24 below; K counts the roundings on the way to a
value, and the majorant sums the magnitudes that they act on."""
import math

import pytest
import torch

from refil_amd import blocks

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def rnd(*shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def close(name, got, want, fp32_error):
    """got (its type rounds by half a step) against want (64 bits) with the fp32 error majorant fp32_error >= 0"""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny                      # below the normal range a step no longer shrinks with the value
    bound = half * (want.abs() + fp32_error) + fp32_error + tiny * (2 * half if got.dtype != F32 else 1)
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound).nan_to_num(nan=math.inf).max()):.3g} x the bound"


# ------------------------------------------------------------------------------------------------ gated linear recurrence
def rec_ref(x, ga, gi, decay, scale, h0, reset, lengths, dy=None, dh_last=None):
    """values and error majorants (see the module's docstring), step by step in 64 bits.

    K: a sigmoid costs |argument| + 4 roundings (the exponent's product, 2^x, the sum, the reciprocal), a = exp(-L) costs L + 5, the root
    and the products around it 8 more."""
    B, T, D = x.shape[0], x.shape[1], x.shape[-1]
    one = (B,) + (1,) * (x.dim() - 2)
    d, x, ga, gi = decay.double(), x.double(), ga.double(), gi.double()
    sp = torch.nn.functional.softplus(d, threshold=700.0)
    rate = scale * sp
    sa, si = torch.sigmoid(ga), torch.sigmoid(gi)
    L = rate * sa
    a = torch.exp(-L)
    beta = torch.sqrt(-torch.expm1(-2 * L))
    u = beta * si * x
    lob = torch.where(L > 0, L / beta.clamp_min(1e-300), torch.zeros_like(L))
    # (the gates' own magnitude: what sits in a masked place is capped, there its sigmoid is 0 or 1 exactly)
    K = 24 + ga.abs().clamp_max(100).amax() + gi.abs().clamp_max(100).amax() + 3 * L.amax()
    h = torch.zeros(B, *x.shape[2:], dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    M = torch.zeros_like(h)
    n = torch.full((B,), T, device=x.device) if lengths is None else lengths.long().clamp(0, T)
    cut = torch.zeros(B, T, dtype=torch.bool, device=x.device) if reset is None else reset.bool()
    y, My, prev, Mprev = torch.zeros_like(x), torch.zeros_like(x), [], []
    for t in range(T):
        prev.append(h)
        Mprev.append(M)
        c, on = cut[:, t].reshape(one), (t < n).reshape(one)
        ah = torch.where(c, torch.zeros_like(h), a[:, t] * h)
        aM = torch.where(c, torch.zeros_like(M), a[:, t] * M)
        h = torch.where(on, ah + u[:, t], h)
        M = torch.where(on, aM + ah.abs() + u[:, t].abs(), M)
        y[:, t] = torch.where(on, h, torch.zeros_like(h))
        My[:, t] = torch.where(on, M, torch.zeros_like(M))
    out = {"y": (y, K * U * My), "h_last": (h, K * U * M)}
    if dy is None:
        return out
    dy = dy.double()
    g = torch.zeros_like(h) if dh_last is None else dh_last.double()
    Mg = g.abs()
    dx, dga, dgi, ex, ea, ei = (torch.zeros_like(x) for _ in range(6))
    dd, ed = torch.zeros(D, dtype=torch.float64, device=x.device), torch.zeros(D, dtype=torch.float64, device=x.device)
    zero = torch.zeros_like(g)
    for t in range(T - 1, -1, -1):
        c, on = cut[:, t].reshape(one), (t < n).reshape(one)
        gt = torch.where(on, g + dy[:, t], zero)
        Mt = torch.where(on, Mg + dy[:, t].abs(), zero)                    # >= |gt|, and the unit its errors come in
        p = torch.where(c, zero, a[:, t] * prev[t])
        Mp = torch.where(c, zero, a[:, t] * (prev[t].abs() + Mprev[t]))
        sx = si[:, t] * x[:, t]
        dx[:, t] = gt * beta[:, t] * si[:, t]
        ex[:, t] = 2 * Mt * beta[:, t] * si[:, t]
        dgi[:, t] = gt * beta[:, t] * sx * (1 - si[:, t])
        ei[:, t] = 2 * Mt * beta[:, t] * sx.abs()                          # 1 - sigmoid cancels: its error is absolute
        first = sx * a[:, t] ** 2 * lob[:, t]
        q = gt * (first - p * L[:, t])
        Mq = 2 * Mt * (first.abs() + Mp * L[:, t])
        dga[:, t] = q * (1 - sa[:, t])
        ea[:, t] = Mq
        dd += q.reshape(-1, D).sum(0)
        ed += Mq.reshape(-1, D).sum(0)
        g = torch.where(on, torch.where(c, zero, a[:, t] * gt), g)
        Mg = torch.where(on, torch.where(c, zero, a[:, t] * (Mt + gt.abs())), Mg)
    ratio = torch.where(sp > 0, torch.sigmoid(d) / sp.clamp_min(1e-300), torch.ones_like(d))
    adds = 64 + T / 16 + x.numel() / D / 256        # additions that a term of ddecay passes through: threads, waves, tiles, then the partial rows
    out.update(dx=(dx, K * U * ex), dga=(dga, K * U * ea), dgi=(dgi, K * U * ei), ddecay=(dd * ratio, (K + adds) * U * ed * ratio), dh0=(g, K * U * Mg))
    return out


def rec_case(B, T, na, D, dtype, seed, ragged=True, h0=True, decay_shift=-3.0):
    shape = (B, T, na, D) if na else (B, T, D)
    kw = dict(h0=rnd(B, *shape[2:], seed=seed + 5) if h0 else None, reset=None, lengths=None)
    if ragged:
        g = torch.Generator().manual_seed(seed + 6)
        ln = torch.randint(0, T + 1, (B,), generator=g)
        ln[0] = T
        if B > 1:
            ln[1] = 0
        if B > 2:
            ln[2] = min(1, T)
        kw["lengths"] = ln.to(torch.int32).to(DEV)
        kw["reset"] = (torch.rand(B, T, generator=g) < 0.1).to(torch.uint8).to(DEV)
    return (rnd(*shape, seed=seed, dtype=dtype), rnd(*shape, seed=seed + 1, dtype=dtype, scale=2.0), rnd(*shape, seed=seed + 2, dtype=dtype, scale=2.0),
            rnd(D, seed=seed + 3) + decay_shift), kw


def rec_check(args, kw, scale=8.0, dh_last=None, seed=99):
    x = args[0]
    dy = rnd(*x.shape, seed=seed, dtype=x.dtype)
    y, h_last, saved = blocks.linrec_forward(*args, scale=scale, save=True, **kw)
    y2, h2, none = blocks.linrec_forward(*args, scale=scale, **kw)
    assert none is None and torch.equal(y, y2) and torch.equal(h_last, h2)
    r = blocks.linrec_backward(dy, *args, saved, scale=scale, dh_last=dh_last, **kw)
    r2 = blocks.linrec_backward(dy, *args, saved, scale=scale, dh_last=dh_last, **kw)
    assert all(torch.equal(p, q) for p, q in zip(r, r2))                      # the same sums every time
    ref = rec_ref(*args, scale, kw["h0"], kw["reset"], kw["lengths"], dy, dh_last)
    got = dict(y=y, h_last=h_last, dx=r[0], dga=r[1], dgi=r[2], ddecay=r[3], dh0=r[4])
    for k, v in got.items():
        close(k, v, *ref[k])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,na,D", [(1, 1, 0, 1), (2, 3, 0, 64), (3, 65, 0, 7), (4, 81, 3, 24), (3, 128, 0, 65), (1, 200, 5, 33), (2, 70, 0, 258), (3, 33, 0, 511), (1, 3, 0, 2)])
def test_linrec_matches_the_definition(B, T, na, D, dtype):
    args, kw = rec_case(B, T, na, D, dtype, seed=100 + B * T + D)
    state = (B, na, D) if na else (B, D)
    rec_check(args, kw, dh_last=rnd(*state, seed=9))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linrec_without_the_optional_inputs(dtype):
    args, kw = rec_case(2, 70, 0, 40, dtype, seed=3, ragged=False, h0=False)
    rec_check(args, kw)


def test_linrec_long_sequence_few_rows():
    """one row, several chunks of the time axis; scale other than the default; slow and fast decays"""
    args, kw = rec_case(1, 1500, 0, 10, F32, seed=21)
    kw["lengths"] = torch.tensor([1400], dtype=torch.int32, device=DEV)
    args = (*args[:3], torch.linspace(-8, 3, 10).to(DEV))
    rec_check(args, kw, scale=2.0)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_linrec_strided_inputs(dtype):
    """x, the gates as slices of one projection [T, B, 3 D + 5]: batch behind time, odd row strides; expanded reset"""
    B, T, D = 3, 37, 20
    fused = rnd(T, B, 3 * D + 5, seed=31, dtype=dtype)
    x, ga, gi = (fused[:, :, i * D + 1:(i + 1) * D + 1].transpose(0, 1) for i in range(3))
    reset = torch.zeros(1, T, dtype=torch.bool, device=DEV)
    reset[0, 11] = True
    kw = dict(h0=rnd(B, D, seed=32), reset=reset.expand(B, T), lengths=None)
    rec_check((x, ga, gi, rnd(D, seed=33) - 3), kw)


def test_linrec_nothing_passes_a_reset_or_an_episodes_end():
    """NaN and Inf behind a reset, in h0 in front of one, and behind an episode's end"""
    B, T, D = 3, 140, 9
    args, kw = rec_case(B, T, 0, D, F32, seed=41, ragged=False)
    x, ga, gi, decay = args
    reset = torch.zeros(B, T, dtype=torch.uint8, device=DEV)
    reset[:, 0] = 1
    reset[:, 70] = 1
    lengths = torch.tensor([T, 100, 90], dtype=torch.int32, device=DEV)
    kw = dict(h0=torch.full((B, D), math.nan, device=DEV), reset=reset, lengths=lengths)
    clean = rec_ref(x, ga, gi, decay, 8.0, torch.zeros(B, D, device=DEV), reset, lengths)
    for t in (x, ga, gi):
        t[1, 100:] = math.nan
        t[2, 95:] = math.inf
    y, h_last, _ = blocks.linrec_forward(x, ga, gi, decay, **kw)
    close("y", y, *clean["y"])
    close("h_last", h_last, *clean["h_last"])
    x[0, 69] = math.nan
    y, h_last, _ = blocks.linrec_forward(x, ga, gi, decay, **kw)
    assert torch.isnan(y[0, 69]).all() and not torch.isnan(y[0, 70:]).any()
    close("y behind the reset", y[0, 70:], clean["y"][0][0, 70:], clean["y"][1][0, 70:])
    close("h_last", h_last, *clean["h_last"])


def test_linrec_gates_at_their_ends():
    """gates at +-inf and at the type's lowest value: a_t = 1 keeps the state, gradients stay finite where the root is 0"""
    B, T, D = 1, 6, 8
    x, ga, gi = rnd(B, T, D, seed=51), torch.zeros(B, T, D, device=DEV), torch.zeros(B, T, D, device=DEV)
    ga[:, 1], ga[:, 2], ga[:, 3] = -math.inf, torch.finfo(F32).min, math.inf
    gi[:, 4], gi[:, 5] = -math.inf, math.inf
    h0, decay, dy = rnd(B, D, seed=52), rnd(D, seed=53) - 2, rnd(B, T, D, seed=54)
    y, h_last, saved = blocks.linrec_forward(x, ga, gi, decay, h0=h0, save=True)
    assert torch.equal(y[:, 1], y[:, 0]) and torch.equal(y[:, 2], y[:, 0])
    grads = blocks.linrec_backward(dy, x, ga, gi, decay, saved, h0=h0)
    assert all(torch.isfinite(g).all() for g in grads)
    ref = rec_ref(x, ga.clamp(-200, 200), gi.clamp(-200, 200), decay, 8.0, h0, None, None, dy)
    for k, v in dict(y=y, h_last=h_last, dx=grads[0], dga=grads[1], dgi=grads[2], ddecay=grads[3], dh0=grads[4]).items():
        close(k, v, *ref[k])


def test_linrec_empty_shapes():
    decay = rnd(4, seed=1)
    for B, T in ((0, 5), (2, 0)):
        x = rnd(B, T, 4, seed=2)
        h0 = rnd(B, 4, seed=3)
        y, h_last, saved = blocks.linrec_forward(x, x, x, decay, h0=h0, save=True)
        assert y.shape == x.shape and torch.equal(h_last, h0)
        dh = rnd(B, 4, seed=4)
        dx, dga, dgi, dd, dh0 = blocks.linrec_backward(x, x, x, x, decay, saved, h0=h0, dh_last=dh)
        assert torch.equal(dh0, dh) and torch.equal(dd, torch.zeros_like(dd)) and dx.shape == x.shape


def test_linrec_lengths_out_of_range_are_clamped():
    args, kw = rec_case(3, 20, 0, 8, F32, seed=61, ragged=False)
    kw["lengths"] = torch.tensor([-5, 1 << 30, 20], dtype=torch.int32, device=DEV)
    y, h_last, _ = blocks.linrec_forward(*args, **kw)
    assert torch.equal(h_last[0], kw["h0"][0]) and not y[0].any()
    kw["lengths"] = None
    full = blocks.linrec_forward(*args, **kw)
    assert torch.equal(y[1:], full[0][1:]) and torch.equal(h_last[1:], full[1][1:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,na,D", [(1, 0, 1), (5, 3, 24), (130, 0, 33), (2, 0, 700)])
def test_linrec_step(B, na, D, dtype):
    """a step is the one-step episode; with slots in any order, padded rows, and into another buffer"""
    shape = (B, na, D) if na else (B, D)
    x, ga, gi = (rnd(*shape, seed=70 + i, dtype=dtype) for i in range(3))
    decay, state = rnd(D, seed=73) - 3, rnd(B + 4, *shape[1:], seed=74)
    ref = rec_ref(x[:, None], ga[:, None], gi[:, None], decay, 8.0, state[:B], None, None)
    st = state.clone()
    y = blocks.linrec_step(x, ga, gi, decay, st)
    close("y", y, ref["y"][0][:, 0], ref["y"][1][:, 0])
    close("state", st[:B], *ref["h_last"])
    assert torch.equal(st[B:], state[B:])
    g = torch.Generator().manual_seed(5)
    slots = torch.randperm(B + 4, generator=g)[:B].to(torch.int32)
    padded = torch.rand(B, generator=g) < 0.3
    padded[0] = False
    slots[padded] = torch.tensor(-1, dtype=torch.int32)
    if B > 3:
        slots[3] = B + 4                                    # out of range: padded as well
        padded[3] = True
    keep = ~padded.to(DEV)
    slots = slots.to(DEV)
    rows = slots[keep].long()
    ref = rec_ref(x[:, None][keep], ga[:, None][keep], gi[:, None][keep], decay, 8.0, state[rows], None, None)
    out = torch.full_like(state, 7.0)
    y = blocks.linrec_step(x, ga, gi, decay, state, slots=slots, state_out=out)
    close("y", y[keep], ref["y"][0][:, 0], ref["y"][1][:, 0])
    assert not y[~keep].any()
    close("state", out[rows], *ref["h_last"])
    rest = torch.ones(B + 4, dtype=torch.bool, device=DEV)
    rest[rows] = False
    assert (out[rest] == 7.0).all()


def test_linrec_step_rows_of_one_slot_are_consecutive_steps():
    B, D = 150, 20
    x, ga, gi, decay, state = rnd(B, D, seed=80), rnd(B, D, seed=81), rnd(B, D, seed=82), rnd(D, seed=83) - 3, rnd(4, D, seed=84)
    slots = torch.randint(0, 3, (B,), generator=torch.Generator().manual_seed(3)).to(torch.int32)
    slots[77] = -1
    st = state.clone()
    y = blocks.linrec_step(x, ga, gi, decay, st, slots=slots.to(DEV))
    for s in range(3):
        rows = (slots == s).nonzero()[:, 0].to(DEV)
        yy, hh, _ = blocks.linrec_forward(x[rows][None], ga[rows][None], gi[rows][None], decay, h0=state[s][None])
        ref = rec_ref(x[rows][None], ga[rows][None], gi[rows][None], decay, 8.0, state[s][None], None, None)
        close("y", y[rows], ref["y"][0][0], ref["y"][1][0])
        close("state", st[s][None], *ref["h_last"])
        close("y of the episode", yy, *ref["y"])
    assert torch.equal(st[3], state[3]) and not y[77].any()


def test_linrec_autograd_and_differences():
    """the autograd function's gradients against central differences in 64 bits of the definition"""
    args, kw = rec_case(2, 9, 0, 5, F32, seed=91)
    x, ga, gi, decay = args
    wy, wh = rnd(2, 9, 5, seed=95), rnd(2, 5, seed=96)
    leaves = [t.clone().requires_grad_(True) for t in (x, ga, gi, decay, kw["h0"])]
    y, h = blocks.linear_recurrence(*leaves[:4], h0=leaves[4], reset=kw["reset"], lengths=kw["lengths"])
    ((y * wy).sum() + (h * wh).sum()).backward()

    def loss(ts):
        r = rec_ref(*ts[:4], 8.0, ts[4], kw["reset"], kw["lengths"])
        return float((r["y"][0] * wy).sum() + (r["h_last"][0] * wh).sum())
    base = [t.detach().double() for t in leaves]
    for i, leaf in enumerate(leaves):
        d = rnd(*leaf.shape, seed=97 + i).double()
        e = 1e-5
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + e * d, base[i] - e * d
        want = (loss(hi) - loss(lo)) / (2 * e)
        got = float((leaf.grad.double() * d).sum())
        assert abs(got - want) <= 1e-5 * (leaf.grad.double().abs() * d.abs()).sum().item() + 1e-8, (i, got, want)
    # only the state's gradient; only one leaf asked for
    x1 = x.clone().requires_grad_(True)
    y, h = blocks.linear_recurrence(x1, ga, gi, decay, h0=kw["h0"])
    (gx,) = torch.autograd.grad((h * wh).sum(), [x1])
    ref = rec_ref(x, ga, gi, decay, 8.0, kw["h0"], None, None, torch.zeros_like(x), wh)
    close("dx", gx, *ref["dx"])
    with torch.no_grad():
        y2, _ = blocks.linear_recurrence(x1, ga, gi, decay, h0=kw["h0"])
    assert torch.equal(y, y2) and not y2.requires_grad


# ------------------------------------------------------------------------------------- norms, gate and residual scale
def norm_ref(x, o, g, wp, sc, wq, alpha, eps, mask, dy=None, dn=None):
    """values and majorants. K = 96: a mean of squares passes 16 sequential and 10 tree additions (32 in the widest rows), the root, the
    gate (|argument| + 4) and the products around them the rest; the second mean and its root count again on the way to the gradients."""
    D = x.shape[-1]
    x = x.double().reshape(-1, D)
    N = x.shape[0]
    z = torch.zeros_like(x)
    one = torch.ones(D, dtype=torch.float64, device=x.device)
    gone = torch.zeros(N, 1, dtype=torch.bool, device=x.device) if mask is None else mask.reshape(-1, 1).bool()
    clean = lambda t: z if t is None else torch.where(gone, z, t.double().reshape(-1, D))
    wp, sc, wq = (one if w is None else w.double() for w in (wp, sc, wq))
    x, oo = torch.where(gone, z, x), clean(o)
    sg = 1.0 if g is None else torch.sigmoid(clean(g))
    K = 96 + (0 if g is None else clean(g).abs().amax().item() if N else 0)
    ro = 1 / torch.sqrt((oo * oo).mean(1, keepdim=True) + eps)
    oh = oo * ro
    v = sc * sg * oh * wp
    y = alpha * x + v
    My = (alpha * x).abs() + v.abs()
    ry = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
    yh = y * ry
    rel = ((My * y.abs()).mean(1, keepdim=True)) * ry * ry         # relative error of the root, in units of K U
    Mh = My * ry + yh.abs() * (1 + rel)
    hide = lambda t: torch.where(gone, torch.zeros_like(t), t)
    out = {"y": (hide(y), K * U * My), "n": (hide(yh * wq), K * U * Mh * wq.abs())}
    if dy is None and dn is None:
        return out
    dy, dn = clean(dy), clean(dn)
    e = dn * wq
    m, Mm = (e * yh).mean(1, keepdim=True), (e.abs() * Mh).mean(1, keepdim=True)
    d = dy + ry * (e - yh * m)
    Md = dy.abs() + ry * (1 + rel) * (e.abs() + 2 * Mh * Mm + yh.abs() * Mm)
    f, Mf = d * sc * sg, Md * (sc * sg).abs()
    e2, Me2 = f * wp, Mf * wp.abs()
    m2, Mm2 = (e2 * oh).mean(1, keepdim=True), (Me2 * oh.abs()).mean(1, keepdim=True)
    out["dx"] = (alpha * d, K * U * abs(alpha) * Md)
    if o is not None:
        out["do"] = (ro * (e2 - oh * m2), 2 * K * U * ro * (Me2 + oh.abs() * Mm2))
    if g is not None:
        out["dgate"] = (f * oh * wp * (1 - sg), 2 * K * U * Mf * (oh * wp).abs())
    adds = 64 + N / 64 + 64                                            # rows of a workgroup, then the partial rows
    for name, t, M in (("dpost_weight", f * oh, Mf * oh.abs()), ("dres_scale", d * sg * oh * wp, Md * (sg * oh * wp).abs()), ("dpre_weight", dn * yh, dn.abs() * Mh)):
        out[name] = (t.sum(0), (2 * K + adds) * U * M.sum(0))
    return out


def norm_check(x, o, g, wp, sc, wq, alpha=1.0, eps=1e-6, mask=None, use_dy=True, use_dn=True, seed=7):
    kw = dict(post_weight=wp, res_scale=sc, pre_weight=wq, alpha=alpha, eps=eps, row_mask=mask)
    dy = rnd(*x.shape, seed=seed, dtype=x.dtype) if use_dy else None
    dn = rnd(*x.shape, seed=seed + 1, dtype=x.dtype) if use_dn else None
    y, n = blocks.norm_gate_forward(x, o, g, **kw)
    y1, _ = blocks.norm_gate_forward(x, o, g, want_n=False, **kw)
    _, n1 = blocks.norm_gate_forward(x, o, g, want_y=False, **kw)
    assert torch.equal(y, y1) and torch.equal(n, n1)
    r = blocks.norm_gate_backward(dy, dn, x, o, g, **kw)
    r2 = blocks.norm_gate_backward(dy, dn, x, o, g, **kw)
    assert all((p is None and q is None) or torch.equal(p, q) for p, q in zip(r, r2))
    ref = norm_ref(x, o, g, wp, sc, wq, alpha, eps, mask, dy, dn)
    got = dict(y=y, n=n, **r._asdict())
    given = dict(do=o, dgate=g, dpost_weight=wp, dres_scale=sc, dpre_weight=wq)
    for k, v in got.items():
        if k in given and given[k] is None:
            assert v is None
            continue
        close(k, v.reshape(ref[k][0].shape), *ref[k])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D", [(1, 1), (3, 8), (70, 33), (9, 130), (5, 520), (3, 1500), (2, 2100), (2, 4100)])
def test_norm_gate_matches_the_definition(N, D, dtype):
    x, o, g = (rnd(N, D, seed=N + D + i, dtype=dtype) for i in range(3))
    wp, sc, wq = (1 + rnd(D, seed=N * D + i, scale=0.2) for i in range(3))
    mask = (torch.arange(N) % 3 == 1).to(torch.uint8).to(DEV)
    norm_check(x, o, g, wp, sc, wq, alpha=0.75, mask=mask)


@pytest.mark.parametrize("D", [8200, 16384])
def test_norm_gate_widest_rows(D):
    for dtype in (F32, F16):
        norm_check(*(rnd(2, D, seed=i, dtype=dtype) for i in range(3)), *(1 + rnd(D, seed=5 + i, scale=0.2) for i in range(3)))


@pytest.mark.parametrize("has_o,has_g,weights,use_dy,use_dn", [(0, 0, 1, 1, 1), (1, 0, 1, 1, 1), (1, 1, 0, 1, 1), (1, 1, 1, 0, 1), (1, 1, 1, 1, 0), (0, 0, 0, 0, 1)])
def test_norm_gate_optional_parts(has_o, has_g, weights, use_dy, use_dn):
    N, D = 21, 48
    o, g = rnd(N, D, seed=2) if has_o else None, rnd(N, D, seed=3) if has_g else None
    ws = [1 + rnd(D, seed=4 + i, scale=0.2) if weights else None for i in range(3)]
    norm_check(rnd(N, D, seed=1), o, g, *ws, use_dy=bool(use_dy), use_dn=bool(use_dn))


def test_norm_gate_shapes_strides_and_masked_rows():
    """agents' rows [B, T, na, D] cut out of a wider projection; rows that the mask leaves out hold NaN and Inf; every row masked; none"""
    B, T, na, D = 2, 3, 5, 12
    wide = rnd(B, T, na, 3 * D + 1, seed=1, dtype=BF16)
    x, o, g = (wide[..., i * D + 1:(i + 1) * D + 1] for i in range(3))
    mask = (torch.rand(B, T, na, generator=torch.Generator().manual_seed(2)) < 0.5).to(DEV)
    wide[mask] = math.nan
    wide[0, 0, 0] = math.inf
    mask[0, 0, 0] = True
    ws = [1 + rnd(D, seed=4 + i, scale=0.2) for i in range(3)]
    norm_check(x, o, g, *ws, mask=mask)
    y, n = blocks.norm_gate_forward(x, o, g, post_weight=ws[0], row_mask=torch.ones_like(mask))
    assert not y.any() and not n.any()
    e = torch.empty(0, D, device=DEV)
    y, n = blocks.norm_gate_forward(e, e, e)
    r = blocks.norm_gate_backward(e, e, e, e, e, post_weight=ws[0], pre_weight=ws[2])
    assert y.shape == n.shape == r.dx.shape == (0, D) and not r.dpost_weight.any() and not r.dpre_weight.any()


def test_norm_gate_many_rows():
    """more rows than the backward has workgroups: a workgroup walks several, the last round is ragged"""
    norm_check(*(rnd(5003, 9, seed=i) for i in range(3)), *(1 + rnd(9, seed=5 + i, scale=0.2) for i in range(3)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [2100, 4100, 6001])
def test_norm_gate_wide_rows_in_several_rounds(D, dtype):
    """a workgroup passes over several wide rows; some of them masked (a few rows on the emulator)"""
    N = 700 if DEV == "cuda" else 3
    x, o, g = (rnd(N, D, seed=s, dtype=dtype) for s in (1, 2, 3))
    norm_check(x, o, g, 1 + 0.1 * rnd(D, seed=4), rnd(D, seed=5), 1 + 0.1 * rnd(D, seed=6), alpha=0.9, mask=(rnd(N, seed=7) > 0.8).to(torch.uint8))


def test_norm_gate_zero_rows_and_gate_ends():
    """rows of zeros (the root is eps alone), gates at +-inf and at the type's lowest value"""
    N, D = 6, 16
    x, o, g = rnd(N, D, seed=1), rnd(N, D, seed=2), rnd(N, D, seed=3)
    x[0], o[0], o[1] = 0, 0, 0
    g[2], g[3], g[4] = -math.inf, math.inf, torch.finfo(F32).min
    y, n = blocks.norm_gate_forward(x, o, g, eps=1e-5)
    r = blocks.norm_gate_backward(rnd(N, D, seed=4), rnd(N, D, seed=5), x, o, g, eps=1e-5)
    ref = norm_ref(x, o, g.clamp(-200, 200), None, None, None, 1.0, 1e-5, None, rnd(N, D, seed=4), rnd(N, D, seed=5))
    for k, v in dict(y=y, n=n, dx=r.dx, do=r.do, dgate=r.dgate).items():
        close(k, v, *ref[k])
    assert torch.equal(y[2], x[2]) and torch.equal(y[4], x[4])


def test_norm_gate_autograd_and_differences():
    N, D = 4, 11
    leaves = [rnd(N, D, seed=i).requires_grad_(True) for i in range(3)] + [(1 + rnd(D, seed=5 + i, scale=0.2)).requires_grad_(True) for i in range(3)]
    a, b = rnd(N, D, seed=20), rnd(N, D, seed=21)
    y, n = blocks.norm_gate_residual(*leaves[:3], post_weight=leaves[3], res_scale=leaves[4], pre_weight=leaves[5], alpha=0.9)
    ((y * a).sum() + (n * b).sum()).backward()

    def loss(t):
        r = norm_ref(*t, 0.9, 1e-6, None)
        return float((r["y"][0] * a).sum() + (r["n"][0] * b).sum())
    base = [t.detach().double() for t in leaves]
    for i, leaf in enumerate(leaves):
        d = rnd(*leaf.shape, seed=30 + i).double()
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        want, got = (loss(hi) - loss(lo)) / 2e-5, float((leaf.grad.double() * d).sum())
        assert abs(got - want) <= 1e-5 * (leaf.grad.double().abs() * d.abs()).sum().item() + 1e-8, (i, got, want)
    none, n = blocks.norm_gate_residual(leaves[0].detach(), pre_weight=leaves[5])
    assert none is None and n.requires_grad


# ------------------------------------------------------------------------------------------------ gated feed-forward block
def act_ref(act, g):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    a, b = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(a * (g + b * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * b * g * g)


def ff_ref(x, wg, wu, bg, bu, act, dh=None):
    """values and majorants. A dot product of n terms in fp32: at most (n + 16) U of the sum of magnitudes (16: the split's dropped terms
    and the last roundings). |act'| <= 1.13, |act''| <= 1.2; the gates' sigmoids cost (3 |g| + 3 |g|^3 / 10 + 8) U of the value. The
    backward starts from pre-activations rounded to the type (half a step of each), and in 16 bits the gradients of the two
    pre-activations are rounded to it once more before the products."""
    F, D = wg.shape
    half = 0.0 if x.dtype == F32 else torch.finfo(x.dtype).eps / 2
    x2, wg2, wu2 = x.double().reshape(-1, D), wg.double(), wu.double()
    z = torch.zeros(F, dtype=torch.float64, device=x.device)
    b0, b1 = (z if b is None else b.double() for b in (bg, bu))
    g, u = x2 @ wg2.t() + b0, x2 @ wu2.t() + b1
    Eg, Eu = (D + 16) * U * (x2.abs() @ wg2.abs().t() + b0.abs()), (D + 16) * U * (x2.abs() @ wu2.abs().t() + b1.abs())
    f, df = act_ref(act, g)
    Ka = (3 * g.abs() + 0.3 * g.abs() ** 3 + 8) * U
    out = {"h": (f * u, 1.13 * Eg * u.abs() + (f.abs() + 1.13 * Eg) * Eu + (Ka + 2 * U) * (f * u).abs())}
    if dh is None:
        return out
    d = dh.double().reshape(-1, F)
    Rg, Ru = Eg + (half + U) * (g.abs() + Eg), Eu + (half + U) * (u.abs() + Eu)
    dg, du = d * u * df, d * f
    Kd = Ka * (1 + g.abs())
    Edg = d.abs() * ((u.abs() + Ru) * (1.2 * Rg + Kd) + Ru * df.abs()) + 4 * U * dg.abs()
    Edu = d.abs() * (1.13 * Rg + Ka * f.abs()) + 4 * U * du.abs()
    tiny = 0.0 if x.dtype == F32 else torch.finfo(x.dtype).tiny * 2 * half
    Edg, Edu = Edg + half * (dg.abs() + Edg) + tiny, Edu + half * (du.abs() + Edu) + tiny
    N = x2.shape[0]
    k = (2 * F + 16) * U
    out["dx"] = (dg @ wg2 + du @ wu2, Edg @ wg2.abs() + Edu @ wu2.abs() + k * (dg.abs() @ wg2.abs() + du.abs() @ wu2.abs()))
    k = (N + 16) * U
    out["dwg"] = (dg.t() @ x2, Edg.t() @ x2.abs() + k * (dg.abs().t() @ x2.abs()))
    out["dwu"] = (du.t() @ x2, Edu.t() @ x2.abs() + k * (du.abs().t() @ x2.abs()))
    out["dbg"] = (dg.sum(0), (Edg + k * dg.abs()).sum(0))
    out["dbu"] = (du.sum(0), (Edu + k * du.abs()).sum(0))
    return out


def ff_check(x, wg, wu, bg, bu, act, seed=11):
    F = wg.shape[0]
    dh = rnd(*x.shape[:-1], F, seed=seed, dtype=x.dtype)
    h, saved = blocks.gated_ff_forward(x, wg, wu, bg, bu, act=act, save=True)
    h2, none = blocks.gated_ff_forward(x, wg, wu, bg, bu, act=act)
    assert none is None and torch.equal(h, h2)
    r = blocks.gated_ff_backward(dh, x, wg, wu, saved, act=act, bias=bg is not None)
    r2 = blocks.gated_ff_backward(dh, x, wg, wu, saved, act=act, bias=bg is not None)
    assert all((p is None and q is None) or torch.equal(p, q) for p, q in zip(r, r2))
    ref = ff_ref(x, wg, wu, bg, bu, act, dh)
    for k, v in dict(h=h, dx=r[0], dwg=r[1], dwu=r[2], dbg=r[3], dbu=r[4]).items():
        if v is None:
            assert bg is None and k in ("dbg", "dbu")
            continue
        close(k, v.reshape(ref[k][0].shape), *ref[k])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,F,act,bias", [(1, 1, 1, "silu", True), (3, 64, 32, "gelu", False), (17, 72, 50, "silu", True), (64, 33, 65, "gelu", True),
                                            (65, 64, 128, "silu", False), (130, 70, 131, "gelu", True), (200, 128, 40, "silu", False)])
def test_gated_ff_matches_the_definition(N, D, F, act, bias, dtype):
    x = rnd(N, D, seed=N + D, dtype=dtype)
    wg, wu = rnd(F, D, seed=1, dtype=dtype, scale=D ** -0.5), rnd(F, D, seed=2, dtype=dtype, scale=D ** -0.5)
    bg, bu = (rnd(F, seed=3, dtype=dtype), rnd(F, seed=4, dtype=dtype)) if bias else (None, None)
    ff_check(x, wg, wu, bg, bu, act)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gated_ff_large_tiles(dtype):
    """enough tiles for the 256 x 256 variant of every product, ragged in rows and columns (fewer compute units on the emulator, fewer tiles)"""
    N, D, F = (2060, 2056, 2052) if DEV == "cuda" else (520, 264, 300)
    K = 64
    x, wg, wu = rnd(N, K, seed=1, dtype=dtype), rnd(F, K, seed=2, dtype=dtype, scale=0.1), rnd(F, K, seed=3, dtype=dtype, scale=0.1)
    h, _ = blocks.gated_ff_forward(x, wg, wu)
    close("h", h, *ff_ref(x, wg, wu, None, None, "silu")["h"])
    F = 72                                                          # dx: N x D
    x, wg, wu = rnd(N, D, seed=4, dtype=dtype), rnd(F, D, seed=5, dtype=dtype, scale=0.02), rnd(F, D, seed=6, dtype=dtype, scale=0.02)
    ff_check(x, wg, wu, None, None, "gelu")
    N, F = 70, (1030 if DEV == "cuda" else 260)                    # dw: 2 F x D
    x, wg, wu = rnd(N, D, seed=7, dtype=dtype), rnd(F, D, seed=8, dtype=dtype, scale=0.02), rnd(F, D, seed=9, dtype=dtype, scale=0.02)
    ff_check(x, wg, wu, rnd(F, seed=10, dtype=dtype), rnd(F, seed=11, dtype=dtype), "silu")


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_ff_whole_rounds_of_tiles(dtype):
    """rows and columns whose 128-row tiles fill the compute units evenly (the shorter tiles would not), forward and dx; the ragged middle; odd
    widths, and rows shorter than a 16-byte load, in as many tiles"""
    k = 1 if DEV == "cuda" else 8
    for N, D, F in ((1024 // k, 64, 1920 // k), (1024 // k, 3840 // k, 64), (1400 // k, 72, 1920 // k), (700 // k, 37, 1000), (700 // k, 5, 1000), (700 // k, 3, 1001)):
        x, wg, wu = rnd(N, D, seed=1, dtype=dtype), rnd(F, D, seed=2, dtype=dtype, scale=D ** -0.5), rnd(F, D, seed=3, dtype=dtype, scale=D ** -0.5)
        ff_check(x, wg, wu, rnd(F, seed=4, dtype=dtype), rnd(F, seed=5, dtype=dtype), "silu")


def test_gated_ff_shapes_and_strides():
    """agents' rows [B, T, na, D] cut out of wider rows, both weights in one fused matrix with padding, one bias alone, rows expanded over one"""
    D, F = 24, 20
    wide = rnd(2, 5, 3, D + 7, seed=1)
    both = rnd(2 * F, D + 3, seed=2, scale=0.2)
    x, wg, wu = wide[..., 5:5 + D], both[:F, 2:2 + D], both[F:, 2:2 + D]
    ff_check(x, wg, wu, None, None, "silu")
    b = rnd(F, seed=3)
    h, _ = blocks.gated_ff_forward(x, wg, wu, None, b)
    close("h", h.reshape(-1, F), *ff_ref(x, wg, wu, None, b, "silu")["h"])
    row = rnd(1, D, seed=4).expand(9, D)
    close("h", blocks.gated_ff(row, wg, wu), *ff_ref(row, wg, wu, None, None, "silu")["h"])
    e = torch.empty(0, D, device=DEV)
    h, saved = blocks.gated_ff_forward(e, wg, wu, save=True)
    dx, dwg, dwu, dbg, dbu = blocks.gated_ff_backward(h, e, wg, wu, saved, bias=True)
    assert h.shape == (0, F) and dx.shape == (0, D) and not dwg.any() and not dwu.any() and not dbg.any() and not dbu.any()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,D", [(5, 130), (40, 131), (70, 192)])
def test_gated_ff_rows_that_begin_inside_words(N, D, dtype):
    """16-bit rows at addresses that are no multiple of four: slices from an odd column on, odd and even strides, inputs alone and weights alone"""
    F = 24
    for off, pad in ((1, 0), (1, 2), (0, 1), (3, 3)):
        x = rnd(N, off + D + pad, seed=1, dtype=dtype)[:, off:off + D]
        both = rnd(2 * F, off + D + pad, seed=2, dtype=dtype, scale=0.2)[:, off:off + D]
        ff_check(x, both[:F], both[F:], None, None, "silu")
        ff_check(x, both[:F].contiguous(), both[F:].contiguous(), None, None, "gelu")
        ff_check(x.contiguous(), both[:F], both[F:], None, None, "silu")


def test_gated_ff_rows_do_not_mix():
    """a NaN row spoils its own row of h and dx alone"""
    x, wg, wu = rnd(100, 40, seed=1), rnd(30, 40, seed=2, scale=0.2), rnd(30, 40, seed=3, scale=0.2)
    h0, _ = blocks.gated_ff_forward(x, wg, wu)
    x[41] = math.nan
    h, saved = blocks.gated_ff_forward(x, wg, wu, save=True)
    keep = torch.arange(100, device=DEV) != 41
    assert torch.isnan(h[41]).all() and torch.equal(h[keep], h0[keep])
    dx = blocks.gated_ff_backward(rnd(100, 30, seed=4), x, wg, wu, saved)[0]
    assert torch.isnan(dx[41]).all() and torch.isfinite(dx[keep]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,F", [(130, 72), (70, 130)])
def test_gated_ff_an_infinite_last_row_stays_where_it_is(N, F, dtype):
    """the last row of a weight / of x is Inf, the tiles read whole 64-blocks of rows behind it: what it does not touch stays finite, and a
    zero in front of it alone makes a NaN"""
    D = 64
    x, wg, wu = rnd(N, D, seed=1, dtype=dtype), rnd(F, D, seed=2, dtype=dtype, scale=0.1), rnd(F, D, seed=3, dtype=dtype, scale=0.1)
    h, saved = blocks.gated_ff_forward(x, wg, wu, save=True)
    dh = rnd(N, F, seed=4, dtype=dtype)
    wi = wu.clone()
    wi[-1, 5] = math.inf
    dx = blocks.gated_ff_backward(dh, x, wg, wi, saved)[0]
    clean = blocks.gated_ff_backward(dh, x, wg, wu, saved)[0]
    others = torch.arange(D, device=DEV) != 5
    assert torch.equal(dx[:, others], clean[:, others]) and torch.isinf(dx[:, 5]).all()
    xi = x.clone()
    xi[-1, 7] = -math.inf
    _, dwg, dwu, _, _ = blocks.gated_ff_backward(dh, xi, wg, wu, saved)
    _, cg, cu, _, _ = blocks.gated_ff_backward(dh, x, wg, wu, saved)
    others = torch.arange(D, device=DEV) != 7
    assert torch.equal(dwg[:, others], cg[:, others]) and torch.equal(dwu[:, others], cu[:, others])
    assert torch.isinf(dwg[:, 7]).all() and torch.isinf(dwu[:, 7]).all()


def test_gated_ff_autograd_and_differences():
    N, D, F = 5, 8, 6
    leaves = [t.requires_grad_(True) for t in (rnd(N, D, seed=1), rnd(F, D, seed=2), rnd(F, D, seed=3), rnd(F, seed=4), rnd(F, seed=5))]
    w = rnd(N, F, seed=6)
    (blocks.gated_ff(*leaves, act="gelu") * w).sum().backward()
    base = [t.detach().double() for t in leaves]
    for i, leaf in enumerate(leaves):
        d = rnd(*leaf.shape, seed=10 + i).double()
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        want = float(((ff_ref(*hi, "gelu")["h"][0] - ff_ref(*lo, "gelu")["h"][0]) * w).sum()) / 2e-5
        got = float((leaf.grad.double() * d).sum())
        assert abs(got - want) <= 1e-5 * (leaf.grad.double().abs() * d.abs()).sum().item() + 1e-8, (i, got, want)


def step_of(v, t):
    """distance of the numbers of type t around v (its subnormal step aside)"""
    return torch.where(v == 0, 0.0, t.eps * torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(1e-300)))))


def ff_ref16(x, wg, wu, bg, bu, act, dh, keep=None):
    """The backward of 16-bit inputs: values, error majorants and, for dx and the weight gradients, the variance of what the roundings do.

    It starts from fp32 pre-activations. dg and du, the gradients of the two, are exact to fp32 errors Edg, Edu where the bias gradients sum them;
    the products read them rounded to the type, off by half a step of the value, and in fp16 by half a subnormal step S / 2 = 2^-25 R more: R is 1
    while the largest |dg|, |du| lies in [1, 61440), else the power of two that brings it into [2^14, 2^15). A rounding error is uniform in
    half a step to either side, independent from element to element: its variance is step^2 / 12. `keep` makes the reference wrong: what it does to
    its pre-activations."""
    F, D = wg.shape
    t = torch.finfo(x.dtype)
    half = t.eps / 2
    x2, wg2, wu2 = x.double().reshape(-1, D), wg.double(), wu.double()
    z = torch.zeros(F, dtype=torch.float64, device=x.device)
    b0, b1 = (z if b is None else b.double() for b in (bg, bu))
    g, u = x2 @ wg2.t() + b0, x2 @ wu2.t() + b1
    if keep is not None:
        g, u = keep(g), keep(u)
    Eg, Eu = (D + 16) * U * (x2.abs() @ wg2.abs().t() + b0.abs()), (D + 16) * U * (x2.abs() @ wu2.abs().t() + b1.abs())
    f, df = act_ref(act, g)
    Ka = (3 * g.abs() + 0.3 * g.abs() ** 3 + 8) * U
    d = dh.double().reshape(-1, F)
    dg, du = d * u * df, d * f
    Edg = d.abs() * ((u.abs() + Eu) * (1.2 * Eg + Ka * (1 + g.abs())) + Eu * df.abs()) + 4 * U * dg.abs()
    Edu = d.abs() * (1.13 * Eg + Ka * f.abs()) + 4 * U * du.abs()
    N = x2.shape[0]
    k = (N + 16) * U
    out = {"dbg": (dg.sum(0), (Edg + k * dg.abs()).sum(0)), "dbu": (du.sum(0), (Edu + k * du.abs()).sum(0))}
    S = 0.0
    if x.dtype == F16:
        top = max(float(dg.abs().max()), float(du.abs().max()))
        R = 1.0 if 1 <= top < 61440 else 2.0 ** (math.floor(math.log2(top)) - 14)
        S = 2.0 ** -24 * R * (2 if abs(math.log2(top) - round(math.log2(top))) < 1e-5 else 1)       # (the fp32 value may sit on the other side of a power)
    out["S"] = S
    Rg, Ru = Edg + half * (dg.abs() + Edg) + S / 2, Edu + half * (du.abs() + Edu) + S / 2
    vg, vu = (step_of(dg, t) ** 2 + S * S) / 12, (step_of(du, t) ** 2 + S * S) / 12
    kx = (2 * F + 16) * U
    dx = dg @ wg2 + du @ wu2
    out["dx"] = (dx, Rg @ wg2.abs() + Ru @ wu2.abs() + kx * (dg.abs() @ wg2.abs() + du.abs() @ wu2.abs()))
    var = {"dx": vg @ wg2 ** 2 + vu @ wu2 ** 2}
    for name, v, R_, va in (("dwg", dg, Rg, vg), ("dwu", du, Ru, vu)):
        out[name] = (v.t() @ x2, R_.t() @ x2.abs() + k * (v.abs().t() @ x2.abs()))
        var[name] = va.t() @ x2 ** 2
    out["var"] = {n: var[n] + (step_of(out[n][0], t) ** 2 + (t.tiny * t.eps) ** 2) / 12 for n in var}        # (the last rounding, its subnormal step)
    return out


def close_or_inf(name, got, want, fp32_error):
    """close(), and where the value itself lies outside the type: Inf of its sign. Rounding to nearest gives Inf from the largest number and half a
    step on (fp16: 65520), so an Inf is right if the value may reach that, and a number is if it may stay below"""
    t = torch.finfo(got.dtype)
    edge = t.max * (1 + t.eps / 4)                  # (its last step is max eps / (2 - eps); half of it is max eps / 4 or a little more)
    inf = torch.isinf(got)
    assert (inf <= (want.abs() + fp32_error >= edge)).all() and (torch.sign(got) == torch.sign(want))[inf].all(), f"{name}: Inf where the value is in range"
    assert (inf >= (want.abs() - fp32_error >= edge * (1 + t.eps))).all(), f"{name}: a number where the value is out of range"
    close(name, torch.where(inf, 0, got), torch.where(inf, 0.0, want), torch.where(inf, 0.0, fp32_error))


def ff_check16(x, wg, wu, bg, bu, act, dh, keep=None):
    """every gradient inside its majorant, and the errors of dx, dw_gate and dw_up no larger in the mean square than the roundings' variance. The mean
    of n squares of a normal variable strays by sqrt(2 / n), n the fewer of the elements and the roundings behind them: six of those, and a tenth for
    steps that are not quite uniform. (fp32 arithmetic adds next to nothing: its roundings are at most 2^-12 of these, K <= 1200 of them to a sum, each of
    a running sum no larger than the root of the summed squares: K 2^-24 of the variance.)"""
    (N, D), F = x.shape, wg.shape[0]
    _, saved = blocks.gated_ff_forward(x, wg, wu, bg, bu, act=act, save=True)
    got = dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), blocks.gated_ff_backward(dh, x, wg, wu, saved, act=act, bias=bg is not None)))
    ref = ff_ref16(x, wg, wu, bg, bu, act, dh, keep)
    for k, v in got.items():
        if v is not None:
            close_or_inf(k, v.reshape(ref[k][0].shape), *ref[k])
    for k in ("dx", "dwg", "dwu"):
        err = got[k].double().reshape(ref[k][0].shape) - ref[k][0]
        fits = torch.isfinite(got[k].reshape(ref[k][0].shape))
        ratio = float((err ** 2 / ref["var"][k])[fits].mean())
        n = N * min(D, 2 * F) if k == "dx" else F * min(D, N)
        assert ratio <= 1.1 + 6 * math.sqrt(2 / n), f"{k}: the mean square error is {ratio:.3g} of the roundings'"


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("N,D,F", [(128, 512, 64), (130, 512, 512), (70, 33, 131)])
@pytest.mark.parametrize("scale", [1e4, 1.0, 1e-3, 3e-6, 1e-7])
def test_gated_ff_half_gradients_over_the_types_range(scale, N, D, F, act):
    """dh as loss scaling makes it, and down to subnormal numbers: the gradients of the pre-activations, which lie outside fp16 on the way, neither
    overflow nor lose digits"""
    x = rnd(N, D, seed=N + D, dtype=F16)
    wg, wu = rnd(F, D, seed=1, dtype=F16, scale=D ** -0.5), rnd(F, D, seed=2, dtype=F16, scale=D ** -0.5)
    ff_check16(x, wg, wu, rnd(F, seed=3, dtype=F16), rnd(F, seed=4, dtype=F16), act, rnd(N, F, seed=5, dtype=F16, scale=scale))


def test_gated_ff_half_gradients_beside_infinities_and_zeros():
    """an Inf in dh spoils its own row of dx, not the scale of the others; gradients that are all zero give zeros"""
    N, D, F = 40, 64, 96
    x, wg, wu = rnd(N, D, seed=1, dtype=F16), rnd(F, D, seed=2, dtype=F16, scale=0.1), rnd(F, D, seed=3, dtype=F16, scale=0.1)
    _, saved = blocks.gated_ff_forward(x, wg, wu, save=True)
    dh = rnd(N, F, seed=4, dtype=F16, scale=1e-6)
    clean = blocks.gated_ff_backward(dh, x, wg, wu, saved)[0]
    dh[7, 3] = math.inf
    dx = blocks.gated_ff_backward(dh, x, wg, wu, saved)[0]
    keep = torch.arange(N, device=DEV) != 7
    assert not torch.isfinite(dx[7]).any() and torch.equal(dx[keep], clean[keep])
    r = blocks.gated_ff_backward(torch.zeros_like(dh), x, wg, wu, saved, bias=True)
    assert not any(t.any() for t in r)


@pytest.mark.parametrize("N,D,F", [(3, 32, 20), (65, 32, 40), (1100, 40, 900), (130, 33, 31)])
def test_gated_ff_largest_fp32_numbers(N, D, F):
    """operands up to the largest fp32 number, whose leading 16-bit piece must not round to Inf: x in front of small weights (few rows, fragments, tiles),
    then weights and x in the backward's products. (1e-30: all three pieces of a weight are normal numbers)"""
    if DEV == "cpu":
        N, F = min(N, 260), min(F, 200)
    top = torch.finfo(F32).max
    x, wg, wu = rnd(N, D, seed=1), rnd(F, D, seed=2, scale=1e-30), rnd(F, D, seed=3, scale=1e-39 ** 0.5)
    x[:, ::3], x[0], x[-1, 1::3] = top, -3.4e38, 3.3962e38
    h, saved = blocks.gated_ff_forward(x, wg, wu, save=True)
    assert torch.isfinite(h).all()
    close("h", h, *ff_ref(x, wg, wu, None, None, "silu")["h"])
    # dw: x as large against small gradients; dx: weights as large against them
    a, b = rnd(F, D, seed=4), rnd(F, D, seed=5)
    saved = torch.stack([rnd(N, F, seed=6), rnd(N, F, seed=7)])
    dh = rnd(N, F, seed=8, scale=1e-6)
    g, u = saved[0].double(), saved[1].double()
    f, df = act_ref("silu", g)
    dg, du = dh.double() * u * df, dh.double() * f
    E = (3 * g.abs() + 16) * U * (1 + g.abs()) * dh.double().abs() * (1 + u.abs())
    a[:, ::4], b[1] = top, -top
    dx, dwg, dwu, _, _ = blocks.gated_ff_backward(dh, x, a, b, saved)
    A, B, X = a.double(), b.double(), x.double()
    close("dx", dx, dg @ A + du @ B, E @ (A.abs() + B.abs()) + (2 * F + 16) * U * (dg.abs() @ A.abs() + du.abs() @ B.abs()))
    for name, got, v in (("dwg", dwg, dg), ("dwu", dwu, du)):
        close(name, got, v.t() @ X, E.t() @ X.abs() + (N + 16) * U * (v.abs().t() @ X.abs()))


# ------------------------------------------------------------------------------------------------ together
def block_pass(x, p, h0, lengths, row_mask, state=None):
    """norm -> recurrence -> norm, gate, residual -> gated feed-forward -> norm, gate, residual, as an agent would stack it; with `state` one
    acting step of it"""
    F = torch.nn.functional
    _, n = blocks.norm_gate_residual(x, pre_weight=p["w0"], row_mask=row_mask)
    ga, gi, g = F.linear(n, p["wa"]), F.linear(n, p["wi"]), F.linear(n, p["wgate"])
    if state is None:
        y, h = blocks.linear_recurrence(n, ga, gi, p["decay"], h0=h0, lengths=lengths)
    else:
        y, h = blocks.linrec_step(n, ga, gi, p["decay"], state), state
    x, n = blocks.norm_gate_residual(x, y, g, post_weight=p["w1"], res_scale=p["s1"], pre_weight=p["w2"], row_mask=row_mask)
    f = F.linear(blocks.gated_ff(n, p["wg"], p["wu"]), p["wd"])
    x, _ = blocks.norm_gate_residual(x, f, None, post_weight=p["w3"], res_scale=p["s3"], row_mask=row_mask)
    return x, h


def block_ref(x, p, h0, lengths, row_mask):
    F = torch.nn.functional
    live = (row_mask == 0).double()[..., None]
    nrm = lambda v, w: v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w
    n = nrm(x, p["w0"]) * live
    ga, gi, g = n @ p["wa"].t(), n @ p["wi"].t(), n @ p["wgate"].t()
    rate = 8.0 * F.softplus(p["decay"])
    h, ys = h0, []
    for t in range(x.shape[1]):
        a = torch.exp(-rate * torch.sigmoid(ga[:, t]))
        on = (t < lengths)[:, None, None]
        h = torch.where(on, a * h + torch.sqrt(1 - a * a) * torch.sigmoid(gi[:, t]) * n[:, t], h)
        ys.append(torch.where(on, h, torch.zeros_like(h)))
    x = (x + p["s1"] * torch.sigmoid(g) * nrm(torch.stack(ys, 1), p["w1"])) * live
    n = nrm(x, p["w2"]) * live
    f = (F.silu(n @ p["wg"].t()) * (n @ p["wu"].t())) @ p["wd"].t()
    return (x + p["s3"] * nrm(f, p["w3"])) * live, h


def block_params(D, F):
    p = {k: 1 + rnd(D, seed=i, scale=0.1) for i, k in enumerate(("w0", "w1", "s1", "w2", "w3", "s3"))}
    p["decay"] = rnd(D, seed=10) - 3
    for i, k in enumerate(("wa", "wi", "wgate")):
        p[k] = rnd(D, D, seed=11 + i, scale=D ** -0.5)
    p["wg"], p["wu"], p["wd"] = rnd(F, D, seed=15, scale=D ** -0.5), rnd(F, D, seed=16, scale=D ** -0.5), rnd(D, F, seed=17, scale=F ** -0.5)
    return p


def test_the_block_as_a_whole_trains_and_acts():
    """The three operators as one residual block of [B, T, n_agents, D]: outputs and every gradient against 64-bit torch, then the same
    episode acted step by step. Bound: the block is a chain of about 12 operators whose relative errors (some 100 U each, the majorants of
    the tests above) add up and are amplified by its Jacobians (norms of rows of order 1: O(1) each): 3e-5 of the largest value."""
    B, T, na, D, F = 3, 10, 2, 16, 24
    p = block_params(D, F)
    x, h0 = rnd(B, T, na, D, seed=30), rnd(B, na, D, seed=31)
    lengths = torch.tensor([T, 4, 7], dtype=torch.int32, device=DEV)
    mask = (torch.rand(B, T, na, generator=torch.Generator().manual_seed(4)) < 0.2).to(torch.uint8).to(DEV)
    names = sorted(p)
    leaves = [x.clone().requires_grad_(True), h0.clone().requires_grad_(True)] + [p[k].clone().requires_grad_(True) for k in names]
    out, h = block_pass(leaves[0], dict(zip(names, leaves[2:])), leaves[1], lengths, mask)
    wo, wh = rnd(*out.shape, seed=40), rnd(*h.shape, seed=41)
    grads = torch.autograd.grad((out * wo).sum() + (h * wh).sum(), leaves)
    l64 = [t.detach().double().requires_grad_(True) for t in leaves]
    out64, h64 = block_ref(l64[0], dict(zip(names, l64[2:])), l64[1], lengths, mask)
    g64 = torch.autograd.grad((out64 * wo.double()).sum() + (h64 * wh.double()).sum(), l64)
    for name, a, b in [("out", out, out64), ("h", h, h64)] + list(zip(["x", "h0"] + names, grads, g64)):
        assert (a.double() - b).abs().max() <= 3e-5 * b.abs().max(), (name, (a.double() - b).abs().max(), b.abs().max())
    with torch.no_grad():
        full, hT = block_pass(x, p, h0, None, mask)
        state, steps = h0.clone(), []
        for t in range(T):
            steps.append(block_pass(x[:, t], p, None, None, mask[:, t], state=state)[0])
        acted = torch.stack(steps, 1)
        assert (acted - full).abs().max() <= 3e-5 * full.abs().max() and (state - hT).abs().max() <= 3e-5 * hT.abs().max()


def test_forward_mode_derivatives_are_refused():
    """a tangent on any differentiable input raises, whether or not the input also requires a gradient; values without one pass, at any level"""
    fw = torch.autograd.forward_ad
    B, T, D, F = 2, 3, 8, 5
    seq, decay, h0, w = [rnd(B, T, D, seed=i) for i in range(3)], rnd(D, seed=3), rnd(B, D, seed=4), 1 + 0.1 * rnd(D, seed=5)
    wg, wu, b = rnd(F, D, seed=6), rnd(F, D, seed=7), rnd(F, seed=8)
    calls = [(lambda x, ga, gi, d, h: blocks.linear_recurrence(x, ga, gi, d, h0=h), [*seq, decay, h0]),
             (lambda x, o, g, a, c, e: blocks.norm_gate_residual(x, o, g, post_weight=a, res_scale=c, pre_weight=e), [*seq, w, w, w]),
             (lambda *a: blocks.gated_ff(*a), [seq[0], wg, wu, b, b]),
             (lambda x, ga, gi, d: blocks.linrec_step(x, ga, gi, d, h0.clone()), [seq[0][:, 0], seq[1][:, 0], seq[2][:, 0], decay])]
    for f, args in calls:
        for i in range(len(args)):
            for needs_grad in (False, True):
                with fw.dual_level(), torch.set_grad_enabled(needs_grad):
                    primal = args[i].clone().requires_grad_(needs_grad)
                    a = list(args)
                    a[i] = fw.make_dual(primal, torch.ones_like(primal))
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        f(*a)
                    f(*args)


def test_linrec_step_tells_torch_that_the_state_changed():
    """a graph that kept the state notices the step; state_out counts, a state that is only read does not; inference tensors have no counter"""
    B, D = 3, 8
    x, ga, gi, decay, state = rnd(B, D, seed=1), rnd(B, D, seed=2), rnd(B, D, seed=3), rnd(D, seed=4), rnd(B, D, seed=5)
    leaf = rnd(B, D, seed=6).requires_grad_(True)
    loss = (leaf * state).sum()
    before = state._version
    blocks.linrec_step(x, ga, gi, decay, state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    out = torch.empty_like(state)
    counts = state._version, out._version
    blocks.linrec_step(x, ga, gi, decay, state, state_out=out)
    assert state._version == counts[0] and out._version > counts[1]
    with torch.inference_mode():
        s = state.clone()
        y = blocks.linrec_step(x, ga, gi, decay, s)
    assert torch.equal(s, out) and not y.requires_grad


def test_linrec_step_refuses_inputs_that_require_a_gradient():
    """it has no backward: under no_grad parameters pass, elsewhere the call raises before anything is written"""
    B, D = 3, 8
    args = [rnd(B, D, seed=1), rnd(B, D, seed=2), rnd(B, D, seed=3), rnd(D, seed=4), rnd(B, D, seed=5)]
    for i in range(5):
        a = list(args)
        a[i] = args[i].clone().requires_grad_(True)
        keep = a[4].detach().clone()
        with pytest.raises(RuntimeError, match="linrec_step: .*no_grad"):
            blocks.linrec_step(*a)
        assert torch.equal(a[4], keep)
        with torch.no_grad():
            y = blocks.linrec_step(*a)
        assert not y.requires_grad and not torch.equal(a[4], keep)


def rec_plan(args, kw, backward):
    """(tiles of the time axis, chunks they are dealt to) of a call, from what it asks for: one state a tile and row is saved, two maps a chunk and row"""
    from refil_amd import _lib
    d = blocks._linrec_desc("rec_plan", *args, 8.0, kw["h0"], kw["reset"], kw["lengths"])
    row = d.B * d.C
    tiles = _lib.lib().refil_linrec_saved_floats(d) // row
    ws = _lib.lib().refil_linrec_workspace_bytes(d, backward) // 4
    sums = ws if not backward else ws - row                          # one chunk: no maps; the backward keeps a partial decay gradient a chunk
    return tiles, 1 if sums == 0 else ws // (3 * row if backward else 2 * row)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ragged", [True, False])
@pytest.mark.parametrize("B,T,D,chunks", [(200, 200, 3, "several"), (1100, 100, 4, "one"), (100, 200, 130, "several"), (40, 260, 300, "several"), (700, 150, 5, "any")])
def test_linrec_workgroups_that_walk_several_tiles(B, T, D, chunks, ragged, dtype):
    """the carry from tile to tile, the LDS halves in turn, loads into the next (backward: the previous) tile, chunks' maps over several tiles: the plan
    that a shape is here for is asserted"""
    args, kw = rec_case(B, T, 0, D, dtype, seed=B + T + D, ragged=ragged, decay_shift=-5.0)
    for backward in (0, 1):
        tiles, n = rec_plan(args, kw, backward)
        assert tiles > n and (n == 1 if chunks == "one" else n > 1 if chunks == "several" else True), (backward, tiles, n)
    rec_check(args, kw, dh_last=rnd(B, D, seed=9))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,D,F,act,bias", [(1, 1, 1, "silu", True), (3, 64, 32, "gelu", False), (17, 72, 50, "silu", True), (64, 33, 65, "gelu", True),
                                            (65, 64, 128, "silu", False), (130, 70, 131, "gelu", True), (200, 128, 40, "silu", False), (600, 200, 333, "silu", True)])
def test_gated_ff_backward_rounds_once_on_the_way(N, D, F, act, bias, dtype):
    """16-bit gradients inside bounds that know the pre-activations as fp32 and round nothing but dg and du in front of the products, and not even those
    in the bias gradients"""
    x = rnd(N, D, seed=N + D, dtype=dtype)
    wg, wu = rnd(F, D, seed=1, dtype=dtype, scale=D ** -0.5), rnd(F, D, seed=2, dtype=dtype, scale=D ** -0.5)
    bg, bu = (rnd(F, seed=3, dtype=dtype), rnd(F, seed=4, dtype=dtype)) if bias else (None, None)
    ff_check16(x, wg, wu, bg, bu, act, rnd(N, F, seed=5, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_those_bounds_notice_pre_activations_kept_in_16_bits(dtype):
    """the reference made wrong in that way (its own pre-activations rounded to the type) leaves the bounds, in the bias gradients and in the mean square"""
    N, D, F = 130, 70, 131
    x, dh = rnd(N, D, seed=N + D, dtype=dtype), rnd(N, F, seed=5, dtype=dtype)
    wg, wu = rnd(F, D, seed=1, dtype=dtype, scale=D ** -0.5), rnd(F, D, seed=2, dtype=dtype, scale=D ** -0.5)
    bg, bu = rnd(F, seed=3, dtype=dtype), rnd(F, seed=4, dtype=dtype)
    ff_check16(x, wg, wu, bg, bu, "silu", dh)
    keep = lambda t: t.to(dtype).double()
    with pytest.raises(AssertionError, match="db[gu]: "):
        ff_check16(x, wg, wu, bg, bu, "silu", dh, keep)
    # (without biases: the mean square; the elements' majorants add up magnitudes and reach further)
    with pytest.raises(AssertionError, match="mean square"):
        ff_check16(x, wg, wu, None, None, "silu", dh, keep)
