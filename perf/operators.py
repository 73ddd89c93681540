"""What is measured of the residual temporal block: a gated linear recurrence over an episode, the norms before and after a block
fused with its gate and residual scale, and a gated feed-forward block -- each in its plain form (elementary torch operations in
32 bits) and, where `own` is true, through refil_amd.blocks.

    recurrence   L_t = c softplus(decay) sigmoid(ga_t),  a_t = exp(-L_t)
                 h_t = [reset_t = 0] a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gi_t) x_t,   y_t = h_t
    norm         N(v; w) = v w / sqrt(mean(v^2) + eps);   y = alpha x + s sigmoid(g) N(o; w_post),   n = N(y; w_pre)
    feed-forward h = act(x Wg^T + bg) * (x Wu^T + bu)

A "train" case is the forward and the backward of one step, a "forward" case what evaluation runs, a "step" case one acting step of
every agent.
"""
import math

import torch

own = False

SCALE = 8.0          # c of the recurrence
EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one acting step of 8 environments x 16 agents, hidden size 64: latency alone
        {"name": "rec_step_act", "op": "rec", "dir": "step", "dtype": "f32", "B": 128, "D": 64, "slots": True},
        # the learner's batch: 32 episodes x 3 imagined copies, 81 steps, 16 agents x 64 hidden units, early ends
        {"name": "rec_train_episode", "op": "rec", "dir": "train", "dtype": "f32", "B": 96, "T": 81, "na": 16, "D": 64, "ragged": True},
        # few long sequences in 16 bits: the sequence has to be split to fill the card
        {"name": "rec_train_long", "op": "rec", "dir": "train", "dtype": "bf16", "B": 4, "T": 8192, "na": 1, "D": 1024, "ragged": False},
        # evaluation of ragged packed rows with resets, odd length and width
        {"name": "rec_forward_odd", "op": "rec", "dir": "forward", "dtype": "f16", "B": 3, "T": 5001, "na": 1, "D": 997, "ragged": True},
        # the norm around one acting step
        {"name": "norm_step_act", "op": "norm", "dir": "forward", "dtype": "f32", "N": 128, "D": 64, "gate": True, "mask": True},
        # the learner's agent rows at the attention width, inactive agents masked
        {"name": "norm_train_agents", "op": "norm", "dir": "train", "dtype": "f32", "N": 41472, "D": 128, "gate": True, "mask": True},
        # wide rows in 16 bits
        {"name": "norm_train_wide", "op": "norm", "dir": "train", "dtype": "bf16", "N": 16384, "D": 2048, "gate": True, "mask": False},
        # odd rows and width, no gate
        {"name": "norm_train_odd", "op": "norm", "dir": "train", "dtype": "f16", "N": 4099, "D": 1001, "gate": False, "mask": False},
        # few rows: the weights' bytes are the cost
        {"name": "ff_forward_rows16", "op": "ff", "dir": "forward", "dtype": "bf16", "N": 16, "D": 1024, "F": 4096, "act": "silu", "bias": False},
        # the learner's agent rows at the attention width, in 32 bits
        {"name": "ff_train_agents", "op": "ff", "dir": "train", "dtype": "f32", "N": 41472, "D": 128, "F": 512, "act": "silu", "bias": True},
        # a large block in 16 bits: the matrix cores are the cost
        {"name": "ff_train_large", "op": "ff", "dir": "train", "dtype": "bf16", "N": 8192, "D": 2048, "F": 8192, "act": "silu", "bias": False},
        # odd rows and widths
        {"name": "ff_train_odd", "op": "ff", "dir": "train", "dtype": "f16", "N": 1537, "D": 520, "F": 1366, "act": "gelu", "bias": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rec", "norm", "ff"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "rec":
        way = rng.choice(["step", "forward", "train", "train"])
        D = _log_int(rng, 16, 4096)
        if way == "step":
            return {"op": op, "dir": way, "dtype": dtype, "B": _log_int(rng, 1, 1024), "D": D, "slots": rng.random() < 0.5}
        na = rng.choice([1, 1, 5, 16]) if D <= 256 else 1
        most = 32e6 / (2 if dtype == "f32" else 1)           # elements: no more than the largest listed case moves
        T = _log_int(rng, 1, min(16384, int(most / (na * D))))
        B = _log_int(rng, 1, max(1, min(256, int(most / (na * D * T)))))
        return {"op": op, "dir": way, "dtype": dtype, "B": B, "T": T, "na": na, "D": D, "ragged": rng.random() < 0.5}
    if op == "norm":
        way = rng.choice(["forward", "train", "train"])
        D = _log_int(rng, 16, 8192)
        N = _log_int(rng, 1, min(100000, int(32e6 / (2 if dtype == "f32" else 1) / D)))
        return {"op": op, "dir": way, "dtype": dtype, "N": N, "D": D, "gate": rng.random() < 0.7, "mask": rng.random() < 0.5}
    way = rng.choice(["forward", "train", "train"])
    D, F = _log_int(rng, 32, 4096), _log_int(rng, 64, 8192)
    most = 8192 * 2048 * 8192 / (16 if dtype == "f32" else 2)
    N = _log_int(rng, 1, max(1, min(16384, int(most / (D * F)))))
    return {"op": op, "dir": way, "dtype": dtype, "N": N, "D": D, "F": F, "act": rng.choice(["silu", "gelu"]), "bias": rng.random() < 0.5}


def work(case):
    """Bytes and operations that a pass cannot do without: each input read once, each output written once."""
    es = BYTES[case["dtype"]]
    if case["op"] == "rec":
        if case["dir"] == "step":
            n = case["B"] * case["D"]
            return {"bytes": n * (4 * es + 8) + 4 * case["D"], "flops": 25 * n}
        n = case["B"] * case["T"] * case["na"] * case["D"]
        state = 4 * case["B"] * case["na"] * case["D"]
        if case["dir"] == "forward":
            return {"bytes": n * 4 * es + 2 * state, "flops": 25 * n}
        return {"bytes": n * 8 * es + 4 * state + 8 * case["D"], "flops": 80 * n}
    if case["op"] == "norm":
        n, g = case["N"] * case["D"], int(case["gate"])
        if case["dir"] == "forward":
            return {"bytes": n * (4 + g) * es + 12 * case["D"], "flops": 20 * n}
        return {"bytes": n * (8 + 2 * g) * es + 24 * case["D"], "flops": 70 * n}
    N, D, F = case["N"], case["D"], case["F"]
    if case["dir"] == "forward":
        return {"bytes": es * (N * D + 2 * F * D + N * F), "flops": 4 * N * D * F}
    return {"bytes": es * (2 * N * D + 4 * F * D + 2 * N * F), "flops": 12 * N * D * F}


# --------------------------------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    s = {}
    if case["op"] == "rec":
        D = case["D"]
        # a_t reaches from 0.9 to 0.999 where its gate is fully open: memories of ten to a thousand steps
        rate = -torch.log(0.9 + 0.099 * uniform(D)) / SCALE
        s["decay"] = torch.log(torch.expm1(rate))
        if case["dir"] == "step":
            B = case["B"]
            for k in ("x", "ga", "gi"):
                s[k] = normal(B, D)
            s["state"] = normal(B + 3 if case["slots"] else B, D, dtype=torch.float32)
            s["state_out"] = s["state"].clone()
            s["slots"] = torch.randperm(B + 3, generator=gen, device=dev)[:B].to(torch.int32) if case["slots"] else None
            return s
        B, T, na = case["B"], case["T"], case["na"]
        shape = (B, T, na, D) if na > 1 else (B, T, D)
        for k in ("x", "ga", "gi"):
            s[k] = normal(*shape)
        s["h0"] = normal(B, *shape[2:], dtype=torch.float32)
        s["lengths"] = s["reset"] = None
        if case["ragged"]:
            s["lengths"] = torch.randint(T // 2, T + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
            s["reset"] = (uniform(B, T) < 0.005).to(torch.uint8)
        if case["dir"] == "train":
            s["dy"] = normal(*shape)
        return s
    if case["op"] == "norm":
        N, D = case["N"], case["D"]
        s["x"], s["o"] = normal(N, D), normal(N, D, scale=0.7)
        s["g"] = normal(N, D) if case["gate"] else None
        s["w_post"], s["w_pre"] = 1.0 + normal(D, scale=0.1, dtype=torch.float32), 1.0 + normal(D, scale=0.1, dtype=torch.float32)
        s["scale"] = 0.5 + 0.5 * uniform(D)
        s["mask"] = (uniform(N) < 0.2).to(torch.uint8) if case["mask"] else None
        if case["dir"] == "train":
            s["dy"], s["dn"] = normal(N, D), normal(N, D)
        return s
    N, D, F = case["N"], case["D"], case["F"]
    s["x"] = normal(N, D)
    s["wg"], s["wu"] = normal(F, D, scale=D ** -0.5), normal(F, D, scale=D ** -0.5)
    s["bg"], s["bu"] = (normal(F, scale=0.1), normal(F, scale=0.1)) if case["bias"] else (None, None)
    if case["dir"] == "train":
        s["dh"] = normal(N, F)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    return s


# ------------------------------------------------------------------------------------------------- passes, both ways
def run(state):
    case = state["case"]
    if own:
        return {"rec": _own_rec, "norm": _own_norm, "ff": _own_ff}[case["op"]](case, state)
    return {"rec": _plain_rec, "norm": _plain_norm, "ff": _plain_ff}[case["op"]](case, state)


def _own_rec(case, s):
    from refil_amd import blocks
    if case["dir"] == "step":
        y = blocks.linrec_step(s["x"], s["ga"], s["gi"], s["decay"], s["state"], scale=SCALE, slots=s["slots"], state_out=s["state_out"])
        return {"y": y, "state": s["state_out"]}
    kw = dict(scale=SCALE, h0=s["h0"], reset=s["reset"], lengths=s["lengths"])
    train = case["dir"] == "train"
    y, h_last, saved = blocks.linrec_forward(s["x"], s["ga"], s["gi"], s["decay"], save=train, **kw)
    if not train:
        return {"y": y, "h_last": h_last}
    dx, dga, dgi, ddecay, dh0 = blocks.linrec_backward(s["dy"], s["x"], s["ga"], s["gi"], s["decay"], saved, **kw)
    return {"y": y, "h_last": h_last, "dx": dx, "dga": dga, "dgi": dgi, "ddecay": ddecay, "dh0": dh0}


def _own_norm(case, s):
    from refil_amd import blocks
    kw = dict(post_weight=s["w_post"], res_scale=s["scale"], pre_weight=s["w_pre"], eps=EPS, row_mask=s["mask"])
    y, n = blocks.norm_gate_forward(s["x"], s["o"], s["g"], **kw)
    if case["dir"] == "forward":
        return {"y": y, "n": n}
    r = blocks.norm_gate_backward(s["dy"], s["dn"], s["x"], s["o"], s["g"], **kw)
    return {"y": y, "n": n, "dx": r.dx, "do": r.do, "dg": r.dgate, "dw_post": r.dpost_weight, "dscale": r.dres_scale, "dw_pre": r.dpre_weight}


def _own_ff(case, s):
    from refil_amd import blocks
    train = case["dir"] == "train"
    h, saved = blocks.gated_ff_forward(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], act=case["act"], save=train)
    if not train:
        return {"h": h}
    dx, dwg, dwu, dbg, dbu = blocks.gated_ff_backward(s["dh"], s["x"], s["wg"], s["wu"], saved, act=case["act"], bias=case["bias"])
    return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu, "dbg": dbg, "dbu": dbu}


# --- plain forms: 32-bit torch operations, one rounding at the end
def _scan(a, u, dim):
    """h_t = a_t h_{t-1} + u_t along `dim` by doubling: after step k every element holds the composition of 2^k maps."""
    n, s = a.shape[dim], 1
    while s < n:
        a0, u0, a1, u1 = a.narrow(dim, 0, n - s), u.narrow(dim, 0, n - s), a.narrow(dim, s, n - s), u.narrow(dim, s, n - s)
        u = torch.cat([u.narrow(dim, 0, s), a1 * u0 + u1], dim)
        a = torch.cat([a.narrow(dim, 0, s), a1 * a0], dim)
        s *= 2
    return a, u


def _plain_rec(case, s):
    dt = s["x"].dtype
    x, ga, gi = (s[k].float() for k in ("x", "ga", "gi"))
    rate = SCALE * torch.log1p(torch.exp(s["decay"]))
    sa, si = 1 / (1 + torch.exp(-ga)), 1 / (1 + torch.exp(-gi))
    L = rate * sa
    a, beta = torch.exp(-L), torch.sqrt(-torch.expm1(-2 * L))
    u = beta * si * x
    if case["dir"] == "step":
        if s["slots"] is None:
            h = a * s["state"] + u
            s["state_out"].copy_(h)
        else:
            rows = s["slots"].long()
            h = a * s["state"][rows] + u
            s["state_out"][rows] = h
        return {"y": h.to(dt), "state": s["state_out"]}
    B, T = x.shape[:2]
    per_step = (B, T) + (1,) * (x.dim() - 2)
    keep = torch.ones(per_step, device=x.device) if s["reset"] is None else (s["reset"] == 0).float().reshape(per_step)
    live = torch.ones(per_step, device=x.device)
    if s["lengths"] is not None:
        live = (torch.arange(T, device=x.device)[None] < s["lengths"][:, None]).float().reshape(per_step)
    h0 = s["h0"]
    ak = a * keep
    dead = live == 0
    scan_a, scan_u = torch.where(dead, torch.ones_like(ak), ak), torch.where(dead, torch.zeros_like(u), u)   # past the end the state stays
    A, U = _scan(scan_a, scan_u, 1)
    h = A * h0[:, None] + U
    out = {"y": (h * live).to(dt), "h_last": h[:, -1]}
    if case["dir"] == "forward":
        return out
    dy = s["dy"].float() * live
    nxt = torch.cat([scan_a[:, 1:], torch.ones_like(scan_a[:, :1])], 1).flip(1)
    dh = _scan(nxt, dy.flip(1), 1)[1].flip(1)                        # dh_t = dy_t + a_{t+1} dh_{t+1}
    prev = torch.cat([h0[:, None], h[:, :-1]], 1)
    q = dh * live * (si * x * a * a * (L / beta) - a * keep * prev * L)        # d(loss)/d(log L)
    sig_over_softplus = torch.sigmoid(s["decay"]) * SCALE / rate
    dims = tuple(range(x.dim() - 1))
    out.update(dx=(dh * live * beta * si).to(dt), dga=(q * (1 - sa)).to(dt), dgi=(dh * live * beta * x * si * (1 - si)).to(dt),
               ddecay=(q.sum(dims)) * sig_over_softplus, dh0=scan_a[:, 0] * dh[:, 0])
    return out


def _plain_norm(case, s):
    dt = s["x"].dtype
    x, o = s["x"].float(), s["o"].float()
    live = torch.ones(x.shape[0], 1, device=x.device) if s["mask"] is None else (s["mask"] == 0).float()[:, None]
    sg = 1.0 if s["g"] is None else 1 / (1 + torch.exp(-s["g"].float()))
    ro = torch.rsqrt((o * o).mean(1, keepdim=True) + EPS)
    oh = o * ro
    y = x + s["scale"] * sg * oh * s["w_post"]
    ry = torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
    yh = y * ry
    out = {"y": (y * live).to(dt), "n": (yh * s["w_pre"] * live).to(dt)}
    if case["dir"] == "forward":
        return out
    dy, dn = s["dy"].float() * live, s["dn"].float() * live
    e = dn * s["w_pre"]
    d = dy + ry * (e - yh * (e * yh).mean(1, keepdim=True))
    f = d * s["scale"] * sg
    e2 = f * s["w_post"]
    out.update(dx=d.to(dt), do=(ro * (e2 - oh * (e2 * oh).mean(1, keepdim=True))).to(dt),
               dg=None if s["g"] is None else (f * oh * s["w_post"] * (1 - sg)).to(dt),
               dw_post=(f * oh).sum(0), dscale=(d * sg * oh * s["w_post"]).sum(0), dw_pre=(dn * yh).sum(0))
    return out


GELU_A, GELU_B = math.sqrt(2 / math.pi), 0.044715          # gelu: 0.5 v (1 + tanh(A (v + B v^3)))


def _plain_ff(case, s):
    dt = s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    if s["bg"] is not None:
        g, u = g + s["bg"].float(), u + s["bu"].float()
    if case["act"] == "silu":
        sg = 1 / (1 + torch.exp(-g))
        act, dact = g * sg, sg * (1 + g * (1 - sg))
    else:
        t = torch.tanh(GELU_A * (g + GELU_B * g * g * g))
        act, dact = 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * GELU_A * (1 + 3 * GELU_B * g * g)
    out = {"h": (act * u).to(dt)}
    if case["dir"] == "forward":
        return out
    dh = s["dh"].float()
    dg, du = dh * u * dact, dh * act
    out.update(dx=(dg @ wg + du @ wu).to(dt), dwg=(dg.t() @ x).to(dt), dwu=(du.t() @ x).to(dt),
               dbg=dg.sum(0).to(dt) if case["bias"] else None, dbu=du.sum(0).to(dt) if case["bias"] else None)
    return out


# ------------------------------------------------------------------------------------------------ definitions, 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    with torch.enable_grad():
        return {"rec": _exact_rec, "norm": _exact_norm, "ff": _exact_ff}[case["op"]](case, s)


def _leaf(t):
    return None if t is None else t.double().requires_grad_(True)


def _exact_rec(case, s):
    decay = s["decay"].double()
    rate = SCALE * torch.nn.functional.softplus(decay, threshold=700.0)
    x, ga, gi = (s[k].double() for k in ("x", "ga", "gi"))

    def maps(ga_, gi_, x_):
        log_a = -rate * torch.sigmoid(ga_)
        return torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a)) * torch.sigmoid(gi_) * x_

    if case["dir"] == "step":
        a, u = maps(ga, gi, x)
        rows = torch.arange(x.shape[0], device=x.device) if s["slots"] is None else s["slots"].long()
        state = s["state"].double()
        y = a * state[rows] + u
        state[rows] = y
        return {"y": y, "state": state}
    T = x.shape[1]
    one = (-1,) + (1,) * (x.dim() - 2)
    h = s["h0"].double()
    ends = torch.full((x.shape[0],), T, device=x.device) if s["lengths"] is None else s["lengths"]
    drop = torch.zeros(x.shape[:2], device=x.device) if s["reset"] is None else s["reset"]
    ends_l, states, y = ends.reshape(one), [], torch.zeros_like(x)
    for t in range(T):
        states.append(h)
        a, u = maps(ga[:, t], gi[:, t], x[:, t])
        new = torch.where(drop[:, t].reshape(one) != 0, u, a * h + u)
        on = t < ends_l
        h = torch.where(on, new, h)
        y[:, t] = torch.where(on, new, torch.zeros_like(new))
    out = {"y": y, "h_last": h}
    if case["dir"] == "forward":
        return out
    dy, grad = s["dy"].double(), torch.zeros_like(h)
    dx, dga, dgi, drate = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(rate)
    for t in range(T - 1, -1, -1):
        on = (t < ends_l).double()
        through = on * (drop[:, t].reshape(one) == 0).double()
        g = (grad + dy[:, t]) * on                                # d loss / d h_t
        sa, si = torch.sigmoid(ga[:, t]), torch.sigmoid(gi[:, t])
        a = torch.exp(-rate * sa)
        root = torch.sqrt(-torch.expm1(-2 * rate * sa))
        dx[:, t] = g * root * si
        dgi[:, t] = g * root * x[:, t] * si * (1 - si)
        dL = g * (a * a / root * si * x[:, t]) - g * through * a * states[t]
        dga[:, t] = dL * rate * sa * (1 - sa)
        drate += (dL * sa).reshape(-1, rate.shape[0]).sum(0)
        grad = g * through * a + grad * (1 - on)
    out.update(dx=dx, dga=dga, dgi=dgi, ddecay=drate * SCALE * torch.sigmoid(decay), dh0=grad)
    return out


def _exact_norm(case, s):
    x, o, g, wp, sc, wq = (_leaf(s[k]) for k in ("x", "o", "g", "w_post", "scale", "w_pre"))
    D = x.shape[1]
    b = o / torch.sqrt(torch.linalg.vector_norm(o, dim=1, keepdim=True) ** 2 / D + EPS) * wp * sc
    y = x + (b if g is None else b * torch.sigmoid(g))
    n = y / torch.sqrt(torch.linalg.vector_norm(y, dim=1, keepdim=True) ** 2 / D + EPS) * wq
    if s["mask"] is not None:
        gone = s["mask"].bool()[:, None]
        y, n = y.masked_fill(gone, 0.0), n.masked_fill(gone, 0.0)
    if case["dir"] == "forward":
        return {"y": y.detach(), "n": n.detach()}
    ins = [x, o, wp, sc, wq] + ([] if g is None else [g])
    d = torch.autograd.grad([y, n], ins, [s["dy"].double(), s["dn"].double()])
    return {"y": y.detach(), "n": n.detach(), "dx": d[0], "do": d[1], "dg": None if g is None else d[5], "dw_post": d[2], "dscale": d[3], "dw_pre": d[4]}


def _exact_ff(case, s):
    x, wg, wu, bg, bu = (_leaf(s[k]) for k in ("x", "wg", "wu", "bg", "bu"))
    g, u = torch.nn.functional.linear(x, wg, bg), torch.nn.functional.linear(x, wu, bu)
    f = torch.nn.functional
    h = (f.silu(g) if case["act"] == "silu" else f.gelu(g, approximate="tanh")) * u
    if case["dir"] == "forward":
        return {"h": h.detach()}
    ins = [x, wg, wu] + ([] if bg is None else [bg, bu])
    d = torch.autograd.grad(h, ins, s["dh"].double())
    return {"h": h.detach(), "dx": d[0], "dwg": d[1], "dwu": d[2], "dbg": None if bg is None else d[3], "dbu": None if bg is None else d[4]}
