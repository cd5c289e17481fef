"""The sequence operators of state space recurrent agents and the gradient clip over many tensors: cases, inputs, plain forms.

Operators (codebase_amd.hip):
  ssm_conv / ssm_conv_grad     short causal depthwise convolution, SiLU epilogue, carried window, episode resets, ragged lengths
  ssm_scan / ssm_scan_grad     selective state space scan h_t = exp(dt_t A) h_{t-1} + dt_t B_t x_t, y_t = C_t h_t + D x_t, gated by silu(z_t)
  clip_grad_norm               global 2-norm over many tensors and the clipped gradients

Layouts follow the library's sequence forwards: [agents P][steps S][batch B][channels C], channels contiguous, any stride elsewhere.
Weights are per network, `sharing` maps agents to networks; the carried states are [P][B][state N][C] and [P][B][W-1][C]."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # acting: one environment step of 2 agents x 64 environments; the window is carried, latency counts
        dict(name="conv_act_f32", op="conv", P=2, S=1, B=64, C=128, W=4, dtype="f32", sharing="", carry=True, reset=False, ragged=False),
        # learning from 512 sampled episodes of 25 steps (26 observations), ended early at different steps
        dict(name="conv_episodes_train_f32", op="conv_train", P=2, S=26, B=512, C=128, W=4, dtype="f32", sharing="", carry=False,
             reset=False, ragged=True),
        # long prompts of four rows, the input being one half of a wider projection
        dict(name="conv_prompt_bf16", op="conv", P=1, S=16384, B=4, C=1024, W=4, dtype="bf16", sharing="", carry=True, reset=False,
             ragged=False),
        # acting: one environment step, the scan's state is carried
        dict(name="scan_act_f32", op="scan", P=2, S=1, B=64, C=128, N=16, G=1, dtype="f32", sharing="", carry=True, reset=True, ragged=False,
             z=True),
        # acting in many environments at once: the state is what has to be read and written
        dict(name="scan_act_wide_bf16", op="scan", P=4, S=1, B=4096, C=256, N=16, G=1, dtype="bf16", sharing="", carry=True, reset=True,
             ragged=False, z=True),
        # a rollout of four agents that share one network, episodes starting anew inside it
        dict(name="scan_rollout_f32", op="scan", P=4, S=128, B=256, C=128, N=16, G=1, dtype="f32", sharing="0000", carry=True, reset=True,
             ragged=False, z=True),
        # learning from 512 sampled episodes of 25 steps
        dict(name="scan_episodes_train_f32", op="scan_train", P=2, S=26, B=512, C=128, N=16, G=1, dtype="f32", sharing="", carry=False,
             reset=False, ragged=True, z=True),
        # learning from 500-step episodes of four agents, resets inside, state carried in and its gradient out
        dict(name="scan_rollout_train_bf16", op="scan_train", P=4, S=501, B=32, C=256, N=16, G=1, dtype="bf16", sharing="", carry=True,
             reset=True, ragged=False, z=True),
        # one long prompt: few rows, the work has to be split over its length
        dict(name="scan_prompt_bf16", op="scan", P=1, S=16384, B=1, C=512, N=16, G=1, dtype="bf16", sharing="", carry=True, reset=False,
             ragged=False, z=True),
        # odd sizes, two groups of input and output maps, agents sharing networks selectively, half precision
        dict(name="scan_odd_train_f16", op="scan_train", P=3, S=37, B=29, C=100, N=10, G=2, dtype="f16", sharing="010", carry=True,
             reset=True, ragged=True, z=True),
        # the gradients of two agents' default networks: 12 small tensors
        dict(name="clip_agents_f32", op="clip", tensors=12, largest=128 * 128, dtype="f32", mixed=False),
        # many tensors of mixed sizes and types
        dict(name="clip_many_mixed", op="clip", tensors=320, largest=1024 * 1024, dtype="bf16", mixed=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv", "conv_train", "scan", "scan", "scan_train", "scan_train", "clip"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "clip":
        n = _log_int(rng, 1, 320)
        return dict(op=op, tensors=n, largest=_log_int(rng, 64, 1024 * 1024), dtype=dtype, mixed=rng.random() < 0.5)
    P = rng.choice([1, 1, 2, 2, 3, 4, 8])
    S = 1 if rng.random() < 0.2 else _log_int(rng, 2, 8192)
    sharing = rng.choice(["", "", "0" * P, "".join(str(i % 2) for i in range(P))])
    case = dict(op=op, P=P, S=S, dtype=dtype, sharing=sharing, carry=rng.random() < 0.6, reset=rng.random() < 0.5, ragged=rng.random() < 0.4)
    if op.startswith("conv"):
        C = _log_int(rng, 8, 1024)
        S = case["S"] = max(1, min(S, 2**25 // (P * C)))
        B = _log_int(rng, 1, max(1, min(4096, 2**25 // (P * S * C))))
        case.update(B=B, C=C, W=rng.choice([2, 3, 4, 4, 4]))
        return case
    G = rng.choice([1, 1, 1, 2])
    N = rng.choice([4, 8, 10, 16, 16, 16, 24, 32])
    C = G * _log_int(rng, 8, 512 // G)
    room = 2**27 if op == "scan" else 2**26
    S = case["S"] = max(1, min(S, room // (P * C * N)))
    B = _log_int(rng, 1, max(1, min(4096, room // (P * S * C * N))))
    case.update(B=B, C=C, N=N, G=G, z=rng.random() < 0.8)
    return case


def _networks(case):
    net = [int(c) for c in case["sharing"]] or list(range(case["P"]))
    return net, max(net) + 1


def _episodes(case, st, gen):
    """resets (an episode starts at this step) and lengths as replayed or collected episodes have them"""
    S, B = case["S"], case["B"]
    if case["reset"]:
        st["reset"] = (torch.rand(S, B, generator=gen, device="cuda") < 1.0 / 25).to(torch.uint8)
    if case["ragged"]:
        st["lengths"] = torch.randint((S + 1) // 2, S + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)


def _clip_sizes(case):
    """(elements, type) of every tensor: weights and biases in turn, sizes spread below the largest"""
    sizes = []
    for i in range(case["tensors"]):
        k = case["largest"] if i % 6 == 2 else max(1, case["largest"] >> (2 * (i % 6)))
        if i % 2 == 1:
            k = max(1, int(math.isqrt(k)) - (i % 3))
        sizes.append((k, "f32" if case["mixed"] and i % 3 == 0 else case["dtype"]))
    return sizes


def _pad(k):
    return (k + 63) // 64 * 64  # a flat buffer's views start on whole cache lines


def _prepare_clip(case, gen):
    # small gradients with a norm above the limit; the clipped ones go into the optimiser's flat buffers, one a type
    sizes = _clip_sizes(case)
    grads = [(torch.randn(k, generator=gen, device="cuda") * (0.5 / (1 + i % 4))).to(DTYPES[d]) for i, (k, d) in enumerate(sizes)]
    flat = {d: torch.zeros(sum(_pad(k) for k, dk in sizes if dk == d), dtype=DTYPES[d], device="cuda") for d in sorted({d for _, d in sizes})}
    at, out = dict.fromkeys(flat, 0), []
    for k, d in sizes:
        out.append(flat[d][at[d]:at[d] + k])
        at[d] += _pad(k)
    return {"grads": grads, "out": out, "flat": flat, "max_norm": 0.5}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] == "clip":
        return dict(_prepare_clip(case, gen), case=case)
    dt = DTYPES[case["dtype"]]
    P, S, B, C = (case[k] for k in "PSBC")
    net, M = _networks(case)
    st = {"case": case, "sharing": tuple(net) if case["sharing"] else None, "net": torch.tensor(net, device="cuda"), "M": M,
          "reset": None, "lengths": None}

    def rn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    _episodes(case, st, gen)
    train = case["op"].endswith("train")
    if case["op"].startswith("conv"):
        W = case["W"]
        st["x"] = rn(P, S, B, 2 * C)[..., :C]  # the first half of the input projection, the gate is the other half
        st["weight"] = rn(M, W, C, scale=1.0 / math.sqrt(W), dtype=torch.float32)
        st["bias"] = rn(M, C, scale=0.1, dtype=torch.float32)
        st["state"] = rn(P, B, W - 1, C) if case["carry"] else None
        if train:
            st["dy"] = rn(P, S, B, C)
            st["dstate"] = rn(P, B, W - 1, C) if case["carry"] else None
        return st
    N, G = case["N"], case["G"]
    st["x"] = torch.nn.functional.silu(rn(P, S, B, C, dtype=torch.float32)).to(dt)
    st["z"] = rn(P, S, B, 2 * C)[..., C:] if case["z"] else None
    st["delta"] = rn(P, S, B, C, scale=0.5)
    rank = (C + 15) // 16
    maps = rn(P, S, B, rank + 2 * G * N)
    st["B"] = maps[..., rank:rank + G * N].unflatten(-1, (G, N))
    st["C"] = maps[..., rank + G * N:].unflatten(-1, (G, N))
    # decay rates 1..N with some spread, step sizes log-uniform in [1e-3, 1e-1] through the softplus
    st["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32)[None, :, None] * (0.8 + 0.4 * torch.rand(M, N, C, generator=gen, device="cuda"))
    step = torch.exp(torch.rand(M, C, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
    st["delta_bias"] = step + torch.log(-torch.expm1(-step))
    st["D"] = 1.0 + rn(M, C, scale=0.1, dtype=torch.float32)
    st["h_in"] = rn(P, B, N, C, scale=0.3, dtype=torch.float32) if case["carry"] else None
    if train:
        st["dy"] = rn(P, S, B, C)
        st["dh"] = rn(P, B, N, C, dtype=torch.float32) if case["carry"] else None
    return st


def work(case):
    e = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "clip":
        sizes = _clip_sizes(case)
        total, bytes_ = sum(k for k, _ in sizes), sum(2 * k * (4 if d == "f32" else 2) for k, d in sizes)  # read once, written once
        return {"bytes": bytes_ + 4, "flops": 3 * total}
    P, S, B, C = (case[k] for k in "PSBC")
    rows, M = P * S * B, _networks(case)[1]
    train, carry = case["op"].endswith("train"), case["carry"]
    extra = (S * B if case["reset"] else 0) + (4 * B if case["ragged"] else 0)
    if case["op"].startswith("conv"):
        W = case["W"]
        state, weights = P * B * (W - 1) * C * e, M * (W + 1) * C * 4
        if not train:
            return {"bytes": rows * C * 2 * e + weights + extra + (2 * state if carry else 0), "flops": rows * C * (2 * W + 5)}
        # a training pass: x in, y out; x and dy in, dx and the weights' gradients out (x counted once)
        return {"bytes": rows * C * 4 * e + 2 * weights + extra + (4 * state if carry else 0), "flops": rows * C * (8 * W + 15)}
    N, G = case["N"], case["G"]
    state, weights = P * B * N * C * 4, M * (N + 2) * C * 4
    seq = 3 + (1 if case["z"] else 0)  # x, delta, y and the gate
    fwd = rows * (C * seq + 2 * G * N) * e + weights + extra + (2 * state if carry else 0)
    if not train:
        return {"bytes": fwd, "flops": rows * C * (7 * N + 12)}
    # a training pass: the inputs and dy once, y, the inputs' gradients and the weights' gradients out
    return {"bytes": rows * (C * (2 * seq) + 4 * G * N) * e + 2 * weights + extra + (4 * state if carry else 0),
            "flops": rows * C * (24 * N + 40)}


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------
def _per_network(t, net, M):
    """sum the per-agent gradients of agents that share a network"""
    return torch.zeros(M, *t.shape[1:], dtype=t.dtype, device=t.device).index_add_(0, net, t)


def _valid(case, st):
    """[S][B]: steps before the sequence's end"""
    S, B = case["S"], case["B"]
    t = torch.arange(S, device="cuda")[:, None]
    if st["lengths"] is None:
        return torch.ones(S, B, dtype=torch.bool, device="cuda")
    return t < st["lengths"].long()[None, :]


def _plain_conv(case, st, train):
    P, S, B, C, W = case["P"], case["S"], case["B"], case["C"], case["W"]
    net, M, dt = st["net"], st["M"], st["x"].dtype
    x, w, bias = st["x"].float(), st["weight"][net], st["bias"][net]
    state = st["state"].float() if st["state"] is not None else torch.zeros(P, B, W - 1, C, device="cuda")
    e = torch.cat([state.transpose(1, 2), x], 1)  # [P][W-1+S][B][C]
    pos = torch.arange(S, device="cuda")[:, None]
    start = torch.full((S, B), -W, dtype=torch.long, device="cuda")  # first position the window at a step may look at
    if st["reset"] is not None:
        start = torch.where(st["reset"] != 0, pos, start).cummax(0).values
    valid = _valid(case, st)
    pre = bias[:, None, None, :].expand(P, S, B, C).clone()
    for j in range(W):
        ok = ((pos - j >= start) & valid)[None, :, :, None]
        pre += torch.where(ok, e[:, W - 1 - j:W - 1 - j + S], 0.0) * w[:, W - 1 - j][:, None, None, :]
    sig = 1.0 / (1.0 + torch.exp(-pre))
    v = valid[None, :, :, None]
    y = torch.where(v, pre * sig, 0.0)
    # the window after the last step
    length = st["lengths"].long() if st["lengths"] is not None else torch.full((B,), S, dtype=torch.long, device="cuda")
    src = length[:, None] - (W - 1) + torch.arange(W - 1, device="cuda")[None, :]  # positions [B][W-1], >= -(W-1)
    last = torch.where(length > 0, start.gather(0, (length - 1).clamp(min=0)[None, :])[0], -W)
    keep = (src >= last[:, None])[None, :, :, None]
    at = (src + W - 1)
    window = torch.where(keep, e.transpose(1, 2).gather(2, at[None, :, :, None].expand(P, B, W - 1, C)), 0.0)
    if not train:
        return {"y": y.to(dt), "state": window.to(dt)} if case["carry"] else {"y": y.to(dt)}
    dpre = torch.where(v, st["dy"].float() * sig * (1.0 + pre * (1.0 - sig)), 0.0)
    de = torch.zeros_like(e)
    dw = torch.zeros(P, W, C, device="cuda")
    for j in range(W):
        ok = ((pos - j >= start) & valid)[None, :, :, None]
        dw[:, W - 1 - j] = (dpre * torch.where(ok, e[:, W - 1 - j:W - 1 - j + S], 0.0)).sum((1, 2))
        de[:, W - 1 - j:W - 1 - j + S] += torch.where(ok, dpre * w[:, W - 1 - j][:, None, None, :], 0.0)
    if st["dstate"] is not None:
        de.transpose(1, 2).scatter_add_(2, at[None, :, :, None].expand(P, B, W - 1, C), torch.where(keep, st["dstate"].float(), 0.0))
    out = {"y": y.to(dt), "dx": de[:, W - 1:].to(dt), "dweight": _per_network(dw, net, M), "dbias": _per_network(dpre.sum((1, 2)), net, M)}
    if case["carry"]:
        out["state"], out["dstate"] = window.to(dt), de[:, :W - 1].transpose(1, 2).to(dt)
    return out


def _plain_scan(case, st, train):
    P, S, B, C, N, G = (case[k] for k in "PSBCNG")
    net, M, dt = st["net"], st["M"], st["x"].dtype
    valid = _valid(case, st)[None, :, :, None]
    x = torch.where(valid, st["x"].float(), 0.0)
    A, D, db = st["A"][net], st["D"][net], st["delta_bias"][net]
    raw = torch.where(valid, st["delta"].float() + db[:, None, None, :], 0.0)
    step = torch.where(valid, torch.where(raw > 20.0, raw, torch.log1p(torch.exp(raw.clamp(max=20.0)))), 0.0)

    def wide(m):  # [P][S][B][G][N] -> [P][S][B][N][C]
        m = torch.where(valid[..., None], m.float(), 0.0)
        return m.transpose(-1, -2).repeat_interleave(C // G, -1)

    Bw, Cw = wide(st["B"]), wide(st["C"])
    a = torch.exp(step[:, :, :, None, :] * A[:, None, None, :, :])
    if st["reset"] is not None:
        a = a * ((st["reset"] == 0) | ~valid[0, :, :, 0])[None, :, :, None, None]  # the state is dropped before this step
    u = (step * x)[:, :, :, None, :] * Bw
    h = st["h_in"] if st["h_in"] is not None else torch.zeros(P, B, N, C, device="cuda")
    hs = torch.empty_like(u)
    for t in range(S):
        h = torch.addcmul(u[:, t], a[:, t], h)
        hs[:, t] = h
    ys = (hs * Cw).sum(3) + D[:, None, None, :] * x
    gate = None
    y = ys
    if st["z"] is not None:
        z = torch.where(valid, st["z"].float(), 0.0)
        sig = 1.0 / (1.0 + torch.exp(-z))
        gate = z * sig
        y = ys * gate
    y = torch.where(valid, y, 0.0).to(dt)
    if not train:
        return {"y": y, "h": h} if case["carry"] else {"y": y}
    dy = torch.where(valid, st["dy"].float(), 0.0)
    out = {"y": y}
    dys = dy
    if gate is not None:
        out["dz"] = (dy * ys * sig * (1.0 + z * (1.0 - sig))).to(dt)
        dys = dy * gate
    e = dys[:, :, :, None, :] * Cw
    dh = st["dh"] if st["dh"] is not None else torch.zeros(P, B, N, C, device="cuda")
    g = torch.empty_like(e)  # the gradient at every step's state
    for t in range(S - 1, -1, -1):
        dh = dh + e[:, t]
        g[:, t] = dh
        dh = dh * a[:, t]
    del e
    prev = torch.empty_like(hs)
    prev[:, 1:] = hs[:, :-1]
    prev[:, 0] = st["h_in"] if st["h_in"] is not None else 0.0

    def narrow(m):  # the sum over a group's channels
        return m.unflatten(-1, (G, C // G)).sum(-1).transpose(-1, -2)

    out["dC"] = narrow(dys[:, :, :, None, :] * hs).to(dt)
    out["dB"] = narrow(g * (step * x)[:, :, :, None, :]).to(dt)
    gb = (g * Bw).sum(3)
    ga = torch.where(valid[..., None], g * a * prev, 0.0)  # through the decay's exponent
    dstep = gb * x + (ga * A[:, None, None, :, :]).sum(3)
    draw_ = torch.where(valid, dstep / (1.0 + torch.exp(-raw)), 0.0)
    out["ddelta"] = draw_.to(dt)
    out["dx"] = torch.where(valid, gb * step + dys * D[:, None, None, :], 0.0).to(dt)
    out["dA"] = _per_network((ga * step[:, :, :, None, :]).sum((1, 2)), net, M)
    out["dD"] = _per_network((dys * x).sum((1, 2)), net, M)
    out["ddelta_bias"] = _per_network(draw_.sum((1, 2)), net, M)
    if case["carry"]:
        out["h"], out["dh"] = h, dh
    return out


def _flat(st, grads):
    """the flat buffers that hold these gradients, the gaps between them zero"""
    return {d: torch.cat([torch.nn.functional.pad(g, (0, _pad(g.numel()) - g.numel())) for g, (_, dk) in zip(grads, _clip_sizes(st["case"])) if dk == d])
            for d in st["flat"]}


def _plain_clip(st):
    norm = torch.sqrt(torch.stack([(g.float() ** 2).sum(dtype=torch.float64) for g in st["grads"]]).sum()).float()
    coef = torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0)
    return {"norm": norm.reshape(1), **_flat(st, [(g.float() * coef).to(g.dtype) for g in st["grads"]])}


# ---- the framework's calls ---------------------------------------------------------------------------------------------------------
def _own_conv(case, st, train):
    from codebase_amd import hip as h

    kw = dict(sharing=st["sharing"], state=st["state"], reset=st["reset"], lengths=st["lengths"])
    out = {}
    if case["carry"]:
        out["y"], out["state"] = h.ssm_conv(st["x"], st["weight"], st["bias"], want_state=True, **kw)
    else:
        out["y"] = h.ssm_conv(st["x"], st["weight"], st["bias"], **kw)
    if train:
        g = h.ssm_conv_grad(st["dy"], st["x"], st["weight"], st["bias"], dstate_out=st["dstate"], **kw)
        out.update(dx=g.x, dweight=g.weight, dbias=g.bias)
        if case["carry"]:
            out["dstate"] = g.state
    return out


def _own_scan(case, st, train):
    from codebase_amd import hip as h

    args = (st["x"], st["delta"], st["A"], st["B"], st["C"])
    kw = dict(D=st["D"], z=st["z"], delta_bias=st["delta_bias"], sharing=st["sharing"], h_in=st["h_in"], reset=st["reset"],
              lengths=st["lengths"])
    record = h.ssm_scan_record(st["x"], case["N"]) if train else None
    out = {}
    if case["carry"]:
        out["y"], out["h"] = h.ssm_scan(*args, want_h=True, record=record, **kw)
    else:
        out["y"] = h.ssm_scan(*args, record=record, **kw)
    if train:
        g = h.ssm_scan_grad(st["dy"], *args, record, dh_out=st["dh"], **kw)
        out.update(dx=g.x, ddelta=g.delta, dA=g.A, dB=g.B, dC=g.C, dD=g.D, ddelta_bias=g.delta_bias)
        if case["z"]:
            out["dz"] = g.z
        if case["carry"]:
            out["dh"] = g.h_in
    return out


def _own_clip(st):
    from codebase_amd import hip as h

    return {"norm": h.clip_grad_norm(st["grads"], st["max_norm"], out=st["out"]), **st["flat"]}


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "clip":
        return _own_clip(state) if own else _plain_clip(state)
    train = op.endswith("train")
    if op.startswith("conv"):
        return (_own_conv if own else _plain_conv)(case, state, train)
    return (_own_scan if own else _plain_scan)(case, state, train)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------
def _exact_conv(case, st, train):
    """position by position through a window that a reset empties; gradients by automatic differentiation"""
    P, S, B, C, W = case["P"], case["S"], case["B"], case["C"], case["W"]
    net = st["net"]

    def leaf(t):
        return t.double().clone().requires_grad_(train)

    x, weight, bias = leaf(st["x"]), leaf(st["weight"]), leaf(st["bias"])
    state = leaf(st["state"]) if st["state"] is not None else torch.zeros(P, B, W - 1, C, dtype=torch.float64, device="cuda")
    w, b = weight[net], bias[net]
    window = [state[:, :, i] for i in range(W - 1)]
    ys = []
    length = st["lengths"].long() if st["lengths"] is not None else torch.full((B,), S, device="cuda")
    for t in range(S):
        live = (t < length)[None, :, None]
        xt = torch.where(live, x[:, t], 0.0)
        if st["reset"] is not None:
            fresh = ((st["reset"][t] != 0)[None, :, None]) & live
            window = [torch.where(fresh, 0.0, v) for v in window]
        taps = window + [xt]
        pre = b[:, None, :] + sum(tap * w[:, i][:, None, :] for i, tap in enumerate(taps))
        ys.append(torch.where(live, pre * torch.sigmoid(pre), 0.0))
        window = [torch.where(live, n, v) for n, v in zip(taps[1:], window)]
    y, state_out = torch.stack(ys, 1), torch.stack(window, 2) if W > 1 else state
    out = {"y": y}
    if case["carry"]:
        out["state"] = state_out
    if train:
        loss = (y * st["dy"].double()).sum()
        if st["dstate"] is not None:
            loss = loss + (state_out * st["dstate"].double()).sum()
        leaves = [x, weight, bias] + ([state] if case["carry"] else [])
        g = torch.autograd.grad(loss, leaves)
        out.update(dx=g[0], dweight=g[1], dbias=g[2])
        if case["carry"]:
            out["dstate"] = g[3]
    return {k: v.detach() for k, v in out.items()}


def _exact_scan(case, st, train):
    """step by step from the definition; gradients by automatic differentiation"""
    P, S, B, C, N, G = (case[k] for k in "PSBCNG")
    net = st["net"]

    def leaf(t):
        return None if t is None else t.double().clone().requires_grad_(train)

    names = ["x", "delta", "B", "C", "z", "A", "D", "delta_bias", "h_in"]
    v = {k: leaf(st[k]) for k in names}
    A, D, db = v["A"][net], v["D"][net], v["delta_bias"][net]
    h = v["h_in"] if v["h_in"] is not None else torch.zeros(P, B, N, C, dtype=torch.float64, device="cuda")
    group = torch.arange(C, device="cuda") // (C // G)
    length = st["lengths"].long() if st["lengths"] is not None else torch.full((B,), S, device="cuda")
    ys = []
    for t in range(S):
        live = (t < length)[None, :, None]
        xt = v["x"][:, t]
        step = torch.nn.functional.softplus(v["delta"][:, t] + db[:, None, :], threshold=60.0)
        Bt, Ct = (v[k][:, t].transpose(-1, -2)[..., group] for k in ("B", "C"))  # [P][B][N][C]
        hp = h
        if st["reset"] is not None:
            hp = torch.where((st["reset"][t] != 0)[None, :, None, None], 0.0, h)
        hn = torch.exp(step[:, :, None, :] * A[:, None]) * hp + (step * xt)[:, :, None, :] * Bt
        yt = (Ct * hn).sum(2) + D[:, None, :] * xt
        if v["z"] is not None:
            zt = v["z"][:, t]
            yt = yt * zt * torch.sigmoid(zt)
        ys.append(torch.where(live, yt, 0.0))
        h = torch.where(live[:, :, None, :], hn, h)
    y = torch.stack(ys, 1)
    out = {"y": y}
    if case["carry"]:
        out["h"] = h
    if train:
        loss = (y * st["dy"].double()).sum()
        if st["dh"] is not None:
            loss = loss + (h * st["dh"].double()).sum()
        used = [k for k in names if v[k] is not None]
        grads = torch.autograd.grad(loss, [v[k] for k in used])
        for k, g in zip(used, grads):
            out["dh" if k == "h_in" else "d" + k] = g
    return {k: t.detach() for k, t in out.items()}


def _exact_clip(st):
    total = sum(float((g.double() * g.double()).sum()) for g in st["grads"])
    norm = math.sqrt(total)
    coef = min(st["max_norm"] / (norm + 1e-6), 1.0)
    return {"norm": torch.tensor([norm], dtype=torch.float64, device="cuda"), **_flat(st, [g.double() * coef for g in st["grads"]])}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "clip":
        return _exact_clip(st)
    train = case["op"].endswith("train")
    if train and case["S"] > 1024:  # differentiating so many steps one by one takes too long
        return None
    return _exact_conv(case, st, train) if case["op"].startswith("conv") else _exact_scan(case, st, train)
