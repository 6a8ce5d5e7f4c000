"""The state-space sequence operators, as cases to be measured: short causal convolution and selective scan over whole
sequences (training: value and gradients; prompts: value and the state that generation goes on from) and both for one
more token on a pool of saved states.

Notation: B sequences, T steps, D channels, N states a channel, G groups of channels that share the input and output
maps (D a multiple of G), K taps.  The scan is
    dt = softplus(delta + delta_bias),  h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t,  y_t = (C_t . h_t + D u_t) silu(z_t)
for every channel, h a vector of N states.  `run` computes it through the framework where `own` is true and by
elementary torch operations in 32 bits where it is false (there the recurrence is an associative scan by doubling).
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one layer of the stock training configuration: hidden size 24, expanded twice, windows of 24 steps, batch 128
        dict(name="conv_train_stock", kind="conv_train", dtype="f32", B=128, T=24, D=48, K=4, ragged=False),
        # long training sequences at a channel count of a wide layer
        dict(name="conv_train_long", kind="conv_train", dtype="bf16", B=8, T=4096, D=2048, K=4, ragged=False),
        # prompts of different lengths in one padded batch that go on from a saved state; odd sizes throughout
        dict(name="conv_prompt_ragged", kind="conv_prompt", dtype="bf16", B=7, T=1531, D=1003, K=4, ragged=True),
        # the scan of the same stock training layer
        dict(name="scan_train_stock", kind="scan_train", dtype="f32", B=128, T=24, D=48, N=16, G=1, ragged=False),
        # the stress configuration's layer (hidden size 512 expanded twice, windows of 256 steps) on a slice of its batch
        dict(name="scan_train_stress", kind="scan_train", dtype="f32", B=64, T=256, D=1024, N=16, G=1, ragged=False),
        # long sequences in 16 bits, few of them: training of a wide layer
        dict(name="scan_train_long", kind="scan_train", dtype="bf16", B=4, T=2048, D=2048, N=16, G=1, ragged=False),
        # ONE long prompt: the case with the least independent work for its length
        dict(name="scan_prompt_long", kind="scan_prompt", dtype="bf16", B=1, T=16384, D=2048, N=16, G=1, ragged=False),
        # prompts of different lengths in one padded batch, grouped maps, odd sizes, a larger state, going on from saved states
        dict(name="scan_prompt_ragged", kind="scan_prompt", dtype="f16", B=6, T=777, D=1004, N=24, G=4, ragged=True),
        # one more token of one sequence: nothing but latency
        dict(name="conv_step_one", kind="conv_step", dtype="bf16", B=1, D=1024, K=4, P=1),
        dict(name="scan_step_one", kind="scan_step", dtype="bf16", B=1, D=1024, N=16, G=1, P=1),
        # one more token of each of 256 sequences whose states lie scattered in a pool
        dict(name="conv_step_batch", kind="conv_step", dtype="bf16", B=256, D=4096, K=4, P=300),
        dict(name="scan_step_batch", kind="scan_step", dtype="bf16", B=256, D=4096, N=16, G=1, P=300),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["conv_train", "conv_prompt", "scan_train", "scan_prompt", "conv_step", "scan_step"])
    c = dict(kind=kind, dtype=rng.choice(["f32", "bf16", "f16"]))
    if kind.endswith("step"):
        c["B"] = _log_uniform(rng, 1, 256)
        c["D"] = _log_uniform(rng, 17, 4096)
        c["P"] = c["B"] + rng.randint(0, 40)
    else:
        c["D"] = _log_uniform(rng, 17, 2048)
        c["T"] = _log_uniform(rng, 1, 8192)
    if kind.startswith("conv"):
        c["K"] = rng.randint(2, 5)
        per = c["D"] * c.get("T", 1)
        most = 67_000_000
    else:
        c["N"] = rng.choice([4, 8, 11, 16, 16, 16, 24, 32])
        c["G"] = rng.choice([1, 1, 2, 4])
        c["D"] = -(-c["D"] // c["G"]) * c["G"]
        if kind == "scan_step":
            c["D"] = min(c["D"], 4096)
        per = c["D"] * c["N"] * c.get("T", 1)
        most = 268_000_000
    if not kind.endswith("step"):
        c["T"] = max(1, min(c["T"], most * c["T"] // per))
        per = min(per, most)
        c["B"] = _log_uniform(rng, 1, max(1, min(128, most // per)))
        c["ragged"] = rng.random() < 0.4
    return c


def _lengths(case, gen):
    """Lengths over the whole range, the first one full, the last one (of three or more) zero."""
    if not case.get("ragged"):
        return None
    B, T = case["B"], case["T"]
    lens = torch.randint(1, T + 1, (B,), generator=gen)
    lens[0] = T
    if B > 2:
        lens[-1] = 0
    return lens.to(torch.int32).cuda()


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    kind, B, D = case["kind"], case["B"], case["D"]
    train = kind.endswith("train")

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=dev, device="cuda") * scale).to(dtype)

    s = dict(case=dict(case), kind=kind)
    rows = (B,) if kind.endswith("step") else (B, case["T"])
    if kind.startswith("conv"):
        K = case["K"]
        s["x"] = normal(*rows, D)
        s["weight"] = normal(D, K, scale=1.0 / math.sqrt(K), dtype=torch.float32)
        s["bias"] = normal(D, scale=0.1, dtype=torch.float32)
        leaves = ["x", "weight", "bias"]
        if kind == "conv_prompt":
            s["initial"] = normal(B, K - 1, D)
    else:
        N, G = case["N"], case["G"]
        u = normal(*rows, D, dtype=torch.float32)
        s["u"] = (u * torch.sigmoid(u)).to(dt)
        s["delta"] = normal(*rows, D, scale=0.5)
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * torch.exp(
            normal(D, N, scale=0.2, dtype=torch.float32))
        s["Bm"] = normal(*rows, G, N)
        s["Cm"] = normal(*rows, G, N)
        s["D"] = 1.0 + normal(D, scale=0.1, dtype=torch.float32)
        s["z"] = normal(*rows, D)
        step = torch.exp(torch.rand(D, generator=dev, device="cuda") * math.log(100.0) + math.log(1e-3))
        s["delta_bias"] = torch.log(torch.expm1(step))       # step sizes between 0.001 and 0.1
        leaves = ["u", "delta", "A", "Bm", "Cm", "D", "z", "delta_bias"]
        if kind == "scan_prompt":
            s["initial"] = normal(B, D, N, dtype=torch.float32)
    if kind.endswith("step"):
        P = case["P"]
        shape = (P, case["K"] - 1, D) if kind == "conv_step" else (P, D, case["N"])
        s["state"] = normal(*shape, dtype=dt if kind == "conv_step" else torch.float32)
        s["state_out"] = s["state"].clone()
        s["slots"] = torch.randperm(P, generator=gen)[:B].to(torch.int32).cuda()
    else:
        s["lengths"] = _lengths(case, gen)
    if train:
        s["dy"] = normal(*rows, D)
        s["leaves"] = leaves
        for name in leaves:
            s[name].requires_grad_(True)
    return s


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"conv_train": _plain_conv_train, "conv_prompt": _plain_conv_prompt, "scan_train": _plain_scan_train,
                "scan_prompt": _plain_scan_prompt, "conv_step": _plain_conv_step, "scan_step": _plain_scan_step}[s["kind"]](s)


def _own(s):
    import timegan_amd as tg
    kind = s["kind"]
    if kind == "conv_train":
        y = tg.short_conv(s["x"], s["weight"], s["bias"], silu=True, lengths=s["lengths"])
        return (y, *torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"]))
    if kind == "conv_prompt":
        return tg.short_conv(s["x"], s["weight"], s["bias"], silu=True, initial_state=s["initial"], lengths=s["lengths"],
                             return_state=True)
    if kind == "conv_step":
        y = tg.short_conv_step(s["x"], s["state"], s["weight"], s["bias"], silu=True, slots=s["slots"],
                               state_out=s["state_out"])
        return y, s["state_out"]
    if kind == "scan_step":
        y = tg.selective_scan_step(s["u"], s["delta"], s["state"], s["A"], s["Bm"], s["Cm"], s["D"], s["z"],
                                   s["delta_bias"], softplus=True, slots=s["slots"], state_out=s["state_out"])
        return y, s["state_out"]
    args = (s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], s["D"], s["z"], s["delta_bias"])
    if kind == "scan_train":
        y = tg.selective_scan(*args, softplus=True, lengths=s["lengths"])
        return (y, *torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"]))
    return tg.selective_scan(*args, softplus=True, initial_state=s["initial"], lengths=s["lengths"], return_state=True)


# ---- the plain forms: elementary torch operations in 32 bits, rounded once at the end ---------------------------------

def _valid(s, T):
    """(B, T, 1) truth values: the steps that a sequence has; None where all have all."""
    if s["lengths"] is None:
        return None
    return (torch.arange(T, device="cuda")[None, :] < s["lengths"][:, None])[..., None]


def _masked(x, valid):
    return x if valid is None else torch.where(valid, x, torch.zeros((), device=x.device))


def _conv_rows(s):
    """(rows with K - 1 earlier ones in front, pre-activation), both over the steps that there are."""
    x, w = s["x"].float(), s["weight"]
    B, T, D = x.shape
    K = w.shape[1]
    valid = _valid(s, T)
    first = s["initial"].float() if "initial" in s else torch.zeros(B, K - 1, D, device="cuda")
    ext = torch.cat([first, _masked(x, valid)], 1)
    pre = s["bias"] + sum(ext[:, k:k + T] * w[:, k] for k in range(K))
    return ext, pre, valid


def _plain_conv_prompt(s):
    ext, pre, valid = _conv_rows(s)
    B, T = s["x"].shape[:2]
    K = s["weight"].shape[1]
    y = _masked(pre * torch.sigmoid(pre), valid).to(s["x"].dtype)
    lens = torch.full((B,), T, device="cuda") if s["lengths"] is None else s["lengths"].long()
    at = lens[:, None] + torch.arange(K - 1, device="cuda")
    return y, ext[torch.arange(B, device="cuda")[:, None], at].to(s["x"].dtype)


def _plain_conv_train(s):
    ext, pre, valid = _conv_rows(s)
    T, K = s["x"].shape[1], s["weight"].shape[1]
    sig = torch.sigmoid(pre)
    y = _masked(pre * sig, valid).to(s["x"].dtype)
    dpre = _masked(s["dy"].float() * sig * (1 + pre * (1 - sig)), valid)
    tail = torch.cat([dpre, torch.zeros_like(dpre[:, :K - 1])], 1)
    dx = _masked(sum(tail[:, K - 1 - k:K - 1 - k + T] * s["weight"][:, k] for k in range(K)), valid)
    dw = torch.stack([(dpre * ext[:, k:k + T]).sum((0, 1)) for k in range(K)], 1)
    return y, dx.to(s["x"].dtype), dw, dpre.sum((0, 1))


def _plain_conv_step(s):
    rows = s["slots"].long()
    ext = torch.cat([s["state"][rows].float(), s["x"].float()[:, None]], 1)
    pre = s["bias"] + (ext * s["weight"].t()).sum(1)
    s["state_out"][rows] = ext[:, 1:].to(s["x"].dtype)
    return (pre * torch.sigmoid(pre)).to(s["x"].dtype), s["state_out"]


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _spread(m, D):
    """The maps of G groups, (..., G, N) -> (..., D, N) in 32 bits."""
    return m.float().repeat_interleave(D // m.shape[-2], dim=-2)


def _gather(m, G):
    """Sum over the channels of a group, (B, T, D, N) -> (B, T, G, N)."""
    B, T, D, N = m.shape
    return m.view(B, T, G, D // G, N).sum(3)


def _recur(a, b):
    """h_t = a_t h_{t-1} + b_t over dimension 1 (h_{-1} = 0), by doubling: spans of 1, 2, 4, ... steps are joined."""
    T, span = a.shape[1], 1
    while span < T:
        b = torch.cat([b[:, :span], torch.addcmul(b[:, span:], a[:, span:], b[:, :-span])], 1)
        if 2 * span < T:
            a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _scan_states(s):
    T, D = s["u"].shape[1:]
    valid = _valid(s, T)
    u, raw = _masked(s["u"].float(), valid), s["delta"].float() + s["delta_bias"]
    dt = _masked(_softplus(raw), valid)
    a = torch.exp(dt[..., None] * s["A"])
    b = (dt * u)[..., None] * _spread(s["Bm"], D)
    if "initial" in s:
        b[:, 0] += a[:, 0] * s["initial"]
    return valid, u, raw, dt, a, _recur(a, b)


def _plain_scan_prompt(s):
    valid, u, _, _, _, h = _scan_states(s)
    z = s["z"].float()
    y = (h * _spread(s["Cm"], u.shape[2])).sum(-1) + s["D"] * u
    return _masked(y * z * torch.sigmoid(z), valid).to(s["u"].dtype), h[:, -1].clone()


def _plain_scan_train(s):
    kept = s["u"].dtype
    valid, u, raw, dt, a, h = _scan_states(s)
    D, G = u.shape[2], s["Bm"].shape[2]
    C, z = _spread(s["Cm"], D), s["z"].float()
    sig = torch.sigmoid(z)
    out = (h * C).sum(-1) + s["D"] * u
    y = _masked(out * z * sig, valid).to(kept)
    dy = _masked(s["dy"].float(), valid)
    dz = (dy * out * sig * (1 + z * (1 - sig))).to(kept)
    dy = dy * z * sig
    dC = _gather(dy[..., None] * h, G)
    # dh_t = C_t dy_t + a_{t+1} dh_{t+1}: the same recurrence from the last step to the first
    later = torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    g = _recur(later, (dy[..., None] * C).flip(1)).flip(1)
    dB = _gather(g * (dt * u)[..., None], G)
    gB = (g * _spread(s["Bm"], D)).sum(-1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    w = g * a * before
    ddt = gB * u + (w * s["A"]).sum(-1)
    ddelta = _masked(ddt * torch.sigmoid(raw), valid)
    dA = (w * dt[..., None]).sum((0, 1))
    return (y, (gB * dt + s["D"] * dy).to(kept), ddelta.to(kept), dA, dB.to(kept), dC.to(kept), (dy * u).sum((0, 1)), dz,
            ddelta.sum((0, 1)))


def _plain_scan_step(s):
    rows, u, z = s["slots"].long(), s["u"].float(), s["z"].float()
    dt = _softplus(s["delta"].float() + s["delta_bias"])
    D = u.shape[1]
    h = torch.exp(dt[..., None] * s["A"]) * s["state"][rows] + (dt * u)[..., None] * _spread(s["Bm"], D)
    y = (h * _spread(s["Cm"], D)).sum(-1) + s["D"] * u
    s["state_out"][rows] = h
    return (y * z * torch.sigmoid(z)).to(s["u"].dtype), s["state_out"]


# ---- what cannot be done without --------------------------------------------------------------------------------------

def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    rows = case["B"] * case.get("T", 1)
    live = rows / 2 if case.get("ragged") else rows        # ragged lengths are half of T in the mean; outputs come whole
    x, xl = rows * case["D"], live * case["D"]
    if kind.startswith("conv"):
        K, state = case["K"], case["B"] * (case["K"] - 1) * case["D"] * e
        taps = case["D"] * (K + 1) * 4
        if kind == "conv_train":       # x, dy in; y, dx out; the taps and their gradients
            return {"bytes": 2 * (x + xl) * e + 2 * taps, "flops": xl * (6 * K + 20)}
        return {"bytes": (x + xl) * e + 2 * state + taps, "flops": xl * (2 * K + 6)}
    N = case["N"]
    maps, maps_l = rows * case["G"] * N, live * case["G"] * N
    state = case["B"] * case["D"] * N * 4
    par = case["D"] * (N + 2) * 4
    if kind == "scan_train":           # u, delta, z, dy in; y, du, ddelta, dz out; both maps and their gradients
        return {"bytes": 4 * (x + xl) * e + 2 * (maps + maps_l) * e + 2 * par, "flops": xl * (22 * N + 40)}
    return {"bytes": (x + 3 * xl) * e + 2 * maps_l * e + 2 * state + par, "flops": xl * (7 * N + 20)}


# ---- the definition in 64 bits, step by step --------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    with torch.no_grad():
        return _exact_conv(s) if s["kind"].startswith("conv") else _exact_scan(s)


def _silu(v):
    return v / (1 + torch.exp(-v))


def _silu_slope(v):
    e = torch.exp(-v)
    return (1 + e + v * e) / (1 + e) ** 2


def _exact_conv(s):
    w, K = s["weight"], s["weight"].shape[1]
    if s["kind"] == "conv_step":
        rows = s["slots"].long()
        window = [s["state"][rows, j] for j in range(K - 1)] + [s["x"]]
        pre = s["bias"].expand_as(s["x"])
        for k, row in enumerate(window):
            pre = pre + row * w[:, k]
        state = s["state_out"].clone()
        for j in range(K - 1):
            state[rows, j] = window[j + 1]
        return _silu(pre), state
    B, T, D = s["x"].shape
    lens = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    y, dx = torch.zeros_like(s["x"]), torch.zeros_like(s["x"])
    dw, db = torch.zeros_like(w), torch.zeros_like(s["bias"])
    last = []
    for b, n in enumerate(lens):
        head = s["initial"][b] if "initial" in s else s["x"].new_zeros(K - 1, D)
        ext = torch.cat([head, s["x"][b, :n]])
        pre = s["bias"].expand(n, D).clone()
        for k in range(K):
            pre += ext[k:k + n] * w[:, k]
        y[b, :n] = _silu(pre)
        last.append(ext[n:n + K - 1])
        if s["kind"] == "conv_train":
            d = s["dy"][b, :n] * _silu_slope(pre)
            dext = torch.zeros_like(ext)
            for k in range(K):
                dext[k:k + n] += d * w[:, k]
                dw[:, k] += (d * ext[k:k + n]).sum(0)
            dx[b, :n] = dext[K - 1:]
            db += d.sum(0)
    return (y, dx, dw, db) if s["kind"] == "conv_train" else (y, torch.stack(last))


def _exact_scan(s):
    A, D = s["A"], s["A"].shape[0]
    wide = lambda m: m.repeat_interleave(D // m.shape[-2], dim=-2)  # noqa: E731
    raw = s["delta"] + s["delta_bias"]
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    if s["kind"] == "scan_step":
        rows = s["slots"].long()
        h = torch.exp(dt[..., None] * A) * s["state"][rows] + (dt * s["u"])[..., None] * wide(s["Bm"])
        state = s["state_out"].clone()
        state[rows] = h
        return ((h * wide(s["Cm"])).sum(-1) + s["D"] * s["u"]) * _silu(s["z"]), state
    B, T = s["u"].shape[:2]
    lens = torch.full((B,), T, device="cuda") if s["lengths"] is None else s["lengths"]
    h = s["initial"].clone() if "initial" in s else A.new_zeros(B, D, A.shape[1])
    train = s["kind"] == "scan_train"
    states, out = [h], torch.zeros_like(s["u"])
    for t in range(T):
        on = (t < lens)[:, None, None]
        new = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * s["u"][:, t])[..., None] * wide(s["Bm"][:, t])
        h = torch.where(on, new, h)
        out[:, t] = torch.where(on[..., 0], (h * wide(s["Cm"][:, t])).sum(-1) + s["D"] * s["u"][:, t], out[:, t])
        if train:
            states.append(h)
    y = out * _silu(s["z"])
    if not train:
        return y, h
    on = (torch.arange(T, device="cuda")[None, :] < lens[:, None])[..., None]
    gate = torch.where(on, s["dy"], torch.zeros_like(s["dy"]))
    dz, dy = gate * out * _silu_slope(s["z"]), gate * _silu(s["z"])
    G, N = s["Bm"].shape[2:]
    du, ddt, dB, dC = torch.zeros_like(dy), torch.zeros_like(dy), torch.zeros_like(s["Bm"]), torch.zeros_like(s["Cm"])
    dA, g = torch.zeros_like(A), torch.zeros_like(h)
    share = lambda m: m.view(B, G, D // G, N).sum(2)  # noqa: E731
    for t in reversed(range(T)):
        live = on[:, t, :, None]
        g = g + dy[:, t, :, None] * wide(s["Cm"][:, t])
        dC[:, t] = share(dy[:, t, :, None] * states[t + 1])
        decay = torch.exp(dt[:, t, :, None] * A)
        gt = torch.where(live, g, torch.zeros_like(g))
        dB[:, t] = share(gt * (dt[:, t] * s["u"][:, t])[..., None])
        gB = (gt * wide(s["Bm"][:, t])).sum(-1)
        du[:, t] = gB * dt[:, t] + s["D"] * dy[:, t]
        w = gt * decay * states[t]
        ddt[:, t] = gB * s["u"][:, t] + (w * A).sum(-1)
        dA += (w * dt[:, t, :, None]).sum(0)
        g = torch.where(live, g * decay, g)
    ddelta = ddt * torch.sigmoid(raw)
    return y, du, ddelta, dA, dB, dC, (dy * s["u"]).sum((0, 1)), dz, ddelta.sum((0, 1))
