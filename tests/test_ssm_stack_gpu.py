"""The `SSM` stack on the GPU: values and all gradients against the same stack written with elementary torch operations in
float64 (autograd), its token-by-token form, its input forms, and the places where it stands in for the GRU -- the TimeGAN
networks, the trainer (eager and as graphs) and the scorer."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def tg():
    import timegan_amd
    return timegan_amd


def plain_layer(layer, x, lengths=None, state=None):
    """SSMLayer.forward by elementary operations, in x's type, differentiable."""
    B, T, _ = x.shape
    p = {k: v.to(x.dtype) for k, v in layer.items()}
    N, K = p["A_log"].shape[1], p["conv_weight"].shape[1]
    R = p["dt_proj.weight"].shape[1]
    x, z = (x @ p["in_proj.weight"].t()).chunk(2, -1)
    ext = torch.cat([x.new_zeros(B, K - 1, x.shape[2]) if state is None else state[0], x], 1)
    x = F.silu(p["conv_bias"] + sum(ext[:, k:k + T] * p["conv_weight"][:, k] for k in range(K)))
    dt, Bm, Cm = (x @ p["x_proj.weight"].t()).split([R, N, N], -1)
    raw = dt @ p["dt_proj.weight"].t() + p["dt_bias"]
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    A = -torch.exp(p["A_log"])
    h = x.new_zeros(B, x.shape[2], N) if state is None else state[1]
    ys = []
    for t in range(T):
        on = torch.ones(B, 1, 1, dtype=torch.bool) if lengths is None else (torch.tensor(lengths) > t)[:, None, None]
        new = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * x[:, t])[..., None] * Bm[:, t, None, :]
        h = torch.where(on, new, h)
        y = (h * Cm[:, t, None, :]).sum(-1) + p["D"] * x[:, t]
        ys.append(torch.where(on[..., 0], y * F.silu(z[:, t]), torch.zeros_like(y)))
    return torch.stack(ys, 1) @ p["out_proj.weight"].t(), h


def plain_stack(m, x, dtype, lengths=None):
    """(output, last layer's scan state, parameters as leaves by name) on the CPU in `dtype`."""
    params = {n: p.detach().cpu().to(dtype).requires_grad_(True) for n, p in m.named_parameters()}
    for k in range(m.num_layers):
        x, h = plain_layer({n.split(".", 2)[2]: p for n, p in params.items() if n.startswith(f"layers.{k}.")}, x, lengths)
    return x, h, params


def near(got, ref, single, what):
    """The kernels round as often as the same formulas in float32 elsewhere, in another order: their distance from 64 bits is
    allowed eight times that of float32 on the CPU (largest element against largest element), plus 64 half steps of the
    largest value for a case that happens to round exactly there."""
    got, ref, single = (v.detach().cpu().double() for v in (got, ref, single))
    assert got.shape == ref.shape, what
    allowed = 8 * float((single - ref).abs().max()) + 64 * 2 ** -24 * float(ref.abs().max())
    assert float((got - ref).abs().max()) <= allowed, f"{what}: {float((got - ref).abs().max()):.3g} allowed {allowed:.3g}"


@pytest.mark.parametrize("kw", [dict(B=4, T=24, In=6, H=24, L=2), dict(B=3, T=33, In=10, H=20, L=1, state_size=9, conv_width=3, expand=1),
                                dict(B=2, T=50, In=5, H=16, L=2, lengths=[50, 17])], ids=str)
def test_value_and_all_gradients(tg, kw):
    B, T, In, H, L = (kw.pop(k) for k in ("B", "T", "In", "H", "L"))
    lengths = kw.pop("lengths", None)
    torch.manual_seed(1)
    m = tg.SSM(In, H, L, batch_first=True, **kw).to(DEV)
    x, dy = torch.randn(B, T, In), torch.randn(B, T, H)
    outs = {}
    for dtype in (torch.float64, torch.float32):
        leaf = x.to(dtype).requires_grad_(True)
        y, h, params = plain_stack(m, leaf, dtype, lengths)
        grads = torch.autograd.grad(y, [leaf] + list(params.values()), dy.to(dtype))
        outs[dtype] = (y, h, dict(zip(["input"] + list(params), grads)))
    leaf = x.to(DEV).requires_grad_(True)
    y, state = m(leaf, lengths=lengths)
    named = dict(m.named_parameters())
    grads = dict(zip(["input"] + list(named), torch.autograd.grad(y, [leaf] + list(named.values()), dy.to(DEV))))
    ref, single = outs[torch.float64], outs[torch.float32]
    near(y, ref[0], single[0], "output")
    near(state.scan[-1], ref[1], single[1], "state")
    for n, g in grads.items():
        near(g, ref[2][n], single[2][n], n)


def test_input_forms_agree(tg):
    torch.manual_seed(2)
    m = tg.SSM(7, 16, 2, batch_first=True).to(DEV)
    t = tg.SSM(7, 16, 2).to(DEV)
    t.load_state_dict(m.state_dict())
    x = torch.randn(4, 21, 7, device=DEV)
    lengths = [5, 21, 1, 13]
    y, s = m(x, lengths=lengths)
    assert not y[0, 5:].any() and not y[2, 1:].any()
    yt, st = t(x.transpose(0, 1), lengths=torch.tensor(lengths))
    single = plain_stack(m, x.cpu(), torch.float32, lengths)[0]
    ref = plain_stack(m, x.cpu().double(), torch.float64, lengths)[0]
    near(y, ref, single, "batch first")
    near(yt.transpose(0, 1), ref, single, "time first")
    packed = torch.nn.utils.rnn.pack_padded_sequence(x, lengths, batch_first=True, enforce_sorted=False)
    yp, sp = m(packed)
    back, lens = torch.nn.utils.rnn.pad_packed_sequence(yp, batch_first=True)
    assert lens.tolist() == lengths
    near(back, ref, single, "packed")
    near(sp.scan[1], s.scan[1].double(), s.scan[1] * (1 + 2 ** -20), "packed state")
    order = sorted(range(4), key=lambda i: -lengths[i])
    srt = torch.nn.utils.rnn.pack_padded_sequence(x[order], [lengths[i] for i in order], batch_first=True)
    ys, _ = m(srt)
    assert ys.sorted_indices is None and torch.equal(ys.batch_sizes, srt.batch_sizes)
    near(torch.nn.utils.rnn.pad_packed_sequence(ys, batch_first=True)[0], ref[order], single[order], "sorted")
    one, _ = m(x[1])
    near(one, ref[1], single[1], "one sequence")
    a, s1 = m(x[:, :8])
    b, s2 = m(x[:, 8:], s1)
    whole = plain_stack(m, x.cpu().double(), torch.float64)[0]
    near(torch.cat([a, b], 1), whole, plain_stack(m, x.cpu(), torch.float32)[0], "two calls")


@pytest.mark.parametrize("pool", [False, True])
def test_tokens_one_by_one(tg, pool):
    torch.manual_seed(3)
    m = tg.SSM(6, 24, 2, batch_first=True).to(DEV)
    x = torch.randn(5, 12, 6, device=DEV)
    ref, h, _ = plain_stack(m, x.cpu().double(), torch.float64)
    single, h32, _ = plain_stack(m, x.cpu(), torch.float32)
    with torch.no_grad():
        if pool:
            state, slots, out, start = m.init_state(9), torch.tensor([7, 0, 3, 8, 1]), [], 0
        else:
            y, state = m(x[:, :7])
            slots, out, start = None, list(y.unbind(1)), 7
        for t in range(start, 12):
            out.append(m.step(x[:, t], state, slots))
    near(torch.stack(out, 1), ref, single, "outputs")
    near(state.scan[1] if slots is None else state.scan[1][slots.to(DEV)], h, h32, "state")
    if pool:
        assert not state.scan[0][[2, 4, 5, 6]].any() and not state.conv[1][[2, 4, 5, 6]].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_sixteen_bit_stack(tg, dtype):
    """Runs in the type throughout; about a dozen roundings of half a step each (2^-8, 2^-11) lie between input and output of
    a layer, and values near the largest one are amplified little: an eighth of the largest value covers two layers of
    bfloat16 four times over."""
    torch.manual_seed(4)
    m = tg.SSM(6, 24, 2, batch_first=True, dtype=dtype).to(DEV)
    x = torch.randn(3, 20, 6).to(dtype)
    y, s = m(x.to(DEV).requires_grad_(True))
    y.float().square().sum().backward()
    assert y.dtype == dtype and s.conv[0].dtype == dtype and s.scan[0].dtype == torch.float32
    assert all(p.grad is not None and p.grad.dtype == dtype and torch.isfinite(p.grad).all() for p in m.parameters())
    ref = plain_stack(m, x.double(), torch.float64)[0].detach()
    assert float((y.detach().cpu().double() - ref).abs().max()) < float(ref.abs().max()) / 8
    with torch.no_grad():
        st = m.init_state(3)
        steps = torch.stack([m.step(x[:, t].to(DEV), st) for t in range(20)], 1)
    assert float((steps.cpu().double() - ref).abs().max()) < float(ref.abs().max()) / 8


@pytest.mark.parametrize("graphs", [False, True])
def test_trainer_on_the_stack(tg, graphs):
    """The three phases with every recurrent layer replaced: losses are finite, every network is updated, and replays of the
    captured steps equal eager steps."""
    cfg = tg.make_cfg(features=5, hidden=12, layers=2, seq_len=24, batch_size=16)
    g = torch.Generator().manual_seed(0)
    batches = [torch.rand(16, 24, 5, generator=g).to(DEV) for _ in range(4)]

    def run(graphs):
        torch.manual_seed(7)
        tr = tg.TimeGANTrainer(cfg, rnn_cls=tg.SSM, use_graphs=graphs, counter_noise=True)
        before = {k: [p.detach().clone() for p in n.parameters()] for k, n in tr.nets.items()}
        losses = []
        for x in batches:
            losses.append(float(torch.as_tensor(tr.embedding_step(x))))
        for x in batches:
            losses.append(float(torch.as_tensor(tr.supervisor_step(x))))
        for x in batches:
            losses += [float(torch.as_tensor(v)) for v in np.ravel(_flat(tr.joint_step(x)))]
        changed = {k: any(not torch.equal(a, b) for a, b in zip(before[k], n.parameters())) for k, n in tr.nets.items()}
        return losses, changed, tr

    losses, changed, tr = run(graphs)
    assert all(math.isfinite(v) for v in losses)
    assert all(changed[k] for k in ("emb", "rec", "sup", "g")), changed
    if graphs:
        eager, _, te = run(False)
        # the same kernels on the same inputs; Adam divides by roots of tiny second moments, which turns last bits of a
        # gradient into up to lr / step of a weight
        for a, b in zip(losses, eager):
            assert abs(a - b) <= 1e-3 * max(1.0, abs(b)), (losses, eager)


def _flat(v):
    if isinstance(v, dict):
        v = list(v.values())
    if isinstance(v, (list, tuple)):
        out = []
        for x in v:
            out += _flat(x)
        return out
    return [] if v is None else [float(torch.as_tensor(v))]


def test_scorer_on_the_stack(tg):
    cfg = {"rnn": {"type": "ssm", "dim_input": 5, "dim_output": 1, "dim_hidden": 8, "num_layers": 1, "dropout": 0.0, "bidirectional": "false"}}
    net = tg.scorer.GeneralRNN(cfg).to(DEV)
    assert isinstance(net.rnn, tg.SSM)
    out = net(torch.rand(24, 7, 5, device=DEV))
    assert out.shape == (24, 7, 1) and bool(((out > 0) & (out < 1)).all())
    rng = np.random.default_rng(0)
    real, synth = rng.random((40, 24, 5)).astype(np.float32), rng.random((40, 24, 5)).astype(np.float32)
    assert 0.0 <= tg.scorer.discriminative_score(real, synth, DEV, hidden=8, steps=3, batch=16, rnn_cls=tg.SSM) <= 0.5
    assert tg.scorer.predictive_score(real, synth, DEV, hidden=8, steps=3, batch=16, rnn_cls=tg.SSM) >= 0.0


def test_a_dropped_trainer_is_not_collected_during_a_capture(tg, monkeypatch):
    """The graphs of a trainer that nobody holds any more go before the next capture begins, not inside it."""
    import gc
    import weakref
    cfg = tg.make_cfg(features=5, hidden=8, layers=1, seq_len=24, batch_size=4)
    x = torch.rand(4, 24, 5, device=DEV)

    def trained():
        tr = tg.TimeGANTrainer(cfg, use_graphs=True)
        for _ in range(3):
            tr.embedding_step(x)
        return tr

    gc.disable()
    try:
        gone = weakref.ref(trained())
        assert gone() is not None, "the trainer is a cycle: only the collector frees it"
    finally:
        gc.enable()
    state = []
    real = torch.cuda.graph.__enter__
    monkeypatch.setattr(torch.cuda.graph, "__enter__", lambda self: (state.append((gone() is None, gc.isenabled())), real(self))[1])
    trained()
    assert state == [(True, False)] and gc.isenabled()
