"""The state-space operators on the GPU against their definition in float64 (ssm_reference.py, which also derives the
bounds): values and gradients over types, odd sizes, groups, lengths, strides; the one-token forms and their pools; streams
and graphs; and the `SSM` stack in the places of the GRU."""
import gc

import pytest
import torch

import ssm_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def tg():
    import timegan_amd
    return timegan_amd


def randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def cuda(v):
    return v.to(DEV) if torch.is_tensor(v) else v


def leaf(v):
    return None if v is None else v.to(DEV).requires_grad_(True)


def case_scan(seed, B, T, D, N, G, dtype, z=True, skip=True, bias=True, initial=True, lengths=None):
    g = torch.Generator().manual_seed(seed)
    c = dict(u=randn(g, B, T, D, dtype=dtype), delta=randn(g, B, T, D, dtype=dtype, scale=0.7),
             A=-torch.exp(randn(g, D, N, scale=0.8)), Bm=randn(g, B, T, G, N, dtype=dtype), Cm=randn(g, B, T, G, N, dtype=dtype),
             D=randn(g, D) if skip else None, z=randn(g, B, T, D, dtype=dtype, scale=2.0) if z else None,
             delta_bias=randn(g, D) - 2.0 if bias else None, initial=randn(g, B, D, N) if initial else None, lengths=lengths)
    c["dy"], c["dfinal"] = randn(g, B, T, D, dtype=dtype), randn(g, B, D, N)
    return c


ORDER = ("u", "delta", "A", "Bm", "Cm", "D", "z", "delta_bias")


def run_scan(tg, c, softplus=True, view=lambda k, v: v, device_lengths=True):
    leaves = {k: leaf(c[k]) for k in ORDER + ("initial",)}
    args = [None if leaves[k] is None else view(k, leaves[k]) for k in ORDER]
    lens = c["lengths"]
    if lens is not None and device_lengths:
        lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    y, h = tg.selective_scan(*args, softplus=softplus, initial_state=leaves["initial"], lengths=lens, return_state=True)
    names = [k for k in leaves if leaves[k] is not None]
    grads = torch.autograd.grad([y, h], [leaves[k] for k in names], [cuda(c["dy"]), cuda(c["dfinal"])])
    return y, h, dict(zip(names, grads))


def check_scan(c, got, softplus=True):
    B, T, D = c["u"].shape
    kw = dict(softplus=softplus, initial=c["initial"], lengths=c["lengths"], dy=c["dy"], dfinal=c["dfinal"])
    args = [c[k] for k in ORDER]
    want, size = ref.scan(*args, **kw), ref.scan(*args, absolute=True, **kw)
    y, h, grads = got
    ref.close(y, want[0], size[0], T, what="y")
    ref.close(h, want[1], size[1], T, what="state")
    rename = {"Bm": "B", "Cm": "C"}
    for k, g in grads.items():
        n = rename.get(k, k)
        ref.close(g, want[2][n], size[2][n], T, B, D, what=f"gradient of {k}")


# one block and several, a block's edge and beyond, every number of lanes per channel (N up to 4, 8, 16, 32, 64), groups
# narrower and wider than a wave, one workgroup per group and several
SIZES = [(1, 1, 1, 1, 1), (2, 15, 5, 3, 1), (3, 16, 17, 4, 1), (2, 17, 64, 8, 2), (5, 33, 48, 16, 1), (2, 40, 150, 16, 2),
         (1, 50, 36, 11, 4), (3, 31, 20, 32, 5), (2, 48, 9, 64, 3), (2, 20, 7, 24, 7), (1, 64, 300, 5, 1)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("B,T,D,N,G", SIZES)
def test_scan_value_and_gradients(tg, B, T, D, N, G, dtype):
    c = case_scan(B * 1000 + T, B, T, D, N, G, dtype)
    check_scan(c, run_scan(tg, c))


@pytest.mark.parametrize("kw", [dict(z=False), dict(skip=False), dict(bias=False), dict(initial=False),
                                dict(z=False, skip=False, bias=False, initial=False)], ids=str)
def test_scan_without_optional_inputs(tg, kw):
    c = case_scan(3, 2, 37, 40, 16, 2, torch.float32, **kw)
    check_scan(c, run_scan(tg, c))


def test_scan_without_softplus_and_with_negative_steps(tg):
    c = case_scan(4, 2, 30, 24, 16, 1, torch.float32, bias=False)
    c["delta"] = c["delta"] * 0.1
    check_scan(c, run_scan(tg, c, softplus=False), softplus=False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lengths", [[40, 0, 1, 16, 17, 39], [0, 0, 0, 0, 0, 0], [1, 40, 3, 15, 32, 33]], ids=str)
def test_scan_lengths_and_what_lies_behind_them(tg, lengths, dtype):
    """Rows behind a sequence's end may hold anything; outputs and gradients there are zero, a sequence of length 0 keeps
    its state, and the state's gradient passes through it."""
    c = case_scan(5, 6, 40, 21, 16, 3, dtype, lengths=lengths)
    on = torch.arange(40)[None, :] < torch.tensor(lengths)[:, None]
    clean = dict(c)
    for k, junk in (("u", float("nan")), ("delta", float("inf")), ("Bm", float("nan")), ("Cm", float("-inf")),
                    ("z", torch.finfo(dtype).min), ("dy", float("nan"))):
        c[k] = torch.where(on.view(6, 40, *[1] * (c[k].dim() - 2)), c[k], torch.full_like(c[k], junk))
    got = run_scan(tg, c)
    check_scan(clean, got)
    assert not got[0].cpu()[~on].any() and not got[2]["u"].cpu()[~on].any() and not got[2]["Bm"].cpu()[~on].any()
    host = run_scan(tg, c, device_lengths=False)
    assert torch.equal(got[0], host[0]) and torch.equal(got[2]["A"], host[2]["A"])


@pytest.mark.parametrize("lengths", [None, [300, 0, 131]], ids=str)
@pytest.mark.parametrize("N,G", [(16, 1), (5, 2), (33, 1)])
def test_scan_in_chunks_of_time(tg, N, G, lengths):
    """Few channels and many steps: the launch is cut along time and joined."""
    B = 3 if lengths else 1
    c = case_scan(6, B, 300, 24, N, G, torch.float32, lengths=lengths)
    check_scan(c, run_scan(tg, c))


def test_scan_with_decays_that_vanish(tg):
    """A = -inf forgets the state at every step; a length that ends inside a block must not turn that into 0 * inf."""
    c = case_scan(7, 2, 300, 8, 4, 1, torch.float32, lengths=[300, 21])
    c["A"] = torch.full_like(c["A"], float("-inf"))
    y, h = tg.selective_scan(*[cuda(c[k]) for k in ORDER], initial_state=cuda(c["initial"]), return_state=True,
                             lengths=torch.tensor(c["lengths"], dtype=torch.int32, device=DEV))
    c["A"] = torch.full_like(c["A"], -1e30)
    args = [c[k] for k in ORDER]
    kw = dict(initial=c["initial"], lengths=c["lengths"])
    want, size = ref.scan(*args, **kw), ref.scan(*args, absolute=True, **kw)
    ref.close(y, want[0], size[0], 300, what="y")
    ref.close(h, want[1], size[1], 300, what="state")


def test_scan_strides_broadcasts_and_offsets(tg):
    """Time-major inputs, halves of a wider tensor, a start off any alignment, channels that are not consecutive, maps shared
    by all sequences: the same numbers, and gradients in the shape of what was passed."""
    c = case_scan(8, 3, 26, 30, 16, 2, torch.bfloat16)
    for k in ("Bm", "Cm"):
        c[k] = c[k][:1].expand(3, -1, -1, -1)
    plain = run_scan(tg, c)
    wide = torch.empty(3, 26, 91, dtype=torch.bfloat16, device=DEV)

    def view(k, v):
        if k == "u":
            return v.transpose(0, 1).contiguous().transpose(0, 1)
        if k == "delta":
            return torch.cat([wide[..., :7] * 0, v, wide[..., :9] * 0], -1)[..., 7:37]
        if k == "z":
            return v.transpose(1, 2).contiguous().transpose(1, 2)
        if k == "Bm":
            return v[:1].expand(3, -1, -1, -1)
        return v

    wide.zero_()
    other = run_scan(tg, c, view=view)
    assert torch.equal(plain[0], other[0]) and torch.equal(plain[1], other[1])
    for k in ("u", "delta", "z", "A", "Cm", "D", "delta_bias", "initial"):
        assert torch.equal(plain[2][k], other[2][k]), k
    total = plain[2]["Bm"].double().sum(0)
    assert torch.allclose(other[2]["Bm"][0].double(), total, rtol=0, atol=float(total.abs().max()) * 3 * 2 ** -8)


def test_offsets_beyond_32_bits(tg):
    """Rows that lie more than 2^31 elements apart."""
    B, T, D, step = 2, 280, 40, 1 << 22
    big = torch.empty(B, T, step, dtype=torch.bfloat16, device=DEV)
    c = case_scan(9, B, T, D, 16, 1, torch.bfloat16)
    views = {k: big[..., i * 64:i * 64 + D] for i, k in enumerate(("u", "delta", "z", "x", "dy"))}
    for k in ("u", "delta", "z"):
        views[k].copy_(c[k])
    views["x"].copy_(c["u"])
    args = [views[k] if k in views else cuda(c[k]) for k in ORDER]
    dense = [cuda(c[k]) for k in ORDER]
    assert B * T * step > 2 ** 31
    assert torch.equal(tg.selective_scan(*args), tg.selective_scan(*dense))
    w = randn(torch.Generator().manual_seed(1), D, 4).to(DEV)
    assert torch.equal(tg.short_conv(views["x"], w), tg.short_conv(cuda(c["u"]), w))
    leaves = [a.detach().requires_grad_(True) for a in args]
    views["dy"].copy_(c["dy"])
    got = torch.autograd.grad(tg.selective_scan(*leaves), leaves, views["dy"])
    leaves = [a.detach().requires_grad_(True) for a in dense]
    for a, b in zip(got, torch.autograd.grad(tg.selective_scan(*leaves), leaves, cuda(c["dy"]))):
        assert torch.equal(a, b)


def test_steps_almost_too_far_apart_to_be_read_in_place(tg):
    B, T, D, step = 1, 20, 24, (1 << 25) - 64
    c = case_scan(11, B, T, D, 16, 1, torch.float32)
    big = torch.empty(T, step, device=DEV)
    views = {k: big.as_strided((B,) + tuple(c[k].shape[1:]), (0, step, 16, 1)[:c[k].dim() - 1] + (1,), 64 * i)
             for i, k in enumerate(("u", "delta", "Bm", "Cm", "z", "dy"))}
    for k, v in views.items():
        v.copy_(c[k])
    leaves = [(views[k] if k in views else cuda(c[k])).detach().requires_grad_(True) for k in ORDER]
    dense = [cuda(c[k]).requires_grad_(True) for k in ORDER]
    y, want = tg.selective_scan(*leaves), tg.selective_scan(*dense)
    assert torch.equal(y, want)
    for a, b in zip(torch.autograd.grad(y, leaves, views["dy"]), torch.autograd.grad(want, dense, cuda(c["dy"]))):
        assert torch.equal(a, b)


def test_gradients_of_more_rows_and_columns_than_one_launch_has_workgroups_for(tg):
    def grads(args):
        leaves = [a.detach().requires_grad_(True) for a in args]
        return torch.autograd.grad(tg.selective_scan(*leaves), leaves, leaves[0].detach())

    dev = torch.Generator(device=DEV).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=dev, device=DEV)  # noqa: E731
    B, T, D, N = 560000, 16, 4, 16                                   # 2 B T N > 2^28
    args = [rnd(B, T, D), rnd(B, T, D), -rnd(D, N).abs(), rnd(B, T, 1, N), rnd(B, T, 1, N), rnd(D)]
    many = grads(args)
    for part in (slice(0, 3), slice(B - 3, B)):
        few = grads([a[part] if a.shape[0] == B else a for a in args])
        for k in (0, 1, 3, 4):
            assert torch.equal(many[k][part], few[k])
    D = 300000                                                       # D (N + 2) > 2^22
    args = [rnd(1, 2, D), rnd(1, 2, D), -rnd(D, N).abs(), rnd(1, 2, 1, N), rnd(1, 2, 1, N), rnd(D)]
    many = grads(args)
    part = slice(D - 32, D)
    few = grads([args[0][..., part], args[1][..., part], args[2][part], args[3], args[4], args[5][part]])
    for k in (2, 5):
        assert torch.equal(many[k][part], few[k]) and torch.equal(many[k][:32], grads(
            [args[0][..., :32], args[1][..., :32], args[2][:32], args[3], args[4], args[5][:32]])[k])


def test_steps_that_lie_far_apart(tg):
    """Steps 2^26 elements apart and more: copied in front of the scan, and the results too where they would lie like that."""
    B, T, D, step = 2, 3, 8, 1 << 26
    c = case_scan(10, B, T, D, 16, 1, torch.bfloat16)
    big = torch.empty(T, step, dtype=torch.bfloat16, device=DEV)
    far = lambda i, *shape: big.as_strided(shape, (64, step, 16, 1)[:len(shape) - 1] + (1,), 1024 * i)  # noqa: E731
    views = {k: far(i, *c[k].shape) for i, k in enumerate(("u", "delta", "Bm", "Cm", "z", "dy"))}
    for k, v in views.items():
        assert v.stride(1) >= step
        v.copy_(c[k])
    leaves = [(views[k] if k in views else cuda(c[k])).detach().requires_grad_(True) for k in ORDER]
    y, h = tg.selective_scan(*leaves, initial_state=cuda(c["initial"]), return_state=True)
    grads = torch.autograd.grad([y, h], leaves, [views["dy"], cuda(c["dfinal"])])
    dense = [cuda(c[k]).requires_grad_(True) for k in ORDER]
    want, state = tg.selective_scan(*dense, initial_state=cuda(c["initial"]), return_state=True)
    assert torch.equal(y, want) and torch.equal(h, state)
    for a, b in zip(grads, torch.autograd.grad([want, state], dense, [cuda(c["dy"]), cuda(c["dfinal"])])):
        assert torch.equal(a, b)
    # (T, B, D) with so many sequences that a step of the result in that order would be too long
    B, T, D = 1 << 16, 2, 1024
    u = torch.randn(T, B, D, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    A, b = -torch.ones(D, 4, device=DEV), torch.ones(1, 1, 1, 4, dtype=torch.bfloat16, device=DEV).expand(B, T, 1, 4)
    y = tg.selective_scan(u, u, A, b, b)
    few = u[-3:].contiguous()
    assert torch.equal(y[-3:], tg.selective_scan(few, few, A, b[-3:], b[-3:]))


# ---- convolution -----------------------------------------------------------------------------------------------------

def case_conv(seed, B, T, D, K, dtype, bias=True, initial=True, lengths=None):
    g = torch.Generator().manual_seed(seed)
    return dict(x=randn(g, B, T, D, dtype=dtype), weight=randn(g, D, K, scale=0.6), bias=randn(g, D) if bias else None,
                initial=randn(g, B, K - 1, D, dtype=dtype) if initial else None, lengths=lengths,
                dy=randn(g, B, T, D, dtype=dtype), dfinal=randn(g, B, K - 1, D, dtype=dtype))


def run_conv(tg, c, act, view=lambda v: v):
    leaves = {k: leaf(c[k]) for k in ("x", "weight", "bias", "initial")}
    lens = None if c["lengths"] is None else torch.tensor(c["lengths"], dtype=torch.int32, device=DEV)
    y, s = tg.short_conv(view(leaves["x"]), leaves["weight"], leaves["bias"], silu=act, initial_state=leaves["initial"], lengths=lens,
                         return_state=True)
    names = [k for k in leaves if leaves[k] is not None]
    grads = torch.autograd.grad([y, s], [leaves[k] for k in names], [cuda(c["dy"]), cuda(c["dfinal"])], allow_unused=True)
    return y, s, dict(zip(names, grads))


def check_conv(c, got, act):
    B, T, D = c["x"].shape
    kw = dict(initial=c["initial"], lengths=c["lengths"], dy=c["dy"], dfinal=c["dfinal"], act=act)
    want, size = (ref.conv(c["x"], c["weight"], c["bias"], absolute=a, **kw) for a in (False, True))
    ref.close(got[0], want[0], size[0], 1, what="y")
    assert torch.equal(got[1].cpu().double(), want[1])
    for k, g in got[2].items():
        ref.close(g, want[2][k], size[2][k], T if k in ("weight", "bias") else 1, B, what=f"gradient of {k}")


@pytest.mark.parametrize("act", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("B,T,D,K", [(1, 1, 1, 2), (2, 3, 8, 4), (3, 7, 24, 8), (2, 8, 16, 4), (2, 9, 33, 3), (1, 130, 40, 5),
                                     (4, 66, 64, 4), (1, 17, 100, 1), (2, 29, 7, 7), (3, 24, 48, 6)])
def test_conv_value_and_gradients(tg, B, T, D, K, dtype, act):
    c = case_conv(B * 100 + T, B, T, D, K, dtype)
    check_conv(c, run_conv(tg, c, act), act)


@pytest.mark.parametrize("kw", [dict(bias=False), dict(initial=False), dict(bias=False, initial=False)], ids=str)
def test_conv_without_optional_inputs(tg, kw):
    c = case_conv(3, 2, 21, 24, 4, torch.float32, **kw)
    check_conv(c, run_conv(tg, c, True), True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", [16, 13])
def test_conv_lengths_and_what_lies_behind_them(tg, D, dtype):
    """Shorter than the taps, zero, a run's edge; NaN behind the end."""
    lengths = [40, 0, 1, 2, 3, 8, 31, 32]
    c = case_conv(5, 8, 40, D, 4, dtype, lengths=lengths)
    on = torch.arange(40)[None, :] < torch.tensor(lengths)[:, None]
    clean = dict(c)
    for k in ("x", "dy"):
        c[k] = torch.where(on[..., None], c[k], torch.full_like(c[k], float("nan")))
    got = run_conv(tg, c, True)
    check_conv(clean, got, True)
    assert not got[0].cpu()[~on].any() and not got[2]["x"].cpu()[~on].any()


@pytest.mark.parametrize("B,T,D,K,dtype", [(3000, 9, 3, 4, torch.float32), (700, 40, 13, 3, torch.bfloat16), (2100, 5, 9, 1, torch.float16),
                                           (5000, 3, 17, 8, torch.float32)])
def test_conv_parameter_gradients_over_many_sequences(tg, B, T, D, K, dtype):
    """More rows of partial sums than are added in one launch."""
    g = torch.Generator().manual_seed(B)
    c = case_conv(B, B, T, D, K, dtype, lengths=torch.randint(0, T + 1, (B,), generator=g).tolist())
    check_conv(c, run_conv(tg, c, True), True)


def test_conv_gradients_of_millions_of_sequences(tg):
    """Two million rows, against sums in 64 bits.  A term is rounded once and goes through two rounds of at most 128 rows of a
    thread, 16 partial sums and 32 threads: less than 384 roundings of 2^-24 each."""
    B, D, K = 2200000, 2, 2
    dev = torch.Generator(device=DEV).manual_seed(1)
    x, dy = (torch.randn(B, 1, D, generator=dev, device=DEV) for _ in range(2))
    w, b = torch.randn(D, K, generator=dev, device=DEV).requires_grad_(True), torch.zeros(D, device=DEV, requires_grad=True)
    dw, db = torch.autograd.grad(tg.short_conv(x, w, b, silu=False), (w, b), dy)
    want, size = (dy.double() * x.double()).sum((0, 1)), (dy.double() * x.double()).abs().sum((0, 1))
    eps = 384 * 2.0 ** -24
    assert ((dw[:, -1].double() - want).abs() <= eps * size).all() and not dw[:, 0].any()
    assert ((db.double() - dy.double().sum((0, 1))).abs() <= eps * dy.double().abs().sum((0, 1))).all()


def test_conv_strides_and_alignment(tg):
    c = case_conv(6, 3, 50, 32, 4, torch.bfloat16)
    plain = run_conv(tg, c, True)
    for view in (lambda v: v.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda v: torch.cat([v, v], -1)[..., 32:],
                 lambda v: torch.cat([v[..., :3], v], -1)[..., 3:],
                 lambda v: v.transpose(1, 2).contiguous().transpose(1, 2)):
        other = run_conv(tg, c, True, view)
        assert torch.equal(plain[0], other[0]) and torch.equal(plain[1], other[1])
        assert torch.equal(plain[2]["x"], other[2]["x"]) and torch.equal(plain[2]["initial"], other[2]["initial"])
        for k in ("weight", "bias"):      # another cut of the sums: both within the bound
            check_conv(c, (other[0], other[1], {k: other[2][k]}), True)


# ---- one token, pools ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("B,D,N,G,K", [(1, 1, 1, 1, 2), (3, 40, 16, 1, 4), (5, 33, 11, 3, 3), (2, 128, 64, 2, 8), (70, 8, 4, 1, 4), (4, 24, 30, 4, 5)])
def test_steps_go_on_from_a_prompt(tg, B, D, N, G, K, dtype):
    """A prompt's states, then tokens one by one, equal the whole sequence at once; y of a step is y of the sequence."""
    T, cut = 12, 7
    c, cc = case_scan(B, B, T, D, N, G, dtype), case_conv(B, B, T, D, K, dtype)
    s = {k: cuda(c[k]) for k in ORDER}
    x, w, b, x0 = (cuda(cc[k]) for k in ("x", "weight", "bias", "initial"))
    head = [s[k][:, :cut] if s[k].dim() > 2 else s[k] for k in ORDER]
    y, h = tg.selective_scan(*head, initial_state=cuda(c["initial"]), return_state=True)
    yc, hc = tg.short_conv(x[:, :cut], w, b, initial_state=x0, return_state=True)
    ys, ycs = [y], [yc]
    for t in range(cut, T):
        ys.append(tg.selective_scan_step(s["u"][:, t], s["delta"][:, t], h, s["A"], s["Bm"][:, t], s["Cm"][:, t], s["D"], s["z"][:, t],
                                         s["delta_bias"])[:, None])
        ycs.append(tg.short_conv_step(x[:, t], hc, w, b)[:, None])
    args = [c[k] for k in ORDER]
    want, size = (ref.scan(*args, initial=c["initial"], absolute=a) for a in (False, True))
    ref.close(torch.cat(ys, 1), want[0], size[0], T, what="y")
    ref.close(h, want[1], size[1], T, what="state")
    want, size = (ref.conv(cc["x"], cc["weight"], cc["bias"], initial=cc["initial"], absolute=a) for a in (False, True))
    ref.close(torch.cat(ycs, 1), want[0], size[0], 1, what="convolution")
    assert torch.equal(hc.cpu().double(), want[1])


@pytest.mark.parametrize("D", [24, 21])
@pytest.mark.parametrize("out_of_place", [False, True])
def test_pools_slots_padding_and_repeats(tg, D, out_of_place):
    """Rows with a slot outside the pool are padding; rows with the same slot are taken in order; states that no row names
    stay as they were, to the bit."""
    B, P, N, K = 300, 40, 16, 4
    g = torch.Generator().manual_seed(2)
    slots = torch.randint(0, 30, (B,), generator=g)
    slots[5], slots[17], slots[200] = -1, 40, -2 ** 31
    c, cc = case_scan(1, B, 1, D, N, 1, torch.float32), case_conv(1, B, 1, D, K, torch.float32)
    pool, cpool = randn(g, P, D, N), randn(g, P, K - 1, D)
    y_want, h_want = torch.zeros(B, D, dtype=torch.float64), pool.double().clone()
    yc_want, x_want = torch.zeros(B, D, dtype=torch.float64), cpool.double().clone()
    for i, p in enumerate(slots.tolist()):
        if 0 <= p < P:
            row = [c[k][i:i + 1] if c[k].dim() > 2 else c[k] for k in ORDER]
            y, h, _ = ref.scan(*row, initial=h_want[p:p + 1])
            y_want[i], h_want[p] = y[0, 0], h[0]
            y, x, _ = ref.conv(cc["x"][i:i + 1], cc["weight"], cc["bias"], initial=x_want[p:p + 1])
            yc_want[i], x_want[p] = y[0, 0], x[0]
    s = {k: cuda(c[k]) for k in ORDER}
    state, cstate = pool.to(DEV), cpool.to(DEV)
    kw = dict(slots=slots.to(torch.int32).to(DEV))
    scan_out, conv_out = (state.clone(), cstate.clone()) if out_of_place else (None, None)
    y = tg.selective_scan_step(s["u"][:, 0], s["delta"][:, 0], state, s["A"], s["Bm"][:, 0], s["Cm"][:, 0], s["D"], s["z"][:, 0],
                               s["delta_bias"], state_out=scan_out, **kw)
    yc = tg.short_conv_step(cuda(cc["x"])[:, 0], cstate, cuda(cc["weight"]), cuda(cc["bias"]), state_out=conv_out, **kw)
    if out_of_place:
        assert torch.equal(state.cpu(), pool) and torch.equal(cstate.cpu(), cpool)
        state, cstate = scan_out, conv_out
    # at most 30 steps on one slot; values stay below 100 in the sum of their absolute terms
    tol = (8 * 30 + 64) * ref.EPS * 100
    assert float((y.cpu().double() - y_want).abs().max()) < tol and float((state.cpu().double() - h_want).abs().max()) < tol
    assert float((yc.cpu().double() - yc_want).abs().max()) < tol and torch.equal(cstate.cpu().double(), x_want)
    assert torch.equal(state.cpu()[30:], pool[30:])
    for i in (5, 17, 200):
        assert not y[i].any() and not yc[i].any()


# ---- streams, graphs, repeats ----------------------------------------------------------------------------------------

def test_same_bits_on_every_call_and_stream(tg):
    c = case_scan(11, 4, 200, 70, 16, 1, torch.bfloat16)
    first = run_scan(tg, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run_scan(tg, c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    for k in first[2]:
        assert torch.equal(first[2][k], second[2][k]), k


def test_captured_and_replayed(tg):
    """Forward, backward and both one-token forms in two graphs, replayed with new inputs, eager work in between."""
    c, cc = case_scan(12, 2, 150, 24, 16, 1, torch.float32), case_conv(12, 2, 150, 24, 4, torch.float32)
    leaves = [leaf(c[k]) for k in ORDER] + [leaf(cc[k]) for k in ("x", "weight", "bias")]
    dy, state, cstate = cuda(c["dy"]), cuda(c["initial"]), cuda(cc["initial"])

    def train():
        x = tg.short_conv(*leaves[8:])
        y = tg.selective_scan(leaves[0] + x, *leaves[1:8])
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    def token():
        with torch.no_grad():
            x = tg.short_conv_step(leaves[8][:, 0], cstate, *leaves[9:])
            return tg.selective_scan_step(x, leaves[1][:, 0], state, leaves[2], leaves[3][:, 0], leaves[4][:, 0], *leaves[5:6], leaves[6][:, 0],
                                          leaves[7])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
        token()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    gc.collect()        # another test's graphs must not be collected, and so destroyed, while these are captured
    gc.disable()
    try:
        with torch.cuda.graph(graphs[0]):
            outs = train()
        with torch.cuda.graph(graphs[1]):
            tok = token()
    finally:
        gc.enable()
    gen = torch.Generator().manual_seed(5)
    for _ in range(4):
        with torch.no_grad():
            for v in (leaves[0], leaves[1], leaves[8], leaves[3]):
                v.copy_(randn(gen, *v.shape))
        before = state.clone(), cstate.clone()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        got, after, y = [o.clone() for o in outs], (state.clone(), cstate.clone()), tok.clone()
        state.copy_(before[0])
        cstate.copy_(before[1])
        want, y_want = train(), token()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(y, y_want) and torch.equal(after[0], state) and torch.equal(after[1], cstate)


def test_only_what_is_asked_for(tg):
    """Frozen inputs get no gradient and change nothing for the others; an unused output counts as zero."""
    c = case_scan(13, 2, 40, 30, 16, 1, torch.float32)
    full = run_scan(tg, c)
    for names in (("u",), ("A",), ("Bm", "z"), ("initial",), ("delta_bias", "D")):
        t = {k: leaf(c[k]) if k in names else cuda(c[k]) for k in ORDER + ("initial",)}
        y, h = tg.selective_scan(*[t[k] for k in ORDER], initial_state=t["initial"], return_state=True)
        for k, g in zip(names, torch.autograd.grad([y, h], [t[k] for k in names], [cuda(c["dy"]), cuda(c["dfinal"])])):
            assert torch.equal(g, full[2][k]), k
    t = {k: leaf(c[k]) for k in ORDER + ("initial",)}
    y, h = tg.selective_scan(*[t[k] for k in ORDER], initial_state=t["initial"], return_state=True)
    got = torch.autograd.grad(h.sum(), [t["u"], t["initial"]])
    kw = dict(initial=c["initial"], dfinal=torch.ones_like(c["dfinal"]))
    want, size = (ref.scan(*[c[k] for k in ORDER], absolute=a, **kw)[2] for a in (False, True))
    ref.close(got[0], want["u"], size["u"], 40, what="u")
    ref.close(got[1], want["initial"], size["initial"], 40, what="initial")
    with pytest.raises(RuntimeError, match="second derivative"):
        u = leaf(c["u"])
        torch.autograd.grad(tg.selective_scan(u, *[cuda(c[k]) for k in ORDER[1:]]).sum(), u, create_graph=True)


def test_slots_of_64_bits(tg):
    """A slot that 32 bits do not hold is padding like every other one outside the pool."""
    pool = torch.randn(3, 3, 8, device=DEV)
    was, x, w = pool.clone(), torch.randn(3, 8, device=DEV), torch.randn(8, 4, device=DEV)
    y = tg.short_conv_step(x, pool, w, slots=torch.tensor([2 ** 32, 1, -2 ** 32], device=DEV))
    assert not y[0].any() and not y[2].any() and y[1].any()
    assert torch.equal(pool[0], was[0]) and torch.equal(pool[2], was[2]) and torch.equal(pool[1, -1], x[1])


def test_steps_refuse_gradients(tg):
    u = torch.zeros(2, 4, device=DEV, requires_grad=True)
    w, s = torch.zeros(4, 4, device=DEV), torch.zeros(2, 3, 4, device=DEV)
    with pytest.raises(RuntimeError, match="no backward"):
        tg.short_conv_step(u, s, w)
    with torch.no_grad():
        tg.short_conv_step(u, s, w)
