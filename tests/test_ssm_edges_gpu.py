"""The state-space operators at the edges of their arguments' ranges, on the GPU: states that grow, rates that are infinite,
results that are changed in place, views and large sizes.  Values against ssm_reference.py (float64), with its bounds."""
import pytest
import torch

import ssm_reference as ref
from test_ssm_gpu import DEV, ORDER, case_scan, check_scan, cuda, randn, run_scan, tg  # noqa: F401

pytestmark = pytest.mark.gpu


def growing_scan(tg, N):  # noqa: F811
    """300 steps of few channels: cut into chunks of 16 or 32 steps (checked).  A step of -0.5 multiplies a state by up to
    e^8, so a chunk of such steps by up to 2^369, far beyond float32."""
    c = case_scan(21, 1, 300, 24, N, 1, torch.float32, bias=False)
    c["A"] = -16 * (0.5 + 0.5 * torch.rand(24, N, generator=torch.Generator().manual_seed(1)))
    assert tg.lib().tgru_scan_workspace_bytes(1, 300, 24, N, 1, 0) > 0
    return c


@pytest.mark.parametrize("N", [16, 5])
def test_a_state_of_zero_stays_zero_where_states_grow(tg, N):  # noqa: F811
    """Nothing enters before the last 8 steps and no gradient behind the first 8: in between all is 0, whatever the chunks
    would make of a state.  8 steps are e^64 at most, and the exponents' errors of 12 half steps times 64 are within
    ref.bound's 8 T = 2400."""
    c = growing_scan(tg, N)
    c["delta"] = torch.full_like(c["delta"], -0.5)
    c["u"][:, :-8] = 0
    c["dy"][:, 8:] = 0
    c["initial"], c["dfinal"] = torch.zeros_like(c["initial"]), torch.zeros_like(c["dfinal"])
    check_scan(c, run_scan(tg, c, softplus=False), softplus=False)


@pytest.mark.parametrize("N", [16, 5])
def test_a_small_state_grows_by_more_than_float_holds(tg, N):  # noqa: F811
    """13 steps in one chunk multiply by up to e^104 = 2^150, what enters is about 1e-30: 1e15 comes out, in both directions.
    12 * 104 half steps from the exponents are within ref.bound."""
    c = growing_scan(tg, N)
    c["delta"] = torch.zeros_like(c["delta"])
    c["delta"][:, 97:110] = -0.5
    for k in ("initial", "dfinal", "u", "dy"):
        c[k] = c[k] * 1e-30
    check_scan(c, run_scan(tg, c, softplus=False), softplus=False)


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("N", [16, 5])
def test_a_token_with_infinite_rates(tg, N, softplus):  # noqa: F811
    """A = -inf forgets the state at every step that is longer than 0; one of length 0 (also softplus of -200) keeps it.  The
    same from a sequence of one step and from the one-token form."""
    c = case_scan(23, 4, 1, 8, N, 1, torch.float32, bias=False)
    c["A"] = torch.full_like(c["A"], float("-inf"))
    zero = -200.0 if softplus else 0.0
    c["delta"] = torch.tensor([0.5, zero, 1.0, zero])[:, None, None].expand(4, 1, 8).contiguous()
    s = {k: cuda(c[k]) for k in ORDER}
    y_seq, h_seq = tg.selective_scan(*[s[k] for k in ORDER], softplus=softplus, initial_state=cuda(c["initial"]), return_state=True)
    state = cuda(c["initial"]).clone()
    y = tg.selective_scan_step(s["u"][:, 0], s["delta"][:, 0], state, s["A"], s["Bm"][:, 0], s["Cm"][:, 0], s["D"], s["z"][:, 0],
                               softplus=softplus)
    c["A"] = torch.full_like(c["A"], -1e30)
    args = [c[k] for k in ORDER]
    want, size = (ref.scan(*args, softplus=softplus, initial=c["initial"], absolute=a) for a in (False, True))
    for got, k, what in ((y_seq, 0, "sequence"), (h_seq, 1, "its state"), (y[:, None], 0, "token"), (state, 1, "its state")):
        ref.close(got, want[k], size[k], 1, what=what)


def test_results_in_order_of_time_can_be_changed_in_place(tg):  # noqa: F811
    """(T, B, D) inputs give results in that order; they are tensors of their own, not views that autograd protects."""
    g = torch.Generator().manual_seed(1)
    x, w, s = randn(g, 6, 3, 16).to(DEV), randn(g, 16, 4).to(DEV), randn(g, 16).to(DEV)
    A, b = -torch.ones(16, 4, device=DEV), randn(g, 3, 6, 1, 4).to(DEV)
    calls = (lambda t: tg.short_conv(t, w), lambda t: tg.short_conv(t, w, return_state=True)[0],
             lambda t: tg.selective_scan(t, t, A, b, b), lambda t: tg.selective_scan(t, t, A, b, b, return_state=True)[0])
    for call in calls:
        leaf = x.clone().requires_grad_(True)
        want = torch.autograd.grad((call(leaf.transpose(0, 1)) * s).sum(), leaf)[0]
        y = call(leaf.transpose(0, 1))
        assert y.stride() == (16, 48, 1) and not y._is_view()
        y.mul_(s)
        assert torch.equal(torch.autograd.grad(y.sum(), leaf)[0], want)
        scale = s.clone().requires_grad_(True)        # a result without a graph, changed by something with one
        y = call(x.transpose(0, 1))
        before = y.clone()
        y.mul_(scale)
        assert torch.equal(torch.autograd.grad(y.sum(), scale)[0], before.sum((0, 1)))


def test_lengths_and_slots_out_of_a_table(tg):  # noqa: F811
    """Columns of an int32 table on the GPU, whose elements are not consecutive."""
    g = torch.Generator().manual_seed(2)
    x, w, pool = randn(g, 3, 6, 8).to(DEV), randn(g, 8, 4).to(DEV), randn(g, 8, 3, 8).to(DEV)
    table = torch.tensor([[6, 5], [2, 0], [3, 1]], dtype=torch.int32, device=DEV)
    assert torch.equal(tg.short_conv(x, w, lengths=table[:, 0]), tg.short_conv(x, w, lengths=[6, 2, 3]))
    first, second = pool.clone(), pool.clone()
    assert torch.equal(tg.short_conv_step(x[:, 0], first, w, slots=table[:, 1]), tg.short_conv_step(x[:, 0], second, w, slots=[5, 0, 1]))
    assert torch.equal(first, second)


def test_a_convolution_of_more_than_2_to_the_34_elements(tg):  # noqa: F811
    """520 sequences, all the same one (so inputs are small), results whole: 35 GB each.  Without the activation a term of
    dweight is an exact product; it goes through 64 steps of a run, at most 80 rows of partial sums in a thread and its
    tree, and 32 threads: less than 256 roundings."""
    B, T, D, K = 520, 4096, 8192, 4
    dev = torch.Generator(device=DEV).manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=dev, device=DEV)  # noqa: E731
    one, dy, w = rnd(1, T, D).bfloat16(), rnd(1, T, D).bfloat16(), rnd(D, K)
    assert B * T * D > 2 ** 34
    results = []
    for n in (1, B):
        x = one.expand(n, T, D).detach().requires_grad_(True)
        weight = w.clone().requires_grad_(True)
        y = tg.short_conv(x, weight, silu=False)
        results.append((y.detach(), *torch.autograd.grad(y, [x, weight], dy.expand(n, T, D))))
        del y
    (y1, dx1, _), (y, dx, dw) = results
    for i in (0, 255, 256, B - 1):
        assert torch.equal(y[i], y1[0]) and torch.equal(dx[i], dx1[0])
    ext = torch.cat([one.new_zeros(1, K - 1, D), one], 1)[0].double()
    for k in range(K):
        terms = dy[0].double() * ext[k:k + T]
        assert ((dw[:, k].double() - B * terms.sum(0)).abs() <= 256 * 2.0 ** -24 * B * terms.abs().sum(0)).all()
    del results, y, dx
    torch.cuda.empty_cache()


def test_accuracy_of_the_activation(tg):  # noqa: F811
    """v sigmoid(v) through a convolution of one tap of 1, relative to the value.  Half steps of float32: exp2 and the reciprocal
    2 each, the sum, the product and the result 1 each; below 0 also |v| for the rounded exponent v log2(e) and 0.22 |v| for the
    constant's own rounding (2^-26.2)."""
    v = torch.linspace(-80, 80, 1 << 20)
    y = tg.short_conv(v.view(-1, 1, 1).to(DEV), torch.ones(1, 1, device=DEV)).cpu().view(-1).double()
    want = v.double() * torch.sigmoid(v.double())
    assert ((y - want).abs() <= (7 - 1.22 * v.double().clamp(max=0)) * ref.EPS * want.abs()).all()


def test_gradients_of_as_many_sequences_as_are_counted(tg):  # noqa: F811
    """2^31 - 256 sequences of one step and one channel, all ones: rows of partial sums are numbered up to the end of 31 bits.  The
    sums go through two rounds of at most 2^19 / 32 / 16 rows in a partial sum (whole numbers below 2^24, exact), 16 partial sums
    and 32 threads, then 4096 rows: less than 384 roundings."""
    B = 2 ** 31 - 256
    one = torch.ones(1, 1, 1, device=DEV).expand(B, 1, 1)
    w, b = torch.full((1, 1), 2.0, device=DEV, requires_grad=True), torch.ones(1, device=DEV, requires_grad=True)
    y = tg.short_conv(one, w, b, silu=False)
    assert bool((y == 3).all())
    dw, db = torch.autograd.grad(y, (w, b), one)
    for g in (dw, db):
        assert abs(float(g) - B) <= 384 * ref.EPS * B
    del y
    torch.cuda.empty_cache()


def test_thousands_of_rows_with_slots_that_come_twice(tg):  # noqa: F811
    """Rows i and 2500 + j with the same slot are two steps of one sequence: the same bits as two calls without repeats."""
    g = torch.Generator().manual_seed(3)
    P, D, N = 2500, 12, 8
    first, second = torch.randperm(P, generator=g).to(DEV).int(), torch.randperm(P, generator=g).to(DEV).int()
    x, u, delta, B, C = (randn(g, 2 * P, *s).to(DEV) for s in ((D,), (D,), (D,), (1, N), (1, N)))
    w, A, cpool, pool = (randn(g, *s).to(DEV) for s in ((D, 4), (D, N), (P, 3, D), (P, D, N)))
    A = -A.abs()
    twice = [cpool.clone(), pool.clone()]
    slots = torch.cat([first, second])
    y = tg.short_conv_step(x, twice[0], w, slots=slots), tg.selective_scan_step(u, delta, twice[1], A, B, C, slots=slots)
    for part, s in ((slice(0, P), first), (slice(P, 2 * P), second)):
        assert torch.equal(tg.short_conv_step(x[part], cpool, w, slots=s), y[0][part])
        assert torch.equal(tg.selective_scan_step(u[part], delta[part], pool, A, B[part], C[part], slots=s), y[1][part])
    assert torch.equal(cpool, twice[0]) and torch.equal(pool, twice[1])


def test_a_token_of_as_many_channels_as_are_counted(tg):  # noqa: F811
    """2^31 - 1 channels of one state: the number of waves must not be rounded up beyond 31 bits."""
    D = 2 ** 31 - 1
    dev = torch.Generator(device=DEV).manual_seed(5)
    u = torch.empty(1, D, dtype=torch.bfloat16, device=DEV).normal_(generator=dev)
    A, state = torch.full((D, 1), -1.0, device=DEV), torch.ones(1, D, 1, device=DEV)
    b = torch.ones(1, 1, 1, dtype=torch.bfloat16, device=DEV)
    y = tg.selective_scan_step(u, u, state, A, b, b)
    for part in (slice(0, 1000), slice(D // 2, D // 2 + 1000), slice(D - 1000, D)):
        few = torch.ones(1, 1000, 1, device=DEV)
        assert torch.equal(tg.selective_scan_step(u[:, part], u[:, part], few, A[:1000], b, b), y[:, part])
        assert torch.equal(few, state[:, part])
    del u, A, state, y
    torch.cuda.empty_cache()


def test_sequences_refuse_dual_tensors(tg):  # noqa: F811
    import torch.autograd.forward_ad as fw
    x, w = torch.zeros(2, 3, 8, device=DEV), torch.zeros(8, 4, device=DEV)
    b = torch.zeros(2, 3, 1, 4, device=DEV)
    with fw.dual_level(), torch.no_grad():
        dual = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: tg.short_conv(dual, w), lambda: tg.selective_scan(dual, x, w, b, b)):
            with pytest.raises(RuntimeError, match="jvp is not implemented"):
                call()
