"""CPU tests of the state-space operators: the float64 reference against differences, the refusals of the public entry points
and of the C ABI, size queries, and the SSM stack's construction.  No kernel is launched."""
import ctypes

import pytest
import torch

import ssm_reference as ref


@pytest.fixture(scope="module")
def tg():
    import timegan_amd
    return timegan_amd


def test_reference_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    B, T, D, N, G, K = 2, 5, 4, 3, 2, 3
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    c = dict(u=rnd(B, T, D), delta=rnd(B, T, D), A=-torch.exp(rnd(D, N)), Bm=rnd(B, T, G, N), Cm=rnd(B, T, G, N), D=rnd(D), z=rnd(B, T, D),
             delta_bias=rnd(D), initial=rnd(B, D, N))
    lengths, dy, dh = [5, 3], rnd(B, T, D), rnd(B, D, N)

    def value(c):
        y, h, _ = ref.scan(*[c[k] for k in ("u", "delta", "A", "Bm", "Cm", "D", "z", "delta_bias")], initial=c["initial"], lengths=lengths)
        return float((y * dy).sum() + (h * dh).sum())

    grads = ref.scan(*[c[k] for k in ("u", "delta", "A", "Bm", "Cm", "D", "z", "delta_bias")], initial=c["initial"], lengths=lengths,
                     dy=dy, dfinal=dh)[2]
    x = dict(x=rnd(B, T, D), weight=rnd(D, K), bias=rnd(D), initial=rnd(B, K - 1, D))
    dx = rnd(B, K - 1, D)

    def cvalue(x):
        y, s, _ = ref.conv(x["x"], x["weight"], x["bias"], initial=x["initial"], lengths=lengths)
        return float((y * dy).sum() + (s * dx).sum())

    cgrads = ref.conv(x["x"], x["weight"], x["bias"], initial=x["initial"], lengths=lengths, dy=dy, dfinal=dx)[2]
    for f, inputs, got in ((value, c, grads), (cvalue, x, cgrads)):
        for k, v in inputs.items():
            d = torch.randn(v.shape, generator=g, dtype=torch.float64)
            e = 1e-5      # central difference: the error is of order e^2 (1e-10) and 2^-52 |f| / e (1e-10)
            num = (f({**inputs, k: v + e * d}) - f({**inputs, k: v - e * d})) / (2 * e)
            assert abs(num - float((got[{"Bm": "B", "Cm": "C"}.get(k, k)] * d).sum())) < 1e-7 * max(1.0, abs(num)), k


def scan_inputs(B=2, T=3, D=4, N=16, G=1, dtype=torch.float32):
    z = lambda *s: torch.zeros(*s, dtype=dtype)  # noqa: E731
    return dict(u=z(B, T, D), delta=z(B, T, D), A=torch.zeros(D, N), B=z(B, T, G, N), C=z(B, T, G, N))


@pytest.mark.parametrize("change,text", [
    (dict(u=torch.zeros(2, 4)), "must be \\(B, T, D\\)"),
    (dict(u=torch.zeros(2, 3, 4, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(u=torch.zeros(2, 0, 4)), "number of steps"),
    (dict(u=torch.zeros(0, 3, 4)), "batch"),
    (dict(delta=torch.zeros(2, 3, 5)), "delta must have shape"),
    (dict(delta=torch.zeros(2, 3, 4, dtype=torch.bfloat16)), "element type"),
    (dict(A=torch.zeros(4)), "A must be"),
    (dict(A=torch.zeros(5, 16)), "A must be"),
    (dict(A=torch.zeros(4, 65)), "1 to 64"),
    (dict(A=torch.zeros(4, 0)), "1 to 64"),
    (dict(A=torch.zeros(4, 16, dtype=torch.int32)), "floating-point"),
    (dict(B=torch.zeros(2, 3, 16)), "dimension of groups"),
    (dict(B=torch.zeros(2, 3, 3, 16)), "divide"),
    (dict(B=torch.zeros(2, 3, 0, 16)), "divide"),
    (dict(B=torch.zeros(2, 3, 1, 15)), "B must have shape"),
    (dict(C=torch.zeros(2, 3, 2, 16)), "C must have shape"),
    (dict(D=torch.zeros(5)), "D must have shape"),
    (dict(z=torch.zeros(2, 3, 4, dtype=torch.float16)), "element type"),
    (dict(delta_bias=torch.zeros(4, 1)), "delta_bias must have shape"),
    (dict(initial_state=torch.zeros(2, 4, 15)), "initial_state must have shape"),
    (dict(lengths=[3]), "batch_size"),
    (dict(lengths=[3, 4]), "between 0 and"),
    (dict(lengths=[3, -1]), "between 0 and"),
    (dict(), "no CPU fallback"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_scan_refusals(tg, change, text):
    kw = {**scan_inputs(), **change}
    with pytest.raises(RuntimeError, match=text):
        tg.selective_scan(**kw)


@pytest.mark.parametrize("change,text", [
    (dict(x=torch.zeros(3, 4)), "must be \\(B, T, D\\)"),
    (dict(x=torch.zeros(2, 3, 4, dtype=torch.int32)), "float32, bfloat16 or float16"),
    (dict(x=torch.zeros(2, 0, 4)), "number of steps"),
    (dict(weight=torch.zeros(5, 4)), "weight must be"),
    (dict(weight=torch.zeros(4, 9)), "1 to 8"),
    (dict(weight=torch.zeros(4, 0)), "1 to 8"),
    (dict(bias=torch.zeros(3)), "bias must have shape"),
    (dict(initial_state=torch.zeros(2, 4, 4)), "initial_state must have shape"),
    (dict(initial_state=torch.zeros(2, 3, 4, dtype=torch.float16)), "element type"),
    (dict(lengths=[4, 1]), "between 0 and"),
    (dict(), "no CPU fallback"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_conv_refusals(tg, change, text):
    kw = {**dict(x=torch.zeros(2, 3, 4), weight=torch.zeros(4, 4)), **change}
    with pytest.raises(RuntimeError, match=text):
        tg.short_conv(**kw)


def test_step_refusals(tg):
    pool = torch.zeros(2, 3, 4)
    kw = dict(x=torch.zeros(2, 4), state=pool, weight=torch.zeros(4, 4))
    both = torch.zeros(30)
    for change, text in [(dict(x=torch.zeros(2, 3, 4)), "must be \\(B, D\\)"), (dict(x=torch.zeros(3, 4)), "holds 2 sequences"),
                         (dict(state=torch.zeros(2, 4, 4)), "state must have shape"), (dict(state=torch.zeros(2, 4, 3).transpose(1, 2)), "dense"),
                         (dict(state=pool.half()), "element type"), (dict(state_out=torch.zeros(3, 3, 4)), "state_out must have shape"),
                         (dict(state=both[:24].view(2, 3, 4), state_out=both[6:].view(2, 3, 4)), "overlap"),
                         (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots must have shape"),
                         (dict(weight=torch.zeros(4, 4, requires_grad=True)), "no backward pass"), (dict(), "no CPU fallback")]:
        with pytest.raises(RuntimeError, match=text):
            tg.short_conv_step(**{**kw, **change})
    s = {k: v[:, 0] if v.dim() > 2 else v for k, v in scan_inputs().items()}
    kw = dict(s, state=torch.zeros(2, 4, 16))
    for change, text in [(dict(u=torch.zeros(2, 3, 4)), "must be \\(B, D\\)"), (dict(state=torch.zeros(2, 4, 15)), "state must have shape"),
                         (dict(state=torch.zeros(2, 4, 16, dtype=torch.bfloat16)), "float32"), (dict(state=torch.zeros(1, 4, 16)), "holds 1"),
                         (dict(B=torch.zeros(2, 16)), "dimension of groups"), (dict(), "no CPU fallback")]:
        with pytest.raises(RuntimeError, match=text):
            tg.selective_scan_step(**{**kw, **change})


def test_step_inputs_that_lie_in_the_state(tg):
    """What a call reads beside the state must not be what it writes."""
    pool = torch.zeros(2, 3, 4)
    with pytest.raises(RuntimeError, match="input overlaps the state"):
        tg.short_conv_step(pool[:, 0], pool, torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tg.short_conv_step(pool[:, 0], pool, torch.zeros(4, 4), state_out=torch.zeros(2, 3, 4))
    s = {k: v[:, 0] if v.dim() > 2 else v for k, v in scan_inputs().items()}
    state = torch.zeros(2, 4, 16)
    for k, v in (("u", state[..., 0].as_strided((2, 4), (64, 1))), ("delta", state.view(2, 64)[:, 8:12]), ("z", state.view(2, 64)[:, 60:]),
                 ("B", state[:, :1]), ("C", state[:, 3:])):
        with pytest.raises(RuntimeError, match="overlaps the state"):
            tg.selective_scan_step(**{**s, "state": state, k: v})
    whole = torch.zeros(2 * 64 + 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):      # next to it is not in it
        tg.selective_scan_step(**{**s, "state": whole[:128].view(2, 4, 16), "u": whole[128:].view(2, 4)})


def test_slots_and_lengths_of_other_integer_types(tg):
    from timegan_amd import ssm
    cpu = torch.device("cpu")
    got = ssm._slots(torch.tensor([0, 5, -1, 2 ** 32, 2 ** 32 + 1, -2 ** 40, 2 ** 31 - 1]), cpu)
    assert got.dtype == torch.int32 and got.tolist() == [0, 5, -1, 2 ** 31 - 1, 2 ** 31 - 1, -1, 2 ** 31 - 1]
    assert ssm._slots([3, -1], cpu).tolist() == [3, -1]
    assert ssm._slots(torch.tensor([200, 7], dtype=torch.uint8), cpu).tolist() == [200, 7]
    for bad in ([0.5, 1.0], torch.tensor([True, False])):
        with pytest.raises(RuntimeError, match="whole numbers"):
            ssm._slots(bad, cpu)


def test_c_abi_refuses_before_it_launches(tg):
    from timegan_amd._lib import ConvArgs, ConvStepArgs, ScanArgs, ScanStepArgs
    lb = tg.lib()
    E_DIMS, E_NULL, E_ALIGN, E_DTYPE = -1, -2, -4, -8
    for fn in (lb.tgru_conv_forward, lb.tgru_conv_backward, lb.tgru_conv_step, lb.tgru_scan_forward, lb.tgru_scan_backward, lb.tgru_scan_step):
        assert fn(None, None) == E_NULL
    conv = lambda **kw: ctypes.byref(ConvArgs(**{**dict(B=2, T=3, D=4, K=4), **kw}))  # noqa: E731
    for bad in (dict(B=0), dict(T=-1), dict(D=0), dict(K=9), dict(K=0), dict(B=1 << 20, T=1 << 20, D=1 << 10)):
        assert lb.tgru_conv_forward(conv(**bad), None) == E_DIMS and lb.tgru_conv_backward(conv(**bad), None) == E_DIMS
    assert lb.tgru_conv_forward(conv(dtype=3), None) == E_DTYPE
    assert lb.tgru_conv_forward(conv(), None) == E_NULL and lb.tgru_conv_backward(conv(), None) == E_NULL
    assert lb.tgru_conv_backward(conv(x=16, weight=16, dweight=16), None) == E_NULL          # no workspace
    scan = lambda **kw: ctypes.byref(ScanArgs(**{**dict(B=2, T=3, D=4, N=16, G=1), **kw}))  # noqa: E731
    for bad in (dict(N=65), dict(N=0), dict(G=3), dict(G=0), dict(T=0), dict(B=1 << 30, T=1 << 20)):
        assert lb.tgru_scan_forward(scan(**bad), None) == E_DIMS and lb.tgru_scan_backward(scan(**bad), None) == E_DIMS
    full = dict(u=16, delta=16, b=16, c=16, a=16, y=16)
    assert lb.tgru_scan_forward(scan(dtype=-1), None) == E_DTYPE
    assert lb.tgru_scan_forward(scan(), None) == E_NULL
    assert lb.tgru_scan_backward(scan(**full), None) == E_NULL                                # no reserve
    assert lb.tgru_scan_backward(scan(**full, reserve=16, workspace=16, dz=16), None) == E_NULL   # dz without z
    assert lb.tgru_scan_forward(scan(**full, reserve=8), None) == E_ALIGN
    step = lambda **kw: ctypes.byref(ConvStepArgs(**{**dict(B=2, P=2, D=4, K=4), **kw}))  # noqa: E731
    assert lb.tgru_conv_step(step(P=1), None) == E_DIMS and lb.tgru_conv_step(step(), None) == E_NULL
    step = lambda **kw: ctypes.byref(ScanStepArgs(**{**dict(B=2, P=2, D=4, N=16, G=1), **kw}))  # noqa: E731
    assert lb.tgru_scan_step(step(P=1), None) == E_DIMS and lb.tgru_scan_step(step(), None) == E_NULL
    assert lb.tgru_error_string(E_DTYPE) not in (b"ok", b"unknown error")


def test_size_queries(tg):
    lb = tg.lib()
    assert lb.tgru_scan_reserve_bytes(0, 1, 1, 1, 1) == 0 and lb.tgru_scan_workspace_bytes(1, 1, 1, 65, 1, 1) == 0
    assert lb.tgru_conv_backward_workspace_bytes(1, 1, 1, 9) == 0
    # 16 fp32 states in front of every 16 steps: one fp32 value per step and channel
    assert lb.tgru_scan_reserve_bytes(2, 64, 48, 16, 1) == 2 * 64 * 48 * 4
    assert lb.tgru_scan_workspace_bytes(64, 256, 1024, 16, 1, 0) == 0         # enough channels: time is not cut
    assert lb.tgru_scan_workspace_bytes(1, 4096, 64, 16, 1, 0) > 0
    assert lb.tgru_scan_workspace_bytes(1, 4096, 64, 16, 1, 1) > lb.tgru_scan_workspace_bytes(1, 4096, 64, 16, 1, 0)
    assert lb.tgru_conv_backward_workspace_bytes(2, 24, 48, 4) >= 2 * 5 * 48 * 4


def test_sizes_whose_state_needs_more_than_31_bits_are_refused(tg):
    assert tg.lib().tgru_scan_workspace_bytes(1, 16, 1 << 25, 64, 1, 1) == 0
    assert tg.lib().tgru_scan_workspace_bytes(1, 16, 1 << 24, 64, 1, 1) > 0


def test_launches_of_more_than_2_to_the_32_threads_are_refused(tg):
    from timegan_amd._lib import ConvArgs, ConvStepArgs, ScanArgs, ScanStepArgs
    lb, E_DIMS, E_NULL = tg.lib(), -1, -2
    scan = lambda B, D: lb.tgru_scan_forward(ctypes.byref(ScanArgs(B=B, T=1, D=D, N=16, G=1)), None)  # noqa: E731
    assert scan(1 << 20, 1024) == E_DIMS and scan(1 << 19, 1024) == E_NULL           # 16 workgroups of 256 a sequence
    step = lambda B, D, N: lb.tgru_scan_step(ctypes.byref(ScanStepArgs(B=B, P=B, D=D, N=N, G=1)), None)  # noqa: E731
    assert step(1 << 20, 1024, 16) == E_DIMS and step(1 << 19, 1024, 16) == E_NULL   # 64 waves a row
    assert step(1 << 20, 1024, 4) == E_NULL and step(1 << 22, 1024, 4) == E_DIMS
    conv = lambda B, D: lb.tgru_conv_step(ctypes.byref(ConvStepArgs(B=B, P=B, D=D, K=4)), None)  # noqa: E731
    assert conv(1 << 22, 1024) == E_DIMS and conv(1 << 21, 1024) == E_NULL
    back = lambda **kw: lb.tgru_conv_backward(ctypes.byref(ConvArgs(B=1, T=1, D=1 << 25, K=4, **kw)), None)  # noqa: E731
    assert back(dweight=16, x=16, weight=16, workspace=16) == E_DIMS and back() == E_NULL


def test_argument_structs_match_the_header(tg, tmp_path):
    """The ctypes mirrors have the layout that a C compiler gives the header's structs."""
    import os
    import subprocess
    from timegan_amd import _lib
    names = {"ConvArgs": "tgru_conv_args", "ConvStepArgs": "tgru_conv_step_args", "ScanArgs": "tgru_scan_args", "ScanStepArgs": "tgru_scan_step_args"}
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lines = ['#include "tgru.h"', "#include <stdio.h>", "int main(void) {"]
    for py, c in names.items():
        for f in getattr(_lib, py)._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {f[0]}));')
        lines.append(f'printf("%zu\\n", sizeof({c}));')
    (tmp_path / "a.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "a.c"), "-o", str(tmp_path / "a")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "a")]).split()]
    want = []
    for py in names:
        cls = getattr(_lib, py)
        want += [getattr(cls, f[0]).offset for f in cls._fields_] + [ctypes.sizeof(cls)]
    assert got == want


def test_ssm_stack_construction(tg):
    m = tg.SSM(6, 24, 2, batch_first=True)
    assert {n.split(".", 2)[2] for n, _ in m.named_parameters()} == {
        "conv_weight", "conv_bias", "dt_bias", "A_log", "D", "in_proj.weight", "x_proj.weight", "dt_proj.weight", "out_proj.weight"}
    s = m.init_state(5)
    assert s.conv[0].shape == (5, 3, 48) and s.scan[1].shape == (5, 48, 16) and s.scan[0].dtype == torch.float32
    m.load_state_dict(tg.SSM(6, 24, 2).state_dict())
    dt = torch.nn.functional.softplus(m.layers[0].dt_bias.detach())
    assert float(dt.min()) > 0.9e-3 and float(dt.max()) < 0.11
    for kw, err in ((dict(bidirectional=True), NotImplementedError), (dict(state_size=65), ValueError), (dict(conv_width=1), ValueError),
                    (dict(dtype=torch.float64), ValueError), (dict(dropout=0.1, num_layers=2), NotImplementedError)):
        with pytest.raises(err):
            tg.SSM(6, 24, **kw)
    with pytest.raises(tg.TgruError, match="no CPU fallback"):
        m(torch.zeros(2, 3, 6))
    with pytest.raises(RuntimeError, match="input.size"):
        m(torch.zeros(2, 3, 5))
