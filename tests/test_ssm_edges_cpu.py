"""What the state-space operators refuse and accept at the edges of their arguments' ranges, without launching a kernel."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from test_ssm_cpu import scan_inputs, tg  # noqa: F401


@pytest.mark.parametrize("grad", [True, False])
def test_steps_refuse_dual_tensors(tg, grad):  # noqa: F811
    """A tangent would be lost without a word: every floating argument of the one-token forms is looked at."""
    conv = dict(x=torch.zeros(2, 4), state=torch.zeros(2, 3, 4), weight=torch.zeros(4, 4), bias=torch.zeros(4), state_out=torch.zeros(2, 3, 4))
    scan = {k: v[:, 0] if v.dim() > 2 else v for k, v in scan_inputs().items()}
    scan |= dict(state=torch.zeros(2, 4, 16), D=torch.zeros(4), z=torch.zeros(2, 4), delta_bias=torch.zeros(4), state_out=torch.zeros(2, 4, 16))
    with fw.dual_level(), torch.set_grad_enabled(grad):
        for fn, args in ((tg.short_conv_step, conv), (tg.selective_scan_step, scan)):
            for k in args:
                dual = fw.make_dual(args[k], torch.ones_like(args[k]))
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    fn(**{**args, k: dual})
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                fn(**args)


def test_slots_out_of_a_table(tg):  # noqa: F811
    """A column of an int32 table is taken like any other whole numbers."""
    table = torch.tensor([[6, 0], [2, 1], [3, 2]], dtype=torch.int32)
    scan = {k: v[:, 0] if v.dim() > 2 else v for k, v in scan_inputs(B=3).items()}
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tg.short_conv_step(torch.zeros(3, 4), torch.zeros(8, 3, 4), torch.zeros(4, 4), slots=table[:, 0])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tg.selective_scan_step(**scan, state=torch.zeros(8, 4, 16), slots=table[:, 0])


def test_convolutions_that_one_launch_holds_are_taken(tg):  # noqa: F811
    """The launch has a thread for 64 steps of 16 bytes of channels, so 2^35 elements are far from 2^32 threads."""
    import ctypes
    from timegan_amd._lib import ConvArgs
    lb, E_DIMS, E_NULL = tg.lib(), -1, -2
    for dims, want in (((32, 131072, 8192), E_NULL), ((520, 4096, 8192), E_NULL), ((1 << 20, 4096, 64), E_NULL), ((1 << 27, 1, 64), E_NULL),
                       ((1, 8, (1 << 31) - 256), E_NULL), ((1, 8, (1 << 31) - 255), E_DIMS), ((1, 1, (1 << 31) - 1), E_DIMS),
                       (((1 << 31) - 256, 1, 1), E_NULL), (((1 << 31) - 255, 1, 1), E_DIMS), (((1 << 31) - 1, 1, 1), E_DIMS),
                       ((1 << 30, 128, 1), E_DIMS), ((1 << 29, 64, 64), E_DIMS), ((1 << 28, 64, 256), E_DIMS)):
        for dtype in (0, 1, 2):
            args = ctypes.byref(ConvArgs(**dict(zip("BTD", dims)), K=4, dtype=dtype))
            assert lb.tgru_conv_forward(args, None) == want and lb.tgru_conv_backward(args, None) == want, (dims, dtype)
        assert (lb.tgru_conv_backward_workspace_bytes(*dims, 4) > 0) == (want == E_NULL)
    for dtype, want in ((0, E_DIMS), (1, E_NULL), (2, E_NULL)):       # 2^32 and 2^31 packs of one step
        assert lb.tgru_conv_forward(ctypes.byref(ConvArgs(B=1 << 26, T=1, D=256, K=4, dtype=dtype)), None) == want


def test_slots_that_would_be_searched_for_seconds_are_refused(tg):  # noqa: F811
    """Rows squared times waves a row, below 2^44; without slots nothing is searched."""
    import ctypes
    from timegan_amd._lib import ConvStepArgs, ScanStepArgs
    lb, E_DIMS, E_NULL = tg.lib(), -1, -2
    conv = lambda B, D, slots=16, dtype=0: lb.tgru_conv_step(ctypes.byref(ConvStepArgs(B=B, P=B, D=D, K=4, slots=slots, dtype=dtype)), None)  # noqa: E731
    assert conv(1 << 21, 256) == E_NULL and conv(1 << 22, 256) == E_DIMS and conv(1 << 22, 256, None) == E_NULL
    assert conv(1 << 21, 257) == E_DIMS and conv(1 << 20, 257) == E_NULL                # five waves a row
    assert conv(1 << 21, 512, dtype=1) == E_NULL and conv(1 << 21, 1024) == E_DIMS
    scan = lambda B, D, slots=16: lb.tgru_scan_step(ctypes.byref(ScanStepArgs(B=B, P=B, D=D, N=16, G=1, slots=slots)), None)  # noqa: E731
    assert scan(1 << 21, 16) == E_NULL and scan(1 << 22, 16) == E_DIMS and scan(1 << 22, 16, None) == E_NULL
    assert scan(1 << 19, 1024) == E_DIMS and scan((1 << 19) - 1, 1024) == E_NULL
