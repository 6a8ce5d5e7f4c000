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
