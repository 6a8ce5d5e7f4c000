"""State-space sequence operators: the short causal convolution and the selective scan, over whole sequences (with
gradients) and for one more token on saved states, and `SSM`, the layer stack around them with nn.GRU's constructor and
forward contract, so that it takes the GRU's place (`rnn_cls=tg.SSM`) in the networks of modules.py and in the scorer.

The reference has no counterpart: its recurrent layer is nn.GRU (outdated_files/TimeGANv1.py:35-38), whose steps follow one
another.  Here a step of a sequence is linear in the state, so time can be cut into chunks that run side by side.

All operators run in libtgru.so (tgru_conv_*, tgru_scan_* of include/tgru.h) through the C++ binding; there is no CPU
fallback.  Sequence tensors are float32, bfloat16 or float16 -- one type per call -- and may be any view whose last
dimension is consecutive (a (T, B, D) tensor is passed as x.transpose(0, 1), half of a projection as a slice); parameters of
any floating type are computed with in float32, and so is everything between input and output.
"""
import math
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn
from torch.nn.utils.rnn import PackedSequence, pack_padded_sequence, pad_packed_sequence

from . import functional as F_
from ._lib import TgruError


def _op():
    mod = F_.cpp_op()
    if mod is None:
        raise TgruError("time-gan_amd/_tgru_torch.so is not built or switched off (python __graft_entry__.py build): the "
                        "state-space operators run through it only")
    return mod


def _lengths(lengths, B: int, T: int, device) -> Optional[torch.Tensor]:
    """int32 lengths on `device`, or None where all are T.  A tensor that is on the GPU already is taken as it is, without
    looking at it (no synchronisation; the kernels take a length as clamped to [0, T]); anything else is checked here."""
    if lengths is None:
        return None
    if isinstance(lengths, torch.Tensor) and lengths.is_cuda:
        if lengths.is_floating_point() or lengths.dtype == torch.bool:
            raise RuntimeError(f"lengths must be whole numbers, got {lengths.dtype}")
        return lengths.contiguous() if lengths.dtype == torch.int32 else lengths.long().clamp(0, T).int()
    lens = [int(v) for v in (lengths.tolist() if isinstance(lengths, torch.Tensor) else lengths)]
    if len(lens) != B:
        raise RuntimeError(f"Expected `len(lengths)` to be equal to batch_size, but got {len(lens)} (batch_size={B})")
    if any(n < 0 or n > T for n in lens):
        raise RuntimeError(f"lengths must be between 0 and the sequence dimension ({T}), got {lens}")
    if all(n == T for n in lens):
        return None
    return torch.tensor(lens, dtype=torch.int32, device=device)


def _slots(slots, device) -> Optional[torch.Tensor]:
    if slots is None:
        return None
    if isinstance(slots, torch.Tensor) and slots.dtype == torch.int32 and slots.device == device:
        return slots.contiguous()
    slots = torch.as_tensor(slots, device=device)
    if slots.is_floating_point() or slots.dtype == torch.bool:
        raise RuntimeError(f"slots must be whole numbers, got {slots.dtype}")
    return slots.long().clamp(-1, 2 ** 31 - 1).int()       # what 32 bits do not hold is outside every pool, and stays so


def short_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, silu: bool = True,
               initial_state: Optional[torch.Tensor] = None, lengths=None, return_state: bool = False):
    """Causal depthwise convolution over time: y[:, t] = act(bias + sum_k weight[:, k] x[:, t - K + 1 + k]).

    x (B, T, D); weight (D, K), 1 <= K <= 8; bias (D); act is v * sigmoid(v), or nothing with silu=False.  What lies in
    front of x is initial_state (B, K - 1, D) in x's type, or zeros.  lengths: steps of each sequence, in [0, T], any order
    (list, CPU tensor, or an integer GPU tensor, which is not looked at on the host); outputs behind a sequence's end are
    0, inputs there are ignored whatever they hold, and no gradient goes there.
    Returns y (B, T, D), or (y, state) with return_state: the last K - 1 inputs of each sequence, the next call's
    initial_state and what short_conv_step goes on from.  Differentiable once (in backward mode) in every floating argument.
    """
    if x.dim() == 3:
        lengths = _lengths(lengths, x.shape[0], x.shape[1], x.device)
    out = _op().short_conv(x, weight, bias, silu, initial_state, lengths, return_state)
    return (out[0], out[1]) if return_state else out[0]


def short_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                    silu: bool = True, slots=None, state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One more step of short_conv for each of B sequences: x (B, D) -> y (B, D).

    state (P, K - 1, D) in x's type, dense, is a pool of states; row i of x belongs to state[slots[i]] (state[i] without
    slots).  The states are updated in place, or written to state_out (same shape) with `state` left as it was.  A row
    whose slot is outside [0, P) is padding: y is 0, no state is touched.  Rows with the same slot are steps of one sequence
    and are taken in order; looking for them costs time that grows with the square of the rows (little up to some thousand
    rows, 15 ms for a scan of 65536 rows; what would take seconds is refused).  slots: dense int32 GPU tensor (no copy), or
    whole numbers in anything torch.as_tensor takes.  x must not overlap the states that are written (refused).  No
    derivatives.
    """
    return _op().short_conv_step(x, state, weight, bias, silu, _slots(slots, x.device), state_out)


def selective_scan(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   delta_bias: Optional[torch.Tensor] = None, *, softplus: bool = True,
                   initial_state: Optional[torch.Tensor] = None, lengths=None, return_state: bool = False):
    """The selective state-space scan.  For every sequence and channel, with N states h,

        dt_t = softplus(delta_t + delta_bias)          (delta_t + delta_bias with softplus=False)
        h_t  = exp(dt_t A) h_{t-1} + dt_t u_t B_t
        y_t  = (C_t . h_t + D u_t) * z_t * sigmoid(z_t)

    u, delta, z (batch, T, channels); A (channels, N), 1 <= N <= 64; B, C (batch, T, G, N): G groups of channels / G
    channels share them (one group: unsqueeze(2)); D, delta_bias (channels).  D, z, delta_bias may be None.
    initial_state (batch, channels, N) float32 or zeros.  lengths and padding as in short_conv; a sequence of length 0
    keeps its initial state.
    States may grow (negative steps, positive rates) as far as float32 holds them and exp(dt A) of one step.
    Returns y, or (y, state) with return_state: the float32 state behind each sequence's last step.  Differentiable once
    (in backward mode) in every floating argument.
    """
    if u.dim() == 3:
        lengths = _lengths(lengths, u.shape[0], u.shape[1], u.device)
    out = _op().selective_scan(u, delta, A, B, C, D, z, delta_bias, softplus, initial_state, lengths, return_state)
    return (out[0], out[1]) if return_state else out[0]


def selective_scan_step(u: torch.Tensor, delta: torch.Tensor, state: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                        C: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        delta_bias: Optional[torch.Tensor] = None, *, softplus: bool = True, slots=None,
                        state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One more step of selective_scan for each of B sequences: u, delta, z (B, channels), B, C (B, G, N) -> y (B, channels).
    state (P, channels, N) float32, dense: a pool of states; slots, state_out, padding and repeated slots as in
    short_conv_step.  No derivatives."""
    return _op().selective_scan_step(u, delta, state, A, B, C, D, z, delta_bias, softplus, _slots(slots, u.device), state_out)


class SSMState(NamedTuple):
    """State of an `SSM` stack between calls, one tensor per layer: the convolutions' last inputs (sequences, K - 1, E)
    and the scans' states (sequences, E, N) in float32."""
    conv: Tuple[torch.Tensor, ...]
    scan: Tuple[torch.Tensor, ...]


class SSMLayer(nn.Module):
    """One selective state-space layer: in_proj to (x, z), short convolution of x, projections of it to the step sizes and
    the input and output maps, selective scan gated by z, out_proj."""

    def __init__(self, input_size: int, hidden_size: int, state_size: int, conv_width: int, expand: int, dt_rank: int,
                 bias: bool, device=None, dtype=None):
        super().__init__()
        kw = dict(device=device, dtype=dtype)
        self.inner, self.state_size, self.conv_width, self.dt_rank = expand * hidden_size, state_size, conv_width, dt_rank
        E = self.inner
        self.in_proj = nn.Linear(input_size, 2 * E, bias=False, **kw)
        self.conv_weight = nn.Parameter(torch.empty(E, conv_width, **kw))
        self.conv_bias = nn.Parameter(torch.empty(E, **kw)) if bias else None
        self.x_proj = nn.Linear(E, dt_rank + 2 * state_size, bias=False, **kw)
        self.dt_proj = nn.Linear(dt_rank, E, bias=False, **kw)
        self.dt_bias = nn.Parameter(torch.empty(E, **kw))
        self.A_log = nn.Parameter(torch.empty(E, state_size, **kw))
        self.D = nn.Parameter(torch.empty(E, **kw))
        self.out_proj = nn.Linear(E, hidden_size, bias=False, **kw)
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        for lin in (self.in_proj, self.x_proj, self.out_proj):
            lin.reset_parameters()
        k = 1.0 / math.sqrt(self.conv_width)
        self.conv_weight.uniform_(-k, k)
        if self.conv_bias is not None:
            self.conv_bias.uniform_(-k, k)
        r = self.dt_rank ** -0.5
        self.dt_proj.weight.uniform_(-r, r)
        # step sizes between 0.001 and 0.1 (their logarithm uniform), decay rates 1 .. N
        dt = torch.exp(torch.rand_like(self.dt_bias, dtype=torch.float32) * math.log(100.0) + math.log(1e-3))
        self.dt_bias.copy_(torch.log(torch.expm1(dt)))
        self.A_log.copy_(torch.log(torch.arange(1, self.state_size + 1, dtype=torch.float32, device=self.A_log.device)).expand_as(self.A_log))
        self.D.fill_(1.0)

    def _maps(self, x: torch.Tensor):
        dt, B, C = self.x_proj(x).split([self.dt_rank, self.state_size, self.state_size], dim=-1)
        return self.dt_proj(dt), -torch.exp(self.A_log.float()), B.unsqueeze(-2), C.unsqueeze(-2)

    def forward(self, x: torch.Tensor, lengths=None, conv_state=None, scan_state=None):
        x, z = self.in_proj(x).chunk(2, dim=-1)
        x, conv_state = short_conv(x, self.conv_weight, self.conv_bias, initial_state=conv_state, lengths=lengths, return_state=True)
        delta, A, B, C = self._maps(x)
        y, scan_state = selective_scan(x, delta, A, B, C, self.D, z, self.dt_bias, initial_state=scan_state, lengths=lengths,
                                       return_state=True)
        return self.out_proj(y), conv_state, scan_state

    def step(self, x: torch.Tensor, conv_state: torch.Tensor, scan_state: torch.Tensor, slots=None) -> torch.Tensor:
        x, z = self.in_proj(x).chunk(2, dim=-1)
        x = short_conv_step(x, conv_state, self.conv_weight, self.conv_bias, slots=slots)
        delta, A, B, C = self._maps(x)
        return self.out_proj(selective_scan_step(x, delta, scan_state, A, B, C, self.D, z, self.dt_bias, slots=slots))


class SSM(nn.Module):
    """A stack of selective state-space layers behind nn.GRU's constructor and forward signature.

    Beyond the GRU's arguments: state_size (states per channel, up to 64), conv_width (taps, up to 8), expand (inner width
    / hidden_size), dt_rank (default ceil(hidden_size / 16)).  Parameters and inputs are float32, bfloat16 or float16, one
    type for all (parameters may stay float32 where only float32 inputs come).
    """

    def __init__(self, input_size: int, hidden_size: int, num_layers: int = 1, bias: bool = True, batch_first: bool = False,
                 dropout: float = 0.0, bidirectional: bool = False, device=None, dtype=None, *, state_size: int = 16,
                 conv_width: int = 4, expand: int = 2, dt_rank: Optional[int] = None):
        super().__init__()
        if bidirectional:
            raise NotImplementedError("bidirectional stacks are not built")
        if dropout and num_layers > 1:
            raise NotImplementedError("inter-layer dropout is not built")
        if not 1 <= state_size <= 64:
            raise ValueError(f"state_size must be between 1 and 64, got {state_size}")
        if not 2 <= conv_width <= 8:
            raise ValueError(f"conv_width must be between 2 and 8, got {conv_width}")
        if dtype not in (None, torch.float32, torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        self.input_size, self.hidden_size, self.num_layers, self.batch_first = input_size, hidden_size, num_layers, batch_first
        self.layers = nn.ModuleList(
            SSMLayer(input_size if k == 0 else hidden_size, hidden_size, state_size, conv_width, expand,
                     dt_rank or math.ceil(hidden_size / 16), bias, device, dtype) for k in range(num_layers))

    def extra_repr(self) -> str:
        return f"{self.input_size}, {self.hidden_size}, num_layers={self.num_layers}, batch_first={self.batch_first}"

    def init_state(self, sequences: int) -> SSMState:
        """Zero states of `sequences` sequences: a pool for step()."""
        w = self.layers[0].in_proj.weight
        return SSMState(tuple(w.new_zeros(sequences, l.conv_width - 1, l.inner) for l in self.layers),
                        tuple(torch.zeros(sequences, l.inner, l.state_size, device=w.device) for l in self.layers))

    def forward(self, input: Union[torch.Tensor, PackedSequence], hx: Optional[SSMState] = None, lengths: Optional[Sequence[int]] = None):
        """(output, state): nn.GRU's forward with an SSMState in the place of h_0 and h_n (sequences along dimension 0).
        `lengths` (padded input only): steps of each sequence, any order, zero allowed; outputs behind them are zero."""
        if isinstance(input, PackedSequence):
            if lengths is not None:
                raise ValueError("lengths go with padded input, not with a PackedSequence")
            x, lens = pad_packed_sequence(input, batch_first=True)
            y, state = self._run(x, hx, lens)
            if input.sorted_indices is not None:
                y, lens = y[input.sorted_indices], lens[input.sorted_indices.cpu()]
            data = pack_padded_sequence(y, lens, batch_first=True).data
            return PackedSequence(data, input.batch_sizes, input.sorted_indices, input.unsorted_indices), state
        if input.dim() == 2:       # one sequence, (T, input_size)
            y, state = self.forward(input.unsqueeze(0 if self.batch_first else 1), hx, lengths)
            return y.squeeze(0 if self.batch_first else 1), state
        if input.dim() != 3:
            raise ValueError(f"SSM: Expected input to be 2D or 3D, got {input.dim()}D instead")
        if input.shape[-1] != self.input_size:
            raise RuntimeError(f"input.size(-1) must be equal to input_size. Expected {self.input_size}, got {input.shape[-1]}")
        if self.batch_first:
            return self._run(input, hx, lengths)
        y, state = self._run(input.transpose(0, 1), hx, lengths)
        return y.transpose(0, 1), state

    def _run(self, x: torch.Tensor, hx: Optional[SSMState], lengths):
        lengths = _lengths(lengths, x.shape[0], x.shape[1], x.device)      # once for all layers
        conv, scan = [], []
        for k, layer in enumerate(self.layers):
            x, c, s = layer(x, lengths, None if hx is None else hx.conv[k], None if hx is None else hx.scan[k])
            conv.append(c)
            scan.append(s)
        return x, SSMState(tuple(conv), tuple(scan))

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: SSMState, slots=None) -> torch.Tensor:
        """One more step of each of B sequences, x (B, input_size) -> (B, hidden_size).  `state` (what forward returned, or
        a pool from init_state with `slots`) is updated in place.  No gradients."""
        slots = _slots(slots, x.device)
        for layer, c, s in zip(self.layers, state.conv, state.scan):
            x = layer.step(x, c, s, slots)
        return x
