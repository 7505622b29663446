"""The gated recurrent core: a recurrence that is linear in its state, so a sequence is one scan (csrc/gated_scan.hip) between two
products (csrc/linear_act.hip) instead of one dependent launch per step.  No counterpart in the reference.

    (gate | value) = x W_in^T + b_in,   f = sigmoid(gate)
    h_t = f_t (m_t h_{t-1}) + (1 - f_t) value_t
    y = h + silu(h W_out^T + b_out)

`GatedCore` is the nn.Module (also `Policy(..., base_kwargs={'recurrent': 'gated'})`, through engine.py); `linear_act` and `gated_scan`
are its two operators as differentiable functions.
"""
import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import ops


def _rows(t, last):
    """[rows, last] view of a tensor, or a copy where its rows share memory or are not contiguous (expanded, transposed)"""
    t = t.reshape(-1, last)
    if (last > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < last):
        t = t.contiguous()
    return t


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, act, residual):
        need = any(ctx.needs_input_grad[:3])
        pre = x.new_empty((x.shape[0], w.shape[0])) if need and ops.LINEAR_ACT[act] else None
        y = ops.linear_act_fwd(x, w, b, act=act, residual=residual, pre=pre)
        ctx.act = act
        ctx.save_for_backward(x, w, pre)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        dense = dy.contiguous()
        if any(need[:3]):
            dx, dw, db = ops.linear_act_bwd(dense, x, w, pre=pre, act=ctx.act, need_dx=need[0], need_dw=need[1], need_db=need[2])
        return dx, dw, db, None, dy if need[4] else None


def linear_act(x, w, b=None, act=None, residual=None):
    """act(x w^T + b) + residual for x [..., K], residual [..., N]; differentiable in every tensor."""
    ops._act_code(act)
    if residual is not None and residual.shape != x.shape[:-1] + w.shape[:1]:
        raise RuntimeError('linear_act: residual must have shape %s (got %s)' % (tuple(x.shape[:-1] + w.shape[:1]), tuple(residual.shape)))
    r = _rows(residual, w.shape[0]) if residual is not None else None
    return _LinearAct.apply(_rows(x, x.shape[-1]), w, b, act, r).view(*x.shape[:-1], w.shape[0])


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, value, h0, masks):
        out, last, saved = ops.gated_scan_fwd(gate, value, h0, masks, save=any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(gate, value, h0, masks, saved)
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast):
        gate, value, h0, masks, saved = ctx.saved_tensors
        if dout is None and dlast is None:
            return None, None, None, None
        dout = torch.zeros_like(value, memory_format=torch.contiguous_format) if dout is None else dout
        if dout.shape[-1] > 1 and dout.stride(-1) != 1:
            dout = dout.contiguous()
        dlast = dlast.contiguous() if dlast is not None else None
        dg, dv, dh0 = ops.gated_scan_bwd(dout, gate, value, h0, masks, saved=saved, dlast=dlast,
                                         need_dh0=h0 is not None and ctx.needs_input_grad[2])
        return dg, dv, dh0, None


def gated_scan(gate, value, h0=None, masks=None):
    """(states [T, N, H], final state [N, H] fp32) of the recurrence; differentiable in gate, value and h0."""
    if gate.dim() != 3 or value.shape != gate.shape:
        raise RuntimeError('gated_scan: gate and value [T, N, H] expected, got %s and %s' % (tuple(gate.shape), tuple(value.shape)))
    unit = lambda t: t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()
    return _GatedScan.apply(unit(gate), unit(value), h0.contiguous() if h0 is not None else None, masks)


class GatedCore(nn.Module):
    """Runs in its parameters' type (fp32, bf16 or fp16); the state is always fp32."""

    def __init__(self, input_size, hidden_size):
        super(GatedCore, self).__init__()
        self.input_size, self.hidden_size = input_size, hidden_size
        self.in_proj = nn.Linear(input_size, 2 * hidden_size)
        self.out_proj = nn.Linear(hidden_size, hidden_size)
        for m in (self.in_proj, self.out_proj):
            nn.init.orthogonal_(m.weight)
            nn.init.constant_(m.bias, 0)
        # gates start with memories of 2 to 128 steps, evenly spread over their logarithm: 1 - f = 1 / tau
        tau = torch.exp(torch.linspace(math.log(2.0), math.log(128.0), hidden_size))
        with torch.no_grad():
            self.in_proj.bias[:hidden_size] = torch.log(tau - 1.0)

    def initial_state(self, n):
        return torch.zeros(n, self.hidden_size, dtype=torch.float32, device=self.in_proj.weight.device)

    def forward(self, x, state=None, masks=None):
        """x [T, N, input_size], state [N, hidden_size] fp32 or None (zeros), masks [T, N] or [T, N, 1] fp32 or None; returns
        (y [T, N, hidden_size], state behind the last step)."""
        H = self.hidden_size
        proj = linear_act(x, self.in_proj.weight, self.in_proj.bias)
        h, last = gated_scan(proj[..., :H], proj[..., H:], state, masks)
        return linear_act(h, self.out_proj.weight, self.out_proj.bias, 'silu', h), last

    @torch.no_grad()
    def step(self, x, state, masks=None):
        """One step for acting: x [N, input_size]; `state` is updated in place; returns y [N, hidden_size]."""
        return ops.gated_core_step(x, self.in_proj.weight, self.in_proj.bias, self.out_proj.weight, self.out_proj.bias, state, masks, state)[0]
