"""AdamW over any list of tensors, in one pass over all of them (csrc/adamw.hip).

Beside `_FlatAdam` (algo/ppo.py), which steps on a policy's one flat fp32 buffer: parameters here may be separate tensors of any
size, fp32 or 16-bit, with fp32 or 16-bit gradients; weight decay is decoupled from the gradient; the moments take 8 bytes or 2
bytes per parameter; 16-bit copies of fp32 parameters (the weights a mixed-precision layer multiplies with) are written in the
same pass.  The step counter and the hyperparameters live in device memory, so a step that was captured into a hipGraph replays
with the right bias corrections.
"""
import ctypes
import operator

import torch

from .. import _hip, ops

f32 = torch.float32
_POINTER, _COUNT, _DENSE, _TYPE = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous, operator.attrgetter('dtype')


class AdamW(object):
    """params: tensors to step on, in place.  grads: their gradients, one tensor each (default: every parameter's .grad, or its
    copy's, at the time of the step).  copies: 16-bit tensors of the parameters' shapes (entries may be None) that receive the
    new parameters rounded to nearest.  max_grad_norm: gradients are scaled as they are read, as clip_grad_norm_ would; they
    stay as they are.  state_bits: 32, or 8 (blocks of 256 values with a common scale, rounded stochastically; `seed` names
    the random sequence).  All tensors are contiguous and on one GPU."""

    def __init__(self, params, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_grad_norm=None, grads=None, copies=None,
                 state_bits=32, seed=0):
        params = list(params)
        if not params:
            raise ValueError('AdamW: no parameters')
        if state_bits not in (32, 8):
            raise ValueError('AdamW: state_bits must be 32 or 8 (got %r)' % (state_bits,))
        self.grads = list(grads) if grads is not None else None
        self.copies = list(copies) if copies is not None else [None] * len(params)
        if len(self.copies) != len(params) or (self.grads is not None and len(self.grads) != len(params)):
            raise ValueError('AdamW: as many gradients and copies as parameters are needed')
        self.param_groups = [{'params': params, 'lr': lr, 'betas': betas, 'eps': eps, 'weight_decay': weight_decay,
                              'max_grad_norm': max_grad_norm}]
        self._copied = [c for c in self.copies if c is not None]
        self._check_hyper()
        self.state_bits, self.seed = state_bits, int(seed)
        self.step_count = 0
        self._dev = None
        self._seen = self._hyper = None

    @property
    def params(self):
        return self.param_groups[0]['params']

    # ------------------------------------------------------------------ host-side state
    def _check_hyper(self):
        g = self.param_groups[0]
        c = g['max_grad_norm']
        if not (g['lr'] >= 0 and g['eps'] >= 0 and g['weight_decay'] >= 0 and all(0 <= b < 1 for b in g['betas']) and
                (c is None or c > 0)):
            raise ValueError('AdamW: lr, eps and weight_decay must be >= 0, betas in [0, 1), max_grad_norm > 0 or None')

    def _allocate(self, dev):
        """Moments: one buffer each; every tensor starts at a multiple of the block."""
        L = _hip.lib()
        block = L.acktr_adamw_block()
        self._offs, off = [], 0
        for p in self.params:
            self._offs.append(off)
            off += -(-p.numel() // block) * block
        self._numel = [p.numel() for p in self.params]
        self._total, self._dev = off, dev
        dt = f32 if self.state_bits == 32 else torch.uint8
        self.mom1 = torch.zeros(off, dtype=dt, device=dev)
        self.mom2 = torch.zeros(off, dtype=dt, device=dev)
        self.scales = torch.zeros(2 * off // block, dtype=f32, device=dev) if self.state_bits == 8 else None
        self._tensors = torch.zeros(len(self.params) * ctypes.sizeof(_hip.AdamwTensor), dtype=torch.uint8, device=dev)
        words = -(-L.acktr_adamw_state_bytes() // 8)
        self._state = torch.zeros(words, dtype=torch.float64, device=dev)
        self._state[6:8].view(torch.int64).copy_(torch.tensor([self.step_count, self.seed]))
        chunk = L.acktr_adamw_chunk()
        count = torch.tensor([-(-n // chunk) for n in self._numel])
        which = torch.repeat_interleave(count)                # {tensor, chunk number} pairs
        first = torch.cumsum(count, 0) - count
        self._chunks = torch.stack((which, torch.arange(which.numel()) - first[which]), 1).to(torch.int32).to(dev)
        # (pointers to what never moves)
        self._fixed = self._state.data_ptr(), self._tensors.data_ptr(), self._chunks.data_ptr(), self._chunks.shape[0]
        self._seen = self._hyper = None

    def _gradients(self):
        if self.grads is not None:
            return self.grads
        out = []
        for i, (p, c) in enumerate(zip(self.params, self.copies)):
            g = p.grad if p.grad is not None else (c.grad if c is not None else None)
            if g is None:
                raise RuntimeError('AdamW: parameter %d has no gradient' % i)
            out.append(g)
        return out

    def _table(self, grads):
        """The device table of tensors, rebuilt (and its entries checked) only when one of them changed: another address, size, type
        or layout."""
        every = self.params + self._copied + grads
        seen = [list(map(_POINTER, every)), list(map(_COUNT, every)), list(map(_TYPE, every)), all(map(_DENSE, every))]
        if seen == self._seen:
            return
        dev = self._dev
        rows = (_hip.AdamwTensor * len(self.params))()
        for i, (p, g, c) in enumerate(zip(self.params, grads, self.copies)):
            for t, what in ((p, 'parameter'), (g, 'gradient'), (c, 'copy')):
                if t is None:
                    continue
                if not t.is_cuda or t.device != dev:
                    raise RuntimeError('AdamW: %s %d is on %s, expected %s' % (what, i, t.device, dev))
                if t.dtype not in ops.DTYPE_CODE:
                    raise RuntimeError('AdamW: %s %d must be bfloat16, float16 or float32 (got %s)' % (what, i, t.dtype))
                if tuple(t.shape) != tuple(p.shape) or not t.is_contiguous():
                    raise RuntimeError('AdamW: %s %d must be contiguous and of the parameter\'s shape %s (got %s)'
                                       % (what, i, tuple(p.shape), tuple(t.shape)))
            if p.numel() != self._numel[i]:
                raise RuntimeError('AdamW: parameter %d changed its size' % i)
            quad = lambda t: t is not None and t.data_ptr() % (4 * t.element_size()) == 0
            rows[i] = _hip.AdamwTensor(p.data_ptr(), g.data_ptr(), None if c is None else c.data_ptr(), p.numel(), self._offs[i],
                                       ops.DTYPE_CODE[p.dtype], ops.DTYPE_CODE[g.dtype],
                                       ops.DTYPE_CODE[c.dtype] if c is not None else 0,
                                       (1 if quad(p) else 0) | (2 if quad(g) else 0) | (4 if quad(c) else 0))
        spans = sorted((t.data_ptr(), t.data_ptr() + t.nbytes) for t in self.params + self._copied if t.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise RuntimeError('AdamW: two of the tensors to be written overlap (the same parameter twice?)')
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('AdamW: the tensors changed since the last step; run prepare() before the capture')
        # (into the same memory: a captured step reads the table there)
        self._tensors.copy_(torch.frombuffer(bytearray(bytes(rows)), dtype=torch.uint8))
        self._seen = seen

    def _place(self):
        """Moments, tables and device state, made where the parameters are when they are first needed."""
        dev = self.params[0].device
        if self._dev != dev:
            if dev.type != 'cuda':
                raise RuntimeError('AdamW: parameters must live on the MI355X device (got %s): this package has no CPU path' % dev)
            if self._dev is not None:
                raise RuntimeError('AdamW: the parameters moved to %s; build a new optimiser' % dev)
            with torch.no_grad():
                self._allocate(dev)

    def prepare(self):
        """Brings the device side up to date with the parameter list and the hyperparameters: outside a graph capture, and before a
        replay when a hyperparameter changed."""
        g = self.param_groups[0]
        self._place()
        b1, b2 = g['betas']
        hyper = (float(g['lr']), float(b1), float(b2), float(g['eps']), float(g['weight_decay']), float(g['max_grad_norm'] or 0.0))
        if hyper != self._hyper:
            self._check_hyper()
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError('AdamW: a hyperparameter changed; run prepare() before the capture')
            with torch.no_grad():
                self._state[:6].copy_(torch.tensor(hyper, dtype=torch.float64))
            self._hyper = hyper
        grads = self._gradients()
        self._table(grads)

    # ------------------------------------------------------------------ torch.optim surface
    def zero_grad(self, set_to_none=False):
        for t in self.grads if self.grads is not None else self.params + self._copied:
            if self.grads is not None:
                t.zero_()
            elif t.grad is not None:
                if set_to_none:
                    t.grad = None
                else:
                    t.grad.detach().zero_()

    def step(self):
        """One step on all tensors: two launches."""
        self.prepare()
        # (a captured step looks the clip norm up when it is replayed, so that one given or taken away later counts)
        clip = self._hyper[5] > 0 or torch.cuda.is_current_stream_capturing()
        ops._launch(_hip.lib().acktr_adamw_step, self._dev.index, 'adamw_step', 20.0 * self._total, *self._fixed, self.mom1.data_ptr(),
                    self.mom2.data_ptr(), self.scales.data_ptr() if self.scales is not None else None, self.state_bits,
                    1 if clip else 0)
        ops._written(self.params + self._copied)
        self.step_count += 1

    def moments(self):
        """(m, v) as fp32, one value per element of the state buffers (tensor k from offsets()[k] on): the buffers themselves, or, of
        8-bit moments, the values they stand for."""
        self._place()
        if self.state_bits == 32:
            return self.mom1, self.mom2
        m, v = torch.empty(self._total, dtype=f32, device=self._dev), torch.empty(self._total, dtype=f32, device=self._dev)
        ops._launch(_hip.lib().acktr_adamw_read_moments, self._dev.index, 'adamw_read_moments', 0.0, self.mom1.data_ptr(),
                    self.mom2.data_ptr(), self.scales.data_ptr(), m.data_ptr(), v.data_ptr(), self._total)
        return m, v

    def offsets(self):
        """Where each tensor's moments start in the state buffers."""
        self._place()
        return list(self._offs)

    def state_dict(self):
        self._place()
        own = lambda t: None if t is None else t.clone()
        return dict(step=self.steps_done(), seed=self.seed, state_bits=self.state_bits, mom1=own(self.mom1), mom2=own(self.mom2),
                    scales=own(self.scales), hyper={k: v for k, v in self.param_groups[0].items() if k != 'params'})

    def load_state_dict(self, sd):
        if sd['state_bits'] != self.state_bits:
            raise ValueError('AdamW: the state holds %d-bit moments, this optimiser %d' % (sd['state_bits'], self.state_bits))
        self._place()
        if sd['mom1'].numel() != self._total:
            raise ValueError('AdamW: the state belongs to other parameters')
        self.param_groups[0].update(sd['hyper'])
        self.step_count, self.seed = int(sd['step']), int(sd['seed'])
        with torch.no_grad():
            self.mom1.copy_(sd['mom1'])
            self.mom2.copy_(sd['mom2'])
            if self.scales is not None:
                self.scales.copy_(sd['scales'])
            self._state[6:8].view(torch.int64).copy_(torch.tensor([self.step_count, self.seed]))

    def steps_done(self):
        """The device's step counter (replays of a captured step count too; synchronises)."""
        return self.step_count if self._dev is None else int(self._state[6:7].view(torch.int64).item())
