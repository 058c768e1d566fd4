"""AdamW over many tensors in one launch, with states in 32 or 8 bits and the running average of the parameters.

Stands where the reference's training loop has its optimizer and `ExponentialMovingAverage` (src/utils/utils.py; the released checkpoint is such an
average): `weights.trainable_parameters` gives the score model's parameters as device tensors, `ema_parameters()` what `load_state_dict` of the score
model takes for a validation run (`fit.inference_epoch`).  All arithmetic runs in libdiffphore_train.so.
"""
from __future__ import annotations

import ctypes as C
from array import array
from operator import attrgetter
from typing import Iterable, Optional

import numpy as np
import torch
from torch.autograd.graph import increment_version

from . import _trainlib
from ._trainlib import TYPES, DptAdamWArgs, Streams, call, need_gpu

BLOCK = 256                # elements of a tensor that share one scale of an 8-bit state; every tensor's slot in the flat buffers is a multiple of it
_MAX_TENSORS = 400         # per launch
_DTYPE, _SHAPE, _DEVICE, _CONTIGUOUS, _ADDRESS = attrgetter("dtype"), torch.Tensor.size, torch.Tensor.get_device, torch.Tensor.is_contiguous, torch.Tensor.data_ptr
_RECORD = np.dtype([("param", "u8"), ("tensor", "i4"), ("index", "i4"), ("left", "i4"), ("decay", "f4"), ("pad", "i4", 2)])


class AdamW:
    """m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps);
    ema = d ema + (1 - d) p.

    params: a list of contiguous tensors of one type on one GPU, or a dict of them.  fp32 parameters are updated in place; bf16 parameters are the
    roundings of fp32 masters kept here.  They are updated at the memory that they have now: assigning other memory to `p.data` later takes a tensor out of
    the optimiser's reach.  no_decay: indices (dict: names) of the tensors without weight decay.

    State is held in flat buffers (`master`, `ema`, `exp_avg`, `exp_avg_sq`), tensor i in the elements 256 * first_block[i] onwards, each slot rounded up to
    256; the padding stays 0.  state_bits=8: 256 elements share an fp32 scale a (their largest magnitude), m = a c|c| / 127^2 with an int8 c,
    v = a (c / 255)^4 with a uint8 c that is never 0 where v > 0; a step's update uses the new m and v before they are rounded to their codes.
    A gradient that is not finite makes its element's parameter and state NaN - with 8-bit states the state of its whole block.

    The step number lives on the device: a captured `step` counts on with every replay (lr and grad_scale can be device tensors for the same
    reason).  One optimiser is used from one stream at a time.  A step is an in-place change of the parameters: a backward pass over activations that were
    formed with the parameters of before raises (a replayed step moves no version counter).

    `lr` may be set between steps.  The other settings and the state buffers are fixed when the optimiser is made: the launches hold their values and
    addresses."""

    _STATE = ("master", "ema", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
    _FIXED = ("betas", "eps", "weight_decay", "ema_decay", "state_bits") + _STATE
    betas, eps, weight_decay, ema_decay, state_bits, master, ema, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale = (property(attrgetter("_" + n)) for n in _FIXED)

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, no_decay: Iterable = (),
                 state_bits: int = 32, ema_decay: Optional[float] = None):
        self.names = list(params) if isinstance(params, dict) else None
        params = list(params.values()) if self.names is not None else list(params)
        if not params:
            raise ValueError("no parameters")
        for i, p in enumerate(params):
            need_gpu(p, f"parameter {i}")
            if p.dtype != params[0].dtype or p.device != params[0].device:
                raise ValueError(f"parameter {i} is {p.dtype} on {p.device}, parameter 0 is {params[0].dtype} on {params[0].device}")
            if not p.is_contiguous():
                raise ValueError(f"parameter {i} is not contiguous")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size(), i) for i, p in enumerate(params) if p.numel())
        for (_, end, i), (start, _, j) in zip(spans, spans[1:]):
            if start < end:
                raise ValueError(f"parameters {i} and {j} share memory")
        if not eps >= 0.0 or not weight_decay >= 0.0 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas = {betas}, eps = {eps}, weight_decay = {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits = {state_bits}: 8 or 32")
        if ema_decay is not None and not 0.0 <= ema_decay <= 1.0:
            raise ValueError(f"ema_decay = {ema_decay}")
        self.lr, self._betas, self._eps, self._weight_decay = lr, (float(betas[0]), float(betas[1])), float(eps), float(weight_decay)
        self._state_bits, self._ema_decay = state_bits, ema_decay
        self.params = params
        self._alias = [p.detach() for p in params]                       # keeps the updated memory alive whatever happens to the tensors
        self.dtype, self.device = params[0].dtype, params[0].device
        number = {n: i for i, n in enumerate(self.names)} if self.names is not None else None
        decay = np.ones(len(params), dtype=np.float32)
        for n in no_decay:
            if (n not in number) if number is not None else not 0 <= int(n) < len(params):
                raise ValueError(f"no_decay: there is no parameter {n!r}")
            decay[number[n] if number is not None else int(n)] = 0.0
        self._numel, self._sizes = [p.numel() for p in params], [p.shape for p in params]
        blocks = [-(-n // BLOCK) for n in self._numel]
        self.first_block = [0]
        for b in blocks:
            self.first_block.append(self.first_block[-1] + b)
        self.n_blocks = self.first_block[-1]
        if self.n_blocks >= 1 << 30:
            raise ValueError("too many elements")

        which = np.repeat(np.arange(len(params), dtype=np.int32), blocks)                # DptAdamWBlock records
        index = np.arange(self.n_blocks, dtype=np.int32) - np.asarray(self.first_block[:-1], dtype=np.int32)[which]
        rec = np.zeros(self.n_blocks, dtype=_RECORD)
        rec["tensor"], rec["index"], rec["decay"] = which, index, decay[which]
        rec["param"] = np.asarray([p.data_ptr() for p in params], dtype=np.uint64)[which] + index.astype(np.uint64) * (BLOCK * params[0].element_size())
        rec["left"] = np.minimum(np.asarray(self._numel, dtype=np.int64)[which] - index.astype(np.int64) * BLOCK, BLOCK)
        self._blocks = torch.from_numpy(rec.view(np.uint8)).to(self.device)

        def flat(dtype=torch.float32):
            return torch.zeros(self.n_blocks * BLOCK, dtype=dtype, device=self.device)
        self._master = self._gather(flat()) if self.dtype == torch.bfloat16 else None
        self._ema = self._gather(flat()) if ema_decay is not None else None
        small = state_bits == 8
        self._exp_avg, self._exp_avg_sq = flat(torch.int8 if small else torch.float32), flat(torch.uint8 if small else torch.float32)
        self._exp_avg_scale, self._exp_avg_sq_scale = (torch.zeros(self.n_blocks, dtype=torch.float32, device=self.device) if small else None for _ in range(2))
        self._counter = torch.tensor([0.0, 1.0, 1.0, 0.0], dtype=torch.float64, device=self.device)
        self._state = [t for t in (getattr(self, n) for n in self._STATE) if t is not None]
        self._changed = self._alias + self._state
        self._args = self._make_args()
        self._streams = Streams(self.device, [self._blocks, self._counter, *self._alias, *self._state])

    @property
    def lr(self) -> float:
        return self._lr

    @lr.setter
    def lr(self, lr):
        self._lr = self._rate(lr)

    @staticmethod
    def _rate(lr) -> float:
        lr = float(lr)
        if not lr >= 0.0:
            raise ValueError(f"lr = {lr}")
        return lr

    # ---- flat buffers ---------------------------------------------------------------------------------------------------
    def views(self, flat: torch.Tensor):
        """The tensors' parts of a flat buffer, in the parameters' shapes: a list, or a dict if the parameters came as one."""
        out = [flat[b * BLOCK:b * BLOCK + n].view(s) for b, n, s in zip(self.first_block, self._numel, self._sizes)]
        return dict(zip(self.names, out)) if self.names is not None else out

    def _gather(self, flat):
        v = self.views(flat)
        for dst, p in zip(v.values() if isinstance(v, dict) else v, self._alias):
            dst.copy_(p)
        return flat

    def ema_parameters(self):
        """The averaged parameters (fp32 views), named as the parameters are."""
        if self.ema is None:
            raise ValueError("ema_decay was not given")
        return self.views(self.ema)

    def moments(self):
        """(exp_avg, exp_avg_sq) as flat fp32 buffers: the state itself, or the values that 8-bit codes stand for."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        m, v = torch.empty((2, self.n_blocks * BLOCK), dtype=torch.float32, device=self.device)
        self._streams.use()
        call("dpt_adamw_moments", _trainlib.lib().dpt_adamw_moments, self.device.index, self.exp_avg.data_ptr(), self.exp_avg_scale.data_ptr(),
             self.exp_avg_sq.data_ptr(), self.exp_avg_sq_scale.data_ptr(), self.n_blocks, m.data_ptr(), v.data_ptr())
        return m, v

    # ---- checkpoints ----------------------------------------------------------------------------------------------------
    def state_dict(self):
        """Copies of the state, with the names and shapes of the tensors that it belongs to (host-synchronising: the step number is read back)."""
        self._streams.use()
        return {"step": int(self._counter[0].item()), "state_bits": self.state_bits, "names": list(self.names) if self.names is not None else None, "sizes": [tuple(s) for s in self._sizes],
                **{n: getattr(self, n).clone() if getattr(self, n) is not None else None for n in self._STATE}}

    def _refresh(self):
        """The bf16 parameters as the roundings of their masters."""
        v = self.views(self.master)
        for p, m in zip(self._alias, v.values() if isinstance(v, dict) else v):
            p.copy_(m)

    def load_state_dict(self, state):
        """The state of `state_dict`, of an optimiser of the same tensors in the same order (a state without `names` or `sizes` is taken by the length of its
        buffers); bf16 parameters become the roundings of the loaded masters (fp32 parameters are not part of the state)."""
        t = int(state["step"])
        if t < 0:
            raise ValueError(f"step = {t}")
        if state["state_bits"] != self.state_bits:
            raise ValueError(f"the state has {state['state_bits']} bits, the optimiser {self.state_bits}")
        names, sizes = state.get("names"), state.get("sizes")
        if sizes is not None and [tuple(s) for s in sizes] != [tuple(s) for s in self._sizes]:
            raise ValueError("the state belongs to tensors of other shapes, or in another order")
        if names is not None and self.names is not None and list(names) != self.names:
            raise ValueError("the state belongs to tensors of other names, or in another order")
        self._streams.use()
        for n in self._STATE:
            mine, given = getattr(self, n), state.get(n)
            if (mine is None) != (given is None) or (mine is not None and (mine.shape != given.shape or mine.dtype != given.dtype)):
                raise ValueError(f"{n} does not fit this optimiser")
        for n in self._STATE:
            if getattr(self, n) is not None:
                getattr(self, n).copy_(state[n])
        if self.master is not None:
            self._refresh()
        self._counter.copy_(torch.tensor([t, self.betas[0] ** t, self.betas[1] ** t, 0.0], dtype=torch.float64))

    # ---- the step -------------------------------------------------------------------------------------------------------
    def _make_args(self):
        a = DptAdamWArgs()
        a.type, a.state_bits = TYPES[self.dtype], self.state_bits
        a.beta1, a.beta2, a.eps, a.weight_decay, a.ema_decay = *self.betas, self.eps, self.weight_decay, self.ema_decay or 0.0
        a.blocks = self._blocks.data_ptr()
        for n in self._STATE:
            setattr(a, n, getattr(self, n).data_ptr() if getattr(self, n) is not None else None)
        a.counter = self._counter.data_ptr()
        return a

    def _scalar(self, x, name):
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{name}: a tensor is wanted, got {type(x).__name__}")
        if x.dtype != torch.float32 or x.numel() != 1 or x.device != self.device:
            raise ValueError(f"{name}: one float32 value on {self.device} is wanted, got {x.numel()} of {x.dtype} on {x.device}")
        return x.data_ptr()

    def step(self, grads=None, lr=None, grad_scale: Optional[torch.Tensor] = None):
        """One step with the gradients `grads` (a list, or a dict as the parameters; by default the parameters' `.grad`), contiguous, in the parameters' type
        or fp32.  A tensor whose gradient is None stays as it is, with its state.  lr: another learning rate for this step, a number or a float32
        tensor on the device.  grad_scale: a float32 tensor on the device that multiplies the gradients."""
        if grads is None:
            grads = [p.grad for p in self.params]
        elif not isinstance(grads, (list, dict)):
            grads = list(grads)
        if isinstance(grads, dict):
            if self.names is None or grads.keys() - set(self.names):
                raise ValueError("grads names tensors that are not parameters")
            grads = [grads.get(n) for n in self.names]
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        # one pass per property over the whole list: some hundreds of small tensors are the common case, and a loop over all of them costs more than the step
        some = grads if type(None) not in set(map(type, grads)) else [g for g in grads if g is not None]
        if not all(issubclass(c, torch.Tensor) for c in set(map(type, some))):
            raise TypeError(f"gradients are tensors or None, got {set(map(type, some))}")
        types = set(map(_DTYPE, some)) or {self.dtype}
        if len(types) > 1 or not types <= {self.dtype, torch.float32}:
            raise TypeError(f"gradients in {types}: all in {self.dtype}, or all in float32")
        fits = list(map(_SHAPE, some)) == (self._sizes if some is grads else [s for s, g in zip(self._sizes, grads) if g is not None])
        if not fits or not set(map(_DEVICE, some)) <= {self.device.index} or not all(map(_CONTIGUOUS, some)):
            for i, (g, s) in enumerate(zip(grads, self._sizes)):
                if g is not None and (g.shape != s or g.get_device() != self.device.index or not g.is_contiguous()):
                    raise ValueError(f"gradient {i} is {tuple(g.shape)} on {g.device}: contiguous {tuple(s)} on {self.device} is wanted")
        ptrs = list(map(_ADDRESS, grads)) if some is grads else [g.data_ptr() if g is not None else 0 for g in grads]
        L = _trainlib.lib()
        self._streams.use()
        a = self._args
        a.grad_type = TYPES[types.pop()]
        a.lr_dev, a.lr = (self._scalar(lr, "lr"), 0.0) if isinstance(lr, torch.Tensor) else (None, self._lr if lr is None else self._rate(lr))
        a.grad_scale = self._scalar(grad_scale, "grad_scale") if grad_scale is not None else None
        for i in range(0, len(ptrs), _MAX_TENSORS):
            part = array("Q", ptrs[i:i + _MAX_TENSORS])
            a.tensor0, a.n_tensors, a.block0, a.last = i, len(part), self.first_block[i], int(i + len(part) == len(ptrs))
            a.n_blocks = self.first_block[i + len(part)] - a.block0
            call("dpt_adamw_step", L.dpt_adamw_step, self.device.index, C.byref(a), part.buffer_info()[0])
        # autograd sees an in-place change, as it would of a torch operator (the aliases share the parameters' counters)
        increment_version(self._changed if some is grads else [p for p, g in zip(self._alias, grads) if g is not None] + self._state)

    def zero_grad(self):
        for p in self.params:
            p.grad = None
