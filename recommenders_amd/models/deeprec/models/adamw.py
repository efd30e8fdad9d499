"""AdamW over many tensors at once, with its states in 32 or in 8 bits (``xdfm_adamw_*`` of include/xdfm.h).

    opt = AdamW(params, grads, weight_decay=[0.01, 0.0, ...], state_bits=8)
    ...                                    # gradients are written into `grads`
    opt.step(lr=1e-3, step=t)              # t = 1, 2, ...: one launch, however many tensors

The addresses of the tensors are laid down once, so they have to stay where they are (parameters and gradients in
place, as ``XDeepFMEngine``'s flat buffers are); their contents are read and written by every step.
"""

import ctypes

import torch

from recommenders_amd import _lib

__all__ = ["AdamW"]

_GRAD_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BLOCK = 64  # elements that share a scale byte


class AdamW(object):
    """One optimizer over ``params`` (fp32) and ``grads`` (fp32, bf16 or fp16), contiguous tensors of one GPU.

    ``weight_decay``: decoupled decay, one number or one per tensor.  ``slot_m``, ``slot_v`` (and ``scale_m``,
    ``scale_v`` with ``state_bits=8``): the states, by default new ones of zeros; fp32 of the parameter's size, or
    uint8 codes of its size and uint8 scales of one per 64 elements.  The lists stay readable as attributes.
    """

    def __init__(self, params, grads, weight_decay=0.01, state_bits=32, slot_m=None, slot_v=None, scale_m=None,
                 scale_v=None):
        params, grads = list(params), list(grads)
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8")
        if len(grads) != len(params):
            raise ValueError("%d parameters, %d gradients" % (len(params), len(grads)))
        if not params:
            raise ValueError("AdamW needs at least one parameter")
        self.device = params[0].device
        if self.device.type != "cuda":
            raise ValueError("AdamW runs on the GPU, the first parameter is on %s" % self.device)
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * len(params)
        if len(decay) != len(params):
            raise ValueError("%d parameters, %d weight_decay" % (len(params), len(decay)))
        self.state_bits = state_bits
        sizes = [p.numel() for p in params]
        blocks = [(n + BLOCK - 1) // BLOCK for n in sizes]
        coded = state_bits == 8
        if not coded and (scale_m is not None or scale_v is not None):
            raise ValueError("32-bit states have no scales")
        dtype = torch.uint8 if coded else torch.float32
        self.params, self.grads = params, grads
        self.slot_m, self.slot_v = self._state(slot_m, sizes, dtype), self._state(slot_v, sizes, dtype)
        self.scale_m = self._state(scale_m, blocks, dtype) if coded else [None] * len(params)
        self.scale_v = self._state(scale_v, blocks, dtype) if coded else [None] * len(params)
        self._check("parameter", params, sizes, (torch.float32,))
        self._check("gradient", grads, sizes, tuple(_GRAD_DTYPE))
        for name, slots, n in (("slot_m", self.slot_m, sizes), ("slot_v", self.slot_v, sizes)):
            self._check(name, slots, n, (dtype,))
        if coded:
            self._check("scale_m", self.scale_m, blocks, (dtype,))
            self._check("scale_v", self.scale_v, blocks, (dtype,))

        def at(t):
            return t.data_ptr() if t is not None and t.numel() else None

        table = (_lib.AdamWTensor * len(params))()
        for k, n in enumerate(sizes):
            table[k] = _lib.AdamWTensor(at(params[k]), at(grads[k]), at(self.slot_m[k]), at(self.slot_v[k]),
                                        at(self.scale_m[k]), at(self.scale_v[k]), n, float(decay[k]),
                                        _GRAD_DTYPE[grads[k].dtype])
        self._info = _lib.AdamWPlanInfo()
        _lib.check(_lib.lib.xdfm_adamw_plan(table, len(params), state_bits, None, 0, ctypes.byref(self._info)))
        image = torch.empty((max(self._info.bytes // 8, 1),), dtype=torch.int64)
        _lib.check(_lib.lib.xdfm_adamw_plan(table, len(params), state_bits, image.data_ptr(), image.numel() * 8,
                                            ctypes.byref(self._info)))
        self._plan = image.to(self.device)  # (a copy from pageable memory: done when this returns)
        self._index = self._plan.device.index
        self._call = (self._plan.data_ptr(), ctypes.byref(self._info))
        self.elements = int(self._info.elements)

    def _state(self, given, sizes, dtype):
        if given is not None:
            return list(given)
        flat = torch.zeros((sum(sizes),), dtype=dtype, device=self.device)
        return list(torch.split(flat, sizes))

    def _check(self, what, tensors, sizes, dtypes):
        if len(tensors) != len(sizes):
            raise ValueError("%d parameters, %d of %s" % (len(sizes), len(tensors), what))
        for k, (t, n) in enumerate(zip(tensors, sizes)):
            if t.dtype not in dtypes:
                raise ValueError("%s %d is %s" % (what, k, t.dtype))
            if t.device != self.device:
                raise ValueError("%s %d is on %s, the first parameter on %s" % (what, k, t.device, self.device))
            if t.numel() != n:
                raise ValueError("%s %d has %d elements instead of %d" % (what, k, t.numel(), n))
            if not t.is_contiguous():
                raise ValueError("%s %d is not contiguous" % (what, k))

    def _enqueue(self, fn, *args):
        """fn(plan, info, *args, stream) on the current stream of the plan's device."""
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        if torch.cuda.current_device() == self._index:
            _lib.check(fn(*self._call, *args, stream))
        else:
            with torch.cuda.device(self._index):
                _lib.check(fn(*self._call, *args, stream))

    def step(self, lr, beta1=0.9, beta2=0.999, eps=1e-8, step=None, opt_state=None, seed=0):
        """One step of every tensor on the current stream.  The step count t (from 1) is ``step``, or is read from
        ``opt_state[3]`` on the device (a float tensor kept by ``xdfm_opt_advance``) so that the call can be captured
        in a HIP graph (a float: it stays at 2^24, where t no longer matters to the step; the rounding of 8-bit states
        goes on by other bits).  ``seed``: of the rounding of 8-bit states."""
        if (step is None) == (opt_state is None):
            raise ValueError("AdamW.step takes either step or opt_state")
        if opt_state is None:
            at = None
        else:
            if (opt_state.dtype != torch.float32 or opt_state.device != self.device or opt_state.numel() < 4
                    or not opt_state.is_contiguous()):
                raise ValueError("opt_state has to be four contiguous floats on %s" % self.device)
            step, at = 0, opt_state.data_ptr()
        args = _lib.AdamWArgs(lr, beta1, beta2, eps, at, step, seed & (2 ** 64 - 1))
        self._enqueue(_lib.lib.xdfm_adamw_step, ctypes.byref(args))

    def _values(self, t, dtype, what):
        if t.dtype != dtype or t.device != self.device or t.numel() != self.elements or not t.is_contiguous():
            raise ValueError("%s has to be %d contiguous elements of %s on %s"
                             % (what, self.elements, dtype, self.device))
        return t.data_ptr()

    def read_state(self, m=None, v=None):
        """The 8-bit states as the values they stand for: (m, v), bf16, the tensors one behind the other."""
        new = [torch.empty((self.elements,), dtype=torch.bfloat16, device=self.device) if t is None else t
               for t in (m, v)]
        self._enqueue(_lib.lib.xdfm_adamw_state_read, self._values(new[0], torch.bfloat16, "m"),
                      self._values(new[1], torch.bfloat16, "v"))
        return tuple(new)

    def write_state(self, m, v):
        """8-bit states from values (fp32, the tensors one behind the other), rounded to the nearest."""
        self._enqueue(_lib.lib.xdfm_adamw_state_write, self._values(m, torch.float32, "m"),
                      self._values(v, torch.float32, "v"))
