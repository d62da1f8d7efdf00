"""The update of a model's weights: AdamW over many tensors in one launch, with
moments in 32 or 8 bits. No counterpart in the reference's runtime; the weights
are those of weights.py or any other float32 torch CUDA tensors.
"""
from __future__ import annotations

import ctypes as C

from ._lib import PRECISION_BF16, PRECISION_F32, AdamwOptions, check, lib, ptr
from .ops import _load, _On, _require

BLOCK = 256  # ILLUMINA_ADAMW_BLOCK


class AdamW:
    """Create with createOptimizer. lr, betas, eps and weightDecay may be changed between steps (a captured step keeps
    the values it was captured with; give lr as a float32 CUDA scalar to change it under a captured step). The optimizer
    must outlive the graphs that captured its steps."""

    def __init__(self, params, lr, betas, eps, weightDecay, decay, momentBits, gradDtype):
        import torch
        self._h = None
        self.params = list(params)
        _require(len(self.params) > 0, "adamw: no tensors")
        for i, p in enumerate(self.params):
            _require(isinstance(p, torch.Tensor) and p.is_cuda and p.dtype == torch.float32 and p.is_contiguous() and not p.is_neg(),
                     f"adamw: parameter {i} must be a contiguous float32 CUDA tensor")
            _require(p.device == self.params[0].device, "adamw: the parameters must be on one device")
        self.device = self.params[0].device
        _require(momentBits in (8, 32), "adamw: momentBits must be 32 or 8")
        _require(gradDtype in (torch.float32, torch.bfloat16), "adamw: gradDtype must be float32 or bfloat16")
        decay = [True] * len(self.params) if decay is None else [bool(d) for d in decay]
        _require(len(decay) == len(self.params), "adamw: decay must have one entry a tensor")
        self.lr, self.betas, self.eps, self.weightDecay = lr, tuple(betas), eps, weightDecay
        self.momentBits, self.gradDtype = momentBits, gradDtype
        n = len(self.params)
        counts = (C.c_longlong * n)(*[p.numel() for p in self.params])
        blocks = C.c_longlong(0)
        check(lib().illumina_adamw_blocks(counts, n, C.byref(blocks)))
        _require(blocks.value > 0, "adamw: every tensor is empty")
        self.blocks = blocks.value
        size, dev = self.blocks * BLOCK, self.device
        if momentBits == 32:
            self.m, self.v = torch.zeros(size, device=dev), torch.zeros(size, device=dev)
            self.mScale = self.vScale = None
        else:
            self.m = torch.zeros(size, dtype=torch.int8, device=dev)
            self.v = torch.zeros(size, dtype=torch.uint8, device=dev)
            self.mScale, self.vScale = torch.zeros(self.blocks, device=dev), torch.zeros(self.blocks, device=dev)
        # the zeros are written on this stream; steps may run on others
        torch.cuda.current_stream(dev).synchronize()
        options = AdamwOptions(device=dev.index, tensors=n,
                               params=(C.c_void_p * n)(*[p.data_ptr() or None for p in self.params]), counts=counts,
                               decay=(C.c_int * n)(*decay), moment_bits=momentBits,
                               grad_precision=PRECISION_F32 if gradDtype == torch.float32 else PRECISION_BF16,
                               m=self.m.data_ptr(), v=self.v.data_ptr(), m_scale=ptr(self.mScale),
                               v_scale=ptr(self.vScale))
        handle = C.c_void_p()
        check(lib().illumina_adamw_create(C.byref(options), C.byref(handle)))
        self._h = handle
        moments = [x for x in (self.m, self.v, self.mScale, self.vScale) if x is not None]
        self._stepper = _load().Stepper(handle.value, self.params, moments, dev.index, gradDtype == torch.bfloat16)

    def step(self, grads, stream=None):
        """One step; grads: one contiguous tensor of gradDtype for each parameter, of its element count. The parameters
        must lie where they lay at creation: a step after p.data = ... or a move of a module is refused (a captured step
        cannot look, and must not be replayed then)."""
        _require(self._h is not None, "adamw: the optimizer was destroyed")
        args = (grads, self.lr, *self.betas, self.eps, self.weightDecay)
        if stream is None:
            return self._stepper.step(*args)
        with _On(self.device, stream):
            return self._stepper.step(*args)

    def moments(self, stream=None):
        """The first and second moments as flat float32 tensors, every parameter from a multiple of 256 elements on.
        With 32 bits these are the moments themselves, with 8 bits new tensors of the values the codes stand for."""
        import torch
        _require(self._h is not None, "adamw: the optimizer was destroyed")
        if self.momentBits == 32:
            return self.m, self.v
        self._stepper.stay()
        with _On(self.device, stream) as handle:
            m = torch.empty(self.blocks * BLOCK, dtype=torch.float32, device=self.device)
            v = torch.empty_like(m)
            check(lib().illumina_adamw_moments(self._h, m.data_ptr(), v.data_ptr(), handle))
        return m, v

    @property
    def steps(self) -> int:
        """Steps taken (waits for the current stream)."""
        _require(self._h is not None, "adamw: the optimizer was destroyed")
        n = C.c_longlong(0)
        with _On(self.device, None) as handle:
            check(lib().illumina_adamw_get_steps(self._h, C.byref(n), handle))
        return n.value

    def state(self) -> dict:
        """What loadState takes: the step count and copies of the moments as they are held (on the current stream)."""
        copy = lambda x: None if x is None else x.clone()  # noqa: E731
        return {"step": self.steps, "m": copy(self.m), "v": copy(self.v), "mScale": copy(self.mScale),
                "vScale": copy(self.vScale)}

    def loadState(self, state: dict) -> None:
        """Sets the step count and the moments (on the current stream)."""
        import torch
        _require(self._h is not None, "adamw: the optimizer was destroyed")
        mine = {"m": self.m, "v": self.v, "mScale": self.mScale, "vScale": self.vScale}
        for name, x in mine.items():
            y = state.get(name)
            _require((x is None) == (y is None) and (x is None or (y.dtype == x.dtype and y.numel() == x.numel())),
                     f"adamw: the state's {name} does not fit")
        _require(int(state["step"]) >= 0, "adamw: the state's step must not be negative")
        for name, x in mine.items():
            if x is not None:
                x.copy_(state[name].reshape(x.shape))
        with _On(self.device, None) as handle:
            check(lib().illumina_adamw_set_steps(self._h, int(state["step"]), handle))

    def destroy(self) -> None:
        if self._h is not None:
            handle, self._h = self._h, None
            check(lib().illumina_adamw_destroy(handle))

    def __del__(self):
        try:
            self.destroy()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


def createOptimizer(params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weightDecay=0.01, decay=None, momentBits=32,
                    gradDtype=None) -> AdamW:
    """AdamW over `params` (contiguous float32 CUDA tensors of one device, updated in place). decay: per tensor, whether
    weight decay applies (default: to all). momentBits 8 keeps the moments as 8-bit codes with a scale for every 256
    elements of a tensor; the second moment's root is held at 1/255 of its block's largest at least, so elements whose
    gradients stay below that are stepped by less than with 32 bits on average. gradDtype: float32 (default) or
    bfloat16. eps is 0 or at least the smallest normal float."""
    import torch
    return AdamW(params, lr, betas, eps, weightDecay, decay, momentBits, gradDtype or torch.float32)
