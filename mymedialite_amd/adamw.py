"""AdamW over the parameter tensors of a model, on torch tensors in HBM (mml_adamw_step_device)."""
from __future__ import annotations

import ctypes

import torch

from . import _native as N

_DTYPES = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16}


def _overlap(tensors):
    """Whether two of the contiguous tensors share memory"""
    spans = sorted((x.data_ptr(), x.data_ptr() + x.numel() * x.element_size())
                   for x in tensors if x.numel())
    return any(x[1] > y[0] for x, y in zip(spans, spans[1:]))


class AdamW:
    """One optimizer for a list of contiguous float32, bfloat16 or float16 tensors on one GPU.

    ``step(grads)`` updates the tensors in place on torch's current stream and returns without
    waiting; it may be captured into a graph, and a replay counts its step.  ``StateBits``: 32, or
    8 for moments as e4m3 codes with one scale per 256 values (``m``, ``v`` and ``m_scale``,
    ``v_scale``; ``v`` then holds the codes of sqrt(v)) and a byte for what both codes leave
    (``rest``), without which changes of less than half a code's spacing, which most are, would be
    lost; a ``state`` that has none goes on without.  LearnRate, Beta1, Beta2, Epsilon and
    WeightDecay may be changed between steps.  ``state``: the dict that ``state()`` returned (its
    tensors are used, not copied), to go on from there."""

    def __init__(self, params, LearnRate=1e-3, Beta1=0.9, Beta2=0.999, Epsilon=1e-8,
                 WeightDecay=0.01, StateBits=32, state=None):
        self.LearnRate, self.Beta1, self.Beta2 = LearnRate, Beta1, Beta2
        self.Epsilon, self.WeightDecay = Epsilon, WeightDecay
        if StateBits not in (8, 32):
            raise ValueError("StateBits must be 8 or 32")
        self._bits = StateBits
        self.params = list(params)
        for p in self.params:
            if not isinstance(p, torch.Tensor) or p.dtype not in _DTYPES:
                raise ValueError("parameters must be float32, bfloat16 or float16 tensors")
            if not p.is_cuda:
                raise ValueError("parameters must be on the GPU")
            if p.device != self.params[0].device:
                raise ValueError("parameters must be on one device")
            if not p.is_contiguous():
                raise ValueError("parameters must be contiguous: they are updated in place")
        if _overlap(self.params):
            raise ValueError("a parameter is listed twice, or two overlap")
        self._device = self.params[0].device if self.params else torch.device("cuda", 0)
        blocks = [-(-p.numel() // N.ADAMW_BLOCK) for p in self.params]
        kind = torch.float32 if StateBits == 32 else torch.float8_e4m3fn
        names = ("m", "v") if StateBits == 32 else ("m", "v", "m_scale", "v_scale", "rest")
        s = dict(state) if state is not None else {}
        if state is not None and "rest" not in s:
            names = names[:4]
        for name in names:
            scale = name.endswith("scale")
            dtype = torch.float32 if scale else torch.uint8 if name == "rest" else kind
            if name not in s:
                if state is not None:
                    raise ValueError(f"state has no {name}")
                zeros = torch.uint8 if dtype == torch.float8_e4m3fn else dtype
                s[name] = [torch.zeros(b if scale else p.shape, device=self._device,
                                       dtype=zeros).view(dtype)
                           for p, b in zip(self.params, blocks)]
            x = list(s[name])
            if len(x) != len(self.params):
                raise ValueError(f"state has {len(x)} {name}, expected {len(self.params)}")
            for y, p, b in zip(x, self.params, blocks):
                shape = (b,) if scale else tuple(p.shape)
                if y.dtype != dtype or tuple(y.shape) != shape or y.device != self._device \
                        or not y.is_contiguous():
                    raise ValueError(f"state's {name} must be contiguous {dtype} tensors of the "
                                     "parameters' (scales: blocks') shapes on their device")
            setattr(self, name, x)
        self._names = names
        if _overlap(self.params + [y for name in names for y in getattr(self, name)]):
            raise ValueError("two of the state's tensors overlap, or one and a parameter")
        if int(s.get("step", 0)) < 0:
            raise ValueError("state's step must not be negative")
        self._count = torch.zeros(N.ADAMW_STATE, dtype=torch.int32, device=self._device)
        self._count[0] = int(s.get("step", 0))
        n = len(self.params)
        self._tensors = (N.AdamwTensor * max(n, 1))()
        for i, p in enumerate(self.params):
            t = self._tensors[i]
            t.param, t.m, t.v = p.data_ptr(), self.m[i].data_ptr(), self.v[i].data_ptr()
            if StateBits == 8:
                t.m_scale, t.v_scale = self.m_scale[i].data_ptr(), self.v_scale[i].data_ptr()
                if "rest" in names:
                    t.rest = self.rest[i].data_ptr()
            t.n, t.param_dtype = p.numel(), _DTYPES[p.dtype]

    @property
    def StateBits(self):
        return self._bits

    def step(self, grads):
        """One step with a gradient per parameter (its shape and device; any of the three types)."""
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        keep = []
        for i, (g, p) in enumerate(zip(grads, self.params)):
            if not isinstance(g, torch.Tensor):
                raise ValueError(f"gradient {i} is not a tensor")
            if g.shape != p.shape or g.device != self._device:
                raise ValueError(f"gradient {i} has not its parameter's shape and device")
            if g.dtype not in _DTYPES:
                raise ValueError(f"gradient {i} must be float32, bfloat16 or float16")
            if not g.is_contiguous():
                g = g.contiguous()
                keep.append(g)
            t = self._tensors[i]
            if p.data_ptr() != (t.param or 0):
                raise ValueError(f"parameter {i} is in other memory than at the start")
            t.grad, t.grad_dtype = g.data_ptr(), _DTYPES[g.dtype]
        a = N.AdamwParams(self.LearnRate, self.Beta1, self.Beta2, self.Epsilon, self.WeightDecay,
                          self._bits)
        N.check(N.lib().mml_adamw_step_device(
            self._tensors, len(self.params), ctypes.byref(a), self._count.data_ptr(),
            self._device.index, torch._C._cuda_getCurrentRawStream(self._device.index)))

    def state(self):
        """{"step", "m", "v"}, with 8 bits {"m_scale", "v_scale"} and {"rest"}: the optimizer's own tensors
        and the number of steps done (waits for the device)."""
        s = {n: getattr(self, n) for n in self._names}
        s["step"] = int(self._count[0])
        return s
