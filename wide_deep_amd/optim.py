"""AdamW over many tensors at once (csrc/adamw.hip, wd_adamw_step in include/wd_hip.h).

Beside the optimizers of the reference's two scopes (wd_opt_dense, wd_sparse_apply_opt), which update one flat buffer each and follow
tf.train: decoupled weight decay per tensor, clipping by the global norm, moments in 32 or in 8 bits, a half copy of the parameters
written by the same pass.  One or two launches a step whatever the number of tensors; nothing is read back, so a step can be captured
into a hipGraph (the step count lives on the device and advances with every replay).  Tensors and gradients are bound at construction:
a program fills the same gradient buffers every step, as the engine does.
"""
import struct

import numpy as np
import torch

from . import capi

BLOCK, CHUNK, PARTIALS, TICKETS = 64, 2048, 2048, 1056           # WD_ADAMW_*
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TENSOR = np.dtype([("p", "<u8"), ("g", "<u8"), ("copy", "<u8"), ("n", "<i8"), ("start", "<i8"), ("decay", "<f4"), ("pad", "<i4")])
_OPTS = struct.Struct("=QQqQQQQQQQQddfffIiiii")     # wd_adamw_t


class AdamW:
    """params, grads: lists of contiguous tensors on one GPU, fp32 and fp32 / fp16 / bf16 (one type for all gradients), bound for good.
    weight_decay: one number or one per tensor.  max_norm: clip by the global norm of all gradients (math.inf: tell it and clip nothing); a step whose norm is not finite
    (elements above 6.5e18 may do that: the squares of eight are added in fp32) changes nothing and is counted in `skipped`.  state_bits: 32, or 8 (m and the root r of the second moment, one byte each; rounding by
    a hash of index, step and `seed`, so runs repeat; elements whose root is below 2^-18 of the largest of their 64 take smaller steps than with 32).  copies: fp16 or bf16 tensors that receive the updated parameters (None where a
    tensor has none).

    Moments are flat buffers over all tensors, tensor k from element `starts[k]` on: `m`, `v` (state_bits 32) or the codes `m`, `r` and
    scales `m_scale`, `r_scale`.  One step at a time: steps of one optimizer may not overlap on two streams."""

    def __init__(self, params, grads, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_norm=None, state_bits=32, copies=None, seed=0):
        params, grads = list(params), list(grads)
        copies = [None] * len(params) if copies is None else list(copies)
        if not params or len(grads) != len(params) or len(copies) != len(params):
            raise ValueError("AdamW: %d parameters, %d gradients, %d copies: at least one, and as many of each" % (len(params), len(grads), len(copies)))
        try:
            decay = [float(weight_decay)] * len(params)
        except TypeError:
            decay = [float(d) for d in weight_decay]
        if len(decay) != len(params):
            raise ValueError("AdamW: %d weight decays for %d parameters" % (len(decay), len(params)))
        self.betas = (float(betas[0]), float(betas[1]))
        if not (0.0 <= self.betas[0] < 1.0 and 0.0 <= self.betas[1] < 1.0 and eps >= 0.0):
            raise ValueError("AdamW: betas in [0, 1) and eps >= 0 are wanted, got %r, %r" % (betas, eps))
        if state_bits not in (8, 32):
            raise ValueError("AdamW: state_bits is 32 or 8, got %r" % (state_bits,))
        if max_norm is not None and not np.float32(max_norm) > 0.0:      # as the kernel gets it
            raise ValueError("AdamW: max_norm must be positive in fp32, got %r" % (max_norm,))
        copy_type = {c.dtype for c in copies if isinstance(c, torch.Tensor)}
        if len(copy_type) > 1 or copy_type - {torch.float16, torch.bfloat16}:
            raise ValueError("AdamW: copies of one half type are wanted, got %s" % sorted(map(str, copy_type)))
        dev = params[0].device
        for k, (p, g, c) in enumerate(zip(params, grads, copies)):
            for what, t, types in (("parameter", p, (torch.float32,)), ("gradient", g, (grads[0].dtype,)), ("copy", c, copy_type)):
                if t is None and what == "copy":
                    continue
                if not isinstance(t, torch.Tensor) or t.dtype not in types or t.dtype not in _DTYPES or t.shape != p.shape or t.device != dev or not t.is_contiguous():
                    raise ValueError("AdamW: %s %d: a contiguous tensor of %s like its parameter (%s on %s) is wanted, got %s" % (
                        what, k, " or ".join(map(str, types)), list(p.shape), dev, "%s %s on %s, strides %s" % (t.dtype, list(t.shape), t.device, t.stride()) if isinstance(t, torch.Tensor) else repr(t)))
        for what, ts in (("parameters", params), ("copies", [c for c in copies if c is not None])):
            spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in ts if t.numel())
            if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
                raise ValueError("AdamW: %s that share memory (one tensor given twice?): every element may be updated once a step" % what)
        if dev.type != "cuda":
            raise capi.WdError("AdamW needs a GPU (MI355X / gfx950); there is no CPU fallback: parameters are on %s" % dev)
        self.params, self.grads, self.copies = params, grads, copies
        self.lr, self.eps, self.max_norm, self.state_bits, self.seed = float(lr), float(eps), max_norm, state_bits, int(seed) & 0xffffffff
        sizes = np.array([p.numel() for p in params], dtype=np.int64)
        padded = -(-sizes // BLOCK) * BLOCK
        self.starts = (np.cumsum(padded) - padded).tolist()
        self.size = int(padded.sum())                     # elements of the flat moment buffers
        if self.size == 0:
            raise ValueError("AdamW: all parameters are empty")
        table = np.zeros(len(params), dtype=_TENSOR)
        table["p"], table["g"] = [p.data_ptr() for p in params], [g.data_ptr() for g in grads]
        table["copy"] = [0 if c is None else c.data_ptr() for c in copies]
        table["n"], table["start"], table["decay"] = sizes, self.starts, decay
        per = -(-sizes // CHUNK)
        chunks = np.empty((int(per.sum()), 2), dtype=np.int32)
        chunks[:, 0] = np.repeat(np.arange(len(params)), per)
        chunks[:, 1] = np.arange(len(chunks)) - np.repeat(np.cumsum(per) - per, per)
        self._tensors = torch.from_numpy(table.view(np.uint8)).to(dev)
        self._chunks = torch.from_numpy(chunks).to(dev)
        n = self.size
        if state_bits == 32:
            self.m, self.v = torch.zeros(n, dtype=torch.float32, device=dev), torch.zeros(n, dtype=torch.float32, device=dev)
            second, scales = self.v, (0, 0)
        else:
            u8 = dict(dtype=torch.uint8, device=dev)
            self.m, self.r = torch.zeros(n, **u8), torch.zeros(n, **u8)
            self.m_scale, self.r_scale = torch.full((n // BLOCK,), 27, **u8), torch.full((n // BLOCK,), 27, **u8)
            second, scales = self.r, (self.m_scale.data_ptr(), self.r_scale.data_ptr())
        self._state = torch.zeros(12, dtype=torch.int32, device=dev)      # wd_adamw_state_t
        self._tickets = torch.empty(TICKETS, dtype=torch.int32, device=dev)
        #: global norm of the gradients of the last step with max_norm, before clipping; the next step writes it
        self.grad_norm = self._state[10:11].view(torch.float32)[0]
        self._partials = torch.zeros(PARTIALS, dtype=torch.float64, device=dev) if max_norm is not None else None
        self._device = dev
        self._head = (self._tensors.data_ptr(), self._chunks.data_ptr(), len(chunks), self.m.data_ptr(), second.data_ptr(), *scales,
                      self._state.data_ptr(), self._tickets.data_ptr(), 0 if self._partials is None else self._partials.data_ptr())
        self._types = (state_bits, _DTYPES[grads[0].dtype], _DTYPES[copy_type.pop()] if copy_type else 2, 0)
        self.set_step(0)

    def _call(self, name, *args):
        if torch._C._cuda_getDevice() != self._device.index:
            with torch.cuda.device(self._device):
                return self._call(name, *args)
        return capi.call(name, *args, torch._C._cuda_getCurrentRawStream(self._device.index))

    def step(self, lr=None):
        """One step on the gradients as they stand.  lr: a number, or a one-element fp32 tensor on the GPU whose value at the time of the
        launch counts (a captured step whose rate moves); None: `self.lr`."""
        rate, dev_rate = (self.lr, 0) if lr is None else (lr, 0)
        if isinstance(lr, torch.Tensor):
            if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != self._device:
                raise ValueError("AdamW.step: lr as a tensor is one fp32 value on %s, got %s %s on %s" % (self._device, lr.dtype, list(lr.shape), lr.device))
            rate, dev_rate = 0.0, lr.data_ptr()
        self._call("wd_adamw_step", _OPTS.pack(*self._head, dev_rate, *self.betas, rate, self.eps, self.max_norm or 0.0, self.seed, *self._types))

    def set_step(self, step, skipped=0):
        """The number of steps done and skipped so far (a restored optimizer)."""
        self._call("wd_adamw_set_step", self._state.data_ptr(), self._tickets.data_ptr(), int(step), *self.betas)
        if skipped:
            self._state[2].fill_(int(skipped))

    @property
    def step_count(self):
        """Steps done (read back from the device)."""
        return int(self._state[:2].view(torch.int64))

    @property
    def skipped(self):
        """Steps skipped for a norm that was not finite (read back from the device)."""
        return int(self._state[2])

    def moments(self, dtype=torch.bfloat16):
        """8-bit moments as numbers: flat (m, r), r the root of the second moment; bf16 holds every value exactly."""
        if self.state_bits != 8:
            raise ValueError("AdamW.moments: the moments are in `m` and `v` as they are (state_bits 32)")
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("AdamW.moments: bf16 or fp32, got %s" % dtype)
        m, r = self.m.new_empty((2, self.size), dtype=dtype).unbind()
        self._call("wd_adamw_unpack", self._head[3], self._head[5], self._head[4], self._head[6], self.size, m.data_ptr(), r.data_ptr(), _DTYPES[dtype])
        return m, r

    def load_moments(self, m, second):
        """Flat fp32 moments of a checkpoint: m and v (state_bits 32), or m and the root of v, rounded to the nearest codes (state_bits 8)."""
        for t in (m, second):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != (self.size,) or t.device != self._device or not t.is_contiguous():
                raise ValueError("AdamW.load_moments: two contiguous fp32 tensors of %d values on %s are wanted" % (self.size, self._device))
        if self.state_bits == 32:
            self.m.copy_(m)
            self.v.copy_(second)
        else:
            self._call("wd_adamw_pack", m.data_ptr(), second.data_ptr(), self.size, self.m.data_ptr(), self.m_scale.data_ptr(), self.r.data_ptr(),
                       self.r_scale.data_ptr())
