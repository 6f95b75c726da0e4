"""The learned heads' operators on torch tensors: layer norm forward and backward, the gradients' norm, AdamW with
moments in 32 or 8 bits (the device-buffer part of include/splatx_hip.h).

`TorchBackend` is a `splatx_hip.Backend` whose further methods take tensors of its device and enqueue on torch's current
stream there: they return at once, like torch's own operations, and a tensor in use on another stream than the current one
is the caller's to order, as with those. What they return or use as workspace comes from torch's allocator on that stream.
`layer_norm` is the differentiable form, and `AdamW` keeps a model's moments and steps its parameters.

torch brings a HIP runtime of its own, and one process must run on one: import this module (or torch) before anything
loads the library.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import os
import struct

import torch

import splatx_hip as sh

ADAMW_BLOCK = 256  # elements that share a scale with 8-bit moments


# The C structs, for programs that have device memory without torch's tensors and call the entry points through `TorchBackend.lib`
# themselves (as the tests of the C boundary do); the methods here go through the extension.
class Queue(C.Structure):
    _fields_ = [("stream", C.c_void_p)]


class LayerNormInputs(C.Structure):
    _fields_ = [("x", C.c_void_p), ("residual", C.c_void_p), ("weight", C.c_void_p), ("bias", C.c_void_p),
                ("rows", C.c_int64), ("width", C.c_int64), ("x_stride", C.c_int64), ("residual_stride", C.c_int64),
                ("eps", C.c_float), ("type", C.c_uint8), ("weight_type", C.c_uint8)]


class LayerNormOutputs(C.Structure):
    _fields_ = [("y", C.c_void_p), ("h", C.c_void_p), ("mean", C.c_void_p), ("rstd", C.c_void_p),
                ("y_stride", C.c_int64), ("h_stride", C.c_int64)]


class LayerNormGradsIn(C.Structure):
    _fields_ = [("dy", C.c_void_p), ("h", C.c_void_p), ("dh", C.c_void_p), ("mean", C.c_void_p), ("rstd", C.c_void_p),
                ("weight", C.c_void_p), ("rows", C.c_int64), ("width", C.c_int64), ("dy_stride", C.c_int64),
                ("h_stride", C.c_int64), ("dh_stride", C.c_int64), ("type", C.c_uint8), ("weight_type", C.c_uint8)]


class LayerNormGrads(C.Structure):
    _fields_ = [("dx", C.c_void_p), ("dweight", C.c_void_p), ("dbias", C.c_void_p), ("dx_stride", C.c_int64),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_int64)]


class NormTensor(C.Structure):
    _fields_ = [("grad", C.c_void_p), ("n", C.c_int64), ("type", C.c_uint8)]


class AdamWTensor(C.Structure):
    _fields_ = [("param", C.c_void_p), ("master", C.c_void_p), ("grad", C.c_void_p), ("exp_avg", C.c_void_p),
                ("exp_avg_sq", C.c_void_p), ("exp_avg_scale", C.c_void_p), ("exp_avg_sq_scale", C.c_void_p),
                ("n", C.c_int64), ("lr", C.c_double), ("weight_decay", C.c_double), ("param_type", C.c_uint8),
                ("grad_type", C.c_uint8), ("taken", C.c_void_p)]


class AdamWParams(C.Structure):
    _fields_ = [("step", C.c_int64), ("seed", C.c_uint64), ("b1", C.c_double), ("b2", C.c_double), ("eps", C.c_double),
                ("grad_norm", C.c_void_p), ("max_norm", C.c_float), ("grad_scale", C.c_float), ("state_bits", C.c_int32),
                ("adopt", C.c_int32)]


_NORM_ROW = struct.Struct("<QqB7x")  # a NormTensor as bytes, for a table of many
# (the public way to the current stream's handle makes an object of it, 2 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _extension():
    """host/torch_ops.cpp, which is built beside the library where torch is: the calls' checks, outputs and launches."""
    path = os.path.join(os.path.dirname(sh.LIB_PATH), "_splatx_torch.so")
    if not os.path.exists(path):
        raise sh.SxRuntimeError(f"the torch extension is not built: {path} (make all in splatx-metal_amd, with torch's and Python's headers)")
    loader = importlib.machinery.ExtensionFileLoader("_splatx_torch", path)
    ops = importlib.util.module_from_spec(importlib.util.spec_from_loader("_splatx_torch", loader))
    ops.set_errors(sh.SxInvalidArgument, sh.SxRuntimeError)
    return ops


def _one_hip_runtime():
    """A stream of one HIP runtime means nothing to another one."""
    with open("/proc/self/maps") as f:
        found = {line.split(None, 5)[5].strip() for line in f if "libamdhip64" in line}
    if len(found) > 1:
        raise sh.SxRuntimeError("two HIP runtimes in this process (" + ", ".join(sorted(found)) +
                                "): import splatx_torch or torch before the library is loaded")


def adamw_blocks(n: int) -> int:
    """Scales of a tensor of n elements with 8-bit moments."""
    return -(-n // ADAMW_BLOCK)


class TorchBackend(sh.Backend):
    """A backend with the learned heads' operators on torch tensors of its device."""

    def __init__(self, device_ordinal: int = 0, lib=None):
        torch.cuda.init()
        lib = lib or sh.load_library()
        if not os.path.samefile(lib._name, sh.LIB_PATH):
            raise sh.SxInvalidArgument(f"the operators on tensors are those of {sh.LIB_PATH}")
        _one_hip_runtime()
        super().__init__(device_ordinal, lib)
        self.device = torch.device("cuda", device_ordinal)
        self._index, self._address, self._ops = device_ordinal, self.handle.value, _extension()
        p, n = C.c_void_p, C.c_int64
        for name, args in (("layer_norm_fwd", (p, p, p, p)), ("layer_norm_bwd", (p, p, p, p)), ("grad_norm", (p, p, n, p, p, n, p)),
                           ("adamw", (p, p, n, p, p))):
            f = getattr(self.lib, "sxh_" + name)
            f.argtypes, f.restype = args, C.c_int32
        for name, args in (("layer_norm_bwd_workspace", (n, n)), ("grad_norm_workspace", (n,))):
            f = getattr(self.lib, "sxh_" + name)
            f.argtypes, f.restype = args, n

    def close(self):
        self._address = 0
        super().close()

    # -- layer norm ------------------------------------------------------------------------------------
    def layer_norm_fwd(self, x, weight=None, bias=None, eps=1e-5, residual=None, stats=True):
        """(y, h, mean, rstd): h = x + residual (x itself without one), y = (h - mean) rstd weight + bias over the last
        dimension; mean and rstd, one per row, are None without `stats`."""
        return self._ops.layer_norm_fwd(self._address, self._index, _raw_stream(self._index), x, weight, bias, eps, residual, stats)

    def layer_norm_bwd(self, dy, h, mean, rstd, weight=None, dh=None, want_dx=True, want_dweight=True, want_dbias=True):
        """(dx, dweight, dbias) of layer_norm_fwd's h, mean and rstd; dx is the gradient of x and of the residual, with the
        gradient dh that reaches h past the norm. dweight and dbias have the weight's type (float32 without one)."""
        return self._ops.layer_norm_bwd(self._address, self._index, _raw_stream(self._index), dy, h, mean, rstd, weight, dh, want_dx,
                                        want_dweight, want_dbias)

    # -- many tensors ------------------------------------------------------------------------------------
    def grad_norm(self, grads):
        """The 2-norm of all the tensors together, as a tensor of one float32 on the device."""
        grads = grads if isinstance(grads, (list, tuple)) else list(grads)
        return self._ops.grad_norm(self._address, self._index, _raw_stream(self._index), grads)

    def adamw_step(self, params, grads, exp_avg, exp_avg_sq, *, step, lr, weight_decay=0.0, b1=0.9, b2=0.999, eps=1e-8,
                   master=None, grad_scale=1.0, grad_norm=None, max_norm=0.0, exp_avg_scale=None, exp_avg_sq_scale=None, seed=0,
                   taken=None, adopt=False):
        """One AdamW step of lists of tensors, in place. `lr` and `weight_decay`: a number, or one for each tensor. `master`:
        float32 copies that the step works on, with 16-bit params. With the scales, exp_avg and exp_avg_sq are float8_e4m3fn
        (or uint8) tensors: m, and the root of v, in units of their block's scale. grad_norm: `grad_norm`'s result of these
        gradients; where it is not finite the step is left out. `taken`: int64 tensors of two elements, each the count of its
        tensor's own steps and a word of the call's; the bias is corrected by them in place of `step`, and a step that is not
        left out adds one. `adopt`: an element of a 16-bit param that is not its master's rounding has been set since the last
        step, and is what this one begins from."""
        self._ops.adamw(self._address, self._index, _raw_stream(self._index), params, grads, exp_avg, exp_avg_sq, step, lr,
                        weight_decay, b1, b2, eps, master, grad_scale, grad_norm, max_norm, exp_avg_scale, exp_avg_sq_scale, seed, taken,
                        adopt)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, backend, x, weight, bias, eps, residual):
        y, h, mean, rstd = backend.layer_norm_fwd(x, weight, bias, eps, residual)
        ctx.backend = backend
        ctx.shapes = tuple(None if t is None else t.shape for t in (weight, bias))
        ctx.save_for_backward(h, mean, rstd, weight)
        ctx.set_materialize_grads(False)
        return (y, h) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, mean, rstd, weight = ctx.saved_tensors
        _, need_x, need_w, need_b, _, need_r = ctx.needs_input_grad
        if dy is None:
            return None, dh, None, None, None, dh if need_r else None
        # (a sum's gradient is one value broadcast; a transposed layer's has its rows in other places)
        dy, dh = (t if t is None or t.dim() == 2 and t.stride(1) == 1 else t.contiguous() for t in (dy, dh))
        dx, dweight, dbias = backward_of(ctx.backend, dy, h, mean, rstd, weight, dh, need_x or need_r, need_w, need_b)
        dweight, dbias = (g if g is None else g.view(shape) for g, shape in zip((dweight, dbias), ctx.shapes))
        return None, dx if need_x else None, dweight, dbias, None, dx if need_r else None


def backward_of(backend, dy, h, mean, rstd, weight, dh, want_dx, want_dweight, want_dbias):
    if not (want_dx or want_dweight or want_dbias):
        return None, None, None
    return backend.layer_norm_bwd(dy, h, mean, rstd, weight, dh if want_dx else None, want_dx, want_dweight, want_dbias)


def layer_norm(backend: TorchBackend, x, weight=None, bias=None, eps=1e-5, residual=None):
    """Differentiable layer norm over the last dimension: y, or (y, x + residual) with a residual. weight and bias have as many
    elements as a row, in any shape, and so have their gradients."""
    return _LayerNorm.apply(backend, x, weight, bias, eps, residual)


class AdamW:
    """AdamW over a model's parameters, with moments in 32 bits or in 8 and a float32 master copy of 16-bit parameters (where
    a parameter has been set since its last step, weights loaded for one, the master follows it).

    `params`: tensors, or dicts with "params" and their own "lr" or "weight_decay". A step takes the gradients from the
    parameters (one without a gradient is left as it is) and clips their norm to `max_norm` (0: does not); a step whose
    norm is not finite is left out with `max_norm` or `skip_nonfinite`. `steps` counts the calls; a parameter's bias is
    corrected by the count of its own steps, those without a gradient and those left out not among them. It does not wait
    for the device."""

    def __init__(self, backend: TorchBackend, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32,
                 max_norm=0.0, skip_nonfinite=False, seed=0):
        if state_bits not in (8, 32):
            raise sh.SxInvalidArgument("state_bits must be 32 or 8")
        self.backend, self.betas, self.eps, self.state_bits = backend, betas, eps, state_bits
        self.max_norm, self.skip_nonfinite, self.seed, self.steps = max_norm, skip_nonfinite, seed, 0
        params = list(params)
        groups = params if params and isinstance(params[0], dict) else [dict(params=params)]
        self.params, self.lr, self.weight_decay = [], [], []
        for g in groups:
            for p in g["params"]:
                self.params.append(p)
                self.lr.append(g.get("lr", lr))
                self.weight_decay.append(g.get("weight_decay", weight_decay))
        self.state = [self._fresh(p) for p in self.params]

    def _fresh(self, p):
        d = p.detach()
        if self.state_bits == 32:
            s = dict(exp_avg=torch.zeros_like(d, dtype=torch.float32), exp_avg_sq=torch.zeros_like(d, dtype=torch.float32))
        else:
            s = {k: torch.zeros(d.shape, dtype=torch.uint8, device=d.device).view(torch.float8_e4m3fn)
                 for k in ("exp_avg", "exp_avg_sq")}
            for k in ("exp_avg_scale", "exp_avg_sq_scale"):
                s[k] = torch.zeros(adamw_blocks(d.numel()), dtype=torch.float32, device=d.device)
        if d.dtype != torch.float32:
            s["master"] = d.float()
        s["taken"] = torch.zeros(2, dtype=torch.int64, device=d.device)
        return s

    def moments(self, i):
        """(m, v) of parameter i as float32 tensors."""
        s = self.state[i]
        if self.state_bits == 32:
            return s["exp_avg"], s["exp_avg_sq"]
        m, root = (self._values(s[k], s[k + "_scale"]) for k in ("exp_avg", "exp_avg_sq"))
        return m, root * root

    @staticmethod
    def _values(codes, scale):
        return (codes.float().view(-1) * scale.repeat_interleave(ADAMW_BLOCK)[:codes.numel()]).view(codes.shape)

    def step(self, grad_scale=1.0):
        """One step with the gradients times `grad_scale`. Returns their norm before it, if it was formed (a device tensor)."""
        self.steps += 1
        at = [i for i, p in enumerate(self.params) if p.grad is not None]
        grads = [self.params[i].grad for i in at]
        norm = self.backend.grad_norm(grads) if self.max_norm > 0 or self.skip_nonfinite else None
        b = self.betas
        # float32 parameters and 16-bit ones with their masters are two calls
        for half in (False, True):
            k = [j for j, i in enumerate(at) if ("master" in self.state[i]) == half]
            if not k:
                continue
            st = [self.state[at[j]] for j in k]
            more = dict(taken=[s["taken"] for s in st])
            if half:
                more.update(master=[s["master"] for s in st], adopt=True)
            if self.state_bits == 8:
                more.update(exp_avg_scale=[s["exp_avg_scale"] for s in st], exp_avg_sq_scale=[s["exp_avg_sq_scale"] for s in st],
                            seed=(self.seed * 2 + half) & (2 ** 64 - 1))
            with torch.no_grad():
                self.backend.adamw_step([self.params[at[j]] for j in k], [grads[j] for j in k], [s["exp_avg"] for s in st],
                                        [s["exp_avg_sq"] for s in st], step=self.steps, lr=[self.lr[at[j]] for j in k],
                                        weight_decay=[self.weight_decay[at[j]] for j in k], b1=b[0], b2=b[1], eps=self.eps,
                                        grad_scale=grad_scale, grad_norm=norm, max_norm=self.max_norm, **more)
        return norm

    def zero_grad(self):
        for p in self.params:
            p.grad = None

    def state_dict(self):
        return dict(steps=self.steps, seed=self.seed, state_bits=self.state_bits,
                    state=[{k: v.clone() for k, v in s.items()} for s in self.state])

    def load_state_dict(self, d):
        if d["state_bits"] != self.state_bits or len(d["state"]) != len(self.state):
            raise sh.SxInvalidArgument("the state is of another form or of other parameters")
        # (a state of before parameters had counts of their own: all took every step)
        state = [{"taken": torch.tensor([d["steps"], 0]), **t} for t in d["state"]]
        for s, t in zip(self.state, state):
            # (a copy would convert: codes as whole numbers are other values than the codes)
            if s.keys() != t.keys() or any(s[k].shape != t[k].shape or s[k].dtype != t[k].dtype for k in s):
                raise sh.SxInvalidArgument("the state is of other parameters")
        for s, t in zip(self.state, state):
            for k in s:
                s[k].copy_(t[k])
        self.steps, self.seed = d["steps"], d["seed"]
