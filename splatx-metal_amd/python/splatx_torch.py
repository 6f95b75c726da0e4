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
import struct

import torch

import splatx_hip as sh

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # SXH_TYPE_*
ADAMW_BLOCK = 256  # elements that share a scale with 8-bit moments
_CODE_TYPES = (torch.float8_e4m3fn, torch.uint8)


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
                ("grad_type", C.c_uint8)]


class AdamWParams(C.Structure):
    _fields_ = [("step", C.c_int64), ("seed", C.c_uint64), ("b1", C.c_double), ("b2", C.c_double), ("eps", C.c_double),
                ("grad_norm", C.c_void_p), ("max_norm", C.c_float), ("grad_scale", C.c_float), ("state_bits", C.c_int32)]


# the two tables' rows as bytes: a step of many tensors fills them each time
_NORM_ROW = struct.Struct("<QqB7x")
_ADAMW_ROW = struct.Struct("<7QqddBB6x")
assert _NORM_ROW.size == C.sizeof(NormTensor) and _ADAMW_ROW.size == C.sizeof(AdamWTensor)

_is_contiguous = torch.Tensor.is_contiguous
_numel = torch.Tensor.numel
_ptr = torch.Tensor.data_ptr


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
        super().__init__(device_ordinal, lib)
        _one_hip_runtime()
        self.device = torch.device("cuda", device_ordinal)
        for name, args in (("layer_norm_fwd", 4), ("layer_norm_bwd", 4)):
            getattr(self.lib, "sxh_" + name).argtypes = [C.c_void_p] * args
        self.lib.sxh_grad_norm.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
        self.lib.sxh_adamw.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p]
        for name, args in (("layer_norm_bwd_workspace", 2), ("grad_norm_workspace", 1)):
            f = getattr(self.lib, "sxh_" + name)
            f.argtypes, f.restype = [C.c_int64] * args, C.c_int64

    def _queue(self):
        return C.byref(Queue(torch.cuda.current_stream(self.device).cuda_stream))

    def _rows(self, t, name, like=None):
        """(tensor as [rows, width], its row stride)"""
        if not isinstance(t, torch.Tensor) or t.device != self.device:
            raise sh.SxInvalidArgument(f"{name} must be a tensor on {self.device}")
        if t.dtype not in TYPES:
            raise sh.SxInvalidArgument(f"{name} must be float32, bfloat16 or float16")
        if like is not None and (t.dtype != like.dtype or t.shape != like.shape):
            raise sh.SxInvalidArgument(f"{name} must have the rows' type and shape")
        if t.dim() != 2:
            if t.dim() == 0:
                raise sh.SxInvalidArgument(f"{name} has no rows")
            try:
                t = t.view(t.shape[:-1].numel(), t.shape[-1])
            except RuntimeError:
                raise sh.SxInvalidArgument(f"{name}: rows of {tuple(t.shape)} with strides {t.stride()} are not evenly spaced") from None
        rows, width = t.shape
        stride = t.stride()
        if width > 1 and stride[1] != 1:
            raise sh.SxInvalidArgument(f"{name}: the elements of a row must lie side by side")
        return t, stride[0] if rows > 1 else width

    def _vector(self, t, name, n, types):
        if not isinstance(t, torch.Tensor) or t.device != self.device:
            raise sh.SxInvalidArgument(f"{name} must be a tensor on {self.device}")
        if t.dtype not in types or t.numel() != n or not t.is_contiguous():
            raise sh.SxInvalidArgument(f"{name} must be {n} contiguous elements of {' or '.join(map(str, types))}")
        return t.data_ptr()

    # -- layer norm ------------------------------------------------------------------------------------
    def layer_norm_fwd(self, x, weight=None, bias=None, eps=1e-5, residual=None, stats=True):
        """(y, h, mean, rstd): h = x + residual (x itself without one), y = (h - mean) rstd weight + bias over the last
        dimension; mean and rstd, one per row, are None without `stats`."""
        x2, x_stride = self._rows(x, "x")
        rows, width = x2.shape
        types = (torch.float32, x.dtype)
        wt = weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32
        w = self._vector(weight, "weight", width, types) if weight is not None else None
        b = self._vector(bias, "bias", width, (wt,)) if bias is not None else None
        y = torch.empty(x.shape, dtype=x.dtype, device=self.device)
        h, r2, r_stride = None, None, 0
        if residual is not None:
            r2, r_stride = self._rows(residual, "residual", x)
            h = torch.empty_like(y)
        mean = rstd = None
        if stats:
            mean, rstd = (torch.empty(x.shape[:-1], dtype=torch.float32, device=self.device) for _ in range(2))
        self._call("layer_norm_fwd",
                   C.byref(LayerNormInputs(x2.data_ptr(), r2.data_ptr() if r2 is not None else None, w, b, rows, width, x_stride,
                                           r_stride, eps, TYPES[x.dtype], TYPES[wt])),
                   C.byref(LayerNormOutputs(y.data_ptr(), h.data_ptr() if h is not None else None,
                                            mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None, width, width)),
                   self._queue())
        return y, x if h is None else h, mean, rstd

    def layer_norm_bwd(self, dy, h, mean, rstd, weight=None, dh=None, want_dx=True, want_dweight=True, want_dbias=True):
        """(dx, dweight, dbias) of layer_norm_fwd's h, mean and rstd; dx is the gradient of x and of the residual, with the
        gradient dh that reaches h past the norm. dweight and dbias have the weight's type (float32 without one)."""
        h2, h_stride = self._rows(h, "h")
        dy2, dy_stride = self._rows(dy, "dy", h)
        rows, width = h2.shape
        w = self._vector(weight, "weight", width, (torch.float32, h.dtype)) if weight is not None else None
        wt = weight.dtype if weight is not None else torch.float32
        dh2, dh_stride = self._rows(dh, "dh", h) if dh is not None else (None, 0)
        m = self._vector(mean, "mean", rows, (torch.float32,))
        s = self._vector(rstd, "rstd", rows, (torch.float32,))
        dx = torch.empty(h.shape, dtype=h.dtype, device=self.device) if want_dx else None
        dweight = torch.empty(width, dtype=wt, device=self.device) if want_dweight else None
        dbias = torch.empty(width, dtype=wt, device=self.device) if want_dbias else None
        work, bytes_ = None, 0
        if want_dweight or want_dbias:
            bytes_ = self.lib.sxh_layer_norm_bwd_workspace(rows, width)
            work = torch.empty(bytes_, dtype=torch.uint8, device=self.device)
        self._call("layer_norm_bwd",
                   C.byref(LayerNormGradsIn(dy2.data_ptr(), h2.data_ptr(), dh2.data_ptr() if dh is not None else None, m, s, w,
                                            rows, width, dy_stride, h_stride, dh_stride, TYPES[h.dtype], TYPES[wt])),
                   C.byref(LayerNormGrads(dx.data_ptr() if want_dx else None, dweight.data_ptr() if want_dweight else None,
                                          dbias.data_ptr() if want_dbias else None, width,
                                          work.data_ptr() if work is not None else None, bytes_)),
                   self._queue())
        return dx, dweight, dbias

    # -- many tensors ------------------------------------------------------------------------------------
    def _tensors(self, ts, name, types):
        """Pointers of a list of contiguous tensors of the device."""
        for t in ts:
            if not isinstance(t, torch.Tensor) or t.device != self.device:
                raise sh.SxInvalidArgument(f"{name} must be tensors on {self.device}")
            if t.dtype not in types:
                raise sh.SxInvalidArgument(f"{name} must be {' or '.join(map(str, types))}, not {t.dtype}")
        if not all(map(_is_contiguous, ts)):
            raise sh.SxInvalidArgument(f"{name} must be contiguous")
        return list(map(_ptr, ts))

    def grad_norm(self, grads):
        """The 2-norm of all the tensors together, as a tensor of one float32 on the device."""
        grads = list(grads)
        ptrs = self._tensors(grads, "grads", tuple(TYPES))
        norm = torch.empty((), dtype=torch.float32, device=self.device)
        bytes_ = self.lib.sxh_grad_norm_workspace(len(grads))
        work = torch.empty(bytes_, dtype=torch.uint8, device=self.device)
        table = b"".join(_NORM_ROW.pack(p, t.numel(), TYPES[t.dtype]) for p, t in zip(ptrs, grads))
        self._call("grad_norm", table, len(grads), norm.data_ptr(), work.data_ptr(), bytes_, self._queue())
        return norm

    def adamw_step(self, params, grads, exp_avg, exp_avg_sq, *, step, lr, weight_decay=0.0, b1=0.9, b2=0.999, eps=1e-8,
                   master=None, grad_scale=1.0, grad_norm=None, max_norm=0.0, exp_avg_scale=None, exp_avg_sq_scale=None, seed=0):
        """One AdamW step of lists of tensors, in place. `lr` and `weight_decay`: a number, or one for each tensor. `master`:
        float32 copies that the step works on, with 16-bit params. With the scales, exp_avg and exp_avg_sq are float8_e4m3fn
        (or uint8) tensors: m, and the root of v, in units of their block's scale. grad_norm: `grad_norm`'s result of these
        gradients; where it is not finite the step is left out."""
        params, grads = list(params), list(grads)
        n = len(params)
        eight = exp_avg_scale is not None
        if eight != (exp_avg_sq_scale is not None):
            raise sh.SxInvalidArgument("exp_avg_scale and exp_avg_sq_scale are given together")
        lists = [params, params if master is None else list(master), grads, list(exp_avg), list(exp_avg_sq)]
        states = _CODE_TYPES if eight else (torch.float32,)
        named = [("params", tuple(TYPES)), ("master", (torch.float32,) if master is not None else tuple(TYPES)),
                 ("grads", tuple(TYPES)), ("exp_avg", states), ("exp_avg_sq", states)]
        if eight:
            lists += [list(exp_avg_scale), list(exp_avg_sq_scale)]
            named += [("exp_avg_scale", (torch.float32,)), ("exp_avg_sq_scale", (torch.float32,))]
        for ts, (name, _) in zip(lists, named):
            if len(ts) != n:
                raise sh.SxInvalidArgument(f"{name}: {len(ts)} tensors for {n} params")
        sizes = list(map(_numel, params))
        for ts, (name, _) in zip(lists[1:5], named[1:5]):
            if list(map(_numel, ts)) != sizes:
                raise sh.SxInvalidArgument(f"{name} must have the params' sizes")
        if eight:
            blocks = list(map(adamw_blocks, sizes))
            for ts, (name, _) in zip(lists[5:], named[5:]):
                if list(map(_numel, ts)) != blocks:
                    raise sh.SxInvalidArgument(f"{name} must have a scale for each {ADAMW_BLOCK} elements of a param")
        ptrs = [self._tensors(ts, name, types) for ts, (name, types) in zip(lists, named)]
        if master is None:
            ptrs[1] = [0] * n
        if not eight:
            ptrs += [[0] * n, [0] * n]
        lrs = lr if isinstance(lr, (list, tuple)) else [lr] * n
        decays = weight_decay if isinstance(weight_decay, (list, tuple)) else [weight_decay] * n
        if len(lrs) != n or len(decays) != n:
            raise sh.SxInvalidArgument("lr and weight_decay are a number, or one for each tensor")
        norm = self._vector(grad_norm, "grad_norm", 1, (torch.float32,)) if grad_norm is not None else None
        table = b"".join(map(_ADAMW_ROW.pack, *ptrs, sizes, lrs, decays, [TYPES[p.dtype] for p in params],
                             [TYPES[g.dtype] for g in grads]))
        self._call("adamw", table, n,
                   C.byref(AdamWParams(step, seed, b1, b2, eps, norm, max_norm, grad_scale, 8 if eight else 32)), self._queue())


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, backend, x, weight, bias, eps, residual):
        y, h, mean, rstd = backend.layer_norm_fwd(x, weight, bias, eps, residual)
        ctx.backend, ctx.has_bias, ctx.has_residual = backend, bias is not None, residual is not None
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
        return None, dx if need_x else None, dweight, dbias, None, dx if need_r else None


def backward_of(backend, dy, h, mean, rstd, weight, dh, want_dx, want_dweight, want_dbias):
    if not (want_dx or want_dweight or want_dbias):
        return None, None, None
    return backend.layer_norm_bwd(dy, h, mean, rstd, weight, dh if want_dx else None, want_dx, want_dweight, want_dbias)


def layer_norm(backend: TorchBackend, x, weight=None, bias=None, eps=1e-5, residual=None):
    """Differentiable layer norm over the last dimension: y, or (y, x + residual) with a residual."""
    return _LayerNorm.apply(backend, x, weight, bias, eps, residual)


class AdamW:
    """AdamW over a model's parameters, with moments in 32 bits or in 8 and a float32 master copy of 16-bit parameters.

    `params`: tensors, or dicts with "params" and their own "lr" or "weight_decay". A step takes the gradients from the
    parameters (one without a gradient is left as it is) and clips their norm to `max_norm` (0: does not); a step whose
    norm is not finite is left out with `max_norm` or `skip_nonfinite`. It does not wait for the device."""

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
            more = {}
            if half:
                more["master"] = [s["master"] for s in st]
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
        for s, t in zip(self.state, d["state"]):
            if s.keys() != t.keys() or any(s[k].shape != t[k].shape for k in s):
                raise sh.SxInvalidArgument("the state is of other parameters")
        for s, t in zip(self.state, d["state"]):
            for k in s:
                s[k].copy_(t[k])
        self.steps, self.seed = d["steps"], d["seed"]
