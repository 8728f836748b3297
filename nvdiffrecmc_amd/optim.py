"""Adam + gradient scale + parameter clamps of one iteration in ONE kernel launch (csrc/optim.hip), and the global norm of many gradient
tensors with clipping by it (csrc/gradnorm.hip): on its own (grad_norm, clip_grad_norm_) or as part of the update (FusedAdam(max_norm=...)).

Same update as torch.optim.Adam(params, lr, betas, eps) without weight decay / amsgrad (the optimizer of the reference,
train.py:452-461), followed by the clamps the reference applies to its parameters after the step (train.py:470-476); the
multiplication of the light gradient by 64 (train.py:439-440) enters as a per-tensor gradient scale.  The step counter lives in
device memory, so the launch can be captured in a HIP graph.
"""
import array
import math
import struct

import torch

from . import _lib

_NORM_TYPES = {math.inf: 0, 1.0: 1, 2.0: 2}                                 # NVDR_NORM_INF / 1 / 2


def _norm_code(norm_type):
    code = _NORM_TYPES.get(float(norm_type))
    if code is None:
        raise ValueError('norm_type must be 1, 2 or inf (got %s)' % norm_type)
    return code


def _max_norm(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError('max_norm must be zero or more (got %s)' % max_norm)
    return max_norm


def _norm(tensors, scales, code, max_norm, out, work, what):
    """gradops.norm, with contiguous copies in the place of tensors whose elements do not fill their memory exactly once (a slice, an expanded
    tensor)."""
    try:
        r = _lib.gradops().norm(tensors, scales, code, max_norm, out, work)
        if isinstance(r, list):
            for i in r:
                tensors[i] = tensors[i].detach().clone(memory_format=torch.contiguous_format)
            r = _lib.gradops().norm(tensors, scales, code, max_norm, out, work)
        return r
    except (TypeError, ValueError) as e:
        raise type(e)('%s: %s' % (what, e)) from None


def grad_norm(tensors, norm_type=2.0, scales=None):
    """The norm of all `tensors` seen as one vector: (sum |scales[k] * g|^p)^(1/p) for norm_type p = 1 or 2, the largest magnitude for
    math.inf; a NaN anywhere gives a NaN.  tensors: a tensor or an iterable of tensors, fp32 / bf16 / fp16 in any mixture and any layout,
    on one GPU.  Returns a 0-d fp32 tensor on that GPU (0 on the CPU for an empty list); nothing waits for it, and no gradient flows through it.
    Sums are kept in fp64."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    code = _norm_code(norm_type)
    if scales is not None:
        scales = array.array('f', scales).tobytes()
        if len(scales) != 4 * len(tensors):
            raise ValueError('grad_norm: %d scales for %d tensors' % (len(scales) // 4, len(tensors)))
    norm = _norm(tensors, scales, code, math.inf, None, None, 'grad_norm')
    return torch.zeros(()) if norm is None else norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scales the gradients of `parameters` in place by min(1, max_norm / (norm + 1e-6)) and returns their norm BEFORE that (0-d fp32 on
    the GPU): torch.nn.utils.clip_grad_norm_ with the norm kept in fp64 and two launches for up to 160 tensors (neighbours in memory, like
    the views of a gradient bucket, count as one).  parameters: a tensor or an iterable; those without a gradient are left out.  A norm
    that is infinite or NaN makes the gradients zero or NaN as it does there, unless error_if_nonfinite is set, which waits for the norm
    and raises before anything is scaled (not inside a graph capture).  max_norm = inf only measures.  Gradients that share memory -- the same
    tensor twice, overlapping views, an expanded tensor -- are refused, and views whose strides take more than
    2^14 steps to tell apart; views that interleave, like columns of a matrix, are not."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    code, max_norm = _norm_code(norm_type), _max_norm(max_norm)
    if error_if_nonfinite:
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError('clip_grad_norm_: error_if_nonfinite reads the norm on the host, which a graph capture does not allow')
        norm = grad_norm([p.grad for p in parameters if p.grad is not None], norm_type).item()
        if not math.isfinite(norm):
            raise RuntimeError('clip_grad_norm_: the norm of the gradients is %s' % norm)
    try:
        norm = _lib.gradops().clip(parameters, True, code, max_norm)
        if not isinstance(norm, list):
            return torch.zeros((), device=parameters[0].device if parameters else None) if norm is None else norm
        # gradients whose elements do not lie side by side: through contiguous copies
        grads = [p.grad for p in parameters if p.grad is not None]
        originals = [grads[i] for i in norm]
        for i in norm:
            grads[i] = grads[i].detach().clone(memory_format=torch.contiguous_format)
        copies = [grads[i] for i in norm]
        norm = _lib.gradops().clip(grads, False, code, max_norm)
        with torch.no_grad():
            for g, copy in zip(originals, copies):
                g.copy_(copy)
        return norm
    except (TypeError, ValueError) as e:
        raise type(e)('clip_grad_norm_: %s' % e) from None


# nvdr_adam_tensor (_lib.NvdrAdamTensor): filling its fields one by one costs 2 us a tensor.  Native mode: a bound or scale beyond fp32 becomes
# infinite as in the structure (in the standard modes struct raises)
_ADAM_ROW = struct.Struct('@QQQQqfff4xQqQqfiQii').pack
_UNBOUNDED = (-math.inf, math.inf, 0, 0, 0, 0)
_LEAST_RATE = 2.0 ** -149                                                    # fp32's smallest number


def _check_bounds(clamps, device):
    """Per-channel bounds are read by the kernel where they lie."""
    for i, c in enumerate(clamps):
        for v in (c[2:4] if c is not None else ()):
            if v is not None and (v.dtype != torch.float32 or v.device != device or not v.is_contiguous() or v.numel() == 0):
                raise ValueError('FusedAdam: the per-channel bounds of parameter %d must be contiguous fp32 tensors on its GPU' % i)


class FusedAdam:
    """params: list of tensors (requires_grad, contiguous fp32, on one GPU).
    clamps[i]: None or (lo, hi[, lo_vec[, hi_vec]]) with lo / hi floats or None and lo_vec / hi_vec optional per-channel bounds
    (fp32 tensors on the same GPU: element e is bounded by lo_vec[e % len(lo_vec)] / hi_vec[e % len(hi_vec)]; Texture2D.clamp_).
    grad_scales[i]: factor applied to the gradient of parameter i inside the update (p.grad itself is left alone).
    lr_scales[i]: learning rate of parameter i relative to lr (the reference runs three Adams with position / material / light
    rates, train.py:336-356).  normalize3[i]: renormalise every texel of three channels after the clamps (the normal map).
    sparse[i]: the tensor is a three-channel texture whose gradient is zero almost everywhere (a nearest-texel lookup): tiles of 64
    texels without gradient and without history are skipped -- same parameters, a fraction of the traffic (csrc/optim.hip).
    zero_grad[i] (with sparse): p.grad is zeroed behind the update (a persistent scatter-add buffer then needs no memset).
    max_norm: the update sees its gradients -- with grad_scales and grad_mult -- scaled by min(1, max_norm / (norm + 1e-6)), norm =
    the norm (norm_type 2, 1 or math.inf) of all tensors that are not frozen: clip_grad_norm_ in front of the step, without its pass over
    the gradients, which stay as they are.  .grad_norm holds the norm of the last step (0-d, device; the next step overwrites it)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, clamps=None, grad_scales=None, lr_scales=None, normalize3=None,
                 sparse=None, zero_grad=None, max_norm=None, norm_type=2.0):
        self.params = list(params)
        if not 1 <= len(self.params) <= 8:
            raise ValueError('FusedAdam: 1..8 parameter tensors')
        for p in self.params:
            if p.dtype != torch.float32 or not p.is_contiguous() or not p.is_cuda or p.device != self.params[0].device:
                raise ValueError('FusedAdam: parameters must be contiguous fp32 tensors on the GPU, all on the same one')
        self.lr, self.betas, self.eps = float(lr), (float(betas[0]), float(betas[1])), float(eps)
        self.clamps = list(clamps) if clamps is not None else [None] * len(self.params)
        _check_bounds(self.clamps, self.params[0].device)
        self.grad_scales = list(grad_scales) if grad_scales is not None else [1.0] * len(self.params)
        self.lr_scales = list(lr_scales) if lr_scales is not None else [1.0] * len(self.params)
        self.normalize3 = list(normalize3) if normalize3 is not None else [False] * len(self.params)
        self.sparse = list(sparse) if sparse is not None else [False] * len(self.params)
        self.zero_grad_after = list(zero_grad) if zero_grad is not None else [False] * len(self.params)
        self.active = [torch.zeros((p.numel() // 3 + 63) // 64, dtype=torch.uint8, device=p.device) if sp else None for p, sp in zip(self.params, self.sparse)]
        self.exp_avg = [torch.zeros_like(p) for p in self.params]
        self.exp_avg_sq = [torch.zeros_like(p) for p in self.params]
        self.max_norm, self._norm_code = (None if max_norm is None else _max_norm(max_norm)), _norm_code(norm_type)
        self._measured = False
        dev = self.params[0].device
        self._norm_out = torch.zeros(2, dtype=torch.float32, device=dev)        # norm, factor
        self._norm_view = self._norm_out[0]
        # what the step begins with, and the parts of the norm: enough for any part of the tensors
        n, types = array.array('q', [p.numel() for p in self.params]).tobytes(), bytes(len(self.params))
        self._norm_work = torch.empty(2 + _lib.load().nvdr_grad_norm_workspace(n, types, len(types), 0), dtype=torch.float64, device=dev)
        self.state = torch.zeros(8, dtype=torch.int32, device=self.params[0].device)     # steps taken, scratch, beta1^t, beta2^t (doubles)

    @property
    def step_count(self):
        return int(self.state[0].item())

    @property
    def grad_norm(self):
        """Norm of the gradients of the last step before clipping (0 before the first one; None without max_norm)."""
        return None if self.max_norm is None else self._norm_view

    def measure_norm(self, grad_mult=1.0):
        """The norm of this iteration's gradients into .grad_norm, and the factor of the updates that follow (max_norm).  step() of all tensors
        does it itself; a caller that updates in subsets calls it once, when every gradient of the iteration is there, in front of the
        first subset."""
        if self.max_norm is None:
            raise RuntimeError('FusedAdam.measure_norm: no max_norm was given')
        live = [i for i in range(len(self.params)) if float(self.lr_scales[i]) != 0.0]
        for i in live:
            if self.params[i].grad is None:
                raise RuntimeError('FusedAdam.step: parameter %d has no gradient' % i)
        scales = array.array('f', [float(self.grad_scales[i]) * float(grad_mult) for i in live]).tobytes()
        _norm([self.params[i].grad for i in live], scales, self._norm_code, self.max_norm, self._norm_out, self._norm_work[2:], 'FusedAdam')
        self._measured = True

    def zero_grad(self, set_to_none=True):
        for p in self.params:
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.zero_()

    def step(self, subset=None, advance=True, grad_mult=1.0):
        """subset: indices of the tensors to update in this launch (None = all); advance=False leaves the step counter alone (every
        launch of an iteration but the last, nvdr_adam_step_partial); grad_mult: extra factor on the gradients of this launch (1 / world
        after a summing all-reduce).  With max_norm a launch of all tensors measures the norm first; subsets need measure_norm() before the
        first of them."""
        if torch.cuda.current_device() != self.state.get_device():          # (launches go to the current device)
            with torch.cuda.device(self.state.device):
                return self.step(subset, advance, grad_mult)
        rows, keep, grad_mult = [], [], float(grad_mult)
        for i in (range(len(self.params)) if subset is None else subset):
            p = self.params[i]
            g = p.grad
            if g is None:
                raise RuntimeError('FusedAdam.step: parameter %d has no gradient' % i)
            if g.dtype is not torch.float32:
                raise RuntimeError('FusedAdam.step: the gradient of parameter %d must be float32 (got %s)' % (i, g.dtype))
            if not g.is_contiguous():
                if self.zero_grad_after[i]:
                    # a copy would be zeroed instead of the buffer the producer scatter-adds into
                    raise RuntimeError('FusedAdam.step: zero_grad needs a contiguous .grad for parameter %d (the persistent scatter-add buffer itself)' % i)
                g = g.contiguous()
            keep.append(g)                          # (the call runs without the interpreter's lock: another thread may drop p.grad meanwhile)
            bounds, c = _UNBOUNDED, self.clamps[i]
            if c is not None:
                lo_vec = c[2] if len(c) > 2 else None
                hi_vec = c[3] if len(c) > 3 else None
                bounds = (-math.inf if c[0] is None else c[0], math.inf if c[1] is None else c[1],
                          lo_vec.data_ptr() if lo_vec is not None else 0, lo_vec.numel() if lo_vec is not None else 0,
                          hi_vec.data_ptr() if hi_vec is not None else 0, hi_vec.numel() if hi_vec is not None else 0)
            # lr_scales[i] == 0 freezes the tensor (the C block's lr_scale 0 means "the plain rate": a zero-initialised block trains, and a rate
            # below fp32's range must not become one)
            rate, active = float(self.lr_scales[i]), self.active[i]
            if 0.0 < rate < _LEAST_RATE:
                rate = _LEAST_RATE
            rows.append(_ADAM_ROW(p.data_ptr(), g.data_ptr(), self.exp_avg[i].data_ptr(), self.exp_avg_sq[i].data_ptr(), p.numel(),
                                  self.grad_scales[i] * grad_mult, *bounds, rate or 1.0, bool(self.normalize3[i]),
                                  active.data_ptr() if active is not None else 0, bool(self.zero_grad_after[i]) and active is not None, rate == 0.0))
        tab, lib, state = b''.join(rows), _lib.load(), self.state.data_ptr()
        hyper = (self.lr, self.betas[0], self.betas[1], self.eps)
        if self.max_norm is not None and subset is None and advance:
            _lib.check(lib.nvdr_adam_step_clipped(tab, len(rows), *hyper, state, self._norm_code, self.max_norm, self._norm_work.data_ptr(),
                                                  self._norm_work.numel(), self._norm_out.data_ptr(), _lib.stream_ptr()), 'adam_step')
            self._measured = False
            return
        factor = None
        if self.max_norm is not None:
            if subset is None:
                self.measure_norm(grad_mult)
            elif not self._measured:
                raise RuntimeError('FusedAdam.step: with max_norm, measure_norm() comes before the first subset of an iteration')
            factor = self._norm_out.data_ptr() + 4
        _lib.check(lib.nvdr_adam_step_factor(tab, len(rows), *hyper, state, bool(advance), factor, _lib.stream_ptr()), 'adam_step')
        self._measured = self._measured and not advance
