"""AdamW over all tensors of a model at once, with moments in 32 bits or in 8.

``multi_tensor_adamw`` is one step on lists of tensors: on CUDA one kernel launch per 360 tensors
(``csrc/adamw_multi.cu``), elsewhere plain PyTorch, which is also what the kernel tests compare with.
``FusedAdamW`` is the optimizer around it for training loops that do not go through the native engine
(which has its own AdamW on flat storage, ``runtime/engine.py``).

8-bit moments: a tensor's values in row order, in blocks of 256, as ``float8_e4m3fn`` numbers and one fp32
factor per block, the smallest power of two with which the block's largest value fits (448), and at least
2^-126.  The first moment is held itself, the second as its square root, which never becomes zero by rounding.
``quantize_moment`` and ``dequantize_moment`` convert.
"""
from __future__ import annotations

import math
import os

import torch

from . import native

STATE_BLOCK = 256       # values per factor of an 8-bit moment


def state_blocks(n: int) -> int:
    """Blocks, and so factors, of an 8-bit moment of ``n`` values."""
    return -(-n // STATE_BLOCK)


def quantize_moment(x, second: bool = False):
    """fp32 tensor -> (e4m3 numbers of its shape, factors of its blocks).  ``second``: ``x`` is a second
    moment, its square root is what is held."""
    flat = x.detach().float().reshape(-1)
    if second:
        flat = flat.sqrt()
    n = flat.numel()
    blocks = torch.nn.functional.pad(flat, (0, state_blocks(n) * STATE_BLOCK - n)).view(-1, STATE_BLOCK)
    top = blocks.abs().amax(1, keepdim=True).clamp(min=2.0 ** -126)
    mantissa, exponent = torch.frexp(top)       # top = mantissa * 2^exponent, mantissa in [1/2, 1)
    exponent = torch.where(mantissa > 448 / 512, exponent - 8, exponent - 9).clamp(min=-126)
    codes = torch.ldexp(blocks, -exponent).to(torch.float8_e4m3fn)
    if second:
        least = (blocks > 0) & (codes.float() == 0)
        codes = torch.where(least, torch.full_like(blocks, 2.0 ** -9), codes.float()).to(torch.float8_e4m3fn)
    scale = torch.ldexp(torch.ones_like(top), exponent)
    return codes.view(-1)[:n].view(x.shape), scale.view(-1)


def dequantize_moment(codes, scale, second: bool = False):
    """The fp32 values that :func:`quantize_moment`'s results stand for."""
    flat = codes.float().reshape(-1)
    x = flat * scale.repeat_interleave(STATE_BLOCK)[:flat.numel()]
    return (x * x if second else x).view(codes.shape)


def _per_tensor(value, n, name):
    if isinstance(value, (list, tuple)):
        if len(value) != n:
            raise ValueError(f"{name}: {n} values required, not {len(value)}")
        return [float(v) for v in value]
    return [float(value)] * n


@torch.no_grad()
def multi_tensor_adamw(params, grads, exp_avgs, exp_avg_sqs, *, lr, betas=(0.9, 0.999), eps=1e-8,
                       weight_decay=0.01, step, masters=None, exp_avg_scales=None, exp_avg_sq_scales=None,
                       grad_scale=None):
    """One AdamW step on every tensor of ``params``, in place::

        g = grad * grad_scale;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        w -= lr * ((m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps) + weight_decay * w)

    All lists have one entry per parameter: contiguous tensors of the parameter's length on one device,
    parameters and gradients of one type (bf16, fp16 or fp32).  ``masters``, for 16-bit parameters: fp32
    weights that are updated and rounded to the parameters (without them the parameters themselves are).
    ``exp_avgs`` and ``exp_avg_sqs`` are fp32, or with ``exp_avg_scales`` and ``exp_avg_sq_scales`` 8-bit
    moments as :func:`quantize_moment` makes them.  ``lr`` and ``weight_decay``: a number, or one per tensor.
    ``step`` counts from 1; a one-element int64 CUDA tensor is read by the kernel, so that a captured step
    goes on counting.  ``grad_scale``: one fp32 value on the device.  Gradients must be finite (a NaN stays in
    its place).  On the GPU a second moment below 2^-126 counts as zero in 8 bits, and ``eps`` must be at least
    2^-63 / sqrt(1 - b2) with them (3.4e-18 for 0.999); with 32 bits it may be 0.  Autograd notices there that
    parameters and masters have changed, not that moments have."""
    params, grads = list(params), list(grads)
    n = len(params)
    lrs, decays = _per_tensor(lr, n, "lr"), _per_tensor(weight_decay, n, "weight_decay")
    masters = list(masters) if masters is not None else []
    exp_avgs, exp_avg_sqs = list(exp_avgs), list(exp_avg_sqs)
    if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
        raise ValueError("8-bit moments need the factors of both")
    m_scales = list(exp_avg_scales) if exp_avg_scales is not None else []
    v_scales = list(exp_avg_sq_scales) if exp_avg_sq_scales is not None else []
    if n == 0:
        return
    if params[0].is_cuda and native_adamw():
        on_device = torch.is_tensor(step)
        args = (params, grads, masters, exp_avgs, exp_avg_sqs, m_scales, v_scales, lrs, decays, betas[0],
                betas[1], eps, 0 if on_device else step, step if on_device else None, grad_scale)
        if not native.direct("multi_adamw")(*args):      # (something that the dispatcher has to see)
            native.ops().multi_adamw(*args)
        return
    for name, got in (("gradients", grads), ("first moments", exp_avgs), ("second moments", exp_avg_sqs)):
        if len(got) != n:
            raise ValueError(f"{name}: {n} tensors required, not {len(got)}")
    for name, got in (("masters", masters), ("factors", m_scales), ("factors", v_scales)):
        if len(got) not in (0, n):
            raise ValueError(f"{name}: {n} tensors required, not {len(got)}")
    if masters and params[0].dtype == torch.float32:
        raise ValueError("fp32 parameters are their own masters")
    t = int(step)
    if t < 1:
        raise ValueError(f"steps count from 1, not {t}")
    for i in range(n):
        _reference_step(params[i], grads[i], masters[i] if masters else None, exp_avgs[i], exp_avg_sqs[i],
                        m_scales[i] if m_scales else None, v_scales[i] if v_scales else None, lrs[i],
                        decays[i], betas, eps, t, grad_scale)


def native_adamw() -> bool:
    """Whether CUDA tensors run the kernel; a missing extension is an error unless it is allowed."""
    if native.available():
        return True
    if os.environ.get("SLAPO_B200_ALLOW_FALLBACK", "0") == "1":
        return False
    raise RuntimeError("slapo_b200 native extension is not built/loaded but CUDA parameters were given")


def _reference_step(param, grad, master, exp_avg, exp_avg_sq, m_scale, v_scale, lr, decay, betas, eps, t,
                    grad_scale):
    b1, b2 = betas
    g = grad.float()
    if grad_scale is not None:
        g = g * grad_scale.to(g.device)
    if m_scale is not None:
        m = dequantize_moment(exp_avg, m_scale)
        v = dequantize_moment(exp_avg_sq, v_scale, second=True)
    else:
        m, v = exp_avg, exp_avg_sq
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    w = master if master is not None else param.float()
    update = (m / (1 - b1 ** t)) / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    w = w - lr * (update + decay * w)
    if master is not None:
        master.copy_(w)
    param.copy_(w)
    if m_scale is not None:
        for codes, scale, x, second in ((exp_avg, m_scale, m, False), (exp_avg_sq, v_scale, v, True)):
            new, factors = quantize_moment(x, second)
            codes.copy_(new)
            scale.copy_(factors)
    else:
        exp_avg.copy_(m)
        exp_avg_sq.copy_(v)


class FusedAdamW(torch.optim.Optimizer):
    """AdamW whose step is one kernel for all tensors of a type: ``FusedAdamW(model.parameters(), lr=...)``.

    ``state_bits``: 32, or 8 for moments of one byte each (rounded by at most 1 / 16 of themselves; ``eps`` as
    :func:`multi_tensor_adamw` says).
    ``master_weights``: keep fp32 copies of 16-bit parameters, which are what is updated (default); without
    them an update below half a step of the parameter's type is lost.  ``capturable``: steps are counted on
    the device, so that a captured ``step()`` can be replayed (with the ``lr`` and ``weight_decay`` of its
    capture; without, capturing a step is refused); parameters that were first updated together then have to
    go on together.
    ``step(grad_scale=...)`` takes a one-element fp32 tensor that multiplies every gradient (clipping, loss
    scaling).  Parameter groups may differ in ``lr``,
    ``weight_decay``, ``betas`` and ``eps``.  Parameters must be contiguous and their gradients dense."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32,
                 master_weights=True, capturable=False):
        if state_bits not in (8, 32):
            raise ValueError(f"moments of 8 or 32 bits, not {state_bits}")
        if lr < 0.0 or eps < 0.0 or weight_decay < 0.0:
            raise ValueError("lr, eps and weight_decay must not be negative")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas in [0, 1) required, not {betas}")
        self.state_bits, self.master_weights, self.capturable = state_bits, master_weights, capturable
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        own = ("state_bits", "master_weights", "capturable")
        return {**super().__getstate__(), **{name: getattr(self, name) for name in own}}

    def _new_state(self, p, counter):
        if not p.is_contiguous():
            raise ValueError(f"a parameter of shape {tuple(p.shape)} is not contiguous")
        if p.dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise ValueError(f"parameters of bf16, fp16 or fp32 required, not {p.dtype}")
        s = {"step": counter if counter is not None else 0}
        if self.master_weights and p.dtype != torch.float32:
            s["master"] = p.detach().float()
        if self.state_bits == 8:
            for name in ("exp_avg", "exp_avg_sq"):
                s[name] = torch.zeros(p.shape, dtype=torch.float8_e4m3fn, device=p.device)
                s[name + "_scale"] = torch.full((state_blocks(p.numel()),), 2.0 ** -126, device=p.device)
        else:
            s["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            s["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return s

    @torch.no_grad()
    def step(self, closure=None, grad_scale=None):
        """One update of every parameter that has a gradient.  What a refused step has not updated keeps its
        state, and its number of steps, unless that is counted on the device together with something that was
        updated."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        runs = {}       # one kernel for each device, type, betas, eps and number of steps
        fresh = {}      # the counters on the device of what is updated for the first time
        new = []        # states that begin with this step
        for group in self.param_groups:
            lr, decay = float(group["lr"]), float(group["weight_decay"])
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    continue
                if grad.layout != torch.strided:
                    raise RuntimeError("FusedAdamW takes dense gradients")
                s = self.state.get(p)
                if not s:
                    s = self._new_state(p, self._new_counter(p, fresh))
                    new.append(s)
                count = s["step"]
                key = (p.device, p.dtype, tuple(group["betas"]), group["eps"],
                       id(count) if torch.is_tensor(count) else count)
                run = runs.get(key)
                if run is None:
                    if not torch.is_tensor(count) and p.is_cuda and torch.cuda.is_current_stream_capturing():
                        # (every replay would be this step again, with its bias corrections)
                        raise RuntimeError("FusedAdamW: a step that is captured needs capturable=True")
                    run = runs[key] = ([], [], [], [], [])
                run[0].append(p)
                run[1].append(grad if grad.is_contiguous() else grad.contiguous())
                run[2].append(s)
                run[3].append(lr)
                run[4].append(decay)
        counters = self._count_on_device(runs.values(), new)
        try:
            for (_, _, betas, eps, _), (params, grads, states, lrs, decays) in runs.items():
                step = states[0]["step"]
                counted = torch.is_tensor(step)
                more = {}
                if "master" in states[0]:
                    more["masters"] = [s["master"] for s in states]
                if "exp_avg_scale" in states[0]:
                    more["exp_avg_scales"] = [s["exp_avg_scale"] for s in states]
                    more["exp_avg_sq_scales"] = [s["exp_avg_sq_scale"] for s in states]
                multi_tensor_adamw(params, grads, [s["exp_avg"] for s in states],
                                   [s["exp_avg_sq"] for s in states], lr=lrs, betas=betas, eps=eps,
                                   weight_decay=decays, step=step if counted else step + 1,
                                   grad_scale=grad_scale, **more)
                if counted:
                    counters.pop(id(step), None)
                else:
                    for s in states:
                        s["step"] = step + 1
                if new:
                    self.state.update(zip(params, states))
        except BaseException:
            for counter in counters.values():       # (of what nothing was updated with)
                counter.sub_(1)
            raise
        return loss

    def _new_counter(self, p, fresh):
        if not (self.capturable and p.is_cuda):
            return None
        if torch.cuda.is_current_stream_capturing():
            # (every replay of the graph would start from zeros)
            raise RuntimeError("FusedAdamW's state is made by its first step: take one before capturing")
        if p.device not in fresh:
            fresh[p.device] = torch.zeros(1, dtype=torch.int64, device=p.device)
        return fresh[p.device]

    def _count_on_device(self, runs, new):
        """Advance the counters on the device, each once, by all of the parameters that share it; by their
        ``id``."""
        if not self.capturable:
            return {}
        updated = {}
        for run in runs:
            for s in run[2]:
                if torch.is_tensor(s["step"]):
                    updated.setdefault(id(s["step"]), [s["step"], 0])[1] += 1
        shared = {}
        for s in [*self.state.values(), *new]:
            if torch.is_tensor(s.get("step")):
                shared[id(s["step"])] = shared.get(id(s["step"]), 0) + 1
        for key, (counter, n) in updated.items():
            if n != shared[key]:
                raise RuntimeError("capturable FusedAdamW: parameters that were first updated together need "
                                   f"their gradients together ({n} of {shared[key]} have one)")
        for counter, _ in updated.values():
            counter.add_(1)
        return {key: counter for key, (counter, _) in updated.items()}

    def load_state_dict(self, state_dict):
        """As ``torch.optim.Optimizer.load_state_dict``; states keep their own types, whatever the
        parameters' is.  Saved moments of another number of bits are refused; masters that are wanted and were
        not saved are made of the parameters, and saved ones that are not wanted are left out."""
        for old in state_dict["state"].values():
            if old and ("exp_avg_scale" in old) != (self.state_bits == 8):
                raise ValueError("the saved moments have another number of bits")
        super().load_state_dict(state_dict)
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        counters = {}
        for index, p in zip(saved, params):
            old = state_dict["state"].get(index)
            if not old:
                continue
            s = self.state[p]
            s.pop("master", None)
            keeps = self.master_weights and p.dtype != torch.float32
            if keeps and "master" not in old:
                s["master"] = p.detach().float()
            for name, value in old.items():
                if name == "step":
                    step = int(value)
                    if self.capturable and p.is_cuda:
                        if (p.device, step) not in counters:
                            counters[p.device, step] = torch.full((1,), step, dtype=torch.int64,
                                                                  device=p.device)
                        s["step"] = counters[p.device, step]
                    else:
                        s["step"] = step
                elif torch.is_tensor(value) and (keeps or name != "master"):
                    s[name] = value.detach().to(device=p.device, copy=True)
