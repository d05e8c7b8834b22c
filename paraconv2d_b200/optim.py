"""SGD for networks of ParaConv2d layers, honouring the optimizer tags the
module sets on its flat parameter vector (reference ptparaconv2d.py:194-198):
``pars.h_lr_factor`` and ``pars.p_lr_factor`` multiply the learning rate of
the [h0 | h] and [p | p0] parts, ``pars.wd_factor`` multiplies the weight
decay ("Multiplies the learning rate / weight decay applied to the parameters
by the optimizer", the reference module's docstring).

The update is torch.optim.SGD's (momentum without dampening or Nesterov,
weight decay added to the gradient):

    d = grad + weight_decay * wd_factor * w
    buf = momentum * buf + d            (buf = d on the first step)
    w -= lr * lr_factor * buf

For a tagged ``pars`` on the GPU it is one fused kernel (``pc2d_param_step``:
one pass over the parameters, the gradient and the momentum buffer); other
parameters, and tagged ones on the CPU, take the same update in torch ops.

:func:`adamw_step` is AdamW over many tensors at once, on the GPU, with the
moments in 32 or in 8 bits; :class:`ParaboloidAdamW` is the optimizer over it,
honouring the same tags.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor
from torch.optim import Optimizer

from . import _lib

_lib.load_op_library()
_adamw_step = torch.ops.paraconv2d_b200.adamw_step.default
_adamw_state_values = torch.ops.paraconv2d_b200.adamw_state_values.default


def paraboloid_split(p: torch.Tensor):
    """(m, d) of a tagged flat parameter vector [h0 | h | p | p0] of
    2*m*(1+d) values, d = ``p.d`` (input channels x window)."""
    d = int(p.d)
    n = p.numel()
    if d < 0 or n % (2 * (d + 1)) != 0:
        raise ValueError(f"a paraboloid parameter vector of {n} values does not split with d = {d}")
    return n // (2 * (d + 1)), d


def sgd_step_reference(w, g, buf, first, nh, lr_h, lr_p, wd, momentum):
    """The update in torch ops (in place on w and buf): the first nh values
    use lr_h, the rest lr_p."""
    d = g.add(w, alpha=wd) if wd != 0 else g
    if momentum != 0:
        if first:
            buf.copy_(d)
        else:
            buf.mul_(momentum).add_(d)
        d = buf
    if nh >= w.numel():
        w.add_(d, alpha=-lr_h)
        return
    flat_w, flat_d = w.view(-1), d.reshape(-1)
    flat_w[:nh].add_(flat_d[:nh], alpha=-lr_h)
    flat_w[nh:].add_(flat_d[nh:], alpha=-lr_p)


class ParaboloidSGD(Optimizer):
    """SGD with the ParaConv2d tags applied per parameter (see the module
    docstring).  Parameters without the tags get plain SGD."""

    def __init__(self, params, lr: float, momentum: float = 0.0, weight_decay: float = 0.0):
        if lr < 0 or momentum < 0 or weight_decay < 0:
            raise ValueError("ParaboloidSGD: lr, momentum and weight_decay must be non-negative")
        super().__init__(params, dict(lr=lr, momentum=momentum, weight_decay=weight_decay))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            lr, mom, wd = group["lr"], group["momentum"], group["weight_decay"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                first = "momentum_buffer" not in state
                if mom != 0 and first:
                    state["momentum_buffer"] = torch.empty_like(p, memory_format=torch.contiguous_format)
                buf = state.get("momentum_buffer")
                if getattr(p, "isParaboloid", False):
                    m, d = paraboloid_split(p)
                    hf, pf, wdf = float(p.h_lr_factor), float(p.p_lr_factor), float(p.wd_factor)
                    if p.is_cuda and p.dtype in (torch.float32, torch.float64):
                        g = p.grad.contiguous()
                        if not p.is_contiguous():
                            raise ValueError("ParaboloidSGD: the paraboloid parameter vector must be contiguous")
                        lib = _lib.cabi()
                        st = lib.pc2d_param_step(0 if p.dtype == torch.float32 else 1, p.data_ptr(), g.data_ptr(),
                                                 buf.data_ptr() if buf is not None else None, m, d, lr, hf, pf, wd,
                                                 wdf, mom, 1 if first else 0,
                                                 torch.cuda.current_stream(p.device).cuda_stream)
                        if st != 0:
                            raise RuntimeError(_lib.status_message(st))
                    else:
                        sgd_step_reference(p, p.grad, buf, first, m * (1 + d), lr * hf, lr * pf, wd * wdf, mom)
                else:
                    sgd_step_reference(p, p.grad, buf, first, p.numel(), lr, lr, wd, mom)
                if mom != 0:
                    state["momentum_buffer"] = buf
        return loss


# ---------------------------------------------------------------------- AdamW

def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor],
               exp_avg_sqs: Sequence[Tensor], step: Tensor, *, lr: Union[float, Tensor],
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               masters: Optional[Sequence[Optional[Tensor]]] = None, scales: Optional[Sequence[Tensor]] = None,
               factors: Optional[Sequence[Optional[Tuple[int, float, float, float]]]] = None,
               grad_scale: Optional[Tensor] = None, seed: int = 0, numbers: Optional[Sequence[int]] = None) -> None:
    """One AdamW step over many tensors, in place, in two launches (and one
    more for every further combination of types, and beyond 320 tensors)::

        t = step + 1;  g = grad * grad_scale
        m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
        w = (1 - lr weight_decay) w - lr m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps)

    ``params``: float32, float16 or bfloat16, dense in any order of their
    dimensions; ``grads`` of the same type or float32.  ``step`` (int64 [1],
    on the GPU) is counted by the call; with it, and with ``lr`` as a float32
    number on the GPU, a captured step can be replayed.  ``grad_scale`` (one
    float32 number on the GPU): what the gradients are multiplied by, as
    clipping their norm needs it.  ``masters``: float32 copies of 16-bit
    parameters (None for the float32 ones among them), which hold the weights;
    the parameters are their roundings.  ``factors``: for each parameter None
    or (split, rate of the first `split` elements, rate of the others, factor
    of the weight decay).

    The moments are float32 of their parameter's shape and strides, or uint8
    [n] with ``scales`` (uint8 [ceil(n/256), 2]): codes of 8-bit floats with
    3 bits of mantissa under an exponent for every 256 elements, rounded
    stochastically by ``seed``, the step, the tensor's number (``numbers``, or
    its place in the list) and the element's place in it (see
    :func:`adamw_new_state`, :func:`adamw_state_values`).  The update is
    computed from the moments before they are rounded.  Where a moment is not
    finite, the state of its 256 elements becomes NaN.

    No tensor that is written may share memory with another one of the call.
    """
    if not params:
        return
    rate, rate_tensor = (0.0, lr) if isinstance(lr, Tensor) else (float(lr), None)
    if masters is not None:
        none = step.new_empty(0, dtype=torch.float32) if any(m is None for m in masters) else None
        masters = [none if m is None else m for m in masters]
    splits, rates = [], []
    if factors is not None:
        if len(factors) != len(params):
            raise ValueError(f"factors must be as many as params ({len(params)}), got {len(factors)}")
        for p, f in zip(params, factors):
            split, first, rest, decay = (p.numel(), 1.0, 1.0, 1.0) if f is None else f
            splits.append(split)
            rates += (first, rest, decay)
    _adamw_step(params, grads, exp_avgs, exp_avg_sqs, masters or [], scales or [], step, rate_tensor, rate, betas[0],
                betas[1], eps, weight_decay, grad_scale, splits, rates, seed, numbers or [])


def adamw_new_state(param: Tensor, bits: int = 32):
    """Zero moments for a parameter: (exp_avg, exp_avg_sq, scales), the last
    one None for 32 bits."""
    if bits == 32:
        return (*(torch.zeros_like(param, dtype=torch.float32, requires_grad=False) for _ in range(2)), None)
    if bits != 8:
        raise ValueError(f"states of 32 or 8 bits, got {bits}")
    n = param.numel()
    return tuple(torch.zeros(s, dtype=torch.uint8, device=param.device) for s in ((n,), (n,), (-(-n // 256), 2)))


@torch.no_grad()
def adamw_state_values(exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor], scales: Sequence[Tensor],
                       dtype: torch.dtype = torch.float32) -> Tuple[List[Tensor], List[Tensor]]:
    """The values of moments in 8 bits, flat, as float32 or bfloat16 (both
    hold them exactly): the lists of the first and of the second moments."""
    exp_avgs = list(exp_avgs)
    if not exp_avgs:
        return [], []
    outs = _adamw_state_values(exp_avgs, list(exp_avg_sqs), list(scales), dtype)
    return outs[:len(exp_avgs)], outs[len(exp_avgs):]


class ParaboloidAdamW(Optimizer):
    """:func:`adamw_step` over a model's parameters (CUDA; float32, float16,
    bfloat16), with the ParaConv2d tags applied: ``h_lr_factor`` and
    ``p_lr_factor`` multiply the learning rate of the two halves of a layer's
    ``pars``, ``wd_factor`` its weight decay.

    ``state_bits``: 32, or 8 for moments of two bytes and a 128th per element
    instead of eight.  ``masters``: keep float32 copies of 16-bit parameters.  ``seed``:
    of the stochastic rounding of 8-bit moments, with a parameter's place among
    all of the optimizer's; ranks that hold the same parameters need the same one.  ``lr`` may be a float32 tensor on the GPU.
    Steps are counted on the GPU, for all parameters that have had the same
    gradients together (one that gets none is left as it is and goes on at its
    own count), so that ``step`` can be captured into a CUDA graph after one
    outside of the same parameters' gradients (a capture that would have to make
    a state or a count raises); the gradients must then stay the same tensors,
    and a step outside of other parameters ends the graph's use."""

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32, masters: bool = False,
                 seed: int = 0):
        if not isinstance(lr, Tensor) and lr < 0 or eps < 0 or weight_decay < 0:
            raise ValueError("ParaboloidAdamW: lr, eps and weight_decay must be non-negative")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError(f"ParaboloidAdamW: betas must be in [0, 1), got {betas}")
        if state_bits not in (8, 32):
            raise ValueError(f"ParaboloidAdamW: states of 32 or 8 bits, got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, masters=bool(masters), seed=int(seed)))

    @staticmethod
    def _not_captured(why):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"ParaboloidAdamW: a parameter cannot be stepped in a capture yet: {why}; take a step with "
                               "the same gradients outside it")

    def _new_state(self, p, group):
        if not p.is_cuda or p.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise NotImplementedError("ParaboloidAdamW: float32, float16 and bfloat16 parameters on the GPU only, got "
                                      f"{p.dtype} on {p.device}")
        self._not_captured("its first step makes its state, which a graph would clear at every replay")
        state = self.state[p]
        state["exp_avg"], state["exp_avg_sq"], scales = adamw_new_state(p, group["state_bits"])
        if scales is not None:
            state["scales"] = scales
        if group["masters"] and p.dtype != torch.float32:
            state["master"] = p.detach().float()

    @torch.no_grad()
    def step(self, closure=None, grad_scale: Optional[Tensor] = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        number, numbers = 0, {}  # places among all parameters: what their random numbers go by
        for group in self.param_groups:
            cohorts = {}  # parameters by the counter that they share
            for p in group["params"]:
                numbers[p] = number
                number += 1
                if p.grad is None:
                    continue
                if "step" not in self.state[p]:
                    self._new_state(p, group)
                    cohorts.setdefault((None, p.device), []).append(p)
                else:
                    cohorts.setdefault((id(self.state[p]["step"]), p.device), []).append(p)
            for (counter, device), members in cohorts.items():
                if counter is None:
                    count = torch.zeros(1, dtype=torch.int64, device=device)
                else:
                    count = self.state[members[0]]["step"]
                    if any(self.state[q].get("step") is count for q in group["params"] if q.grad is None):
                        # the others stay where they are
                        self._not_captured("it gets a count of its own, which a graph would start anew at every replay")
                        count = count.clone()
                for p in members:
                    self.state[p]["step"] = count
                states = [self.state[p] for p in members]
                factors = None
                if any(getattr(p, "isParaboloid", False) for p in members):
                    factors = []
                    for p in members:
                        if getattr(p, "isParaboloid", False):
                            m, d = paraboloid_split(p)
                            factors.append((m * (1 + d), p.h_lr_factor, p.p_lr_factor, p.wd_factor))
                        else:
                            factors.append(None)
                adamw_step(members, [p.grad for p in members], [s["exp_avg"] for s in states],
                           [s["exp_avg_sq"] for s in states], count, lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"],
                           masters=[s.get("master") for s in states] if group["masters"] else None,
                           scales=[s["scales"] for s in states] if group["state_bits"] == 8 else None,
                           factors=factors, grad_scale=grad_scale, seed=group["seed"],
                           numbers=[numbers[p] for p in members] if group["state_bits"] == 8 else None)
        return loss

    def load_state_dict(self, state_dict):
        """As for every optimizer; the states keep the types they were saved
        in, and parameters whose counts are equal share one again."""
        super().load_state_dict(state_dict)
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            counts = {}
            for p, place in zip(group["params"], saved["params"]):
                state = state_dict["state"].get(place)
                if not state:
                    continue
                mine = self.state[p]
                for name, value in state.items():
                    # (the base class would have turned them into the parameter's type)
                    mine[name] = value.to(device=p.device, copy=True) if isinstance(value, Tensor) else value
                mine["step"] = counts.setdefault((int(mine["step"]), p.device), mine["step"])
