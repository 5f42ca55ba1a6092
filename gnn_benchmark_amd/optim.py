"""AdamW over many tensors at once, one launch for up to 48 of them, states in 32 or in 8 bits.

``AdamW`` is a ``torch.optim.Optimizer`` for ``gcn.train_step`` / ``sage.train_step`` and any other loop;
``adamw_step`` is the step on plain lists of tensors.  A step counts itself on the device, so it can be captured into a
HIP graph and replayed.

States in 8 bits are in the format of ``fp8`` (e4m3 codes, blocks of 128 elements, power-of-two scales): ``exp_avg`` is m
rounded to nearest, ``exp_avg_sq`` holds sqrt(v) -- half the range in powers of two -- rounded to one of its two
neighbours with the odds of the distance, because a step at ``beta2 = 0.999`` moves sqrt(v) by far less than half a code
and rounding to nearest would never let it move.  The random bits come from a hash of (seed, tensor, step, element): the
same calls give the same bits, on every rank.
"""
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import ext
from .fp8 import BLOCK

_FLOATS = {torch.float32, torch.bfloat16}
_OWN_KEYS = ("state_bits", "min_8bit_size", "seed")
# of torch's groups: how its step runs, or (refused unless off) by which rule
_TORCH_KEYS = ("amsgrad", "maximize", "foreach", "capturable", "differentiable", "fused", "decoupled_weight_decay")


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], steps: torch.Tensor, *, lr: Union[float, torch.Tensor],
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               masters: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None, seed: int = 0, first: int = 0) -> None:
    """One step in place: parameters, states and ``steps`` (int32 [len(params)], steps taken so far) are updated.

    Parameters: all fp32, or all bf16 with fp32 ``masters`` (the values that are updated; the parameters receive them
    rounded).  Gradients: all fp32 or all bf16.  States: fp32 ``exp_avgs`` / ``exp_avg_sqs``, or float8_e4m3fn codes of m
    and sqrt(v) with ``exp_avg_scales`` / ``exp_avg_sq_scales`` (float8_e8m0fnu, one for each 128 elements).  ``lr``: a
    number, or an fp32 scalar on the device that is read when the step runs.  No tensor that is written may overlap another
    that is written or read, gradients and a learning rate on the device among them (that is refused).  ``first``: number
    of the first tensor for the 8-bit states' random bits, where a list is split over calls."""
    ext.train_ops().adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, lr, betas[0], betas[1], eps, weight_decay, masters,
                               exp_avg_scales, exp_avg_sq_scales, seed & 0xFFFFFFFF, first)


class _Run:
    """Parameters of one kind in a group and their array of step counts.  ``kept[i]``: what ``state[params[i]]["step"]`` was
    made to be, the i-th entry; None while params[i] has no state (its count is zero then)."""
    __slots__ = ("bits", "params", "steps", "kept")

    def __init__(self, bits: int, params: List[torch.Tensor], steps: torch.Tensor):
        self.bits, self.params, self.steps, self.kept = bits, params, steps, [None] * len(params)


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s update and arguments, each parameter group in a few launches.

    ``state_bits`` 8 keeps both states of tensors of at least ``min_8bit_size`` elements in 8 bits (2 bytes an element
    instead of 8), the others in 32.  bf16 parameters keep an fp32 master in their state.  A step can be captured into a
    HIP graph once it has run eagerly (the states exist then); ``lr`` may be an fp32 scalar tensor on the device, which a
    captured step reads anew at every replay.  A parameter, state or step count that a program changes is found by the next
    step, which has to be an eager one; steps captured before go on as they were.  Sparse gradients are refused."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits: int = 32,
                 min_8bit_size: int = 4096, seed: int = 0):
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8")
        if not isinstance(lr, torch.Tensor) and lr < 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"Invalid betas: {betas}")
        if eps < 0.0 or weight_decay < 0.0:
            raise ValueError("eps and weight_decay must not be negative")
        self._runs, self._captured = {}, []
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, min_8bit_size=min_8bit_size, seed=seed))

    def __setstate__(self, state):
        super().__setstate__(state)
        self._runs, self._captured = {}, []

    # ------------------------------------------------------------------ states
    @staticmethod
    def _kind(p: torch.Tensor, group) -> Tuple[torch.device, torch.dtype, int]:
        bits = 8 if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"] else 32
        return p.device, p.dtype, bits

    def _new_state(self, p: torch.Tensor, bits: int) -> dict:
        if not p.is_cuda or p.dtype not in _FLOATS or not p.is_contiguous():
            raise RuntimeError("Input mismatch: AdamW takes contiguous float32 or bfloat16 parameters on a GPU (HIP) device")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW's states do not exist yet: run one step before capturing one")
        state = {}
        flat = (p.numel(),)
        if bits == 32:
            for key in ("exp_avg", "exp_avg_sq"):
                state[key] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        else:
            for key in ("exp_avg", "exp_avg_sq"):
                # the zero code and the scale byte of an empty block
                state[key] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                state[key + "_scales"] = torch.ones(-(-flat[0] // BLOCK), dtype=torch.uint8,
                                                    device=p.device).view(torch.float8_e8m0fnu)
        if p.dtype == torch.bfloat16:
            state["master"] = p.detach().float()
        return state

    def _kept_step(self, p: torch.Tensor):
        """What ``state[p]["step"]`` is; None where p has no state."""
        state = self.state.get(p)
        return state.get("step", 0) if state else None

    def _prepare(self, index: int, group) -> list:
        """The group's parameters in an order that puts those of one kind (device, type, state) side by side, with one
        array of step counts for each kind: [_Run].  ``state[p]["step"]`` is p's entry of it.  What a program changes from
        outside -- parameters, their order, states taken away or put in place, step counts -- is found by comparing with
        what the arrays were made from, object by object, and the arrays are made again from the states."""
        ps = group["params"]
        kinds = [self._kind(p, group) for p in ps]
        before, known = self._runs.get(index, ([], None))
        if (known is not None and len(known) == len(ps)
                and all(p is q and kind == k for p, kind, (q, k) in zip(ps, kinds, known))
                and all(self._kept_step(p) is kept for run in before for p, kept in zip(run.params, run.kept))):
            return before
        by_kind = {}
        for p, kind in zip(ps, kinds):
            by_kind.setdefault(kind, []).append(p)
        if any(kind[0].type != "cuda" for kind in by_kind):
            raise RuntimeError("Input mismatch: AdamW takes parameters on a GPU (HIP) device")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW's parameters or states are new or were changed: run one step before capturing one")
        runs = []
        for kind, members in by_kind.items():
            steps = torch.tensor([int(self._kept_step(p) or 0) for p in members], dtype=torch.int32, device=kind[0])
            for old in before:  # the array stays where it is if it can: captured steps raise it there
                if (old.steps.device == kind[0] and old.bits == kind[2] and len(old.params) == len(members)
                        and all(p is q for p, q in zip(old.params, members))):
                    steps = old.steps.copy_(steps)
            run = _Run(kind[2], members, steps)
            for i, p in enumerate(members):
                if self._kept_step(p) is not None:
                    self.state[p]["step"] = run.kept[i] = run.steps[i]
            runs.append(run)
        self._runs[index] = runs, list(zip(ps, kinds))
        return runs

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        number = 0  # of a tensor among all groups', for its random bits
        for index, group in enumerate(self.param_groups):
            for run in self._prepare(index, group):
                ps, at = run.params, 0
                while at < len(ps):  # stretches of parameters that have a gradient: each has its own count of steps
                    if ps[at].grad is None:
                        at += 1
                        continue
                    end = at
                    while end < len(ps) and ps[end].grad is not None:
                        end += 1
                    self._step_stretch(group, run, at, end, number + at)
                    at = end
                number += len(ps)
        return loss

    def _step_stretch(self, group, run: "_Run", at: int, end: int, number: int) -> None:
        ps, bits, states = run.params[at:end], run.bits, []
        for i, p in enumerate(ps, at):
            if p.grad.is_sparse:
                raise RuntimeError("AdamW does not take sparse gradients")
            state = self.state[p]
            if not state:
                state.update(self._new_state(p, bits))
                state["step"] = run.kept[i] = run.steps[i]
            states.append(state)
        if torch.cuda.is_current_stream_capturing() and not any(run.steps is t for t in self._captured):
            self._captured.append(run.steps)  # the graph writes there as long as it lives, whatever becomes of the run
        grads = [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p in ps]
        adamw_step(ps, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], run.steps[at:end],
                   lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                   masters=[s["master"] for s in states] if ps[0].dtype == torch.bfloat16 else None,
                   exp_avg_scales=[s["exp_avg_scales"] for s in states] if bits == 8 else None,
                   exp_avg_sq_scales=[s["exp_avg_sq_scales"] for s in states] if bits == 8 else None,
                   seed=group["seed"], first=number)

    # ------------------------------------------------------------------ checkpoints
    def load_state_dict(self, state_dict) -> None:
        """Takes over a ``state_dict`` of this class, or one of ``torch.optim.AdamW`` (``Adam`` where it has no weight decay;
        groups of a torch that does not say how its decay works are taken for AdamW's) with fp32 states where this
        optimizer's states are in 32 bits.  Groups that step by another rule -- ``maximize``, ``amsgrad``, a weight decay that
        is added to the gradient, another class of optimizer -- are refused, and so are states that do not fit; a refusal
        leaves this optimizer as it was.  The states are new tensors: a step captured before is captured again.  (torch's
        own loading casts states to their parameter's type, which would turn 8-bit codes and fp32 states of bf16
        parameters into something else.)"""
        saved = state_dict["param_groups"]
        for g in saved:
            self._refuse_another_rule(g)
        sizes = [len(g["params"]) for g in saved]
        if sizes != [len(g["params"]) for g in self.param_groups]:
            super().load_state_dict({"state": {}, "param_groups": saved})  # says which sizes differ
        groups = [{**{k: own[k] for k in _OWN_KEYS}, **{k: v for k, v in g.items() if k not in _TORCH_KEYS}}
                  for g, own in zip(saved, self.param_groups)]
        states = {}
        for g, own in zip(groups, self.param_groups):
            for i, p in zip(g["params"], own["params"]):
                old = state_dict["state"].get(i)
                if old:
                    states[p] = self._taken_over(old, self._new_state(p, self._kind(p, g)[2]))
        super().load_state_dict({"state": {}, "param_groups": groups})
        self.state.update(states)
        self._runs = {}

    @staticmethod
    def _refuse_another_rule(group) -> None:
        if "state_bits" in group:  # this class's
            return
        why = None
        if "amsgrad" not in group or "betas" not in group:
            why = "not torch.optim.Adam's or AdamW's"
        elif group["amsgrad"] or group.get("maximize"):
            why = "amsgrad" if group["amsgrad"] else "maximize"
        elif group["weight_decay"] != 0 and group.get("decoupled_weight_decay") is False:
            why = "a weight decay that is added to the gradient"
        if why:
            raise RuntimeError(f"Input mismatch: the saved parameter groups step by another rule ({why})")

    @staticmethod
    def _taken_over(old, state: dict) -> dict:
        """The saved state ``old`` in the place of the fresh one."""
        for key, t in state.items():
            src = old.get(key)
            if key == "master" and src is None:
                continue
            if src is None or src.dtype != t.dtype or src.shape != t.shape:
                raise RuntimeError(f"Input mismatch: the saved {key} does not fit this optimizer's states (type and "
                                   "shape have to be the same)")
            t.copy_(src)
        state["step"] = int(old["step"])
        return state
