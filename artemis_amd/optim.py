"""AdamW over many tensors at once, moments in 32 or 8 bits (``include/artemis_ops.h``: a launch takes up to 90
tensors, 59 with 8-bit moments).  ``adamw_step`` and ``adamw_step_8bit`` are the steps as functions on lists of tensors; ``AdamW``
is the optimizer around them (``train.py --optimizer adamw | adamw8``).

The 8-bit moments: 256 consecutive elements share an int32 base; a uint8 code counts from it in steps of
an eighth of a binade (v: 255 codes, m: a sign and 127), rounded up or down at random with the right mean, so
that a second moment that changes by a thousandth a step still moves.  State takes 2 + 8/256 bytes for a
parameter instead of 8.
"""
from __future__ import annotations

import torch

from . import _lib

GROUP = 256   # elements that share a base


def _step(*args):
    if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
        # the step number goes into the kernels' arguments: a replay would repeat it
        raise RuntimeError("an AdamW step cannot be captured into a graph: every replay would be the same step")
    _lib.load_ops_host().adamw(*args)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2):
    """Step number ``step`` (from 1) of AdamW, in place: lists of contiguous tensors of one type (fp32, bf16 or
    fp16; gradients of the same) on one device that do not overlap, moments fp32.

        p *= 1 - lr * weight_decay;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        p -= lr / (1 - b1^step) * m / (sqrt(v) / sqrt(1 - b2^step) + eps)
    """
    _step(params, grads, exp_avgs, exp_avg_sqs, [], [], 32, step, lr, *betas, eps, weight_decay, 0)


def adamw_step_8bit(params, grads, exp_avg_codes, exp_avg_bases, exp_avg_sq_codes, exp_avg_sq_bases, step, *,
                    lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, seed=0):
    """The same with moments in 8 bits: uint8 codes like the parameters, one int32 base for each 256 elements (the
    last group may be short); zeros stand for 0.  ``seed`` goes into the random rounding, with the step and the
    element's place in the list of tensors: the same call gives the same bits.  A gradient that is not finite
    spoils the moments of its group."""
    _step(params, grads, exp_avg_codes, exp_avg_sq_codes, exp_avg_bases, exp_avg_sq_bases, 8, step, lr, *betas, eps,
          weight_decay, seed)


def moments_from_8bit(codes, bases, signed):
    """The fp32 values (a list of tensors like ``codes``) that 8-bit moments stand for; ``signed``: of first
    moments (exp_avg), not second ones."""
    return _lib.load_ops_host().moments_from_8bit(codes, bases, signed)


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is one kernel launch for each 90 tensors (8 bit: 59).  ``moment_bits`` 32 or 8.  Parameters on HIP
    devices, contiguous, fp32, bf16 or fp16; dense gradients."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, moment_bits=32, seed=0):
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, moment_bits=moment_bits, seed=seed)
        self._check(defaults)
        super().__init__(params, defaults)

    @staticmethod
    def _check(group):
        if group["moment_bits"] not in (32, 8):
            raise ValueError(f"moment_bits must be 32 or 8, got {group['moment_bits']}")
        if not group["lr"] >= 0 or not group["eps"] >= 0 or not group["weight_decay"] >= 0:
            raise ValueError(f"lr={group['lr']}, eps={group['eps']} and weight_decay={group['weight_decay']} must be >= 0")
        if not (0 <= group["betas"][0] < 1 and 0 <= group["betas"][1] < 1):
            raise ValueError(f"betas must lie in [0, 1), got {group['betas']}")

    def add_param_group(self, param_group):
        self._check({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def _start(self, p, bits):
        state = self.state[p]
        state["step"] = 0
        n = (p.numel() + GROUP - 1) // GROUP
        for name in ("exp_avg", "exp_avg_sq"):
            if bits == 32:
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            else:
                state[name + "_codes"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
                state[name + "_bases"] = torch.zeros(n, dtype=torch.int32, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            bits = group["moment_bits"]
            # one launch takes tensors of one type, device and step number
            calls = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                state = self.state[p] or self._start(p, bits)
                calls.setdefault((p.dtype, p.device, state["step"] + 1), []).append((p, p.grad.contiguous(), state))
            for (_, _, number), items in calls.items():
                ps, gs = [i[0] for i in items], [i[1] for i in items]
                args = dict(lr=float(group["lr"]), betas=group["betas"], eps=group["eps"],
                            weight_decay=group["weight_decay"])
                if bits == 32:
                    adamw_step(ps, gs, [i[2]["exp_avg"] for i in items], [i[2]["exp_avg_sq"] for i in items], number, **args)
                else:
                    adamw_step_8bit(ps, gs, *[[i[2][n] for i in items] for n in (
                        "exp_avg_codes", "exp_avg_bases", "exp_avg_sq_codes", "exp_avg_sq_bases")], number,
                        seed=group["seed"], **args)
                for i in items:  # (a refused step is not counted)
                    i[2]["step"] = number
        return loss

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the base class casts state to the parameter's type; codes, bases and fp32 moments keep their own
        given = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(given, params):
            for name, value in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(value):
                    self.state[p][name] = value.to(device=p.device, copy=True)
