"""AdamW over many tensors in few launches, its states in 32 bits or in 8, and Muon over
many matrices.

``adamw_step`` and ``muon_step`` are the steps themselves over lists of tensors; ``AdamW``
and ``Muon`` the optimisers that hold the states.  The steps are HIP kernels behind the C
ABI (csrc/torch_sequence.cpp, csrc/adamw.hip, csrc/muon.hip); there is no torch or CPU
fallback.  No counterpart in the reference, which trains with torch's optimisers.
"""
import math

import torch

from ._native import torch_binding

__all__ = ["adamw_step", "AdamW", "muon_step", "Muon"]

_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_GROUP = 32   # values that share a scale


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2, exp_avg_scales=None, exp_avg_sq_scales=None, masters=None,
               seed=0):
    """One AdamW step, in place, over lists of tensors:

        m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
        p = p (1 - lr wd) - lr / (1 - b1^step) m / (sqrt(v / (1 - b2^step)) + eps)

    Arguments:
        params: tensors of one type (float32 or bfloat16) on one device, dense in memory
        grads: their gradients, of the same type and shapes
        exp_avgs, exp_avg_sqs: m and v, float32 in the parameters' shapes and layouts;
            or, with the scales, 8-bit states: float8_e4m3fn tensors of as many values
            (in the parameter's order in memory) that hold m and sqrt(v), each 32 of
            them with one power-of-two scale
        step: int, the step's number, from 1
        lr, betas, eps, weight_decay: floats
        exp_avg_scales, exp_avg_sq_scales: the scales, float8_e8m0fnu tensors of
            ceil(n / 32) values; give both or neither
        masters: float32 tensors in the parameters' shapes that the step moves in the
            parameters' place; each parameter becomes its master's rounding
        seed: int, of the random rounding of 8-bit states (a call's result depends on
            its arguments alone)

    The tensors that it writes do not overlap; one that comes twice is refused.  The
    step's number is part of the launch: a step captured in a graph keeps it.
    """
    torch_binding().adamw(params, grads, exp_avgs, exp_avg_sqs, int(step), float(lr),
                          float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
                          exp_avg_scales, exp_avg_sq_scales, masters, int(seed))


class _Optimizer(torch.optim.Optimizer):
    def load_state_dict(self, state_dict):
        """As torch's, but the states keep their own types (torch casts them to the
        parameter's)."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, own):
            for name, value in saved.get(i, {}).items():
                if isinstance(value, torch.Tensor):
                    self.state[p][name] = value.to(p.device).clone(memory_format=torch.preserve_format)


class AdamW(_Optimizer):
    """AdamW on ``adamw_step``.

    Arguments:
        params: parameters or groups of them, float32 or bfloat16 on the GPU
        lr, betas, eps, weight_decay: as torch.optim.AdamW
        state_bits: 32, or 8: the moments in 8 bits (2.1 bytes a parameter, not 8)
        master_weights: bool, keep 32-bit values of bfloat16 parameters, which
            otherwise lose steps smaller than their rounding (taken from the parameters
            at the first step; a parameter set by hand afterwards is not seen)
        seed: int, of the 8-bit states' random rounding
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *,
                 state_bits=32, master_weights=True, seed=0):
        assert state_bits in (8, 32), 'state_bits must be 8 or 32'
        assert lr >= 0 and eps >= 0 and weight_decay >= 0, \
            'lr, eps and weight_decay must not be negative'
        assert all(0 <= b < 1 for b in betas), 'betas must be in [0, 1)'
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, master_weights=master_weights,
                                      seed=seed))

    def _new_state(self, p, group):
        n, dev = p.numel(), p.device
        state = {"step": 0}
        for name in ("exp_avg", "exp_avg_sq"):
            if group["state_bits"] == 32:
                state[name] = torch.zeros_like(p, dtype=torch.float32,
                                               memory_format=torch.preserve_format)
            else:
                state[name] = torch.zeros(n, dtype=torch.uint8, device=dev).view(_E4M3)
                state[name + "_scale"] = torch.zeros(-(-n // _GROUP), dtype=torch.uint8,
                                                     device=dev).view(_E8M0)
        if p.dtype != torch.float32 and group["master_weights"]:
            state["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        """One step for every parameter that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # what is refused is refused before anything moves, or is not counted
        for group in self.param_groups:
            for p in group["params"]:
                assert p.grad is None or not p.grad.is_sparse, 'AdamW does not take sparse gradients'
        ordinal = 0
        for group in self.param_groups:
            # one call for the parameters of one type and device that took as many steps
            calls = {}
            try:
                for p in group["params"]:
                    ordinal += 1
                    if p.grad is None:
                        continue
                    state = self.state[p]
                    if not state:
                        state.update(self._new_state(p, group))
                    state["step"] = int(state["step"]) + 1
                    key = (p.dtype, p.device, state["step"], "master" in state)
                    if key not in calls:
                        calls[key] = ([], [], [], ordinal)
                    calls[key][0].append(p)
                    calls[key][1].append(p.grad)
                    calls[key][2].append(state)
                for key in list(calls):
                    self._call(group, key, *calls[key])
                    del calls[key]
            except Exception:
                for _, _, states, _ in calls.values():
                    for state in states:
                        state["step"] -= 1
                raise
        return loss

    @staticmethod
    def _call(group, key, params, grads, states, first):
        _, _, step, master = key
        lists = {k: [s[k] for s in states] for k in ("exp_avg", "exp_avg_sq")}
        eight = group["state_bits"] == 8
        scales = [[s[k + "_scale"] for s in states] if eight else None for k in lists]
        adamw_step(params, grads, lists["exp_avg"], lists["exp_avg_sq"], step, group["lr"],
                   group["betas"], group["eps"], group["weight_decay"], *scales,
                   [s["master"] for s in states] if master else None,
                   group["seed"] + 7919 * first)


def _rate(lr, adjust_lr_fn, shape):
    rows, cols = shape
    if rows == 0 or cols == 0:
        return 0.0
    if adjust_lr_fn == "match_rms_adamw":
        return lr * 0.2 * math.sqrt(max(rows, cols))
    return lr * math.sqrt(max(1.0, rows / cols))


def muon_step(params, grads, momenta, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True,
              ns_coefficients=(3.4445, -4.775, 2.0315), eps=1e-7, ns_steps=5, adjust_lr_fn=None,
              masters=None):
    """One Muon step, in place, over lists of matrices:

        m = momentum m + (1 - momentum) g
        u = momentum m + (1 - momentum) g  (nesterov; else u = m)
        X = u / max(|u|, eps),  ns_steps times  X = c0 X + (c1 A + c2 A^2) X,  A = X X^T
        p = p (1 - lr weight_decay) - lr adjust X

    Arguments:
        params: contiguous matrices of one type (float32 or bfloat16) on one device
        grads: their gradients, of the same type and shapes
        momenta: m, contiguous float32 in the parameters' shapes
        lr, weight_decay, momentum, eps: floats
        ns_coefficients: c0, c1, c2; such that X's values stay below 60
        ns_steps: int, 1 to 100
        adjust_lr_fn: None or "original": adjust = sqrt(max(1, rows / cols));
            "match_rms_adamw": 0.2 sqrt(max(rows, cols))
        masters: contiguous float32 matrices in the parameters' shapes that the step moves
            in the parameters' place; each parameter becomes its master's rounding

    X and A are held to 22 bits whatever the parameters' type, values below 2^-12 to 2^-35
    (of an update whose values are all of one size, 20 bits at 2^30 of them).  The matrices
    that it writes do not overlap; one that comes twice is refused.  The rates are part of
    the launch: a step captured in a graph keeps them.
    """
    assert adjust_lr_fn in (None, "original", "match_rms_adamw"), \
        'adjust_lr_fn must be None, "original" or "match_rms_adamw"'
    assert all(p.dim() == 2 for p in params), 'muon_step takes matrices'
    rates = [_rate(float(lr), adjust_lr_fn, p.shape) for p in params]
    torch_binding().muon(params, grads, momenta, rates, float(lr), float(weight_decay),
                         float(momentum), bool(nesterov), tuple(map(float, ns_coefficients)),
                         float(eps), int(ns_steps), masters)


class Muon(_Optimizer):
    """Muon on ``muon_step``, for the matrices of a network (the others take AdamW).

    Arguments:
        params: matrices or groups of them, contiguous, float32 or bfloat16 on the GPU
        lr, weight_decay, momentum, nesterov, ns_coefficients, eps, ns_steps,
            adjust_lr_fn: as ``muon_step``
        master_weights: bool, keep 32-bit values of bfloat16 parameters, which otherwise
            lose steps smaller than their rounding (taken from the parameters at the first
            step; a parameter set by hand afterwards is not seen)
    """

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True,
                 ns_coefficients=(3.4445, -4.775, 2.0315), eps=1e-7, ns_steps=5, adjust_lr_fn=None, *,
                 master_weights=True):
        assert lr >= 0 and eps >= 0 and weight_decay >= 0, \
            'lr, eps and weight_decay must not be negative'
        assert 0 <= momentum < 1, 'momentum must be in [0, 1)'
        assert 1 <= ns_steps <= 100, 'ns_steps must be from 1 to 100'
        assert adjust_lr_fn in (None, "original", "match_rms_adamw"), \
            'adjust_lr_fn must be None, "original" or "match_rms_adamw"'
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum,
                                      nesterov=nesterov, ns_coefficients=tuple(ns_coefficients),
                                      eps=eps, ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn,
                                      master_weights=master_weights))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2:
                self.param_groups.pop()
                raise AssertionError('Muon takes matrices; give the other parameters to AdamW')

    @torch.no_grad()
    def step(self, closure=None):
        """One step for every matrix that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                assert p.grad is None or not p.grad.is_sparse, 'Muon does not take sparse gradients'
        for group in self.param_groups:
            # one call for the matrices of one type and device
            calls = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                    if p.dtype != torch.float32 and group["master_weights"]:
                        state["master"] = p.detach().float()
                calls.setdefault((p.dtype, p.device, "master" in state), []).append((p, state))
            for (_, _, master), found in calls.items():
                muon_step([p for p, _ in found], [p.grad for p, _ in found],
                          [s["momentum_buffer"] for _, s in found], group["lr"], group["weight_decay"],
                          group["momentum"], group["nesterov"], group["ns_coefficients"], group["eps"],
                          group["ns_steps"], group["adjust_lr_fn"],
                          [s["master"] for _, s in found] if master else None)
        return loss
