"""AdamW over many tensors in few launches, its states in 32 bits or in 8.

``adamw_step`` is the step itself over lists of tensors; ``AdamW`` the optimiser that
holds the states.  The step is a HIP kernel behind the C ABI
(csrc/torch_sequence.cpp, csrc/adamw.hip); there is no torch or CPU fallback.  No
counterpart in the reference, which trains with torch's optimisers.
"""
import torch

from ._native import torch_binding

__all__ = ["adamw_step", "AdamW"]

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


class AdamW(torch.optim.Optimizer):
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
