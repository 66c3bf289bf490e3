"""AdamW over many tensors at once, with states in 32 bits or in 8.

``adamw_step`` is the operator: one step over lists of tensors in one launch.
``AdamW`` is the optimizer around it, for the parameters of ``fp8_linear``,
``fp8_grouped_linear`` and the norms. States in 8 bits are e4m3 codes of the
first moment and of the second's root with a scale for each 128 elements: 2.06
bytes a parameter in the place of 8. No counterpart in the reference, which is
forward only (src/cutie/rms_norm/bench.py).
"""

from __future__ import annotations

import torch

from .ops import FP8_DTYPE, require_binding


def adamw_state(param: torch.Tensor, bits: int = 32):
    """A state of zeros for ``param``: a float32 tensor of its shape, or (codes, scales) for ``bits`` = 8."""
    if bits == 32:
        return torch.zeros_like(param, dtype=torch.float32, memory_format=torch.contiguous_format)
    if bits != 8:
        raise ValueError(f"states have 32 or 8 bits, got {bits}")
    codes = torch.zeros(param.shape, dtype=torch.uint8, device=param.device).view(FP8_DTYPE)
    return codes, torch.zeros(-(-param.numel() // 128), dtype=torch.float32, device=param.device)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.0, grad_scale: torch.Tensor | None = None, seed: int = 0) -> None:
    """One step of AdamW over lists of tensors, in place, on the current stream.

    params: contiguous bf16, fp16 or fp32 tensors of one dtype; grads: of their
    shapes, of the same dtype, or fp32, or bf16 for fp32 params. exp_avgs,
    exp_avg_sqs: float32 tensors, or pairs (codes, scales) of ``adamw_state(p,
    8)``, where exp_avg_sqs hold the second moment's root. For each element, in
    fp32: g' = g grad_scale, m' = b1 m + (1 - b1) g', v' = b2 v + (1 - b2) g'^2,
    p' = p (1 - lr weight_decay) - lr / (1 - b1^step) m' / (sqrt(v' / (1 -
    b2^step)) + eps). Codes are rounded at random (the mean is kept: small
    steps of a moment are not lost), by a hash of seed, step, the tensor's place in
    the list and the element: the same call gives the same bits. An infinite
    gradient leaves NaN in its group of 128 states.

    step counts from 1: an int, or an int64 tensor on the GPU that is read when the
    kernel runs (for captured steps); lr: a number or a float32 tensor likewise;
    grad_scale: a float32 tensor, what clipping leaves of the gradients.
    Parameters and states that share memory with one another, or with a
    gradient, are refused.
    """
    beta1, beta2 = betas
    require_binding().adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, float(beta1), float(beta2),
                                 float(eps), float(weight_decay), grad_scale, int(seed))


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is one launch for each dtype of parameters (``adamw_step``).

    state_bits: 32, or 8 for e4m3 codes of both moments. ``capturable`` keeps
    the step count on the GPU, so that a step may be captured into a CUDA graph and
    replayed; lr may then be a float32 tensor on the GPU that the program
    changes; the step before the capture makes the states.
    ``step(grad_scale=...)`` takes the factor of a clipped norm. Parameters
    without a gradient are left as they are. Refused are sparse gradients and
    parameters that are not contiguous; a refused step does not count for the
    parameters that it leaves as they were.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, seed: int = 0, capturable: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not isinstance(lr, torch.Tensor) and not lr >= 0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"eps and weight_decay must not be negative, got {eps}, {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      seed=seed, capturable=capturable))

    def load_state_dict(self, state_dict):
        """As torch's, but states keep their own dtypes (torch casts them to the parameters')."""
        super().load_state_dict(state_dict)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        own = [(p, group) for group in self.param_groups for p in group["params"]]
        shared = {}
        for i, (p, group) in zip(ids, own):
            saved = state_dict["state"].get(i)
            if saved is None:
                continue
            state = {k: v.detach().clone().to(p.device) if isinstance(v, torch.Tensor) else v for k, v in saved.items()}
            step = int(state["step"])
            if group["capturable"]:
                key = (id(group), p.device, step)
                if key not in shared:
                    shared[key] = torch.full((), step, dtype=torch.int64, device=p.device)
                step = shared[key]
            state["step"] = step
            self.state[p] = state

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: torch.Tensor | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for number, group in enumerate(self.param_groups):
            own = [p for p in group["params"] if p.grad is not None]
            if own:
                self._step_group(group, own, grad_scale, int(group["seed"]) + (number << 16))
        return loss

    def _step_group(self, group, own, grad_scale, seed):
        if any(p.grad.is_sparse for p in own):
            raise ValueError("AdamW takes no sparse gradients")
        fresh = [p for p in own if not self.state[p]]
        if torch.cuda.is_current_stream_capturing() and (fresh or not group["capturable"]):
            raise RuntimeError("a captured step needs capturable=True and one step before it, which makes the states")
        lr = group["lr"] if group["capturable"] else float(group["lr"])
        self._make_states(group, fresh)
        self._count(group, own)
        # a launch for the parameters of one age and of the same dtypes
        lists = {}
        for p in own:
            age = self.state[p]["step"]
            key = (id(age) if group["capturable"] else age, p.dtype, p.grad.dtype, p.device)
            lists.setdefault(key, []).append(p)
        names = ("exp_avg", "exp_avg_sq")
        lists, done = list(lists.values()), 0
        try:
            for ps in lists:
                states = [self.state[p] for p in ps]
                if group["state_bits"] == 8:
                    m, v = ([(s[name], s[name + "_scale"]) for s in states] for name in names)
                else:
                    m, v = ([s[name] for s in states] for name in names)
                adamw_step(ps, [p.grad for p in ps], m, v, step=states[0]["step"], lr=lr, betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"], grad_scale=grad_scale, seed=seed + done)
                done += 1
        except BaseException:
            self._take_back(group, [p for ps in lists[done:] for p in ps])
            raise

    def _make_states(self, group, fresh):
        """Zeros. On the GPU, parameters that begin together share their count."""
        counts = {}
        for p in fresh:
            state = self.state[p]
            for name in ("exp_avg", "exp_avg_sq"):
                value = adamw_state(p, group["state_bits"])
                if group["state_bits"] == 8:
                    state[name], state[name + "_scale"] = value
                else:
                    state[name] = value
            if not group["capturable"]:
                state["step"] = 0
            else:
                if p.device not in counts:
                    counts[p.device] = torch.zeros((), dtype=torch.int64, device=p.device)
                state["step"] = counts[p.device]

    def _sharers(self, group, own):
        """For each count on the GPU that parameters of `own` have: those of them, and all of the group's that have it."""
        sharers, now = {}, {}
        for p in group["params"]:
            if self.state[p]:
                sharers.setdefault(id(self.state[p]["step"]), []).append(p)
        for p in own:
            now.setdefault(id(self.state[p]["step"]), []).append(p)
        return [(ps, sharers[key]) for key, ps in now.items()]

    def _add(self, ps, sharers, n):
        step = self.state[ps[0]]["step"]
        if len(ps) < len(sharers):  # some stay behind: the others count on their own from here
            step = step.clone()
            for p in ps:
                self.state[p]["step"] = step
        step.add_(n)

    def _count(self, group, own):
        if not group["capturable"]:
            for p in own:
                self.state[p]["step"] += 1
            return
        shared = self._sharers(group, own)
        if any(len(ps) < len(all_) for ps, all_ in shared) and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured step needs a gradient for every parameter that has had the same steps")
        for ps, all_ in shared:
            self._add(ps, all_, 1)

    def _take_back(self, group, own):
        """Parameters whose step was refused have not made it."""
        if not group["capturable"]:
            for p in own:
                self.state[p]["step"] -= 1
        elif not torch.cuda.is_current_stream_capturing():  # a capture that fails has counted nothing
            for ps, all_ in self._sharers(group, own):
                self._add(ps, all_, -1)
