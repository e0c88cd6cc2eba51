"""The end of a training step: the gradients' global norm and the AdamW step, each over any number
of tensors in a few launches (csrc/optim.hip), with the two states in fp32 or in 8 bits.

The reference keeps torch's AdamW and moves its moments to host memory (solution/adam_host.py);
here the moments stay on the GPU, and the step runs over all tensors at once.  Everything
that changes from step to step (the step count, a clipping norm, a loss scale) is read from
device memory, so a step never waits for the GPU and can be captured into a graph.

    norm = optim.grad_norm(grads)
    optim.adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr=2e-4, norm=norm, max_norm=1.0)

`AdamW` is the torch optimizer around them.  8-bit states are codes of the 8-bit dynamic map, 256
values to a scale: the signed map (quant.dynamic_map) for the first moment, an unsigned one with
a bit more of fraction for the second.
"""

import torch

from . import ops

STATE_BLOCK = 256      # values that share a scale of an 8-bit state
ZERO_SIGNED = 127      # the signed map's code of 0; the unsigned one's is 0


def _on_gpu(tensors, name):
    for t in tensors:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{name} takes GPU tensors")


def _list(tensors):
    return tensors if type(tensors) is list else list(tensors)


def grad_norm(grads, grad_scale=None):
    """The 2-norm over all values of the tensors `grads` (fp32, fp16 or bf16, mixed or not), an
    fp32 scalar tensor on their device; divided by `grad_scale` (one fp32 value on the device,
    the loss scale the gradients still carry) where that is given.  Squares and sums are fp64, in
    a fixed order."""
    grads = _list(grads)
    if not grads:
        raise ValueError("grad_norm takes at least one gradient")
    return ops.lists().grad_norm(grads, grad_scale)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.01, scales=None, norm=None, max_norm=None, grad_scale=None,
               found_inf=None):
    """One AdamW step over the parameters, in place; `step` (one fp32 value on the device, the
    steps so far) goes up by one.

    With c = min(1, max_norm / (norm + 1e-6)) / grad_scale (1 where not given), t the new step and
    g = grad * c:
        m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps)
    Parameters are fp32, fp16 or bf16 (gradients alike), the arithmetic fp32, each parameter
    rounded once.  States are fp32, or with `scales = (exp_avg_scales, exp_avg_sq_scales)` uint8
    codes with one fp32 scale per 256 values in storage order (`zero_state8` makes them); the
    moments' recurrence and the choice of codes are then fp64.  A block of an 8-bit state that
    gets a value which is not finite becomes NaN as a whole.

    norm: `grad_norm` of the (unscaled) gradients; max_norm: the clipping bound, needed with it.
    lr: a number, or one fp32 value on the device.  grad_scale, found_inf: as GradScaler hands
    them to a fused optimizer; found_inf != 0 leaves parameters, states and step as they were."""
    _on_gpu([step], "adamw_step")
    if (norm is None) != (max_norm is None):
        raise ValueError("norm and max_norm are given together or not at all")
    b1, b2 = betas
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError(f"betas must lie in [0, 1), got {betas}")
    if not eps >= 0.0 or not weight_decay >= 0.0 or (max_norm is not None and not max_norm > 0.0):
        raise ValueError(f"eps {eps}, weight_decay {weight_decay}, max_norm {max_norm}")
    lr_dev = lr if isinstance(lr, torch.Tensor) else None
    ms, vs = ([], []) if scales is None else map(_list, scales)
    ops.lists().adamw_step(_list(params), _list(grads), _list(exp_avgs), _list(exp_avg_sqs), ms,
                           vs, step,
                           0.0 if lr_dev is not None else float(lr), lr_dev, float(b1),
                           float(b2), float(eps), float(weight_decay), norm,
                           1.0 if max_norm is None else float(max_norm), grad_scale, found_inf)


@torch.no_grad()
def state_values(codes, scale, signed):
    """The fp32 values of an 8-bit state: uint8 `codes` (any shape) with `scale` fp32
    [ceil(n / 256)]; signed: the first moment's map, else the second's."""
    _on_gpu([codes, scale], "state_values")
    return ops.load().state_values(codes, scale, bool(signed))


def zero_state8(param):
    """(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale) of 8-bit states that stand for
    zeros, for a parameter."""
    blocks = -(-param.numel() // STATE_BLOCK)
    codes = [torch.full_like(param, z, dtype=torch.uint8, memory_format=torch.preserve_format)
             for z in (ZERO_SIGNED, 0)]
    return *codes, *(torch.zeros(blocks, dtype=torch.float32, device=param.device)
                     for _ in range(2))


def _not_captured(p, what):
    """Tensors that a capture makes are made anew by every replay: states would start over."""
    if p.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"AdamW: {what} cannot be captured; take it before the capture")


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update (decoupled weight decay, no amsgrad) on `adamw_step`.

    state_bits 8 keeps the two moments of every parameter of at least `min_8bit_size` values in
    8 bits.  max_grad_norm clips the gradients of all groups by their global norm within the
    step, without a pass of its own over them.  lr may be a one-value fp32 tensor on the device.
    Parameters whose gradient is None are passed over, and their step count with them.
    GradScaler hands its scale and its overflow flag to the step instead of unscaling.
    A step can be captured into a graph once each of its parameters has taken one."""

    _step_supports_amp_scaling = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *,
                 state_bits=32, min_8bit_size=4096, max_grad_norm=None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, got {state_bits}")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr {lr}")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"eps {eps}, weight_decay {weight_decay}")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"max_grad_norm {max_grad_norm}")
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None  # of the last step, where it clips
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, min_8bit_size=min_8bit_size))

    def _new_state(self, p, group):
        if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]:
            names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
            return dict(zip(names, zero_state8(p)))
        return {k: torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
                for k in ("exp_avg", "exp_avg_sq")}

    def _cohorts(self, group):
        """The group's parameters with a gradient, by their step tensor, device and kind of state.
        Parameters that have always stepped together share one step tensor; where only some of
        its owners step now, those get a copy."""
        owners, fresh = {}, {}
        for p in group["params"]:
            st = self.state[p]
            if p.grad is not None:
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW takes no sparse gradients")
                if not st:
                    _not_captured(p, "a parameter's first step")
                    st.update(self._new_state(p, group))
                    if p.device not in fresh:
                        fresh[p.device] = torch.zeros((), dtype=torch.float32, device=p.device)
                    st["step"] = fresh[p.device]
            if st:
                owners.setdefault(id(st["step"]), []).append(p)
        out = []
        for ps in owners.values():
            live = [p for p in ps if p.grad is not None]
            if not live:
                continue
            step = self.state[live[0]]["step"]
            if len(live) < len(ps):
                _not_captured(live[0],
                              "a step of some of the parameters that stepped together so far")
                step = step.clone()
            kinds = {}
            for p in live:
                kinds.setdefault("exp_avg_scale" in self.state[p], []).append(p)
            for i, (bits8, some) in enumerate(kinds.items()):
                own = step if i == 0 else step.clone()  # each launch counts its own step up
                for p in some:
                    self.state[p]["step"] = own
                out.append((bits8, some, own))
        return out

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        grad_scale = getattr(self, "grad_scale", None)
        found_inf = getattr(self, "found_inf", None)
        work = [(group, c) for group in self.param_groups for c in self._cohorts(group)]
        norm = None
        if self.max_grad_norm is not None and work:
            norm = grad_norm([p.grad for _, (_, ps, _) in work for p in ps], grad_scale)
            self.grad_norm = norm
        for group, (bits8, ps, step) in work:
            st = [self.state[p] for p in ps]
            scales = ([s["exp_avg_scale"] for s in st],
                      [s["exp_avg_sq_scale"] for s in st]) if bits8 else None
            adamw_step(ps, [p.grad for p in ps], [s["exp_avg"] for s in st],
                       [s["exp_avg_sq"] for s in st], step, lr=group["lr"],
                       betas=group["betas"], eps=group["eps"],
                       weight_decay=group["weight_decay"], scales=scales, norm=norm,
                       max_norm=self.max_grad_norm, grad_scale=grad_scale, found_inf=found_inf)
        return loss

    def __setstate__(self, state):
        """Groups of another AdamW's checkpoint get this one's own settings."""
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("state_bits", 32)
            group.setdefault("min_8bit_size", 4096)

    def load_state_dict(self, state_dict):
        """As Optimizer's, but states keep their own types (Optimizer would give them the
        parameter's), and parameters with the same step count share one step tensor again."""
        super().load_state_dict(state_dict)
        saved, steps = state_dict["state"], {}
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        group_of = {p: k for k, g in enumerate(self.param_groups) for p in g["params"]}
        for i, p in zip(ids, params):
            for name, value in saved.get(i, {}).items():
                if name == "step":
                    kind = (group_of[p], float(value), p.device,
                            "exp_avg_scale" in saved[i])
                    if kind not in steps:
                        steps[kind] = torch.tensor(kind[1], dtype=torch.float32,
                                                   device=p.device)
                    self.state[p][name] = steps[kind]
                elif isinstance(value, torch.Tensor):
                    if not name.endswith("_scale"):  # laid out like the parameter
                        dtype = torch.uint8 if value.dtype == torch.uint8 else torch.float32
                        own = torch.empty_like(p, dtype=dtype,
                                               memory_format=torch.preserve_format)
                        own.copy_(value)
                    else:
                        own = value.detach().clone().to(p.device)
                    self.state[p][name] = own


def patch_trainer():
    """transformers' Trainer takes this AdamW where its arguments name torch's AdamW
    (adamw_torch, adamw_torch_fused) or the 8-bit one (adamw_8bit, adamw_bnb_8bit) and ask for
    nothing else of it; returns whether transformers' Trainer is importable."""
    try:
        from transformers import Trainer
    except Exception:
        return False
    original = Trainer.get_optimizer_cls_and_kwargs
    if getattr(original, "_mindx_adamw", False):
        return True

    def get_optimizer_cls_and_kwargs(args, model=None):
        name = getattr(args.optim, "value", args.optim)
        if name not in ("adamw_torch", "adamw_torch_fused", "adamw_8bit", "adamw_bnb_8bit") or \
                getattr(args, "optim_args", None) or not torch.cuda.is_available():
            return original(args, model)
        return AdamW, {"lr": args.learning_rate, "betas": (args.adam_beta1, args.adam_beta2),
                       "eps": args.adam_epsilon, "state_bits": 8 if "8bit" in name else 32}

    get_optimizer_cls_and_kwargs._mindx_adamw = True
    get_optimizer_cls_and_kwargs._mindx_original = original
    Trainer.get_optimizer_cls_and_kwargs = staticmethod(get_optimizer_cls_and_kwargs)
    return True
