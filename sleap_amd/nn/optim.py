"""AdamW for the commands that fit models (tools/train_benchmark_model.py, tools/train_config_models.py) and for networks of token
operators: torch's optimizer interface (parameter groups, schedulers, state_dict) over `ops.adamw_step`, one launch per 128 tensors (108 with amsgrad).

The reference fits with tf.keras.optimizers.Adam(amsgrad=True) (sleap/nn/config/optimization.py, sleap/nn/training.py); without
weight decay this is Adam, with `amsgrad=True` its running maximum."""
import torch

from .. import ops


def _taken(p):
    return isinstance(p, torch.Tensor) and p.is_cuda and p.dtype in (torch.float32, torch.float16, torch.bfloat16) and p.is_contiguous()


class AdamW(torch.optim.Optimizer):
    """m, v (and the running maximum of v with `amsgrad`) are float32 whatever the parameter's type; see `ops.adamw_step`.

    Parameters are contiguous float32 / float16 / bfloat16 CUDA tensors; dense gradients of their type (one of another layout is copied).
    `step()` counts on the host and refuses to be captured into a graph (it would repeat one step count): capture `ops.adamw_step` with
    `step` and `lr` as tensors instead."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False):
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and all(0 <= b < 1 for b in betas)):
            raise ValueError(f"AdamW: lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad, decoupled_weight_decay=True))  # (the last: what a saved state says of itself)

    def add_param_group(self, group):
        params = [group["params"]] if isinstance(group["params"], torch.Tensor) else list(group["params"])
        if len({id(p) for p in params}) != len(params):
            raise ValueError("AdamW: the same parameter twice in a group")
        if group.get("maximize") or not group.get("decoupled_weight_decay", True):
            raise ValueError("AdamW: a group that maximizes, or whose weight decay is not decoupled")
        for p in params:
            if not _taken(p):
                raise ValueError("AdamW: parameters are contiguous float32, float16 or bfloat16 CUDA tensors (there is no CPU fallback)")
        super().add_param_group({**group, "params": params})

    def load_state_dict(self, state_dict):
        """As torch's, but the states keep float32 (torch's casts them to their parameter's type). Takes what torch's Adam and AdamW saved
        (their step is a tensor), unless they maximize or decay otherwise. A state with decay that does not say how it decays (no
        `decoupled_weight_decay` in its groups: older releases of torch, Adam as well as AdamW, and of this class) is refused until the key is
        added."""
        loaded = {}

        def look(_, saved):
            for group in saved["param_groups"]:
                if group.get("maximize"):
                    raise ValueError("AdamW: a state of an optimizer with maximize")
                if group.get("weight_decay") and not group.get("decoupled_weight_decay", False):
                    raise ValueError("AdamW: a state of an optimizer whose weight decay is not decoupled, or that does not say that it is (decoupled_weight_decay=True in its groups)")
            loaded.update(saved)

        def keep(_):
            for group in self.param_groups:
                group["decoupled_weight_decay"] = True  # whatever a state without decay said
            saved = [i for g in loaded["param_groups"] for i in g["params"]]
            for p, i in zip((p for g in self.param_groups for p in g["params"]), saved):
                for name, value in loaded["state"].get(i, {}).items():
                    if name == "step":
                        value = int(value)
                    elif isinstance(value, torch.Tensor):
                        value = value.detach().to(device=p.device, dtype=torch.float32, copy=True).contiguous()
                    self.state[p][name] = value

        # behind the hooks that may change the state, ahead of those that may read what was loaded
        hooks = self.register_load_state_dict_pre_hook(look), self.register_load_state_dict_post_hook(keep, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: step() counts on the host: capture ops.adamw_step with its step and lr as tensors")
        for group in self.param_groups:
            names = ("exp_avg", "exp_avg_sq", "max_exp_avg_sq") if group["amsgrad"] else ("exp_avg", "exp_avg_sq")
            sets = {}  # parameters of one step count step together
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW: dense gradients only")
                s = self.state[p]
                if not s:
                    s["step"] = 0
                for name in names:
                    if name not in s:
                        s[name] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                sets.setdefault(s["step"] + 1, []).append((p, s))
            for count, items in sets.items():
                grads = [p.grad if p.grad.is_contiguous() and not p.grad.is_neg() else p.grad.resolve_neg().contiguous() for p, _ in items]
                m, v, *w = ([s[name] for _, s in items] for name in names)
                ops.adamw_step([p for p, _ in items], grads, m, v, max_exp_avg_sqs=w[0] if w else None, step=count, lr=group["lr"],
                               betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"])
                for _, s in items:
                    s["step"] = count
        return loss


def adam(params, lr):
    """What the fitting commands step with: `AdamW` without decay, which is Adam, on a GPU; torch's Adam on the CPU and
    for parameters that `AdamW` does not take (another type or layout)."""
    params = list(params)
    if all(_taken(p) for p in params):
        return AdamW(params, lr=lr, weight_decay=0.0)
    return torch.optim.Adam(params, lr=lr)
