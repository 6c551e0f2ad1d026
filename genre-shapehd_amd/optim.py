"""The optimiser of the training commands with a bound on the gradients: Adam whose step takes the global clip with it."""
import torch

from .toolbox.grad_clip.functions.grad_clip import _native, clip_adam_step_


def own_steps(states):
    """the `state` of an optimiser's state_dict with a `step` of its own in every entry (torch.optim.Adam counts in place, and loads
    and saves keep tensors that are shared)"""
    return {k: dict(st, step=st["step"].clone()) if isinstance(st, dict) and torch.is_tensor(st.get("step")) else st for k, st in states.items()}


class ClipAdam(torch.optim.Adam):
    """torch.optim.Adam (state_dicts go from one to the other) on GPU tensors, as if
    torch.nn.utils.clip_grad_norm_(all parameters, max_grad_norm) had run before every step, in a few launches for the whole
    network: the gradients are read twice and never written.  The norm that a step found is left in `grad_norm`, on the GPU.

    Not for capture in a HIP graph: a replay would repeat the step that was captured, its count with it.  The moments are fp32
    whatever the weights' type.  Parameters without a gradient are passed over, as they are there."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, max_grad_norm=None, decoupled_weight_decay=False):
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise ValueError("max_grad_norm must not be negative, got %r" % (max_grad_norm,))
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled_weight_decay=decoupled_weight_decay)
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None

    def __getstate__(self):                                            # (copies and pickles)
        return dict(super().__getstate__(), max_grad_norm=self.max_grad_norm, grad_norm=self.grad_norm)

    def state_dict(self):
        """torch.optim.Adam's (parameters that are stepped together share one `step` here, which stays inside)"""
        out = super().state_dict()
        return dict(out, state=own_steps(out["state"]))

    def load_state_dict(self, state_dict):
        """torch.optim.Adam's too.  torch casts what it loads to the weights' type, in which a resumed run would not be the one that
        was saved (an fp16 second moment is zero below 3e-8): the moments are taken from the given state, in fp32"""
        given = []                                                     # as the hooks leave it
        hooks = [self.register_load_state_dict_pre_hook(lambda _, sd: given.append(sd)),
                 self.register_load_state_dict_post_hook(lambda _: self._keep_moments(given[-1]), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _keep_moments(self, given):
        keys = [k for group in given["param_groups"] for k in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for key, p in zip(keys, params):
            for name in ("exp_avg", "exp_avg_sq"):
                if name in given["state"].get(key, {}) and self.state[p][name].dtype != torch.float32:
                    self.state[p][name] = given["state"][key][name].detach().to(p.device, torch.float32, copy=True)

    def _moments(self, p):
        st = self.state[p]
        if not st:
            st["step"] = torch.tensor(0.0, dtype=torch.float32, device="cpu")
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        return st

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("ClipAdam: a step cannot be captured: its count of steps lives on the host")
        # what is stepped together: the same options and the same number of steps behind it (`step` tensors are shared by those)
        batches, every = [], []
        for group in self.param_groups:
            if any(group.get(k) for k in ("amsgrad", "maximize", "capturable", "differentiable")):
                raise RuntimeError("ClipAdam: amsgrad, maximize, capturable and differentiable are not supported")
            counts, found = {}, {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                st = self._moments(p)
                key = id(st["step"])
                if key not in counts:
                    counts[key] = int(st["step"])
                found.setdefault(counts[key], []).append((p, p.grad, st))
                every.append(p.grad)
            batches += [(group, count, members) for count, members in found.items()]
        if not every:
            return loss
        factor = None
        if self.max_grad_norm is not None:
            self.grad_norm, factor = _native.grad_norm(every, float(self.max_grad_norm), 2)
        for group, count, members in batches:
            params, grads, states = zip(*members)
            params, grads = list(params), list(grads)
            for i in _native.laid_otherwise(params, grads):
                grads[i] = torch.empty_like(params[i]).copy_(grads[i])
            for name in ("exp_avg", "exp_avg_sq"):                     # (moments of weights whose layout has changed, or loaded ones)
                for i in _native.laid_otherwise(params, [s[name] for s in states]):
                    states[i][name] = torch.empty_like(params[i], dtype=torch.float32).copy_(states[i][name])
            clip_adam_step_(params, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], count + 1, lr=float(group["lr"]),
                            betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                            decoupled=group.get("decoupled_weight_decay", False), factor=factor)
            now = torch.tensor(float(count + 1), dtype=torch.float32, device="cpu")
            for s in states:
                s["step"] = now
        return loss


def adam(params, lr, betas, clip_grad=None):
    """the optimiser of the training commands: torch.optim.Adam, or with a bound on the gradients' norm ClipAdam"""
    if clip_grad is None:
        return torch.optim.Adam(params, lr=lr, betas=betas)
    return ClipAdam(params, lr=lr, betas=betas, max_grad_norm=clip_grad)
