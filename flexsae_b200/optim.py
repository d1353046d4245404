"""The optimizer step behind the decoder losses: gradient norm, AdamW with 32-bit or 8-bit states,
AdamW on a decoder whose rows are kept at unit length.

The reference ends at the gradients (torch-ext/flex_sae/hierarchical_kernels.py:288-299); its callers
take the step with the optimizer of their choice.  Here one launch updates all tensors of a model:

    from flexsae_b200 import optim
    opt = optim.AdamW([{"params": [w_enc, b_enc, b_dec]},
                       {"params": [w_dec], "unit_rows": True}], lr=1e-4, max_norm=1.0)
    loss.backward()
    opt.step()
    opt.zero_grad()

``AdamW`` is a ``torch.optim.Optimizer`` over four functions that can be called on their own:
``grad_norm``, ``adamw_step``, ``adamw8_step``, ``adamw_unit_rows_step``.  They work in place on lists of
tensors, on the current stream, without a synchronisation; a step's number, its clipping factor and
whether it takes place at all (it does not when the gradient norm is not finite) are decided on the
device, so a step can be captured in a CUDA graph and replayed.  Results are the same bits every time,
so replicas that step on the same gradients stay equal.
"""
from __future__ import annotations

from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _native as nv
from . import losses as _losses

#: elements that share one scale of the 8-bit states
BLOCK = 256
#: types of the 8-bit states: first moment, second moment
STATE8_DTYPES = (torch.float8_e4m3fn, torch.float8_e5m2)

_ADAMW, _ADAMW8, _UNIT_ROWS = 0, 1, 2      # kinds of step in the binding
_Tensors = Sequence[torch.Tensor]
_Masters = Sequence[Optional[torch.Tensor]]


def state8_blocks(numel: int) -> int:
    """Number of scales that go with ``numel`` 8-bit values."""
    return -(-numel // BLOCK)


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.numel() == 0 or all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _step(kind: int, params, grads, exp_avgs, scales, exp_avg_sqs, sq_scales, masters, step, lr, betas, eps, weight_decay, norm,
          max_norm, seed=0) -> None:
    _losses.launch_count += nv.binding().step(kind, params, grads, exp_avgs, scales, exp_avg_sqs, sq_scales, masters, step, lr,
                                              tuple(betas), eps, weight_decay, norm, max_norm, seed)


def grad_norm(grads: _Tensors) -> torch.Tensor:
    """``sqrt(sum of squares)`` over all tensors of a list (float32, bfloat16 or float16, mixed) as a
    0-dim float32 tensor: the ``norm`` of the step functions.  The squares are added in 64 bits in a
    fixed order: the result is reproducible, and finite whenever float32 can hold it."""
    norm, launches = nv.binding().grad_norm(grads)
    _losses.launch_count += launches
    return norm


def adamw_step(params: _Tensors, grads: _Tensors, exp_avgs: _Tensors, exp_avg_sqs: _Tensors, step: torch.Tensor, *,
               lr: Union[float, torch.Tensor], betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.01, masters: Optional[_Masters] = None, norm: Optional[torch.Tensor] = None,
               max_norm: Optional[float] = None) -> None:
    """One AdamW step over lists of tensors, in place:

        g = c grad                       m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    ``params`` (float32, bfloat16 or float16, mixed), ``grads`` of the same types or float32, float32
    states in their parameters' layout.  ``step``: int64 on the device, steps taken so far; t is one
    more, and the call leaves t there.  ``masters``: float32 copies of 16-bit parameters that hold the
    exact values (None where a parameter has none); the parameters are their roundings (to nearest: without a master, a
    16-bit parameter loses changes below half its spacing).  ``lr``: a number, or a float32 tensor on the
    device (which a captured graph follows).  ``norm``: the norm of all gradients, from ``grad_norm``;
    with it c = min(1, max_norm / (norm + 1e-6)), and a norm that is not finite leaves everything as it
    was.  A tensor given twice, or tensors that overlap (``step``, ``lr`` and ``norm`` among them), are refused."""
    _step(_ADAMW, params, grads, exp_avgs, None, exp_avg_sqs, None, masters, step, lr, betas, eps, weight_decay, norm, max_norm)


def adamw8_step(params: _Tensors, grads: _Tensors, exp_avgs: _Tensors, exp_avg_scales: _Tensors, exp_avg_sqs: _Tensors,
                exp_avg_sq_scales: _Tensors, step: torch.Tensor, *, lr: Union[float, torch.Tensor],
                betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                masters: Optional[_Masters] = None, norm: Optional[torch.Tensor] = None, max_norm: Optional[float] = None,
                seed: int = 0) -> None:
    """``adamw_step`` with states of 8 bits: ``exp_avgs`` float8_e4m3fn and ``exp_avg_sqs`` float8_e5m2 in
    their parameters' layout, each with one float32 scale for every ``BLOCK`` elements in memory order
    (``state8_blocks(numel)`` of them; the value is code * scale).  The parameter is computed from the
    new moments before they are rounded; then each goes at random to one of its two neighbours, so that
    the rounding is right on average (rounding to nearest would never move a second moment, which a
    step changes by a thousandth).  The random bits are a function of (seed, t, position in the list,
    element).  A second moment is stored as at least 2^-16 of its scale.  An infinity or a NaN
    stays with its own element (a first moment's infinity as a NaN, which e4m3 has in its place)."""
    _step(_ADAMW8, params, grads, exp_avgs, exp_avg_scales, exp_avg_sqs, exp_avg_sq_scales, masters, step, lr, betas, eps,
          weight_decay, norm, max_norm, seed)


def adamw_unit_rows_step(params: _Tensors, grads: _Tensors, exp_avgs: _Tensors, exp_avg_sqs: _Tensors, step: torch.Tensor, *,
                         lr: Union[float, torch.Tensor], betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                         weight_decay: float = 0.01, masters: Optional[_Masters] = None, norm: Optional[torch.Tensor] = None,
                         max_norm: Optional[float] = None) -> None:
    """``adamw_step`` for decoders [F, D] (contiguous, D up to 8192) whose rows are kept at unit length: the
    gradient's component along its row is taken out first (g -= (g.w / w.w) w), and after the step
    the row is divided by its length.  A row of zeros has no direction and no length: its gradient stays whole, and where the step
    leaves it zeros it is not divided.  An infinity or NaN in a parameter or gradient reaches its row.  Sums over a row are
    held in 32 bits: a row shorter than 2^-55 counts as zeros, one longer than 2^64 is left as it was, with its moments,
    and a gradient whose product with its row passes 2^128 counts as infinite."""
    _step(_UNIT_ROWS, params, grads, exp_avgs, None, exp_avg_sqs, None, masters, step, lr, betas, eps, weight_decay, norm, max_norm)


class AdamW(torch.optim.Optimizer):
    """AdamW over the functions above, as a ``torch.optim.Optimizer``.

    Per parameter group, beside ``lr`` (a number or a float32 tensor on the device), ``betas``, ``eps`` and
    ``weight_decay``: ``state_bits`` (32 or 8), ``master_weights`` (float32 copies of 16-bit parameters in
    the state), ``unit_rows`` (parameters [F, D] kept at unit rows; 32-bit states only) and ``seed`` (8-bit
    states).  ``max_norm`` clips the norm over the gradients of all groups; ``skip_nonfinite`` measures
    that norm without clipping.  With either, a step whose norm is not finite does not take place, and
    ``norm`` holds the norm of the last step (a 0-dim tensor on the device).

    A parameter without a gradient is passed over; its own step count does not move.  All parameters
    live on one device.  A parameter with a master copy is its rounding after every step: who changes one
    changes both.  A step may be captured in a CUDA graph once every parameter has its states, that is
    after a step outside of it (a capture that would have to make them is refused)."""

    def __init__(self, params: Iterable, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, *, state_bits: int = 32, master_weights: bool = False,
                 unit_rows: bool = False, seed: int = 0, max_norm: Optional[float] = None, skip_nonfinite: bool = False):
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        self.max_norm, self.skip_nonfinite = max_norm, skip_nonfinite
        self.norm: Optional[torch.Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights, unit_rows=unit_rows, seed=seed))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_group(group, group["params"])
        except (ValueError, TypeError):
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(group: dict, params: Sequence[torch.Tensor]) -> None:
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {group['state_bits']}")
        if not 0 <= group["seed"] < 2 ** 32:
            raise ValueError(f"seed must be in [0, 2**32), got {group['seed']}")
        if group["unit_rows"] and group["state_bits"] != 32:
            raise ValueError("unit_rows goes with 32-bit states")
        for p in params:
            if p.dtype not in nv.DTYPE_CODES:
                raise TypeError(f"parameters must be float32, bfloat16 or float16, got {p.dtype}")
            if group["unit_rows"] and p.dim() != 2:
                raise ValueError(f"unit rows need [F, D] parameters, got {tuple(p.shape)}")

    def _new_state(self, p: torch.Tensor, group: dict, step: torch.Tensor) -> Dict[str, torch.Tensor]:
        kinds = STATE8_DTYPES if group["state_bits"] == 8 else (torch.float32, torch.float32)
        state = {"step": step, "exp_avg": torch.zeros_like(p, dtype=kinds[0], memory_format=torch.preserve_format),
                 "exp_avg_sq": torch.zeros_like(p, dtype=kinds[1], memory_format=torch.preserve_format)}
        if group["state_bits"] == 8:
            for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                state[name] = torch.zeros(state8_blocks(p.numel()), dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype != torch.float32:
            state["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)
        return state

    def _cohorts(self, group: dict) -> List[List[torch.Tensor]]:
        """The group's parameters with gradients, those that share a step count together."""
        active = [p for p in group["params"] if p.grad is not None]
        new = [p for p in active if not self.state[p]]
        capturing = active and active[0].is_cuda and torch.cuda.is_current_stream_capturing()
        if new:
            if capturing:      # every replay would set them back to zero
                raise RuntimeError("the optimizer's states have to exist before a step is captured: take one step outside of the graph")
            step = torch.zeros((), dtype=torch.int64, device=new[0].device)
            for p in new:
                self.state[p].update(self._new_state(p, group, step))
        if len(active) < len(group["params"]):      # who sits a step out keeps a count of its own
            moving = {id(self.state[p]["step"]) for p in active}
            left: Dict[int, torch.Tensor] = {}         # together, so that they go on in one step
            for p in group["params"]:
                if p.grad is None and self.state.get(p) and id(self.state[p]["step"]) in moving:
                    if capturing:      # every replay would copy the count again
                        raise RuntimeError("a parameter that takes part in steps outside of the captured one has no gradient in it")
                    step = self.state[p]["step"]
                    if id(step) not in left:
                        left[id(step)] = step.clone()
                    self.state[p]["step"] = left[id(step)]
        counts: Dict[int, List[torch.Tensor]] = {}
        for p in active:
            counts.setdefault(id(self.state[p]["step"]), []).append(p)
        return list(counts.values())

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.norm = None
        if self.max_norm is not None or self.skip_nonfinite:
            grads = [p.grad for group in self.param_groups for p in group["params"] if p.grad is not None]
            if grads:
                self.norm = grad_norm(grads)
        for index, group in enumerate(self.param_groups):
            for ps in self._cohorts(group):
                self._step_cohort(index, group, ps)
        return loss

    def _step_cohort(self, index: int, group: dict, ps: List[torch.Tensor]) -> None:
        states = [self.state[p] for p in ps]

        def column(name: str) -> List[Optional[torch.Tensor]]:
            return [s.get(name) for s in states]

        grads, masters = [p.grad for p in ps], column("master")
        kw = dict(lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                  masters=masters if any(t is not None for t in masters) else None, norm=self.norm, max_norm=self.max_norm)
        if group["state_bits"] == 8:
            # groups of one seed, and cohorts of a group at the same count, round independently
            place = next(k for k, p in enumerate(group["params"]) if p is ps[0])
            seed = (group["seed"] + 0x9E3779B9 * index + 0x85EBCA6B * place) % 2 ** 32
            adamw8_step(ps, grads, column("exp_avg"), column("exp_avg_scale"), column("exp_avg_sq"), column("exp_avg_sq_scale"),
                        states[0]["step"], seed=seed, **kw)
        else:
            step = adamw_unit_rows_step if group["unit_rows"] else adamw_step
            step(ps, grads, column("exp_avg"), column("exp_avg_sq"), states[0]["step"], **kw)

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "max_norm": self.max_norm, "skip_nonfinite": self.skip_nonfinite, "norm": None}

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        for group in self.param_groups:                 # a copy pickled by an earlier version knows fewer options
            for name, value in self.defaults.items():
                group.setdefault(name, value)

    def _completed(self, state_dict: dict) -> dict:
        """``state_dict``, its groups with this optimizer's values for the options that they do not have."""
        saved, mine = state_dict["param_groups"], self.param_groups
        if len(saved) != len(mine):                     # refused by the base class
            return state_dict
        own = [{name: group[name] for name in self.defaults} for group in mine]
        return {**state_dict, "param_groups": [{**options, **group} for options, group in zip(own, saved)]}

    @staticmethod
    def _check_names(i: int, state: dict, names: Iterable[str]) -> None:
        missing = [name for name in names if name not in state]
        if missing:
            raise ValueError(f"the state of parameter {i} has no {', '.join(missing)}: it is not one of AdamW")

    def _check_loaded(self, state_dict: dict) -> None:
        """Refuses a state that these steps would not continue: of another rule, without the moments in the group's form, or with
        options that do not go together or with the parameters."""
        if len(state_dict["param_groups"]) != len(self.param_groups):      # refused by the base class
            return
        for group, mine in zip(state_dict["param_groups"], self.param_groups):
            self._check_group(group, mine["params"])
            for name in ("maximize", "amsgrad"):
                if group.get(name):
                    raise ValueError(f"the state was saved with {name}=True, which this optimizer does not have")
            # torch's Adam family says how the decay is applied; of its members only Adam and AdamW know amsgrad
            if "momentum_decay" in group or ("decoupled_weight_decay" in group and "amsgrad" not in group):
                raise ValueError("the state is not one of torch.optim.AdamW: its optimizer follows another rule")
            if not group.get("decoupled_weight_decay", True) and group.get("weight_decay", 0) != 0:
                raise ValueError("the state was saved by an optimizer that adds weight_decay to the gradient (torch.optim.Adam)")
            for i, p in zip(group["params"], mine["params"]):
                state = state_dict["state"].get(i)
                if not state:
                    continue
                eight = group.get("state_bits") == 8
                self._check_names(i, state, ("step", "exp_avg", "exp_avg_sq"))
                for name in ("exp_avg", "exp_avg_sq", "master"):
                    if name in state and state[name].shape != p.shape:
                        raise ValueError(f"{name} of parameter {i} has shape {tuple(state[name].shape)}, the parameter {tuple(p.shape)}")
                kinds = (state["exp_avg"].dtype, state["exp_avg_sq"].dtype)
                if eight and kinds != STATE8_DTYPES:
                    raise TypeError(f"the moments of parameter {i} are {kinds[0]} and {kinds[1]}: a group with 8-bit states takes {STATE8_DTYPES}")
                if not eight and any(k.itemsize < 2 for k in kinds):
                    raise TypeError(f"the moments of parameter {i} are {kinds[0]} and {kinds[1]}: a group with 32-bit states takes neither")
                if eight:
                    self._check_names(i, state, ("exp_avg_scale", "exp_avg_sq_scale"))
                    for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                        if state[name].shape != (state8_blocks(p.numel()),):
                            raise ValueError(f"{name} of parameter {i} has shape {tuple(state[name].shape)}, ({state8_blocks(p.numel())},) goes with it")
                    if not (_same_layout(state["exp_avg"], p) and _same_layout(state["exp_avg_sq"], p)):
                        raise ValueError(f"the 8-bit states of parameter {i} were saved in another memory layout: their scales go with "
                                         f"256 elements that lie side by side (strides {state['exp_avg'].stride()}, the parameter's {p.stride()})")

    def load_state_dict(self, state_dict: dict) -> None:
        """Restores a ``state_dict``, also one of ``torch.optim.AdamW`` for 32-bit states: the states keep their own types
        (the base class would turn them into the parameters'), parameters of a group that stand at the same step
        share their count again, and a group keeps its own value of each option that the saved one does not have.  A state
        of another rule (``maximize``, ``amsgrad``, decay added to the gradient), or with moments of other types than ``state_bits`` has, is refused, with
        nothing changed; so are 8-bit states saved from a parameter of another memory layout."""
        loaded: Dict[str, dict] = {}

        def before(_, state: dict) -> dict:             # behind the hooks of the program, which may replace the state
            state = self._completed(state)
            self._check_loaded(state)
            loaded.update(state)
            return state

        def after(_) -> None:                           # ahead of its hooks, which see the states as they are to be
            self._restore(loaded)

        handles = [self.register_load_state_dict_pre_hook(before), self.register_load_state_dict_post_hook(after, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for handle in handles:
                handle.remove()

    def _restore(self, state_dict: dict) -> None:
        saved_ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [(p, group) for group in self.param_groups for p in group["params"]]
        for i, (p, group) in zip(saved_ids, params):
            for name, value in state_dict["state"].get(i, {}).items():
                if name == "master" and p.dtype == torch.float32:
                    del self.state[p][name]             # the parameter holds its own value
                elif name == "step":
                    self.state[p][name] = torch.as_tensor(value).to(device=p.device, dtype=torch.int64).clone()
                elif name in ("exp_avg_scale", "exp_avg_sq_scale"):
                    self.state[p][name] = value.to(p.device).clone()
                elif name in ("exp_avg", "exp_avg_sq", "master"):
                    dtype = torch.float32 if group["state_bits"] == 32 else value.dtype
                    kept = torch.empty_like(p, dtype=dtype, memory_format=torch.preserve_format)
                    self.state[p][name] = kept.copy_(value)
            if self.state.get(p) and group["master_weights"] and p.dtype != torch.float32 and "master" not in self.state[p]:
                self.state[p]["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)
        for group in self.param_groups:
            counts: Dict[int, torch.Tensor] = {}
            for p in group["params"]:
                if self.state.get(p):
                    step = self.state[p]["step"]
                    self.state[p]["step"] = counts.setdefault(int(step), step)
