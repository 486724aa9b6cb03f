"""AdamW over many tensors in one launch, moments in 32 or in 8 bits (include/cp4/adamw.h), and Muon over many
matrices (include/cp4/muon.h).

``AdamW`` and ``Muon`` are the optimizers of a training loop; ``adamw_step`` and ``muon_step`` are the same steps for a
program that keeps its own lists.  All arithmetic is in the HIP library; there is no eager fallback.  AdamW's count
of steps lives on the device, so a step records into a HIP graph and counts its replays.
"""
import torch

from . import capi

BLOCK = 256                      # values that share the scale of their 8-bit moments


def counter(device="cuda"):
    """A new count of steps for ``adamw_step``: [t, beta1^t, beta2^t, 0] in float64."""
    return torch.tensor([0.0, 1.0, 1.0, 0.0], dtype=torch.float64, device=device)


def empty_moments(param, bits=32):
    """(exp_avg, exp_avg_sq, scales) of a tensor before its first step; scales is None for 32 bits."""
    if bits == 32:
        zeros = lambda: torch.zeros(param.shape, dtype=torch.float32, device=param.device)
        return zeros(), zeros(), None
    if bits != 8:
        raise ValueError("moments have 32 or 8 bits")
    blocks = -(-param.numel() // BLOCK)
    return (torch.zeros(param.shape, dtype=torch.int8, device=param.device),
            torch.zeros(param.shape, dtype=torch.uint8, device=param.device),
            torch.zeros(2, blocks, dtype=torch.float32, device=param.device))


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, counter, *, lr, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.01, scales=None, copies=None, max_norm=None, grad_scale=1.0, stream=None):
    """One AdamW step of all ``params`` (contiguous float32, bfloat16 or float16), in place.

    grads: one each, of any of the three types (None: that parameter is left alone).  exp_avgs and
    exp_avg_sqs: float32, or int8 and uint8 with ``scales`` [2, ceil(n / 256)] float32 (first the first
    moment's), as ``empty_moments`` makes them.  counter: see ``counter``.  copies: tensors (or None)
    that receive the new parameters rounded to their type.  ``grad_scale`` multiplies all gradients.
    With ``max_norm`` they are scaled down to that norm together; the norm is returned (a device
    scalar), and a step whose norm is infinite or NaN changes nothing.
    """
    run = capi._native.adamw_step
    args = (params, grads, exp_avgs, exp_avg_sqs, scales, copies, None,
            [(lr, betas[0], betas[1], eps, weight_decay, counter)], max_norm, grad_scale, stream)
    return run(*args) if stream is None else capi._ordered(stream, run, *args)


def moment_values(exp_avgs, exp_avg_sqs, scales, out=None, stream=None):
    """The values that lists of 8-bit moments stand for, as two lists of float32 tensors (``out``: where
    they go)."""
    if out is None:
        make = lambda: [torch.empty(m.shape, dtype=torch.float32, device=m.device) for m in exp_avgs]
        if stream is not None:
            return capi._ordered(stream, lambda: moment_values(exp_avgs, exp_avg_sqs, scales, (make(), make())))
        out = make(), make()
    capi._native.adamw_moments(exp_avgs, exp_avg_sqs, scales, out[0], out[1], False, stream)
    return out


def set_moments(exp_avgs, exp_avg_sqs, scales, values, stream=None):
    """Rounds ``values`` (as ``moment_values`` gives them) into lists of 8-bit moments."""
    capi._native.adamw_moments(exp_avgs, exp_avg_sqs, scales, values[0], values[1], True, stream)


class AdamW(torch.optim.Optimizer):
    """AdamW, all parameters of a group in one launch (one for every 75 of the same types, 57
    with 8-bit moments).

    state_bits: 32, or 8 for the moments of parameters of at least ``min_8bit_size`` values.
    masters: 16-bit parameters are copies of float32 ones that the optimizer keeps (``True``) or
    are stepped in their own 16 bits.  max_norm: all gradients together are scaled down to this norm;
    ``step`` returns nothing then, the norm is ``last_norm``, and a step whose norm is not finite
    changes nothing.  Groups may have rates of their own (lr, betas, eps, weight_decay).

    Steps are counted for each parameter, from its own first gradient on and only where it has one.  Parameters of a
    group whose counts have parted are launched apart."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32,
                 min_8bit_size=4096, masters=True, max_norm=None):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("lr, eps and weight_decay must be 0 or more, the betas in [0, 1)")
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm must be above 0")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits, self.min_8bit_size = state_bits, min_8bit_size
        self.masters, self.max_norm, self.last_norm = masters, max_norm, None

    def __getstate__(self):
        """What a copy or a pickle takes along (torch's optimizers keep all of theirs in groups)."""
        own = ("state_bits", "min_8bit_size", "masters", "max_norm", "last_norm")
        return {**super().__getstate__(), **{k: getattr(self, k) for k in own}}

    def _state(self, p):
        s = self.state[p]
        if not s:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: a parameter's first step makes its state, and a replay would make it anew; take "
                                   "that step before the capture")
            bits = 8 if self.state_bits == 8 and p.numel() >= self.min_8bit_size else 32
            s["exp_avg"], s["exp_avg_sq"], scales = empty_moments(p, bits)
            if scales is not None:
                s["scales"] = scales
            if self.masters and p.dtype != torch.float32:
                s["master"] = p.detach().float()
        return s

    def _count(self, states, idle):
        """Gives each of ``states`` (of a group's parameters that are about to step) the count of its own steps
        and returns the counts and whose is whose.  Parameters that have always stepped together share one, a launch
        between them; one that others keep as it is (``idle``: the ids of those) is copied for the ones that go on."""
        counts, place, of = [], {}, []
        for s in states:
            old = s.get("counter")
            k = place.get(id(old))
            if k is None:
                new = old
                if old is None:
                    new = counter(s["exp_avg"].device)
                elif id(old) in idle:
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: parameters that have stepped together so far part here; take such a "
                                           "step before the capture, a replay would repeat the copy of their count")
                    new = old.clone()
                k = place[id(old)] = len(counts)
                counts.append(new)
            if old is not counts[k]:
                s["counter"] = counts[k]
            of.append(k)
        idle.update(map(id, counts))                                 # (another group's parameters do not share them)
        return counts, of

    @torch.no_grad()
    def step(self, closure=None, grad_scale=1.0):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        params, grads, ms, vs, scales, copies, of, groups = [], [], [], [], [], [], [], []
        idle, parts = set(), []
        for group in self.param_groups:
            states = []
            for p in group["params"]:
                g = p.grad
                if g is None:
                    if p in self.state:
                        idle.add(id(self.state[p].get("counter")))
                    continue
                if not p.is_contiguous():
                    raise ValueError("AdamW takes contiguous parameters")
                s = self._state(p)
                states.append(s)
                master = s.get("master")
                params.append(p if master is None else master)
                copies.append(None if master is None else p)
                grads.append(g if g.is_contiguous() else g.contiguous())
                ms.append(s["exp_avg"])
                vs.append(s["exp_avg_sq"])
                scales.append(s.get("scales"))
            parts.append((group, states))
        for group, states in parts:
            counts, whose = self._count(states, idle)
            of += [len(groups) + k for k in whose] if groups else whose
            rates = group["lr"], *group["betas"], group["eps"], group["weight_decay"]
            groups += [(*rates, c) for c in counts]
        if groups:
            self.last_norm = capi._native.adamw_step(params, grads, ms, vs, scales, copies, of, groups,
                                                     self.max_norm, grad_scale, None)
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but every state keeps its own type (torch would cast it to its parameter's).  A state of
        ``torch.optim.AdamW`` is taken as well: its moments as 32-bit ones, its count of steps with the powers of the betas."""
        of = {}                                                      # the saved group of each saved state
        for saved in state_dict["param_groups"]:
            of.update((i, saved) for i in saved["params"])
            if saved.get("amsgrad") or saved.get("maximize"):
                raise ValueError("AdamW: a state with amsgrad or maximize is not this optimizer's")
        for i, s in state_dict["state"].items():
            if s and "counter" not in s and "step" not in s and "counter" not in of.get(i, {}):
                raise ValueError("AdamW: moments without a count of steps")
        super().load_state_dict(state_dict)
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            group.pop("counter", None)                               # (states saved before parameters had their own)
            shared = {}                                              # counts that are equal go on as one
            for i, p in zip(saved["params"], group["params"]):
                if not state_dict["state"].get(i):
                    continue
                state = dict(state_dict["state"][i])
                count = state.pop("counter", saved.get("counter"))
                step = state.pop("step", None)
                if count is None:
                    t, (beta1, beta2) = float(step), group["betas"]
                    count = torch.tensor([t, beta1 ** t, beta2 ** t, 0.0], dtype=torch.float64)
                    state = {k: state[k].float() for k in ("exp_avg", "exp_avg_sq")}
                    if self.masters and p.dtype != torch.float32:
                        state["master"] = p.detach().float()
                key = tuple(count.tolist())
                if key not in shared:
                    shared[key] = count.detach().to(p.device, torch.float64, copy=True)
                self.state[p] = {k: t.detach().to(p.device, copy=True) for k, t in state.items()}
                self.state[p]["counter"] = shared[key]


def muon_step(params, grads, momenta, *, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, eps=1e-7,
              copies=None, stream=None):
    """One Muon step of all ``params`` (contiguous float32, bfloat16 or float16), in place: each matrix along its
    momentum, orthogonalised by ``steps`` Newton-Schulz products (up to 16), times ``lr sqrt(max(1, rows / cols))``.

    A parameter is [..., rows, cols]: a stack of matrices that are orthogonalised one by one (None: its momentum alone is
    updated).  grads: one each, of any of the three types (None: that parameter is left alone).  momenta: float32 of the same shape, zero before the first step.
    copies: tensors (or None) that receive the new parameters rounded to their type.  A matrix whose momentum is not
    finite becomes NaN.  What is written must not overlap another tensor of the call.  A step that is captured into a graph keeps
    the settings it was captured with."""
    run = capi._native.muon_step
    args = (params, grads, momenta, copies, None, lr, momentum, nesterov, weight_decay, eps, steps, stream)
    return run(*args) if stream is None else capi._ordered(stream, run, *args)


def orthogonalize(updates, steps=5, eps=1e-7, out=None, stream=None):
    """The matrices of ``updates`` (a tensor or a list of them, [..., rows, cols] each) with their singular values brought
    to about 1 (0.68 to 1.21) by ``steps`` Newton-Schulz products, each of its own type.  ``out``: where they go, of any of
    the three types (a contiguous matrix itself may be its own)."""
    if isinstance(updates, torch.Tensor):
        return orthogonalize([updates], steps, eps, None if out is None else [out], stream)[0]
    if stream is not None:
        return capi._ordered(stream, _orthogonalize, updates, steps, eps, out, stream)
    return _orthogonalize(updates, steps, eps, out, None)


def _orthogonalize(updates, steps, eps, out, stream):
    if out is None:
        out = [torch.empty(u.shape, dtype=u.dtype, device=u.device) for u in updates]
    updates = [u.detach() if u.is_contiguous() else u.detach().contiguous() for u in updates]
    capi._native.muon_step(None, updates, None, None, out, 0.0, 0.0, False, 0.0, eps, steps, stream)
    return out


class Muon(torch.optim.Optimizer):
    """Muon for parameters that are matrices or stacks of them ([..., rows, cols]): factors, adapters, dense
    layers.  Biases and norms belong to ``AdamW``.  Three launches for up to 72 parameters whose shorter sides round up to
    the same multiple of 16 up to 64, 17 (22 where a long depth is taken in parts) for up to 16 larger ones.  A step that is
    captured into a graph keeps the settings it was captured with.

    masters: 16-bit parameters are copies of float32 ones that the optimizer keeps (``True``) or are stepped in their own
    16 bits.  Groups may have settings of their own (lr, momentum, nesterov, weight_decay, steps, eps)."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, eps=1e-7, masters=True):
        if not (lr >= 0 and weight_decay >= 0 and 0 <= momentum < 1):
            raise ValueError("lr and weight_decay must be 0 or more, momentum in [0, 1)")
        if not eps >= 1e-30 or not 1 <= steps <= 16:
            raise ValueError("eps must be 1e-30 or more, steps 1 to 16")
        self.masters = masters
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, eps=eps))

    def __getstate__(self):
        return {**super().__getstate__(), "masters": self.masters}

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        if any(p.dim() < 2 for p in self.param_groups[-1]["params"]):
            self.param_groups.pop()
            raise ValueError("Muon takes parameters of two dimensions or more; leave the others to AdamW")

    def _state(self, p):
        s = self.state[p]
        if not s:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("Muon: a parameter's first step makes its state, and a replay would make it anew; take "
                                   "that step before the capture")
            s["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            if self.masters and p.dtype != torch.float32:
                s["master"] = p.detach().float()
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params, grads, momenta, copies = [], [], [], []
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if not p.is_contiguous():
                    raise ValueError("Muon takes contiguous parameters")
                s = self._state(p)
                master = s.get("master")
                params.append(p if master is None else master)
                copies.append(None if master is None else p)
                grads.append(g if g.is_contiguous() else g.contiguous())
                momenta.append(s["momentum_buffer"])
            if params:
                capi._native.muon_step(params, grads, momenta, copies, None, group["lr"], group["momentum"], group["nesterov"],
                                       group["weight_decay"], group["eps"], group["steps"], None)
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but every state keeps its own type (torch would cast it to its parameter's).  What is not a state of
        this optimizer is refused before anything of it is taken."""
        if any(k not in saved for saved in state_dict["param_groups"] for k in self.defaults):
            raise ValueError("Muon: a saved group without " + ", ".join(self.defaults))
        for s in state_dict["state"].values():
            if s and not isinstance(s.get("momentum_buffer"), torch.Tensor):
                raise ValueError("Muon: a state without a momentum")
        super().load_state_dict(state_dict)
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            for i, p in zip(saved["params"], group["params"]):
                state = state_dict["state"].get(i)
                if not state:
                    continue
                kept = {"momentum_buffer": state["momentum_buffer"].detach().to(p.device, torch.float32, copy=True)}
                if self.masters and p.dtype != torch.float32:
                    kept["master"] = state["master"].detach().to(p.device, copy=True) if "master" in state else p.detach().float()
                self.state[p] = kept
