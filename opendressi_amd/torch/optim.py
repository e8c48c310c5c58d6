"""AdamW over many parameter tensors at once, with moments in 32 or in 8 bits:
the optimizer of what is trained through the surface (vertices, textures,
environments, a neural shader's weights). No counterpart in the reference's
surface, whose optimizer is part of its graph.
"""
from __future__ import annotations

import ctypes as C
import math
from collections import OrderedDict

import numpy as np
import torch
from torch.autograd.graph import increment_version

from .._lib import AdamwSet, AdamwTensor, check, lib
from ..ops import TYPE_CODES, _addr
from .context import RasterizeHipContext

# an entry of the table of parameters (dressi_adamw_tensor)
_ENTRY = np.dtype([("param", "<u8"), ("grad", "<u8"), ("master", "<u8"), ("n", "<u8"),
                   ("state", "<u8"), ("type", "<u4"), ("set", "<u4")])
BLOCK = 32  # elements that share an exponent; a parameter's share is padded to whole ones


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill its memory without gaps or overlaps, in
    whatever order of its dimensions."""
    if t.is_contiguous():
        return True
    step = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != step:
            return False
        step *= size
    return True


def _layout(t: torch.Tensor) -> tuple[tuple, tuple]:
    """(shape, stride): the order in which t's elements lie."""
    return tuple(t.shape), t.stride()


def _row_major(layout: tuple) -> bool:
    return torch.empty_strided(*layout, device="meta").is_contiguous()


def _same_order(p: torch.Tensor, layout: tuple, packed: bool) -> bool:
    """Whether p's elements lie in the order of `layout`; packed: that order is
    row-major, in which another shape changes nothing."""
    if packed and p.is_contiguous():
        return True
    shape, stride = layout
    return p.shape == shape and (p.stride() == stride or all(
        n == 1 or a == b for n, a, b in zip(shape, p.stride(), stride)))


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) in one launch for up to 64 tensors.

    Per element, with gradient g and step t of its parameter:

        m = m beta1 + g (1 - beta1)
        v = v beta2 + g^2 (1 - beta2)
        p = p (1 - lr weight_decay)
            - m / (sqrt(v) / sqrt(1 - beta2^t) + eps) lr / (1 - beta1^t)

    `params` is an iterable of parameters or of groups with their own lr,
    betas, eps and weight_decay. Parameters are float32, bfloat16 or float16
    on the context's device, densely stored, no two in the same memory (a step
    takes them all at once); they are updated in place, in
    float32, on torch's current stream.

    state_bits 32 keeps the moments in float32; 8 keeps them in a byte each,
    with a scale byte for every 32 (2.06 bytes an element in place of 8).
    Their rounding is random, from a hash of element, step and `seed`, and
    right on average, so that the slow second moment still moves; the same
    seed gives the same bits. A gradient that is not finite makes the moments
    of its 32 neighbours NaN as well.

    master_weights keeps a float32 copy of 16-bit parameters, of which they
    are roundings; without it a small update of a 16-bit parameter is lost.
    Where such a parameter is written by others between steps (clamped,
    loaded), the copy takes the new value.

    The state of a parameter lies in the order its elements have in memory at
    its first step. Where that order changes later (channels_last), its steps
    go through copies in the old one.

    max_grad_norm multiplies the gradients by
    min(1, max_grad_norm / (norm + 1e-6)), norm the 2-norm over all of them,
    without a host round trip; `grad_norm` then holds the last step's norm.

    A parameter whose grad is None is left as it is, and so is its step.

    capturable keeps the step counts on the device, so that a step can be
    captured into a graph (at the learning rates of the capture); every
    parameter then needs a gradient in every step. A graph holds the state by
    its address: once a step has been captured, groups cannot be added, and
    loaded state has to lie in the order of the present one.

    Hooks registered on the optimizer run; torch's global optimizer hooks do
    not."""

    def __init__(self, ctx: RasterizeHipContext, params, lr: float = 1e-3, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32,
                 max_grad_norm: float | None = None, master_weights: bool = True, seed: int = 0,
                 capturable: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if max_grad_norm is not None and (not 0.0 < max_grad_norm < math.inf or
                                          C.c_float(max_grad_norm).value == 0.0):
            # the step takes it in 32 bits, where zero says not to clip
            raise ValueError(f"max_grad_norm must be above 0, got {max_grad_norm}")
        if isinstance(params, (set, frozenset)):
            raise TypeError("parameters need an order, in which their state lies: not a set")
        self.ctx = ctx
        self.state_bits = state_bits
        self.max_grad_norm = max_grad_norm
        self.master_weights = bool(master_weights)
        self.seed = int(seed) & 0xffffffff
        self.capturable = bool(capturable)
        self._captured = False  # a graph holds the state's addresses
        self.grad_norm = None
        self._params: list[torch.Tensor] = []  # in the order of their shares
        self._steps: list[int] = []
        self._groups: list[dict] = []  # each parameter's
        self._pre_hooks: OrderedDict = OrderedDict()
        self._post_hooks: OrderedDict = OrderedDict()
        # of state_dict and load_state_dict, before and after
        self._save_hooks = OrderedDict(), OrderedDict()
        self._load_hooks = OrderedDict(), OrderedDict()
        self._layouts: list[tuple] = []  # shape and stride of the order its share is in
        self._fresh: set[int] = set()  # those whose share no step or state has touched
        self._expect: list[tuple] = []  # each parameter with its size, type and (unpacked) layout
        self._sets: list[tuple[dict, int]] = []  # each group with the place of its first parameter
        self._even = True  # every group's parameters have taken the same steps
        self._total = 0
        self._moments: tuple[torch.Tensor, torch.Tensor] | None = None
        self._scales: tuple[torch.Tensor | None, torch.Tensor | None] = (None, None)
        self.master = None
        self._scratch = None
        self._counts = self._device_sets = None  # of the sets, where capturable
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    # ---- layout ----

    def add_param_group(self, param_group) -> None:
        """Adds a group; its parameters' state follows the others', at zero."""
        if self._captured:
            raise RuntimeError("AdamW: a step has been captured into a graph, whose replays write "
                               "the state where it is: no group can be added")
        group = dict(param_group)
        if isinstance(group["params"], (set, frozenset)):
            raise TypeError("a group's parameters need an order, in which their state lies: "
                            "not a set")
        group["params"] = [group["params"]] if isinstance(group["params"], torch.Tensor) \
            else list(group["params"])
        for p in group["params"]:
            self._check_param(p)
        _check_apart(self._params + group["params"])
        for k, v in self.defaults.items():
            group.setdefault(k, v)
        _check_hyper(group)
        super().add_param_group(group)
        group = self.param_groups[-1]
        if group["params"]:
            self._sets.append((group, len(self._params)))
        for p in group["params"]:
            self._fresh.add(len(self._params))
            self._layouts.append(_layout(p))
            self._params.append(p)
            self._steps.append(0)
            self._groups.append(group)
        at = 0
        table = (AdamwTensor * len(self._params))()
        view = np.frombuffer(table, dtype=_ENTRY) if len(table) else np.empty(0, _ENTRY)
        for i, p in enumerate(self._params):
            view[i] = (0, 0, 0, p.numel(), at, TYPE_CODES[p.dtype], 0)
            at += _share(p)
        for k, (_, first) in enumerate(self._sets):
            view["set"][first:] = k
        if self.capturable:
            new = torch.zeros(len(self._sets), dtype=torch.int64, device=self.ctx.device)
            if self._counts is not None:
                new[:len(self._counts)] = self._counts
            self._counts = new
            self._device_sets = torch.empty(len(new) * lib.dressi_adamw_set_bytes(),
                                            dtype=torch.uint8, device=self.ctx.device)
        self._grow(at)
        if self.master is not None:
            where = self.master.data_ptr()
            for i, p in enumerate(self._params):
                if p.dtype != torch.float32:
                    view["master"][i] = where
                    where += 4 * _share(p)
        self._expect_layouts()
        self._table, self._view, self._total = table, view, at
        self._fields = view["param"], view["grad"]
        self._hyper = (AdamwSet * len(self._sets))()

    def _expect_layouts(self) -> None:
        """What a step looks for; the layout is None for row-major order."""
        self._expect = [(p, p.numel(), p.dtype, None if _row_major(at) else at)
                        for p, at in zip(self._params, self._layouts)]

    def _check_param(self, p) -> None:
        if not isinstance(p, torch.Tensor):
            raise TypeError(f"a parameter must be a torch.Tensor, got {type(p).__name__}")
        if p.dtype not in TYPE_CODES:
            raise TypeError(f"a parameter must be float32, bfloat16 or float16, got {p.dtype}")
        if p.device != self.ctx.device:
            raise ValueError(f"a parameter is on {p.device}, the context on {self.ctx.device}")
        if not _dense(p):
            raise ValueError(f"a parameter of shape {tuple(p.shape)} and strides {p.stride()} "
                             "is not densely stored")

    def _grow(self, total: int) -> None:
        """State for `total` elements: what is there, then zeros (and the new
        16-bit parameters' master copies)."""
        dev = self.ctx.device

        def grown(t, n, dtype):
            new = torch.zeros(n, dtype=dtype, device=dev)
            if t is not None:
                new[:t.numel()] = t
            return new

        kind = torch.float32 if self.state_bits == 32 else torch.uint8
        m, v = self._moments or (None, None)
        self._moments = grown(m, total, kind), grown(v, total, kind)
        if self.state_bits == 8:
            self._scales = tuple(grown(s, total // BLOCK, torch.uint8) for s in self._scales)
        narrow = [p for p in self._params if p.dtype != torch.float32]
        if self.master_weights and narrow:
            old = 0 if self.master is None else self.master.numel()
            self.master = grown(self.master, sum(map(_share, narrow)), torch.float32)
            at = 0
            for p in narrow:
                if at >= old:
                    self.master[at:at + p.numel()] = _flat(p.detach())
                at += _share(p)
        if self._scratch is None:
            self._scratch = torch.empty(lib.dressi_adamw_scratch(), dtype=torch.uint8, device=dev)
            if self.max_grad_norm is not None:
                self.grad_norm = torch.zeros((), device=dev)

    # ---- the step ----

    def step(self, closure=None):
        """One step with the parameters' present gradients; returns the
        closure's loss, if there is a closure."""
        if not self._pre_hooks and not self._post_hooks:
            return self._step(closure)
        args, kwargs = (closure,), {}
        for hook in list(self._pre_hooks.values()):
            new = hook(self, args, kwargs)
            if new is not None:
                args, kwargs = new
        loss = self._step(*args, **kwargs)
        for hook in list(self._post_hooks.values()):
            hook(self, args, kwargs)
        return loss

    # torch would wrap step for its hooks and profiler label, 7 us a call; a torch that does not
    # know this mark wraps it all the same
    step.hooked = True

    def register_step_pre_hook(self, hook):
        """hook(optimizer, args, kwargs) before each step; it may return new
        (args, kwargs). Returns a handle whose remove() takes it out."""
        return _register(self._pre_hooks, hook)

    def register_step_post_hook(self, hook):
        """hook(optimizer, args, kwargs) after each step."""
        return _register(self._post_hooks, hook)

    def register_state_dict_pre_hook(self, hook, prepend: bool = False):
        """hook(optimizer) before each state_dict."""
        return _register(self._save_hooks[0], hook, prepend)

    def register_state_dict_post_hook(self, hook, prepend: bool = False):
        """hook(optimizer, state_dict) after each state_dict; it may return
        another dict."""
        return _register(self._save_hooks[1], hook, prepend)

    def register_load_state_dict_pre_hook(self, hook, prepend: bool = False):
        """hook(optimizer, state_dict) before each load_state_dict, with a
        shallow copy of the dict; it may return another."""
        return _register(self._load_hooks[0], hook, prepend)

    def register_load_state_dict_post_hook(self, hook, prepend: bool = False):
        """hook(optimizer) after each load_state_dict."""
        return _register(self._load_hooks[1], hook, prepend)

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_current_stream_capturing()
        if capturing and not self.capturable:
            raise RuntimeError("AdamW.step cannot be captured into a graph without "
                               "capturable=True: its step count is the host's")
        dev = self.ctx.device.index
        kept = []  # copies that the launch reads
        moved = []  # parameters in another order than their state, with their copies
        live, params, grads = [], [], []
        for i, (p, n, kind, order) in enumerate(self._expect):
            g = p.grad
            if g is None:
                continue
            # a parameter's and its gradient's storage may have been replaced or reordered
            if (g.dtype is not kind or p.dtype is not kind or g.numel() != n or p.numel() != n
                    or g.get_device() != dev or p.get_device() != dev
                    or g.layout is not torch.strided
                    or not (g.is_contiguous() and p.is_contiguous() if order is None else
                            (p.shape, p.stride()) == order and g.stride() == order[1])):
                q, g = self._reorder(i, p, g, n, kind)
                kept.append(g)
                if q is not p:
                    moved.append((p, q))
                    p = q
            live.append(i)
            params.append(p.data_ptr())
            grads.append(g.data_ptr())
        if not live:
            if self.grad_norm is not None:
                self.grad_norm.zero_()  # the norm of nothing
            return loss
        every = len(live) == len(self._expect)
        steps = self._steps
        if every and self._even:
            # all in step: a set for each group, as the table has it
            table, hyper = self._table, self._hyper
            self._fields[0][:], self._fields[1][:] = params, grads
            for e, (g, first) in zip(hyper, self._sets):
                e.lr, e.eps, e.weight_decay = g["lr"], g["eps"], g["weight_decay"]
                e.beta1, e.beta2 = g["betas"]
                e.step = steps[first] + 1
            now = steps if self.capturable else [t + 1 for t in steps]
        elif self.capturable:
            raise RuntimeError("AdamW: a capturable step needs every parameter's gradient")
        else:
            now = list(steps)
            index, sets, of = {}, [], []
            for i in live:
                now[i] += 1
                k = index.setdefault((id(self._groups[i]), now[i]), len(sets))
                if k == len(sets):
                    sets.append((self._groups[i], now[i]))
                of.append(k)
            view = self._view[live].copy()
            view["set"], view["param"], view["grad"] = of, params, grads
            table = (AdamwTensor * len(live)).from_buffer(view)
            hyper = (AdamwSet * len(sets))(*(
                (g["lr"], *g["betas"], g["eps"], g["weight_decay"], t) for g, t in sets))
        if capturing:
            self._captured = True
        ctx = self.ctx
        with ctx.lock:
            ctx._ctx.use_torch_stream()
            check(lib.dressi_adamw_step(
                ctx._ctx.handle, table, len(live), hyper, len(hyper), self.state_bits, self._total,
                self._moments[0].data_ptr(), self._moments[1].data_ptr(),
                _addr(self._scales[0]), _addr(self._scales[1]), self.seed, self.max_grad_norm or 0.0,
                self._scratch.data_ptr(), _addr(self.grad_norm), _addr(self._counts),
                _addr(self._device_sets)))
        if moved:
            with torch.no_grad():
                for p, q in moved:
                    p.copy_(q)
        # written in place: a backward pass over the values before the step has to refuse them
        increment_version(self._params if every else [self._params[i] for i in live])
        self._steps = now
        self._even = self._even and every
        if self._fresh:
            self._fresh.difference_update(live)
        return loss

    def _reorder(self, i: int, p, g, n: int, kind) -> tuple[torch.Tensor, torch.Tensor]:
        """The parameter (a copy, where its order is not its state's) and the
        gradient, both in the state's order; refuses what the kernel cannot
        take."""
        if g.layout is not torch.strided:
            raise RuntimeError("AdamW: sparse gradients are not supported")
        if g.numel() != n or p.numel() != n or g.dtype is not kind or p.dtype is not kind \
                or g.device != self.ctx.device or p.device != g.device:
            raise ValueError(f"parameter {i} or its gradient changed its size, type or device: "
                             f"{p.dtype} {tuple(p.shape)} on {p.device}, {g.dtype} "
                             f"{tuple(g.shape)} on {g.device}")
        layout, there = self._layouts[i], True
        if _same_order(p, layout, self._expect[i][3] is None):
            layout = _layout(p)
        elif not _dense(p):
            raise ValueError(f"parameter {i} is no longer densely stored")
        elif i in self._fresh:
            # zeros, and a master copy of which the kernel takes what is still the parameter's
            layout = self._layouts[i] = _layout(p)
            self._expect[i] = (p, n, kind, None if p.is_contiguous() else layout)
        elif tuple(p.shape) != layout[0]:
            raise ValueError(f"parameter {i} changed its shape from {layout[0]} to "
                             f"{tuple(p.shape)}, and its order")
        else:
            there = False

        def ordered(t):
            if t.stride() == layout[1]:
                return t
            return torch.empty_strided(*layout, dtype=kind, device=t.device).copy_(t)

        with torch.no_grad():
            return p if there else ordered(p), ordered(g)

    # ---- state ----

    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(m, v) of all parameters, flat, in the parameters' order, each
        parameter's share in its memory order (of its first step) and padded with zeros to a
        multiple of 32. With 32-bit state they are the optimizer's own
        float32 buffers, with 8-bit state the values that the codes stand for,
        in bfloat16, which holds them exactly."""
        if self.state_bits == 32:
            return self._moments
        m = torch.empty(self._total, dtype=torch.bfloat16, device=self.ctx.device)
        v = torch.empty_like(m)
        with self.ctx.lock:
            self.ctx._ctx.use_torch_stream()
            check(lib.dressi_adamw_values(
                self.ctx._ctx.handle, self._total, self._moments[0].data_ptr(),
                self._moments[1].data_ptr(), _addr(self._scales[0]), _addr(self._scales[1]),
                m.data_ptr(), v.data_ptr()))
        return m, v

    def state_dict(self) -> dict:
        """Flat state: "step" (one count a parameter), "exp_avg" and
        "exp_avg_sq" as they are kept (with "exp_avg_scale" and
        "exp_avg_sq_scale" in 8 bits), "master" where there is one (the
        16-bit parameters' copies, laid out like the moments), "layout" (the
        shape and stride of each parameter's share), and the groups'
        hyperparameters."""
        for hook in list(self._save_hooks[0].values()):
            hook(self)
        steps = list(self._steps)
        if self.capturable:
            ends = [at for _, at in self._sets[1:]] + [len(steps)]
            for t, (_, a), b in zip(self._counts.tolist(), self._sets, ends):
                steps[a:b] = [t] * (b - a)
        layout = [_layout(p) if p.numel() == n and _same_order(p, at, order is None) else at
                  for (p, n, _, order), at in zip(self._expect, self._layouts)]
        out = {"step": steps, "seed": self.seed, "layout": layout,
               "exp_avg": self._moments[0], "exp_avg_sq": self._moments[1],
               "param_groups": [{k: v for k, v in g.items() if k != "params"}
                                for g in self.param_groups]}
        if self.state_bits == 8:
            out["exp_avg_scale"], out["exp_avg_sq_scale"] = self._scales
        if self.master is not None:
            out["master"] = self.master
        for hook in list(self._save_hooks[1].values()):
            new = hook(self, out)
            out = out if new is None else new
        return out

    def __getstate__(self):
        raise TypeError("an AdamW is not copied or pickled: its context and its flat state are "
                        "its own; take its state_dict to another one")

    def load_state_dict(self, state_dict: dict) -> None:
        """Takes over the state of an optimizer of the same parameters and
        state_bits. "seed", "master" and "param_groups" may be missing: then
        they stay as they are; without "layout" the state is taken to be in
        the parameters' present order. Where a parameter lies in another order
        than its state, its steps go through copies in the state's."""
        state_dict = dict(state_dict)
        for hook in list(self._load_hooks[0].values()):
            new = hook(self, state_dict)
            state_dict = state_dict if new is None else new
        steps = [int(t) for t in state_dict["step"]]
        if len(steps) != len(self._params) or min(steps, default=0) < 0:
            raise ValueError(f"state of {len(steps)} parameters for {len(self._params)}")
        named = {"exp_avg": self._moments[0], "exp_avg_sq": self._moments[1]}
        if self.state_bits == 8:
            named["exp_avg_scale"], named["exp_avg_sq_scale"] = self._scales
        if self.master is not None and "master" in state_dict:
            named["master"] = self.master
        for k, t in named.items():
            src = state_dict[k]
            if src.dtype != t.dtype or src.shape != t.shape:
                raise ValueError(f"{k} must be {t.dtype} {tuple(t.shape)}, got {src.dtype} "
                                 f"{tuple(src.shape)}")
        layouts = self._check_layouts(state_dict.get("layout"))
        if self._captured and not all(
                a == b or _row_major(a) and order is None
                for a, b, (_, _, _, order) in zip(layouts, self._layouts, self._expect)):
            raise ValueError("a step has been captured into a graph, which takes the state in "
                             "the order that it had then")
        groups = state_dict.get("param_groups")
        if groups is not None:
            if len(groups) != len(self.param_groups):
                raise ValueError(f"{len(groups)} groups for {len(self.param_groups)}")
            for g in groups:
                _check_hyper(g)
        ends = [at for _, at in self._sets[1:]] + [len(steps)]
        even = all(len(set(steps[a:b])) == 1 for (_, a), b in zip(self._sets, ends))
        if self.capturable and not even:
            raise ValueError("a capturable optimizer's groups have one step count each")
        seed = int(state_dict.get("seed", self.seed)) & 0xffffffff
        # nothing is refused from here on
        for mine, g in zip(self.param_groups, groups or ()):
            mine.update({k: v for k, v in g.items() if k != "params"})
        for k, t in named.items():
            t.copy_(state_dict[k])
        self._steps, self._even = steps, even
        self._fresh.clear()
        self._layouts = layouts
        self._expect_layouts()
        if self.capturable:
            self._counts.copy_(torch.tensor([steps[a] for _, a in self._sets]))
        self.seed = seed
        for hook in list(self._load_hooks[1].values()):
            hook(self)

    def _check_layouts(self, layouts) -> list[tuple]:
        """A state dict's, one for each parameter and of its shape; None: the
        parameters' own."""
        if layouts is None:
            return [_layout(p) if _dense(p) else at
                    for p, at in zip(self._params, self._layouts)]
        if len(layouts) != len(self._params):
            raise ValueError(f"layouts of {len(layouts)} parameters for {len(self._params)}")
        out = []
        for i, (p, (shape, stride)) in enumerate(zip(self._params, layouts)):
            shape, stride = tuple(shape), tuple(stride)
            if shape != tuple(p.shape):
                raise ValueError(f"state of a parameter {i} of shape {shape}, not "
                                 f"{tuple(p.shape)}")
            if len(stride) != len(shape) or min(stride, default=0) < 0 or \
                    not _dense(torch.empty_strided(shape, stride, device="meta")):
                raise ValueError(f"parameter {i}'s share has strides {stride}")
            out.append((shape, stride))
        return out


def _register(hooks: OrderedDict, hook, prepend: bool = False):
    """Adds a hook; the handle's remove() takes it out."""
    handle = torch.utils.hooks.RemovableHandle(hooks)
    hooks[handle.id] = hook
    if prepend:
        hooks.move_to_end(handle.id, last=False)
    return handle


def _share(p: torch.Tensor) -> int:
    """Elements of the flat buffers that belong to a parameter."""
    return -(-p.numel() // BLOCK) * BLOCK


def _flat(t: torch.Tensor) -> torch.Tensor:
    """A densely stored tensor's elements in memory order."""
    return torch.as_strided(t, (t.numel(),), (1,))


def _check_apart(params) -> None:
    """Refuses a parameter that is there twice, or two that share memory."""
    spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size(), i)
                   for i, p in enumerate(params) if p.numel())
    for (_, end, i), (begin, _, k) in zip(spans, spans[1:]):
        if begin < end:
            raise ValueError(f"parameters {min(i, k)} and {max(i, k)} are the same or share memory")
    if len(set(map(id, params))) != len(params):
        raise ValueError("an empty parameter is there twice")


def _check_hyper(g: dict) -> None:
    b1, b2 = g["betas"]
    for name, v, ok in (("lr", g["lr"], 0.0 <= g["lr"] < math.inf),
                        ("betas", g["betas"], 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0),
                        ("eps", g["eps"], 0.0 <= g["eps"] < math.inf),
                        ("weight_decay", g["weight_decay"],
                         0.0 <= g["weight_decay"] < math.inf)):
        if not ok:
            raise ValueError(f"invalid {name}: {v}")
