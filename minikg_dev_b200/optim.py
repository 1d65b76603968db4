"""AdamW over many tensors in one launch, with the moments held in 32 or in 8 bits.

``AdamW`` updates what a rule model trains: the producer's embeddings, LSTMs and linear layer (dozens
of small tensors) and the facts' scores (one tensor of every fact).  It is a
``torch.optim.Optimizer`` (parameter groups, learning-rate schedulers, ``zero_grad``, closures,
step hooks), and a step is one ``mkg_adamw_step`` call per group and pair of element types, that is
one launch for up to 800 tensors.  Nothing is copied to the device and the step counts live there, so
a step can be captured in a CUDA graph (``proof.ProofRunner.capture(optimizer=...)`` does).

``state_bits=8`` holds each moment in one byte and shares a power of two between 256 values: 2.03
bytes a parameter in place of 8.  First moments have 4 significant bits, second moments 4 over 34
binades; a second moment above 0 is never held as 0.  What is held is the sum in fp64 rounded once; the
update takes the sum in fp32.
"""
from __future__ import annotations

import copy
import ctypes
import math
from collections import Counter, OrderedDict, defaultdict
from itertools import accumulate

import torch
from torch.utils.hooks import RemovableHandle

from . import _native as N

_TYPES = list(N.DTYPES)  # by their numbers
_CODES = ("exp_avg_codes", "exp_avg_scale", "exp_avg_sq_codes", "exp_avg_sq_scale")


def _run(buffer, at, n):
    """``buffer[at:at + n]`` of a flat buffer, in one operation."""
    return torch.as_strided(buffer, (n,), (1,), at)


def _blocks(at, n):
    """The blocks of scales of ``n`` moments that start at ``at``: (first, how many)."""
    return at // N.ADAMW_BLOCK, -(-n // N.ADAMW_BLOCK)


class _Plan:
    """Sizes, offsets into the flat moments and step-count indexes of a group's parameters."""

    def __init__(self, numel, offset, index):
        self.numel, self.offset, self.index = list(numel), list(offset), list(index)
        table = ctypes.c_int64 * len(self.numel)
        self.tables = tuple(table(*v) for v in (self.numel, self.offset, self.index))

    def __reduce__(self):  # ctypes arrays do not pickle
        return _Plan, (self.numel, self.offset, self.index)


class AdamW(torch.optim.Optimizer):
    """``p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)`` on dense,
    contiguous CUDA parameters (float32, bfloat16 or float16; gradients in any of the three), all on
    one device.  Arithmetic is fp32 and each parameter is rounded to its type once.

    Gradients of another type than their parameter's: a 16-bit parameter whose ``grad_dtype`` is torch's default
    gets ``grad_dtype = None`` here, so a program may give it a gradient in 32 bits (autograd's own stay in
    its type); for a float32 parameter the program sets it.

    ``lr`` is a number or a float32 CUDA tensor of one element; a captured step reads the tensor
    at every replay, a number is kept as it was at capture.  Parameters without a gradient are left
    alone and their step count with them.  A step can be captured after ``load_kernels()`` or a first step;
    gradients must then stay where they are (``zero_grad(set_to_none=False)``).  Not offered: sparse or complex gradients, ``amsgrad``,
    ``maximize``; non-contiguous parameters and parameters that share memory are refused.  Two steps
    of one optimizer must not run at the same time.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, got {state_bits}")
        self.state_bits = int(state_bits)
        self._plan = []     # a _Plan per group
        self._buffers = {}  # flat moments, scales, step counts, the ticket word
        self._total = self._tensors = 0
        self._captured = []  # what captured steps read and write, kept as long as the optimizer
        self._before_load, self._after_load = OrderedDict(), OrderedDict()
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    # ------------------------------------------------------------------ parameters and their state
    def _check_group(self, group) -> None:
        lr, (b1, b2), eps, wd = group["lr"], group["betas"], group["eps"], group["weight_decay"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32 or not lr.is_cuda:
                raise ValueError("AdamW: a tensor lr must be one float32 value on the parameters' device")
        elif not (lr >= 0.0 and math.isfinite(lr)):
            raise ValueError(f"AdamW: lr must be finite and not negative, got {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {(b1, b2)}")
        if not (eps >= 0.0 and wd >= 0.0 and math.isfinite(eps) and math.isfinite(wd)):
            raise ValueError(f"AdamW: eps and weight_decay must be finite and not negative, got {eps}, {wd}")

    def add_param_group(self, param_group) -> None:
        before = len(self.param_groups)
        super().add_param_group(param_group)
        try:
            group = self.param_groups[-1]
            self._check_group(group)
            for p in group["params"]:
                if p.dtype not in N.DTYPES:
                    raise TypeError(f"AdamW: parameters must be float32, bfloat16 or float16, got {p.dtype}")
                if p.layout != torch.strided or not p.is_contiguous():
                    raise ValueError("AdamW: parameters must be dense and contiguous")
            every = [p for g in self.param_groups for p in g["params"]]
            for p in group["params"]:
                N.require_cuda(p, "AdamW parameters")
                if p.device != every[0].device:
                    raise ValueError(f"AdamW: parameters on {every[0].device} and {p.device}")
            spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in every if p.numel())
            if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
                raise ValueError("AdamW: parameters share memory")
            if isinstance(group["lr"], torch.Tensor) and every and group["lr"].device != every[0].device:
                raise ValueError(f"AdamW: a tensor lr must be on {every[0].device}, got {group['lr'].device}")
            self._extend(group["params"])
        except Exception:
            del self.param_groups[before:]
            raise
        self._open_gradients(group["params"])

    @staticmethod
    def _open_gradients(params) -> None:
        """16-bit parameters may have gradients of any type; a type that the program has set stays.  float32 ones
        are left alone: torch would no longer widen 16-bit gradients before it adds them up."""
        for p in params:
            if p.dtype != torch.float32 and p.grad_dtype == p.dtype:
                p.grad_dtype = None

    def _extend(self, params) -> None:
        """Room in the flat buffers for one more group; a graph captured before has to be captured again (it
        updates the former moments, which stay allocated)."""
        numel = [p.numel() for p in params]
        room = [-(-n // N.ADAMW_BLOCK) * N.ADAMW_BLOCK for n in numel]
        offset = [self._total + x for x in accumulate(room, initial=0)][:-1]
        plan = _Plan(numel, offset, range(self._tensors, self._tensors + len(numel)))
        total, tensors = self._total + sum(room), self._tensors + len(numel)
        buffers = self._allocated(params[0].device, total, tensors) if params else self._buffers
        self._plan.append(plan)  # from here on nothing needs memory
        self._total, self._tensors, self._buffers = total, tensors, buffers
        if params:
            self._views()

    def _allocated(self, dev, total: int, tensors: int) -> dict:
        """Flat buffers of that many moments and tensors, with what the present ones hold."""
        held = torch.float32 if self.state_bits == 32 else torch.uint8
        want = {"exp_avg": (total, held), "exp_avg_sq": (total, held), "steps": (tensors, torch.int64),
                "ticket": (1, torch.int32)}
        if self.state_bits == 8:
            want |= {k: (total // N.ADAMW_BLOCK, torch.float32) for k in ("exp_avg_scale", "exp_avg_sq_scale")}
        buffers = {}
        for name, (n, dtype) in want.items():
            b = buffers[name] = torch.zeros(max(n, 1), dtype=dtype, device=dev)
            if name in self._buffers and name != "ticket":
                b[:self._buffers[name].numel()].copy_(self._buffers[name])
        return buffers

    def _views(self) -> None:
        """``state[p]``: each parameter's part of the flat buffers."""
        b = self._buffers
        steps = b["steps"].unbind()
        for group, plan in zip(self.param_groups, self._plan):
            for p, n, at, i in zip(group["params"], plan.numel, plan.offset, plan.index):
                m, v = (torch.as_strided(b[k], p.shape, p.stride(), at) for k in ("exp_avg", "exp_avg_sq"))
                if self.state_bits == 32:
                    self.state[p] = {"step": steps[i], "exp_avg": m, "exp_avg_sq": v}
                else:
                    sm, sv = (_run(b[k], *_blocks(at, n)) for k in ("exp_avg_scale", "exp_avg_sq_scale"))
                    self.state[p] = {"step": steps[i], **dict(zip(_CODES, (m, sm, v, sv)))}

    def _state_struct(self, buffers=None) -> N.AdamwState:
        b = buffers or self._buffers
        return N.AdamwState(b["exp_avg"].data_ptr(), b["exp_avg_sq"].data_ptr(), N.ptr(b.get("exp_avg_scale")),
                            N.ptr(b.get("exp_avg_sq_scale")), b["steps"].data_ptr(), b["ticket"].data_ptr(),
                            self._total, self._tensors)

    def __getstate__(self):  # what others attach (hooks, a scheduler's step) stays here, as with torch's optimizers
        return {k: self.__dict__[k] for k in ("defaults", "param_groups", "state_bits", "_plan", "_buffers", "_total",
                                              "_tensors")}

    def __setstate__(self, state) -> None:
        self._captured = []
        self.state, self._before_load, self._after_load = defaultdict(dict), OrderedDict(), OrderedDict()
        super().__setstate__(state)
        if self._buffers:
            self._views()  # unpickled tensors share no memory
        for group in self.param_groups:
            self._open_gradients(group["params"])

    # ------------------------------------------------------------------ the step
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if len(self._plan) != len(self.param_groups):
            raise RuntimeError("AdamW: parameter groups are added with add_param_group")
        for group, plan in zip(self.param_groups, self._plan):
            params = group["params"]
            if len(params) != len(plan.numel):
                raise RuntimeError("AdamW: a group's parameters changed after it was added")
            if params:
                self._launch(group, params, plan)
        return loss

    def load_kernels(self) -> None:
        """Loads what ``step`` launches with the present gradients, without a step: before a capture."""
        for group in self.param_groups:
            kinds = Counter((p.dtype, p.grad.dtype) for p in group["params"] if p.grad is not None)
            for (p_dtype, g_dtype), n in kinds.items():  # the kernel goes by how many tensors there are
                none = (ctypes.c_int64 * n)()
                self._call(group, p_dtype, g_dtype, none, none, none, none, none)

    def _call(self, group, p_dtype, g_dtype, p_at, g_at, numel, offset, index) -> None:
        self._check_group(group)
        dev, lr = self._buffers["steps"].device, group["lr"]
        on_device = isinstance(lr, torch.Tensor)
        if on_device and lr.device != dev:
            raise ValueError(f"AdamW: a tensor lr must be on {dev}, got {lr.device}")
        b1, b2 = group["betas"]
        hyper = N.AdamwParams(0.0 if on_device else float(lr), float(b1), float(b2), float(group["eps"]),
                              float(group["weight_decay"]), lr.data_ptr() if on_device else None, N.DTYPES[p_dtype],
                              N.DTYPES[g_dtype], self.state_bits, 0)
        with N.on_device(dev):
            N.check(N.load().mkg_adamw_step(hyper, self._state_struct(), len(numel), p_at, g_at, numel, offset, index,
                                            N.stream_handle(dev)), "adamw_step")
            if torch.cuda.is_current_stream_capturing():
                self._captured.append((self._buffers, lr, [p.grad for p in group["params"]]))

    def _launch(self, group, params, plan) -> None:
        dev, n = self._buffers["steps"].device, len(params)
        table = ctypes.c_int64 * n
        p_at, g_at, kinds, at = table(), table(), (ctypes.c_int32 * n)(), (ctypes.c_int64 * 2)()
        status = N.gather_gradients()(params, n, dev.index, plan.tables[0], p_at, g_at, kinds, at)
        if status:
            raise self._refusal(status, params[at[0]], dev)
        held = []  # contiguous copies of gradients, until the launch
        if at[1] and 0 <= kinds[0] < 16:
            parts = ((kinds[0], None),)
        else:
            every = list(kinds)
            for i, k in enumerate(every):
                if k >= 16:
                    held.append(params[i].grad.detach().resolve_neg().contiguous())
                    every[i], g_at[i] = k - 16, held[-1].data_ptr()
            parts = [(k, [i for i, other in enumerate(every) if other == k]) for k in sorted(set(every) - {-1})]
        for kind, only in parts:
            tables, updated = (p_at, g_at, *plan.tables), params
            if only is not None and len(only) < n:
                short = ctypes.c_int64 * len(only)
                tables, updated = [short(*(t[i] for i in only)) for t in tables], [params[i] for i in only]
            self._call(group, _TYPES[kind % 4], _TYPES[kind // 4], *tables)
            torch.autograd.graph.increment_version(updated)

    @staticmethod
    def _refusal(status, p, dev) -> Exception:
        if status == 2:
            return RuntimeError("AdamW: gradients must be dense")
        if status == 3:
            return RuntimeError("AdamW: a parameter changed its size or layout, or its gradient has another size")
        if status == 4:
            return RuntimeError(f"AdamW: parameters and gradients must be on {dev}")
        if status == 5:
            return TypeError(f"AdamW: parameters of {p.dtype} with gradients of {p.grad.dtype}")
        return RuntimeError("AdamW: a parameter or gradient without memory of its own")

    # ------------------------------------------------------------------ the moments
    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(exp_avg, exp_avg_sq) of every parameter, in the order of the groups, as flat fp32 arrays in
        which each parameter starts on a multiple of 256 values: the optimizer's own buffers, or the
        values that the 8-bit ones stand for."""
        if not self._buffers:
            return torch.empty(0), torch.empty(0)
        if self.state_bits == 32:
            return self._buffers["exp_avg"][:self._total], self._buffers["exp_avg_sq"][:self._total]
        return self._unpacked(self._buffers)

    def _unpacked(self, buffers):
        dev = buffers["steps"].device
        m, v = (torch.empty(max(self._total, 1), dtype=torch.float32, device=dev) for _ in range(2))
        with N.on_device(dev):
            N.check(N.load().mkg_adamw_unpack(self._state_struct(buffers), m.data_ptr(), v.data_ptr(),
                                              N.stream_handle(dev)), "adamw_unpack")
        return m[:self._total], v[:self._total]

    def state_dict(self):
        """``torch.optim.Optimizer.state_dict`` with the step counts as ``torch.optim.AdamW`` has them (float32
        on the host), which continues from moments in 32 bits."""
        out = super().state_dict()
        steps = self._buffers["steps"].tolist() if self._buffers else []
        out["state"] = {k: {**e, "step": torch.tensor(float(steps[k]), dtype=torch.float32, device="cpu")}
                        for k, e in out["state"].items()}
        return out

    @staticmethod
    def _hooked(hooks, hook, prepend):
        handle = RemovableHandle(hooks)
        hooks[handle.id] = hook
        if prepend:
            hooks.move_to_end(handle.id, last=False)
        return handle

    def register_load_state_dict_pre_hook(self, hook, prepend: bool = False):
        """``hook(optimizer, state_dict)`` before a load; a dict that it returns is loaded instead."""
        return self._hooked(self._before_load, hook, prepend)

    def register_load_state_dict_post_hook(self, hook, prepend: bool = False):
        """``hook(optimizer)`` after a load."""
        return self._hooked(self._after_load, hook, prepend)

    def load_state_dict(self, state_dict) -> None:
        """Loads a state dict of this class or of ``torch.optim.AdamW`` into the buffers in place: moments
        given as fp32 values are rounded to what 8 bits hold, moments given in 8 bits are read as the
        values they stand for.  Parameters without an entry start anew.  Groups take over every key of
        the saved ones, as copies; a tensor ``lr`` is written in place."""
        state_dict = dict(state_dict)  # hooks may replace its entries
        for hook in list(self._before_load.values()):
            given = hook(self, state_dict)
            state_dict = state_dict if given is None else given
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("AdamW: the state dict has other parameter groups")
        dev = self._buffers["steps"].device if self._buffers else None
        rates = []  # the saved groups, copied: keys of others (a scheduler's initial_lr) come along
        for have, new in zip(self.param_groups, groups):
            new = {k: v.detach().to(device=dev, copy=True) if isinstance(v, torch.Tensor) else copy.deepcopy(v)
                   for k, v in new.items() if k != "params"}
            if "betas" in new:
                new["betas"] = tuple(new["betas"])
            rates.append(new)
            merged = have | new
            if isinstance(have["lr"], torch.Tensor):
                merged["lr"] = have["lr"]  # a captured step reads this tensor
            self._check_group(merged)
            if new.get("amsgrad") or new.get("maximize") or (new.get("decoupled_weight_decay") is False
                                                             and merged["weight_decay"]):
                raise ValueError("AdamW: the state dict is of an optimizer with amsgrad, maximize or coupled decay")
        entries = []
        for group, new, plan in zip(self.param_groups, groups, self._plan):
            for p, key, n, at, i in zip(group["params"], new["params"], plan.numel, plan.offset, plan.index):
                e = state_dict["state"].get(key)
                if e is None:
                    continue
                if "exp_avg" not in e and _CODES[0] not in e:
                    raise ValueError("AdamW: a state dict entry without moments")
                names = ("exp_avg", "exp_avg_sq") if "exp_avg" in e else (_CODES[0], _CODES[2])
                if any(e[k].numel() != n for k in names):
                    raise ValueError("AdamW: a state dict entry of another size")
                entries.append((e, n, at, i))
        if self._buffers:
            self._load_moments(entries)
        for have, new in zip(self.param_groups, rates):
            for k, v in new.items():
                if k == "lr" and isinstance(have["lr"], torch.Tensor):
                    have["lr"].copy_(torch.as_tensor(v).reshape(have["lr"].shape))
                elif k != "params":
                    have[k] = v
        for hook in list(self._after_load.values()):
            hook(self)

    def _load_moments(self, entries) -> None:
        """The flat buffers from (entry, size, offset, step-count index) of each parameter that has one."""
        dev = self._buffers["steps"].device
        m, v = (torch.zeros(max(self._total, 1), dtype=torch.float32, device=dev) for _ in range(2))
        codes = {k: torch.zeros(max(self._total, 1), dtype=torch.uint8, device=dev) for k in ("exp_avg", "exp_avg_sq")}
        codes |= {k: torch.zeros(max(self._total // N.ADAMW_BLOCK, 1), dtype=torch.float32, device=dev)
                  for k in _CODES[1::2]}
        codes |= {k: self._buffers[k] for k in ("steps", "ticket")}
        coded = [x for x in entries if "exp_avg" not in x[0]]
        for e, n, at, _ in coded:
            blocks = _blocks(at, n)
            for buffer, name, run in zip(("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"), _CODES,
                                         ((at, n), blocks, (at, n), blocks)):
                _run(codes[buffer], *run).copy_(e[name].reshape(-1))
        if coded:
            m, v = (x.contiguous() for x in self._unpacked(codes))
        counts = [0] * max(self._tensors, 1)
        for e, n, at, i in entries:
            counts[i] = int(e["step"])
        steps = torch.tensor(counts, dtype=torch.int64)
        plain = [x for x in entries if "exp_avg" in x[0]]
        for buffer, name in ((m, "exp_avg"), (v, "exp_avg_sq")):
            if plain:
                torch._foreach_copy_([_run(buffer, at, n) for _, n, at, _ in plain],
                                     [e[name].detach().reshape(-1) for e, *_ in plain])
        if bool((v < 0).any()):
            raise ValueError("AdamW: a state dict entry with negative second moments")
        self._buffers["steps"].copy_(steps)
        if self.state_bits == 32:
            self._buffers["exp_avg"][:self._total].copy_(m[:self._total])
            self._buffers["exp_avg_sq"][:self._total].copy_(v[:self._total])
        else:
            with N.on_device(dev):
                N.check(N.load().mkg_adamw_pack(self._state_struct(), m.data_ptr(), v.data_ptr(),
                                                N.stream_handle(dev)), "adamw_pack")
