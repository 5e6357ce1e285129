"""AdamW over many tensors at once, with 32-bit or 8-bit state.

An mHC-rewired model trains hundreds of tensors of a few values each beside a
few large ones; ``AdamW.step`` is one kernel launch for each type of parameter
in a group (one per 1000 tensors), whatever their number.

The state of a group is one flat buffer a kind, allocated when the group is
added; ``state[p]`` holds views of it.  With ``state_bits=8`` the two moments
take a byte an element each, as 8-bit floats in units of a power of two per
256 elements: ``exp_avg`` of the first moment, ``exp_avg_sq_root`` of the square
root of the second.  They are rounded up or down by a hash of (seed, step,
place), so that a moment's small changes are kept on average; runs with the
same seed are the same bit for bit.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _capi as C
from . import _kernels as K

BLOCK = 256  # elements that share a scale; a tensor's state starts at a multiple of it
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_M32 = 0xFFFFFFFF


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one stretch of memory, each once."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _alike(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one shape have their elements in one order in memory."""
    return all(s == t for n, s, t in zip(a.shape, a.stride(), b.stride()) if n > 1) or not a.numel()


def _apart(params) -> bool:
    """Whether no two of them share memory: blocks of one launch would race for it."""
    spans = sorted((p.data_ptr(), p.numel() * p.element_size()) for p in params if p.numel())
    return all(a + size <= b for (a, size), (b, _) in zip(spans, spans[1:]))


class _States(dict):
    """Optimizer.state: a parameter's views of the flat buffers are made when they are
    first asked for (hundreds of parameters, four buffers each), those of all when the
    state is walked."""

    def __init__(self, owner):
        super().__init__()
        self.owner, self.where = owner, {}

    def __missing__(self, p):
        if p not in self.where:  # a group has been added
            self.where = self.owner._where()
        pack, i = self.where[p]
        self[p] = pack.state_of(i)
        return self[p]

    def _all(self):
        self.where = self.owner._where()
        return [(p, self[p]) for p in self.where]

    def __len__(self):
        return len(self.owner._where())

    def __contains__(self, p):
        return p in self.owner._where()

    def __iter__(self):
        return iter(self.owner._where())

    def keys(self):
        return self.owner._where().keys()

    def values(self):
        return [s for _, s in self._all()]

    def items(self):
        return self._all()

    def get(self, p, default=None):
        return self[p] if p in self else default


class _Pack:
    """The parameters of one group that share a type and a device, and their state."""

    def __init__(self, params, bits: int, master: bool, salt: int):
        self.params, self.bits, self.salt = params, bits, salt
        self.dtype, self.device = params[0].dtype, params[0].device
        self.steps = [0] * len(params)
        sizes = [p.numel() for p in params]
        offsets = [0]
        for s in sizes:
            offsets.append(offsets[-1] + -(-s // BLOCK) * BLOCK)
        total = offsets.pop()
        self.sizes, self.offsets, self.total = sizes, offsets, total
        self._arrays()
        # every gradient must lie in memory as its parameter does
        self.plain = all(p.is_contiguous() for p in params)
        self.strides = [p.stride() for p in params]
        self.code, self.where = C.dtype_code(self.dtype), params[0].get_device()
        zeros = lambda k, dt: torch.zeros(max(k, 1), dtype=dt, device=self.device)[:k]  # noqa: E731
        f8, f32 = torch.float8_e4m3fn, torch.float32
        if bits == 8:
            scales = total // BLOCK
            smallest = torch.finfo(f32).tiny
            self.buffers = {"exp_avg": zeros(total, f8), "exp_avg_scale": zeros(scales, f32),
                            "exp_avg_sq_root": zeros(total, f8),
                            "exp_avg_sq_root_scale": zeros(scales, f32)}
            self.buffers["exp_avg_scale"].fill_(smallest)
            self.buffers["exp_avg_sq_root_scale"].fill_(smallest)
        else:
            self.buffers = {"exp_avg": zeros(total, f32), "exp_avg_sq": zeros(total, f32)}
        if master:
            self.buffers["master"] = zeros(total, f32)
            for p, o in zip(params, offsets):
                self.view("master", p, o).copy_(p.detach())

    def _arrays(self) -> None:
        n = len(self.sizes)
        self.numel = (ctypes.c_int64 * n)(*self.sizes)
        self.off = (ctypes.c_int64 * n)(*self.offsets)
        # written by each step's look at the parameters, read by its launch
        self.p_ptr, self.g_ptr = (ctypes.c_uint64 * n)(), (ctypes.c_uint64 * n)()

    def __getstate__(self) -> dict:
        arrays = ("numel", "off", "p_ptr", "g_ptr")
        state = {k: v for k, v in self.__dict__.items() if k not in arrays}
        # 8-bit floats go as bytes: pickle does not know them
        state["buffers"] = {k: b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b
                            for k, b in self.buffers.items()}
        return state

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self.buffers = {k: b.view(torch.float8_e4m3fn) if b.dtype == torch.uint8 else b
                        for k, b in state["buffers"].items()}
        self._arrays()

    def view(self, key: str, p: torch.Tensor, offset: int) -> torch.Tensor:
        """p's part of a buffer, laid out as p is; of a scale, its blocks."""
        b = self.buffers[key]
        if key.endswith("_scale"):
            return b[offset // BLOCK:offset // BLOCK + -(-p.numel() // BLOCK)]
        return b.as_strided(p.shape, p.stride(), b.storage_offset() + offset)

    def state_of(self, i: int) -> dict:
        return {k: self.view(k, self.params[i], self.offsets[i]) for k in self.buffers}

    def launch(self, group, seed: int, grad_scale) -> None:
        n = len(self.params)
        at = ctypes.addressof
        if self.plain and C.host().gather(self.params, at(self.numel), self.code, self.where,
                                          at(self.p_ptr), at(self.g_ptr)) \
                and self.steps.count(self.steps[0]) == n:
            t = self.steps[0] + 1
            if self.total:
                self._call(group, t, seed, grad_scale, n, self.p_ptr, self.g_ptr, self.numel,
                           self.off)
                C.host().changed(self.params)
                C.host().changed(list(self.buffers.values()))
            self.steps = [t] * n
            return
        # parameters without a gradient, gradients in another order, or an error
        self._check_forms()
        grads = [p.grad for p in self.params]
        grads = [g if g is None or g.layout == torch.strided and not g.is_neg() and
                 g.stride() == p.stride() else self._as_param(p, g)
                 for p, g in zip(self.params, grads)]
        by_step: dict[int, list[int]] = {}  # those of each number of steps in a launch of their own
        for i, g in enumerate(grads):
            if g is not None:
                by_step.setdefault(self.steps[i], []).append(i)
        for t, which in by_step.items():
            k = len(which)
            self._call(group, t + 1, seed, grad_scale, k,
                       (ctypes.c_uint64 * k)(*(self.params[i].data_ptr() for i in which)),
                       (ctypes.c_uint64 * k)(*(grads[i].data_ptr() for i in which)),
                       (ctypes.c_int64 * k)(*(self.numel[i] for i in which)),
                       (ctypes.c_int64 * k)(*(self.offsets[i] for i in which)))
            for i in which:
                self.steps[i] = t + 1
            C.host().changed([*(self.params[i] for i in which), *self.buffers.values()])

    def _check_forms(self) -> None:
        """The kernel goes by the sizes, type, device and layout that the state was made
        for; a parameter may have been given other memory since (``p.data = ...``,
        ``model.half()``)."""
        for p, size, strides in zip(self.params, self.numel, self.strides):
            laid_out = p.is_contiguous() if self.plain else p.stride() == strides
            if not laid_out or (p.numel(), p.dtype, p.device) != (size, self.dtype, self.device):
                raise ValueError("a parameter has another type, device, size or layout than when "
                                 "its optimizer was made")
            g = p.grad
            if g is not None and (g.shape, g.dtype, g.device) != (p.shape, p.dtype, p.device):
                raise ValueError("a gradient does not fit its parameter")

    @staticmethod
    def _as_param(p, g):
        if g.layout != torch.strided:
            raise ValueError("AdamW does not take sparse gradients")
        return torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device=p.device).copy_(g)

    def _call(self, group, t, seed, grad_scale, n, params, grads, numel, offsets):
        b1, b2 = group["betas"]
        b = self.buffers
        second = "exp_avg_sq_root" if self.bits == 8 else "exp_avg_sq"
        key = (seed * 0x9E3779B9 + t * 0x85A308D3 + self.salt * 0x3C6EF372) & _M32
        K.adamw_step(self.device, n, params, grads, numel, offsets, self.dtype, self.bits,
                     b["exp_avg"], b.get("exp_avg_scale"), b[second], b.get(second + "_scale"),
                     b.get("master"), b1, 1.0 - b1, b2, 1.0 - b2,
                     1.0 - group["lr"] * group["weight_decay"], group["lr"] / (1.0 - b1 ** t),
                     1.0 / math.sqrt(1.0 - b2 ** t), group["eps"], grad_scale, key)


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) for CUDA parameters in fp32, fp16 or bf16.

        m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
        p = (1 - lr weight_decay) p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    params: as for torch.optim.AdamW (groups may set lr, betas, eps and
      weight_decay).  Each is dense in memory, in any order of its axes, and none
      shares memory with another of its group.
    state_bits: 32, or 8 for moments of a byte an element.
    master_weights: keep 16-bit parameters in fp32 beside them; updates are made
      on those and the parameter receives the rounded values.  A parameter that has
      been given other values since (a checkpoint) goes on from them.
    seed: of the 8-bit state's rounding.

    A parameter without a gradient is left alone.  A non-finite gradient makes its
    element NaN for good: skip such steps (torch.amp.GradScaler does).  One whose
    square overflows (above 1.8e19) makes v infinite: its element then only decays."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, master_weights: bool = False,
                 seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        self.state_bits, self.master_weights = int(state_bits), bool(master_weights)
        self.seed = int(seed)
        self._packs: list[list[_Pack]] = []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state = _States(self)

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._packs.append(self._build(group, len(self._packs)))
        except Exception:
            self.param_groups.pop()
            raise

    def _build(self, group, index: int) -> list[_Pack]:
        self._check_group(group)
        by: dict = {}
        for p in group["params"]:
            if p.dtype not in _FLOATS:
                raise ValueError(f"unsupported parameter dtype {p.dtype}; expected float32, "
                                 "float16 or bfloat16")
            if p.layout != torch.strided or not _dense(p):
                raise ValueError("a parameter must fill its memory densely, got strides "
                                 f"{p.stride() if p.layout == torch.strided else p.layout}")
            C.require_cuda(p)
            by.setdefault((p.dtype, p.device), []).append(p)
        packs = []
        for k, ((dtype, _), ps) in enumerate(by.items()):
            if not _apart(ps):
                raise ValueError("parameters of a group share memory")
            pack = _Pack(ps, self.state_bits, self.master_weights and dtype != torch.float32,
                         64 * index + k)
            packs.append(pack)
        return packs

    @staticmethod
    def _check_group(group) -> None:
        lr, (b1, b2) = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor):
            raise ValueError("lr must be a number, not a tensor")
        if not lr >= 0.0:
            raise ValueError(f"lr must be >= 0, got {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be in [0, 1), got {(b1, b2)}")
        if not group["eps"] >= 0.0:
            raise ValueError(f"eps must be >= 0, got {group['eps']}")
        if not group["weight_decay"] >= 0.0:
            raise ValueError(f"weight_decay must be >= 0, got {group['weight_decay']}")

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: torch.Tensor | None = None):
        """One update.  grad_scale: a device scalar that the gradients are multiplied by
        (an inverse loss scale, a clipping coefficient), read by the kernel.

        A step cannot be captured in a CUDA graph: replays would repeat its bias
        corrections and its rounding."""
        if grad_scale is not None and not (isinstance(grad_scale, torch.Tensor)
                                           and grad_scale.numel() == 1):
            raise ValueError("grad_scale must be a CUDA tensor of one number, got "
                             + (f"shape {tuple(grad_scale.shape)}"
                                if isinstance(grad_scale, torch.Tensor) else repr(grad_scale)))
        for packs in self._packs:
            for pack in packs:
                with K._on(pack.device):
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("an AdamW step cannot be captured: its count of steps is "
                                           "an argument of the kernel, the same at every replay")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group, packs in zip(self.param_groups, self._packs):
            self._check_group(group)
            for pack in packs:
                pack.launch(group, self.seed, grad_scale)
        return loss

    def state_buffers(self, group: int = 0, dtype: torch.dtype | None = None) -> dict:
        """The flat buffers that hold a group's state (for one parameter type, where the
        group has several), by name.  Each parameter's part starts at a multiple of
        256 elements, in the group's order."""
        packs = [p for p in self._packs[group] if dtype in (None, p.dtype)]
        if len(packs) != 1:
            raise ValueError(f"{len(packs)} buffers match: give the parameters' dtype")
        return packs[0].buffers

    def set_step(self, step: int) -> None:
        """The number of updates already made (of every parameter), for resuming."""
        if step < 0:
            raise ValueError(f"step must be >= 0, got {step}")
        for packs in self._packs:
            for pack in packs:
                pack.steps = [int(step)] * len(pack.params)

    # ----------------------------------------------------- save and resume --
    def __getstate__(self) -> dict:
        """For copies and pickles: what the class keeps, but for the views, which are made
        on use.  Not what others have hung on this instance: a scheduler's wrapped ``step``
        would go on stepping the original."""
        return {k: self.__dict__[k] for k in ("defaults", "param_groups", "state_bits",
                                              "master_weights", "seed", "_packs")}

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        self.state = _States(self)

    def _where(self) -> dict:
        return {p: (pack, i) for packs in self._packs for pack in packs
                for i, p in enumerate(pack.params)}

    def state_dict(self) -> dict:
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        where, state, groups, k = self._where(), {}, [], 0
        for g in self.param_groups:
            ids = list(range(k, k + len(g["params"])))
            k += len(ids)
            groups.append({**{n: v for n, v in g.items() if n != "params"}, "params": ids})
            for i, p in zip(ids, g["params"]):
                pack, at = where[p]
                state[i] = {"step": pack.steps[at], **pack.state_of(at)}
        saved = {"state": state, "param_groups": groups, "state_bits": self.state_bits,
                 "seed": self.seed}
        for hook in self._optimizer_state_dict_post_hooks.values():
            other = hook(self, saved)
            saved = saved if other is None else other
        return saved

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        state_dict = dict(state_dict)  # a hook may change it
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            other = hook(self, state_dict)
            state_dict = state_dict if other is None else other
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("loaded state dict has other parameter groups")
        if state_dict["state_bits"] != self.state_bits:
            raise ValueError(f"loaded state has {state_dict['state_bits']} bits, this optimizer "
                             f"{self.state_bits}")
        where = self._where()
        pairs = [(p, state_dict["state"][i]) for g, s in zip(self.param_groups, groups)
                 for p, i in zip(g["params"], s["params"])]
        for p, saved in pairs:  # all of it is checked before any of it is taken
            own = where[p][0].state_of(where[p][1])
            if set(saved) != {"step", *own} or any(saved[n].shape != v.shape for n, v in own.items()):
                raise ValueError("loaded state does not fit its parameter")
            # scales belong to blocks of memory
            if self.state_bits == 8 and not all(_alike(saved[n], v) for n, v in own.items()):
                raise ValueError("loaded 8-bit state is laid out otherwise than its parameter")
        for p, saved in pairs:
            pack, i = where[p]
            for n, v in pack.state_of(i).items():
                # 8-bit codes are copied as bytes: a cast could round them
                if v.dtype == torch.float8_e4m3fn:
                    v.view(torch.uint8).copy_(saved[n].view(torch.uint8))
                else:
                    v.copy_(saved[n])
            pack.steps[i] = int(saved["step"])
        self.seed = int(state_dict["seed"])
        for g, s in zip(self.param_groups, groups):
            g.update({n: v for n, v in s.items() if n != "params"})
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)
