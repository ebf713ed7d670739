"""AdamW over all parameters in one launch, moments in 32 or 8 bits (csrc/tt_adamw.hip).

``AdamW`` is a torch.optim.Optimizer (parameter groups, schedulers, state_dict) for device
parameters of any number and size; ``MultiTensorAdamW`` is the step under it over plain tensors
and their gradients (TwoTowerTrainStep takes it).  The step counts live on the device: a step
captured in a HIP graph advances on every replay (with the learning rate of the capture).
"""
from __future__ import annotations

import copy
import ctypes
from itertools import chain
from typing import Dict, List, Optional, Sequence

import numpy as np
import torch
from torch.optim.optimizer import _global_optimizer_post_hooks as _post_hooks
from torch.optim.optimizer import _global_optimizer_pre_hooks as _pre_hooks

from . import _lib
from ._lib import check, lib, require_device, stream_ptr

_increment_version = torch._C._increment_version  # torch.autograd.graph.increment_version of a list
MAX_TENSORS = 416  # per launch (TT_ADAMW_MAX_TENSORS)
_TENSOR = np.dtype([("p", "u8"), ("exp_avg", "u8"), ("exp_avg_sq", "u8"), ("scale_m", "u8"),
                    ("scale_v", "u8"), ("step", "u8"), ("ticket", "u8"), ("n", "i8"),
                    ("dtype", "i4"), ("blocks", "i4")])  # tt_adamw_tensor


def _round_up(n: int, q: int) -> int:
    return (n + q - 1) // q * q


def _check_state(i: int, s: Dict, n: int) -> None:
    """Refuses entries of a saved state that are not parameter i's, of n elements."""
    for k in ("step", "exp_avg", "exp_avg_sq"):
        if k not in s:
            raise ValueError(f"the state dict is not AdamW's: no {k!r}")
    codes = not torch.as_tensor(s["exp_avg"]).is_floating_point()
    for k in ("exp_avg", "exp_avg_sq"):
        t = torch.as_tensor(s[k])
        if t.numel() != n:
            raise ValueError(f"AdamW state: {k} of parameter {i} has {t.numel()} elements, the "
                             f"parameter {n}")
        if t.is_floating_point() == codes:
            raise ValueError(f"AdamW state: of parameter {i}'s moments one is in codes, one is not")
        if codes:
            sc = s.get(k + "_scale")
            if sc is None or torch.as_tensor(sc).numel() != -(-n // 256):
                raise ValueError(f"AdamW state: {k} of parameter {i} is in codes and needs "
                                 f"{-(-n // 256)} scales")


class MultiTensorAdamW:
    """Moments and launch tables of one list of device tensors (one device).

    exp_avg / exp_avg_sq of all tensors lie in one buffer each: f32 with every tensor at a multiple
    of 64 elements, or 8-bit codes at multiples of 256 with a scale per 256 (f32 buffers too)."""

    def __init__(self, tensors: Sequence[torch.Tensor], state_bits: int = 32):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        self.bits = state_bits
        self.sizes = [t.numel() for t in tensors]
        for i, t in enumerate(tensors):
            self._check(t, f"parameter {i}")
        self.device = dev = tensors[0].device
        self._dev_index = tensors[0].get_device()
        if any(t.device != dev for t in tensors):
            raise ValueError("the parameters of one table must be on one device")
        at = np.concatenate([[0], np.cumsum([_round_up(n, 64) for n in self.sizes])])
        at8 = np.concatenate([[0], np.cumsum([_round_up(n, 256) for n in self.sizes])])
        self.offsets, self.total = at[:-1].tolist(), int(at[-1])
        self._off8 = at8[:-1].tolist()
        if state_bits == 32:
            self.exp_avg = torch.zeros(self.total, dtype=torch.float32, device=dev)
            self.exp_avg_sq = torch.zeros_like(self.exp_avg)
            self.scale_m = self.scale_v = None
        else:
            self.exp_avg = torch.zeros(int(at8[-1]), dtype=torch.int8, device=dev)
            self.exp_avg_sq = torch.zeros(int(at8[-1]), dtype=torch.uint8, device=dev)
            self.scale_m = torch.zeros(int(at8[-1]) // 256, dtype=torch.float32, device=dev)
            self.scale_v = torch.zeros_like(self.scale_m)
        k = len(tensors)
        self.steps = torch.zeros(k, dtype=torch.int64, device=dev)
        self._tickets = torch.zeros(k, dtype=torch.int32, device=dev)
        self._off_dev = torch.tensor(self.offsets, dtype=torch.int64, device=dev)
        # elements a block: 1024 (one pass of its four waves) while that leaves the card fewer
        # than 8192 blocks, at most 16 passes (more saves nothing: the launch is then long)
        total = sum(self.sizes)
        self.chunk = 1024 * min(16, max(1, total // (1024 * 8192)))
        self._n_items = [-(-n // self.chunk) for n in self.sizes]
        self._item0 = np.concatenate([[0], np.cumsum(self._n_items)]).tolist()
        items = np.empty((self._item0[-1], 2), np.int32)
        for i, m in enumerate(self._n_items):
            items[self._item0[i]:self._item0[i + 1], 0] = i
            items[self._item0[i]:self._item0[i + 1], 1] = np.arange(m)
        self._items = torch.from_numpy(items).to(dev)
        self.bind(tensors)

    @staticmethod
    def _check(t, name):
        require_device(t, name)
        if t.dtype not in _lib.DTYPES:
            raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous, got strides {t.stride()}")

    def bind(self, tensors: Sequence[torch.Tensor]) -> None:
        """(Re)builds the device table for the tensors' present addresses (same sizes; after a
        parameter's storage was replaced).  Copies to the device: not inside a graph capture."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: take one step (or load a state) before capturing one in a "
                               "HIP graph: its tables are built then")
        if [t.numel() for t in tensors] != self.sizes:
            raise ValueError("AdamW: a parameter changed its size")
        spans = []
        tab = np.zeros(len(tensors), _TENSOR)
        esz = self.exp_avg.element_size()
        for i, t in enumerate(tensors):
            self._check(t, f"parameter {i}")
            if t.device != self.device:
                raise ValueError(f"parameter {i} is on {t.device}, its moments on {self.device}")
            off = self.offsets[i] if self.bits == 32 else self._off8[i]
            r = tab[i]
            r["p"] = t.data_ptr()
            r["exp_avg"] = self.exp_avg.data_ptr() + off * esz
            r["exp_avg_sq"] = self.exp_avg_sq.data_ptr() + off * esz
            if self.bits == 8:
                r["scale_m"] = self.scale_m.data_ptr() + off // 256 * 4
                r["scale_v"] = self.scale_v.data_ptr() + off // 256 * 4
            r["step"] = self.steps.data_ptr() + 8 * i
            r["ticket"] = self._tickets.data_ptr() + 4 * i
            r["n"], r["dtype"], r["blocks"] = t.numel(), _lib.DTYPES[t.dtype], self._n_items[i]
            if t.numel():
                spans.append((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), i))
        spans.sort()
        for a, b in zip(spans, spans[1:]):
            if b[0] < a[1]:
                raise ValueError(f"parameters {a[2]} and {b[2]} share memory: one step would move "
                                 "it twice")
        with _lib.on_device(tensors[0]):
            new = torch.from_numpy(tab.view(np.uint8).copy()).to(self.device)
            if getattr(self, "_tab", None) is None:
                self._tab = new
            else:  # in place, in stream order: a captured step goes on with the new addresses
                self._tab.copy_(new)
        self.ptrs = [t.data_ptr() for t in tensors]
        self.dtypes = [t.dtype for t in tensors]

    def step(self, grads: Sequence[Optional[torch.Tensor]], lr: float, betas, eps: float,
             weight_decay: float, first: int = 0) -> bool:
        """One step of tensors first .. first + len(grads) - 1 (the others stay); a gradient None
        leaves its tensor and its step count as they are.  True if all moved."""
        sizes, dtypes, dev = self.sizes, self.dtypes, self._dev_index
        with _lib.on_device(self._tab):
            keep = []
            ptrs = []
            for i, g in enumerate(grads, first):
                if g is None or sizes[i] == 0:
                    ptrs.append(None)
                    continue
                if (g.layout is not torch.strided or g.dtype is not dtypes[i]
                        or g.numel() != sizes[i] or g.get_device() != dev):
                    raise ValueError(f"AdamW: the gradient of parameter {i} must be a dense "
                                     f"{dtypes[i]} tensor of {sizes[i]} elements on "
                                     f"{self.device}, got {g.dtype} {tuple(g.shape)} "
                                     f"({g.layout}) on {g.device}")
                if not g.is_contiguous():
                    g = g.detach().contiguous()
                    keep.append(g)
                ptrs.append(g.data_ptr())
            st = stream_ptr()
            for a in range(0, len(ptrs), MAX_TENSORS):
                part = ptrs[a:a + MAX_TENSORS]
                i0, i1 = self._item0[first + a], self._item0[first + a + len(part)]
                check(lib().tt_adamw_step(
                    self._tab.data_ptr(), self._items.data_ptr() + 8 * i0, i1 - i0, first + a,
                    (ctypes.c_void_p * len(part))(*part), len(part), self.chunk, self.bits, lr,
                    betas[0], betas[1], eps, weight_decay, st), "tt_adamw_step")
        return None not in ptrs

    def moments(self, out=None):
        """(exp_avg, exp_avg_sq) of all tensors as f32 buffers, tensor i's at offsets[i]: the state
        itself with 32 bits; decoded with 8 (into the pair ``out`` if given)."""
        if self.bits == 32 and out is None:
            return self.exp_avg, self.exp_avg_sq
        if out is None:
            out = tuple(torch.zeros(self.total, dtype=torch.float32, device=self.device)
                        for _ in range(2))
        for t in out:
            if (t.dtype != torch.float32 or t.numel() != self.total or t.device != self.device
                    or not t.is_contiguous() or t.data_ptr() % 16):
                raise ValueError(f"out must be two contiguous float32 buffers of {self.total} "
                                 f"elements on {self.device}, 16-byte aligned")
        if self.bits == 32:
            out[0].copy_(self.exp_avg)
            out[1].copy_(self.exp_avg_sq)
            return out
        with _lib.on_device(self._tab):
            check(lib().tt_adamw_decode(
                self._tab.data_ptr(), self._items.data_ptr(), self._items.shape[0], self.chunk,
                self._off_dev.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), stream_ptr()),
                "tt_adamw_decode")
        return out

    def state_of(self, i: int, shape) -> Dict[str, torch.Tensor]:
        """Tensor i's entries as views of the buffers."""
        off = self.offsets[i] if self.bits == 32 else self._off8[i]
        n = self.sizes[i]
        s = {"step": self.steps[i], "exp_avg": self.exp_avg[off:off + n].view(shape),
             "exp_avg_sq": self.exp_avg_sq[off:off + n].view(shape)}
        if self.bits == 8:
            b = slice(off // 256, off // 256 + -(-n // 256))
            s["exp_avg_scale"], s["exp_avg_sq_scale"] = self.scale_m[b], self.scale_v[b]
        return s

    def load_state(self, states: Dict[int, Dict]) -> None:
        """Sets the moments and counts of the tensors in ``states`` (index -> entries as state_of
        gives them, or f32 moments as torch.optim.AdamW saves them); the others become zero."""
        for i, s in states.items():
            _check_state(i, s, self.sizes[i])
        full = None
        if self.bits == 8 and any(torch.as_tensor(s["exp_avg"]).is_floating_point()
                                  for s in states.values()):
            full = tuple(torch.zeros(self.total, dtype=torch.float32, device=self.device)
                         for _ in range(2))
            # coded as a whole below; entries that come as codes are set after that
            for i, s in states.items():
                for t, k in zip(full, ("exp_avg", "exp_avg_sq")):
                    src = torch.as_tensor(s[k])
                    if src.is_floating_point():
                        t[self.offsets[i]:self.offsets[i] + self.sizes[i]].copy_(src.reshape(-1))
        for t in (self.exp_avg, self.exp_avg_sq, self.scale_m, self.scale_v, self.steps):
            if t is not None:
                t.zero_()
        if full is not None:
            with _lib.on_device(self._tab):
                check(lib().tt_adamw_encode(
                    self._tab.data_ptr(), self._items.data_ptr(), self._items.shape[0],
                    self.chunk, self._off_dev.data_ptr(), full[0].data_ptr(),
                    full[1].data_ptr(), stream_ptr()), "tt_adamw_encode")
        for i, s in states.items():
            mine = self.state_of(i, (self.sizes[i],))
            mine["step"].fill_(int(float(s["step"])))
            codes = not torch.as_tensor(s["exp_avg"]).is_floating_point()
            if codes and self.bits == 32:  # 8-bit state into 32 bits: the values it stands for
                for k, top, power in (("exp_avg", 127.0, 2), ("exp_avg_sq", 255.0, 4)):
                    q = torch.as_tensor(s[k]).reshape(-1).to(self.device).double()
                    sc = torch.as_tensor(s[k + "_scale"]).to(self.device).double()
                    val = torch.sign(q) * (q.abs() / top) ** power
                    mine[k].copy_(val * sc.repeat_interleave(256)[:q.numel()])
            elif codes or self.bits == 32:
                for k, dst in mine.items():
                    if k != "step":
                        dst.copy_(torch.as_tensor(s[k]).reshape(dst.shape))


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay for device parameters (f32 or bf16), one launch per
    parameter group and step (416 tensors each).

    ``state_bits=8`` keeps both moments in 8-bit codes (2 bytes a parameter instead of 8, one f32
    scale per 256); the moments a code stands for: ``moments``.  bf16 parameters are updated in f32
    and rounded once a step.  Parameters must be contiguous and must not share memory.  state_dict
    holds the moments as they are kept; load_state_dict also takes torch.optim.AdamW's, and either
    width into either."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        self.state_bits = state_bits
        self._tables: List = []  # (MultiTensorAdamW, [(group index, first, params)])
        self._captured = False  # a HIP graph holds a step with these tables
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, group) -> None:
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            self._check_group(g)
            if getattr(self, "_captured", False):
                raise RuntimeError("AdamW: a step of this optimizer was captured in a HIP graph, "
                                   "whose replays would go on with the moments of before: add "
                                   "parameter groups first")
        except Exception:
            self.param_groups.pop()
            raise
        if getattr(self, "_tables", None):  # keep the moments, lay the tables out anew
            self._tables = []
            self._build()

    @staticmethod
    def _check_group(g):
        lr, (b1, b2), eps, wd = g["lr"], g["betas"], g["eps"], g["weight_decay"]
        if isinstance(lr, torch.Tensor):
            raise TypeError("lr must be a number (a tensor would have to be read back every step)")
        if not lr >= 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"Invalid betas: {(b1, b2)}")
        if not eps >= 0.0:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not wd >= 0.0:
            raise ValueError(f"Invalid weight_decay value: {wd}")
        if len({id(p) for p in g["params"]}) != len(g["params"]):
            raise ValueError("a parameter group holds one parameter twice")

    # ------------------------------------------------------------------ tables
    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._tables, self._captured = [], False  # built for the copy's own parameters when needed

    def _build(self) -> None:
        """Tables for the present groups, with the moments that self.state holds."""
        by_dev: Dict = {}
        for gi, g in enumerate(self.param_groups):
            for p in g["params"]:
                require_device(p, "parameter")
                tensors, spans = by_dev.setdefault(p.device, ([], []))
                if not spans or spans[-1][0] != gi:
                    spans.append((gi, len(tensors), []))
                tensors.append(p)
                spans[-1][2].append(p)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: take one step (or load a state) before capturing one in a "
                               "HIP graph: its tables are built then")
        tables = []
        for tensors, spans in by_dev.values():
            t = MultiTensorAdamW([p.detach() for p in tensors], self.state_bits)
            had = {i: self.state[p] for i, p in enumerate(tensors) if self.state.get(p)}
            if had:
                t.load_state(had)
            tables.append((t, spans))
        self._tables = tables
        self.state.clear()
        for t, spans in tables:
            for _, first, ps in spans:
                for j, p in enumerate(ps):
                    self.state[p] = t.state_of(first + j, p.shape)

    def step(self, closure=None):
        """One step of every parameter that has a gradient."""
        if (_pre_hooks or _post_hooks or self._optimizer_step_pre_hooks
                or self._optimizer_step_post_hooks):
            return self._hooked_step(closure)
        return self._step(closure)

    # torch wraps every optimizer's step in a profiler range (some 5 us of host time, as much as the
    # whole launch of a small set); marked as wrapped, step runs the registered hooks itself
    step.hooked = True

    def _hooked_step(self, closure):
        args, kwargs = (self, closure), {}
        for hook in chain(_pre_hooks.values(), self._optimizer_step_pre_hooks.values()):
            new = hook(self, args, kwargs)
            if new is not None:
                args, kwargs = new
        out = self._step(*args[1:], **kwargs)
        for hook in chain(self._optimizer_step_post_hooks.values(), _post_hooks.values()):
            hook(self, args, kwargs)
        return out

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if not self._tables:
            self._build()
        if not self._captured and torch.cuda.is_current_stream_capturing():
            self._captured = True
        for t, spans in self._tables:
            ptrs = [p.data_ptr() for _, _, ps in spans for p in ps]
            dtypes = [p.dtype for _, _, ps in spans for p in ps]
            if ptrs != t.ptrs or dtypes != t.dtypes:
                if self._captured and dtypes != t.dtypes:
                    raise RuntimeError("AdamW: a parameter changed its type after a step was "
                                       "captured in a HIP graph, which reads gradients of the old")
                t.bind([p.detach() for _, _, ps in spans for p in ps])  # a storage was replaced
            for gi, first, ps in spans:
                g = self.param_groups[gi]
                whole = t.step([p.grad for p in ps], g["lr"], g["betas"], g["eps"],
                               g["weight_decay"], first)
                # (written by their addresses: autograd refuses a backward pass over the old values)
                _increment_version(ps if whole else [p for p in ps if p.grad is not None])
        return loss

    # ------------------------------------------------------------------ state
    def moments(self, out=None):
        """(exp_avg, exp_avg_sq) of all parameters as f32 buffers in the groups' order, each
        parameter's at the next multiple of 64 elements (32 bits: the state itself; 8 bits: decoded,
        into the pair ``out`` if given)."""
        if not self._tables:
            self._build()
        if len(self._tables) != 1:
            raise ValueError("moments() needs all parameters on one device; use moments_of")
        return self._tables[0][0].moments(out)

    def moments_of(self, param):
        """(exp_avg, exp_avg_sq) of one parameter in f32, in its shape."""
        if not self._tables:
            self._build()
        for t, spans in self._tables:
            i = 0
            for _, _, ps in spans:
                for p in ps:
                    if p is param:
                        m, v = t.moments()
                        o, n = t.offsets[i], t.sizes[i]
                        return m[o:o + n].view(p.shape), v[o:o + n].view(p.shape)
                    i += 1
        raise ValueError("not a parameter of this optimizer")

    def load_state_dict(self, state_dict: Dict) -> None:
        """Moments, counts and groups (all of their entries, as torch restores them) become the saved
        ones.  A state that does not fit is refused before anything changes."""
        state_dict = state_dict.copy()
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            new = hook(self, state_dict)
            if new is not None:
                state_dict = new
        groups, saved = self.param_groups, state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in saved]:
            raise ValueError("loaded state dict's parameter groups do not match this optimizer's")
        restored = []
        for g, s in zip(groups, saved):
            for key in ("amsgrad", "maximize"):
                if s.get(key):
                    raise ValueError(f"the saved optimizer has {key}=True, which this one does not do")
            new = {**g, **copy.deepcopy({k: v for k, v in s.items() if k != "params"})}
            if isinstance(new["lr"], torch.Tensor):
                new["lr"] = float(new["lr"])
            self._check_group(new)
            restored.append(new)
        ids = [i for g in saved for i in g["params"]]
        params = [p for g in groups for p in g["params"]]
        # (the saved state may be this optimizer's own views: copied before they are overwritten)
        states = {p: {k: v.clone() if isinstance(v, torch.Tensor) else v
                      for k, v in state_dict["state"][i].items()}
                  for i, p in zip(ids, params) if i in state_dict["state"]}
        for i, p in enumerate(params):
            if p in states:
                _check_state(i, states[p], p.numel())
        if not self._tables:
            self._build()
        for g, new in zip(groups, restored):
            g.update(new)
        for t, spans in self._tables:  # in place: a captured step goes on from the loaded state
            at = [p for _, _, ps in spans for p in ps]
            t.load_state({i: states[p] for i, p in enumerate(at) if p in states})
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)
