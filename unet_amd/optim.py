"""K17: ``clip_grad_norm_`` + ``AdamW.step`` of the reference's training loop as two HIP passes.

The reference does (train.py:1553-1559, optimizer arguments train.py:183-193, 2214-2241)::

    torch.nn.utils.clip_grad_norm_(model.parameters(), GRAD_CLIP)      # one norm per parameter GROUP of our optimizer
    optimizer.step()                                                    # torch.optim.AdamW(betas=(0.7596, 0.9203), wd=0)

which torch runs as ~12 launches per group (per-tensor norms, stack + norm, clamp, a multi-tensor scale of every
gradient, four multi-tensor AdamW launches).  ``ClipAdamW`` is a ``torch.optim.Optimizer`` with the same
``param_groups`` / ``state_dict`` layout as ``torch.optim.AdamW`` (``step``, ``exp_avg``, ``exp_avg_sq`` per parameter,
so the reference's checkpoints load) that does the same arithmetic in three launches per group
(``csrc/optim.hip``): partial sums of g², one block for the norm and the clip factor, one pass that
updates p, m, v from the clipped gradient.  The clipped gradient is not written back (nothing reads it: the loop drops
the gradients right after the step); ``total_norm(group)`` returns the pre-clip norm like ``clip_grad_norm_`` does.
Nothing synchronises with the host, so the step can be captured in a HIP graph.

The moments live in two flat fp32 buffers per group; ``state[p]["exp_avg"]`` etc. are views into them.

``state_bits=8`` (an option of the optimizer or of one group) keeps both moments in 8 bits (``csrc/optim8.hip``): 2 bytes of
state an element instead of 8, and 16 bytes of memory traffic a step instead of 28.  ``state[p]`` then holds ``exp_avg``
(e4m3 codes, ``torch.float8_e4m3fn``) and ``exp_avg_sq_root`` (e4m3 codes of sqrt(exp_avg_sq)), each with an fp32 ``*_scale`` per
block of 256 elements: value = code * scale.  Tensors with fewer than ``min_8bit_numel`` elements (norms, biases) keep fp32
moments.  Checkpoints convert both ways when they are loaded.
"""
from __future__ import annotations

import ctypes as C
from typing import Iterable, List, Optional

import torch

from . import _lib
from .ops import check, _stream


class _Group:
    """Device tables of one parameter group (built at the first step, rebuilt if the parameter list changes)."""

    def __init__(self, params: List[torch.nn.Parameter]):
        dev = params[0].device
        self.params = params
        start4, off = [], 0
        for p in params:
            if p.dtype != torch.float32 or not p.is_contiguous() or p.device != dev:
                raise TypeError("ClipAdamW: parameters must be contiguous fp32 tensors on one device (fp32 master "
                                "weights, as in the reference)")
            start4.append(off)
            off += (p.numel() + 3) // 4
        start4.append(off)
        if off >= 1 << 31:
            raise ValueError("ClipAdamW: more than 2^33 parameters in one group")
        self.flat = 4 * off
        self.start4 = torch.tensor(start4, dtype=torch.int64).to(torch.int32).to(dev)        # values < 2^31
        self.numel = torch.tensor([p.numel() for p in params], dtype=torch.int64).to(torch.int32).to(dev)
        self.p_ptrs = torch.tensor([p.data_ptr() for p in params], dtype=torch.int64, device=dev)
        self.ptr_key = tuple(p.data_ptr() for p in params)
        self.m = torch.zeros(self.flat, dtype=torch.float32, device=dev)
        self.v = torch.zeros(self.flat, dtype=torch.float32, device=dev)
        self.step = torch.zeros(len(params), dtype=torch.float32, device=dev)     # one counter per tensor, as torch
        self.coef = torch.zeros(8, dtype=torch.float32, device=dev)
        self.lr = torch.zeros((), dtype=torch.float32, device=dev)
        self.lr_host = None
        lib = _lib.load()
        # sub-tables of at most OPT_MAX_TENSORS tensors: (first, count, flat elements, first partial, blocks)
        self.batches, nb = [], 0
        for a in range(0, len(params), _lib.OPT_MAX_TENSORS):
            b = min(len(params), a + _lib.OPT_MAX_TENSORS)
            flat = 4 * (start4[b] - start4[a])
            blocks = int(lib.unet_opt_blocks(flat))
            self.batches.append((a, b - a, flat, nb, blocks))
            nb += blocks
        self.partial = torch.zeros(max(nb, 1), dtype=torch.float32, device=dev)
        self.n_partial = nb


BLOCK = 256                 # csrc/optim8.hip: elements of a tensor that share one scale
FP8_MAX, FP8_LEAST = 448.0, 2.0 ** -9
CODES = ("exp_avg", "exp_avg_sq_root")         # the e4m3 entries of a tensor's state
TINY = 2.0 ** -100          # a block below this is stored as zeros
WIDE = 0x80000000           # include/unet_hip.h unet_adamw8_apply: slot of a tensor with fp32 moments


def quantise_moment(x: torch.Tensor, root: bool):
    """fp32 moment -> (e4m3 codes of x's shape, fp32 scale per block of 256 elements).  ``root``: x is sqrt(exp_avg_sq), whose
    positive values must not become zero."""
    n = x.numel()
    flat = torch.nn.functional.pad(x.reshape(-1).float(), (0, -n % BLOCK)).view(-1, BLOCK)
    top = flat.abs().amax(1, keepdim=True)
    some = top >= TINY
    y = torch.where(some, flat * (top.reciprocal() * FP8_MAX), torch.zeros_like(flat))
    if root:
        y = torch.where(some & (flat > 0), y.clamp_min(FP8_LEAST), y)
    scale = torch.where(some, top / FP8_MAX, torch.zeros_like(top)).view(-1)
    return y.to(torch.float8_e4m3fn).view(-1)[:n].view(x.shape), scale


def dequantise_moment(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The fp32 values that codes and scales of one tensor stand for."""
    n = codes.numel()
    return codes.reshape(-1).float() * scale.float().repeat_interleave(BLOCK)[:n]


def _load_moments(st):
    """(exp_avg, exp_avg_sq) of a state in either form as flat fp32, or None for a tensor that has not been stepped."""
    if "exp_avg" not in st:
        return None
    if "exp_avg_scale" in st:
        return (dequantise_moment(st["exp_avg"], st["exp_avg_scale"]),
                dequantise_moment(st["exp_avg_sq_root"], st["exp_avg_sq_root_scale"]).square())
    return st["exp_avg"].reshape(-1), st["exp_avg_sq"].reshape(-1)


def _dense_fp32(grads) -> bool:
    """One question a pass: with as many tensors as layers, three questions a tensor take 1.6 times as long."""
    live = [g for g in grads if g is not None]
    try:
        return all([g.is_contiguous() for g in live]) and {g.dtype for g in live} <= {torch.float32}
    except RuntimeError:                # a sparse layout that cannot say
        return False


class _Group8:
    """Device tables of a parameter group with 8-bit moments: code buffers for its large tensors, fp32 buffers for the rest."""

    def __init__(self, params: List[torch.nn.Parameter], min_numel: int):
        dev = params[0].device
        self.params, self.min_numel = params, min_numel
        start, slot, blocks, self.end8, self.end32 = [], [], 0, 0, 0
        for p in params:
            if p.dtype != torch.float32 or not p.is_contiguous() or p.device != dev:
                raise TypeError("ClipAdamW: parameters must be contiguous fp32 tensors on one device (fp32 master "
                                "weights, as in the reference)")
            if p.numel() >= 1 << 31:
                raise ValueError("ClipAdamW: a tensor of 2^31 or more elements cannot keep 8-bit moments")
            start.append(blocks)
            nb = -(-p.numel() // BLOCK)
            blocks += nb
            if p.numel() >= min_numel:
                slot.append(self.end8 // BLOCK)
                self.end8 += nb * BLOCK
            else:
                slot.append(WIDE | (self.end32 // 4))
                self.end32 += -(-p.numel() // 4) * 4
        start.append(blocks)
        if blocks * (BLOCK // 4) >= 1 << 31 or self.end32 >= 1 << 33:
            raise ValueError("ClipAdamW: more than 2^33 parameters in one group")
        as_u32 = lambda v: torch.tensor(v, dtype=torch.int64).to(torch.int32).to(dev)        # the low 32 bits
        self.start256, self.slot = as_u32(start), as_u32(slot)
        self.numel = as_u32([p.numel() for p in params])
        self.p_ptrs = torch.tensor([p.data_ptr() for p in params], dtype=torch.int64, device=dev)
        self.ptrs = [p.data_ptr() for p in params]
        self.device = dev.index
        zeros = lambda n, dt: torch.zeros(max(n, BLOCK), dtype=dt, device=dev)
        self.m8, self.r8 = (zeros(self.end8, torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
        self.m_scale, self.r_scale = (zeros(self.end8 // BLOCK, torch.float32) for _ in range(2))
        self.m, self.v = (zeros(self.end32, torch.float32) for _ in range(2))
        self.step = torch.zeros(len(params), dtype=torch.float32, device=dev)
        self.bc = torch.zeros((len(params), 2), dtype=torch.float32, device=dev)
        self.coef = torch.zeros(8, dtype=torch.float32, device=dev)
        self.lr = torch.zeros((), dtype=torch.float32, device=dev)
        self.lr_host = None
        lib = _lib.load()
        # sub-tables of at most OPT_MAX_TENSORS tensors: (first, count, blocks, first partial of the norm pass / of the step)
        batches, n1, n2 = [], 0, 0
        for a in range(0, len(params), _lib.OPT_MAX_TENSORS):
            b = min(len(params), a + _lib.OPT_MAX_TENSORS)
            nb = start[b] - start[a]
            if nb == 0:
                continue
            batches.append((a, b - a, nb, n1, n2))
            n1 += int(lib.unet_adamw8_norm_blocks(nb))
            n2 += int(lib.unet_adamw8_blocks(nb))
        self.n_norm, self.n_step = n1, n2
        self.partial = torch.zeros(max(n2, 1), dtype=torch.float32, device=dev)
        self.partial64 = torch.zeros(max(n1, 1), dtype=torch.float64, device=dev)
        # the fixed arguments of a batch's three calls (tables of 4-byte entries, but 8 bytes a pointer and a bias correction)
        part, at = self.partial.data_ptr(), lambda t, a: t.data_ptr() + a * t.element_size()
        self.calls = [(a, n,
                       (at(self.start256, a), at(self.numel, a), nb, at(self.partial64, p1)),
                       (at(self.step, a), at(self.bc, 2 * a)),
                       (at(self.p_ptrs, a), at(self.start256, a), at(self.numel, a), at(self.slot, a), nb, self.m8.data_ptr(),
                        self.r8.data_ptr(), self.m_scale.data_ptr(), self.r_scale.data_ptr(), self.m.data_ptr(), self.v.data_ptr(),
                        self.coef.data_ptr(), at(self.bc, 2 * a)), part + 4 * p2)
                      for a, n, nb, p1, p2 in batches]
        self.views = []
        for p, s, b in zip(params, slot, start):
            n = p.numel()
            if s & WIDE:
                a = 4 * (s & ~WIDE)
                self.views.append({"exp_avg": self.m[a:a + n].view_as(p), "exp_avg_sq": self.v[a:a + n].view_as(p)})
            else:
                a, nb = s * BLOCK, -(-n // BLOCK)
                self.views.append({"exp_avg": self.m8[a:a + n].view_as(p), "exp_avg_scale": self.m_scale[s:s + nb],
                                   "exp_avg_sq_root": self.r8[a:a + n].view_as(p), "exp_avg_sq_root_scale": self.r_scale[s:s + nb]})

    def fill(self, states) -> None:
        """Moments and step counts from the tensors' loaded states, in either form, or from an earlier table's views."""
        coded = [(st, v) for st, v in zip(states, self.views) if "exp_avg_scale" in v]
        if coded and all("exp_avg_scale" in st for st, _ in coded):
            # the usual case, all of the large tensors held in codes already: one gather a buffer
            for name, buf in zip(CODES, (self.m8, self.r8)):
                parts = []
                for st, v in coded:
                    parts.append(st[name].reshape(-1).to(torch.float8_e4m3fn).view(torch.uint8))
                    if v[name].numel() % BLOCK:
                        parts.append(parts[-1].new_zeros(-v[name].numel() % BLOCK))
                buf[:self.end8].view(torch.uint8).copy_(torch.cat(parts))        # (from wherever the states were loaded)
            for name, buf in zip(("exp_avg_scale", "exp_avg_sq_root_scale"), (self.m_scale, self.r_scale)):
                buf[:self.end8 // BLOCK].copy_(torch.cat([st[name].reshape(-1) for st, _ in coded]))
        else:                                   # some of them have not been stepped yet, or come from fp32
            for st, v in coded:
                if "exp_avg_scale" in st:
                    for k in v:
                        v[k].copy_(st[k].reshape(v[k].shape))
        for st, view in zip(states, self.views):
            if "exp_avg" in st and not ("exp_avg_scale" in view and "exp_avg_scale" in st):
                m, v = _load_moments(st)
                if "exp_avg_scale" in view:
                    new = quantise_moment(m, False) + quantise_moment(v.sqrt(), True)
                    keys = ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")
                else:
                    new, keys = (m, v), ("exp_avg", "exp_avg_sq")
                for k, t in zip(keys, new):
                    view[k].copy_(t.reshape(view[k].shape))
        steps = [st.get("step") for st in states]
        on_device = [t for t in steps if isinstance(t, torch.Tensor) and t.is_cuda]
        fetched = iter(torch.stack([t.float() for t in on_device]).tolist() if on_device else ())
        self.step.copy_(torch.tensor([0.0 if t is None else next(fetched) if isinstance(t, torch.Tensor) and t.is_cuda else float(t)
                                      for t in steps]))
        for st, view, step in zip(states, self.views, self.step.unbind()):
            for k in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_root", "exp_avg_sq_root_scale"):
                st.pop(k, None)
            st.update(view, step=step)


class ClipAdamW(torch.optim.Optimizer):
    def __init__(self, params: Iterable, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 max_grad_norm: Optional[float] = None, state_bits: int = 32, min_8bit_numel: int = 4096):
        """Arguments as ``torch.optim.AdamW`` (amsgrad / maximize are not offered: the reference never sets them).
        ``max_grad_norm``: clip the global L2 norm of each parameter group's gradients to this value inside ``step()``
        (``None`` or 0: no clipping); a group may override it with its own ``max_grad_norm`` entry.
        ``state_bits``: 32 (fp32 moments) or 8 (see the module docstring); ``min_8bit_numel``: tensors with fewer elements
        keep fp32 moments.  A group may override both; a loaded checkpoint does not."""
        if not 0.0 <= eps or not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0 or weight_decay < 0.0:
            raise ValueError("ClipAdamW: invalid hyper-parameter")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      max_grad_norm=max_grad_norm, state_bits=state_bits, min_8bit_numel=min_8bit_numel))
        self._groups = {}
        self.clips_gradients = True        # GraphedTrainStep / Trainer: do not clip a second time

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        if group["state_bits"] not in (8, 32) or not group["min_8bit_numel"] >= 0:
            self.param_groups.pop()
            raise ValueError(f"ClipAdamW: state_bits must be 8 or 32 and min_8bit_numel not negative, got {group['state_bits']} "
                             f"and {group['min_8bit_numel']}")

    # -- tables -------------------------------------------------------------------------------
    def _tables8(self, gi: int, group) -> Optional[_Group8]:
        g = self._groups.get(gi)
        ptrs = [p.data_ptr() for p in group["params"] if p.requires_grad]
        if not isinstance(g, _Group8) or g.ptrs != ptrs or g.min_numel != group["min_8bit_numel"]:
            params = [p for p in group["params"] if p.requires_grad]
            if not params:
                return None
            g = _Group8(params, group["min_8bit_numel"])
            g.fill([self.state[p] for p in params])
            self._groups[gi] = g
        return g

    def _tables(self, gi: int, group) -> _Group:
        if group["state_bits"] == 8:
            return self._tables8(gi, group)
        params = [p for p in group["params"] if p.requires_grad]
        if not params:
            return None
        g = self._groups.get(gi)
        key = tuple(p.data_ptr() for p in params)
        if not isinstance(g, _Group) or g.ptr_key != key:
            old = g
            g = _Group(params)
            starts = g.start4.cpu().tolist()
            for i, p in enumerate(params):
                a, n = 4 * starts[i], p.numel()
                st = self.state[p]
                # a state loaded from a checkpoint (or moments of a previous table) move into the flat buffers
                moments = _load_moments(st)
                if moments is not None:
                    g.m[a:a + n].copy_(moments[0])
                    g.v[a:a + n].copy_(moments[1])
                for k in ("exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale"):
                    st.pop(k, None)
                st["exp_avg"] = g.m[a:a + n].view_as(p)
                st["exp_avg_sq"] = g.v[a:a + n].view_as(p)
                prev = st.get("step")
                if prev is not None:
                    g.step[i] = float(prev)
                st["step"] = g.step[i]
            del old
            self._groups[gi] = g
        return g

    def load_state_dict(self, state_dict):
        """As ``torch.optim.Optimizer.load_state_dict``, except for three things torch's version loses: it replaces
        every param_group by the saved one, so a ``torch.optim.AdamW`` checkpoint of the reference (no
        ``max_grad_norm`` key) would silently switch the clip off, a device-scalar ``lr`` (graph-captured steps
        read it through its pointer) would become a float no captured step sees, and the codes of 8-bit moments would be
        cast to the parameters' fp32."""
        before = [(g.get("max_grad_norm"), g.get("lr"), g["state_bits"], g["min_8bit_numel"]) for g in self.param_groups]
        bare, codes = dict(state_dict, state={}), {}
        for i, st in state_dict["state"].items():
            if "exp_avg_scale" in st:
                codes[i] = {k: st[k] for k in CODES}
                st = {k: v for k, v in st.items() if k not in CODES}
            bare["state"][i] = st
        super().load_state_dict(bare)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(saved, [p for g in self.param_groups for p in g["params"]]):
            if i in codes:
                self.state[p].update({k: t.to(p.device, torch.float8_e4m3fn) for k, t in codes[i].items()})
        for group, (max_norm, lr, bits, min_numel) in zip(self.param_groups, before):
            group["state_bits"], group["min_8bit_numel"] = bits, min_numel     # the moments convert, see _load_moments
            if "max_grad_norm" not in group:
                group["max_grad_norm"] = max_norm
            if isinstance(lr, torch.Tensor):
                lr.fill_(float(group["lr"]))      # keep the tensor (and its address), take the loaded value
                group["lr"] = lr
        self._groups = {}                  # the loaded moments are copied into fresh flat buffers at the next step

    def total_norm(self, group_index: int = 0) -> torch.Tensor:
        """Global L2 norm of the group's gradients at the last ``step()`` (before clipping), a device scalar."""
        return self._groups[group_index].coef[3]

    def moment_buffers(self, group_index: int = 0) -> dict:
        """The flat buffers behind a group's ``state`` (live, not copies), in parameter order.  ``state_bits=32``: ``exp_avg``,
        ``exp_avg_sq``, tensors padded to 4 elements.  ``state_bits=8``: those hold the tensors below ``min_8bit_numel``; the
        others are in ``exp_avg8`` / ``exp_avg_sq_root8`` (e4m3 codes, tensors padded to 256 elements) with one fp32 scale per
        256 codes in ``exp_avg8_scale`` / ``exp_avg_sq_root8_scale``."""
        g, group = self._groups.get(group_index), self.param_groups[group_index]
        eight = group["state_bits"] == 8
        if g is None or isinstance(g, _Group8) != eight or (eight and g.min_numel != group["min_8bit_numel"]):
            g = self._tables(group_index, group)      # nothing yet, or other options than the last step's
        if g is None:
            return {}
        if not isinstance(g, _Group8):
            return {"exp_avg": g.m, "exp_avg_sq": g.v}
        nb = g.end8 // BLOCK
        return {"exp_avg": g.m[:g.end32], "exp_avg_sq": g.v[:g.end32], "exp_avg8": g.m8[:g.end8], "exp_avg8_scale": g.m_scale[:nb],
                "exp_avg_sq_root8": g.r8[:g.end8], "exp_avg_sq_root8_scale": g.r_scale[:nb]}

    # -- step -----------------------------------------------------------------------------------
    def _apply8(self, lib, g: _Group8, group, grads, max_norm: float, lr_ptr: int) -> None:
        """One step of an 8-bit group: norm first if it clips, otherwise the norm falls out of the step."""
        st = torch._C._cuda_getCurrentRawStream(g.device)
        b1, b2 = (float(b) for b in group["betas"])
        eps, decay = float(group["eps"]), float(group["weight_decay"])
        clips, coef = max_norm > 0.0, g.coef.data_ptr()
        arrs = [(C.c_void_p * c[1])(*grads[c[0]:c[0] + c[1]]) for c in g.calls]
        sums = (g.partial64.data_ptr(), g.n_norm, 1) if clips else (None, 0, 0)
        if clips:
            for (_, n, norm, _, _, _), arr in zip(g.calls, arrs):
                check(lib.unet_adamw8_sqnorm(arr, n, *norm, st), "unet_adamw8_sqnorm")
        for (_, n, _, prep, _, _), arr in zip(g.calls, arrs):
            check(lib.unet_adamw8_prepare(arr, n, *sums, max_norm, lr_ptr, coef, prep[0], b1, b2, prep[1], st), "unet_adamw8_prepare")
        for (_, n, _, _, table, p2), arr in zip(g.calls, arrs):
            check(lib.unet_adamw8_apply(arr, n, *table, None if clips else p2, b1, b2, eps, decay, st), "unet_adamw8_apply")
        if not clips:
            check(lib.unet_adamw8_prepare(None, 0, g.partial.data_ptr(), g.n_step, 0, 0.0, lr_ptr, coef, None, b1, b2, None, st),
                  "unet_adamw8_prepare")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _lib.load()
        for gi, group in enumerate(self.param_groups):
            g = self._tables(gi, group)
            if g is None:
                continue
            lr = group["lr"]
            if isinstance(lr, torch.Tensor) and lr.is_cuda and lr.dtype == torch.float32 and lr.numel() == 1:
                lr_ptr = lr.data_ptr()                               # a device scalar the caller updates in place
            else:
                lr = float(lr)
                if lr != g.lr_host:
                    g.lr.fill_(lr)
                    g.lr_host = lr
                lr_ptr = g.lr.data_ptr()
            if isinstance(g, _Group8):
                grads = [p.grad for p in g.params]
                if not _dense_fp32(grads):
                    raise TypeError("ClipAdamW: gradients must be contiguous dense fp32 tensors")
                ptrs = [None if gr is None else gr.data_ptr() for gr in grads]
                if any(ptrs) and g.calls:
                    max_norm = float(group.get("max_grad_norm") or 0.0)
                    if g.device == torch._C._cuda_getDevice():
                        self._apply8(lib, g, group, ptrs, max_norm, lr_ptr)
                    else:
                        with torch.cuda.device(g.device):
                            self._apply8(lib, g, group, ptrs, max_norm, lr_ptr)
                continue
            grads = []
            for p in g.params:
                gr = p.grad
                if gr is None:
                    grads.append(None)
                    continue
                if gr.dtype != torch.float32 or not gr.is_contiguous() or gr.is_sparse:
                    raise TypeError("ClipAdamW: gradients must be contiguous dense fp32 tensors")
                grads.append(gr.data_ptr())
            if all(x is None for x in grads):
                continue
            st = _stream()
            beta1, beta2 = group["betas"]
            max_norm = group.get("max_grad_norm") or 0.0
            arrs = []
            for a, n, flat, p0, blocks in g.batches:
                arr = (C.c_void_p * n)(*grads[a:a + n])
                arrs.append(arr)
                check(lib.unet_grad_sqnorm(arr, n, g.start4[a:].data_ptr(), g.numel[a:].data_ptr(), flat,
                                           g.partial[p0:].data_ptr(), g.step[a:].data_ptr(), st), "unet_grad_sqnorm")
            check(lib.unet_clip_adamw_prepare(g.partial.data_ptr(), g.n_partial, float(max_norm), lr_ptr,
                                              g.coef.data_ptr(), st), "unet_clip_adamw_prepare")
            for (a, n, flat, p0, blocks), arr in zip(g.batches, arrs):
                check(lib.unet_clip_adamw_apply(arr, n, g.p_ptrs[a:].data_ptr(), g.start4[a:].data_ptr(),
                                                g.numel[a:].data_ptr(), flat, g.m.data_ptr(), g.v.data_ptr(),
                                                g.coef.data_ptr(), g.step[a:].data_ptr(), float(beta1), float(beta2),
                                                float(group["eps"]),
                                                float(group["weight_decay"]), st), "unet_clip_adamw_apply")
        return loss
