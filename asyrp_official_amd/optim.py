"""AdamW over many tensors at once on the HIP library (csrc/adamw.hip): the optimiser of the DeltaBlock training step.

The reference steps its DeltaBlock with a torch optimiser (diffusion_latent.py:288-290, 349-350).  `AdamW` takes the same place:
    opt = AdamW(model.layer_0.parameters(), lr=1e-4, state_bits=8, max_norm=1.0)
    opt.zero_grad(); loss.backward(); opt.step()
"""
import math
import operator
import struct

import torch

from . import _lib
from .engine import AsyrpDeviceError

_raw_stream = torch._C._cuda_getCurrentRawStream      # the current stream's handle (torch.cuda.current_stream() without its object)

BLOCK = 256          # values that share one exponent of the 8-bit moments; every parameter's moments start on a multiple of it


class _Moments:
    """The flat moments of one parameter group: parameter i's values lie at offsets[i]."""

    def __init__(self, params, bits, device):
        self.params, self.bits, self.device = list(params), bits, device
        self.numels = [p.numel() for p in self.params]
        self.offsets, n = [], 0
        for k in self.numels:
            self.offsets.append(n)
            n += -(-k // BLOCK) * BLOCK
        self.n = n
        if bits == 32:
            self.m, self.v = (torch.zeros(n, device=device, dtype=torch.float32) for _ in range(2))
            self.me = self.ve = None
        else:
            self.m, self.v = (torch.zeros(n, device=device, dtype=torch.uint8) for _ in range(2))
            self.me, self.ve = (torch.zeros(n // BLOCK, device=device, dtype=torch.uint8) for _ in range(2))
        self.steps = torch.zeros(max(1, len(self.params)), device=device, dtype=torch.int32)

    def of(self, params):
        return len(self.params) == len(params) and all(map(operator.is_, self.params, params))

    def views(self, i):
        """What self.state holds of parameter i: views of the flat moments (8 bits: codes and exponent bytes)."""
        at, k, p = self.offsets[i], self.numels[i], self.params[i]
        d = {"step": self.steps[i], "exp_avg": self.m[at:at + k].view(p.shape), "exp_avg_sq": self.v[at:at + k].view(p.shape)}
        if self.bits == 8:
            e = slice(at // BLOCK, at // BLOCK + -(-k // BLOCK))
            d["exp_avg_scale"], d["exp_avg_sq_scale"] = self.me[e], self.ve[e]
        return d


class AdamW(torch.optim.Optimizer):
    """One step: p <- p (1 - lr weight_decay) - lr m^ / (sqrt(v^) + eps) with bias-corrected moments (decoupled weight decay), for every parameter that has a
    gradient, in a few launches whatever their number.

    params: float32, float16 or bfloat16 parameters on one GPU, contiguous; gradients of the same type.  state_bits: 32, or 8 (blocks of 256
    values with a power-of-two scale each, rounded at random by the counter hash of csrc/adamw.hip under `seed`; two runs with one seed are alike to the bit).
    max_norm: clips all gradients by their global norm (factor min(1, max_norm / (norm + 1e-6))); the gradients themselves keep
    their values, `grad_norm` (device, float32) holds the last norm, and a step whose norm is not finite changes nothing, its step counts included.
    Without max_norm values that are not finite go their way into the parameters; 8-bit moments keep a block that holds one as NaN.

    Step counts, moments and the norm live on the device, so a step may be captured into a graph once the moments are there (after the first step, or
    `prepare()`); gradients then have to keep their addresses, and lr, where it changes, has to be a float32 tensor on the device (it is
    read when the step runs)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_norm=None, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if max_norm is not None and not 0.0 < float(max_norm) < float("inf"):
            raise ValueError(f"max_norm must be positive and finite, got {max_norm}")
        self.state_bits, self.max_norm, self.seed = int(state_bits), None if max_norm is None else float(max_norm), int(seed) & 0xFFFFFFFF
        self.grad_norm, self._moments = None, {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(g):
        b1, b2 = g["betas"]
        if isinstance(g["lr"], torch.Tensor):
            if g["lr"].numel() != 1:
                raise ValueError("lr as a tensor holds one value")
        elif not 0.0 <= g["lr"] < float("inf"):
            raise ValueError(f"lr must be finite and not negative, got {g['lr']}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must lie in [0, 1), got {g['betas']}")
        if not 0.0 <= g["eps"] < float("inf") or not 0.0 <= g["weight_decay"] < float("inf"):
            raise ValueError("eps and weight_decay must be finite and not negative")
        if len(set(map(id, g["params"]))) != len(g["params"]):
            raise ValueError("a parameter stands in the group twice")
        for p in g["params"]:
            if p.dtype not in _lib.DTYPES:
                raise ValueError(f"parameters must be float32, float16 or bfloat16, got {p.dtype}")

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "max_norm": self.max_norm, "seed": self.seed}

    def __setstate__(self, st):
        super().__setstate__(st)
        self.grad_norm, self._moments = None, {}          # rebuilt from self.state

    # ---- moments ---------------------------------------------------------------------------------------
    def _device(self):
        index = None
        for g in self.param_groups:
            for p in g["params"]:
                d = p.get_device()                         # -1 on the CPU
                if d != index:
                    if d < 0:
                        raise AsyrpDeviceError("AdamW steps only parameters on an MI355X (device type 'cuda' under ROCm): there is no CPU path")
                    if index is not None:
                        raise AsyrpDeviceError(f"parameters on cuda:{index} and cuda:{d}: one optimiser steps one device")
                    index = d
        return None if index is None else torch.device("cuda", index)

    def _group_moments(self, k, device):
        g, mo = self.param_groups[k], self._moments.get(k)
        if mo is not None and mo.device == device and mo.of(g["params"]):
            return mo
        for p in g["params"]:
            if not p.is_contiguous():
                raise ValueError("parameters must be contiguous")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the moments have to be there before a step is captured (every replay would start from new ones): step once or call prepare() first")
        mo = _Moments(g["params"], self.state_bits, device)
        for i, p in enumerate(mo.params):                 # moments that are there already: loaded ones, or those of an unpickled copy
            views, old = mo.views(i), self.state.get(p) or {}
            for key, view in views.items():
                if key in old:
                    view.copy_(torch.as_tensor(old[key]).reshape(view.shape))
            self.state[p] = views
        self._moments[k] = mo
        return mo

    def prepare(self):
        """Allocates the moments (the first step does it otherwise)."""
        device = self._device()
        if device is not None:
            with torch.no_grad():
                for k in range(len(self.param_groups)):
                    self._group_moments(k, device)

    @torch.no_grad()
    def moments(self):
        """[(exp_avg, exp_avg_sq)] of each group as flat float32 tensors, every parameter's values filled up with zeros to a multiple of 256.  32-bit
        moments are the optimiser's own buffers, 8-bit ones the values that their codes stand for."""
        device, out = self._device(), []
        for k in range(len(self.param_groups)):
            mo = self._group_moments(k, device)
            if mo.bits == 32:
                out.append((mo.m, mo.v))
                continue
            m, v = (torch.empty(mo.n, device=device, dtype=torch.float32) for _ in range(2))
            _lib.check(_lib.load().asyrp_adamw_moments(device.index, *(t.data_ptr() for t in (mo.m, mo.v, mo.me, mo.ve)), mo.n, m.data_ptr(), v.data_ptr(),
                                                       _raw_stream(device.index)))
            out.append((m, v))
        return out

    def load_state_dict(self, state_dict):
        """Takes what state_dict() of an optimiser with the same state_bits gave.  Moments, step counts and a learning rate on the device that are there
        already take their values in place, so that a captured step goes on with what was loaded.  What does not fit is refused before anything has changed."""
        taken = {}
        # the state does not go through the base class, which would convert it to the parameters' type: it is taken out behind all hooks in front, and
        # put in place in front of all hooks behind
        front = self.register_load_state_dict_pre_hook(lambda _, sd: taken.update(self._take_state(sd)) or {**sd, "state": {}})
        behind = self.register_load_state_dict_post_hook(lambda _: self._put_state(**taken), prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            front.remove()
            behind.remove()

    def _take_state(self, sd):
        """What _put_state needs of a state dict and of what is there, or ValueError."""
        saved, groups = sd["state"], sd["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("loaded state dict has other parameter groups")
        for i, p in [(i, p) for g, mine in zip(groups, self.param_groups) for i, p in zip(g["params"], mine["params"])]:
            st = saved.get(i)
            if not st:
                continue
            want = {"exp_avg": tuple(p.shape), "exp_avg_sq": tuple(p.shape)}
            if self.state_bits == 8:
                want["exp_avg_scale"] = want["exp_avg_sq_scale"] = (-(-p.numel() // BLOCK),)
            codes = [k for k in st if k != "step" and isinstance(st[k], torch.Tensor) and st[k].dtype == torch.uint8]
            if set(st) != {"step", *want} or torch.as_tensor(st["step"]).numel() != 1 or any(tuple(torch.as_tensor(st[k]).shape) != shape for k, shape in want.items()) \
                    or len(codes) != (4 if self.state_bits == 8 else 0):
                raise ValueError(f"loaded state of parameter {i} is not one of AdamW with {self.state_bits}-bit moments and shape {tuple(p.shape)}")
        return dict(saved=saved, ids=[g["params"] for g in groups], moments=self._moments, norm=self.grad_norm, rates=[g["lr"] for g in self.param_groups])

    @torch.no_grad()
    def _put_state(self, saved, ids, moments, norm, rates):
        self._moments, self.grad_norm = moments, norm
        for g, lr in zip(self.param_groups, rates):
            if isinstance(lr, torch.Tensor) and lr.is_cuda:
                lr.fill_(float(g["lr"]))
                g["lr"] = lr
        for k, mo in list(moments.items()):
            if not mo.of(self.param_groups[k]["params"]):
                del moments[k]
                continue
            for i, p in enumerate(mo.params):
                views, st = mo.views(i), saved.get(ids[k][i]) or {}
                for key, view in views.items():
                    view.copy_(torch.as_tensor(st[key]).reshape(view.shape)) if key in st else view.zero_()
                self.state[p] = views
        for i, p in [(i, p) for mine, g in zip(ids, self.param_groups) for i, p in zip(mine, g["params"])]:
            if saved.get(i) and p not in self.state:
                self.state[p] = {k: t.detach().clone() if isinstance(t, torch.Tensor) else t for k, t in saved[i].items()}

    # ---- the step --------------------------------------------------------------------------------------
    @staticmethod
    def _hyper(g, device):
        """((lr, address of lr on the device), (beta1, beta2, eps, weight decay)) of a group as it is now, or ValueError: before anything is launched for any group."""
        lr, at = g["lr"], 0
        if isinstance(lr, torch.Tensor) and lr.is_cuda:
            if lr.dtype != torch.float32 or lr.device != device or lr.numel() != 1:
                raise ValueError(f"lr as a device tensor must be one float32 value on {device}")
            lr, at = 0.0, lr.data_ptr()
        (b1, b2), eps, decay = g["betas"], float(g["eps"]), float(g["weight_decay"])
        lr, b1, b2 = float(lr), float(b1), float(b2)
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must lie in [0, 1), got {g['betas']}")
        if not (math.isfinite(lr) and 0.0 <= eps < math.inf and math.isfinite(decay)):
            raise ValueError(f"lr, eps and weight_decay must be finite and eps not negative, got {lr}, {eps}, {decay}")
        return (lr, at), (b1, b2, eps, decay)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        device = self._device()
        if device is None:
            return loss
        lib, stream, todo = _lib.load(), _raw_stream(device.index), []
        held = []                                          # copies of gradients laid out otherwise live until the launches are queued
        for k, g in enumerate(self.param_groups):
            mo, by_type = self._group_moments(k, device), {}
            for p, n, at, i in zip(mo.params, mo.numels, mo.offsets, range(len(mo.params))):
                grad = p.grad
                if grad is None:
                    continue
                if grad.dtype != p.dtype or grad.layout != torch.strided or grad.numel() != n or grad.get_device() != device.index:
                    raise ValueError(f"the gradient of a {p.dtype} parameter {tuple(p.shape)} must be dense, of its type, size and device")
                if p.numel() != n or not p.is_contiguous():
                    raise ValueError("parameters must be contiguous and keep their size")
                if not grad.is_contiguous():
                    grad = grad.contiguous()
                    held.append(grad)
                flat, params = by_type.setdefault(p.dtype, ([], []))
                flat += (p.data_ptr(), grad.data_ptr(), n, at, i)
                params.append(p)
            if by_type:
                lr, hyper = self._hyper(g, device)
                todo += [(lr, hyper, mo, _lib.DTYPES[dtype], len(params), struct.pack(f"{len(flat)}q", *flat), params) for dtype, (flat, params) in by_type.items()]
        if not todo:
            return loss
        sumsq, clip = None, (0, 0.0, 0, 0)
        if self.max_norm is not None:
            counts = [-(-n // _lib.ADAMW_TABLE) * _lib.ADAMW_PARTIALS for _, _, _, _, n, _, _ in todo]
            sumsq = torch.empty(sum(counts), device=device, dtype=torch.float64)
            if self.grad_norm is None or self.grad_norm.device != device:
                self.grad_norm = torch.zeros((), device=device, dtype=torch.float32)
            at = sumsq.data_ptr()
            clip = (at, self.max_norm, self.grad_norm.data_ptr(), sum(counts))
            for (_, _, _, dtype, n, table, _), c in zip(todo, counts):
                _lib.check(lib.asyrp_grad_sumsq(device.index, table, n, dtype, at, stream))
                at += 8 * c
        for (lr, lr_device), hyper, mo, dtype, n, table, params in todo:
            spec = _lib.ADAMW.pack(lr, *hyper, lr_device, mo.steps.data_ptr(), *clip[:3], mo.m.data_ptr(), mo.v.data_ptr(),
                                   *((mo.me.data_ptr(), mo.ve.data_ptr()) if mo.bits == 8 else (0, 0)), clip[3], mo.bits, self.seed)
            scratch = torch.empty(4 * (n + 1) + n, device=device, dtype=torch.float32)
            _lib.check(lib.asyrp_adamw_step(device.index, spec, table, n, dtype, scratch.data_ptr(), stream))
            torch.autograd.graph.increment_version(params)   # the engine uploads parameters whose version has moved
        return loss
