"""FusedAdam — ``torch.optim.Adam`` semantics over a parameter arena, one HIP launch per step.

The reference builds ``partial(Adam, lr=lr, betas=betas)`` (experiments/basic_conf.py:55,67;
gradient_penalty_conf.py:9-10) and calls ``optimizer.step()`` once per update
(Trainer.py:135,157).  Here every parameter, gradient and moment of a module lives in one flat
``Arena`` (cgan3d_amd.engine), so the whole update is a single elementwise kernel
(``cgan3d_adam``).  It is a real ``torch.optim.Optimizer``: ``param_groups`` drive the learning
rate (so ``MultiStepLR`` works unchanged) and ``state_dict`` carries torch-Adam-shaped state
(``step``, ``exp_avg``, ``exp_avg_sq`` per parameter) for checkpoint interchange.

FusedMuon — the same arena under the Muon optimiser: momentum, its Newton-Schulz orthogonalisation and
the update of every weight that is a matrix (convolution weights flattened to [first axis, the rest]),
Adam for the vectors (biases, BatchNorm scales and shifts), from one host call (``cgan3d_muon_step``).
``Trainer`` builds either from its ``partial(...)`` (``optimizer_from_partial``).
"""
from __future__ import annotations

import math
from contextlib import nullcontext
from functools import partial

import torch

from .. import ops
from ..engine import Arena


def adam_hyper_from_partial(optim_class) -> dict:
    """lr / betas / eps of a ``partial(torch.optim.Adam, ...)`` config entry."""
    func = optim_class.func if isinstance(optim_class, partial) else optim_class
    if func is not torch.optim.Adam:
        raise NotImplementedError(f"the HIP step implements Adam only (got {getattr(func, '__name__', func)})")
    kw = dict(optim_class.keywords) if isinstance(optim_class, partial) else {}
    for bad in ("weight_decay", "amsgrad", "maximize"):
        if kw.get(bad):
            raise NotImplementedError(f"Adam({bad}=...) is not used by the reference configs")
    betas = kw.get("betas", (0.9, 0.999))
    return {"lr": float(kw.get("lr", 1e-3)), "betas": (float(betas[0]), float(betas[1])),
            "eps": float(kw.get("eps", 1e-8))}


def optimizer_from_partial(optim_class, arena: Arena, weight_clip=None):
    """The arena optimiser of a config entry: ``partial(FusedMuon, ...)`` or ``partial(torch.optim.Adam, ...)``."""
    func = optim_class.func if isinstance(optim_class, partial) else optim_class
    if func is FusedMuon:
        kw = dict(optim_class.keywords) if isinstance(optim_class, partial) else {}
        if isinstance(optim_class, partial) and optim_class.args:
            raise TypeError("partial(FusedMuon, ...) takes keywords only: the Trainer passes the arena")
        return FusedMuon(arena, **{"weight_clip": weight_clip, **kw})
    return FusedAdam(arena, **adam_hyper_from_partial(optim_class), weight_clip=weight_clip)


class FusedAdam(torch.optim.Optimizer):
    def __init__(self, arena: Arena, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_clip=None):
        super().__init__(arena.params, dict(lr=lr, betas=betas, eps=eps))
        self.arena = arena
        dev = arena.flat.device
        # device-resident [lr, beta1, beta2, eps, step, clip] so a captured step replays correctly
        self.hyper = torch.tensor([lr, betas[0], betas[1], eps, 0.0, weight_clip or 0.0], device=dev,
                                  dtype=torch.float32)
        self.ticket = ops.tickets(1, dev)[0]  # launch ticket of the fused update + repack
        self._host_step = 0
        self._host_lr = lr
        for p, name in zip(arena.params, arena.names):
            off = self._offset(p)
            n = p.numel()
            self.state[p] = {"exp_avg": arena.exp_avg[off:off + n].view_as(p),
                             "exp_avg_sq": arena.exp_avg_sq[off:off + n].view_as(p)}

    def _offset(self, p):
        return (p.data_ptr() - self.arena.flat.data_ptr()) // 4

    def sync_hyper(self):
        """Push a changed learning rate (LR scheduler) to the device scalar."""
        lr = float(self.param_groups[0]["lr"])
        if lr != self._host_lr:
            self.hyper[0].fill_(lr)
            self._host_lr = lr

    def launch(self, packs=None):
        """Enqueue one update (step counter advanced on the device); no host sync.  One launch
        (cgan3d_adam_pack: the step tick rides on the Adam kernel, its last block out advances it).
        With ``packs`` (an ops.PackSet over this arena's weights) the packed copies are refreshed in
        the same launch — each updated parameter written straight into its packed positions; those
        are scattered 2-byte stores, measured slower than a separate coalesced repack launch for the
        generator (37 us against 11 + 11), so the engine repacks separately."""
        a = self.arena
        ops.adam_pack(a.flat, a.grad, a.exp_avg, a.exp_avg_sq, self.hyper, self.ticket, packs)
        self._opt_called = True  # what torch's LR schedulers check optimizer.step() for
        if not ops.recording():  # a recorded plan counts its steps when it runs (note_step)
            self._host_step += 1

    def note_step(self):
        """Count one update issued by a replayed launch plan (the device counter ticks itself)."""
        self._opt_called = True
        self._host_step += 1

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        self.sync_hyper()
        self.launch()
        return loss

    def zero_grad(self, set_to_none: bool = True):
        self.arena.grad.zero_()
        self.arena.rebind_grads()

    def state_dict(self):
        step = float(self.hyper[4].item())  # device counter (correct under graph replay too)
        for p in self.arena.params:
            self.state[p]["step"] = torch.tensor(step)
        return super().state_dict()

    def load_state_dict(self, state_dict):
        views = {p: (self.state[p]["exp_avg"], self.state[p]["exp_avg_sq"]) for p in self.arena.params}
        super().load_state_dict(state_dict)
        step = 0
        for p in self.arena.params:
            st = self.state[p]
            m, v = views[p]
            m.copy_(st["exp_avg"])
            v.copy_(st["exp_avg_sq"])
            st["exp_avg"], st["exp_avg_sq"] = m, v
            step = int(st.get("step", torch.tensor(0.0)).item())
        self._host_step = step
        self.hyper[4].fill_(float(step))
        self._host_lr = None
        self.sync_hyper()


class FusedMuon(torch.optim.Optimizer):
    """Muon over a parameter arena.  Two parameter groups: the matrices (``lr``, ``momentum``,
    ``weight_decay``, ``nesterov``) and the vectors (``lr`` = ``vector_lr``, ``betas``, ``eps``: Adam without
    decay); a learning-rate scheduler drives both.

    ``adjust_lr``: "original" multiplies lr by sqrt(max(1, rows / cols)), "match_rms_adamw" by
    0.2 sqrt(max(rows, cols)) (updates of Adam's size).  The arena's ``exp_avg`` holds the matrices'
    momentum and the vectors' first moment."""

    def __init__(self, arena: Arena, lr=0.02, momentum=0.95, weight_decay=0.0, nesterov=True, ns_steps=5,
                 ns_coefficients=ops.NS_COEFFICIENTS, eps=1e-7, adjust_lr="original", vector_lr=3e-4,
                 vector_betas=(0.9, 0.999), vector_eps=1e-8, weight_clip=None):
        scales = {"original": lambda r, c: math.sqrt(max(1.0, r / c)),
                  "match_rms_adamw": lambda r, c: 0.2 * math.sqrt(max(r, c))}
        if adjust_lr not in scales:
            raise ValueError(f"FusedMuon: adjust_lr {adjust_lr!r} (one of {sorted(scales)})")
        if lr < 0 or vector_lr < 0 or weight_decay < 0 or not 0 <= momentum < 1:
            raise ValueError(f"FusedMuon: lr {lr}, vector_lr {vector_lr} and weight_decay {weight_decay} may not be "
                             f"negative, momentum {momentum} must be in [0, 1)")
        if not (0 <= vector_betas[0] < 1 and 0 <= vector_betas[1] < 1):
            raise ValueError(f"FusedMuon: vector_betas {vector_betas} must be in [0, 1)")
        ops._ns_args(ns_steps, ns_coefficients, eps, "FusedMuon")
        mats = [p for p in arena.params if p.dim() >= 2]
        vecs = [p for p in arena.params if p.dim() < 2]
        super().__init__([dict(params=mats, lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov),
                          dict(params=vecs, lr=vector_lr, betas=tuple(vector_betas), eps=vector_eps)], {})
        self.arena = arena
        self.ns_steps, self.ns_coefficients, self.eps = int(ns_steps), tuple(ns_coefficients), float(eps)
        matrices, vectors, off = [], [], 0
        for p in arena.params:
            n = p.numel()
            if p.dim() >= 2:
                r, c = p.shape[0], n // p.shape[0] if n else 0
                if n:
                    matrices.append((off, r, c, scales[adjust_lr](r, c)))
                self.state[p] = {"momentum_buffer": arena.exp_avg[off:off + n].view_as(p)}
            else:
                if vectors and sum(vectors[-1]) == off:  # neighbours are one segment
                    vectors[-1] = (vectors[-1][0], vectors[-1][1] + n)
                else:
                    vectors.append((off, n))
                self.state[p] = {"exp_avg": arena.exp_avg[off:off + n].view_as(p),
                                 "exp_avg_sq": arena.exp_avg_sq[off:off + n].view_as(p)}
            off += n
        self.segs = ops.MuonSegments(arena.numel, matrices, vectors)
        dev = arena.flat.device
        # device-resident, so that a recorded plan or captured graph follows the schedulers
        self._host = self._group_hyper()
        self.hyper = torch.tensor(self._host[:4] + [0.0, weight_clip or 0.0] + self._host[4:], dtype=torch.float32,
                                  device=dev)
        # owned: a plan or graph that holds a step keeps the address; steps of one optimiser are ordered anyway
        with torch.cuda.device(dev) if dev.type == "cuda" else nullcontext():  # its size goes by the current device
            need = self.segs.ws_bytes()
        self.ws = torch.empty(need, dtype=torch.uint8, device=dev)
        self._host_step = 0

    def _group_hyper(self):
        m, v = self.param_groups
        return [float(m["lr"]), float(m["momentum"]), float(m["weight_decay"]), float(bool(m["nesterov"])),
                float(v["lr"]), float(v["betas"][0]), float(v["betas"][1]), float(v["eps"])]

    def sync_hyper(self):
        """Push what a scheduler (or the user) changed in the parameter groups to the device scalars."""
        now = self._group_hyper()
        for i, (new, old) in enumerate(zip(now, self._host)):
            if new != old:
                self.hyper[i if i < 4 else i + 2].fill_(new)
        self._host = now

    def launch(self, packs=None):
        """Enqueue one update (step counter advanced on the device); no host sync."""
        if packs is not None:
            raise NotImplementedError("FusedMuon: packed weight copies are refreshed by the engine's repack launch")
        a = self.arena
        ops.muon_step(a.flat, a.grad, a.exp_avg, a.exp_avg_sq, self.segs, self.hyper, self.ns_steps,
                      self.ns_coefficients, self.eps, ws=self.ws)
        self._opt_called = True  # what torch's LR schedulers check optimizer.step() for
        if not ops.recording():  # a recorded plan counts its steps when it runs (note_step)
            self._host_step += 1

    note_step = FusedAdam.note_step
    step = FusedAdam.step
    zero_grad = FusedAdam.zero_grad

    def state_dict(self):
        step = float(self.hyper[4].item())  # device counter (correct under graph replay too)
        for p in self.arena.params:
            self.state[p]["step"] = torch.tensor(step)
        return super().state_dict()

    def load_state_dict(self, state_dict):
        views = {p: {k: t for k, t in self.state[p].items() if k != "step"} for p in self.arena.params}
        super().load_state_dict(state_dict)
        step = 0
        for p in self.arena.params:
            st = self.state[p]
            for k, t in views[p].items():
                t.copy_(st[k])
                st[k] = t
            step = int(st.get("step", torch.tensor(0.0)).item())
        self._host_step = step
        self.hyper[4].fill_(float(step))
        self._host = [None] * len(self._host)
        self.sync_hyper()
