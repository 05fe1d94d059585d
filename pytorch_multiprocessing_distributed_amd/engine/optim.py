"""Fused SGD (momentum / Nesterov / weight decay) over the flat arena.

Math is exactly ``torch.optim.SGD`` (torch:optim/sgd.py:383-477) as used by
the reference (lr 0.1, momentum 0.9, wd 1e-4, nesterov; main.py:51-55):

    g   = g + wd * p
    buf = g                      (first step)   | m * buf + (1 - dampening) * g
    g   = g + m * buf            (nesterov)     | buf
    p   = p - lr * g

but the whole model is ONE kernel launch over the flat param/grad/momentum
arenas (K16) instead of ~5 multi-tensor launches.  It subclasses
``torch.optim.Optimizer`` so ``torch.optim.lr_scheduler.MultiStepLR`` (the
reference scheduler, main.py:57-59) drives ``param_groups[0]['lr']``.

:class:`Muon` updates the convolution weights along their orthogonalised momentum instead
(Newton-Schulz, ops/functional.py newton_schulz), and everything else with the rule above.
"""
from __future__ import annotations

import torch

from ..ops.functional import NS_COEFFS, prims_for
from ..parallel.flat import flatten_module, get_flat


class FusedSGD(torch.optim.Optimizer):
    def __init__(self, module, lr=0.1, momentum=0.9, weight_decay=1e-4, nesterov=True,
                 dampening=0.0):
        if nesterov and (momentum <= 0 or dampening != 0):
            raise ValueError("Nesterov momentum requires a momentum and zero dampening")
        inner = getattr(module, "module", module)
        self.flat = get_flat(inner) or flatten_module(inner)
        defaults = dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov,
                        dampening=dampening)
        super().__init__(self.flat.params, defaults)
        self.momentum_arena = torch.zeros_like(self.flat.param_arena)
        self.flat.companions.append(self.momentum_arena)   # follows arena relayouts
        self.steps = 0
        # device-resident learning rate: the SGD kernel reads it, so a captured
        # HIP graph of the step follows scheduler updates (see graph_safe())
        self.lr_dev = None
        self._lr_cached = None

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        g = self.param_groups[0]
        P = prims_for(self.flat.param_arena)
        if self.lr_dev is not None and not torch.cuda.is_current_stream_capturing():
            self.sync_lr()
        P.sgd_nesterov_(self.flat.param_arena, self.flat.grad_arena, self.momentum_arena,
                        g["lr"], g["momentum"], g["weight_decay"], g["nesterov"],
                        self.steps == 0, g["dampening"], self.lr_dev)
        self.steps += 1
        return loss

    def graph_safe(self):
        """Switch to the device-resident LR (call before capturing a step)."""
        if self.lr_dev is None:
            self.lr_dev = torch.zeros(1, dtype=torch.float32, device=self.flat.device)
            self._lr_cached = None
            self.sync_lr()
        return self

    def sync_lr(self):
        lr = float(self.param_groups[0]["lr"])
        if lr != self._lr_cached:
            self.lr_dev.fill_(lr)
            self._lr_cached = lr

    def zero_grad(self, set_to_none: bool = False):
        # grads are views into the arena: always zero in place
        self.flat.zero_grad()

    # ------------------------------------------------------ resume state
    def state_dict(self):
        # momentum per parameter name: independent of the arena layout (which the
        # data-parallel wrapper re-orders after its first iteration)
        mom = {n: self.momentum_arena[o: o + p.numel()].detach().cpu().clone()
               for n, p, o in zip(self.flat.names, self.flat.params, self.flat.offsets)}
        return {"steps": self.steps, "momentum": mom,
                "param_groups": [{k: v for k, v in g.items() if k != "params"}
                                 for g in self.param_groups]}

    def load_state_dict(self, sd):
        self.steps = int(sd["steps"])
        mom = sd["momentum"]
        if isinstance(mom, dict):
            for n, p, o in zip(self.flat.names, self.flat.params, self.flat.offsets):
                self.momentum_arena[o: o + p.numel()].copy_(mom[n].to(self.momentum_arena.device))
        else:   # flat arena in construction order (older resume files)
            self.momentum_arena.copy_(mom.to(self.momentum_arena.device))
        for g, s in zip(self.param_groups, sd["param_groups"]):
            g.update(s)


class Muon(FusedSGD):
    """Momentum orthogonalised by Newton-Schulz for matrices, fused SGD for the rest, over the flat
    arenas: one launch for every momentum and the rest's update, then the grouped
    orthogonalisation, whose last product adds to the parameters in place.

        buf = m buf + g;  u = g + m buf (nesterov) | buf
        p   = p (1 - lr wd) - lr max(1, rows / cols)^0.5 NS(u)

    ``matrices``: the parameters to treat so, each as [out channels, everything else] (default: every
    parameter of four dimensions, the convolution weights).  ``param_groups[0]`` holds them,
    ``param_groups[1]`` the rest with the ``rest_*`` settings of :class:`FusedSGD`; a scheduler drives
    both learning rates."""

    def __init__(self, module, lr=0.02, momentum=0.95, weight_decay=0.0, nesterov=True, ns_steps=5,
                 ns_coeffs=NS_COEFFS, eps=1e-7, rest_lr=0.1, rest_momentum=0.9, rest_weight_decay=1e-4,
                 rest_nesterov=True, matrices=None):
        if (nesterov and momentum <= 0) or (rest_nesterov and rest_momentum <= 0):
            raise ValueError("Nesterov momentum requires a momentum")
        if int(ns_steps) < 1:
            raise ValueError(f"Muon needs at least one Newton-Schulz step, got {ns_steps}")
        inner = getattr(module, "module", module)
        self.flat = get_flat(inner) or flatten_module(inner)
        chosen = {id(p) for p in (matrices if matrices is not None else
                                  [p for p in self.flat.params if p.dim() == 4])}
        if any(p.dim() < 2 for p in self.flat.params if id(p) in chosen):
            raise ValueError("Muon orthogonalises matrices: a chosen parameter has fewer than two dimensions")
        known = {id(p) for p in self.flat.params}
        if not chosen <= known:
            raise ValueError("Muon: a chosen parameter is not a trainable parameter of the module")
        mats = [p for p in self.flat.params if id(p) in chosen]
        rest = [p for p in self.flat.params if id(p) not in chosen]
        torch.optim.Optimizer.__init__(self, [
            dict(params=mats, lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov),
            dict(params=rest, lr=rest_lr, momentum=rest_momentum, weight_decay=rest_weight_decay,
                 nesterov=rest_nesterov)], {})
        self.ns = (int(ns_steps), tuple(float(c) for c in ns_coeffs), float(eps))
        # what the orthogonalisation refuses, it refuses here rather than in the middle of a step
        if any(max(p.shape[0], p.numel() // p.shape[0]) > 2 ** 20 for p in mats):
            raise ValueError("Muon: matrices of at most 2^20 rows and columns")
        one = torch.zeros(1, 1, device=self.flat.device)
        prims_for(one).newton_schulz_([one], [one.clone()], *self.ns, [1.0])
        self.momentum_arena = torch.zeros_like(self.flat.param_arena)
        self.flat.companions.append(self.momentum_arena)   # follows arena relayouts
        self.update_arena = torch.zeros_like(self.flat.param_arena)   # written and read within a step
        self.steps = 0
        self.lr_dev = None
        self._lr_cached = None
        self._views = None
        self._chosen = chosen

    def _matrix_views(self):
        """(updates, parameters, rates' factors, kinds) of the current arena layout."""
        fl = self.flat
        if self._views is None or self._views[0] != fl.version:
            upd, par, fac = [], [], []
            kinds = torch.zeros(fl.numel // 4, dtype=torch.uint8)
            for p, o in zip(fl.params, fl.offsets):
                if id(p) not in self._chosen:
                    continue
                n, rows = p.numel(), p.shape[0]
                kinds[o // 4: (o + n + 3) // 4] = 1
                # physical order: the columns of a channels-last weight come permuted, which the
                # orthogonalisation commutes with
                upd.append(self.update_arena[o: o + n].view(rows, n // rows))
                par.append(fl.param_arena[o: o + n].view(rows, n // rows))
                fac.append(-max(1.0, rows / (n // rows)) ** 0.5)
            self._views = (fl.version, upd, par, fac, kinds.to(fl.device))
        return self._views[1:]

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        m, r = self.param_groups
        fl = self.flat
        P = prims_for(fl.param_arena)
        if self.lr_dev is not None and not torch.cuda.is_current_stream_capturing():
            self.sync_lr()
        upd, par, fac, kinds = self._matrix_views()
        rule = [(float(g["lr"]), float(g["momentum"]), float(g["weight_decay"]), bool(g["nesterov"])) for g in (m, r)]
        P.muon_prep_(fl.param_arena, fl.grad_arena, self.momentum_arena, self.update_arena, kinds, rule[0], rule[1],
                     self.lr_dev, self.steps == 0)
        steps, coeffs, eps = self.ns
        if upd:
            dev_lr = None if self.lr_dev is None else self.lr_dev[:1]
            alpha = fac if dev_lr is not None else [f * rule[0][0] for f in fac]
            P.newton_schulz_(upd, par, steps, coeffs, eps, alpha, 1.0, dev_lr)
        self.steps += 1
        return loss

    def graph_safe(self):
        """Switch to device-resident learning rates (call before capturing a step)."""
        self._matrix_views()            # its upload cannot be captured
        if self.lr_dev is None:
            self.lr_dev = torch.zeros(2, dtype=torch.float32, device=self.flat.device)
            self._lr_cached = None
            self.sync_lr()
        return self

    def sync_lr(self):
        lr = tuple(float(g["lr"]) for g in self.param_groups)
        if lr != self._lr_cached:
            self.lr_dev[0].fill_(lr[0])
            self.lr_dev[1].fill_(lr[1])
            self._lr_cached = lr
