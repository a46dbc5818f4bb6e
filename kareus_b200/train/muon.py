"""Muon over the flat buffers of :class:`.optimizer.DistributedAdamW`: orthogonalised momentum for the layers' weight matrices,
AdamW for every other parameter.

A matrix takes ``kernels.muon_step`` on views of the flat parameter, gradient, momentum (``exp_avg``) and master buffers; its
``exp_avg_sq`` stays zero, so checkpoints have the layout of AdamW's.  The update has the root mean square of an AdamW update
(``0.2 * sqrt(max(rows, columns))`` times an orthogonal matrix), so learning rate, weight decay and gradient clipping mean the same for
both kinds of parameters.

An update needs a whole matrix.  With data parallelism gradients are all-reduced (AdamW's reduce-scatter cuts through matrices),
each matrix has one owner that holds its momentum and master values and computes its update, and the owners broadcast the new
weights; AdamW's parameters stay sharded.  Weights that tensor parallelism cuts are refused."""
from __future__ import annotations

from typing import Iterable, List, Optional, Tuple

import torch
import torch.distributed as dist

from .. import kernels as K
from ..config import TrainConfig
from .optimizer import _ALIGN, DistributedAdamW, cosine_lr


class DistributedMuon(DistributedAdamW):
    def __init__(self, params: Iterable[torch.nn.Parameter], cfg: TrainConfig, matrices: Iterable[torch.nn.Parameter], dp_group=None,
                 dp_size: int = 1, dp_rank: int = 0, mp_group=None, tp_size: int = 1):
        if tp_size != 1:
            raise ValueError("Muon needs whole weight matrices: tensor parallelism cuts them (tp must be 1)")
        super().__init__(params, cfg, dp_group=dp_group, dp_size=dp_size, dp_rank=dp_rank, mp_group=mp_group, tp_rank=0)
        wanted = {id(p) for p in matrices}
        # (first element, rows, columns) of every matrix; a parameter may hold several, one behind the other
        self.matrices: List[Tuple[int, int, int]] = []
        for p, off in zip(self.params, self.offsets):
            if id(p) not in wanted:
                continue
            if p.dim() != 2:
                raise ValueError(f"Muon takes matrices, got a parameter of shape {tuple(p.shape)}")
            parts = int(getattr(p, "matrices", 1))
            if p.shape[0] % parts:
                raise ValueError(f"{p.shape[0]} rows are not {parts} matrices")
            rows = p.shape[0] // parts
            self.matrices += [(off + i * rows * p.shape[1], rows, p.shape[1]) for i in range(parts)]
        # what is left for AdamW, as ranges of the flat space
        self.adamw_ranges: List[Tuple[int, int]] = []
        at = 0
        for off, rows, cols in sorted(self.matrices):
            if off > at:
                self.adamw_ranges.append((at, off))
            at = -(-(off + rows * cols) // _ALIGN) * _ALIGN       # ranges start where parameters do
        if at < self.total:
            self.adamw_ranges.append((at, self.total))
        # owners: the largest matrices first, each to the rank with the least work so far
        load = [0] * self.dp
        self.owner = [0] * len(self.matrices)
        for i in sorted(range(len(self.matrices)), key=lambda i: -_work(*self.matrices[i][1:])):
            self.owner[i] = min(range(self.dp), key=load.__getitem__)
            load[self.owner[i]] += _work(*self.matrices[i][1:])
        # momentum and master of the matrices that this rank owns; at dp == 1 the flat buffers hold them
        self._own = {}
        if self.dp > 1:
            for i, (off, rows, cols) in enumerate(self.matrices):
                if self.owner[i] == self.dp_rank:
                    w = self.param_flat[off:off + rows * cols]
                    self._own[i] = (torch.zeros(rows * cols, dtype=self.m.dtype, device=w.device), w.to(self.m.dtype).clone())
        self._apart = set(self._own)

    def _state(self, i: int):
        """(momentum, master) of matrix ``i``, flat; the caller owns it."""
        if self.dp > 1:
            return self._own[i]
        off, rows, cols = self.matrices[i]
        return self.m[off:off + rows * cols], self.master[off:off + rows * cols]

    def _reduce_grads(self) -> torch.Tensor:
        if self.dp > 1:
            dist.all_reduce(self.grad_flat, group=self.dp_group)
        return self.grad_flat

    def _grad_norm_all(self) -> torch.Tensor:
        """Global L2 norm; every data-parallel rank holds all gradients."""
        total = K.sumsq(self.grad_flat)
        for a, b in self.norm_exclude:
            total = total - K.sumsq(self.grad_flat[a:b])
        total = total.reshape(1).clone()
        if self.mp_group is not None:
            dist.all_reduce(total, group=self.mp_group)
        return total.sqrt()[0]

    def step(self, lr: Optional[float] = None) -> torch.Tensor:
        cfg = self.cfg
        g = self._reduce_grads()
        norm = self._grad_norm_all()
        self.last_grad_norm = norm
        scale_t = None
        if cfg.grad_clip and cfg.grad_clip > 0:
            scale_t = torch.clamp(cfg.grad_clip / (norm + 1e-6), max=1.0).to(torch.float32).reshape(1)
        self.step_count += 1
        lr = cosine_lr(self.step_count - 1, cfg) if lr is None else lr
        for a, b in self.adamw_ranges:
            a, b = max(a, self.lo), min(b, self.hi)
            if b > a:
                self._adamw(g, a, b, lr, scale_t)
        if self.dp > 1:
            dist.all_gather_into_tensor(self.param_flat, self.param_flat[self.lo:self.hi].clone(), group=self.dp_group)
        for i, (off, rows, cols) in enumerate(self.matrices):
            if self.owner[i] != self.dp_rank:
                continue
            m, master = self._state(i)
            shape, end = (rows, cols), off + rows * cols
            K.muon_step(self.param_flat[off:end].view(shape), g[off:end].view(shape), m.view(shape), master.view(shape), lr=lr,
                        momentum=cfg.muon_momentum, weight_decay=cfg.weight_decay, steps=cfg.muon_steps, grad_scale_tensor=scale_t)
        if self.dp > 1:
            for i, (off, rows, cols) in enumerate(self.matrices):
                dist.broadcast(self.param_flat[off:off + rows * cols], src=self._rank_of(self.owner[i]), group=self.dp_group)
        return norm

    def _adamw(self, g, a: int, b: int, lr: float, scale_t) -> None:
        cfg, lo = self.cfg, self.lo
        args = (self.param_flat[a:b], g[a:b], self.m[a - lo:b - lo], self.v[a - lo:b - lo], self.master[a - lo:b - lo], lr, cfg.betas[0],
                cfg.betas[1], cfg.eps, cfg.weight_decay, self.step_count)
        if g.is_cuda and g.dtype == torch.float32:
            from ..kernels import cuda as KC
            KC.adamw_step(*args, 1.0, grad_scale_tensor=scale_t)
        else:
            K.ref.adamw_step(*args, float(scale_t.item()) if scale_t is not None else 1.0)

    def _rank_of(self, dp_rank: int) -> int:
        return dist.get_global_rank(self.dp_group, dp_rank) if self.dp_group is not None else dp_rank

    # ------------------------------------------------------------------ checkpoint
    def gather_state(self) -> dict:
        out = super().gather_state()
        if self.dp > 1:
            for i, (off, rows, cols) in enumerate(self.matrices):
                end = off + rows * cols
                for name, k in (("exp_avg", 0), ("fp32_param", 1)):
                    if self.owner[i] == self.dp_rank:
                        out[name][off:end].copy_(self._own[i][k])
                    dist.broadcast(out[name][off:end], src=self._rank_of(self.owner[i]), group=self.dp_group)
        return out

    def scatter_state(self, full: dict, step: int) -> None:
        super().scatter_state(full, step)
        for i, (m, master) in self._own.items():
            off, rows, cols = self.matrices[i]
            m.copy_(full["exp_avg"][off:off + rows * cols])
            master.copy_(full["fp32_param"][off:off + rows * cols])

    def state_dict(self) -> dict:
        sd = super().state_dict()
        sd["muon"] = {i: tuple(t for t in self._own[i]) for i in self._own}
        return sd

    def load_state_dict(self, sd: dict) -> None:
        own = sd.get("muon", {})              # a state of AdamW has none; neither has one of a single rank
        if set(own) != set(self._own):
            raise ValueError("owners of the weight matrices differ from the checkpoint's")
        # the flat master buffer holds no current values of matrices with an owner: their weights stay (another rank's, which come
        # with the model) or follow from the owner's
        weights = [self.param_flat[off:off + rows * cols].clone() for off, rows, cols in self.matrices] if self.dp > 1 else []
        super().load_state_dict(sd)
        for (off, rows, cols), w in zip(self.matrices, weights):
            self.param_flat[off:off + rows * cols].copy_(w)
        for i, state in own.items():
            off, rows, cols = self.matrices[i]
            for mine, theirs in zip(self._own[i], state):
                mine.copy_(theirs)
            self.param_flat[off:off + rows * cols].copy_(self._own[i][1].to(self.param_flat.dtype))


def _work(rows: int, cols: int) -> int:
    side = min(rows, cols)
    return side * side * (3 * max(rows, cols) + side)
