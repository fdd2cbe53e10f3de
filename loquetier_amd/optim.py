"""AdamW over the weights of all adapters at once: one launch, and one for the call's tables by 144 tensors, where torch's
optimizers run a chain of launches an adapter (the reference keeps a trainer, and so an optimizer, an adapter:
src/loquetier_src/trainer_utils.py)."""
from __future__ import annotations

import struct
from typing import Any, Callable, Dict, List, Optional, Tuple

import torch

from .ops import _kernels as kernel


class _Set:
    """The tensors of one type on one device: their flat states."""

    def __init__(self, params: List[torch.Tensor], groups: List[int], bits: int, master: bool):
        dev, dtype = params[0].device, params[0].dtype
        self.params = params
        self.first = [0]  # each tensor's first block, and the end
        for p in params:
            self.first.append(self.first[-1] - (-p.numel() // kernel.ADAMW_BLOCK))
        blocks = self.first[-1]
        n = blocks * kernel.ADAMW_BLOCK
        state = torch.float8_e4m3fn if bits == 8 else torch.float32
        zeros = lambda size, dt: torch.zeros(size, dtype=dt, device=dev)
        self.tensors: Dict[str, Optional[torch.Tensor]] = dict(
            exp_avg=zeros(n, torch.uint8).view(state) if bits == 8 else zeros(n, state),
            exp_avg_sq=zeros(n, torch.uint8).view(state) if bits == 8 else zeros(n, state),
            avg_scale=zeros(blocks, torch.float32) if bits == 8 else None,
            sq_scale=zeros(blocks, torch.float32) if bits == 8 else None,
            # (zeros are the rounding of no weight but 0: each one takes its place at the first step)
            master=zeros(n, torch.float32) if master and dtype != torch.float32 else None,
            step=zeros(len(params), torch.int32))
        self.groups, self.group = groups, kernel.put_ints(dev, [], groups)[1]
        self.workspace = kernel.Workspace(dev)

    def regroup(self, groups: List[int]) -> None:
        """Other groups of the tensors (-1: none, and the tensor stays as it is), in the place that captured steps read."""
        if groups != self.groups:
            kernel.put_words(self.group, struct.pack(f"{len(groups)}i", *groups))
            self.groups = groups

    def __getstate__(self) -> Dict[str, Any]:
        # (the workspace is for the steps captured here; torch pickles no tensors of 8-bit floats, so they go as bytes)
        tensors = {n: t if t is None or t.dtype != torch.float8_e4m3fn else t.view(torch.uint8) for n, t in self.tensors.items()}
        return dict({n: v for n, v in self.__dict__.items() if n != "workspace"}, tensors=tensors)

    def __setstate__(self, state: Dict[str, Any]) -> None:
        self.__dict__.update(state)
        self.tensors = {n: t if t is None or t.dtype != torch.uint8 else t.view(torch.float8_e4m3fn) for n, t in self.tensors.items()}
        self.workspace = kernel.Workspace(self.group.device)

    def parts(self, i: int) -> Dict[str, Optional[torch.Tensor]]:
        """A tensor's share of the states, whole blocks."""
        first, end = self.first[i:i + 2]
        flat = slice(first * kernel.ADAMW_BLOCK, end * kernel.ADAMW_BLOCK)
        of = dict(avg_scale=slice(first, end), sq_scale=slice(first, end), step=slice(i, i + 1))
        return {n: None if t is None else t[of.get(n, flat)] for n, t in self.tensors.items()}


class AdamW(torch.optim.Optimizer):
    """`AdamW(params, lr, betas, eps, weight_decay)` with decoupled weight decay, as torch.optim.AdamW's arguments: params
    are tensors or groups of them (an adapter a group, say) on GPUs, fp16, bf16 or float32, contiguous, each in one group once.

    state_bits 32: averages in float; 8: in e4m3 with a float scale each for 256 weights.  master: float weights beside 16-bit ones,
    which are their rounding (small updates add up that a 16-bit weight would lose); a weight that somebody sets is taken over
    at the next step.  A tensor without a gradient stays as it is, its average's age too, so adapters may take steps by turns; one whose
    group is taken out of `param_groups` stays too, where it lies, and goes on if it comes back.

    Step counts live on the device, so `step` may be captured into a graph after one eager step; the groups' rates too: `step`
    writes those that have changed, between replays `update_rates` does.  Nothing waits for the GPU."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, master: bool = True):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self.state_bits, self.master = state_bits, bool(master)
        self._sets: List[_Set] = []
        self._order: List[List[int]] = []  # the groups' tensors by id, as the sets have them
        self._captured = False  # whether a step was
        # what was written, and the tables: the newest, and smaller ones that a captured step may read
        self._rates: Dict[torch.device, Tuple[tuple, List[torch.Tensor]]] = {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self) -> Dict[str, Any]:
        return dict(super().__getstate__(), state_bits=self.state_bits, master=self.master, _sets=self._sets)

    def __setstate__(self, state: Dict[str, Any]) -> None:
        super().__setstate__(state)
        if "_sets" in state:  # (a copy, or what was pickled: the rates' tables are for the steps captured here)
            self._rates, self._order, self._captured = {}, [], False

    def add_param_group(self, param_group: Dict[str, Any]) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        lr, (b1, b2) = float(group["lr"]), group["betas"]
        if lr < 0 or group["eps"] < 0 or group["weight_decay"] < 0 or not (0 <= b1 < 1 and 0 <= b2 < 1):
            self.param_groups.pop()
            raise ValueError("lr, eps and weight_decay must not be negative, betas lie in [0, 1)")

    def _prepare(self) -> None:
        """States of the tensors that have none yet, and the groups of those that have."""
        order = [list(map(id, group["params"])) for group in self.param_groups]
        if order == self._order:
            return
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the states must be made, and tensors take their groups, before a graph is captured: run an eager step")
        group_of = {i: g for g, ids in enumerate(order) for i in ids}
        have = {id(p) for s in self._sets for p in s.params}
        kinds: Dict[tuple, Tuple[list, list]] = {}
        for group in self.param_groups:
            for p in group["params"]:
                if id(p) in have:
                    continue
                if not p.is_cuda or not p.is_contiguous() or p.dtype not in (torch.float16, torch.bfloat16, torch.float32):
                    raise RuntimeError("No suitable kernel: parameters must be contiguous fp16, bf16 or float32 tensors on a GPU")
                ps, gs = kinds.setdefault((p.device, p.dtype), ([], []))
                ps.append(p), gs.append(group_of[id(p)])
        rows = min((tables[0].size(0) for _, tables in self._rates.values()), default=0)
        groups = [[group_of.get(id(p), -1) for p in s.params] for s in self._sets]
        if self._captured and any(g != was and g >= rows for s, now in zip(self._sets, groups) for g, was in zip(now, s.groups)):
            raise RuntimeError("a captured step's table has no row for a group that others were put before: append them")
        for s, now in zip(self._sets, groups):  # (a group that was taken out, or moved up because another was)
            s.regroup(now)
        self._sets += [_Set(ps, gs, self.state_bits, self.master) for ps, gs in kinds.values()]
        self._order = order

    def update_rates(self) -> None:
        """Writes the groups' lr, betas, eps and weight decay to the device where they have changed (step does so itself; a captured
        step reads what is there at its replay)."""
        self._prepare()
        now = tuple((float(g["lr"]), float(g["betas"][0]), float(g["betas"][1]), float(g["eps"]), float(g["weight_decay"]))
                    for g in self.param_groups)
        for dev in {s.params[0].device for s in self._sets}:
            was = self._rates.get(dev)
            if was is not None and was[0] == now:
                continue
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("rates changed while a graph is captured: call update_rates before")
            tables = was[1] if was is not None else []
            if not tables or tables[-1].size(0) < len(now):
                tables.append(torch.empty(len(now), 5, device=dev))
            for table in tables:  # (rows that no group has any more are zeros)
                rows = [*now, *[(0.0,) * 5] * table.size(0)][:table.size(0)]
                kernel.put_words(table, struct.pack(f"{table.numel()}f", *[v for row in rows for v in row]))
            self._rates[dev] = (now, tables)

    @torch.no_grad()
    def step(self, closure: Optional[Callable[[], torch.Tensor]] = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.update_rates()
        self._captured = self._captured or bool(self._sets) and torch.cuda.is_current_stream_capturing()
        for s in self._sets:
            grads = [p.grad for p in s.params]
            if any(g is not None and not g.is_contiguous() for g in grads):
                grads = [g if g is None else g.contiguous() for g in grads]
            if any(g is not None for g in grads):
                t = s.tensors
                kernel.adamw_step(s.params, grads, t["exp_avg"], t["exp_avg_sq"], t["step"], self._rates[s.params[0].device][1][-1],
                                  s.group, t["avg_scale"], t["sq_scale"], t["master"], s.workspace)
        return loss

    def state_of(self, param: torch.Tensor) -> Dict[str, torch.Tensor]:
        """Copies of a tensor's step count and averages (and float weights), float tensors of its shape."""
        self._prepare()
        for s in self._sets:
            for i, p in enumerate(s.params):
                if p is not param:
                    continue
                t = s.parts(i)
                values = lambda name, scale: (t[name].clone() if scale is None else (
                    t[name].view(-1, kernel.ADAMW_BLOCK).float() * scale[:, None]).flatten())[:p.numel()].view(p.shape)
                out = dict(step=t["step"][0].clone(), exp_avg=values("exp_avg", t["avg_scale"]),
                           exp_avg_sq=values("exp_avg_sq", t["sq_scale"]))
                if self.state_bits == 8:
                    out["exp_avg_sq"] = out["exp_avg_sq"].square()
                if t["master"] is not None:
                    out["master"] = t["master"][:p.numel()].view(p.shape).clone()
                return out
        raise KeyError("not one of the optimizer's tensors")

    def _kinds(self) -> List[List[Tuple[_Set, int]]]:
        """Where the tensors' states are, those of a type on a device together in the groups' order: as one set would hold them
        if all had been there from the start."""
        where = {id(p): (s, i) for s in self._sets for i, p in enumerate(s.params)}
        kinds: Dict[tuple, List[Tuple[_Set, int]]] = {}
        for group in self.param_groups:
            for p in group["params"]:
                if id(p) in where:
                    kinds.setdefault((p.device, p.dtype), []).append(where[id(p)])
        return list(kinds.values())

    def _shapes(self) -> List[List[Tuple[int, ...]]]:
        return [[tuple(s.params[i].shape) for s, i in kind] for kind in self._kinds()]

    def state_dict(self) -> Dict[str, Any]:
        out = super().state_dict()
        if self._sets:
            self._prepare()  # (of a group that has joined since the last step too)
        sets = []
        for kind in self._kinds():
            parts = [s.parts(i) for s, i in kind]
            join = lambda ts: None if ts[0] is None else torch.cat([t.view(torch.uint8) for t in ts]).view(ts[0].dtype)
            sets.append({n: join([p[n] for p in parts]) for n in parts[0]})
        out["state"] = {"bits": self.state_bits, "sets": sets, "shapes": self._shapes()}
        return out

    def load_state_dict(self, state_dict: Dict[str, Any]) -> None:
        """Takes over what `state_dict` gave; what is not of these tensors is refused before anything changes."""
        state, kinds = state_dict["state"], []
        if "sets" not in state:
            raise ValueError("the saved states are not this optimizer's")
        if state["sets"]:
            self._prepare()
            kinds = [[s.parts(i) for s, i in kind] for kind in self._kinds()]
            shape = lambda tensors: {n: None if t is None else (t.dtype, tuple(t.shape)) for n, t in tensors.items()}
            mine = [{n: None if t is None else (t.dtype, (sum(p[n].size(0) for p in parts),)) for n, t in parts[0].items()} for parts in kinds]
            if (state["bits"] != self.state_bits or mine != [shape(s) for s in state["sets"]] or
                    # (tensors of other sizes may fill as many blocks; states without shapes are of an older program)
                    state.get("shapes", self._shapes()) != self._shapes()):
                raise ValueError("the saved states are of other tensors, or of another number of bits")
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        if not state["sets"]:  # (saved before its first step)
            for s in self._sets:
                for t in s.tensors.values():
                    if t is not None:
                        t.view(torch.uint8).zero_()
        for parts, saved in zip(kinds, state["sets"]):
            for name, t in saved.items():
                if t is not None:
                    for part, of in zip(parts, t.split([p[name].size(0) for p in parts])):
                        part[name].view(torch.uint8).copy_(of.view(torch.uint8))
