"""A paged key-value cache on the device: the pool of pages, the requests' page tables and their care, and the calls of a
step that read them (the reference keeps both in Python lists, kernel_src/src/loquetier/utils/kvcache.py, and hands
pointers to its init_kv / append_kv / batch_prefill / batch_decode, kernel_src/csrc/loquetier_ops.cc:90-273).

Nothing here waits for the GPU except `check`, and lists of more than 3584 entries, which are copied where shorter ones travel in a
launch's arguments (tensors on the device are read where they lie)."""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .ops import _kernels as kernel

Ints = Union[torch.Tensor, Sequence[int]]


class KvStep(NamedTuple):
    """The tables of one step, shared by its layers."""
    q_indptr: torch.Tensor   # int32 [S + 1] rows of the sequences
    kv_len: torch.Tensor     # int32 [S] tokens in the cache, the new ones too
    positions: torch.Tensor  # int32 [rows], -1: a row of no sequence
    slots: torch.Tensor      # int64 [rows]
    requests: torch.Tensor   # int32 [S]


class PagedKvCache:
    """`n_pages` pages of `page_size` tokens for all layers, [n_pages, n_layers, 2 (keys, values), kv_heads, page_size, head_dim] as the
    reference's pages are laid out, and up to `max_requests` requests of up to `max_tokens` tokens each (`extend` refuses more, so
    a rotation table of `max_tokens` positions serves), known by their number.  All calls are ordered on the current stream and
    may be captured into a graph after one eager pass."""

    def __init__(self, n_pages: int, n_layers: int, kv_heads: int, head_dim: int, max_requests: int, max_tokens: int,
                 page_size: int = 16, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if dtype not in kernel._DTYPE_CODE or head_dim not in kernel._ATTENTION_DIMS:  # (now, not once its pages hold keys)
            raise RuntimeError(f"No suitable kernel. dtype={dtype} head_dim={head_dim}")
        self.pool = torch.zeros(n_pages, n_layers, 2, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.page_size, self.kv_heads, self.max_tokens = page_size, kv_heads, int(max_tokens)
        ints = dict(dtype=torch.int32, device=self.pool.device)
        self.table = torch.full((max_requests, -(-max_tokens // page_size)), -1, **ints)
        self.length = torch.zeros(max_requests, **ints)
        self.refs = torch.zeros(n_pages, **ints)
        self.status = torch.zeros(1, **ints)
        self.workspace = kernel.Workspace(self.pool.device)

    def _ints(self, v: Ints) -> torch.Tensor:
        if isinstance(v, torch.Tensor):
            return v
        return kernel.put_ints(self.pool.device, [], [int(i) for i in v])[1]

    def layer(self, i: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of a layer, [n_pages, kv_heads, page_size, head_dim] views."""
        return self.pool[:, i, 0], self.pool[:, i, 1]

    def extend(self, requests: Ints, counts: Ints, n_rows: Optional[int] = None) -> KvStep:
        """Room for counts[s] new tokens of requests[s], in the batch's order, and the step's tables.  n_rows: rows of the batch
        (the counts' sum, which a caller with counts on the device names).  The places are given out before they are written: the
        step's `attend` calls, all layers', come before the next `fork` or `free` of its requests and the next `compact`."""
        if n_rows is None:
            if isinstance(counts, torch.Tensor):
                raise RuntimeError("n_rows is needed where the counts are on the device")
            n_rows = sum(int(c) for c in counts)
        requests = self._ints(requests)
        return KvStep(*kernel.kv_extend(self.table, self.length, self.refs, requests, self._ints(counts), n_rows, self.page_size,
                                        self.status, self.workspace, self.max_tokens), requests)

    def fork(self, parents: Ints, children: Ints) -> None:
        kernel.kv_fork(self.pool, self.table, self.length, self.refs, self._ints(parents), self._ints(children), self.status,
                       self.workspace)

    def free(self, requests: Ints) -> None:
        kernel.kv_free(self.table, self.length, self.refs, self._ints(requests), self.page_size, self.status)

    def compact(self) -> None:
        """Packs the pages in use to the pool's front.  Between steps: the slots of a step that was extended before name pages as they
        lay then."""
        kernel.kv_compact(self.pool, self.table, self.refs, self.workspace)

    def plan(self, step: KvStep, q_heads: int) -> kernel.AttentionPlan:
        """The step's attention plan, for all its layers."""
        return kernel.AttentionPlan(step.q_indptr, step.kv_len, self.table, step.positions.size(0), q_heads, self.kv_heads,
                                    self.page_size, step.requests)

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: KvStep, plan: kernel.AttentionPlan,
               table: torch.Tensor, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
               eps: float = 1e-6, scale: Optional[float] = None) -> torch.Tensor:
        """A layer's attention from its projections' outputs [rows, heads, head_dim] (views of one tensor will do): norms and rotation,
        keys and values to the cache, attention.  table: rope_table's."""
        k_cache, v_cache = self.layer(layer)
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        kernel.qk_norm_rope(q_out, None, q, k, table, step.positions, q_weight, k_weight, eps, v, k_cache, v_cache, step.slots)
        # in place: rows of no sequence have no position, so their queries are zero, and stay
        kernel.paged_attention(q_out, q_out, k_cache, v_cache, plan, scale, self.workspace)
        return q_out

    def check(self) -> None:
        """Raises where a call since the last check was refused (waits for the GPU)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            names = {_lib.SMLM_KV_BAD_REQUEST: "a request that is unknown, named twice or not empty",
                     _lib.SMLM_KV_TOO_LONG: "a request longer than max_tokens", _lib.SMLM_KV_ROWS: "more tokens than rows",
                     _lib.SMLM_KV_NO_PAGES: "no free pages"}
            raise RuntimeError("the cache refused a call: " + ", ".join(n for b, n in names.items() if bits & b))
