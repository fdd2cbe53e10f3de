"""Python surface of the HIP library, with the names and argument order of the
reference's pybind module `loquetier.ops._kernels`
(kernel_src/csrc/loquetier_ops.cc:365-374) for the SMLM entries, plus the
fused forward, the backward and the plan builder this build adds.

Tensors are torch tensors on a ROCm device; the calls are asynchronous on
torch's current stream of that device.  Nothing here computes on the host.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Dict, Optional, Tuple

import torch

from .. import _lib

_DTYPE_CODE = {torch.float16: _lib.SMLM_DTYPE_F16, torch.bfloat16: _lib.SMLM_DTYPE_BF16}

class Workspace:
    """Scratch memory for the kernels (plans of unplanned calls, k-split partial sums, the rounded v and
    dV, and their transposed copies for the weight gradients).

    The C ABI allocates nothing: every call is handed a buffer at least as large as its
    `*_workspace_size` query says.  A Workspace owns such a buffer.  It only ever grows, a
    buffer that was handed out is never freed while the Workspace lives (a captured HIP graph
    keeps the raw address of the buffer it was captured with), and it refuses to grow while
    its stream is being captured: size it first, with `reserve` or with one eager pass.
    Calls that share a Workspace must be ordered on one stream."""

    def __init__(self, device: torch.device, nbytes: int = 0):
        self.device = torch.device(device)
        self._buf: Optional[torch.Tensor] = None
        self._retired = []
        if nbytes:
            self.reserve(nbytes)

    def reserve(self, nbytes: int) -> torch.Tensor:
        if self._buf is None or self._buf.numel() < nbytes:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(
                    f"the workspace must grow to {nbytes} bytes during a graph capture: reserve it "
                    "before capturing (Workspace.reserve, or one eager pass of the same calls)")
            if self._buf is not None:
                self._retired.append(self._buf)
            self._buf = torch.empty(max(nbytes, 1 << 20) * 3 // 2, dtype=torch.uint8, device=self.device)
        return self._buf


# default workspaces, one per (device index, stream handle): calls on one stream are ordered,
# so they can share one buffer.  Callers that want to own the memory pass `workspace=`.
_WORKSPACES: Dict[Tuple[int, int], Workspace] = {}


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev: torch.device) -> int:
    # (the handle itself where torch hands it out: building a torch.cuda.Stream object around it costs
    # microseconds per call)
    if _raw_stream is None:
        return torch.cuda.current_stream(dev).cuda_stream
    return _raw_stream(dev.index if dev.index is not None else torch.cuda.current_device())


class _NoSwitch:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_SWITCH = _NoSwitch()


def _on(dev: torch.device):
    """Context that makes `dev` the current device; nothing to do (and nothing spent) when it already is."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return _NO_SWITCH
    return torch.cuda.device(dev)


def _workspace(dev: torch.device, nbytes: int, own: Optional[Workspace] = None) -> torch.Tensor:
    if own is not None:
        buf = own.reserve(nbytes)
        if buf.device != dev:
            raise RuntimeError(f"workspace lives on {buf.device}, the tensors on {dev}")
        return buf
    key = (dev.index if dev.index is not None else torch.cuda.current_device(), _stream(dev))
    ws = _WORKSPACES.get(key)
    if ws is None:
        ws = _WORKSPACES[key] = Workspace(dev)
    return ws.reserve(nbytes)


def _host():
    """The native host path (loaded at the first call that can take it: it needs the built libraries)."""
    return _lib._host or _lib.host(_workspace)


def _check_input(t: torch.Tensor, name: str) -> None:
    # CHECK_INPUT of kernel_src/csrc/loquetier_ops.cc:32-38
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _check_dim(d: int, t: torch.Tensor, name: str) -> None:
    if t.dim() != d:
        raise RuntimeError(f"{name} must be a {d}D tensor")


def _dtype_code(t: torch.Tensor) -> int:
    code = _DTYPE_CODE.get(t.dtype)
    if code is None:
        raise RuntimeError(f"No suitable kernel. dtype={t.dtype}")
    return code


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def smlm_forward_cutlass_tmp_size(num_problems: int) -> int:
    """Bytes of the `tmp` tensor `smlm_forward_cutlass` expects
    (reference: smlm_forward_tmp_size, smlm_forward_cutlass.cuh:48-52)."""
    return _lib.size_query("smlm_tmp_size", int(num_problems))


def smlm_forward_cutlass_workspace_size(T: int, num_problems: int, d_in: int, d_out: int) -> int:
    """Bytes of a `tmp` that smlm_forward_cutlass uses as its ONLY scratch (plan and k-split partial sums of a
    [T, d_in] x [d_in, d_out] batch of num_problems segments): a caller that passes a tmp of at least this size
    owns every byte the call touches.  No counterpart in the reference, whose 60 bytes a problem hold all it needs."""
    return _lib.size_query("smlm_gemm_workspace_size", int(T), int(num_problems), int(d_in), int(d_out))


def smlm_forward_cutlass(y: torch.Tensor, x: torch.Tensor, w_ptr: torch.Tensor, s: torch.Tensor,
                         tmp: torch.Tensor, is_row_major: bool) -> None:
    """Grouped GEMM y[s_i:s_{i+1}] = x[s_i:s_{i+1}] @ W_i, overwriting y.

    Same contract as dispatch_smlm_forward_cutlass
    (kernel_src/csrc/loquetier_ops.cc:277-319): y [T,d_out], x [T,d_in] fp16 or
    bf16, w_ptr int64 [S] device addresses, s int32 [S+1], tmp uint8 of exactly
    smlm_forward_cutlass_tmp_size(S) bytes.  Unlike the reference it does not
    block the host.  The kernels here need more scratch than that tmp holds: with a tmp of the
    reference's size it comes from a buffer this module keeps per (device, stream); a tmp of
    smlm_forward_cutlass_workspace_size(T, S, d_in, d_out) bytes or more (16-byte aligned) is
    used itself, and the call then touches no memory the caller did not hand it.
    """
    for t, n in ((y, "y"), (x, "x"), (w_ptr, "w_ptr"), (s, "s"), (tmp, "tmp")):
        _check_input(t, n)
    _check_dim(2, y, "y")
    _check_dim(2, x, "x")
    _check_dim(1, w_ptr, "w_ptr")
    _check_dim(1, s, "s")
    _check_dim(1, tmp, "tmp")
    num_problems = s.size(0) - 1
    d_in, d_out = x.size(1), y.size(1)
    w_ld = d_out if is_row_major else d_in
    if w_ptr.dtype != torch.int64 or s.dtype != torch.int32:
        raise RuntimeError("w_ptr must be int64 and s must be int32")
    if w_ptr.size(0) != num_problems or y.size(0) != x.size(0) or y.dtype != x.dtype:
        raise RuntimeError("inconsistent shapes: w_ptr [S], s [S+1], x [T,d_in], y [T,d_out]")
    code = _dtype_code(x)
    T = x.size(0)
    dev = tmp.device
    with _on(dev):
        need = _lib.size_query("smlm_gemm_workspace_size", T, num_problems, d_in, d_out)
        own = tmp.size(0) >= need and tmp.size(0) != smlm_forward_cutlass_tmp_size(num_problems)
        if not own and tmp.size(0) != smlm_forward_cutlass_tmp_size(num_problems):
            raise RuntimeError(f"CHECK_EQ(tmp.size(0), smlm_forward_tmp_size(num_problems)) failed: "
                               f"{tmp.size(0)} vs {smlm_forward_cutlass_tmp_size(num_problems)}")
        if own and tmp.data_ptr() % 16:
            raise RuntimeError("a tmp that serves as the workspace must be 16-byte aligned")
        ws = tmp if own else _workspace(dev, need)
        rc = _lib.load().smlm_gemm(y.data_ptr(), x.data_ptr(), w_ptr.data_ptr(), s.data_ptr(),
                                   ws.data_ptr(), ws.numel(), T, num_problems, d_in, d_out, w_ld,
                                   int(bool(is_row_major)), code, 0.0, None, _stream(dev))
    if rc == _lib.SMLM_ERR_DTYPE:
        raise RuntimeError(f"No suitable kernel. dtype={x.dtype}")
    _lib.check(rc, "smlm_forward_cutlass")


def smlm_forward_cutlass_static(y: torch.Tensor, x: torch.Tensor, w_ptr: torch.Tensor, s: torch.Tensor,
                                is_row_major: bool, beta: float = 0.0,
                                seg_scale: Optional[torch.Tensor] = None) -> None:
    """smlm_forward_cutlass without `tmp` and without any allocation (smlm_gemm_static): the
    scratch is an array inside the library, SMLM_STATIC_SCRATCH_BYTES per GPU, shared by all
    calls on that GPU -- keep them on one stream.  Raises when the batch needs more."""
    for t, n in ((y, "y"), (x, "x"), (w_ptr, "w_ptr"), (s, "s")):
        _check_input(t, n)
    _check_dim(2, y, "y")
    _check_dim(2, x, "x")
    _check_dim(1, w_ptr, "w_ptr")
    _check_dim(1, s, "s")
    num_problems = s.size(0) - 1
    if w_ptr.dtype != torch.int64 or s.dtype != torch.int32:
        raise RuntimeError("w_ptr must be int64 and s must be int32")
    if w_ptr.size(0) != num_problems or y.size(0) != x.size(0) or y.dtype != x.dtype:
        raise RuntimeError("inconsistent shapes: w_ptr [S], s [S+1], x [T,d_in], y [T,d_out]")
    if seg_scale is not None and (seg_scale.dtype != torch.float32 or seg_scale.numel() != num_problems
                                  or not seg_scale.is_cuda):
        raise RuntimeError("seg_scale must be a device float32 tensor with one entry per segment")
    code = _dtype_code(x)
    d_in, d_out = x.size(1), y.size(1)
    dev = x.device
    with _on(dev):
        rc = _lib.load().smlm_gemm_static(y.data_ptr(), x.data_ptr(), w_ptr.data_ptr(), s.data_ptr(),
                                          x.size(0), num_problems, d_in, d_out,
                                          d_out if is_row_major else d_in, int(bool(is_row_major)), code,
                                          float(beta), _ptr(seg_scale), _stream(dev))
    _lib.check(rc, "smlm_forward_cutlass_static")


_PUT_BYTES = 4 * 3584  # more words than four launches carry are copied


def put_ints(device: torch.device, words64, words32) -> Tuple[torch.Tensor, torch.Tensor]:
    """Small host tables as device tensors (int64, int32) that share one allocation, without waiting for the device:
    the words travel in a launch's arguments (smlm_put_words); long tables in one copy."""
    n64, n32 = len(words64), len(words32)
    try:
        data = struct.pack(f"={n64}q{n32 + (n32 & 1)}i", *words64, *words32, *((0,) * (n32 & 1)))
    except struct.error as e:
        raise RuntimeError(f"a table entry does not fit its type: {e}") from None
    if len(data) > _PUT_BYTES or (data and torch.device(device).type != "cuda"):
        buf = torch.frombuffer(bytearray(data), dtype=torch.int64).to(device)
    else:
        buf = torch.empty(len(data) // 8, dtype=torch.int64, device=device)
        dev = buf.device
        with _on(dev):
            rc = _lib.load().smlm_put_words(buf.data_ptr(), data, len(data), _stream(dev))
        _lib.check(rc, "put_ints")
    return buf[:n64], buf[n64:].view(torch.int32)[:n32]


class SegmentPlan:
    """Tile plan of one flat batch: built once from (segment, adapter ids) and
    shared by every LoRA linear of the step (the reference rebuilds its
    per-problem table inside every kernel call,
    smlm_forward_cutlass.cuh:76-79).

    seg_key: None (every segment its own group), int32 adapter ids, int64 weight addresses, or a
    PAIR of int64 address tensors (wa_ptr, wb_ptr) as the reference's add_lora.forward is handed
    them (kernel_utils.py:115-119): segments are then grouped where both addresses agree, and one
    plan serves both GEMMs of the fused forward (per-segment tables).

    defer=True (plans keyed by int32 adapter ids or by a pair of address tensors): nothing is
    launched here; the first smlm_lora_forward(_multi) or smlm_lora_backward call that gets the
    plan builds it -- for batches of few enough segments inside its first launch, at no launch of
    its own -- and every other user builds it with the plan launch first (ensure_built)."""

    def __init__(self, segment: torch.Tensor, seg_key: Optional[torch.Tensor], T: int,
                 buf: Optional[torch.Tensor] = None, defer: bool = False):
        _check_input(segment, "segment")
        if segment.dtype != torch.int32 or segment.dim() != 1:
            raise RuntimeError("segment must be a 1D int32 tensor")
        self.segment = segment
        self.S = segment.size(0) - 1
        self.T = int(T)
        self.seg_key2 = None
        if isinstance(seg_key, (tuple, list)):
            if len(seg_key) != 2 or any(k.dtype != torch.int64 for k in seg_key):
                raise RuntimeError("a pair key is two int64 tensors of weight addresses")
            seg_key, self.seg_key2 = seg_key
        self.seg_key = seg_key
        if seg_key is None:
            kind = _lib.SMLM_KEY_NONE
        elif self.seg_key2 is not None:
            kind = _lib.SMLM_KEY_PTR2
        elif seg_key.dtype == torch.int32:
            kind = _lib.SMLM_KEY_I32
        elif seg_key.dtype == torch.int64:
            kind = _lib.SMLM_KEY_PTR
        else:
            raise RuntimeError("seg_key must be int32 adapter ids or int64 addresses")
        for key in (seg_key, self.seg_key2):
            if key is not None:
                _check_input(key, "seg_key")
                if key.dim() != 1 or key.size(0) != self.S:
                    raise RuntimeError("seg_key must have one entry per segment")
        self.kind = kind
        dev = segment.device
        nbytes = _lib.size_query("smlm_plan_size", self.T, self.S)
        if buf is None:
            buf = torch.empty(max(nbytes, 64), dtype=torch.uint8, device=dev)
        elif buf.dtype != torch.uint8 or buf.numel() < nbytes or buf.device != dev:
            raise RuntimeError(f"plan buffer must be a uint8 tensor of >= {nbytes} bytes on {dev}")
        self.buf = buf
        self.built = False
        if not (defer and kind in (_lib.SMLM_KEY_I32, _lib.SMLM_KEY_PTR2)):
            self.ensure_built()

    def ensure_built(self) -> None:
        if self.built:
            return
        dev = self.segment.device
        with _on(dev):
            if self.kind == _lib.SMLM_KEY_PTR2:
                rc = _lib.load().smlm_plan_build2(self.buf.data_ptr(), self.buf.numel(), self.segment.data_ptr(),
                                                  self.seg_key.data_ptr(), self.seg_key2.data_ptr(), self.T,
                                                  self.S, _stream(dev))
            else:
                rc = _lib.load().smlm_plan_build(self.buf.data_ptr(), self.buf.numel(), self.segment.data_ptr(),
                                                 _ptr(self.seg_key), self.kind, self.T, self.S, _stream(dev))
        _lib.check(rc, "smlm_plan_build")
        self.built = True

    @staticmethod
    def nbytes(T: int, S: int) -> int:
        return _lib.size_query("smlm_plan_size", int(T), int(S))

    def header(self) -> Tuple[int, int, int, int]:
        """(n_tiles, n_groups, rows covered, key kind used) -- synchronises; for tests."""
        self.ensure_built()
        h = self.buf[:16].view(torch.int32).cpu()
        return int(h[0]), int(h[1]), int(h[2]), int(h[3])


def _check_table(t: torch.Tensor, plan: SegmentPlan, name: str) -> None:
    _check_input(t, name)
    if t.dtype != torch.int64 or t.dim() != 1:
        raise RuntimeError(f"{name} must be a 1D int64 tensor of device addresses")
    if plan.kind != _lib.SMLM_KEY_I32 and t.size(0) != plan.S:
        raise RuntimeError(f"{name} needs one entry per segment unless the plan is keyed by adapter id")


def _check_scale(seg_scale: Optional[torch.Tensor], plan: SegmentPlan) -> None:
    if seg_scale is not None and (seg_scale.dtype != torch.float32 or seg_scale.dim() != 1
                                  or seg_scale.size(0) != plan.S or not seg_scale.is_cuda):
        raise RuntimeError("seg_scale must be a device float32 tensor with one entry per segment")


def smlm_gemm_planned(y: torch.Tensor, x: torch.Tensor, w_ptrs: torch.Tensor, plan: SegmentPlan,
                      is_row_major: bool = False, seg_scale: Optional[torch.Tensor] = None,
                      beta: float = 0.0, workspace: Optional[Workspace] = None) -> None:
    """Grouped GEMM over a prebuilt plan: y[seg] = beta*y[seg] + scale*x[seg] @ W_seg.
    w_ptrs is indexed by adapter id when the plan was built from int32 adapter ids,
    by segment otherwise."""
    for t, n in ((y, "y"), (x, "x")):
        _check_input(t, n)
    _check_dim(2, y, "y")
    _check_dim(2, x, "x")
    _check_table(w_ptrs, plan, "w_ptrs")
    _check_scale(seg_scale, plan)
    plan.ensure_built()
    if y.dtype != x.dtype or y.size(0) != x.size(0) or x.size(0) != plan.T:
        raise RuntimeError("x [T,d_in] and y [T,d_out] must share dtype and T with the plan")
    code = _dtype_code(x)
    T, d_in, d_out = x.size(0), x.size(1), y.size(1)
    w_ld = d_out if is_row_major else d_in
    dev = x.device
    with _on(dev):
        need = _lib.size_query("smlm_gemm_planned_workspace_size", T, d_in, d_out)
        ws = _workspace(dev, need, workspace)
        rc = _lib.load().smlm_gemm_planned(y.data_ptr(), x.data_ptr(), w_ptrs.data_ptr(), w_ptrs.size(0),
                                           plan.buf.data_ptr(), ws.data_ptr(), ws.numel(), T, plan.S,
                                           d_in, d_out, w_ld, int(bool(is_row_major)), code,
                                           float(beta), _ptr(seg_scale), _stream(dev))
    _lib.check(rc, "smlm_gemm_planned")


class DropoutSpec:
    """Dropout of the training rows of x inside the operator (struct smlm_dropout):
    seg_p float32 [S] on the device, the dropout probability of each segment's
    adapter; rows = number of training rows (they come first in the batch);
    (seed, offset) name the mask stream -- the backward of a layer must be given
    the pair its forward used.  Replaces the nn.Dropout calls and the torch.cat of
    MixedLoraLinear.forward (src/loquetier_src/models/mixed_lora.py:185-192)."""

    def __init__(self, seg_p: torch.Tensor, rows: int, seed: int, offset: int,
                 mask_bits: Optional[torch.Tensor] = None):
        _check_input(seg_p, "seg_p")
        if seg_p.dtype != torch.float32 or seg_p.dim() != 1:
            raise RuntimeError("seg_p must be a 1D float32 tensor")
        if rows < 0:
            raise RuntimeError("rows must not be negative")
        if mask_bits is not None:
            _check_input(mask_bits, "mask_bits")
            if mask_bits.dtype != torch.uint8:
                raise RuntimeError("mask_bits must be a uint8 tensor")
        self.seg_p, self.rows = seg_p, int(rows)
        self.seed, self.offset = int(seed) & (2 ** 64 - 1), int(offset) & (2 ** 64 - 1)
        self.mask_bits = mask_bits

    @staticmethod
    def mask_nbytes(rows: int, h_in) -> int:
        """Size of mask_bits for `rows` training rows; h_in: one width or one per projection."""
        widths = [h_in] if isinstance(h_in, int) else list(h_in)
        return sum(int(rows) * (int(h) // 8) for h in widths)

    def with_offset(self, offset: int) -> "DropoutSpec":
        return DropoutSpec(self.seg_p, self.rows, self.seed, offset, self.mask_bits)

    def struct(self, plan: "SegmentPlan", widths):
        if self.seg_p.size(0) != plan.S or self.seg_p.device != plan.segment.device:
            raise RuntimeError("seg_p must have one entry per segment of the plan, on its device")
        if self.mask_bits is not None and self.mask_bits.numel() < self.mask_nbytes(self.rows, widths):
            raise RuntimeError(f"mask_bits needs {self.mask_nbytes(self.rows, widths)} bytes")
        return _lib.Dropout(self.seg_p.data_ptr(), self.rows, self.seed, self.offset, _ptr(self.mask_bits))


def _opts(plan: SegmentPlan, dropout: Optional["DropoutSpec"], widths, adapter_rank: Optional[torch.Tensor],
          n_weights: int, packed_ranks: bool = False, checked: bool = False):
    """struct smlm_lora_opts for a call (None when there is nothing to say).  The returned
    object keeps the dropout struct alive.  checked: the arguments were looked at by an earlier call."""
    if packed_ranks and adapter_rank is None:
        raise RuntimeError("packed_ranks needs adapter_rank: the kernels must know each adapter's stored rank")
    if dropout is None and adapter_rank is None:
        return None
    if adapter_rank is not None and not checked:
        _check_input(adapter_rank, "adapter_rank")
        if adapter_rank.dtype != torch.int32 or adapter_rank.dim() != 1 or adapter_rank.size(0) < n_weights:
            raise RuntimeError("adapter_rank must be a 1D int32 tensor with one entry per weight table entry")
    opts = _lib.LoraOpts()
    if dropout is not None:
        opts._drop = dropout.struct(plan, widths)
        opts.dropout = C.pointer(opts._drop)
    opts.adapter_rank = _ptr(adapter_rank)
    opts.packed_ranks = int(bool(packed_ranks))
    return opts


def smlm_lora_forward(y: torch.Tensor, x: torch.Tensor, a_ptrs: torch.Tensor, b_ptrs: torch.Tensor,
                      plan: SegmentPlan, rank: int, seg_scale: Optional[torch.Tensor] = None,
                      beta: float = 0.0, v_out: Optional[torch.Tensor] = None,
                      dropout: Optional[DropoutSpec] = None,
                      adapter_rank: Optional[torch.Tensor] = None,
                      workspace: Optional[Workspace] = None, packed_ranks: bool = False,
                      cache: Optional[dict] = None) -> None:
    """y = beta*y + seg_scale * round(x A^T) B^T in one stream-ordered call (two launches).
    a_ptrs / b_ptrs are indexed by adapter id when the plan was built from int32
    adapter ids, by segment otherwise.  cache: see smlm_lora_forward_multi."""
    smlm_lora_forward_multi([y], [x], [a_ptrs], [b_ptrs], plan, rank, seg_scale=seg_scale, beta=beta,
                            v_out=None if v_out is None else [v_out], dropout=dropout,
                            adapter_rank=adapter_rank, workspace=workspace, packed_ranks=packed_ranks,
                            cache=cache)


_FWD_MULTI_SIZES: Dict[Tuple, int] = {}


class _Checked:
    """What a checked call leaves behind for the next call from the same place: what its tensors looked
    like (a later call is compared with that, cheaply) and the argument blocks that do not change."""
    __slots__ = ("descs", "same", "code", "dev", "arrs", "h_in", "h_out", "a_arr", "b_arr", "n_weights", "need",
                 "opts")

    def matches(self, tensor_lists, objects) -> bool:
        """tensor_lists: the call's data tensors, list by list; objects: the tables and other tensors that are
        expected to be the very objects of the checked call."""
        for o, mine in zip(objects, self.same):
            if o is not mine:
                return False
        k = 0
        descs = self.descs
        for ts in tensor_lists:
            for t in ts:
                if k == len(descs):
                    return False
                d = descs[k]
                k += 1
                if t is None:
                    if d is not None:
                        return False
                elif d is None or t.shape != d[0] or t.dtype != d[1] or t.device != d[2] or not t.is_contiguous():
                    return False
        return k == len(descs)


def _descs(tensor_lists):
    return [None if t is None else (t.shape, t.dtype, t.device) for ts in tensor_lists for t in ts]


def _mask(ts) -> int:
    m = 0
    for i, t in enumerate(ts):
        if t is not None:
            m |= 1 << i
    return m


def _fill(arr, ts):
    for i, t in enumerate(ts):
        arr[i] = None if t is None else t.data_ptr()
    return arr


def _remember(cache: dict, key, hit: "_Checked") -> None:
    if len(cache) >= 32:
        cache.clear()
    cache[key] = hit


def _fwd_multi_workspace_size(T: int, widths_in: Tuple[int, ...], rank: int) -> int:
    key = (T, widths_in, rank)
    n = _FWD_MULTI_SIZES.get(key)
    if n is None:
        need = C.c_size_t(0)
        arr = (C.c_int * len(widths_in))(*widths_in)
        _lib.check(_lib.load().smlm_lora_fwd_multi_workspace_size(len(widths_in), T, arr, rank, C.byref(need)),
                   "smlm_lora_fwd_multi_workspace_size")
        n = _FWD_MULTI_SIZES[key] = need.value
    return n


def smlm_lora_forward_multi(ys, xs, a_ptrs, b_ptrs, plan: SegmentPlan, rank: int,
                            seg_scale: Optional[torch.Tensor] = None, beta: float = 0.0,
                            v_out=None, stages: int = 3, dropout: Optional[DropoutSpec] = None,
                            adapter_rank: Optional[torch.Tensor] = None,
                            workspace: Optional[Workspace] = None, packed_ranks: bool = False,
                            dims=None, cache: Optional[dict] = None) -> None:
    """The fused forward for several projections of one batch (q/k/v/o, gate/up/down)
    in two launches.  Lists of equal length; entries of xs may be the same tensor.
    stages: 1 = shrink only, 2 = expand only (after a shrink call with the same
    arguments, workspace and stream), 3 = both.  A shrink-only call may pass None for
    the ys, an expand-only call None for the xs, and an expand-only call skips the
    projections whose y is None (q, k and v of one shrink call can be expanded one at a
    time); `dims` = [(h_in, h_out), ...] then names the shapes the missing tensors have.  dropout: the training rows of x are
    dropped inside the shrink kernel; projection i uses the stream offset + i.
    adapter_rank (int32, indexed like the tables): true ranks of adapters stored
    zero-padded to `rank`; the padding is then not read.  packed_ranks: the adapters are stored
    AT their true rank rounded up to 8 (A_a [r_a, h_in], B_a [h_out, r_a]) instead of padded.
    cache: a dict the caller keeps (one per layer): after a call has been checked, later calls with
    tensors of the same shapes, dtype, device and contiguity and the same tables skip the checks and
    reuse the argument blocks that do not change.  Not for calls with dropout, nor for those of one
    projection that the native host path takes: it checks every call."""
    n = len(ys)
    if n == 1 and dropout is None and stages == 3 and dims is None and len(xs) == len(a_ptrs) == len(b_ptrs) == 1 and (
            v_out is None or len(v_out) == 1) and _host().forward(
                ys[0], xs[0], a_ptrs[0], b_ptrs[0], plan, rank, seg_scale, beta, None if v_out is None else v_out[0],
                adapter_rank, workspace, packed_ranks):
        return  # (one projection, plain: checked and launched by the native host path)
    key = None
    if cache is not None and dropout is None and len(xs) == n:  # (a dropout descriptor is checked call by call)
        scale_list = () if seg_scale is None else (seg_scale,)
        key = ("fwd", n, stages, plan.T, plan.S, plan.kind, rank, bool(packed_ranks), _mask(xs), _mask(ys),
               None if v_out is None else _mask(v_out), len(scale_list),
               dims if dims is None or isinstance(dims, tuple) else tuple(tuple(d_) for d_ in dims))
        hit = cache.get(key)
        if hit is not None and hit.matches((xs, ys, v_out or (), scale_list), (*a_ptrs, *b_ptrs, adapter_rank)):
            dev = hit.dev
            with _on(dev):
                ws = _workspace(dev, hit.need, workspace)
                opts = hit.opts
                if not plan.built and not (stages & _lib.SMLM_STAGE_SHRINK):
                    plan.ensure_built()
                if not plan.built:  # a deferred plan: this call builds it
                    opts = _opts(plan, None, None, adapter_rank, hit.n_weights, packed_ranks, checked=True) \
                        or _lib.LoraOpts()
                    opts.build_seg_indptr = plan.segment.data_ptr()
                    if plan.kind == _lib.SMLM_KEY_PTR2:
                        opts.build_seg_key_a = plan.seg_key.data_ptr()
                        opts.build_seg_key_b = plan.seg_key2.data_ptr()
                    else:
                        opts.build_seg_adapter = plan.seg_key.data_ptr()
                y_arr, x_arr, v_arr = hit.arrs
                rc = _lib.load().smlm_lora_fwd_multi_ex(
                    n, _fill(y_arr, ys), _fill(x_arr, xs), None if v_out is None else _fill(v_arr, v_out),
                    hit.a_arr, hit.b_arr, hit.n_weights, hit.h_in, hit.h_out, plan.buf.data_ptr(), ws.data_ptr(),
                    ws.numel(), plan.T, plan.S, rank, hit.code, float(beta), _ptr(seg_scale), int(stages),
                    None if opts is None else C.byref(opts), _stream(dev))
            _lib.check(rc, "smlm_lora_forward")
            plan.built = True
            return
    if not (1 <= n <= 8) or len(xs) != n or len(a_ptrs) != n or len(b_ptrs) != n or \
            (v_out is not None and len(v_out) != n):
        raise RuntimeError("between 1 and 8 projections, all lists of one length")
    _check_scale(seg_scale, plan)
    given = [t for t in list(xs) + list(ys) if t is not None]
    if not given:
        raise RuntimeError("nothing to work on: every x and y is None")
    first = given[0]
    for i in range(n):
        if (ys[i] is None and stages == 3) or (xs[i] is None and stages != 2):
            raise RuntimeError("only a shrink-only call may leave out y, only an expand-only call x")
        if (xs[i] is None or ys[i] is None) and dims is None:
            raise RuntimeError("dims=[(h_in, h_out), ...] must name the shapes of the tensors left out")
        for t, name in ((ys[i], "y"), (xs[i], "x")):
            if t is None:
                continue
            _check_input(t, name)
            _check_dim(2, t, name)
            if t.dtype != first.dtype or t.size(0) != plan.T or t.device != first.device:
                raise RuntimeError("x [T,h_in] and y [T,h_out] must share dtype, device and T with the plan")
            if dims is not None and t.size(1) != dims[i][0 if name == "x" else 1]:
                raise RuntimeError(f"{name} of projection {i} does not have the width dims names")
        _check_table(a_ptrs[i], plan, "a_ptrs")
        _check_table(b_ptrs[i], plan, "b_ptrs")
        if v_out is not None and v_out[i] is not None:
            vo = v_out[i]
            if vo.dtype != first.dtype or tuple(vo.shape) != (plan.T, rank) or not vo.is_contiguous():
                raise RuntimeError("v_out must be a contiguous [T, rank] tensor of x's dtype")
    code = _dtype_code(first)
    dev = first.device
    VP, CI = C.c_void_p * n, C.c_int * n
    widths_in = [dims[i][0] if xs[i] is None else xs[i].size(1) for i in range(n)]
    h_in = CI(*widths_in)
    h_out = CI(*[dims[i][1] if ys[i] is None else ys[i].size(1) for i in range(n)])
    vo_arr = None if v_out is None else VP(*[_ptr(t) for t in v_out])
    with _on(dev):
        need = _fwd_multi_workspace_size(plan.T, tuple(widths_in), rank)
        ws = _workspace(dev, need, workspace)
        n_weights = min(t.size(0) for t in list(a_ptrs) + list(b_ptrs))
        opts = _opts(plan, dropout, widths_in, adapter_rank, n_weights, packed_ranks)
        a_arr, b_arr = VP(*[t.data_ptr() for t in a_ptrs]), VP(*[t.data_ptr() for t in b_ptrs])
        if key is not None:  # (every check has passed: the next call like this one takes the short way)
            hit = _Checked()
            hit.descs = _descs((xs, ys, v_out or (), () if seg_scale is None else (seg_scale,)))
            hit.same = (*a_ptrs, *b_ptrs, adapter_rank)
            hit.code, hit.dev, hit.arrs, hit.h_in, hit.h_out = code, dev, (VP(), VP(), VP()), h_in, h_out
            hit.a_arr, hit.b_arr, hit.n_weights, hit.need = a_arr, b_arr, n_weights, need
            hit.opts = _opts(plan, None, None, adapter_rank, n_weights, packed_ranks, checked=True)
            _remember(cache, key, hit)
        if not plan.built:
            if stages & _lib.SMLM_STAGE_SHRINK:  # a deferred plan: this call builds it
                opts = opts or _lib.LoraOpts()
                opts.build_seg_indptr = plan.segment.data_ptr()
                if plan.kind == _lib.SMLM_KEY_PTR2:
                    opts.build_seg_key_a = plan.seg_key.data_ptr()
                    opts.build_seg_key_b = plan.seg_key2.data_ptr()
                else:
                    opts.build_seg_adapter = plan.seg_key.data_ptr()
            else:
                plan.ensure_built()
        rc = _lib.load().smlm_lora_fwd_multi_ex(
            n, VP(*[_ptr(t) for t in ys]), VP(*[_ptr(t) for t in xs]), vo_arr,
            a_arr, b_arr,
            n_weights, h_in, h_out,
            plan.buf.data_ptr(), ws.data_ptr(), ws.numel(), plan.T, plan.S, rank, code, float(beta),
            _ptr(seg_scale), int(stages), None if opts is None else C.byref(opts), _stream(dev))
    _lib.check(rc, "smlm_lora_forward")
    plan.built = True


def smlm_lora_backward(dx: torch.Tensor, da_ptrs: torch.Tensor, db_ptrs: torch.Tensor,
                       dy: torch.Tensor, x: torch.Tensor, v: Optional[torch.Tensor],
                       a_ptrs: torch.Tensor, b_ptrs: torch.Tensor, plan: SegmentPlan, rank: int,
                       part_scale: Optional[torch.Tensor] = None,
                       dropout: Optional[DropoutSpec] = None,
                       adapter_rank: Optional[torch.Tensor] = None,
                       workspace: Optional[Workspace] = None, packed_ranks: bool = False,
                       is_row_major: bool = False, cache: Optional[dict] = None,
                       zero_dx_tail: bool = False) -> None:
    """dX rows of the train partitions and per-adapter dA / dB (see include/smlm.h).
    `plan` = SegmentPlan(part_indptr, part_adapter int32, n_rows).  dropout: the
    forward's stream with seg_p per partition; x is the tensor before dropout.
    is_row_major: weights and gradients in the reference's other layout, A [h_in, r], B [r, h_out]."""
    smlm_lora_backward_multi([dx], [da_ptrs], [db_ptrs], [dy], [x], None if v is None else [v], [a_ptrs],
                             [b_ptrs], plan, rank, part_scale=part_scale, dropout=dropout,
                             adapter_rank=adapter_rank, workspace=workspace, packed_ranks=packed_ranks,
                             is_row_major=is_row_major, cache=cache, zero_dx_tail=zero_dx_tail)


_BWD_MULTI_SIZES: Dict[Tuple, int] = {}


def _bwd_opts(plan, adapter_rank, n_weights, packed_ranks, stages, is_row_major, checked, dropout=None, widths=None,
              dx_rows=0):
    """struct smlm_lora_opts of a backward call (None when there is nothing to say)."""
    opts = _opts(plan, dropout, widths, adapter_rank, n_weights, packed_ranks, checked=checked)
    if dx_rows:
        opts = opts or _lib.LoraOpts()
        opts.dx_rows = int(dx_rows)
    if stages:
        opts = opts or _lib.LoraOpts()
        opts.bwd_stages = int(stages)
    if is_row_major:
        opts = opts or _lib.LoraOpts()
        opts.w_row_major = 1
    return opts


def _bwd_multi_workspace_size(n_rows: int, P: int, NA: int, widths_in: Tuple[int, ...],
                              widths_out: Tuple[int, ...], rank: int) -> int:
    key = (n_rows, P, NA, widths_in, widths_out, rank)
    n = _BWD_MULTI_SIZES.get(key)
    if n is None:
        need = C.c_size_t(0)
        CI = C.c_int * len(widths_in)
        _lib.check(_lib.load().smlm_lora_bwd_multi_workspace_size(len(widths_in), n_rows, P, NA, CI(*widths_in),
                                                                  CI(*widths_out), rank, C.byref(need)),
                   "smlm_lora_bwd_multi_workspace_size")
        n = _BWD_MULTI_SIZES[key] = need.value
    return n


def smlm_lora_backward_multi(dxs, da_ptrs, db_ptrs, dys, xs, vs, a_ptrs, b_ptrs, plan: SegmentPlan, rank: int,
                             part_scale: Optional[torch.Tensor] = None,
                             dropout: Optional[DropoutSpec] = None,
                             adapter_rank: Optional[torch.Tensor] = None,
                             workspace: Optional[Workspace] = None, packed_ranks: bool = False,
                             stages: int = 0, is_row_major: bool = False,
                             cache: Optional[dict] = None, zero_dx_tail: bool = False) -> None:
    """The backward of several projections of one batch (q/k/v/o, gate/up/down) in one set of
    launches; lists of equal length, one entry per projection, each what smlm_lora_backward
    takes.  vs: None, or the saved intermediate of every projection.  The results equal
    per-projection calls bit for bit.  dropout: projection i uses the stream offset + i and
    the keep bits of the projections lie end to end (as smlm_lora_forward_multi leaves them).
    stages: 0 = everything; else SMLM_BWD_* bits (1 products v / dV, 2 dX, 4 weight gradients): the stages
    may be issued as separate calls with the same arguments, workspace and stream, in that order.
    is_row_major: the weights and their gradients are A [h_in, r], B [r, h_out] (the layout the reference's
    backward lines are written for, kernel_utils.py:139-145) instead of PEFT's A [r, h_in], B [h_out, r].
    cache: as in smlm_lora_forward_multi (the same dict may serve a layer's forward and backward).
    zero_dx_tail: the dx tensors cover more rows than the plan (the whole batch): the call also sets their rows from
    plan.T on to zero, inside one of its launches where it can (all dx must then have the same number of rows)."""
    n = len(dxs)
    key = None
    if cache is not None and dropout is None:  # (a dropout descriptor is checked call by call)
        scale_list = () if part_scale is None else (part_scale,)
        key = ("bwd", n, stages, plan.T, plan.S, plan.kind, rank, bool(packed_ranks), bool(is_row_major),
               vs is None, len(scale_list), bool(zero_dx_tail))
        hit = cache.get(key)
        if hit is not None and hit.matches((dxs, dys, xs, vs or (), da_ptrs, db_ptrs, scale_list),
                                           (*a_ptrs, *b_ptrs, adapter_rank)):
            dev = hit.dev
            with _on(dev):
                ws = _workspace(dev, hit.need, workspace)
                opts = hit.opts
                if not plan.built and stages and not (stages & _lib.SMLM_BWD_PRODUCTS):
                    plan.ensure_built()
                if not plan.built:  # a deferred plan: this call builds it
                    opts = _bwd_opts(plan, adapter_rank, hit.n_weights, packed_ranks, stages, is_row_major, True,
                                     dx_rows=dxs[0].size(0) if zero_dx_tail else 0) or _lib.LoraOpts()
                    opts.build_seg_indptr = plan.segment.data_ptr()
                    opts.build_seg_adapter = plan.seg_key.data_ptr()
                dx_arr, dy_arr, x_arr, v_arr, da_arr, db_arr = hit.arrs
                rc = _lib.load().smlm_lora_bwd_multi_ex(
                    n, _fill(dx_arr, dxs), _fill(da_arr, da_ptrs), _fill(db_arr, db_ptrs), _fill(dy_arr, dys),
                    _fill(x_arr, xs), None if vs is None else _fill(v_arr, vs), hit.a_arr, hit.b_arr,
                    plan.buf.data_ptr(), ws.data_ptr(), ws.numel(), plan.T, plan.S, hit.n_weights, hit.h_in,
                    hit.h_out, rank, hit.code, _ptr(part_scale), None if opts is None else C.byref(opts),
                    _stream(dev))
            _lib.check(rc, "smlm_lora_backward")
            plan.built = True
            return
    lists = (da_ptrs, db_ptrs, dys, xs, a_ptrs, b_ptrs) + (() if vs is None else (vs,))
    if not (1 <= n <= 8) or any(len(l) != n for l in lists):
        raise RuntimeError("between 1 and 8 projections, all lists of one length")
    if plan.kind != _lib.SMLM_KEY_I32:
        raise RuntimeError("the backward plan must be built from int32 adapter ids")
    n_rows = plan.T
    NA = a_ptrs[0].size(0)
    dtype = dys[0].dtype
    for i in range(n):
        for t, name in ((dxs[i], "dx"), (dys[i], "dy"), (xs[i], "x"), (da_ptrs[i], "da_ptrs"),
                        (db_ptrs[i], "db_ptrs"), (a_ptrs[i], "a_ptrs"), (b_ptrs[i], "b_ptrs")):
            _check_input(t, name)
        if dys[i].size(0) < n_rows or xs[i].size(0) < n_rows or dxs[i].size(0) < n_rows:
            raise RuntimeError("dy, x and dx need at least plan.T rows")
        v = None if vs is None else vs[i]
        if dxs[i].dtype != dtype or xs[i].dtype != dtype or dys[i].dtype != dtype or \
                (v is not None and v.dtype != dtype):
            raise RuntimeError("dx, dy, x, v must share one dtype")
        if any(t.size(0) != NA for t in (a_ptrs[i], b_ptrs[i], da_ptrs[i], db_ptrs[i])):
            raise RuntimeError("pointer tables must all have one entry per adapter")
        if vs is not None and (v is None or v.size(0) < n_rows or v.size(1) != rank or not v.is_contiguous()):
            raise RuntimeError("v must be a contiguous [>=n_rows, rank] tensor (of every projection or of none)")
        if dxs[i].size(1) != xs[i].size(1):
            raise RuntimeError("dx and x must have the same width")
        if any(t is not None and t.device != dys[0].device for t in (dxs[i], dys[i], xs[i], v)):
            raise RuntimeError("dx, dy, x, v must share one device")
    code = _dtype_code(dys[0])
    widths_in = tuple(t.size(1) for t in xs)
    widths_out = tuple(t.size(1) for t in dys)
    dev = dys[0].device
    VP, CI = C.c_void_p * n, C.c_int * n
    with _on(dev):
        need = _bwd_multi_workspace_size(n_rows, plan.S, NA, widths_in, widths_out, rank)
        ws = _workspace(dev, need, workspace)
        if dropout is not None and dropout.rows < n_rows:
            raise RuntimeError("the dropout descriptor must cover the backward's rows")
        dx_rows = 0
        if zero_dx_tail:
            dx_rows = dxs[0].size(0)
            if any(t.size(0) != dx_rows for t in dxs):
                raise RuntimeError("zero_dx_tail: every dx must have the same number of rows")
        opts = _bwd_opts(plan, adapter_rank, NA, packed_ranks, stages, is_row_major, False, dropout,
                         list(widths_in), dx_rows)
        arr = lambda ts: VP(*[t.data_ptr() for t in ts])
        a_arr, b_arr, h_in, h_out = arr(a_ptrs), arr(b_ptrs), CI(*widths_in), CI(*widths_out)
        if key is not None:  # (every check has passed: the next call like this one takes the short way)
            hit = _Checked()
            hit.descs = _descs((dxs, dys, xs, vs or (), da_ptrs, db_ptrs, () if part_scale is None else (part_scale,)))
            hit.same = (*a_ptrs, *b_ptrs, adapter_rank)
            hit.code, hit.dev, hit.arrs, hit.h_in, hit.h_out = code, dev, tuple(VP() for _ in range(6)), h_in, h_out
            hit.a_arr, hit.b_arr, hit.n_weights, hit.need = a_arr, b_arr, NA, need
            hit.opts = _bwd_opts(plan, adapter_rank, NA, packed_ranks, stages, is_row_major, True, dx_rows=dx_rows)
            _remember(cache, key, hit)
        if not plan.built:  # a deferred plan: this call builds it (inside its first launch where it can)
            if stages and not (stages & _lib.SMLM_BWD_PRODUCTS):
                plan.ensure_built()
            else:
                opts = opts or _lib.LoraOpts()
                opts.build_seg_indptr = plan.segment.data_ptr()
                opts.build_seg_adapter = plan.seg_key.data_ptr()
        rc = _lib.load().smlm_lora_bwd_multi_ex(
            n, arr(dxs), arr(da_ptrs), arr(db_ptrs), arr(dys), arr(xs), None if vs is None else arr(vs),
            a_arr, b_arr, plan.buf.data_ptr(), ws.data_ptr(), ws.numel(), n_rows, plan.S, NA,
            h_in, h_out, rank, code, _ptr(part_scale),
            None if opts is None else C.byref(opts), _stream(dev))
    _lib.check(rc, "smlm_lora_backward")
    plan.built = True


def rms_norm(output: torch.Tensor, rms_output: torch.Tensor, input: torch.Tensor, weight: torch.Tensor,
             epsilon: float) -> None:
    """output = input * rms * weight, rms_output = 1 / sqrt(mean(input^2) + epsilon) per row.

    Same arguments and checks as dispatch_rms_norm
    (kernel_src/csrc/loquetier_ops.cc:326-358): input/output [rows, cols] fp16
    or bf16, weight [cols] of the same dtype, rms_output float32 [rows, 1].
    """
    for t, n in ((output, "output"), (rms_output, "rms_output"), (input, "input"), (weight, "weight")):
        _check_input(t, n)
    _check_dim(2, input, "input")
    _check_dim(2, rms_output, "rms_output")
    _check_dim(1, weight, "weight")
    if output.shape != input.shape:
        raise RuntimeError("output and input must have the same shape")
    if rms_output.size(0) != input.size(0) or rms_output.size(1) != 1:
        raise RuntimeError("rms_output must be [rows, 1]")
    if rms_output.dtype != torch.float32:
        raise RuntimeError("rms_output must be float32")
    if weight.size(0) != input.size(1):
        raise RuntimeError("weight must have one entry per column of input")
    if input.dtype != weight.dtype or input.dtype != output.dtype:
        raise RuntimeError("input, weight and output must share one dtype")
    rows, cols = input.shape
    if input.dtype not in _DTYPE_CODE or cols % 8 != 0:
        raise RuntimeError(f"No suitable kernel. dtype={input.dtype} columns={cols}")
    dev = input.device
    with _on(dev):
        rc = _lib.load().smlm_rms_norm_fwd(output.data_ptr(), rms_output.data_ptr(), input.data_ptr(),
                                           weight.data_ptr(), rows, cols, float(epsilon),
                                           _DTYPE_CODE[input.dtype], _stream(dev))
    _lib.check(rc, "rms_norm")


def rms_norm_backward(dx: torch.Tensor, dw: torch.Tensor, grad_output: torch.Tensor, x: torch.Tensor,
                      w: torch.Tensor, rms: torch.Tensor) -> None:
    """dx [rows, cols] and dw [cols] of RMSNorm from the upstream gradient and the
    forward's saved tensors (the reference computes them with tensor expressions,
    src/loquetier_src/kernel_utils.py:169-176)."""
    for t, n in ((dx, "dx"), (dw, "dw"), (grad_output, "grad_output"), (x, "x"), (w, "w"), (rms, "rms")):
        _check_input(t, n)
    if dx.shape != x.shape or grad_output.shape != x.shape or dw.shape != w.shape:
        raise RuntimeError("dx / grad_output must match x and dw must match w")
    if rms.dtype != torch.float32 or rms.numel() != x.size(0):
        raise RuntimeError("rms must be float32 with one entry per row")
    if not (dx.dtype == dw.dtype == grad_output.dtype == x.dtype == w.dtype):
        raise RuntimeError("dx, dw, grad_output, x, w must share one dtype")
    rows, cols = x.shape
    code = _dtype_code(x)
    dev = x.device
    with _on(dev):
        need = _lib.size_query("smlm_rms_norm_bwd_workspace_size", rows, cols)
        ws = _workspace(dev, need)
        rc = _lib.load().smlm_rms_norm_bwd(dx.data_ptr(), dw.data_ptr(), grad_output.data_ptr(),
                                           x.data_ptr(), w.data_ptr(), rms.data_ptr(), ws.data_ptr(),
                                           ws.numel(), rows, cols, code, _stream(dev))
    _lib.check(rc, "rms_norm_backward")


def segments_build(req_adapter: torch.Tensor, req_len: torch.Tensor):
    """Run-length segments from per-request (adapter id, token count), on the device.

    The device version of the loop in ModelGeneration.generate
    (src/loquetier_src/model_generation.py:267-283).  Both inputs are int32 [R]
    device tensors.  Returns (seg_adapter [R], seg_len [R], seg_indptr [R+1],
    n_seg [2]) as int32 device tensors; n_seg holds (segment count, total rows)
    and is not read back here, so nothing waits for the device.  Entries past
    n_seg[0] are empty segments; pass the arrays on whole (S = R)."""
    for t, n in ((req_adapter, "req_adapter"), (req_len, "req_len")):
        _check_input(t, n)
        _check_dim(1, t, n)
        if t.dtype != torch.int32:
            raise RuntimeError(f"{n} must be int32")
    if req_adapter.numel() != req_len.numel():
        raise RuntimeError("req_adapter and req_len must have one entry per request")
    dev, R = req_adapter.device, req_adapter.numel()
    seg_adapter = torch.empty(R, dtype=torch.int32, device=dev)
    seg_len = torch.empty(R, dtype=torch.int32, device=dev)
    seg_indptr = torch.empty(R + 1, dtype=torch.int32, device=dev)
    n_seg = torch.empty(2, dtype=torch.int32, device=dev)
    with _on(dev):
        rc = _lib.load().smlm_segments_build(_ptr(req_adapter), _ptr(req_len), R, _ptr(seg_adapter),
                                             _ptr(seg_len), seg_indptr.data_ptr(), n_seg.data_ptr(),
                                             _stream(dev))
    _lib.check(rc, "segments_build")
    return seg_adapter, seg_len, seg_indptr, n_seg


def segment_scales(seg_adapter: torch.Tensor, table: Optional[torch.Tensor] = None,
                   segment: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
                   part_seg: Optional[torch.Tensor] = None):
    """(seg_scale, part_seg, part_scale) of a step, in one launch: table[seg_adapter] float32 [S] (None without a
    table), the segment (int64) each row of `starts` lies in, and that segment's scale.  part_seg: known already, instead
    of segment and starts; without either there are no partitions and both come back as None."""
    dev, S = seg_adapter.device, seg_adapter.numel()
    for t, n, dt in ((seg_adapter, "seg_adapter", torch.int32), (table, "table", torch.float32),
                     (segment, "segment", torch.int32), (starts, "starts", torch.int32), (part_seg, "part_seg", torch.int64)):
        if t is not None:
            _check_input(t, n)
            _check_dim(1, t, n)
            if t.dtype != dt or t.device != dev:
                raise RuntimeError(f"{n} must be {dt} on {dev}")
    if starts is not None and (segment is None or segment.numel() != S + 1):
        raise RuntimeError("segment must have one entry more than seg_adapter")
    seg_out = None if table is None else torch.empty(S, dtype=torch.float32, device=dev)
    P = starts.numel() if starts is not None else (0 if part_seg is None else part_seg.numel())
    if starts is not None:
        part_seg = torch.empty(P, dtype=torch.int64, device=dev)
    part_out = torch.empty(P, dtype=torch.float32, device=dev) if table is not None and part_seg is not None else None
    with _on(dev):
        rc = _lib.load().smlm_segment_scales(_ptr(seg_adapter), S, _ptr(table), 0 if table is None else table.numel(),
                                             _ptr(seg_out), _ptr(segment), _ptr(starts), P, _ptr(part_seg), _ptr(part_out),
                                             _stream(dev))
    _lib.check(rc, "segment_scales")
    return seg_out, part_seg, part_out


# ---- between the projections: rotation of queries and keys, the cache's pages, attention over them --------------------

def _heads_fit(t: torch.Tensor) -> bool:
    """Whether the kernels read a tensor [rows, heads, head_dim] where it lies (its address has to be 16-byte aligned too)."""
    return (t.size(2) == 1 or t.stride(2) == 1) and not any(s % 8 for n, s in zip(t.shape[:2], t.stride()[:2]) if n > 1)


def _check_heads(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None, written: bool = False) -> None:
    """[rows, heads, head_dim] of any strides the kernels read: views of one projection's output need no copy."""
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    _check_dim(3, t, name)
    if t.numel() and not _heads_fit(t):
        raise RuntimeError(f"{name} must have its head's dimensions next to each other and strides that are multiples of 8")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise RuntimeError(f"{name} must share q's dtype and device")
    if written and any(s == 0 for n, s in zip(t.shape, t.stride()) if n > 1):
        raise RuntimeError(f"{name} is written and must not be expanded")


def _heads(t: Optional[torch.Tensor]) -> _lib.Heads:
    if t is None:
        return _lib.Heads()
    # (the stride of a dimension of one names nothing)
    return _lib.Heads(t.data_ptr(), t.stride(0) if t.size(0) > 1 else 0, t.stride(1) if t.size(1) > 1 else 0)


def _check_ints(dev: torch.device, dtype: torch.dtype, dim: int, **tensors) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        _check_input(t, name)
        _check_dim(dim, t, name)
        if t.dtype != dtype or t.device != dev:
            raise RuntimeError(f"{name} must be {dtype} on {dev}")


def _check_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, like: torch.Tensor, kv_heads: int) -> Tuple[int, int, int]:
    """Strides (page, head, place) of two caches [n_pages, kv_heads, page_size, head_dim]."""
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if not t.is_cuda:
            raise RuntimeError(f"{n} must be a CUDA tensor")
        _check_dim(4, t, n)
        if t.dtype != like.dtype or t.device != like.device:
            raise RuntimeError(f"{n} must share q's dtype and device")
        if t.size(3) != like.size(2) or t.size(1) != kv_heads or t.size(2) < 1:
            raise RuntimeError(f"{n} must be [n_pages, {kv_heads}, page_size, {like.size(2)}]")
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise RuntimeError("k_cache and v_cache must have the same shape and strides")
    strides = tuple(s if n > 1 else 0 for n, s in zip(k_cache.shape, k_cache.stride()))
    if strides[3] != 1 or any(s % 8 for s in strides[:3]):
        raise RuntimeError("the caches must have a head's dimensions next to each other and strides that are multiples of 8")
    return strides[:3]


def rope_table(n_positions: int, rot_dim: int, base: float = 10000.0, device=None,
               inv_freq: Optional[torch.Tensor] = None) -> torch.Tensor:
    """float32 [n_positions, rot_dim] for qk_norm_rope: by position rot_dim / 2 cosines, then the sines.  The angles,
    position times base ** (-2 j / rot_dim) (or times inv_freq[j], for scaled variants), are taken in 64 bits: far positions lose
    whole turns in 32."""
    if rot_dim <= 0 or rot_dim % 16 or n_positions < 0:
        raise RuntimeError("rot_dim must be a positive multiple of 16")
    if inv_freq is None:
        inv_freq = float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    if inv_freq.dim() != 1 or inv_freq.numel() != rot_dim // 2:
        raise RuntimeError("inv_freq must have rot_dim / 2 entries")
    angle = torch.arange(n_positions, dtype=torch.float64)[:, None] * inv_freq.detach().double().cpu()
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def _rope_args(q, k, table, positions, q_weight, k_weight, eps) -> _lib.QkRope:
    _check_heads(q, "q")
    _check_heads(k, "k", q)
    T, Hq, D = q.shape
    if k.size(0) != T or k.size(2) != D:
        raise RuntimeError("q and k must have the same rows and head size")
    if Hq < 1 or k.size(1) < 1:
        raise RuntimeError("q and k must have heads")
    if q.dtype not in _DTYPE_CODE or D % 16 or not 0 < D <= 512:
        raise RuntimeError(f"No suitable kernel. dtype={q.dtype} head_dim={D}")
    dev = q.device
    _check_ints(dev, torch.float32, 2, table=table)
    rot = table.size(1)
    if rot % 16 or not 0 < rot <= D:
        raise RuntimeError(f"table must be [positions, rot_dim], rot_dim a multiple of 16 of at most {D}")
    _check_ints(dev, torch.int32, 1, positions=positions)
    if positions.size(0) != T:
        raise RuntimeError("positions must have one entry per row")
    _check_ints(dev, q.dtype, 1, q_weight=q_weight, k_weight=k_weight)
    for w in (q_weight, k_weight):
        if w is not None and w.size(0) != D:
            raise RuntimeError(f"a weight must have {D} entries")
    a = _lib.QkRope()
    a.q, a.k = _heads(q), _heads(k)
    a.q_weight, a.k_weight, a.table, a.positions = _ptr(q_weight), _ptr(k_weight), table.data_ptr(), positions.data_ptr()
    a.rows, a.q_heads, a.kv_heads, a.head_dim, a.rot_dim, a.table_rows = T, Hq, k.size(1), D, rot, table.size(0)
    a.dtype, a.eps = _DTYPE_CODE[q.dtype], float(eps)
    return a


def qk_norm_rope(q_out: torch.Tensor, k_out: Optional[torch.Tensor], q: torch.Tensor, k: torch.Tensor, table: torch.Tensor,
                 positions: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, v: Optional[torch.Tensor] = None,
                 k_cache: Optional[torch.Tensor] = None, v_cache: Optional[torch.Tensor] = None,
                 slots: Optional[torch.Tensor] = None) -> None:
    """Queries [rows, q_heads, head_dim] and keys [rows, kv_heads, head_dim], each head scaled to a root mean square of one and
    by its weight [head_dim] (where there is one), then rotated by the row's position (see include/smlm.h).  table: rope_table's;
    positions: int32 [rows], below 0 for padding.  q_out may be q, k_out may be k.

    With the caches (k_cache, v_cache [n_pages, kv_heads, page_size, head_dim], any strides) and slots (int64 [rows],
    page * page_size + place, -1: not cached) the keys and v also go there; k_out may then be None."""
    if _host().rope(q_out, k_out, q, k, table, positions, q_weight, k_weight, eps, v, k_cache, v_cache, slots):
        return
    a = _rope_args(q, k, table, positions, q_weight, k_weight, eps)
    _check_heads(q_out, "q_out", q, True)
    if q_out.shape != q.shape:
        raise RuntimeError("q_out and q must have the same shape")
    if k_out is not None:
        _check_heads(k_out, "k_out", q, True)
        if k_out.shape != k.shape:
            raise RuntimeError("k_out and k must have the same shape")
    a.q_out, a.k_out = _heads(q_out), _heads(k_out)
    cache = (v, k_cache, v_cache, slots)
    if any(t is not None for t in cache):
        if any(t is None for t in cache):
            raise RuntimeError("v, k_cache, v_cache and slots come together")
        _check_heads(v, "v", q)
        if v.shape != k.shape:
            raise RuntimeError("v and k must have the same shape")
        a.page_stride, a.head_stride, a.slot_stride = _check_caches(k_cache, v_cache, q, k.size(1))
        if any(s == 0 for n, s in zip(k_cache.shape, k_cache.stride()) if n > 1):
            raise RuntimeError("the caches are written and must not be expanded")
        _check_ints(q.device, torch.int64, 1, slots=slots)
        if slots.size(0) != q.size(0):
            raise RuntimeError("slots must have one entry per row")
        a.v, a.slots = _heads(v), slots.data_ptr()
        a.n_pages, a.page_size = k_cache.size(0), k_cache.size(2)
        if a.n_pages > 0:
            a.k_cache, a.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    if k_out is None and k_cache is None:
        raise RuntimeError("k_out may be left out only where keys go to a cache")
    if k_out is None and a.n_pages == 0:
        raise RuntimeError("the cache has no pages")
    dev = q.device
    with _on(dev):
        rc = _lib.load().smlm_qk_norm_rope_fwd(C.byref(a), _stream(dev))
    _lib.check(rc, "qk_norm_rope")


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, dq_weight: Optional[torch.Tensor],
                          dk_weight: Optional[torch.Tensor], gq: torch.Tensor, gk: torch.Tensor, q: torch.Tensor,
                          k: torch.Tensor, table: torch.Tensor, positions: torch.Tensor,
                          q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                          eps: float = 1e-6, workspace: Optional[Workspace] = None) -> None:
    """Gradients of qk_norm_rope's inputs from those of its outputs, the weights' summed over rows and heads in a fixed
    order.  q, k, table, positions, weights: as in the forward."""
    a = _rope_args(q, k, table, positions, q_weight, k_weight, eps)
    for t, n, like in ((dq, "dq", q), (gq, "gq", q), (dk, "dk", k), (gk, "gk", k)):
        _check_heads(t, n, q, n in ("dq", "dk"))
        if t.shape != like.shape:
            raise RuntimeError(f"{n} must have its tensor's shape")
    for d, w, n in ((dq_weight, q_weight, "dq_weight"), (dk_weight, k_weight, "dk_weight")):
        if (d is None) != (w is None):
            raise RuntimeError(f"{n} and its weight come together")
        if d is not None:
            _check_ints(q.device, q.dtype, 1, **{n: d})
            if d.shape != w.shape:
                raise RuntimeError(f"{n} must match its weight")
    dev = q.device
    if q.size(0) == 0:
        for d in (dq_weight, dk_weight):
            if d is not None:
                d.zero_()
        return
    with _on(dev):
        ws = None
        if q_weight is not None or k_weight is not None:
            ws = _workspace(dev, _lib.size_query("smlm_qk_norm_rope_bwd_workspace_size", a.rows, a.q_heads, a.kv_heads,
                                                 a.head_dim), workspace)
        rc = _lib.load().smlm_qk_norm_rope_bwd(C.byref(a), C.byref(_heads(gq)), C.byref(_heads(gk)), C.byref(_heads(dq)),
                                               C.byref(_heads(dk)), _ptr(dq_weight), _ptr(dk_weight), _ptr(ws),
                                               0 if ws is None else ws.numel(), _stream(dev))
    _lib.check(rc, "qk_norm_rope_backward")


def _kv_state(table, length, refs, status, **lists) -> Tuple[torch.device, int, int, int]:
    _check_input(table, "table")
    dev = table.device
    _check_ints(dev, torch.int32, 2, table=table)
    _check_ints(dev, torch.int32, 1, length=length, refs=refs, status=status, **lists)
    if length is not None and length.size(0) != table.size(0):
        raise RuntimeError("length must have one entry per row of table")
    if status is not None and status.numel() != 1:
        raise RuntimeError("status must have one entry")
    return dev, table.size(0), table.size(1), refs.size(0)


def _kv_pool(pool: torch.Tensor, dev: torch.device, N: int) -> Tuple[int, int, int]:
    """(blocks, page_size, bytes of a place) of a pool [n_pages, ..., page_size, head_dim]."""
    _check_input(pool, "pool")
    if pool.dim() < 3 or pool.device != dev or pool.size(0) != N:
        raise RuntimeError("pool must be [n_pages, ..., page_size, head_dim], one page per entry of refs, on the tables' device")
    place = pool.size(-1) * pool.element_size()
    blocks = 1
    for n in pool.shape[1:-2]:
        blocks *= n
    if place == 0 or place % 16 or blocks == 0 or pool.size(-2) == 0:
        raise RuntimeError(f"No suitable kernel. {place} bytes a place")
    return blocks, pool.size(-2), place


def kv_extend(table: torch.Tensor, length: torch.Tensor, refs: torch.Tensor, requests: torch.Tensor, counts: torch.Tensor,
              n_rows: int, page_size: int, status: Optional[torch.Tensor] = None, workspace: Optional[Workspace] = None,
              max_tokens: Optional[int] = None):
    """Room for counts[s] more tokens of requests[s], pages taken lowest number first, on the device (see include/smlm.h
    for the state's tensors and `status`, which a call that cannot be done marks, changing nothing else).

    Returns (q_indptr int32 [S + 1], kv_len int32 [S], positions int32 [n_rows], slots int64 [n_rows]): what qk_norm_rope and
    AttentionPlan read.  n_rows: the counts' sum, or more (rows past it get position and slot -1).  max_tokens: what a request
    may have, where that is less than its row of the table has places for."""
    done = _host().kv_extend(table, length, refs, requests, counts, n_rows, page_size, status, workspace, max_tokens)
    if done is not None:
        return done
    dev, R, M, N = _kv_state(table, length, refs, status, requests=requests, counts=counts)
    if requests.numel() != counts.numel():
        raise RuntimeError("requests and counts must have one entry per sequence")
    if n_rows < 0 or page_size < 1:
        raise RuntimeError("n_rows and page_size must not be negative")
    if max_tokens is not None and max_tokens < 0:
        raise RuntimeError("max_tokens must not be negative")
    most = 0x7fffffff if max_tokens is None else min(int(max_tokens), 0x7fffffff)
    S = requests.numel()
    q_indptr = torch.empty(S + 1, dtype=torch.int32, device=dev)
    kv_len = torch.empty(S, dtype=torch.int32, device=dev)
    positions = torch.empty(n_rows, dtype=torch.int32, device=dev)
    slots = torch.empty(n_rows, dtype=torch.int64, device=dev)
    with _on(dev):
        ws = _workspace(dev, _lib.size_query("smlm_kv_workspace_size", R, N, S), workspace)
        rc = _lib.load().smlm_kv_extend_upto(_ptr(table), _ptr(length), _ptr(refs), _ptr(requests), _ptr(counts),
                                             q_indptr.data_ptr(), _ptr(kv_len), _ptr(positions), _ptr(slots), ws.data_ptr(),
                                             ws.numel(), R, M, N, S, n_rows, page_size, most, _ptr(status), _stream(dev))
    _lib.check(rc, "kv_extend")
    return q_indptr, kv_len, positions, slots


def kv_free(table: torch.Tensor, length: torch.Tensor, refs: torch.Tensor, requests: torch.Tensor, page_size: int,
            status: Optional[torch.Tensor] = None) -> None:
    """Gives the requests' pages back (those that a fork shares stay with the others).  Each request by itself: one that is
    unknown marks `status`, and the others are freed all the same."""
    if _host().kv_free(table, length, refs, requests, page_size, status):
        return
    dev, R, M, N = _kv_state(table, length, refs, status, requests=requests)
    if page_size < 1:
        raise RuntimeError("page_size must be positive")
    with _on(dev):
        rc = _lib.load().smlm_kv_free(_ptr(table), _ptr(length), _ptr(refs), _ptr(requests), R, M, N, requests.numel(), page_size,
                                      _ptr(status), _stream(dev))
    _lib.check(rc, "kv_free")


def kv_fork(pool: torch.Tensor, table: torch.Tensor, length: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor,
            children: torch.Tensor, status: Optional[torch.Tensor] = None, workspace: Optional[Workspace] = None) -> None:
    """children[i], empty so far, becomes a second parents[i]: full pages shared, the filled places of a part-filled last
    page copied.  pool: [n_pages, ..., page_size, head_dim], contiguous (PagedKvCache.pool)."""
    if _host().kv_fork(pool, table, length, refs, parents, children, status, workspace):
        return
    dev, R, M, N = _kv_state(table, length, refs, status, parents=parents, children=children)
    blocks, P, place = _kv_pool(pool, dev, N)
    if parents.numel() != children.numel():
        raise RuntimeError("parents and children must have one entry per fork")
    K = children.numel()
    with _on(dev):
        ws = _workspace(dev, _lib.size_query("smlm_kv_workspace_size", R, N, K), workspace)
        rc = _lib.load().smlm_kv_fork(_ptr(pool), _ptr(table), _ptr(length), _ptr(refs), _ptr(parents), _ptr(children),
                                      ws.data_ptr(), ws.numel(), R, M, N, K, blocks, P, place, _ptr(status), _stream(dev))
    _lib.check(rc, "kv_fork")


def kv_compact(pool: torch.Tensor, table: torch.Tensor, refs: torch.Tensor, workspace: Optional[Workspace] = None) -> None:
    """Packs the pages in use to the pool's front; table and refs follow (slots that kv_extend gave out before do not)."""
    dev, R, M, N = _kv_state(table, None, refs, None)
    blocks, P, place = _kv_pool(pool, dev, N)
    with _on(dev):
        ws = _workspace(dev, _lib.size_query("smlm_kv_workspace_size", R, N, 0), workspace)
        rc = _lib.load().smlm_kv_compact(_ptr(pool), _ptr(table), _ptr(refs), ws.data_ptr(), ws.numel(), R, M, N, blocks, P, place,
                                         _stream(dev))
    _lib.check(rc, "kv_compact")


def kv_copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """pool[dst[i]] = pool[src[i]] for int32 lists of pages; no page may be written twice, or read and written."""
    _check_input(pool, "pool")
    dev = pool.device
    _check_ints(dev, torch.int32, 1, src=src, dst=dst)
    if src.numel() != dst.numel():
        raise RuntimeError("src and dst must have one entry per copy")
    N = pool.size(0) if pool.dim() else 0
    blocks, P, place = _kv_pool(pool, dev, N)
    with _on(dev):
        rc = _lib.load().smlm_kv_copy_pages(_ptr(pool), _ptr(src), _ptr(dst), src.numel(), N, blocks, P, place, _stream(dev))
    _lib.check(rc, "kv_copy_pages")


_ATTENTION_DIMS = (64, 128)  # head sizes of paged_attention


class AttentionPlan:
    """How the card shares out the attention of one batch (see include/smlm.h): built once a step, for all its layers.

    q_indptr int32 [S + 1]: rows of the sequences in the batch's n_rows, never decreasing (or the plan holds nothing); kv_len
    int32 [S]: tokens of each in the cache, the new ones too; page_table int32 [R, M] (its contents are read by the attention
    calls); requests int32 [S]: the sequences' rows of page_table (None: 0, 1, ...).  The tensors are read when the plan's launches run, and kept."""

    def __init__(self, q_indptr: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor, n_rows: int, q_heads: int,
                 kv_heads: int, page_size: int, requests: Optional[torch.Tensor] = None):
        buf = _host().attention_plan(q_indptr, kv_len, page_table, n_rows, q_heads, kv_heads, page_size, requests)
        if buf is not None:
            self.buf, self.S, self.T = buf, q_indptr.size(0) - 1, n_rows
            self.q_indptr, self.kv_len, self.page_table, self.requests = q_indptr, kv_len, page_table, requests
            self.q_heads, self.kv_heads, self.page_size = q_heads, kv_heads, page_size
            return
        _check_input(q_indptr, "q_indptr")
        dev = q_indptr.device
        _check_ints(dev, torch.int32, 1, q_indptr=q_indptr, kv_len=kv_len, requests=requests)
        _check_ints(dev, torch.int32, 2, page_table=page_table)
        self.S = q_indptr.size(0) - 1
        if self.S < 0 or kv_len.size(0) != self.S or (requests is not None and requests.size(0) != self.S):
            raise RuntimeError("q_indptr needs one entry more than there are sequences, kv_len and requests one for each")
        if requests is None and page_table.size(0) < self.S:
            raise RuntimeError("page_table needs a row for each sequence")
        if q_heads < 1 or kv_heads < 1 or q_heads % kv_heads:
            raise RuntimeError("q_heads must be a multiple of kv_heads")
        if n_rows < 0 or page_size < 1:
            raise RuntimeError("n_rows and page_size must not be negative")
        self.q_indptr, self.kv_len, self.page_table, self.requests = q_indptr, kv_len, page_table, requests
        self.T, self.q_heads, self.kv_heads, self.page_size = int(n_rows), int(q_heads), int(kv_heads), int(page_size)
        self.buf = torch.empty(_lib.size_query("smlm_attn_plan_size", self.T, self.S, self.q_heads, self.kv_heads),
                               dtype=torch.uint8, device=dev)
        R, M = page_table.shape
        with _on(dev):
            rc = _lib.load().smlm_attn_plan_build(self.buf.data_ptr(), self.buf.numel(), q_indptr.data_ptr(), _ptr(kv_len),
                                                  _ptr(requests), self.T, self.S, R, M, self.page_size, self.q_heads,
                                                  self.kv_heads, _stream(dev))
        _lib.check(rc, "AttentionPlan")


def paged_attention(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, plan: AttentionPlan,
                    scale: Optional[float] = None, workspace: Optional[Workspace] = None) -> None:
    """Causal attention of the batch's rows q [rows, q_heads, head_dim] over the pages of k_cache and v_cache [n_pages, kv_heads,
    page_size, head_dim] (any strides), prompts' chunks and single tokens in one call.  scale: head_dim ** -0.5 by default.
    Rows that see no token become zero; rows of no sequence are left as they were.  out may be q."""
    if _host().paged_attention(out, q, k_cache, v_cache, plan, scale, workspace):
        return
    _check_heads(q, "q")
    _check_heads(out, "out", q, True)
    if out.shape != q.shape:
        raise RuntimeError("out and q must have the same shape")
    T, Hq, D = q.shape
    if T != plan.T or Hq != plan.q_heads:
        raise RuntimeError(f"the plan is for {plan.T} rows of {plan.q_heads} heads")
    if plan.buf.device != q.device:
        raise RuntimeError(f"the plan lives on {plan.buf.device}, q on {q.device}")
    if q.dtype not in _DTYPE_CODE or D not in _ATTENTION_DIMS:
        raise RuntimeError(f"No suitable kernel. dtype={q.dtype} head_dim={D}")
    page, head, place = _check_caches(k_cache, v_cache, q, plan.kv_heads)
    if k_cache.size(2) != plan.page_size:
        raise RuntimeError(f"the plan is for pages of {plan.page_size} tokens")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1.0e38:
        raise RuntimeError("scale must be positive")
    dev = q.device
    R, M = plan.page_table.shape
    with _on(dev):
        ws = None
        need = _lib.size_query("smlm_paged_attn_workspace_size", T, plan.S, M, plan.page_size, Hq, plan.kv_heads, D)
        if need:
            ws = _workspace(dev, need, workspace)
        rc = _lib.load().smlm_paged_attn(C.byref(_heads(out)), C.byref(_heads(q)), _ptr(k_cache), _ptr(v_cache), page, head, place,
                                         _ptr(plan.page_table), plan.buf.data_ptr(), plan.buf.numel(), _ptr(ws),
                                         0 if ws is None else ws.numel(), T, plan.S, R, M, k_cache.size(0), plan.page_size, Hq,
                                         plan.kv_heads, D, _DTYPE_CODE[q.dtype], scale, _stream(dev))
    _lib.check(rc, "paged_attention")
