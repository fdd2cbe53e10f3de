"""What the operators around a fine-tuning step refuse, through the C ABI, before any launch (no GPU needed: made-up addresses are never
read), and from Python for tensors that are not on a GPU."""
import ctypes as C

import pytest
import torch

from loquetier_amd import _lib as lib, optim
from loquetier_amd.kernel_utils import add_rms_norm, linear_cross_entropy
from loquetier_amd.ops import _kernels as K

ARG, DTYPE, ALIGN, WORKSPACE, LIMIT = -1, -2, -3, -4, -6
A = 1 << 20  # an aligned address
LOTS = 1 << 60


@pytest.fixture(scope="module")
def L():
    return lib.load()


NORM = dict(out=A, rms=A, h=A, x=A, residual=A, w=A, out8=A, scale=A, group=0, rows=4, cols=256, eps=1e-6, dtype=1, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), ARG), (dict(cols=0), ARG), (dict(cols=252), ALIGN), (dict(dtype=2), DTYPE), (dict(group=64), ARG), (dict(cols=(1 << 24) + 8), LIMIT),
    (dict(group=128, cols=200), ALIGN), (dict(out8=None), ARG), (dict(scale=None), ARG), (dict(x=None), ARG), (dict(w=None), ARG),
    (dict(residual=None), ARG), (dict(out=None, h=None, out8=None, scale=None), ARG), (dict(out=A + 8), ALIGN), (dict(h=A + 2), ALIGN),
    (dict(x=A + 4), ALIGN), (dict(residual=A + 8), ALIGN), (dict(w=A + 2), ALIGN), (dict(out8=A + 1), ALIGN), (dict(rows=(1 << 30) + 1), LIMIT),
    (dict(rows=0), 0), (dict(rows=0, x=None), 0)])
def test_add_rms_norm(L, change, code):
    assert L.smlm_add_rms_norm_fwd(*{**NORM, **change}.values()) == code


BACK = dict(dh=A, dw=A, g=A, gh=A, h=A, w=A, rms=A, workspace=A, workspace_bytes=LOTS, rows=4, cols=256, dtype=1, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), ARG), (dict(rows=0), ARG), (dict(cols=12), ALIGN), (dict(dtype=7), DTYPE), (dict(dh=None), ARG), (dict(dw=None), ARG),
    (dict(g=None), ARG), (dict(h=None), ARG), (dict(w=None), ARG), (dict(rms=None), ARG), (dict(workspace=None), ARG),
    (dict(workspace_bytes=256), WORKSPACE), (dict(gh=A + 8), ALIGN), (dict(dh=A + 8), ALIGN), (dict(workspace=A + 8), ALIGN)])
def test_add_rms_norm_backward(L, change, code):
    assert L.smlm_add_rms_norm_bwd(*{**BACK, **change}.values()) == code


LOSS = dict(loss=A, lse=A, means=A, weight=A, kept=A, kept_bytes=LOTS, x=A, w=A, labels=A, partition=A, P=2, workspace=A,
            workspace_bytes=LOTS, T=4, H=64, V=100, dtype=1, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), ARG), (dict(H=0), ARG), (dict(V=0), ARG), (dict(H=60), ALIGN), (dict(dtype=2), DTYPE), (dict(H=(1 << 22) + 8), LIMIT),
    (dict(T=(1 << 28) + 1), LIMIT), (dict(V=(1 << 28) + 1), LIMIT), (dict(T=1 << 28, V=1 << 28), LIMIT), (dict(P=-1), ARG),
    (dict(means=None), ARG), (dict(weight=None), ARG), (dict(loss=None), ARG), (dict(lse=None), ARG), (dict(x=None), ARG),
    (dict(w=None), ARG), (dict(labels=None), ARG), (dict(workspace=None), ARG), (dict(x=A + 8), ALIGN), (dict(w=A + 2), ALIGN),
    (dict(kept=A + 8), ALIGN), (dict(workspace=A + 8), ALIGN), (dict(kept_bytes=100), WORKSPACE), (dict(workspace_bytes=100), WORKSPACE),
    (dict(T=0, partition=None), 0)])
def test_loss(L, change, code):
    assert L.smlm_vocab_loss_fwd(*{**LOSS, **change}.values()) == code


LOSS_KEPT = dict(dx=A, grad=A, kept=A, kept_bytes=LOTS, w=A, partition=A, weight=A, P=2, T=4, H=64, V=100, dtype=1, stream=None)
LOSS_BACK = dict(dx=A, dw=A, grad=A, loss=A, lse=A, x=A, w=A, labels=A, partition=A, weight=A, P=2, workspace=A, workspace_bytes=LOTS,
                 T=4, H=64, V=100, dtype=1, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), ARG), (dict(H=4), ALIGN), (dict(dtype=3), DTYPE), (dict(P=-1), ARG), (dict(weight=None), ARG), (dict(dx=None), ARG),
    (dict(grad=None), ARG), (dict(kept=None), ARG), (dict(w=None), ARG), (dict(dx=A + 8), ALIGN), (dict(kept=A + 8), ALIGN),
    (dict(w=A + 8), ALIGN), (dict(kept_bytes=100), WORKSPACE), (dict(T=0, dx=None), 0)])
def test_loss_backward_of_what_was_kept(L, change, code):
    assert L.smlm_vocab_loss_bwd_kept(*{**LOSS_KEPT, **change}.values()) == code


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), ARG), (dict(H=4), ALIGN), (dict(dtype=3), DTYPE), (dict(P=-1), ARG), (dict(weight=None), ARG), (dict(dx=None, dw=None), ARG),
    (dict(T=0), ARG), (dict(T=0, dw=None), 0), (dict(grad=None), ARG), (dict(loss=None), ARG), (dict(lse=None), ARG), (dict(x=None), ARG),
    (dict(w=None), ARG), (dict(labels=None), ARG), (dict(workspace=None), ARG), (dict(dx=A + 8), ALIGN), (dict(dw=A + 8), ALIGN),
    (dict(x=A + 8), ALIGN), (dict(workspace_bytes=100), WORKSPACE)])
def test_loss_backward(L, change, code):
    assert L.smlm_vocab_loss_bwd(*{**LOSS_BACK, **change}.values()) == code


def test_loss_sizes(L):
    n = C.c_size_t()
    size = L.smlm_vocab_loss_workspace_size
    assert size(4, 64, 100, 0, None) == ARG and size(4, 64, 100, 6, C.byref(n)) == ARG and size(4, 64, 100, -1, C.byref(n)) == ARG
    assert size(4, 60, 100, 0, C.byref(n)) == ALIGN and size(1 << 28, 64, 1 << 28, 0, C.byref(n)) == LIMIT
    assert all(size(4, 64, 100, what, C.byref(n)) == 0 and n.value > 0 for what in range(6))


@pytest.mark.parametrize("T", [1, 4, 32, 33, 64, 65, 300])
@pytest.mark.parametrize("V", [1 << 22, (1 << 22) + 1, 1 << 26, 1 << 28])
def test_loss_pieces_fit_their_offsets(L, T, V):
    """Exponentials and G live 512 MiB at a time (a tile more of the vocabulary at most), also where G of few rows is held twice, in 64 rows: rows
    are found by offsets of 32 bits."""
    n = C.c_size_t()
    # (beside them a few numbers a row; with the rows' gradient up to 512 partial tiles of 256 x 256 floats)
    for what, besides in ((2, 1 << 20), (1, 130 << 20), (3, 130 << 20)):
        assert L.smlm_vocab_loss_workspace_size(T, 8, V, what, C.byref(n)) == 0
        assert n.value <= (512 << 20) + 2 * 256 * max(T, 64) + besides


def test_loss_rows_that_no_launch_takes(L):
    n = C.c_size_t()
    for T, code in (((1 << 28) - 16, 0), ((1 << 28) - 15, LIMIT), (1 << 28, LIMIT)):  # (a workgroup for 16 rows: 2^32 threads are too many)
        assert all(L.smlm_vocab_loss_workspace_size(T, 8, 50, what, C.byref(n)) == code for what in range(6))


def adam(L, n=2, workspace=A, room=LOTS, sizes=(10, 300), params=(A, A + 1024), **change):
    where, at, count = (C.c_void_p * n)(*params[:n]), (C.c_void_p * n)(*([A] * n)), (C.c_int64 * n)(*sizes[:n])
    a = lib.AdamW(params=C.addressof(where), grads=C.addressof(at), sizes=C.addressof(count), step=A, group=A, hyper=A, exp_avg=A,
                  exp_avg_sq=A, avg_scale=A, sq_scale=A, master=A, n_tensors=n, n_groups=1, state_bits=8, dtype=1)
    for k, v in change.items():
        setattr(a, k, v)
    return L.smlm_adamw_step(C.byref(a), workspace, room, None)


@pytest.mark.parametrize("change,code", [
    (dict(n_tensors=-1), ARG), (dict(n_groups=-1), ARG), (dict(state_bits=16), ARG), (dict(dtype=3), DTYPE), (dict(dtype=2), ARG),
    (dict(params=(A, None)), ARG), (dict(sizes=(10, -1)), LIMIT), (dict(sizes=(10, (1 << 40) + 1)), LIMIT),
    (dict(sizes=(1 << 40, 1 << 40)), LIMIT), (dict(step=None), ARG), (dict(group=None), ARG), (dict(hyper=None), ARG),
    (dict(exp_avg=None), ARG), (dict(exp_avg_sq=None), ARG), (dict(avg_scale=None), ARG), (dict(sq_scale=None), ARG),
    (dict(workspace=None), ARG), (dict(exp_avg=A + 8), ALIGN), (dict(exp_avg_sq=A + 4), ALIGN), (dict(master=A + 4), ALIGN),
    (dict(workspace=A + 8), ALIGN), (dict(room=8), WORKSPACE), (dict(n_tensors=0), 0)])
def test_adamw(L, change, code):
    assert adam(L, **change) == code


def test_adamw_without_arguments(L):
    n = C.c_size_t()
    assert L.smlm_adamw_step(None, A, LOTS, None) == ARG
    assert L.smlm_adamw_workspace_size(-1, C.byref(n)) == ARG and L.smlm_adamw_workspace_size(3, None) == ARG
    assert L.smlm_adamw_workspace_size(3, C.byref(n)) == 0 and n.value > 0


def test_tensors_that_are_not_on_a_gpu():
    x, w, v = torch.zeros(4, 64).half(), torch.ones(64).half(), torch.ones(100, 64).half()
    with pytest.raises(RuntimeError):
        add_rms_norm.apply(x, x, w)
    with pytest.raises(RuntimeError):
        K.add_rms_norm(torch.empty_like(x), None, None, x, None, w, 1e-6)
    with pytest.raises(RuntimeError):
        linear_cross_entropy.apply(x, v, torch.zeros(4, dtype=torch.int64))
    f = torch.zeros(256)
    with pytest.raises(RuntimeError):
        K.adamw_step([x], [x], f, f, torch.zeros(1, dtype=torch.int32), torch.zeros(1, 5), torch.zeros(1, dtype=torch.int32))
    p = torch.nn.Parameter(x)
    p.grad = torch.zeros_like(p)
    with pytest.raises(RuntimeError):
        optim.AdamW([p]).step()
