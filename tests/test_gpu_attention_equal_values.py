"""Attention over values that are all alike gives that value: its weights add up to one as the second product meets them, whatever their
rounding to the element type.

Of every 32 keys one has the weight 1, and the others just short of the middle between two numbers of the type, so that each rounds down by
nearly the most that there is, u = eps / 2 of itself, whoever sums which of them; were they added up before that rounding, the result would be
u (1 - 2^-5) 15.5 / 16.5 = 0.91 u of itself too small, and the value, just under a power of two, has its neighbour 2 u / 2 of it away: the result
would be another number.  Added up as rounded, what is left is float arithmetic: a lane's sum of at most 2000 / 16 + 16 terms and some 16 steps
more, 2^-16 of the value at most, where half a step to the neighbour is 2^-12."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TDT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def K(gpu_device):
    from loquetier_amd import _lib
    from loquetier_amd.ops import _kernels
    _lib.load()
    return _kernels


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,cached", [(1, 60), (1, 1000), (3, 1500), (1, 20000), (40, 1000), (200, 900)])
def test_equal_values(K, dt, D, new, cached):
    t = TDT[dt]
    u = torch.finfo(t).eps / 2
    value = 2 - 2 * u  # the largest number under two
    length, P = new + cached, 16
    pages = -(-length // P)
    kc, vc = torch.zeros(pages, 2, P, D, dtype=t, device="cuda"), torch.full((pages, 2, P, D), value, dtype=t, device="cuda")
    kc[..., 0] = -1.0
    kc[::2, :, 3, 0] = 0.0
    q = torch.zeros(new, 4, D, dtype=t, device="cuda")
    q[..., 0] = 1.0
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    plan = K.AttentionPlan(ints([0, new]), ints([length]), ints([list(range(pages))]), new, 4, 2, P)
    out = torch.empty_like(q)
    K.paged_attention(out, q, kc, vc, plan, scale=math.log(2) - math.log1p(u * (1 - 2 ** -5)))
    assert bool((out == value).all()), f"{(out.float() - value).abs().max().item() / (2 * u)} steps off"
