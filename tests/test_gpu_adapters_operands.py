"""GPU: adapters on operands at the edges of what a binding takes, and values
at the edges of their types.  Bounds are those that test_gpu_adapters derives.
"""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import adapters, linear
from test_gpu_adapters import DEV, case, check, reference

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("stride", [0, 1, 260, 267])
def test_a_single_row_of_any_stride(stride):
    """The row stride of one row means nothing, of the activations as of the others."""
    print(f"adapters: one row, stride {stride}", flush=True)
    x, (base,), banks, (held,), slots = case(1, 264, (40,), (16, 5), 16, torch.bfloat16, "one", seed=20)
    at = lambda t: t.clone().as_strided(t.shape, (stride, 1))
    y = at(base)
    linear.PackedLinearOperators().bind_adapters(at(x), banks, slots, y).launch()
    torch.cuda.synchronize()
    check(y, x, base, held, slots)


def classes(base, x, held, slots):
    """What the formula gives where an adapter holds infinities: +-inf, NaN, or 0
    for a finite value; t itself is far from 0 in these cases."""
    want = torch.zeros(base.shape, dtype=torch.float64)
    for s, (down, up, scale) in enumerate(held):
        mine = torch.nonzero(slots.cpu() == s)[:, 0]
        t = x.cpu().double()[mine] @ down.double().t() * scale
        for r in range(down.shape[0]):
            want[mine] += torch.where(torch.isinf(up[:, r].double())[None], t[:, r, None] * up[:, r].double()[None], 0.0)
    return want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,ranks,capacity", [
    (1, 264, (16,), 16), (12, 520, (16, 5), 16),            # one launch
    (12, 520, (40, 33), 40), (12, 5128, (8, 12), 16),       # 16-row tiles as they stand
    (300, 264, (16, 3), 16), (300, 264, (256, 70), 256),    # in order of adapters
    (1100, 264, (16, 9), 16), (1100, 264, (64, 33), 64), (1100, 264, (128, 100), 128),  # prompts
    (1100, 264, (200, 16), 200),
])
def test_infinities_in_the_second_matrix(m, k, ranks, capacity, dtype):
    """A product with an infinity is that infinity, whatever bits the row's
    intermediate value takes to hold; two of one sign stay, of two signs are NaN."""
    print(f"adapters: infinities in B, m={m} ranks={ranks} {dtype}", flush=True)
    n = 72
    x, (base,), (bank,), (held,), slots = case(m, k, (n,), ranks, capacity, dtype, "own", seed=21)
    x.abs_()
    held = list(held)
    for s, r in enumerate(ranks):
        down, up, scale = held[s]
        # t far from 0, of either sign; one exactly a power of two: its later parts are 0
        down = (down.abs() + 0.05) * torch.where(torch.arange(r) % 3 == 1, -1.0, 1.0)[:, None].to(dtype)
        down[r - 1] = 0
        down[r - 1, 0] = 1.0
        up = up.clone()
        up[3, 0], up[20, 1 % r], up[21, r - 1] = float("inf"), float("-inf"), float("inf")
        up[40, 0] = up[40, r // 2] = float("inf")
        up[71, 0], up[71, r - 1] = float("inf"), float("-inf")
        held[s] = (down.to(dtype), up, 0.5)
        bank.load(s, held[s][0].to(DEV), up.to(DEV), 0.5)
    x[:, 0] = 2.0
    want = classes(base, x, held, slots)
    y = torch.empty_like(base)
    linear.PackedLinearOperators().bind_adapters(x, bank, slots, y, bases=base).launch()
    torch.cuda.synchronize()
    got = y.cpu().double()
    assert torch.isnan(want).any() and torch.isinf(want).any()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    assert torch.equal(torch.sign(got)[torch.isinf(want)], torch.sign(want)[torch.isinf(want)])
    # every other element is what it is without them
    clean = [(d, torch.where(torch.isinf(u), torch.zeros_like(u), u), s) for d, u, s in held]
    value, bound = reference(x, base, clean, slots)
    finite = want == 0
    assert ((got - value).abs() <= bound)[finite].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,rank,capacity", [(5, 1, 16), (5, 3, 40), (40, 1, 16), (300, 2, 64), (300, 1, 256), (1100, 1, 16),
                                             (1100, 2, 64), (1100, 1, 128), (1100, 1, 200)])
def test_a_base_that_cancels_the_adapter(m, rank, capacity, dtype):
    """The base is minus what the adapter adds, rounded: what is left is that rounding,
    and holds whatever the intermediate value was held to.  x has one entry per row,
    so that a row's t is one product, exact in binary32, times the scale (half
    a step of it off); the second product sums 3 * rank products of its parts (each
    addition off by at most 2^-23 of what is added), the base is one more, and y
    is rounded once.  (A t of two bf16 parts, off by 2^-17, is past this bound.)"""
    print(f"adapters: cancellation m={m} rank={rank} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(22)
    n, k, scale = 488, 264, 1.2345678806304932  # a binary32 number with all its bits
    bank = adapters.AdapterBank(n, k, slots=2, max_rank=capacity, dtype=dtype, device=DEV)
    x = torch.zeros((m, k), dtype=dtype)
    x[torch.arange(m), torch.arange(m) * 7 % k] = (torch.rand(m, generator=gen) + 1).to(dtype)
    slots = (torch.arange(m) % 2).to(torch.int32)
    want, off = torch.zeros((m, n), dtype=torch.float64), torch.zeros((m, n), dtype=torch.float64)
    for s in range(2):
        down, up = (torch.randn(shape, generator=gen).to(dtype) for shape in ((rank, k), (n, rank)))
        bank.load(s, down.to(DEV), up.to(DEV), scale)
        t = x[s::2].double() @ down.double().t() * scale
        want[s::2] = t @ up.double().t()
        off[s::2] = t.abs() @ up.double().abs().t() * (2.0 ** -24 + (3 * rank + 1) * 2.0 ** -23)
    base = (-want).to(dtype)
    y = torch.empty((m, n), dtype=dtype, device=DEV)
    linear.PackedLinearOperators().bind_adapters(x.to(DEV), bank, slots.to(DEV), y, bases=base.to(DEV)).launch()
    torch.cuda.synchronize()
    want += base.double()
    off += base.double().abs() * 2.0 ** -23
    half, least = (2.0 ** -8, 0.0) if dtype is torch.bfloat16 else (2.0 ** -11, 2.0 ** -25)
    worst = ((y.cpu().double() - want).abs() / (off + half * (want.abs() + off) + least)).max().item()
    print(f"  off by {worst:.2f} of the bound", flush=True)
    assert worst <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,capacity", [(7, 16), (7, 40), (300, 16), (300, 200), (1100, 32), (1100, 128), (1100, 256)])
def test_an_infinite_row_is_infinite_and_nan_is_nan(m, capacity, dtype):
    """Rank 1: an infinity of x makes t one, and y the base plus it times B; a NaN of x
    makes its row NaN."""
    print(f"adapters: infinite rows m={m} capacity={capacity} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(23)
    n, k = 72, 264
    bank = adapters.AdapterBank(n, k, slots=1, max_rank=capacity, dtype=dtype, device=DEV)
    down, up = torch.ones((1, k), dtype=dtype), torch.randn((n, 1), generator=gen).to(dtype)
    up[5] = 0
    bank.load(0, down.to(DEV), up.to(DEV), 0.75)
    x = torch.randn((m, k), generator=gen).to(dtype)
    x[0, 3], x[m // 2, 9], x[m - 1, 11] = float("inf"), float("-inf"), float("nan")
    base = torch.randn((m, n), generator=gen).to(dtype)
    y = torch.empty((m, n), dtype=dtype, device=DEV)
    slots = torch.zeros(m, dtype=torch.int32, device=DEV)
    linear.PackedLinearOperators().bind_adapters(x.to(DEV), bank, slots, y, bases=base.to(DEV)).launch()
    torch.cuda.synchronize()
    got = y.cpu()
    for row, sign in ((0, 1.0), (m // 2, -1.0)):
        want = sign * float("inf") * up[:, 0].float()
        assert torch.equal(torch.isnan(got[row]), torch.isnan(want)) and int(torch.isnan(want).sum()) == 1
        assert torch.equal(got[row].float().nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
    assert torch.isnan(got[m - 1]).all()
    rest = [r for r in range(1, m - 1) if r != m // 2]
    assert torch.isfinite(got[rest]).all()
