"""GPU: low-rank adapters beside a shared projection (cubic_adapters) against
their formula in 64 bits.

Tolerance, per element, from the arithmetic: t is a binary32 sum of k products
(each addition off by at most 2^-23 of the magnitudes added), enters the second
product as two 16-bit parts (off by 2^-17 of itself in bf16, by 2^-22 of its row's
largest in fp16), the second sum has 2 * rank products, the sum with the base
one rounding, and y is rounded once to its type (half a step).
"""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import adapters, linear, quantization as qz

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
HALF_STEP = {torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25)}


def make_bank(gen, n, k, ranks, capacity, dtype, scale=1.5):
    """A bank whose slot s has rank ranks[s] (0: left empty), and its adapters."""
    bank = adapters.AdapterBank(n, k, slots=len(ranks), max_rank=capacity, dtype=dtype, device=DEV)
    bank.up.fill_(float("nan"))  # load has to clear what the kernel reads
    bank.down.fill_(float("nan"))
    held = []
    for s, r in enumerate(ranks):
        down = (torch.randn((r, k), generator=gen) * k ** -0.5).to(dtype)
        up = (torch.randn((n, r), generator=gen) * 0.3).to(dtype)
        held.append((down, up, scale + s))
        if r:
            bank.load(s, down.to(DEV), up.to(DEV), scale + s)
    return bank, held


def reference(x, base, held, slots):
    """y and its bound, float64 on the CPU."""
    x, y = x.cpu().double(), base.cpu().double()
    step, tiny = HALF_STEP[base.dtype]
    bound = torch.zeros_like(y)
    k = x.shape[1]
    for s, (down, up, scale) in enumerate(held):
        mine = torch.nonzero(slots.cpu() == s)[:, 0]
        if not len(mine) or not down.shape[0]:
            continue
        a, b, xs = down.double(), up.double(), x[mine]
        t, off = xs @ a.t(), (xs.abs() @ a.abs().t()) * (k + 8) * 2.0 ** -23
        if base.dtype is torch.bfloat16:
            off = off + t.abs() * 2.0 ** -17
        else:
            off = off + t.abs().amax(1, keepdim=True) * 2.0 ** -22
        bound[mine] += scale * (off @ b.abs().t() + (t.abs() @ b.abs().t()) * (2 * len(a) + 4) * 2.0 ** -23)
        delta = scale * (t @ b.t())
        bound[mine] += (y[mine].abs() + delta.abs()) * 2.0 ** -23
        y[mine] += delta
    return y, bound + step * (y.abs() + bound) + tiny


def check(got, x, base, held, slots):
    want, bound = reference(x, base, held, slots)
    off = (got.cpu().double() - want).abs()
    worst = (off / bound.clamp_min(1e-300)).max().item()
    assert torch.isfinite(got).all() and worst <= 1.0, f"off by {worst} of the bound"


def rows_of(pattern, m, slots, gen):
    if pattern == "own":
        return torch.arange(m) % slots
    if pattern == "one":
        return torch.full((m,), slots - 1)
    if pattern == "none":
        return torch.full((m,), -1)
    if pattern == "runs":  # requests of ragged lengths, as a packed batch has them
        return (torch.arange(m) * 7 // max(1, m)) % slots
    return torch.randint(-1, slots + 1, (m,), generator=gen)  # any order, -1 and one past the bank


def case(m, k, ns, ranks, capacity, dtype, pattern, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=gen).to(dtype).to(DEV)
    bases = [torch.randn((m, n), generator=gen).to(dtype).to(DEV) for n in ns]
    banks, held = zip(*(make_bank(gen, n, k, ranks, capacity, dtype) for n in ns))
    slots = rows_of(pattern, m, len(ranks), gen).to(torch.int32).to(DEV)
    return x, bases, banks, held, slots


CASES = [
    # m, k, ns, ranks, capacity, pattern
    (1, 8, (1,), (1,), 1, "one"),
    (1, 4096, (4096, 1024, 1024), (16,), 16, "one"),
    (5, 1024, (64,), (8, 3, 0), 8, "mixed"),
    (16, 1032, (40, 24), (16, 9), 16, "own"),
    (17, 2056, (1001,), (12, 6, 3, 12, 1), 12, "mixed"),
    (64, 512, (256, 264), (16,) * 64, 16, "own"),
    (33, 48, (33, 31, 7), (33, 64, 1), 64, "mixed"),
    (128, 2048, (392,), (128, 17), 128, "runs"),
    (129, 1024, (512,), (64, 32, 16), 64, "runs"),       # two row tiles per workgroup
    (200, 3080, (129,), (256, 200), 256, "mixed"),       # widest rank
    (1024, 264, (96, 8), (24, 48), 48, "mixed"),
    (1025, 520, (256,), (16, 8, 4), 16, "runs"),         # four row tiles per workgroup
    (1300, 256, (72, 136, 48), (128, 100), 128, "mixed"),
    (1111, 264, (65,), (256, 31), 256, "mixed"),
    (40, 256, (64,) * 8, (40, 8), 40, "mixed"),          # every member of a full group
    (70, 64, (16,), (4, 4), 4, "none"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,ns,ranks,capacity,pattern", CASES)
def test_against_the_formula(m, k, ns, ranks, capacity, pattern, dtype):
    print(f"adapters m={m} k={k} ns={ns} ranks={ranks[:4]} {pattern} {dtype}", flush=True)
    x, bases, banks, held, slots = case(m, k, ns, ranks, capacity, dtype, pattern)
    outputs = tuple(torch.full_like(b, float("nan")) for b in bases)
    ops = linear.PackedLinearOperators()
    ops.bind_adapters(x, banks, slots, outputs, bases=bases).launch()
    inplace = tuple(b.clone() for b in bases)
    ops.bind_adapters(x, banks, slots, inplace).launch()
    torch.cuda.synchronize()
    none = (slots < 0) | (slots >= len(ranks))
    for s, r in enumerate(ranks):
        if not r:
            none |= slots == s
    for y, z, base, h in zip(outputs, inplace, bases, held):
        check(y, x, base, h, slots)
        assert torch.equal(y, z)
        assert torch.equal(y[none].view(torch.int16), base[none].view(torch.int16))


def test_a_row_does_not_depend_on_its_batch():
    print("adapters: rows of m=1300, 300, 40 and 1 agree bit for bit", flush=True)
    # ranks past and within what the one-launch kernel of few rows takes
    for dtype, ranks in ((torch.bfloat16, (64, 16, 40)), (torch.float16, (64, 16, 40)),
                         (torch.bfloat16, (16, 3, 9)), (torch.float16, (24, 32, 7))):
        x, (base,), (bank,), _, slots = case(1300, 2056, (264,), ranks, max(ranks), dtype, "mixed", seed=3)
        whole = torch.empty_like(base)
        ops = linear.PackedLinearOperators()
        ops.bind_adapters(x, bank, slots, whole, bases=base).launch()
        order = torch.randperm(1300, generator=torch.Generator().manual_seed(1)).to(DEV)
        for count in (300, 40, 1):
            pick = order[:count]
            part = torch.empty((count, 264), dtype=dtype, device=DEV)
            ops.bind_adapters(x[pick].contiguous(), bank, slots[pick].contiguous(), part,
                              bases=base[pick].contiguous()).launch()
            torch.cuda.synchronize()
            assert torch.equal(part, whole[pick])


def test_strided_operands_and_column_slices():
    print("adapters: x, base and output with row strides; q, k, v slices of one output", flush=True)
    dtype = torch.bfloat16
    x, bases, banks, held, slots = case(37, 256, (48, 24, 40), (16, 8), 16, dtype, "mixed", seed=4)
    wide_x = torch.full((37, 264 + 8), float("nan"), dtype=dtype, device=DEV)
    wide_x[:, 8:264] = x
    fused = torch.full((37, 120), 7.0, dtype=dtype, device=DEV)  # q, k, v, and 8 columns beside them
    slices = (fused[:, :48], fused[:, 48:72], fused[:, 72:112])
    for s, b in zip(slices, bases):
        s.copy_(b)
    linear.PackedLinearOperators().bind_adapters(wide_x[:, 8:264], banks, slots, slices).launch()
    odd = torch.full((37, 51), float("nan"), dtype=dtype, device=DEV)  # rows at odd addresses
    linear.PackedLinearOperators().bind_adapters(x, banks[0], slots, odd[:, 1:49], bases=bases[0]).launch()
    torch.cuda.synchronize()
    for s, b, h in zip(slices, bases, held):
        check(s, x, b, h, slots)
    assert torch.equal(odd[:, 1:49], slices[0])
    assert (fused[:, 112:] == 7).all() and odd[:, 0].isnan().all() and odd[:, 49:].isnan().all()


def test_non_finite_values_stay_in_their_rows():
    print("adapters: infinities and NaN in rows and adapters reach only their rows", flush=True)
    for dtype in (torch.bfloat16, torch.float16):
        for m in (30, 150, 1100):
            x, (base,), (bank,), (held,), slots = case(m, 264, (72,), (16, 8, 12), 16, dtype, "mixed", seed=5)
            x[3, 5], x[9, 100] = float("inf"), float("nan")
            slots[3], slots[9] = 0, 1
            bank.down[2, 1, 7] = float("nan")
            bank.up[2, 4, 0] = float("inf")
            y = torch.empty_like(base)
            linear.PackedLinearOperators().bind_adapters(x, bank, slots, y, bases=base).launch()
            torch.cuda.synchronize()
            bad = (slots == 2)
            bad[3] = bad[9] = True
            assert not torch.isfinite(y[bad].float()).all(1).any()
            clean = x.clone()
            clean[3, 5] = clean[9, 100] = 0
            keep = torch.nonzero(~bad)[:, 0]
            check(y[keep], clean[keep], base[keep], held, slots[keep])


def test_large_intermediate_in_half_precision():
    print("adapters: fp16 with an intermediate past fp16's range and one below it", flush=True)
    gen = torch.Generator().manual_seed(6)
    bank = adapters.AdapterBank(64, 512, slots=2, max_rank=8, dtype=torch.float16, device=DEV)
    big = torch.full((8, 512), 16.0, dtype=torch.float16)
    big += torch.randn((8, 512), generator=gen).half()
    held = []
    for s, (down, up) in enumerate(((big, 2.0 ** -10), (big * 2.0 ** -14, 64.0))):
        u = (torch.randn((64, 8), generator=gen) * up).half()
        held.append((down, u, 1.0 if s == 0 else 2.0 ** -3))
        bank.load(s, down.to(DEV), u.to(DEV), held[-1][2])
    x = (torch.rand((20, 512), generator=gen) * 32).half().to(DEV)
    x[10:] *= 2.0 ** -12
    slots = (torch.arange(20) // 10).to(torch.int32).to(DEV)
    base = torch.zeros((20, 64), dtype=torch.float16, device=DEV)
    y = torch.empty_like(base)
    linear.PackedLinearOperators().bind_adapters(x, bank, slots, y, bases=base).launch()
    torch.cuda.synchronize()
    check(y, x, base, held, slots)


def test_replay_follows_slots_and_bank():
    print("adapters: a captured launch follows new row slots, a reloaded and a cleared slot", flush=True)
    dtype = torch.bfloat16
    x, (base,), (bank,), (held,), slots = case(48, 1032, (264,), (16, 16, 8), 16, dtype, "own", seed=7)
    y = torch.zeros_like(base)
    binding = linear.PackedLinearOperators().bind_adapters(x, bank, slots, y, bases=base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a launch on a stream of its own
        binding.launch()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    check(y, x, base, held, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        binding.launch()
    gen = torch.Generator().manual_seed(8)
    held = list(held)
    for turn in range(4):
        if turn == 1:
            slots.copy_(torch.randint(-1, 3, (48,), generator=gen).to(torch.int32))
        if turn == 2:
            held[1] = ((torch.randn((5, 1032), generator=gen) * 0.03).to(dtype),
                       torch.randn((264, 5), generator=gen).to(dtype), 0.25)
            bank.load(1, held[1][0].to(DEV), held[1][1].to(DEV), 0.25)
        if turn == 3:
            bank.clear(0)
            held[0] = (torch.zeros((0, 1032)), torch.zeros((264, 0)), 0.0)
        y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = y.clone()
        check(replayed, x, base, held, slots)
        binding.launch()  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(y, replayed)


def test_adapted_linear_is_the_projection_with_its_adapters():
    print("adapted linear: single matrix and a group, one binding", flush=True)
    gen = torch.Generator().manual_seed(9)
    k, ns, m = 512, (256, 256), 24
    weights = [qz.quantize_cubic(torch.randn((n, k), generator=gen) * 0.02, bits=4, group_in=128).to(DEV) for n in ns]
    x = torch.randn((m, k), generator=gen).to(torch.bfloat16).to(DEV)
    banks, held = zip(*(make_bank(gen, n, k, (16, 4), 16, torch.bfloat16) for n in ns))
    slots = torch.randint(-1, 2, (m,), generator=gen).to(torch.int32).to(DEV)
    ops = linear.PackedLinearOperators()
    shared = [ops.linear(x, w) for w in weights]
    group = tuple(torch.empty_like(s) for s in shared)
    ops.bind_adapted_linear(x, weights, group, banks, slots).launch()
    alone = torch.empty_like(shared[0])
    binding = ops.bind_adapted_linear(x, weights[0], alone, banks[0], slots)
    binding.launch()
    binding.launch()  # the projection writes the output anew each time
    torch.cuda.synchronize()
    for y, base, h in zip(group, shared, held):
        check(y, x, base, h, slots)
    assert torch.equal(alone, group[0]) and binding.output is alone


def test_binding_refuses_what_it_cannot_run():
    x, bases, banks, _, slots = case(6, 64, (16, 24), (8, 8), 8, torch.bfloat16, "own")
    bind = linear.PackedLinearOperators().bind_adapters
    with pytest.raises(ValueError, match="one base and one output"):
        bind(x, banks, slots, bases[:1])
    with pytest.raises(ValueError, match="row slots"):
        bind(x, banks, slots.long(), bases)
    with pytest.raises(ValueError, match="row slots"):
        bind(x, banks, slots[:5], bases)
    with pytest.raises(ValueError, match="differ from the activations"):
        bind(x[:, :56].contiguous(), banks, slots, bases)
    with pytest.raises(ValueError, match="aligned"):
        bind(x[:, 1:57], banks, slots, bases)
    with pytest.raises(ValueError, match="invalid ABI"):
        bind(x, banks, slots, [bases[1], bases[0]])
    with pytest.raises(ValueError, match="invalid ABI"):
        bind(x, banks[0], slots, torch.empty((16, 6), dtype=x.dtype, device=DEV).t())
    with pytest.raises(ValueError, match="alias"):
        bind(x, [banks[0], banks[0]], slots, [bases[0], bases[0]])
    with pytest.raises(ValueError, match="alias"):
        bind(x, banks[0], slots, x[:, :16])
    both = torch.empty((6, 24), dtype=x.dtype, device=DEV)
    with pytest.raises(ValueError, match="alias"):  # output columns over another's base
        bind(x, [banks[0], banks[0]], slots, [both[:, :16], bases[0]], bases=[bases[0], both[:, 8:]])
    with pytest.raises(ValueError, match="one CUDA device"):
        bind(x, banks[0], slots.cpu(), bases[0])
    binding = bind(x, banks[0], slots, bases[0])
    slots.set_(torch.zeros(7, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="changed after binding"):
        binding.launch()
