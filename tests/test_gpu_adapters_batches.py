"""GPU: adapters over the ways a batch can lie: rows tiled in order of adapters or
as they stand, banks of many slots, prompts in 64-row tiles; and adapters together
with vocabulary sampling as a decode step uses them.  Bounds are those that
test_gpu_adapters derives.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cubic_serve_amd import linear, quantization as qz, sampling
from test_gpu_adapters import DEV, case, check, make_bank, rows_of

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def launch(x, banks, slots, bases):
    outputs = tuple(torch.full_like(b, float("nan")) for b in bases)
    linear.PackedLinearOperators().bind_adapters(x, banks, slots, outputs, bases=bases).launch()
    torch.cuda.synchronize()
    return outputs


def test_rows_in_order_of_adapters_and_as_they_stand_agree():
    """A bank of at most 255 slots has its rows tiled in order of adapters, a larger
    one as they stand: the same adapters give the same bits."""
    for dtype in DTYPES:
        gen = torch.Generator().manual_seed(11)
        n, k, ranks = 72, 1040, (12, 3, 0, 16, 7)
        small, held = make_bank(gen, n, k, ranks, 24, dtype)
        large, _ = make_bank(gen, n, k, (0,) * 300, 24, dtype)
        for s, (down, up, scale) in enumerate(held):
            if len(down):
                large.load(s, down.to(DEV), up.to(DEV), scale)
        for m in (17, 31, 128, 129, 255, 257, 512, 1000, 1024):
            for pattern in ("own", "one", "none", "runs", "mixed"):
                print(f"adapters: order m={m} {pattern} {dtype}", flush=True)
                x = torch.randn((m, k), generator=gen).to(dtype).to(DEV)
                base = torch.randn((m, n), generator=gen).to(dtype).to(DEV)
                slots = rows_of(pattern, m, len(ranks), gen)
                slots[slots >= len(ranks)] = -1
                slots = slots.to(torch.int32).to(DEV)
                got, = launch(x, small, slots, (base,))
                check(got, x, base, held, slots)
                other, = launch(x, large, slots, (base,))
                assert torch.equal(got, other)


@pytest.mark.parametrize("slots", [255, 256, 400])
def test_a_bank_of_many_slots(slots):
    for m in (20, 300, 1024):
        print(f"adapters: {slots} slots m={m}", flush=True)
        ranks = tuple(1 + s % 8 for s in range(slots))
        x, bases, banks, held, rows = case(m, 264, (40, 24), ranks, 8, torch.bfloat16, "mixed", seed=slots + m)
        for y, base, h in zip(launch(x, banks, rows, bases), bases, held):
            check(y, x, base, h, rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,ranks,capacity", [(16392, (72, 128, 9), 128), (16384, (256, 100), 256)])
def test_long_prompts_of_large_ranks(k, ranks, capacity, dtype):
    """Enough rows and columns for the 64-row tiles of the down product, the
    last of them ragged."""
    m = 2101
    print(f"adapters: prompts m={m} k={k} ranks={ranks} {dtype}", flush=True)
    x, bases, banks, held, slots = case(m, k, (72,), ranks, capacity, dtype, "runs", seed=12)
    slots[700:720] = torch.arange(20, dtype=torch.int32, device=DEV) % 4 - 1  # a tile of several requests
    got, = launch(x, banks, slots, bases)
    check(got, x, bases[0], held[0], slots)
    few = torch.randperm(m, generator=torch.Generator().manual_seed(2))[:40].to(DEV)
    part, = launch(x[few], banks, slots[few].contiguous(), (bases[0][few],))
    assert torch.equal(part, got[few])


@pytest.mark.parametrize("ranks,capacity", [((16, 5) * 6, 16), ((64, 40, 33) * 4, 64), ((128, 65) * 6, 128), ((200, 8) * 5, 200)])
def test_prompts_of_many_requests(ranks, capacity):
    """Columns that end inside a turn, tiles with rows of every adapter, and
    outputs that are column slices of one matrix."""
    for dtype in DTYPES:
        m, k, ns = 1090, 1032, (200, 72)
        print(f"adapters: prompts ranks={ranks[:2]} {dtype}", flush=True)
        x, bases, banks, held, slots = case(m, k, ns, ranks, capacity, dtype, "mixed", seed=13)
        both = torch.full((m, 280), 3.0, dtype=dtype, device=DEV)
        outputs = (both[:, :200], both[:, 208:])
        linear.PackedLinearOperators().bind_adapters(x, banks, slots, outputs, bases=bases).launch()
        torch.cuda.synchronize()
        for y, base, h in zip(outputs, bases, held):
            check(y, x, base, h, slots)
        assert (both[:, 200:208] == 3.0).all()


def test_two_streams_and_two_graphs():
    """Bindings have workspaces of their own: two of them at once, and two graphs
    replayed in turn, each keep their results."""
    print("adapters: two bindings on two streams, two graphs", flush=True)
    sets = []
    for seed in (14, 15):
        x, bases, banks, held, slots = case(300, 2056, (264,), (16, 40, 8), 40, torch.bfloat16, "mixed", seed=seed)
        y = torch.empty_like(bases[0])
        binding = linear.PackedLinearOperators().bind_adapters(x, banks, slots, y, bases=bases)
        binding.launch()
        torch.cuda.synchronize()
        check(y, x, bases[0], held[0], slots)
        sets.append((binding, y, y.clone()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for (binding, y, _), stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                y.fill_(float("nan"))
                binding.launch()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for _, y, want in sets)
    graphs = []
    for binding, y, _ in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            y.zero_()
            binding.launch()
    for turn in range(4):
        for (binding, y, want), graph in zip(sets, graphs):
            y.fill_(float("nan"))
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for _, y, want in sets)
        sets[turn % 2][0].launch()


def test_decode_step_adapters_then_a_token():
    """A step's end as a server runs it: the shared head with every request's
    adapter, then a token per row from its logits, captured and replayed while
    inputs, slots and settings change, against the eager step."""
    print("adapters and vocabulary sampling: a captured decode step", flush=True)
    gen = torch.Generator().manual_seed(16)
    rows, k, vocab, dtype = 24, 512, 4096, torch.bfloat16
    head = qz.quantize_cubic(torch.randn((vocab, k), generator=gen) * 0.1, bits=4, group_in=128).to(DEV)
    bank, held = make_bank(gen, vocab, k, (16, 4, 8), 16, dtype)
    x = torch.randn((rows, k), generator=gen).to(dtype).to(DEV)
    slots = torch.zeros(rows, dtype=torch.int32, device=DEV)
    logits = torch.empty((rows, vocab), dtype=dtype, device=DEV)
    full = lambda v, dt: torch.full((rows,), v, dtype=dt, device=DEV)
    params = dict(temperatures=full(1.0, torch.float32), top_ks=full(0, torch.int64), top_ps=full(1.0, torch.float32),
                  min_ps=full(0.0, torch.float32), uniforms=full(0.5, torch.float32))
    ops = linear.PackedLinearOperators()
    project = ops.bind_adapted_linear(x, head, logits, bank, slots)
    plan = sampling.VocabSamplingPlan(logits=logits, **params)
    live = torch.tensor([rows], dtype=torch.int32, device=DEV)

    def step():
        project.launch()
        plan.launch(live)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(4):
        x.copy_(torch.randn((rows, k), generator=gen))
        slots.copy_(torch.randint(-1, 3, (rows,), generator=gen))
        params["temperatures"].copy_(torch.tensor([0.0, 0.7, 1.0])[torch.arange(rows) % 3])
        params["top_ks"].copy_(torch.tensor([0, 40, 5, 1])[torch.arange(rows) % 4])
        params["top_ps"].copy_(torch.tensor([1.0, 0.9])[torch.arange(rows) % 2])
        params["uniforms"].copy_(torch.rand(rows, generator=gen))
        count = (rows, 5, 0, 19)[turn]
        live.fill_(count)
        plan.tokens.fill_(-9)
        graph.replay()
        torch.cuda.synchronize()
        seen = logits.clone(), plan.tokens.clone(), plan.logprobs.clone()
        check(logits, x, ops.linear(x, head), held, slots)
        assert (seen[1][count:] == -9).all() and (seen[1][:count] >= 0).all()
        # greedy rows: the first of the largest logits
        for r in range(0, count, 3):
            assert int(seen[1][r]) == int(np.argmax(seen[0][r].float().cpu().numpy()))
        step()
        torch.cuda.synchronize()
        assert torch.equal(logits, seen[0]) and torch.equal(plan.tokens, seen[1])
        assert torch.equal(plan.logprobs[:count], seen[2][:count])


@pytest.mark.parametrize("m,k,n", [(1, 1024, 40), (12, 6000, 40), (40, 520, 72), (300, 520, 72), (1100, 520, 72),
                                   (2101, 16384, 24)])
def test_what_lies_past_a_rank_is_not_used(m, k, n):
    """A's rows past a slot's rank hold NaN and infinities, and another row of x
    does: neither reaches a row that has no part in them."""
    print(f"adapters: past the rank m={m}", flush=True)
    ranks = (5, 17, 66, 1)
    x, bases, banks, held, slots = case(m, k, (n,), ranks, 72, torch.bfloat16, "mixed", seed=17)
    for s, r in enumerate(ranks):
        banks[0].down[s, r:] = float("nan")
        banks[0].down[s, (r + 72) // 2:] = float("inf")
    got, = launch(x, banks, slots, bases)
    check(got, x, bases[0], held[0], slots)
    if m > 1:
        spoilt = x.clone()
        spoilt[m // 2] = float("nan")
        other, = launch(spoilt, banks, slots, bases)
        rest = torch.arange(m, device=DEV) != m // 2
        assert torch.equal(other[rest], got[rest])


def test_joined_partitions_agree_with_added_ones():
    """Many partitions of K: joined in a launch of their own in batches of some
    size, added by the up kernel in smaller ones, with the same bits."""
    for dtype in DTYPES:
        print(f"adapters: joined partitions {dtype}", flush=True)
        x, bases, banks, held, slots = case(300, 8200, (264, 41), (48, 20, 7), 48, dtype, "mixed", seed=18)
        whole = launch(x, banks, slots, bases)
        for y, base, h in zip(whole, bases, held):
            check(y, x, base, h, slots)
        for rows in (65, 64, 17, 9, 1):
            part = launch(x[:rows], banks, slots[:rows], [b[:rows] for b in bases])
            assert all(torch.equal(p, w[:rows]) for p, w in zip(part, whole))


@pytest.mark.parametrize("m,ld", [(600, 1 << 21), (1100, 1 << 21), (40, 1 << 23)])
def test_rows_that_lie_far_apart(m, ld):
    """Row strides whose last rows start past 2^31 bytes, or past 2^30 elements in
    all, in batches that are otherwise tiled in order of adapters."""
    print(f"adapters: rows {ld} elements apart, m={m}", flush=True)
    x, bases, banks, held, slots = case(m, 264, (41,), (16, 7, 12), 16, torch.bfloat16, "mixed", seed=19)
    far = lambda t: torch.empty((m, ld), dtype=t.dtype, device=DEV)[:, :t.shape[1]].copy_(t)
    got = far(bases[0])
    linear.PackedLinearOperators().bind_adapters(far(x), banks, slots, got).launch()
    torch.cuda.synchronize()
    check(got, x, bases[0], held[0], slots)
    near, = launch(x, banks, slots, bases)
    assert torch.equal(got, near)
