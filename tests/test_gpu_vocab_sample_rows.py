"""GPU: vocabulary sampling where its counts and lists are at their limits, on
several streams, and its refusals.  The definition and its bounds are those of
test_gpu_vocab_sample.
"""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import sampling
from test_gpu_vocab_sample import BF16, DEV, FP16, FP32, check, run, settings

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_more_columns_of_a_logit_than_a_counter_holds(dtype):
    """Rows of one chunk with 65535, 65536, 70000 and 200000 columns of one bit
    pattern, among others and alone."""
    print(f"sample full counters {dtype}", flush=True)
    gen = torch.Generator().manual_seed(21)
    logits = (torch.randn((200, 200000), generator=gen)).to(dtype)
    for r, number in enumerate((65535, 65536, 70000, 131072, 200000)):
        where = torch.randperm(200000, generator=gen)[:number]
        logits[r, where] = (2.0, -1.0, 0.0, 3.0, 1.0)[r]
    logits = logits.to(DEV)
    u = torch.rand(200, generator=gen)
    for top_k, top_p in ((0, 1.0), (60000, 0.9)):
        check(run(logits, 1.0, top_k, top_p, 0.0, u), rows=6)


# few chunks, many, and one per row
@pytest.mark.parametrize("rows,width", [(8, 60001), (100, 140003), (140, 50002)])
def test_wide_bins_of_32_bit_logits(rows, width):
    """More distinct columns in a bin of the first digit than are gathered, a key
    held by more columns than are ranked at once, logits that were 16-bit ones, and
    negative numbers about zero."""
    print(f"sample 32-bit rows={rows} width={width}", flush=True)
    gen = torch.Generator().manual_seed(rows)
    logits = torch.randn((rows, width), generator=gen) * 2
    logits[0] = 1.0 + torch.rand(width, generator=gen) / 8
    logits[1] = (logits[1] * 0.5).round()
    logits[2] = logits[2].bfloat16().float()
    logits[3] = -torch.rand(width, generator=gen) * 1e-6
    logits[3, ::5] = -0.0
    logits[3, 1::5] = 0.0
    logits[4] = torch.where(torch.rand(width, generator=gen) < 0.999, float("-inf"), logits[4])
    logits[5] = torch.rand(width, generator=gen) * 1e-30
    logits = logits.to(DEV)
    u = torch.rand(rows, generator=gen)
    for temperature, top_k, top_p, min_p in ((1.0, 0, 1.0, 0.0), (0.7, width // 2, 0.8, 0.0), (1.0, 300, 0.95, 0.1),
                                             (1.5, 0, 0.5, 0.0)):
        check(run(logits, temperature, top_k, top_p, min_p, u), rows=6)


def test_rows_agree_whatever_their_batch():
    """A row's token and log-probability depend on the row alone: chunks differ
    with the number of rows, results do not."""
    for dtype in (BF16, FP16, FP32):
        print(f"sample rows in batches {dtype}", flush=True)
        gen = torch.Generator().manual_seed(22)
        logits = (torch.randn((130, 40003), generator=gen) * 2.5).to(dtype).to(DEV)
        params = settings(130, gen)
        whole = run(logits, *params)
        for rows in (60, 7, 1):
            part = run(logits[:rows], *(p[:rows] for p in params))
            assert torch.equal(part.tokens, whole.tokens[:rows])
            assert torch.equal(part.logprobs, whole.logprobs[:rows])


def test_two_plans_on_two_streams():
    print("sample two plans at once, two graphs in turn", flush=True)
    gen = torch.Generator().manual_seed(23)
    plans, graphs = [], []
    for dtype in (BF16, FP32):
        logits = (torch.randn((20, 60000), generator=gen) * 3).to(dtype).to(DEV)
        plan = run(logits, *settings(20, gen))
        check(plan)
        plans.append((plan, plan.tokens.clone(), plan.logprobs.clone()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def agree():
        torch.cuda.synchronize()
        for plan, tokens, logprobs in plans:
            assert torch.equal(plan.tokens, tokens) and torch.equal(plan.logprobs, logprobs)
            plan.tokens.fill_(-9), plan.logprobs.fill_(9.0)
        torch.cuda.synchronize()

    for _ in range(5):
        for (plan, *_), stream in zip(plans, streams):
            with torch.cuda.stream(stream):
                plan.launch()
    agree()
    for plan, *_ in plans:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            plan.launch()
    for _ in range(4):
        for graph in graphs:
            graph.replay()
        agree()
        for plan, *_ in plans:
            plan.launch()
        agree()


def test_plan_refusals():
    rows = 4
    full = lambda v, dt=FP32, n=rows: torch.full((n,), v, dtype=dt, device=DEV)
    good = dict(logits=torch.zeros((rows, 64), device=DEV), temperatures=full(1.0), top_ks=full(0, torch.int64),
                top_ps=full(1.0), min_ps=full(0.0), uniforms=full(0.5))
    plan = sampling.VocabSamplingPlan(**good)
    for changes in ({"logits": good["logits"].double()}, {"logits": good["logits"][0]}, {"logits": good["logits"].t()},
                    {"logits": good["logits"][:, ::2]}, {"logits": good["logits"][:0]},
                    {"logits": good["logits"][:1].expand(rows, 64)}, {"temperatures": full(1.0, n=3)},
                    {"temperatures": full(1.0, torch.float64)}, {"top_ks": full(0, torch.int32)},
                    {"top_ps": full(1.0).cpu()}, {"min_ps": full(0.0, n=8)[::2]}, {"visible_width": 65},
                    {"visible_width": 0}, {"visible_width": True}, {"visible_width": 8.0},
                    {"logits": torch.zeros((rows, (1 << 20) + 1), dtype=BF16, device=DEV)}):
        with pytest.raises(ValueError):
            sampling.VocabSamplingPlan(**{**good, **changes})
    for live in (-1, 5, True, 2.0, torch.tensor([1], dtype=torch.int32), torch.tensor([1], device=DEV),
                 torch.zeros(0, dtype=torch.int32, device=DEV)):
        with pytest.raises(ValueError, match="live row count"):
            plan.launch(live)
    plan.launch()
    good["uniforms"].set_(full(0.5, n=6))
    with pytest.raises(ValueError, match="changed after binding"):
        plan.launch()


def test_plan_is_not_made_under_capture():
    print("sample plan under capture", flush=True)
    full = lambda v, dt=FP32: torch.full((4,), v, dtype=dt, device=DEV)
    good = dict(logits=torch.zeros((4, 64), device=DEV), temperatures=full(1.0), top_ks=full(0, torch.int64),
                top_ps=full(1.0), min_ps=full(0.0), uniforms=full(0.5))
    plan = sampling.VocabSamplingPlan(**good)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before graph capture"):
            sampling.VocabSamplingPlan(**good)
        plan.launch()
    graph.replay()
    torch.cuda.synchronize()
    assert plan.tokens.tolist() == [32] * 4


def test_rows_that_lie_far_apart():
    """Rows that start past 2^32 bytes."""
    for dtype, stride in ((BF16, 1 << 30), (FP32, 1 << 29)):
        print(f"sample rows {stride} elements apart", flush=True)
        gen = torch.Generator().manual_seed(24)
        near = (torch.randn((4, 20001), generator=gen) * 3).to(dtype).to(DEV)
        far = torch.empty(3 * stride + 20001, dtype=dtype, device=DEV).as_strided((4, 20001), (stride, 1))
        far.copy_(near)
        params = settings(4, gen)
        plan = run(far, *params)
        check(plan)
        assert torch.equal(plan.tokens, run(near, *params).tokens)
        del far, plan
