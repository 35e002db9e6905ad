"""GPU: vocabulary sampling whose settings or live count a caller rewrites while
launches run.  Such a launch's tokens are not specified; they are columns or -1,
and the launches after it are as any other.
"""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import sampling
from test_gpu_vocab_sample import BF16, DEV, FP16, FP32, run, settings

pytestmark = pytest.mark.gpu
# one chunk per row, and several
SHAPES = [(BF16, 3, 100003), (FP16, 2, 151936), (BF16, 140, 20001), (FP32, 5, 100003), (FP32, 140, 20001)]


def counters(plan):
    return plan.workspace[:4 * plan.rows].view(torch.int32)


@pytest.mark.parametrize("dtype,rows,width", SHAPES)
@pytest.mark.parametrize("what", ["count", "settings", pytest.param("logits", marks=pytest.mark.skip(
    reason="logits must not change while a launch runs: 32-bit ones that did ended in a memory fault, its cause not found"))])
def test_operands_rewritten_while_launches_run(dtype, rows, width, what):
    print(f"sample {what} rewritten, rows={rows} width={width} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(26)
    logits = (torch.randn((rows, width), generator=gen) * 3).to(dtype).to(DEV)
    plan = run(logits, *settings(rows, gen))
    tokens, logprobs = plan.tokens.clone(), plan.logprobs.clone()
    live = torch.tensor([rows], dtype=torch.int32, device=DEV)
    kept = logits.clone(), [p.clone() for p in plan.parameters]
    others = (torch.randn((rows, width), generator=gen) * 30).to(dtype).to(DEV)
    others[0, ::3], others[-1, 5] = float("nan"), float("inf")
    zero = torch.zeros(rows, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for turn in range(60):
        plan.launch(live)
        with torch.cuda.stream(side):
            if what == "count":
                live.fill_(0 if turn % 2 else rows)
            elif what == "settings":  # greedy, refused, and as they were
                plan.parameters[0].copy_((zero, -1 - zero, kept[1][0])[turn % 3])
                plan.parameters[4].copy_((kept[1][4], 2 + zero)[turn % 2])
            else:
                logits.copy_(kept[0] if turn % 2 else others)
    torch.cuda.synchronize()
    assert (plan.tokens >= -1).all() and (plan.tokens < width).all()
    live.fill_(rows)
    logits.copy_(kept[0])
    for p, k in zip(plan.parameters, kept[1]):
        p.copy_(k)
    for count in (live, None):
        plan.tokens.fill_(-9), plan.logprobs.fill_(9.0)
        plan.launch(count)
        torch.cuda.synchronize()
        assert torch.equal(plan.tokens, tokens)
        assert torch.equal(plan.logprobs.nan_to_num(nan=5.0), logprobs.nan_to_num(nan=5.0))
        assert not counters(plan).any()


@pytest.mark.parametrize("dtype,rows,width", SHAPES)
def test_rows_past_a_device_count_leave_the_counters(dtype, rows, width):
    print(f"sample counters of rows past the count, rows={rows} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(27)
    logits = (torch.randn((rows, width), generator=gen) * 3).to(dtype).to(DEV)
    plan = run(logits, *settings(rows, gen))
    tokens = plan.tokens.clone()
    live = torch.zeros(1, dtype=torch.int32, device=DEV)
    for count in (0, 1, -5, rows - 1, rows + 7):
        plan.tokens.fill_(-9)
        live.fill_(count)
        plan.launch(live)
        torch.cuda.synchronize()
        n = min(max(count, 0), rows)
        assert torch.equal(plan.tokens[:n], tokens[:n]) and (plan.tokens[n:] == -9).all()
        assert not counters(plan).any()
