"""GPU: 16-bit vocabulary sampling where one logit fills a chunk's counter (65536
columns and more of one bit pattern), the largest of the row among them.  The
definition and its bounds are those of test_gpu_vocab_sample.
"""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import sampling
from test_gpu_vocab_sample import BF16, DEV, FP16, FP32, check

pytestmark = pytest.mark.gpu
FULL = 65536


def bits(pattern, dtype):
    return torch.tensor([pattern - (1 << 16 if pattern >= 1 << 15 else 0)], dtype=torch.int16).view(dtype)


def rows_of(width, dtype, gen):
    """Rows whose largest logit, or NaN, fills a counter (an even pattern's carries
    into its neighbour, an odd one's is lost), where the width has room."""
    one, top = (0x3F80, 0x7F80) if dtype is BF16 else (0x3C00, 0x7C00)
    low = -4.0 - torch.rand(width, generator=gen).to(dtype)
    rows = [bits(p, dtype).expand(width).clone() for p in (0, one, one + 1, 0x8000 | one, 0x8000 | one + 1, 0x8000 | top - 1)]
    for pattern in (one, one + 1, 0x8000 | one, 0x8000 | one + 1, 0x0000, 0x8000):
        for number in (FULL, FULL + 1, 75968, 2 * FULL):
            row = low.clone()
            row[:number] = bits(pattern, dtype)
            if pattern & 0x7fff == one + 1 and number == FULL:  # the largest of all, once
                row[number // 2] = bits(one + 2 if pattern < 0x8000 else 0x8000 | one, dtype)
            rows.append(row)
    masked = torch.full((width,), float("-inf"), dtype=dtype)
    masked[-FULL:] = bits(one + 1, dtype)
    rows.append(masked)
    signed = torch.zeros(width, dtype=dtype)
    signed[::2] = -0.0
    rows.append(signed)
    for pattern in (top, top + 1, 0x7FFF, 0xFFFF, 0x8000 | top + 2):  # +inf and NaN
        row = low.clone()
        row[:FULL] = bits(pattern, dtype)
        rows.append(row)
    return torch.stack(rows)


# one chunk, several, and one again where rows fill the chip
@pytest.mark.parametrize("dtype,rows,width", [(FP16, 1, 65536), (FP16, 1, 131072), (FP16, 0, 151936), (BF16, 128, 151936),
                                              (BF16, 300, 70001)])
def test_the_largest_logit_fills_a_counter(dtype, rows, width):
    gen = torch.Generator().manual_seed(width)
    made = rows_of(width, dtype, gen)
    bad = torch.isnan(made).any(1) | torch.isposinf(made).any(1)
    largest = made == made.amax(1, keepdim=True)
    number = largest.sum(1)
    u = torch.rand(len(made), generator=gen)
    for at in range(len(made)) if rows == 1 else [slice(None)]:
        batch = made[at] if rows != 1 else made[at:at + 1]
        mine = slice(at, at + 1) if rows == 1 else at
        batch = torch.cat([batch, batch.new_zeros((max(0, rows - len(batch)), width))])
        count, kept = len(batch), len(made[mine])
        column = lambda v, dt=FP32: torch.full((count,), v, dtype=dt, device=DEV)
        uniforms = torch.zeros(count)
        uniforms[:kept] = u[mine]
        plan = sampling.VocabSamplingPlan(
            logits=batch.to(DEV), temperatures=column(0.0), top_ks=column(0, torch.int64), top_ps=column(1.0),
            min_ps=column(0.0), uniforms=uniforms.to(DEV))
        # the largest, or nothing but its equals: the next lies past min-p
        for temperature, min_p in ((0.0, 0.0), (1.0, 1.0), (1e-3, 0.5)):
            print(f"sample full counter {dtype} rows={count} width={width} {at} T={temperature}", flush=True)
            plan.parameters[0].fill_(temperature), plan.parameters[3].fill_(min_p)
            plan.tokens.fill_(-9), plan.valid.fill_(True), plan.logprobs.fill_(9.0)
            plan.launch()
            torch.cuda.synchronize()
            n = number[mine] if temperature else torch.ones_like(number[mine])
            nth = (u[mine].double() * n).long() + 1 if temperature else n
            token = (largest[mine].cumsum(1) < nth[:, None]).sum(1)
            got, ok, lp = (t.cpu()[:kept] for t in (plan.tokens, plan.valid, plan.logprobs))
            assert got.tolist() == torch.where(bad[mine], -1, token).tolist()
            assert torch.equal(ok, ~bad[mine]) and torch.equal(lp.isnan(), bad[mine])
            # the sums are exact here: the logarithm, then binary32's half step
            want = -n.double().log()
            assert ((lp.double() - want).abs() <= want.abs() * (2.0 ** -24 + 2.0 ** -50))[~bad[mine]].all()
        if rows != 1:  # every column weighs something, top-k cuts among equals
            plan.parameters[0].fill_(50.0), plan.parameters[1].fill_(70000), plan.parameters[3].fill_(0.0)
            plan.launch()
            torch.cuda.synchronize()
            check(plan, rows=12)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_more_rows_than_a_grid_holds(dtype):
    """4194304 workgroups of 1024 threads are more than one launch takes."""
    rows, width = (1 << 22) + 37, 4
    print(f"sample rows={rows} {dtype}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(25)
    logits = torch.randn((rows, width), generator=gen, device=DEV).to(dtype)
    logits[5, 2] = float("nan")
    column = lambda v, dt=FP32: torch.full((rows,), v, dtype=dt, device=DEV)
    params = dict(temperatures=column(0.0), top_ks=column(0, torch.int64), top_ps=column(1.0), min_ps=column(0.0),
                  uniforms=torch.rand(rows, generator=gen, device=DEV))
    params["temperatures"][-50:] = 1.0
    plan = sampling.VocabSamplingPlan(logits=logits, **params)
    plan.tokens.fill_(-9)
    live = torch.tensor([rows - 3], dtype=torch.int32, device=DEV)
    plan.launch(live)
    torch.cuda.synchronize()
    first = (logits == logits.amax(1, keepdim=True)).int().argmax(1)
    first[5] = -1
    assert torch.equal(plan.tokens[:-50], first[:-50]) and not plan.valid[5] and plan.valid[6]
    last = sampling.VocabSamplingPlan(logits=logits[-50:], **{k: v[-50:] for k, v in params.items()})
    last.launch()
    torch.cuda.synchronize()
    check(last)
    assert torch.equal(plan.tokens[-50:-3], last.tokens[:-3]) and torch.equal(plan.logprobs[-50:-3], last.logprobs[:-3])
    assert (plan.tokens[-3:] == -9).all()
