"""GPU: sampling from the whole vocabulary (cubic_vocab_sample) against its
definition in extended precision.

Tokens have to be equal, except where the definition itself is undecided within
the arithmetic's error: a weight is off by at most half of 2^-43 (fixed point,
the largest weight being 1) and by 2^-44 of itself (the exponent's product and
the polynomial), so a sum over V columns is off by at most V 2^-44 + its own
2^-44, and a comparison with a border that is nearer than that may go either way.
The reference evaluates both ways and gives every token that can come out;
nearly always that is one.  A log-probability is off by that relative error of
the kept mass, by 2^-45 of the exponent and by binary32's half step.
"""
from __future__ import annotations

import itertools
import math

import numpy as np
import pytest
import torch

from cubic_serve_amd import sampling

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def possible(row, temperature, top_k, top_p, min_p, u):
    """[(token, logprob)] that may come out; [(-1, nan)] for a refused row."""
    row = np.asarray(row, np.float64)
    ok = (0 <= temperature < math.inf and 0 < top_p <= 1 and 0 <= min_p <= 1 and 0 <= u < 1
          and not np.isnan(row).any() and not np.isposinf(row).any() and np.isfinite(row).any())
    if not ok:
        return [(-1, math.nan)]
    order = np.argsort(-(row + 0.0), kind="stable")
    if temperature == 0:
        return [(int(order[0]), 0.0)]
    z = (row[order].astype(np.longdouble) - row[order[0]]) / np.longdouble(temperature)
    weight = np.exp(z)
    mass = np.cumsum(weight)
    count = len(row) if top_k <= 0 or top_k > len(row) else int(top_k)
    error = len(row) * 2.0 ** -44 + float(mass[-1]) * 2.0 ** -44
    found = {}
    for dp, dm, du in itertools.product((0, -1, 1), repeat=3):
        total = mass[count - 1]
        keep = min(count, 1 + int(np.searchsorted(mass[:count], top_p * total + dp * error, side="left")))
        if top_p == 1:
            keep = count
        # w >= min-p is z >= ln min-p: decided where they are 2^-40 apart, and
        # for equal logits (z = 0; e^z rounds to 1 for more than those)
        likely = (z >= (math.log(min_p) if min_p else -math.inf) + dm * 2.0 ** -40) | (z == 0)
        keep = max(1, min(keep, int(likely.sum())))
        at = int(np.searchsorted(mass[:keep], u * mass[keep - 1] + du * error, side="right"))
        at = min(at, keep - 1)
        while at > 0 and weight[at] == 0:
            at -= 1
        found.setdefault(int(order[at]), float(z[at] - np.log(mass[keep - 1])))
    return list(found.items())


def run(logits, temperature, top_k, top_p, min_p, u, **kwargs):
    rows = logits.shape[0]
    column = lambda v, dt: torch.as_tensor(v, dtype=dt).expand(rows).contiguous().to(DEV)
    plan = sampling.VocabSamplingPlan(
        logits=logits, temperatures=column(temperature, FP32), top_ks=column(top_k, torch.int64),
        top_ps=column(top_p, FP32), min_ps=column(min_p, FP32), uniforms=column(u, FP32), **kwargs)
    plan.launch()
    torch.cuda.synchronize()
    return plan


def check(plan, width=None, rows=None):
    logits = plan.logits[:, :plan.width].float().cpu().numpy()
    params = [p.cpu().numpy() for p in plan.parameters]
    tokens, valid, logprobs = plan.tokens.cpu(), plan.valid.cpu(), plan.logprobs.cpu()
    undecided = 0
    for r in range(logits.shape[0] if rows is None else rows):
        t, k, p, m, u = (float(params[0][r]), int(params[1][r]), *(float(x[r]) for x in params[2:]))
        want = dict(possible(logits[r], t, k, p, m, u))
        got = int(tokens[r])
        assert got in want, f"row {r}: token {got}, of {list(want)[:4]} (T={t} k={k} p={p} min-p={m} u={u})"
        assert bool(valid[r]) == (got >= 0)
        undecided += len(want) > 1
        lp = float(logprobs[r])
        if got < 0:
            assert math.isnan(lp)
        elif len(want) == 1:
            z = abs(want[got])
            slack = 2.0 ** -24 * z + logits.shape[1] * 2.0 ** -44 + (z + 60) * 2.0 ** -45 + 2.0 ** -44
            assert abs(lp - want[got]) <= slack, f"row {r}: logprob {lp}, {want[got]}"
    return undecided


def settings(rows, gen):
    """Every kind of setting, by row."""
    pick = lambda values: torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=gen)]
    return (pick([0.0, 0.3, 0.7, 1.0, 1.0, 1.7, 50.0]), pick([0, -1, 1, 2, 20, 50, 1000, 10 ** 9]),
            pick([1.0, 1.0, 0.95, 0.9, 0.5, 0.1, 1e-6]), pick([0.0, 0.0, 0.05, 0.3, 1.0, 1e-4]),
            torch.rand(rows, generator=gen))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (5, 7), (40, 333), (64, 4096), (48, 8193), (70, 32768),
                                        (16, 65537), (9, 151936), (300, 2048)])
def test_against_the_definition(rows, width, dtype):
    print(f"sample rows={rows} width={width} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(rows * width)
    logits = (torch.randn((rows, width), generator=gen) * 3).to(dtype).to(DEV)
    undecided = check(run(logits, *settings(rows, gen)))
    assert undecided <= 1 + rows // 20


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_ties_masks_and_extreme_values(dtype):
    print(f"sample ties, masks, extremes {dtype}", flush=True)
    gen = torch.Generator().manual_seed(5)
    width, low = 20011, torch.finfo(dtype).min
    rows = []
    rows.append(torch.zeros(width))                                             # all equal
    rows.append(torch.full((width,), low))                                      # all the lowest finite value
    rows.append(torch.where(torch.rand(width, generator=gen) < 0.01, 1.5, -math.inf))  # a mask, equal values
    one = torch.full((width,), -math.inf)
    one[width - 1] = -7.0                                                       # one column left, the last
    rows.append(one)
    few = torch.full((width,), low)
    few[[3, 77, 4096, 9001]] = torch.tensor([2.0, 2.0, 1.0, 2.0])               # lowest as a mask
    rows.append(few)
    rows.append(torch.randint(-2, 3, (width,), generator=gen).float())          # five values
    signed = torch.zeros(width)
    signed[::2] = -0.0                                                          # +0 and -0 tie
    rows.append(signed)
    rows.append(torch.randn(width, generator=gen) * 1e-3 + 100)                 # far from 0, close together
    rows.append(torch.randn(width, generator=gen) * (torch.finfo(dtype).max / 8))  # huge spread
    rows.append(torch.randn(width, generator=gen) * (1e-40 if dtype != FP16 else 1e-7))  # subnormal
    alone = torch.randn(width, generator=gen)
    alone[123] = 60.0                                                           # one column with nearly all mass
    rows.append(alone)
    base = torch.stack(rows).to(dtype)
    for params in ((1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 3, 1.0, 1.0),
                   (0.0, 0, 1.0, 0.0), (2.0, width - 1, 0.999, 1e-3), (1e-30, 0, 1.0, 0.0), (1e30, 0, 0.25, 0.0)):
        for u in (0.0, 0.25, 0.5, 0.7321, 1 - 2.0 ** -24):
            check(run(base.to(DEV), *params, u))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_uniform_rows_are_counted_exactly(dtype):
    """Equal logits: the token is the column floor(u K), K columns kept."""
    width = 30000
    logits = torch.full((8, width), -3.0, dtype=dtype, device=DEV)
    u = torch.tensor([0.0, 0.125, 0.5, 0.75, 0.99993896484375, 0.3, 0.6, 0.9])
    for top_k, kept in ((0, width), (1000, 1000), (1, 1)):
        plan = run(logits, 1.0, top_k, 1.0, 0.0, u)
        want = [int(math.floor(float(np.float32(v)) * kept)) for v in u]
        assert plan.tokens.tolist() == want
        assert torch.allclose(plan.logprobs.cpu(), torch.full((8,), -math.log(kept)), rtol=2.0 ** -23, atol=0)
    plan = run(logits, 1.0, 0, 0.5, 0.0, u)  # exactly half of the columns
    assert plan.tokens.tolist() == [int(math.floor(float(np.float32(v)) * (width // 2))) for v in u]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_refused_rows(dtype):
    print(f"sample refused rows {dtype}", flush=True)
    gen = torch.Generator().manual_seed(6)
    logits = torch.randn((16, 5000), generator=gen).to(dtype)
    logits[0, 4999] = math.nan
    logits[1, 0] = math.inf
    logits[2] = -math.inf
    logits[3, 17] = -math.nan
    logits[4, :4999] = -math.inf
    t, k, p, m, u = torch.ones(16), torch.zeros(16, dtype=torch.int64), torch.ones(16), torch.zeros(16), \
        torch.full((16,), 0.5)
    t[5], t[6], t[7] = -1.0, math.nan, math.inf
    p[8], p[9], p[10] = 0.0, 1.5, math.nan
    m[11], m[12] = -0.1, math.nan
    u[13], u[14] = 1.0, math.nan
    plan = run(logits.to(DEV), t, k, p, m, u)
    check(plan)
    assert [r for r in range(16) if plan.tokens[r] >= 0] == [4, 15]


@pytest.mark.parametrize("rows,width,spread", [(70, 120000, None), (260, 60001, None), (64, 151936, 3.0)])
def test_many_distinct_logits(rows, width, spread):
    """fp16 logits of more distinct values than a chunk's list, or than the
    search's LDS, holds: all finite bit patterns, or N(0, 3)."""
    print(f"sample distinct rows={rows} width={width} {spread}", flush=True)
    gen = torch.Generator().manual_seed(width)
    if spread:
        logits = (torch.randn((rows, width), generator=gen) * spread).half()
        temperature = 1.0
    else:
        logits = torch.randint(-32768, 32768, (rows, width), generator=gen, dtype=torch.int32).to(torch.int16)
        logits = logits.view(torch.float16)
        logits = torch.where(torch.isfinite(logits), logits, torch.zeros((), dtype=FP16))
        temperature = 2e4
    few = torch.arange(0, rows, max(1, rows // 12))
    _, top_k, top_p, min_p, u = settings(rows, gen)
    plan = run(logits.to(DEV), temperature, top_k, top_p, min_p, u)
    part = sampling.VocabSamplingPlan.__new__(sampling.VocabSamplingPlan)
    part.logits, part.width = plan.logits[few.to(DEV)], plan.width
    part.parameters = [p[few.to(DEV)] for p in plan.parameters]
    part.tokens, part.valid, part.logprobs = (t[few.to(DEV)] for t in (plan.tokens, plan.valid, plan.logprobs))
    check(part)


def test_rows_with_strides_and_a_visible_width():
    print("sample strided rows, visible width", flush=True)
    gen = torch.Generator().manual_seed(7)
    for dtype, cols in itertools.product((BF16, FP16, FP32), (1003, 40001)):
        store = torch.full((24, cols + 13), math.nan, dtype=dtype)
        store[:, 5:5 + cols] = (torch.randn((24, cols), generator=gen) * 2).to(dtype)
        logits = store.to(DEV)[:, 5:]  # rows at any alignment, NaN before and behind
        check(run(logits, *settings(24, gen), visible_width=cols))
        plan = run(logits, 1.0, 0, 1.0, 0.0, 0.5, visible_width=1)
        assert plan.tokens.tolist() == [0] * 24 and plan.logprobs.abs().max() == 0


def test_live_rows_and_replay():
    """Rows past the live count keep their outputs; a captured launch follows
    new logits, parameters and counts."""
    print("sample live rows, captured replays", flush=True)
    gen = torch.Generator().manual_seed(8)
    for dtype, width in ((BF16, 50001), (FP32, 9000)):
        logits = (torch.randn((33, width), generator=gen) * 3).to(dtype).to(DEV)
        plan = run(logits, *settings(33, gen))
        live = torch.tensor([33], dtype=torch.int32, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            plan.launch(live)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.launch(live)
        for count in (33, 7, 0, 20, 33):
            plan.logits.copy_((torch.randn((33, width), generator=gen) * 3).to(dtype))
            for p, v in zip(plan.parameters, settings(33, gen)):
                p.copy_(v)
            live.fill_(count)
            for t, v in ((plan.tokens, -9), (plan.logprobs, 7.0)):
                t.fill_(v)
            plan.valid.fill_(False)
            graph.replay()
            torch.cuda.synchronize()
            check(plan, rows=count)
            assert (plan.tokens[count:] == -9).all() and (plan.logprobs[count:] == 7).all()
            replayed = plan.tokens.clone()
            plan.launch(count)  # eager work between the replays
            torch.cuda.synchronize()
            assert torch.equal(plan.tokens, replayed)


def test_agrees_with_the_candidate_sampler():
    """Same order, filters and draws as the root sampler over gathered
    candidates: all 20 logits of a row, its Philox number given back."""
    print("sample against the root sampler", flush=True)
    gen = torch.Generator().manual_seed(9)
    rows = 256
    logits = torch.randn((rows, 20), generator=gen).to(BF16).to(DEV)
    params = [torch.full((rows,), 0.8, device=DEV), torch.full((rows,), 0.9, device=DEV),
              torch.full((rows,), 12, dtype=torch.int64, device=DEV),
              torch.arange(rows, device=DEV) + 5, torch.zeros(rows, dtype=torch.int64, device=DEV)]
    out = [torch.empty(rows, dtype=torch.int64, device=DEV), torch.empty(rows, dtype=torch.bool, device=DEV)]
    ops = [logits[None].contiguous(), torch.arange(20, device=DEV).expand(1, rows, 20).contiguous(), *params, *out]
    sampling.RootTopKTopPSamplingPrimitive(*ops).launch(*ops)

    def philox(key, counter):  # first word for (ordinal, 0, 0, 0), key (seed, 0)
        c, k = [counter, 0, 0, 0], [key, 0]
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        x = c[0] - (1 << 32) if c[0] >> 31 else c[0]
        return np.float32(-x - 1 if x < 0 else x) * np.float32(4.6566127342e-10)

    u = torch.tensor([float(philox(s + 5, 0)) for s in range(rows)])
    plan = run(logits, 0.8, 12, 0.9, 0.0, u)
    check(plan)
    assert (plan.tokens != out[0]).sum() <= 1  # a draw next to a border may fall either way in binary32
