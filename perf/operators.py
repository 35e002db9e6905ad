"""Cases of the operators that serve many requests in one step: low-rank
adapters beside a shared projection, and sampling from the whole vocabulary.

``run`` computes them from elementary torch operations (``own`` false) or
through the package's entry points (``own`` true); both work on what
``prepare`` makes.  A case is a dict of plain values with a ``kind``:

  adapt   y = base + scale * B (A x) per row, A and B those of the row's
          request; ``ns`` lists the widths of the projections that share x
          (q, k, v or gate, up), ``rank`` the largest rank.  Request i owns
          adapter slot i % slots, every eighth request has none; with
          ``ragged`` the ranks of the slots are rank, rank/2, rank/4, ...
  sample  one token per row from logits over the whole vocabulary under
          temperature, top-k, top-p and min-p, from given uniform numbers.
          ``mode`` says which settings the rows carry.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed() -> list[dict]:
    return [
        # one sequence's decode step: q, k, v of a Qwen3-8B-shaped layer, latency only
        {"name": "adapt_qkv_m1", "kind": "adapt", "m": 1, "k": 4096, "ns": "4096,1024,1024",
         "requests": 1, "slots": 1, "rank": 16, "ragged": False, "dtype": "bf16"},
        # a decode batch in which every request has an adapter of its own
        {"name": "adapt_qkv_m64", "kind": "adapt", "m": 64, "k": 4096, "ns": "4096,1024,1024",
         "requests": 64, "slots": 64, "rank": 16, "ragged": False, "dtype": "bf16"},
        # a verify step, 64 sequences x (3 drafts + 1), some sharing an adapter, down projection
        {"name": "adapt_down_m256", "kind": "adapt", "m": 256, "k": 12288, "ns": "4096",
         "requests": 64, "slots": 16, "rank": 64, "ragged": True, "dtype": "bf16"},
        # a small layer of odd sizes, fp16
        {"name": "adapt_odd_m333_f16", "kind": "adapt", "m": 333, "k": 2056, "ns": "1001",
         "requests": 9, "slots": 5, "rank": 12, "ragged": True, "dtype": "fp16"},
        # a chunk of prompts, gate and up
        {"name": "adapt_gateup_m2048", "kind": "adapt", "m": 2048, "k": 4096, "ns": "12288,12288",
         "requests": 7, "slots": 4, "rank": 32, "ragged": False, "dtype": "bf16"},
        # a long chunk on a Llama-3-70B-shaped o projection, large ranks, fp16
        {"name": "adapt_o70b_m4096_f16", "kind": "adapt", "m": 4096, "k": 8192, "ns": "8192",
         "requests": 16, "slots": 8, "rank": 128, "ragged": True, "dtype": "fp16"},
        # one sequence, small vocabulary: latency only
        {"name": "sample_r1_v32768", "kind": "sample", "rows": 1, "vocab": 32768, "mode": "nucleus",
         "dtype": "bf16"},
        # a decode batch whose requests each bring their own settings
        {"name": "sample_r64_mixed", "kind": "sample", "rows": 64, "vocab": 151936, "mode": "mixed",
         "dtype": "bf16"},
        # the same over logits that a grammar has masked
        {"name": "sample_r64_masked", "kind": "sample", "rows": 64, "vocab": 151936, "mode": "masked",
         "dtype": "bf16"},
        # rollouts: plain sampling at temperature 1 from the whole distribution
        {"name": "sample_r256_open_f16", "kind": "sample", "rows": 256, "vocab": 151936, "mode": "open",
         "dtype": "fp16"},
        # logits that a processor left in 32 bits, odd width
        {"name": "sample_r48_v128001_f32", "kind": "sample", "rows": 48, "vocab": 128001, "mode": "mixed",
         "dtype": "fp32"},
    ]


def _log(rng, low: int, high: int, step: int = 1) -> int:
    """A multiple of ``step``, spread over the logarithm of [low, high]."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(value / step)) * step))


def draw(rng) -> dict:
    if rng.random() < 0.55:
        k = _log(rng, 512, 12288, 8)
        members = rng.choice((1, 1, 2, 3))
        # multiples of 8 as projections have, and any width
        ns = [_log(rng, 256, 12288, rng.choice((8, 8, 8, 1))) for _ in range(members)]
        # no dearer than the largest listed chunk
        most = max(1, min(8192, int(1.0e8 // (k + 2 * sum(ns)))))
        m = _log(rng, 1, most)
        requests = _log(rng, 1, min(m, 128))
        return {"kind": "adapt", "m": m, "k": k, "ns": ",".join(map(str, ns)), "requests": requests,
                "slots": _log(rng, 1, min(requests, 64)), "rank": _log(rng, 4, 128),
                "ragged": rng.random() < 0.5, "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    return {"kind": "sample", "rows": _log(rng, 1, 128 if dtype == "fp32" else 256),
            "vocab": _log(rng, 8000, 151936), "mode": rng.choice(("mixed", "nucleus", "masked", "open")),
            "dtype": dtype}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _device() -> torch.device:
    return torch.device("cuda:0")


def _widths(case: dict) -> list[int]:
    return [int(n) for n in case["ns"].split(",")]


def _rank(case: dict, slot: int) -> int:
    return max(1, case["rank"] >> (slot % 3)) if case["ragged"] else case["rank"]


def _requests(case: dict, seed: int) -> list[tuple[int, int, int]]:
    """(first row, end row, slot or -1) of every request: ragged lengths of at
    least one row that fill the batch."""
    m, q = case["m"], case["requests"]
    cuts = np.random.default_rng(seed).choice(m - 1, q - 1, replace=False) + 1 if q > 1 else []
    edges = [0, *sorted(int(c) for c in cuts), m]
    return [(edges[i], edges[i + 1], -1 if i % 8 == 7 else i % case["slots"]) for i in range(q)]


def _adapt_inputs(case: dict, seed: int) -> dict:
    """Activations N(0, 1), A as an initialised then trained adapter has it
    (entries near 1/sqrt(k)), B smaller, the shared projection's output N(0, 1)."""
    gen = torch.Generator(device=_device()).manual_seed(seed)
    dtype, m, k, slots = DTYPES[case["dtype"]], case["m"], case["k"], case["slots"]
    normal = lambda shape, std: (torch.randn(shape, generator=gen, device=_device()) * std).to(dtype)
    requests = _requests(case, seed)
    rows = torch.empty(m, dtype=torch.int32)
    for first, end, slot in requests:
        rows[first:end] = slot
    adapters = [[(normal((_rank(case, s), k), k ** -0.5), normal((n, _rank(case, s)), 0.05),
                  2.0 / (1 + s % 2)) for s in range(slots)] for n in _widths(case)]
    return {"requests": requests, "row_slots": rows.to(_device()), "x": normal((m, k), 1.0),
            "adapters": adapters, "bases": [normal((m, n), 1.0) for n in _widths(case)]}


def _sample_inputs(case: dict, seed: int) -> dict:
    """Logits N(0, 3); the settings that requests bring, by row."""
    gen = torch.Generator(device=_device()).manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.randn((rows, vocab), generator=gen, device=_device()) * 3
    if case["mode"] == "masked":  # a grammar admits about one token in fifty
        admitted = torch.rand((rows, vocab), generator=gen, device=_device()) < 0.02
        admitted[:, vocab // 2] = True
        logits.masked_fill_(~admitted, -math.inf)
    settings = {  # (temperature, top-k, top-p, min-p), row r takes entry r % len
        "nucleus": [(0.7, 0, 0.9, 0.0)],
        "open": [(1.0, 0, 1.0, 0.0)],
        "masked": [(0.7, 50, 0.95, 0.0), (1.0, 0, 1.0, 0.0)],
        "mixed": [(0.7, 20, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.05),
                  (0.6, 0, 0.95, 0.0), (1.3, 1000, 0.98, 0.01), (0.8, 50, 1.0, 0.0)],
    }[case["mode"]]
    chosen = [settings[r % len(settings)] for r in range(rows)]
    column = lambda i, dtype: torch.tensor([s[i] for s in chosen], dtype=dtype, device=_device())
    return {"logits": logits.to(DTYPES[case["dtype"]]), "temperatures": column(0, torch.float32),
            "top_ks": column(1, torch.int64), "top_ps": column(2, torch.float32),
            "min_ps": column(3, torch.float32),
            "uniforms": torch.rand(rows, generator=gen, device=_device())}


def prepare(case: dict, seed: int) -> dict:
    if case["kind"] == "sample":
        state = {"kind": "sample", **_sample_inputs(case, seed)}
        if own:
            from cubic_serve_amd import sampling

            state["plan"] = sampling.VocabSamplingPlan(
                logits=state["logits"], temperatures=state["temperatures"], top_ks=state["top_ks"],
                top_ps=state["top_ps"], min_ps=state["min_ps"], uniforms=state["uniforms"])
        return state
    state = {"kind": "adapt", **_adapt_inputs(case, seed)}
    if own:
        from cubic_serve_amd import adapters, linear

        banks = []
        for n, slots in zip(_widths(case), state["adapters"]):
            bank = adapters.AdapterBank(n, case["k"], slots=len(slots), max_rank=case["rank"],
                                        dtype=state["x"].dtype, device=_device())
            for slot, (down, up, scale) in enumerate(slots):
                bank.load(slot, down, up, scale)
            banks.append(bank)
        state["outputs"] = tuple(torch.empty_like(b) for b in state["bases"])
        state["binding"] = linear.PackedLinearOperators().bind_adapters(
            state["x"], banks, state["row_slots"], state["outputs"], bases=state["bases"])
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _adapt_plain(state: dict) -> tuple:
    outputs = []
    for base, slots in zip(state["bases"], state["adapters"]):
        y = base.clone()
        for first, end, slot in state["requests"]:
            if slot >= 0:
                down, up, scale = slots[slot]
                low = state["x"][first:end].float() @ down.float().t()
                delta = low @ up.float().t()
                y[first:end] = (base[first:end].float() + scale * delta).to(base.dtype)
        outputs.append(y)
    return tuple(outputs)


def _sample_plain(state: dict) -> tuple:
    logits = state["logits"].double()
    rows, vocab = logits.shape
    values, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    temperature = state["temperatures"].double()[:, None]
    greedy = temperature == 0
    z = (values - values[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature)
    weight = torch.exp(z)
    mass = torch.cumsum(weight, 1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    top_k = state["top_ks"][:, None]
    count = torch.where((top_k <= 0) | (top_k > vocab), vocab, top_k)
    total = torch.gather(mass, 1, count - 1)
    nucleus = (before < state["top_ps"].double()[:, None] * total).sum(1, keepdim=True)
    likely = (weight >= state["min_ps"].double()[:, None]).sum(1, keepdim=True)
    kept = torch.minimum(torch.minimum(count, nucleus), likely).clamp_(min=1)
    kept = torch.where(greedy, 1, kept)
    kept_mass = torch.gather(mass, 1, kept - 1)
    position = (mass <= state["uniforms"].double()[:, None] * kept_mass).sum(1, keepdim=True)
    position = torch.minimum(position, kept - 1)
    logprob = torch.log(torch.gather(weight, 1, position) / kept_mass)
    return (torch.gather(ids, 1, position)[:, 0], torch.isfinite(values[:, 0]), logprob[:, 0].float())


def run(state: dict):
    if state["kind"] == "sample":
        if not own:
            return _sample_plain(state)
        plan = state["plan"]
        plan.launch()
        return plan.tokens, plan.valid, plan.logprobs
    if not own:
        return _adapt_plain(state)
    state["binding"].launch()
    return state["outputs"]


def work(case: dict) -> dict:
    if case["kind"] == "sample":
        logits = case["rows"] * case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        # per row: four settings, the uniform number, the token, its validity and log-probability;
        # per logit: a subtraction, a scaling, an exponential, a sum
        return {"bytes": logits * size + case["rows"] * (24 + 13), "flops": 4 * logits}
    m, k, ns = case["m"], case["k"], _widths(case)
    slots = {i % case["slots"] for i in range(case["requests"]) if i % 8 != 7}
    ranks = sum(_rank(case, s) for s in slots)
    mean = ranks / max(1, len(slots))
    return {"bytes": 2 * (m * k + 2 * m * sum(ns)) + 4 * m + 2 * ranks * (len(ns) * k + sum(ns)),
            "flops": int(2 * m * mean * (len(ns) * k + sum(ns)))}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, on the host
# ---------------------------------------------------------------------------
def _adapt_exact(case: dict, seed: int) -> tuple:
    given = _adapt_inputs(case, seed)
    wide = lambda t: t.cpu().double().numpy()
    x, slot_of = wide(given["x"]), given["row_slots"].cpu().numpy()
    outputs = []
    for base, slots in zip(given["bases"], given["adapters"]):
        y = wide(base)
        for slot, (down, up, scale) in enumerate(slots):
            mine = np.flatnonzero(slot_of == slot)
            if mine.size:
                y[mine] += scale * ((x[mine] @ wide(down).T) @ wide(up).T)
        outputs.append(y)
    return tuple(outputs)


def _sample_exact(case: dict, seed: int) -> tuple:
    given = {name: t.cpu() for name, t in _sample_inputs(case, seed).items()}
    logits = given["logits"].double().numpy()
    temperatures, top_ps, min_ps, uniforms = (
        given[name].double().numpy() for name in ("temperatures", "top_ps", "min_ps", "uniforms"))
    tokens, valid, logprobs = [], [], []
    for r, row in enumerate(logits):
        best = row.max()
        if temperatures[r] == 0:
            tokens.append(int(np.flatnonzero(row == best)[0]))
            logprobs.append(0.0)
        else:
            chance = np.exp((row - best) / temperatures[r])
            order = np.argsort(-row, kind="stable")
            limit = int(given["top_ks"][r])
            if 0 < limit < len(order):
                order = order[:limit]
            ranked = np.cumsum(chance[order])
            keep = np.searchsorted(ranked, top_ps[r] * ranked[-1], side="left") + 1
            keep = min(keep, len(order), int((chance[order] >= min_ps[r]).sum()))
            where = min(int(np.searchsorted(ranked[:keep], uniforms[r] * ranked[keep - 1], side="right")),
                        keep - 1)
            tokens.append(int(order[where]))
            logprobs.append(math.log(chance[order[where]] / ranked[keep - 1]))
        valid.append(bool(np.isfinite(best)))
    return np.array(tokens), np.array(valid), np.array(logprobs)


def exact(case: dict, seed: int):
    return _sample_exact(case, seed) if case["kind"] == "sample" else _adapt_exact(case, seed)
