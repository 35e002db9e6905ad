"""Cases of the operators around block-scaled 8-bit products and in front of the
samplers: row norms and gated activations whose output is 8 bits with scales, the
products of such activations with block-scaled weights, and penalties, biases and
grammar masks on logits.

``run`` computes them from elementary torch operations (``own`` false) or
through the package's entry points (``own`` true); both work on what
``prepare`` makes.  A case is a dict of plain values with a ``kind``:

  norm    h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight per row;
          ``out`` is "8" (y in e4m3 with a scale for each 128 columns) or "16"
          (y in the inputs' type); with ``residual`` h is an output too
  gated   e4m3 and scales of silu(gate) * up (``gated``), or of up alone; both
          are halves of one matrix, as a grouped projection leaves them
  gemm    y = x w^T over e4m3 values, x with a scale for each row and 128
          columns, w with one for each 128 x 128; ``ns`` lists the widths of
          the projections that share x
  logits  repetition, presence and frequency penalties, biases and a grammar's
          mask on the logits of ``requests`` * (``depth`` + 1) rows: row (c, d) has
          the first d of request c's drafts behind its history
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128
TOP = 448.0           # the largest e4m3 value
SMALLEST = 2.0 ** -96  # a group's largest magnitude counts as at least this
EPSILON = 1e-6


def listed() -> list[dict]:
    return [
        # one sequence's decode step, the norm before q, k, v: latency only
        {"name": "norm_m1_k4096", "kind": "norm", "m": 1, "k": 4096, "out": "8", "residual": True, "dtype": "bf16"},
        # a ragged batch of a small model whose next product is not in 8 bits
        {"name": "norm_m333_k2056_f16", "kind": "norm", "m": 333, "k": 2056, "out": "16", "residual": True,
         "dtype": "fp16"},
        # a chunk of prompts of a Llama-3-70B-shaped model
        {"name": "norm_m4096_k8192", "kind": "norm", "m": 4096, "k": 8192, "out": "8", "residual": True,
         "dtype": "bf16"},
        # a verify step (64 rows) before a Qwen3-8B-shaped down projection
        {"name": "gated_m64_k12288", "kind": "gated", "m": 64, "k": 12288, "gated": True, "dtype": "bf16"},
        # attention's output before o, a ragged chunk of prompts, no gate
        {"name": "quantize_m1999_k4104_f16", "kind": "gated", "m": 1999, "k": 4104, "gated": False, "dtype": "fp16"},
        # q, k, v of one sequence: the weight stream
        {"name": "gemm_qkv_m1", "kind": "gemm", "m": 1, "k": 4096, "ns": "4096,1024,1024", "dtype": "bf16"},
        # the lm_head of a verify step
        {"name": "gemm_head_m64", "kind": "gemm", "m": 64, "k": 4096, "ns": "151936", "dtype": "bf16"},
        # a ragged batch on odd widths, fp16 outputs
        {"name": "gemm_odd_m333_f16", "kind": "gemm", "m": 333, "k": 2064, "ns": "1001,520", "dtype": "fp16"},
        # prompts on a Llama-3-70B-shaped o projection: the matrix cores
        {"name": "gemm_o70b_m4096", "kind": "gemm", "m": 4096, "k": 8192, "ns": "8192", "dtype": "bf16"},
        # one sequence, small vocabulary: latency only
        {"name": "logits_c1_v32768", "kind": "logits", "requests": 1, "depth": 0, "vocab": 32768, "prompt": 300,
         "output": 100, "masked": False, "dtype": "bf16"},
        # a verify step under a grammar, 64 sequences x (3 drafts + 1), long prompts
        {"name": "logits_c64_d3_masked", "kind": "logits", "requests": 64, "depth": 3, "vocab": 151936, "prompt": 8000,
         "output": 1500, "masked": True, "dtype": "bf16"},
        # 32-bit logits of an odd width
        {"name": "logits_c48_v128001_f32", "kind": "logits", "requests": 48, "depth": 0, "vocab": 128001, "prompt": 2000,
         "output": 600, "masked": False, "dtype": "fp32"},
    ]


def _log(rng, low: int, high: int, step: int = 1) -> int:
    """A multiple of ``step``, spread over the logarithm of [low, high]."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(value / step)) * step))


def draw(rng) -> dict:
    kind = rng.choice(("norm", "gated", "gemm", "gemm", "logits"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind in ("norm", "gated"):
        k = _log(rng, 64, 16384, rng.choice((8, 8, 8, 1)))
        m = _log(rng, 1, max(1, min(16384, (4096 * 8192) // k)))
        if kind == "norm":
            return {"kind": kind, "m": m, "k": k, "out": rng.choice(("8", "8", "16")),
                    "residual": rng.random() < 0.8, "dtype": dtype}
        return {"kind": kind, "m": m, "k": k, "gated": rng.random() < 0.7, "dtype": dtype}
    if kind == "gemm":
        k = _log(rng, 256, 12288, 16)
        # multiples of 8 as projections have, and any width
        ns = [_log(rng, 128, 16384, rng.choice((8, 8, 8, 1))) for _ in range(rng.choice((1, 1, 2, 3)))]
        # no dearer than the largest listed chunk
        most = max(1, min(4096, int(4096 * 8192 * 8192 // (k * sum(ns)))))
        return {"kind": kind, "m": _log(rng, 1, most), "k": k, "ns": ",".join(map(str, ns)), "dtype": dtype}
    depth = rng.choice((0, 0, 1, 3, 7))
    return {"kind": kind, "requests": _log(rng, 1, 256 // (depth + 1)), "depth": depth,
            "vocab": _log(rng, 8000, 151936), "prompt": _log(rng, 1, 8000), "output": _log(rng, 1, 1500),
            "masked": rng.random() < 0.5, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _device() -> torch.device:
    return torch.device("cuda:0")


def _blocks(size: int) -> int:
    return (size + BLOCK - 1) // BLOCK


def _widths(case: dict) -> list[int]:
    return [int(n) for n in case["ns"].split(",")]


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=_device()).manual_seed(seed)


def _norm_inputs(case: dict, seed: int) -> dict:
    """A layer's output N(0, 1) and the residual stream N(0, 2) with a few large
    channels; weights near one."""
    gen, dtype, (m, k) = _generator(seed), DTYPES[case["dtype"]], (case["m"], case["k"])
    normal = lambda *shape: torch.randn(shape, generator=gen, device=_device())
    channels = torch.where(torch.rand(k, generator=gen, device=_device()) < 0.01, 30.0, 2.0)
    return {"x": normal(m, k).to(dtype), "residual": (normal(m, k) * channels).to(dtype) if case["residual"] else None,
            "weight": (1 + 0.2 * normal(k)).to(dtype)}


def _gated_inputs(case: dict, seed: int) -> dict:
    """Gate and up as one grouped projection leaves them, N(0, 2)."""
    both = torch.randn((case["m"], 2 * case["k"]), generator=_generator(seed), device=_device()) * 2
    both = both.to(DTYPES[case["dtype"]])
    return {"gate": both[:, :case["k"]] if case["gated"] else None, "up": both[:, case["k"]:]}


def _quantized_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 values and scales for each 128 columns of 32-bit rows."""
    m, k = x.shape
    groups = torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k)).view(m, _blocks(k), BLOCK)
    most = groups.abs().amax(2).clamp_min(SMALLEST)
    values = (groups * (TOP / most)[:, :, None]).view(m, -1)[:, :k]
    return values.to(torch.float8_e4m3fn), most / TOP


def _quantized_blocks(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 values and scales for each 128 x 128 of a 32-bit matrix."""
    n, k = w.shape
    rows, columns = _blocks(n), _blocks(k)
    tiles = torch.nn.functional.pad(w, (0, columns * BLOCK - k, 0, rows * BLOCK - n))
    tiles = tiles.view(rows, BLOCK, columns, BLOCK)
    most = tiles.abs().amax((1, 3)).clamp_min(SMALLEST)
    values = (tiles * (TOP / most)[:, None, :, None]).view(rows * BLOCK, -1)[:n, :k]
    return values.to(torch.float8_e4m3fn).contiguous(), most / TOP


def _gemm_inputs(case: dict, seed: int) -> dict:
    """Activations N(0, 1) with a few large channels, weights N(0, 0.02), both
    as the quantiser leaves them."""
    gen, (m, k) = _generator(seed), (case["m"], case["k"])
    normal = lambda *shape: torch.randn(shape, generator=gen, device=_device())
    channels = torch.where(torch.rand(k, generator=gen, device=_device()) < 0.01, 20.0, 1.0)
    return {"x": _quantized_rows(normal(m, k) * channels),
            "weights": [_quantized_blocks(normal(n, k) * 0.02) for n in _widths(case)]}


def _logits_inputs(case: dict, seed: int) -> dict:
    """Logits N(0, 3); tokens as text has them, few often and many seldom; of
    every two requests one has biases; a grammar admits about one token in fifty."""
    gen, dev = _generator(seed), _device()
    requests, rows, vocab = case["requests"], case["requests"] * (case["depth"] + 1), case["vocab"]
    uniform = lambda *shape: torch.rand(shape, generator=gen, device=dev)

    def tokens(most: int) -> torch.Tensor:  # [requests, most], padded with -1
        drawn = (vocab * uniform(requests, most) ** 4).long().clamp_max(vocab - 1)
        lengths = 1 + (uniform(requests, 1) * most).long()
        return torch.where(torch.arange(most, device=dev) < lengths, drawn, -1)

    biases = torch.where(torch.arange(requests, device=dev)[:, None] % 2 == 0,
                         torch.randn((requests, 16), generator=gen, device=dev) * 4, 0.0)
    settings = [(1.1, 0.0, 0.0), (1.0, 0.5, 0.3), (1.05, 0.2, 0.1), (1.3, 0.0, 0.0), (1.0, 0.0, 0.0)]
    column = lambda i: torch.tensor([settings[r % 5][i] for r in range(requests)], device=dev)
    given = {"logits": (torch.randn((rows, vocab), generator=gen, device=dev) * 3).to(DTYPES[case["dtype"]]),
             "prompts": tokens(case["prompt"]), "outputs": tokens(case["output"]),
             # places of their own in the vocabulary, so that no token is named twice
             "bias_tokens": (torch.arange(16, device=dev) * (vocab // 16)).repeat(requests, 1)
             + (uniform(requests, 16) * (vocab // 16)).long(), "biases": biases,
             "repetition": column(0), "presence": column(1), "frequency": column(2),
             "drafts": (vocab * uniform(case["depth"], requests) ** 4).long().clamp_max(vocab - 1), "mask": None}
    if case["masked"]:
        bits = uniform(rows, _blocks(vocab) * BLOCK) < 0.02
        shifted = bits.view(rows, -1, 32).long() << torch.arange(32, device=dev)
        words = shifted.sum(2)[:, :(vocab + 31) // 32]
        given["mask"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int().contiguous()
    return given


def _prepare_norm(case: dict, seed: int) -> dict:
    state = _norm_inputs(case, seed)
    state["eight"] = case["out"] == "8"
    if own:
        from cubic_serve_amd import blockscale, linear

        x = state["x"]
        state["quantized"] = blockscale.BlockScaledActivations.empty(*x.shape, device=x.device) if state["eight"] else None
        state["output"] = None if state["eight"] else torch.empty_like(x)
        state["stream"] = torch.empty_like(x) if case["residual"] else None
        state["binding"] = linear.PackedLinearOperators().bind_norm(
            x, state["weight"], epsilon=EPSILON, residual=state["residual"], residual_output=state["stream"],
            output=state["output"], quantized=state["quantized"])
    return state


def _prepare_gated(case: dict, seed: int) -> dict:
    state = _gated_inputs(case, seed)
    if own:
        from cubic_serve_amd import blockscale, linear

        up = state["up"]
        state["quantized"] = blockscale.BlockScaledActivations.empty(*up.shape, device=up.device)
        state["binding"] = linear.PackedLinearOperators().bind_quantize(up, state["quantized"], gate=state["gate"])
    return state


def _prepare_gemm(case: dict, seed: int) -> dict:
    state = _gemm_inputs(case, seed)
    state["dtype"] = DTYPES[case["dtype"]]
    if own:
        from cubic_serve_amd import blockscale, linear

        values, scales = state["x"]
        x = blockscale.BlockScaledActivations(values, scales)
        weights = [blockscale.BlockScaledMatrix(*w) for w in state["weights"]]
        state["y"] = [torch.empty((case["m"], n), dtype=state["dtype"], device=values.device) for n in _widths(case)]
        state["binding"] = linear.PackedLinearOperators().bind_block_linear_group(x, weights, state["y"])
    return state


def _prepare_logits(case: dict, seed: int) -> dict:
    given = _logits_inputs(case, seed)
    logits, requests, vocab = given["logits"], case["requests"], case["vocab"]
    state = {name: given[name] for name in ("logits", "repetition", "presence", "frequency", "drafts", "mask")}
    if own:
        from cubic_serve_amd import penalties

        history = penalties.TokenHistory(requests, vocab, device=logits.device)
        slots = torch.arange(requests, dtype=torch.int32, device=logits.device)
        history.append_prompt(slots, given["prompts"])
        history.append(slots, given["outputs"])
        for slot in range(0, requests, 2):
            history.set_bias(slot, given["bias_tokens"][slot], given["biases"][slot])
        state["plan"] = penalties.LogitPenaltyPlan(
            logits=logits, history=history, slots=slots, repetition=state["repetition"],
            presence=state["presence"], frequency=state["frequency"],
            draft_tokens=state["drafts"] if case["depth"] else None, token_mask=state["mask"],
            outputs=torch.empty_like(logits))
        return state
    # what a program without such a history keeps: a table of counts, which tokens
    # a prompt has, and a table of biases
    def table(tokens: torch.Tensor) -> torch.Tensor:
        counts = torch.zeros((requests, vocab + 1), dtype=torch.int32, device=logits.device)
        ones = torch.ones_like(tokens, dtype=torch.int32)
        return counts.scatter_add_(1, torch.where(tokens < 0, vocab, tokens), ones)[:, :vocab].contiguous()

    state["counts"], state["prompted"] = table(given["outputs"]), table(given["prompts"]) > 0
    state["bias"] = torch.zeros((requests, vocab), device=logits.device).scatter_(1, given["bias_tokens"], given["biases"])
    return state


def prepare(case: dict, seed: int) -> dict:
    make = {"norm": _prepare_norm, "gated": _prepare_gated, "gemm": _prepare_gemm, "logits": _prepare_logits}
    return {"kind": case["kind"], **make[case["kind"]](case, seed)}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _norm_plain(state: dict) -> tuple:
    h = state["x"].float()
    if state["residual"] is not None:
        h = h + state["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPSILON) * state["weight"].float()
    y = _quantized_rows(y) if state["eight"] else (y.to(state["x"].dtype),)
    return y if state["residual"] is None else (*y, h.to(state["x"].dtype))


def _gated_plain(state: dict) -> tuple:
    y = state["up"].float()
    if state["gate"] is not None:
        gate = state["gate"].float()
        y = gate * torch.sigmoid(gate) * y
    return _quantized_rows(y)


def _gemm_plain(state: dict) -> tuple:
    spread = lambda s, rows, columns: s.repeat_interleave(BLOCK, 1)[:, :columns][:rows]
    values, scales = state["x"]
    m, k = values.shape
    x = values.float() * spread(scales, m, k)

    def product(weight: tuple) -> torch.Tensor:
        w, s = weight
        n = w.shape[0]
        return (x @ (w.float() * spread(s.repeat_interleave(BLOCK, 0), n, k)).t()).to(state["dtype"])

    return tuple(map(product, state["weights"]))


def _logits_plain(state: dict) -> torch.Tensor:
    logits, (depth, requests) = state["logits"], state["drafts"].shape
    vocab = logits.shape[1]
    value = logits.float().view(requests, depth + 1, vocab)
    counts = state["counts"][:, None].expand(requests, depth + 1, vocab)
    if depth:  # row d has the first d drafts behind it
        ahead = torch.arange(depth + 1, device=logits.device)[:, None] > torch.arange(depth, device=logits.device)
        drafts = state["drafts"].t()[:, None].expand(requests, depth + 1, depth)
        counts = counts.scatter_add(2, drafts, ahead.int()[None].expand(requests, depth + 1, depth))
    given = counts > 0
    setting = lambda name: state[name][:, None, None]
    repeated = torch.where(value > 0, value / setting("repetition"), value * setting("repetition"))
    value = torch.where(given | state["prompted"][:, None], repeated, value)
    value = value - setting("frequency") * counts - setting("presence") * given.float()
    value = (value + state["bias"][:, None]).view(-1, vocab)
    if state["mask"] is not None:
        column = torch.arange(vocab, device=logits.device)
        admitted = (state["mask"][:, column >> 5] >> (column & 31)) & 1
        value = torch.where(admitted != 0, value, -math.inf)
    return value.to(logits.dtype)


def run(state: dict):
    kind = state["kind"]
    if not own:
        plain = {"norm": _norm_plain, "gated": _gated_plain, "gemm": _gemm_plain, "logits": _logits_plain}
        return plain[kind](state)
    if kind == "logits":
        state["plan"].launch()
        return state["plan"].outputs
    state["binding"].launch()
    if kind == "gemm":
        return tuple(state["y"])
    if kind == "norm" and not state["eight"]:
        outputs = (state["output"],)
    else:
        outputs = (state["quantized"].values, state["quantized"].scales)
    return (*outputs, state["stream"]) if state.get("stream") is not None else outputs


def work(case: dict) -> dict:
    if case["kind"] == "logits":
        requests, rows, vocab = case["requests"], case["requests"] * (case["depth"] + 1), case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        mask = rows * ((vocab + 31) // 32) * 4 if case["masked"] else 0
        # the mean history's tokens and counts, once per request; five operations on each of its tokens
        history = requests * (case["prompt"] + case["output"]) // 2
        return {"bytes": 2 * rows * vocab * size + mask + 8 * history, "flops": 5 * history * (case["depth"] + 1)}
    m, k = case["m"], case["k"]
    scales = 4 * m * _blocks(k)
    if case["kind"] == "gemm":
        n = sum(_widths(case))
        blocks = sum(_blocks(w) for w in _widths(case)) * _blocks(k)
        return {"bytes": m * k + scales + n * k + 4 * blocks + 2 * m * n, "flops": 2 * m * n * k}
    out = m * k + scales
    if case["kind"] == "gated":
        return {"bytes": m * k * (4 if case["gated"] else 2) + out, "flops": m * k * (8 if case["gated"] else 3)}
    if case["out"] == "16":
        out = 2 * m * k
    return {"bytes": m * k * (6 if case["residual"] else 2) + 2 * k + out, "flops": 8 * m * k}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _wide(t: torch.Tensor) -> np.ndarray:
    return t.cpu().double().numpy()


def _exact_scaled(y: np.ndarray) -> tuple:
    """What e4m3 values stand for before their rounding, and the scales."""
    starts = np.arange(0, y.shape[1], BLOCK)
    most = np.maximum(np.maximum.reduceat(np.abs(y), starts, axis=1), SMALLEST)
    return y * TOP / np.repeat(most, BLOCK, axis=1)[:, :y.shape[1]], most / TOP


def _norm_exact(case: dict, seed: int) -> tuple:
    given = _norm_inputs(case, seed)
    h = _wide(given["x"])
    if given["residual"] is not None:
        h = h + _wide(given["residual"])
    y = h / np.sqrt(np.mean(np.square(h), axis=1, keepdims=True) + EPSILON) * _wide(given["weight"])
    y = _exact_scaled(y) if case["out"] == "8" else (y,)
    return y if given["residual"] is None else (*y, h)


def _gated_exact(case: dict, seed: int) -> tuple:
    given = _gated_inputs(case, seed)
    y = _wide(given["up"])
    if given["gate"] is not None:
        gate = _wide(given["gate"])
        y = gate / (1 + np.exp(-gate)) * y
    return _exact_scaled(y)


def _gemm_exact(case: dict, seed: int) -> tuple:
    """Block by block of K, each block's product under its scales, in 64 bits."""
    given = _gemm_inputs(case, seed)
    (xv, xs), k = given["x"], case["k"]
    outputs = []
    for wv, ws in given["weights"]:
        n = wv.shape[0]
        y = torch.zeros((case["m"], n), dtype=torch.float64, device=xv.device)
        for b in range(_blocks(k)):
            part = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            rows = ws[:, b].double().repeat_interleave(BLOCK)[:n]
            y += (xv[:, part].double() @ wv[:, part].double().t()) * xs[:, b, None].double() * rows
        outputs.append(y.cpu().numpy())
    return tuple(outputs)


def _logits_exact(case: dict, seed: int) -> np.ndarray:
    given = _logits_inputs(case, seed)
    value, depth, vocab = _wide(given["logits"]), case["depth"], case["vocab"]
    host = {name: given[name].cpu().numpy() for name in ("prompts", "outputs", "drafts", "bias_tokens")}
    setting = {name: _wide(given[name]) for name in ("repetition", "presence", "frequency", "biases")}
    words = None if given["mask"] is None else given["mask"].cpu().numpy().view(np.uint8)
    for r, row in enumerate(value):
        c, d = divmod(r, depth + 1)
        said = host["outputs"][c]
        counts = np.bincount(np.concatenate([said[said >= 0], host["drafts"][:d, c]]), minlength=vocab)
        seen = counts > 0
        seen[host["prompts"][c][host["prompts"][c] >= 0]] = True
        repetition = setting["repetition"][c]
        row[seen] *= np.where(row[seen] > 0, 1 / repetition, repetition)
        row -= setting["frequency"][c] * counts + setting["presence"][c] * (counts > 0)
        row[host["bias_tokens"][c]] += setting["biases"][c]
        if words is not None:
            row[np.unpackbits(words[r], bitorder="little")[:vocab] == 0] = -np.inf
    return value


def exact(case: dict, seed: int):
    make = {"norm": _norm_exact, "gated": _gated_exact, "gemm": _gemm_exact, "logits": _logits_exact}
    return make[case["kind"]](case, seed)
