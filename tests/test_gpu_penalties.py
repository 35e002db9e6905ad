"""GPU: token histories, and penalties, biases and masks on logits against their
formulas in 64 bits.

Tolerance: at most four roundings in 32 bits, each 2^-24 of at most |l| (r + 1 / r) +
|f| c + |p| + |b| with r the repetition, and half a step of the output's type.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from cubic_serve_amd import blockscale, linear, penalties, sampling

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}
LEAST = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -150}


class Model:
    """A history restated on the host."""

    def __init__(self, slots, vocab):
        self.counts, self.prompt = np.zeros((slots, vocab), np.int64), np.zeros((slots, vocab), bool)
        self.bias, self.slots, self.vocab = np.zeros((slots, vocab)), slots, vocab

    def take(self, row_slots, tokens, prompt, live=None):
        tokens = tokens[:, None] if tokens.ndim == 1 else tokens
        for slot, row in list(zip(row_slots.tolist(), tokens.tolist()))[:live]:
            for t in row:
                if 0 <= slot < self.slots and 0 <= t < self.vocab:
                    if prompt:
                        self.prompt[slot, t] = True
                    else:
                        self.counts[slot, t] += 1

    def apply(self, logits, slots, settings, drafts=None, mask=None, width=None):
        """(values in 64 bits, bound without the output's rounding)."""
        value = logits.detach().cpu().double().numpy().copy()
        bound = np.zeros_like(value)
        depth = 0 if drafts is None else drafts.shape[0]
        width = value.shape[1] if width is None else width
        for r in range(value.shape[0]):
            c, d = divmod(r, depth + 1)
            slot, (rep, pres, freq) = int(slots[c]), (float(s[c]) if s is not None else None for s in settings)
            rep, pres, freq = 1.0 if rep is None else rep, pres or 0.0, freq or 0.0
            row = value[r, :width]
            if not (0 < rep < math.inf and math.isfinite(pres) and math.isfinite(freq)):
                row[:] = np.nan
                continue
            if 0 <= slot < self.slots:
                counts = self.counts[slot, :width].copy()
                for t in [] if drafts is None else drafts[:d, c].tolist():
                    if 0 <= t < width:
                        counts[t] += 1
                seen = self.prompt[slot, :width] | (counts > 0)
                with np.errstate(invalid="ignore"):
                    bound[r, :width] = 4 * 2.0 ** -24 * (np.abs(row) * (rep + 1 / rep) + abs(freq) * counts + abs(pres)
                                                         + np.abs(self.bias[slot, :width]))
                    row[:] = np.where(seen, np.where(row > 0, row / rep, row * rep), row)
                    row -= np.where(counts > 0, freq * counts + pres, 0)
                    row += self.bias[slot, :width]
            if mask is not None:
                bits = np.unpackbits(mask[r].cpu().numpy().view(np.uint8), bitorder="little")[:width]
                row[bits == 0] = -np.inf
        return value, bound


def compare(got, want, bound):
    dtype, got = got.dtype, got.detach().cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    fine = np.isfinite(want)
    limit = np.abs(want[fine]) * HALF_STEP[dtype] + bound[fine] * (1 + HALF_STEP[dtype]) + LEAST[dtype]
    off = np.abs(got[fine] - want[fine])
    assert (off <= limit).all(), (off / limit).max()


def make(slots, vocab, seed, prompt=60, output=40):
    """A history and its model, tokens drawn with repeats."""
    gen = torch.Generator().manual_seed(seed)
    h, m = penalties.TokenHistory(slots, vocab, DEV), Model(slots, vocab)
    for length, is_prompt in ((prompt, True), (output, False)):
        tokens = (vocab * torch.rand((slots, length), generator=gen) ** 3).long()
        tokens[:, length // 2:] = torch.where(torch.rand((slots, length - length // 2), generator=gen) < 0.2, -1, tokens[:, length // 2:])
        order = torch.randperm(slots, generator=gen).int()
        (h.append_prompt if is_prompt else h.append)(order.to(DEV), tokens.to(DEV))
        m.take(order, tokens, is_prompt)
    for slot in range(0, slots, 2):
        ids = torch.randperm(vocab, generator=gen)[:5].tolist()
        values = [-math.inf, 3.5, -2.0, 0.25, 100.0][:len(ids)]
        h.set_bias(slot, ids, values)
        m.bias[slot, ids] = values
    return h, m, gen


def draw_settings(n, gen):
    return (0.7 + torch.rand(n, generator=gen), torch.randn(n, generator=gen), torch.randn(n, generator=gen) * 0.5)


def draw_mask(rows, width, gen, share=0.5):
    bits = (torch.rand((rows, (width + 31) // 32 * 32), generator=gen) < share).numpy()
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy()).to(DEV)


@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (FP16, FP16), (FP32, FP32), (BF16, FP32), (FP16, FP32)])
@pytest.mark.parametrize("sequences,depth,vocab", [(1, 0, 1), (2, 0, 7), (3, 1, 33), (5, 0, 1000), (4, 3, 8192), (2, 8, 8193), (7, 2, 20011)])
def test_penalties(sequences, depth, vocab, dtype, out):
    print(f"penalties sequences={sequences} depth={depth} vocab={vocab} {dtype} {out}", flush=True)
    h, m, gen = make(sequences + 2, vocab, 1)
    rows = sequences * (depth + 1)
    whole = (torch.randn((rows, vocab + 3), generator=gen) * 4).to(dtype).to(DEV)
    logits = whole[:, :vocab]  # rows at any alignment
    slots = torch.randperm(sequences + 2, generator=gen)[:sequences].int()
    settings = draw_settings(sequences, gen)
    drafts = (vocab * torch.rand((depth, sequences), generator=gen) ** 3).long() if depth else None
    if depth > 1:
        drafts[1] = drafts[0]  # the same draft twice
        drafts[0, 0] = -1
    mask = draw_mask(rows, vocab, gen) if sequences % 2 == 0 else None
    want = m.apply(logits, slots, settings, drafts, mask)
    result = torch.full((rows, vocab + 5), 7.0, dtype=out, device=DEV)
    plan = penalties.LogitPenaltyPlan(
        logits=logits, history=h, slots=slots.to(DEV), repetition=settings[0].to(DEV), presence=settings[1].to(DEV),
        frequency=settings[2].to(DEV), draft_tokens=None if drafts is None else drafts.to(DEV), token_mask=mask,
        outputs=result[:, :vocab])
    plan.launch()
    compare(result[:, :vocab], *want)
    assert (result[:, vocab:] == 7).all()
    if out is dtype:  # the same, in place
        after = whole.clone()
        plan = penalties.LogitPenaltyPlan(
            logits=after[:, :vocab], history=h, slots=slots.to(DEV), repetition=settings[0].to(DEV),
            presence=settings[1].to(DEV), frequency=settings[2].to(DEV),
            draft_tokens=None if drafts is None else drafts.to(DEV), token_mask=mask)
        plan.launch()
        assert plan.outputs is plan.logits
        assert torch.equal(after[:, :vocab].nan_to_num(9), result[:, :vocab].nan_to_num(9))
        assert torch.equal(after[:, vocab:], whole[:, vocab:])


def test_long_histories():
    """Lists longer than a chunk's columns, up to every token."""
    vocab, sequences = 30000, 3
    h, m = penalties.TokenHistory(sequences, vocab, DEV), Model(sequences, vocab)
    gen = torch.Generator().manual_seed(2)
    tokens = torch.stack([torch.randperm(vocab, generator=gen), torch.randint(0, vocab, (vocab,), generator=gen),
                          torch.full((vocab,), 5)])
    slots = torch.arange(sequences, dtype=torch.int32)
    h.append(slots.to(DEV), tokens.to(DEV))
    m.take(slots, tokens, False)
    assert h.sizes.sum(1).tolist()[::2] == [vocab, 1] and h.counts(2)[5].item() == vocab
    for s in range(sequences):
        assert np.array_equal(h.counts(s).cpu().numpy(), m.counts[s])
    logits = (torch.randn((2 * sequences, vocab), generator=gen) * 4).to(BF16).to(DEV)
    settings = draw_settings(sequences, gen)
    drafts = torch.tensor([[0, 29999, 6]])
    want = m.apply(logits, slots, settings, drafts)
    args = dict(history=h, slots=slots.to(DEV), repetition=settings[0].to(DEV), presence=settings[1].to(DEV),
                frequency=settings[2].to(DEV), draft_tokens=drafts.to(DEV))
    plan = penalties.LogitPenaltyPlan(logits=logits, outputs=torch.empty_like(logits), **args)
    plan.launch()
    compare(plan.outputs, *want)
    penalties.LogitPenaltyPlan(logits=logits, **args).launch()
    assert torch.equal(logits, plan.outputs)


@pytest.mark.parametrize("inplace", [False, True])
def test_settings_slots_and_masks_at_the_edges(inplace):
    vocab, sequences = 10000, 12
    h, m, gen = make(8, vocab, 3)
    logits = (torch.randn((sequences, vocab), generator=gen) * 4).to(FP32).to(DEV)
    logits[0, :50], logits[1, 7], logits[2, 3] = -math.inf, math.inf, math.nan
    slots = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, -1, 8, 1 << 20, 0], dtype=torch.int32)  # one slot twice, three outside
    rep, pres, freq = torch.full((sequences,), 1.2), torch.zeros(sequences), torch.zeros(sequences)
    rep[3], rep[4], rep[5], pres[6], freq[7] = 0.0, -1.0, math.nan, math.inf, math.nan  # refused
    mask = draw_mask(sequences, vocab, gen)
    mask[0], mask[1], mask[9] = -1, 0, 0  # everything, nothing
    before = logits.clone()
    want = m.apply(logits, slots, (rep, pres, freq), None, mask)
    plan = penalties.LogitPenaltyPlan(logits=logits, history=h, slots=slots.to(DEV), repetition=rep.to(DEV),
                                      presence=pres.to(DEV), frequency=freq.to(DEV), token_mask=mask,
                                      outputs=None if inplace else torch.empty_like(logits))
    plan.launch()
    compare(plan.outputs, *want)
    assert torch.isnan(plan.outputs[3:8]).all() and (plan.outputs[1] == -math.inf).all()
    if not inplace:
        assert torch.equal(logits.nan_to_num(9), before.nan_to_num(9))
    # no settings: biases and mask only
    plan = penalties.LogitPenaltyPlan(logits=before, history=h, slots=slots.to(DEV), outputs=torch.empty_like(before))
    plan.launch()
    compare(plan.outputs, *m.apply(before, slots, (None, None, None)))


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("live", [0, 1, 4, 5])
def test_rows_past_the_live_count_and_columns_past_the_width(live, inplace):
    vocab, sequences, depth = 9000, 5, 1
    h, m, gen = make(sequences, vocab + 100, 4)
    slots, settings = torch.arange(sequences, dtype=torch.int32), draw_settings(sequences, gen)
    drafts = torch.randint(0, vocab + 100, (depth, sequences), generator=gen)
    source = (torch.randn((2 * sequences, vocab + 50), generator=gen) * 4).to(BF16).to(DEV)
    want, bound = m.apply(source, slots, settings, drafts, None, vocab)
    for how in (live, torch.tensor([live, 99], dtype=torch.int32, device=DEV), torch.tensor([live - 7 if live == 0 else live], dtype=torch.int32, device=DEV)):
        logits = source.clone()
        out = None if inplace else torch.full_like(logits, 7.0)
        plan = penalties.LogitPenaltyPlan(logits=logits, history=h, slots=slots.to(DEV), repetition=settings[0].to(DEV),
                                          presence=settings[1].to(DEV), frequency=settings[2].to(DEV),
                                          draft_tokens=drafts.to(DEV), outputs=out, visible_width=vocab)
        plan.launch(how)
        got = plan.outputs
        compare(got[:2 * live, :vocab], want[:2 * live, :vocab], bound[:2 * live, :vocab])
        rest = source if inplace else torch.full_like(source, 7.0)
        assert torch.equal(got[2 * live:], rest[2 * live:]) and torch.equal(got[:, vocab:], rest[:, vocab:])


def test_history_appends_clears_and_biases():
    vocab, slots = 500, 6
    h, m, gen = make(slots, vocab, 5)
    rows = torch.tensor([2, 2, 0, -1, 6, 5], dtype=torch.int32)   # a slot twice, two outside
    tokens = torch.tensor([[1, 1, 2], [1, 3, -1], [500, 499, -5], [4, 4, 4], [4, 4, 4], [7, 1 << 40, 8]])
    h.append(rows.to(DEV), tokens.to(DEV))
    m.take(rows, tokens, False)
    h.append(rows.to(DEV), tokens[:, 0].int().to(DEV), live_rows=3)
    m.take(rows, tokens[:, 0], False, 3)
    h.append_prompt(rows.to(DEV), tokens[:, 1:].to(DEV), torch.tensor([2], dtype=torch.int32, device=DEV))  # rows at a stride
    m.take(rows, tokens[:, 1:], True, 2)
    h.set_bias(0, torch.tensor([9, 10], device=DEV), torch.tensor([1.5, -1.0]))
    m.bias[0] = 0
    m.bias[0, [9, 10]] = 1.5, -1.0
    h.set_bias(2, [], [])
    m.bias[2] = 0

    def check():
        marks = h.state[:, :, 0].contiguous().cpu().numpy().view(np.uint32)
        assert np.array_equal(marks & ((1 << 30) - 1), m.counts) and np.array_equal(marks >> 31 != 0, m.prompt)
        for s in range(slots):  # every token that has anything is listed, once
            assert np.array_equal(h.biases(s).cpu().numpy(), m.bias[s].astype(np.float32))
            listed = [t for b, n in enumerate(h.sizes[s].tolist()) for t in h.listed[s, 4096 * b:4096 * b + n].tolist()]
            assert len(set(listed)) == len(listed)
            assert set(np.flatnonzero((m.counts[s] > 0) | m.prompt[s] | (m.bias[s] != 0))) <= set(listed)
            assert np.array_equal(np.flatnonzero(marks[s] >> 30 & 1), np.sort(listed))

    check()
    h.clear(torch.tensor([1, 1, -1, 3, 9], dtype=torch.int32, device=DEV))
    h.clear(5)
    for s in (1, 3, 5):
        m.counts[s], m.prompt[s], m.bias[s] = 0, False, 0
    check()
    assert not h.sizes[1::2].any()
    h.append(torch.tensor([1], dtype=torch.int32, device=DEV), torch.tensor([[3, 3]], device=DEV))
    m.take(torch.tensor([1]), torch.tensor([[3, 3]]), False)
    check()


def test_captured_step_follows_its_operands():
    """Penalties and the emitted tokens' append in one graph, replayed over changing logits."""
    vocab, sequences, depth = 12000, 6, 1
    h, m, gen = make(sequences, vocab, 6)
    slots, settings = torch.arange(sequences, dtype=torch.int32), draw_settings(sequences, gen)
    logits = torch.empty((2 * sequences, vocab), dtype=BF16, device=DEV)
    drafts = torch.zeros((depth, sequences), dtype=torch.int64, device=DEV)
    emitted = torch.full((sequences, 2), -1, dtype=torch.int64, device=DEV)
    mask = torch.full((2 * sequences, vocab // 32), -1, dtype=torch.int32, device=DEV)
    plan = penalties.LogitPenaltyPlan(logits=logits, history=h, slots=slots.to(DEV), repetition=settings[0].to(DEV),
                                      presence=settings[1].to(DEV), frequency=settings[2].to(DEV), draft_tokens=drafts,
                                      token_mask=mask, outputs=torch.empty_like(logits))
    on_device = slots.to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.launch()
        h.append(on_device, emitted)
    assert np.array_equal(h.counts(0).cpu().numpy(), m.counts[0])  # nothing ran yet
    for turn in range(4):
        logits.copy_((torch.randn((2 * sequences, vocab), generator=gen) * 4).to(BF16))
        drafts.copy_(torch.randint(0, 50, (depth, sequences), generator=gen))
        emitted.copy_(torch.randint(-1, 50, (sequences, 2), generator=gen))
        mask.copy_(draw_mask(2 * sequences, vocab, gen))
        torch.cuda.synchronize()
        want = m.apply(logits, slots, settings, drafts.cpu(), mask)
        graph.replay()
        torch.cuda.synchronize()
        compare(plan.outputs, *want)
        m.take(slots, emitted.cpu(), False)
        for s in range(sequences):
            assert np.array_equal(h.counts(s).cpu().numpy(), m.counts[s])


def test_rows_that_lie_far_apart():
    """Logits rows past 2^31 elements, a history past 2^31 entries."""
    vocab, slots = 1 << 21, 1100
    h, m = penalties.TokenHistory(slots, vocab, DEV), Model(1, vocab)
    tokens = torch.tensor([[0, 5, 5, vocab - 1]])
    last = torch.tensor([slots - 1], dtype=torch.int32)
    h.append(last.to(DEV), tokens.to(DEV))
    h.set_bias(slots - 1, [vocab - 2], [2.0])
    m.take(torch.tensor([0]), tokens, False)
    m.bias[0, vocab - 2] = 2.0
    stride = (1 << 31) + 64
    whole = torch.empty(stride + 100, dtype=BF16, device=DEV)
    logits = whole.as_strided((2, 100), (stride, 1))
    logits.copy_((torch.randn((2, 100), generator=torch.Generator().manual_seed(7)) * 4).to(BF16))
    settings = torch.tensor([1.5]), torch.tensor([0.5]), torch.tensor([0.25])
    drafts = torch.tensor([[7]])
    want = m.apply(logits, torch.tensor([0]), settings, drafts)
    out = torch.empty((2, 100), dtype=FP32, device=DEV)
    penalties.LogitPenaltyPlan(logits=logits, history=h, slots=last.to(DEV), repetition=settings[0].to(DEV),
                               presence=settings[1].to(DEV), frequency=settings[2].to(DEV), draft_tokens=drafts.to(DEV),
                               outputs=out).launch()
    compare(out, *want)
    assert h.counts(slots - 1)[vocab - 1].item() == 1
    h.clear(slots - 1)
    assert not h.state[slots - 1].any() and not h.sizes.any()


def test_head_penalties_sampling_chain():
    """norm -> block-scaled lm_head -> penalties -> vocabulary sampling -> history, three steps."""
    m, hidden, vocab = 5, 256, 4000
    gen = torch.Generator(device=DEV).manual_seed(8)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    weight, head = (1 + 0.1 * normal(hidden)).to(BF16), blockscale.quantize_block_scaled(normal(vocab, hidden) * 0.2)
    x, logits = normal(m, hidden).to(BF16), torch.empty((m, vocab), dtype=BF16, device=DEV)
    ops, q = linear.PackedLinearOperators(), blockscale.BlockScaledActivations.empty(m, hidden, DEV)
    h, slots = penalties.TokenHistory(m, vocab, DEV), torch.arange(m, dtype=torch.int32, device=DEV)
    full = lambda v, dtype=FP32: torch.full((m,), v, dtype=dtype, device=DEV)
    plan = penalties.LogitPenaltyPlan(logits=logits, history=h, slots=slots, frequency=full(100.0),
                                      outputs=torch.empty((m, vocab), device=DEV))
    sample = sampling.VocabSamplingPlan(logits=plan.outputs, temperatures=full(0.0), top_ks=full(0, torch.int64),
                                        top_ps=full(1.0), min_ps=full(0.0), uniforms=full(0.5))
    bindings = (ops.bind_norm(x, weight, epsilon=1e-6, quantized=q), ops.bind_block_linear(q, head, logits))
    taken = []
    for step in range(3):
        for binding in bindings:
            binding.launch()
        plan.launch()
        sample.launch()
        h.append(slots, sample.tokens)
        torch.cuda.synchronize()
        left = logits.clone()
        for t in taken:  # the largest of those not taken yet
            left[torch.arange(m), t] = -math.inf
        assert sample.valid.all()
        assert torch.equal(left[torch.arange(m), sample.tokens], left.amax(1))
        taken.append(sample.tokens.clone())


def test_verify_step_with_penalties():
    """Draft positions see the drafts before them: MTPVerifyPlan over penalised logits accepts
    what the penalised argmax says, and its emitted tokens go into the history."""
    c, depth, vocab = 4, 2, 3000
    gen = torch.Generator().manual_seed(9)
    h, m = penalties.TokenHistory(c, vocab, DEV), Model(c, vocab)
    slots = torch.arange(c, dtype=torch.int32)
    logits = (torch.randn((c * (depth + 1), vocab), generator=gen) * 3).to(BF16)
    top = logits.float().argmax(1).view(c, depth + 1)
    drafts = torch.stack([top[:, 0], top[:, 0]])           # the second draft repeats the first ...
    logits.view(c, depth + 1, vocab)[torch.arange(c), 1, top[:, 0]] = 50.0  # ... which is row 1's largest logit
    frequency = torch.tensor([0.0, 100.0, 0.0, 100.0])     # and stays so where it is not penalised
    params = dict(history=h, slots=slots.to(DEV), frequency=frequency.to(DEV), draft_tokens=drafts.to(DEV))
    plan = penalties.LogitPenaltyPlan(logits=logits.to(DEV), outputs=torch.empty(logits.shape, dtype=BF16, device=DEV), **params)
    q_scores = torch.full((depth, c, 20), float("nan"), dtype=BF16)
    q_ids = torch.full((depth, c, 20), -1, dtype=torch.int64)
    q_scores[:, :, 0], q_ids[:, :, 0] = 1.0, drafts
    flat = lambda v, dtype: torch.full((depth, c), v, dtype=dtype, device=DEV)
    verify = sampling.MTPVerifyPlan(
        logits=plan.outputs, q_scores=q_scores.to(DEV), q_token_ids=q_ids.to(DEV), draft_tokens=drafts.to(DEV),
        temperatures=flat(0.0, FP32), top_ps=flat(1.0, FP32), top_ks=flat(20, torch.int64),
        seeds=flat(0, torch.int64), ordinals=flat(0, torch.int64))
    plan.launch()
    verify.launch()
    h.append(slots.to(DEV), verify.emitted)
    torch.cuda.synchronize()
    assert verify.merged[:, 0].tolist() == [2, 1, 2, 1]
    for s in range(c):
        assert h.counts(s).sum().item() == verify.merged[s, 0].item() + 1
        assert h.counts(s)[drafts[0, s]].item() == (2 if s % 2 == 0 else 1)


def test_a_plan_whose_history_was_given_other_memory():
    h = penalties.TokenHistory(2, 100, DEV)
    logits, slots = torch.zeros((2, 100), dtype=BF16, device=DEV), torch.arange(2, dtype=torch.int32, device=DEV)
    plan = penalties.LogitPenaltyPlan(logits=logits, history=h, slots=slots)
    plan.launch()
    h.state.data = h.state.clone()
    for refused in (plan.launch, lambda: plan.launch(1), lambda: h.append(slots, slots), lambda: h.set_bias(0, [1], [1.0]),
                    lambda: penalties.LogitPenaltyPlan(logits=logits, history=h, slots=slots)):
        with pytest.raises(ValueError, match="other memory|changed after binding"):
            refused()
    assert not logits.any()


def test_refusals():
    h = penalties.TokenHistory(3, 100, DEV)
    logits, slots = torch.zeros((3, 90), dtype=BF16, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    ok = dict(logits=logits, history=h, slots=slots)
    f = torch.ones(3, device=DEV)
    bad = [(dict(logits=logits.double()), "row-major"), (dict(logits=logits.cpu()), "CUDA"), (dict(logits=logits[:2]), "rows"),
           (dict(slots=slots.long()), "slots"), (dict(slots=slots.cpu()), "slots"), (dict(repetition=f.double()), "float32"),
           (dict(presence=f[:2]), "float32"), (dict(frequency=f.cpu()), "float32"), (dict(visible_width=0), "width"),
           (dict(visible_width=91), "width"), (dict(draft_tokens=torch.zeros((1, 2), dtype=torch.int64, device=DEV)), "draft"),
           (dict(draft_tokens=torch.zeros((9, 3), dtype=torch.int64, device=DEV)), "draft"),
           (dict(draft_tokens=torch.zeros((1, 3), dtype=torch.int64, device=DEV)), "rows"),
           (dict(token_mask=torch.zeros((3, 2), dtype=torch.int32, device=DEV)), "bitmask"),
           (dict(token_mask=torch.zeros((2, 3), dtype=torch.int32, device=DEV)), "bitmask"),
           (dict(outputs=torch.empty((3, 90), dtype=FP16, device=DEV)), "outputs"), (dict(outputs=logits), "alias"),
           (dict(outputs=torch.empty((3, 91), dtype=BF16, device=DEV)), "outputs"),
           (dict(logits=torch.zeros((3, 101), dtype=BF16, device=DEV)), "width")]
    for change, match in bad:
        with pytest.raises(ValueError, match=match):
            penalties.LogitPenaltyPlan(**(ok | change))
    with pytest.raises(TypeError):
        penalties.LogitPenaltyPlan(**(ok | dict(history=None)))
    plan = penalties.LogitPenaltyPlan(**ok)
    for live in (-1, 4, 1.0, torch.tensor([1], device=DEV), torch.tensor([1], dtype=torch.int32)):
        with pytest.raises(ValueError, match="live"):
            plan.launch(live)
    for tokens in (torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(3, device=DEV), torch.zeros(3, dtype=torch.int64),
                   torch.zeros((3, 0), dtype=torch.int64, device=DEV), torch.zeros((2, 3), dtype=torch.int64, device=DEV).t()):
        with pytest.raises(ValueError):
            h.append(slots, tokens)
    for args in ((3, [1], [1.0]), (0, [1, 1], [1.0, 2.0]), (0, [100], [1.0]), (0, [-1], [1.0]), (0, [1], [math.nan]),
                 (0, [1], [math.inf]), (0, [1], [1e39]), (0, [1, 2], [1.0])):
        with pytest.raises(ValueError):
            h.set_bias(*args)
    for slot in (-1, 3, 1.0, True):
        with pytest.raises(ValueError):
            h.clear(slot)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="before graph capture"):
            h.set_bias(0, [1], [1.0])
    logits.resize_((3, 80))
    with pytest.raises(ValueError, match="changed after binding"):
        plan.launch()


@pytest.mark.parametrize("name", ["logits", "slots", "frequency", "drafts", "mask", "outputs"])
def test_operands_with_another_layout_after_binding(name):
    """The same memory and number of elements, read another way."""
    n, vocab = 32, 64
    h = penalties.TokenHistory(n, vocab, DEV)
    t = dict(logits=torch.zeros((2 * n, vocab), dtype=BF16, device=DEV), slots=torch.arange(n, dtype=torch.int32, device=DEV),
             frequency=torch.ones(n, device=DEV), drafts=torch.zeros((1, n), dtype=torch.int64, device=DEV),
             mask=torch.full((2 * n, 2), -1, dtype=torch.int32, device=DEV), outputs=torch.zeros((2 * n, vocab), dtype=BF16, device=DEV))
    plan = penalties.LogitPenaltyPlan(logits=t["logits"], history=h, slots=t["slots"], frequency=t["frequency"],
                                      draft_tokens=t["drafts"], token_mask=t["mask"], outputs=t["outputs"])
    plan.launch()
    if t[name].ndim == 2:
        t[name].t_()
    else:
        t[name].data = t[name].view(FP32 if t[name].dtype is torch.int32 else torch.int32)
    for live in (None, 1):
        with pytest.raises(ValueError, match="changed after binding"):
            plan.launch(live)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_columns_that_no_list_names_beside_an_append(dtype):
    """Lists that grow while a launch reads them: which of the two comes first is open, token by token, but a workgroup goes
    one way as a whole, so the columns that nobody names keep their logits.  (Presence alone, each token appended once: a
    named column holds its logit or that minus 1, whole numbers.)"""
    vocab, sequences, length = 50000, 16, 8
    side = torch.cuda.Stream()
    gen = torch.Generator().manual_seed(11)
    slots = torch.arange(sequences, dtype=torch.int32, device=DEV)
    logits = torch.randint(-60, 60, (sequences, vocab), generator=gen).to(dtype).to(DEV)
    for turn in range(4):
        h = penalties.TokenHistory(sequences, vocab, DEV)
        plan = penalties.LogitPenaltyPlan(logits=logits, history=h, slots=slots, presence=torch.ones(sequences, device=DEV),
                                          outputs=torch.full_like(logits, 7.0))
        # (not token 0, which an unwritten place of a list names)
        named = torch.stack([1 + torch.randperm(vocab - 1, generator=gen)[:20 * length] for _ in range(sequences)]).to(DEV)
        steps = [named[:, i:i + length].contiguous() for i in range(0, 20 * length, length)]
        torch.cuda.synchronize()
        results = []
        for step in steps:
            with torch.cuda.stream(side):
                h.append(slots, step)
            plan.launch()
            results.append(plan.outputs.clone())
        torch.cuda.synchronize()
        given = torch.zeros((sequences, vocab), dtype=torch.bool, device=DEV).scatter_(1, named, True)
        for got in results:
            assert torch.equal(got[~given], logits[~given])
            assert ((got == logits) | (got == logits - 1))[given].all()
        plan.launch()
        assert torch.equal(plan.outputs, torch.where(given, logits - 1, logits))
