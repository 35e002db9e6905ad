"""Penalties for repeated tokens, biases and grammar masks between the lm_head and
the samplers, and the history of tokens that they read.

A ``TokenHistory`` keeps on the device, per request slot, how often each token was
put out, which tokens the prompt has, and biases.  A ``LogitPenaltyPlan`` applies
them to a step's logits, which a VocabSamplingPlan, an MTPVerifyPlan or a greedy
sampler then reads.  In a verify step the row of depth d counts the first d drafts
as put out, so ``draft_tokens`` are those of MTPVerifyPlan; what it emits goes into
the history with ``append(slots, plan.emitted)``.

No counterpart in the reference's verify path.  The kernels are cubic_history_*
and cubic_logit_penalties; there is no eager fallback.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from . import _native
from .linear import operand_identity
from .sampling import _CANDIDATE_DTYPES

MAX_DEPTH = 8  # kMaxPenaltyDepth of the C ABI
BUCKET = 4096  # kHistoryBucket: tokens of the vocabulary that share a list


def _live(live, most: int, device: torch.device, what: str) -> tuple[int, int | None]:
    """(host count, device count or None) of a launch argument."""
    if live is None:
        return most, None
    if isinstance(live, Tensor):
        if live.dtype != torch.int32 or live.device != device or live.numel() < 1 or not live.is_contiguous():
            raise ValueError(f"live {what} count must be a device int32 tensor")
        return most, live.data_ptr()
    if type(live) is not int or not 0 <= live <= most:
        raise ValueError(f"live {what} count must be an int in 0..{most} or a device int32 tensor")
    return live, None


class TokenHistory:
    """Tokens and biases of ``slots`` requests over ``vocab`` tokens.

    ``state`` int32 [slots, vocab, 2] (a token's mark and its bias' bits) and ``listed``
    int32 [slots, vocab]: 12 bytes per slot and token; ``sizes`` int32 [slots, ceil(vocab / 4096)].  Its methods enqueue on the
    current stream and order nothing against other streams; but for ``set_bias``
    they may be captured, and read their tensors when they run.
    """

    def __init__(self, slots: int, vocab: int, device: torch.device | str = "cuda"):
        if type(slots) is not int or not 1 <= slots < 1 << 20:
            raise ValueError("history slots must be an int in 1..2^20 - 1")
        if type(vocab) is not int or not 1 <= vocab <= 1 << 24:
            raise ValueError("history vocabulary must be an int in 1..2^24")
        self.slots, self.vocab = slots, vocab
        # (their addresses are copied by every launch)
        self._tables = (torch.zeros((slots, vocab, 2), dtype=torch.int32, device=device),
                        torch.zeros((slots, vocab), dtype=torch.int32, device=device),
                        torch.zeros((slots, (vocab + BUCKET - 1) // BUCKET), dtype=torch.int32, device=device))
        self._storages = tuple(t.untyped_storage() for t in self._tables)
        self.device = self.state.device
        self._args = (*(t.data_ptr() for t in self._tables), slots, vocab)

    state = property(lambda self: self._tables[0])
    listed = property(lambda self: self._tables[1])
    sizes = property(lambda self: self._tables[2])

    def _check_tables(self) -> None:
        if tuple(t.data_ptr() for t in self._tables) != self._args[:3]:
            raise ValueError("a history's tensors were given other memory")

    def _check_slots(self, row_slots: Tensor) -> None:
        if not isinstance(row_slots, Tensor):
            raise TypeError("history slots must be a tensor")
        if row_slots.dtype != torch.int32 or row_slots.ndim != 1 or row_slots.numel() < 1 \
                or row_slots.device != self.device or not row_slots.is_contiguous():
            raise ValueError("history slots must be a contiguous int32 [rows] tensor on the history's device")

    def _slot(self, slot: int) -> int:
        if type(slot) is not int or not 0 <= slot < self.slots:
            raise ValueError(f"history slot must be an int in 0..{self.slots - 1}")
        return slot

    def _call(self, name: str, *args) -> None:
        self._check_tables()
        if self.device.type != "cuda":
            raise ValueError("a token history must be on a CUDA device")
        with _native.on_device(self.device.index):
            _native.call(name, *self._args, *args, _native.stream_of(self.device.index))

    def _append(self, row_slots: Tensor, tokens: Tensor, prompt: bool, live_rows) -> None:
        self._check_slots(row_slots)
        if not isinstance(tokens, Tensor):
            raise TypeError("history tokens must be a tensor")
        if tokens.ndim == 1:
            tokens = tokens[:, None]
        if tokens.dtype not in (torch.int32, torch.int64) or tokens.ndim != 2 or min(tokens.shape) < 1 \
                or tokens.shape[0] != row_slots.numel() or tokens.device != self.device \
                or (tokens.shape[1] > 1 and tokens.stride(1) != 1) \
                or (tokens.shape[0] > 1 and tokens.stride(0) < tokens.shape[1]):
            raise ValueError("history tokens must be row-major int32 or int64 [rows] or [rows, length] on its device")
        rows, length = tokens.shape
        live, live_ptr = _live(live_rows, rows, self.device, "row")
        self._call("cubic_history_append", row_slots.data_ptr(), tokens.data_ptr(), tokens.element_size(),
                   tokens.stride(0), rows, length, int(prompt), live, live_ptr)

    def append(self, row_slots: Tensor, tokens: Tensor, live_rows: int | Tensor | None = None) -> None:
        """Count ``tokens`` [rows] or [rows, length] as outputs of ``row_slots``.  Tokens
        outside the vocabulary (-1 pads) and slots outside the history (-1) are
        skipped; a slot may come more than once."""
        self._append(row_slots, tokens, False, live_rows)

    def append_prompt(self, row_slots: Tensor, tokens: Tensor, live_rows: int | Tensor | None = None) -> None:
        """Mark ``tokens`` as the prompts' (repetition penalises them, the others do not)."""
        self._append(row_slots, tokens, True, live_rows)

    def clear(self, slots: int | Tensor) -> None:
        """Empty a slot, or the slots of an int32 [rows] tensor: tokens and biases."""
        if isinstance(slots, Tensor):
            self._check_slots(slots)
            self._call("cubic_history_clear", slots.data_ptr(), slots.numel(), 0, 0)
        else:
            self._call("cubic_history_clear", None, 1, self._slot(slots), 0)

    def set_bias(self, slot: int, tokens, values) -> None:
        """Replace a slot's biases: distinct token ids and as many numbers, finite or
        -infinity (which bans a token).  Empty ones remove them.  Waits for the
        device where they lie there; not under capture."""
        self._slot(slot)
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("biases must be set before graph capture")
        listed = lambda v: v.tolist() if isinstance(v, Tensor) else list(v)
        ids, numbers = listed(tokens), [float(v) for v in listed(values)]
        if len(ids) != len(numbers) or len(set(ids)) != len(ids):
            raise ValueError("biases need distinct tokens and a number for each")
        if any(type(t) is not int or not 0 <= t < self.vocab for t in ids):
            raise ValueError(f"biased tokens must be ints in 0..{self.vocab - 1}")
        if any(math.isnan(v) or v == math.inf or abs(v) > 3e38 and v != -math.inf for v in numbers):
            raise ValueError("biases must be finite or -infinity")
        self._call("cubic_history_clear", None, 1, slot, 1)
        if ids:
            on_device = (torch.tensor(ids, dtype=torch.int32, device=self.device),
                         torch.tensor(numbers, dtype=torch.float32, device=self.device))
            self._call("cubic_history_bias", slot, *(t.data_ptr() for t in on_device), len(ids))

    def counts(self, slot: int) -> Tensor:
        """How often each token was put out, int32 [vocab]."""
        return self.state[self._slot(slot), :, 0] & ((1 << 30) - 1)

    def biases(self, slot: int) -> Tensor:
        """Each token's bias, float32 [vocab]."""
        return self.state[self._slot(slot), :, 1].contiguous().view(torch.float32)


class LogitPenaltyPlan:
    """Penalties, biases and a grammar's mask on logits, in one launch.

    With c the times that token t is among the outputs of row's request (its drafts
    before the row included):

        l = l / repetition if l > 0 else l * repetition   (t in the prompt, or c > 0)
        l = l - frequency * c - (presence if c > 0 else 0)
        l = l + bias, and -inf where the token's mask bit is 0

    in 32 bits, rounded once.  ``logits`` [sequences * (depth + 1), V] bf16, fp16 or
    fp32 (rows may be padded), ``slots`` int32 [sequences]: -1 (or any slot outside
    the history) takes the mask only.  ``repetition``, ``presence`` and ``frequency``
    float32 [sequences] or None; one that is no finite number, or a repetition that
    is not positive, makes its sequence's rows NaN, which the samplers refuse.
    ``draft_tokens`` int64 [depth, sequences] make depth + 1 rows per sequence, as
    MTPVerifyPlan has them.  ``token_mask`` int32 [rows, words], bit t % 32 of word t /
    32 admits t.  ``outputs`` None changes the logits in place; else it is
    [rows, V] of their type or float32, in memory of its own.  All operands are read when
    the launch runs.
    """

    def __init__(self, *, logits: Tensor, history: TokenHistory, slots: Tensor, repetition: Tensor | None = None,
                 presence: Tensor | None = None, frequency: Tensor | None = None,
                 draft_tokens: Tensor | None = None, token_mask: Tensor | None = None,
                 outputs: Tensor | None = None, visible_width: int | None = None):
        if not isinstance(history, TokenHistory):
            raise TypeError("penalties need a TokenHistory")
        optional = (repetition, presence, frequency, draft_tokens, token_mask, outputs)
        if not isinstance(logits, Tensor) or not isinstance(slots, Tensor) or \
                any(t is not None and not isinstance(t, Tensor) for t in optional):
            raise TypeError("penalty operands must be tensors")
        row_major = lambda t: (t.ndim == 2 and min(t.shape) >= 1 and (t.stride(1) == 1 or t.shape[1] == 1)
                               and (t.stride(0) >= t.shape[1] or t.shape[0] == 1))
        if logits.dtype not in _CANDIDATE_DTYPES or logits.device.type != "cuda" or not row_major(logits):
            raise ValueError("penalised logits must be row-major CUDA bf16, fp16 or fp32 [rows, V]")
        device = logits.device
        history._check_tables()
        history._check_slots(slots)
        if history.device != device:
            raise ValueError("logits and history must be on one CUDA device")
        self.sequences, self.depth = slots.numel(), 0
        if draft_tokens is not None:
            self.depth = draft_tokens.shape[0] if draft_tokens.ndim == 2 else 0
            if draft_tokens.dtype != torch.int64 or draft_tokens.shape != (self.depth, self.sequences) \
                    or not 1 <= self.depth <= MAX_DEPTH or draft_tokens.device != device or not draft_tokens.is_contiguous():
                raise ValueError(f"draft tokens must be contiguous int64 [depth, sequences], depth in 1..{MAX_DEPTH}")
        rows = self.sequences * (self.depth + 1)
        if logits.shape[0] != rows:
            raise ValueError(f"{self.sequences} sequences of depth {self.depth} need {rows} rows of logits")
        self.width = logits.shape[1] if visible_width is None else visible_width
        if type(self.width) is not int or not 1 <= self.width <= min(logits.shape[1], history.vocab):
            raise ValueError("visible width must be in 1..V and at most the history's vocabulary")
        for t in (repetition, presence, frequency):
            if t is not None and (t.dtype != torch.float32 or t.shape != (self.sequences,) or t.device != device
                                  or not t.is_contiguous()):
                raise ValueError("penalties must be contiguous float32 [sequences] on the logits' device")
        words = 0
        if token_mask is not None:
            if token_mask.dtype != torch.int32 or token_mask.ndim != 2 or token_mask.shape[0] != rows \
                    or token_mask.shape[1] * 32 < self.width or token_mask.device != device or not token_mask.is_contiguous():
                raise ValueError("grammar bitmask must be contiguous int32 [rows, words] over the visible width")
            words = token_mask.shape[1]
        if outputs is None:
            outputs = logits
        elif outputs.dtype not in (logits.dtype, torch.float32) or outputs.shape != logits.shape \
                or outputs.device != device or not row_major(outputs):
            raise ValueError("penalty outputs must be row-major [rows, V] of the logits' type or float32")
        elif any(outputs.untyped_storage().data_ptr() == t.untyped_storage().data_ptr()
                 for t in (logits, slots, repetition, presence, frequency, draft_tokens, token_mask) if t is not None):
            raise ValueError("penalty outputs must not alias their operands")
        self.logits, self.history, self.outputs = logits, history, outputs
        operands = [t for t in (logits, outputs, slots, *optional[:5]) if t is not None]
        stride = lambda t: max(t.stride(0), t.shape[1])
        self._head = (logits.data_ptr(), _CANDIDATE_DTYPES[logits.dtype], stride(logits), self.sequences, self.depth, self.width)
        self._tail = (*history._args, slots.data_ptr(), *(_native.ptr(t) for t in optional[:5]), words, outputs.data_ptr(),
                      _CANDIDATE_DTYPES[outputs.dtype], stride(outputs), None)
        # the call with all sequences live
        self._call = _native.BoundCall("cubic_logit_penalties", *self._head, self.sequences, None, *self._tail[:-1])
        # what a launch looks at: whether every operand still has its memory (which is held) and layout
        self._held = tuple(t.untyped_storage() for t in operands)
        self._operands = tuple(operands)
        self._identity = self._look()
        self._index = device.index

    def _look(self) -> list:
        return [*operand_identity(self._operands), *[t.data_ptr() for t in self.history._tables]]

    def launch(self, live_sequences: int | Tensor | None = None) -> None:
        """Enqueue on the current stream.  The rows of sequences at or past
        ``live_sequences`` (a host int, or a device int32 tensor whose first element
        is read when the launch runs) keep their outputs."""
        if self._look() != self._identity:
            raise ValueError("penalty operands changed after binding")
        index = self._index
        live = None if live_sequences is None else _live(live_sequences, self.sequences, self.history.device, "sequence")
        if live is None and _native.current_device() == index:
            self._call.launch(_native.stream_of(index))
            return
        with _native.on_device(index):
            if live is None:
                self._call.launch(_native.stream_of(index))
            else:
                _native.call("cubic_logit_penalties", *self._head, *live, *self._tail, _native.stream_of(index))
