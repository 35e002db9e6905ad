"""CPU: what token histories and logit penalties refuse before anything is launched."""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import _native, penalties

HISTORY = dict(state=16, listed=16, sizes=16, slots=4, vocab=100)
BAD_HISTORY = [(dict(state=None), "null history"), (dict(listed=None), "null history"), (dict(sizes=None), "null history"), (dict(slots=0), "history of"),
               (dict(slots=1 << 20), "history of"), (dict(vocab=0), "history of"), (dict(vocab=(1 << 24) + 1), "history of"),
               (dict(state=20), "misaligned history"), (dict(sizes=18), "misaligned history")]
APPEND = HISTORY | dict(rows_slots=16, tokens=16, bytes=8, ld=5, rows=2, length=5, prompt=0, live=2, count=None, stream=None)
CLEAR = HISTORY | dict(row_slots=None, rows=1, slot=0, only=0, stream=None)
BIAS = HISTORY | dict(slot=0, ids=16, values=16, count=3, stream=None)
PENALTIES = (dict(logits=16, dtype=0, ld=100, sequences=2, depth=1, width=100, live=2, count=None) | HISTORY
             | dict(row_slots=16, rep=None, pres=None, freq=None, drafts=16, mask=None, words=0, out=32, out_dtype=0, ldo=100,
                    bound=None, stream=None))


@pytest.mark.parametrize("change,match", BAD_HISTORY)
@pytest.mark.parametrize("name,ok", [("cubic_history_append", APPEND), ("cubic_history_clear", CLEAR), ("cubic_history_bias", BIAS),
                                     ("cubic_logit_penalties", PENALTIES)])
def test_histories_refused(name, ok, change, match):
    with pytest.raises(ValueError, match=match):
        _native.call(name, *(ok | change).values())


@pytest.mark.parametrize("name,ok,change,match", [
    ("cubic_history_append", APPEND, dict(tokens=None), "null"), ("cubic_history_append", APPEND, dict(rows_slots=None), "null"),
    ("cubic_history_append", APPEND, dict(bytes=2), "int32 or int64"), ("cubic_history_append", APPEND, dict(rows=0), "rows"),
    ("cubic_history_append", APPEND, dict(rows=1 << 24), "rows"), ("cubic_history_append", APPEND, dict(length=0), "length"),
    ("cubic_history_append", APPEND, dict(ld=4), "row stride"), ("cubic_history_append", APPEND, dict(live=3), "live_rows"),
    ("cubic_history_append", APPEND, dict(live=-1), "live_rows"), ("cubic_history_append", APPEND, dict(tokens=20), "misaligned"),
    ("cubic_history_clear", CLEAR, dict(slot=4), "slot 4"), ("cubic_history_clear", CLEAR, dict(slot=-1), "slot -1"),
    ("cubic_history_clear", CLEAR, dict(rows=0), "rows"),
    ("cubic_history_bias", BIAS, dict(slot=4), "slot 4"), ("cubic_history_bias", BIAS, dict(count=0), "biases"),
    ("cubic_history_bias", BIAS, dict(count=101), "biases"), ("cubic_history_bias", BIAS, dict(ids=None), "null"),
    ("cubic_logit_penalties", PENALTIES, dict(logits=None), "null"), ("cubic_logit_penalties", PENALTIES, dict(dtype=3), "dtype"),
    ("cubic_logit_penalties", PENALTIES, dict(out_dtype=1), "logits' type"), ("cubic_logit_penalties", PENALTIES, dict(dtype=2), "logits' type"),
    ("cubic_logit_penalties", PENALTIES, dict(sequences=0), "sequences"), ("cubic_logit_penalties", PENALTIES, dict(depth=9), "depth"),
    ("cubic_logit_penalties", PENALTIES, dict(depth=-1), "depth"), ("cubic_logit_penalties", PENALTIES, dict(sequences=1 << 23), "sequences"),
    ("cubic_logit_penalties", PENALTIES, dict(width=0), "width"), ("cubic_logit_penalties", PENALTIES, dict(width=101), "width"),
    ("cubic_logit_penalties", PENALTIES, dict(ld=99), "row strides"), ("cubic_logit_penalties", PENALTIES, dict(ldo=99), "row strides"),
    ("cubic_logit_penalties", PENALTIES, dict(drafts=None), "drafts"), ("cubic_logit_penalties", PENALTIES, dict(mask=16, words=3), "mask"),
    ("cubic_logit_penalties", PENALTIES, dict(live=3), "live_sequences"), ("cubic_logit_penalties", PENALTIES, dict(logits=17), "misaligned"),
    ("cubic_logit_penalties", PENALTIES, dict(drafts=20), "misaligned"), ("cubic_logit_penalties", PENALTIES, dict(out=16, out_dtype=2), "in place"),
    ("cubic_logit_penalties", PENALTIES, dict(out=16, ldo=101), "in place")])
def test_arguments_refused(name, ok, change, match):
    with pytest.raises(ValueError, match=match):
        _native.call(name, *(ok | change).values())


def test_history_on_the_host_is_refused():
    h = penalties.TokenHistory(2, 10, "cpu")
    slots, tokens = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int64)
    for call in (lambda: h.append(slots, tokens), lambda: h.append_prompt(slots, tokens), lambda: h.clear(0), lambda: h.set_bias(0, [1], [1.0]),
                 lambda: penalties.LogitPenaltyPlan(logits=torch.zeros((1, 10)), history=h, slots=slots)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for slots, vocab in ((0, 10), (1 << 20, 10), (2, 0), (2, (1 << 24) + 1), (2.0, 10)):
        with pytest.raises(ValueError):
            penalties.TokenHistory(slots, vocab, "cpu")


@pytest.mark.parametrize("name", ["state", "listed", "sizes"])
def test_a_history_whose_tensors_were_given_other_memory(name):
    """Launches copy their addresses."""
    history = penalties.TokenHistory(2, 100, device="cpu")
    with pytest.raises(AttributeError):
        setattr(history, name, getattr(history, name).clone())
    getattr(history, name).data = getattr(history, name).clone()
    with pytest.raises(ValueError, match="other memory"):
        history.clear(0)
