"""Host logic of vocabulary sampling (no GPU): refusals of the plan and of the C
entry, and the workspace query."""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import _native, sampling

BF16, F16, F32 = 0, 1, 2
FINE = 0x10000  # an aligned address that no refused call reads


def entry(**changes):
    args = dict(logits=FINE, dtype=BF16, stride=100, rows=4, width=100, live=4, count=None, t=FINE, k=FINE, p=FINE,
                m=FINE, u=FINE, tokens=FINE, valid=FINE, logprobs=None, workspace=FINE, nbytes=1 << 30)
    args.update(changes)
    return _native.call("cubic_vocab_sample", *args.values(), None)


@pytest.mark.parametrize("changes,match", [
    *(({name: None}, "null operand") for name in ("logits", "t", "k", "p", "m", "u", "tokens", "valid")),
    ({"dtype": 3}, "dtype"), ({"dtype": -1}, "dtype"), ({"rows": 0}, "rows=0"), ({"rows": 1 << 24}, "rows="),
    ({"width": 0}, "width=0"), ({"width": 101}, "row_stride"), ({"width": (1 << 20) + 1, "stride": 1 << 21}, "width="),
    ({"live": -1}, "live_rows"), ({"live": 5}, "live_rows"), ({"logits": FINE + 1}, "aligned"),
    ({"dtype": F32, "logits": FINE + 2}, "aligned"), ({"workspace": None}, "workspace"),
    ({"workspace": FINE + 8}, "workspace"), ({"nbytes": 0}, "workspace")])
def test_entry_refuses_before_any_launch(changes, match):
    with pytest.raises(Exception, match=match):
        entry(**changes)


def test_workspace_query():
    query = _native.lib().cubic_vocab_sample_workspace_bytes
    for rows, width, dtype in ((0, 9, 0), (-1, 9, 0), (1 << 24, 9, 0), (4, 0, 0), (4, (1 << 20) + 1, 0), (4, 9, 3), (4, 9, -1)):
        assert query(rows, width, dtype) == -1
    for dtype in (BF16, F16, F32):
        for rows in (1, 3, 48, 64, 255, 256, 1000):
            for width in (1, 7, 8192, 16384, 128001, 1 << 20):
                need = query(rows, width, dtype)
                # counters, heads and lists: below 16 bytes per column and
                # 256 KiB per workgroup
                assert 0 < need <= 16 * rows * width + max(256, rows) * (1 << 18)
                with pytest.raises(Exception, match="workspace"):
                    entry(rows=rows, live=rows, width=width, stride=width, dtype=dtype, nbytes=need - 1)


def test_plan_refuses_host_tensors_and_other_types():
    rows = 3
    args = dict(logits=torch.zeros((rows, 9)), temperatures=torch.ones(rows), top_ks=torch.zeros(rows, dtype=torch.int64),
                top_ps=torch.ones(rows), min_ps=torch.zeros(rows), uniforms=torch.zeros(rows))
    with pytest.raises(ValueError, match="CUDA"):
        sampling.VocabSamplingPlan(**args)
    with pytest.raises(TypeError, match="tensors"):
        sampling.VocabSamplingPlan(**{**args, "top_ks": [0] * rows})
