"""Host logic of the adapters (no GPU): refusals of the bank, of the binding
and of the C entry, the workspace query, and the bank's layout."""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import _native, adapters


def bank(**changes):
    args = dict(n=24, k=64, slots=3, max_rank=12, device="cpu")
    args.update(changes)
    return adapters.AdapterBank(args.pop("n"), args.pop("k"), **args)


@pytest.mark.parametrize("changes,match", [
    ({"k": 60}, "multiple of 8"), ({"n": 0}, "width"), ({"slots": 0}, "slot count"),
    ({"max_rank": 257}, "rank"), ({"max_rank": 0}, "rank"), ({"max_rank": True}, "rank"),
    ({"dtype": torch.float32}, "BF16"), ({"n": 1 << 27}, "2\\^30")])
def test_bank_refusals(changes, match):
    with pytest.raises(ValueError, match=match):
        bank(**changes)


def test_bank_layout_and_slots():
    b = bank()
    assert b.down.shape == (3, 16, 64) and b.up.shape == (3, 24, 16) and b.ranks.tolist() == [0, 0, 0]
    b.down.fill_(9), b.up.fill_(9)
    down, up = torch.randn((5, 64)).bfloat16(), torch.randn((24, 5)).bfloat16()
    b.load(1, down, up, 0.5)
    assert torch.equal(b.down[1, :5], down) and torch.equal(b.up[1, :, :5], up)
    assert not b.down[1, 5:].any() and not b.up[1, :, 5:].any()
    assert b.ranks.tolist() == [0, 5, 0] and b.scales.tolist() == [0, 0.5, 0]
    assert (b.down[[0, 2]] == 9).all() and (b.up[[0, 2]] == 9).all()
    b.clear(1)
    assert b.ranks.tolist() == [0, 0, 0]
    for slot in (-1, 3, 1.0):
        with pytest.raises(ValueError, match="slot"):
            b.load(slot, down, up)
        with pytest.raises(ValueError, match="slot"):
            b.clear(slot)
    with pytest.raises(ValueError, match="rank 13"):
        b.load(0, torch.zeros((13, 64)).bfloat16(), torch.zeros((24, 13)).bfloat16())
    with pytest.raises(ValueError, match="needs down"):
        b.load(0, down, up.t().contiguous())
    with pytest.raises(ValueError, match="dtype"):
        b.load(0, down.float(), up)


def test_binding_refuses_host_tensors():
    b = bank()
    x, y = torch.zeros((2, 64)).bfloat16(), torch.zeros((2, 24)).bfloat16()
    slots = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        adapters.bind_adapters(x, b, slots, y)
    with pytest.raises(TypeError, match="AdapterBank"):
        adapters.bind_adapters(x, [b, y], slots, [y, y])
    with pytest.raises(TypeError, match="tensors"):
        adapters.bind_adapters(x, b, [0, 0], y)
    with pytest.raises(ValueError, match="1..8 banks"):
        adapters.bind_adapters(x, [b] * 9, slots, [y] * 9)


def test_overlap_of_row_major_matrices():
    t = torch.zeros((4, 32))
    share = adapters._overlap
    assert share(t, t) and share(t, t[1:]) and share(t[:, :8], t[:, 4:12])
    assert not share(t[:, :8], t[:, 8:]) and not share(t[:, 8:], t[:, :8])
    assert not share(t[:2], t[2:]) and not share(t, torch.zeros((4, 32)))
    assert share(t[:, :8], t.view(8, 16)[:, 8:])  # other strides: by extent


def tables(ns, caps):
    c = _native.ctypes
    j = len(ns)
    ptrs = lambda: (c.c_void_p * j)(*([4096] * j))
    strides = lambda: (c.c_int64 * j)(*ns)
    return ((c.c_int64 * j)(*ns), (c.c_int * j)(*caps), ptrs(), ptrs(), ptrs(), ptrs(), ptrs(), strides(),
            ptrs(), strides())


def test_workspace_query():
    lib, c = _native.lib(), _native.ctypes
    caps = lambda *v: (c.c_int * len(v))(*v)
    assert lib.cubic_adapters_workspace_bytes(64, 4096, 3, caps(16, 16, 24)) == 4 * 64 * 64 * 4
    assert lib.cubic_adapters_workspace_bytes(1, 8, 1, caps(8)) == 64
    sizes = [lib.cubic_adapters_workspace_bytes(m, 12288, 1, caps(64)) for m in (1, 64, 65, 4096)]
    assert sizes == sorted(sizes)  # covers every smaller m
    for bad in ((0, 8, 1, caps(8)), (1, 8, 9, caps(*[8] * 9)), (1, 8, 1, caps(12)), (1, 8, 1, caps(264)),
                (1 << 24, 8, 1, caps(8)), (1, (1 << 20) + 8, 1, caps(8)), (1, 8, 1, None)):
        assert lib.cubic_adapters_workspace_bytes(*bad) == -1


@pytest.mark.parametrize("m,k,ldx,slots,ns,caps,dtype,ws,match", [
    (4, 64, 64, 2, (16,), (8,), 2, 1 << 20, "dtype"),
    (0, 64, 64, 2, (16,), (8,), 0, 1 << 20, "extents"),
    (4, 64, 64, 0, (16,), (8,), 0, 1 << 20, "extents"),
    (4, 60, 64, 2, (16,), (8,), 0, 1 << 20, "k % 8"),
    (4, 64, 60, 2, (16,), (8,), 0, 1 << 20, "k % 8"),
    (4, 64, 1 << 24, 2, (16,), (8,), 0, 1 << 20, "ldx <= 2"),
    (4, 64, 64, 2, (16,), (12,), 0, 1 << 20, "multiple of 8"),
    (4, 64, 64, 2, (16,), (264,), 0, 1 << 20, "multiple of 8"),
    (4, 64, 64, 2, (16, 0), (8, 8), 0, 1 << 20, "width"),
    (4, 64, 64, 2, (1 << 27,), (8,), 0, 1 << 20, "width"),
    (4, 64, 64, 2, (16,), (8,), 0, 64, "workspace"),
    (4, 64, 64, 2, (16,) * 9, (8,) * 9, 0, 1 << 20, "members=9"),
])
def test_entry_refuses_before_any_launch(m, k, ldx, slots, ns, caps, dtype, ws, match):
    with pytest.raises(ValueError, match=match):
        _native.call("cubic_adapters", 4096, ldx, 4096, m, k, slots, len(ns), *tables(ns, caps), dtype,
                     4096, ws, None)


def test_entry_refuses_null_and_misaligned_operands():
    t = tables((16,), (8,))
    with pytest.raises(ValueError, match="null"):
        _native.call("cubic_adapters", 4096, 64, None, 4, 64, 2, 1, *t, 0, 4096, 1 << 20, None)
    with pytest.raises(ValueError, match="16-byte"):
        _native.call("cubic_adapters", 4104, 64, 4096, 4, 64, 2, 1, *t, 0, 4096, 1 << 20, None)
    with pytest.raises(ValueError, match="workspace"):
        _native.call("cubic_adapters", 4096, 64, 4096, 4, 64, 2, 1, *t, 0, None, 1 << 20, None)
    t[2][0] = None
    with pytest.raises(ValueError, match="member 0"):
        _native.call("cubic_adapters", 4096, 64, 4096, 4, 64, 2, 1, *t, 0, 4096, 1 << 20, None)
    t[2][0] = 4104
    with pytest.raises(ValueError, match="16-byte"):
        _native.call("cubic_adapters", 4096, 64, 4096, 4, 64, 2, 1, *t, 0, 4096, 1 << 20, None)


def test_binding_notices_a_bank_given_other_tensors():
    """The launch holds the bank's addresses: a bank whose tensors are replaced,
    not written, is refused."""
    b = bank()
    x, slots, y = torch.zeros((2, 64)).bfloat16(), torch.zeros(2, dtype=torch.int32), torch.zeros((2, 24)).bfloat16()
    launch = adapters._AdapterLaunch(x, (b,), slots, (y,), (y,), torch.empty(16, dtype=torch.uint8))
    launch.validate()
    b.load(1, torch.ones((5, 64)).bfloat16(), torch.ones((24, 5)).bfloat16())
    launch.validate()
    b.down = b.down.clone()
    with pytest.raises(ValueError, match="changed after binding"):
        launch.validate()


@pytest.mark.parametrize("m,k,ns,caps", [
    ((1 << 23) + 64, 1032, (8,) * 8, (256,) * 8),  # partitions to be joined
    ((1 << 24) - 1, 64, (1 << 16,), (8,)),         # rows by columns
    (1 << 23, 1 << 20, (8,), (8,)),                # rows by partitions of K
])
def test_entry_refuses_extents_past_a_grid(m, k, ns, caps):
    with pytest.raises(ValueError, match="past a launch"):
        _native.call("cubic_adapters", 4096, k, 4096, m, k, 2, len(ns), *tables(ns, caps), 0, 4096, 1 << 50, None)
