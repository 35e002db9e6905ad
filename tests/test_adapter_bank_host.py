"""Adapter banks (no GPU): what loading leaves behind, and what a binding notices."""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import adapters


def bank(**changes):
    args = dict(n=24, k=64, slots=3, max_rank=12, device="cpu")
    args.update(changes)
    return adapters.AdapterBank(args.pop("n"), args.pop("k"), **args)


def adapter(rank, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((rank, 64), generator=gen).bfloat16(), torch.randn((24, rank), generator=gen).bfloat16()


def test_loading_parameters_records_no_history():
    b = bank()
    for turn in range(3):
        down, up = (torch.nn.Parameter(t) for t in adapter(5, turn))
        b.load(1, down, up, torch.nn.Parameter(torch.tensor(0.5)))
    for t in (b.down, b.up, b.scales, b.ranks):
        assert not t.requires_grad and t.grad_fn is None
    assert torch.equal(b.down[1, :5], down.detach()) and torch.equal(b.up[1, :, :5], up.detach())


def test_a_refused_load_leaves_the_slot_as_it_was():
    b = bank()
    held = adapter(5)
    b.load(1, *held, 0.5)
    before = [t.clone() for t in (b.down, b.up, b.scales, b.ranks)]
    for scale in ("large", None, torch.ones(2), 1j):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            b.load(1, *adapter(7, 1), scale)
        assert all(torch.equal(t, u) for t, u in zip((b.down, b.up, b.scales, b.ranks), before))


CHANGES = {
    "other storage": lambda b: b.ranks.set_(torch.zeros(3, dtype=torch.int32)),
    "other data": lambda b: setattr(b.down, "data", torch.zeros_like(b.down)),
    "freed": lambda b: b.up.untyped_storage().resize_(0),
    "grown": lambda b: b.scales.resize_(1 << 12),
    "moved": lambda b: b.ranks.set_(torch.zeros(9, dtype=torch.int32)[3:6]),
    "replaced": lambda b: setattr(b, "up", b.up.clone()),
}


@pytest.mark.parametrize("change", CHANGES)
def test_a_binding_notices_a_bank_whose_memory_is_another(change):
    """The launch holds the bank's addresses; writing to the bank keeps them."""
    b = bank()
    x, slots, y = torch.zeros((2, 64)).bfloat16(), torch.zeros(2, dtype=torch.int32), torch.zeros((2, 24)).bfloat16()
    launch = adapters._AdapterLaunch(x, (b,), slots, (y,), (y,), torch.empty(16, dtype=torch.uint8))
    b.load(2, *adapter(5))
    launch.validate()
    CHANGES[change](b)
    with pytest.raises(ValueError, match="changed after binding"):
        launch.validate()


@pytest.mark.parametrize("name,shape,dtype", [
    ("down", (3, 8, 64), torch.bfloat16), ("down", (2, 16, 64), torch.bfloat16), ("down", (3, 16, 64), torch.float16),
    ("up", (3, 24, 8), torch.bfloat16), ("up", (3, 23, 16), torch.bfloat16), ("up", (3, 24, 16), torch.float32),
    ("scales", (2,), torch.float32), ("scales", (3,), torch.float64), ("ranks", (2,), torch.int32),
    ("ranks", (3,), torch.int64)])
def test_a_bank_whose_tensors_do_not_fit_it_is_not_bound(name, shape, dtype):
    """The launch reads the extents that the bank was made with."""
    b = bank()
    x, slots, y = torch.zeros((2, 64)).bfloat16(), torch.zeros(2, dtype=torch.int32), torch.zeros((2, 24)).bfloat16()
    setattr(b, name, torch.zeros(shape, dtype=dtype))
    with pytest.raises(ValueError, match=f"adapter bank's {name}"):
        adapters.bind_adapters(x, b, slots, y)


def test_a_bank_whose_matrices_lie_in_another_order_is_not_bound():
    x, slots, y = torch.zeros((2, 64)).bfloat16(), torch.zeros(2, dtype=torch.int32), torch.zeros((2, 24)).bfloat16()
    for name in ("down", "up"):
        b = bank()
        setattr(b, name, getattr(b, name).transpose(1, 2).contiguous().transpose(1, 2))
        with pytest.raises(ValueError, match=f"adapter bank's {name}"):
            adapters.bind_adapters(x, b, slots, y)
    b = bank()
    b.scales = torch.zeros(6)[::2]
    with pytest.raises(ValueError, match="adapter bank's scales"):
        adapters.bind_adapters(x, b, slots, y)
