"""Low-rank adapters of many requests beside a shared packed projection.

Every row of a step belongs to a request, and every request may have its own
adapter of the projection: y[i] = base[i] + scale * up (down x[i]), with down
[rank, k] and up [n, rank] those of row i's slot.  An ``AdapterBank`` holds the
adapters of one [n, k] projection in device slots; a binding takes one bank per
projection that shares x (q, k, v; gate, up) and a device table of each row's
slot, which is read when the launch runs, as are the slots themselves: a captured
launch follows later changes of both.

``PackedLinearOperators.bind_adapters`` adds to given projection outputs and
``bind_adapted_linear`` binds the shared projection with it.  No counterpart in
the reference.  The kernels are cubic_adapters (one launch for few rows, else
a down and an up launch, with one between them that joins partial sums of
long K); there is no eager fallback.
"""
from __future__ import annotations

from typing import Sequence

import torch
from torch import Tensor

from . import _native
from .linear import DTYPE_IDS, MAX_GROUP_MEMBERS, PackedOperatorBinding

MAX_RANK = 256  # kMaxAdapterRank of the C ABI


def _positive(value, name: str, limit: int) -> int:
    if type(value) is not int or not 1 <= value <= limit:
        raise ValueError(f"adapter {name} must be an int in 1..{limit}")
    return value


class AdapterBank:
    """Adapters of one [n, k] projection in ``slots`` device slots.

    ``down`` is [slots, capacity, k] and ``up`` [slots, n, capacity], with
    capacity ``max_rank`` rounded up to a multiple of 8; ``ranks`` int32 and
    ``scales`` float32 [slots].  A slot is empty (rank 0, rows pass through)
    until ``load`` fills it.
    """

    def __init__(self, n: int, k: int, *, slots: int, max_rank: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        self.n, self.k = _positive(n, "width", (1 << 30) - 1), _positive(k, "K", 1 << 20)
        self.slots = _positive(slots, "slot count", (1 << 20) - 1)
        self.max_rank = _positive(max_rank, "rank", MAX_RANK)
        self.capacity = (max_rank + 7) // 8 * 8
        if dtype not in DTYPE_IDS:
            raise ValueError("adapters serve BF16 or FP16 activations")
        if k % 8:
            raise ValueError("adapters need K to be a multiple of 8")
        if n * self.capacity >= 1 << 30:
            raise ValueError("adapter width times rank must stay below 2^30")
        self.dtype, self.device = dtype, torch.device(device)
        self.down = torch.zeros((slots, self.capacity, k), dtype=dtype, device=self.device)
        self.up = torch.zeros((slots, n, self.capacity), dtype=dtype, device=self.device)
        self.scales = torch.zeros(slots, dtype=torch.float32, device=self.device)
        self.ranks = torch.zeros(slots, dtype=torch.int32, device=self.device)

    def check(self) -> None:
        """Whether the tensors are as the bank was made: a launch reads those extents."""
        for name, shape, dtype in (("down", (self.slots, self.capacity, self.k), self.dtype),
                                   ("up", (self.slots, self.n, self.capacity), self.dtype),
                                   ("scales", (self.slots,), torch.float32), ("ranks", (self.slots,), torch.int32)):
            t = getattr(self, name)
            if t.shape != shape or t.dtype is not dtype or not t.is_contiguous() or t.device != self.down.device:
                raise ValueError(f"adapter bank's {name} must be contiguous {dtype} {list(shape)} on one device")

    def _slot(self, slot: int) -> int:
        if type(slot) is not int or not 0 <= slot < self.slots:
            raise ValueError(f"adapter slot must be an int in 0..{self.slots - 1}")
        return slot

    @torch.no_grad()  # of trained parameters too: no history in the bank
    def load(self, slot: int, down: Tensor, up: Tensor, scale: float = 1.0) -> None:
        """Put an adapter (down [rank, k], up [n, rank]) into a slot, on the
        device's current stream: order it against launches on other streams."""
        self._slot(slot)
        if down.ndim != 2 or up.ndim != 2 or down.shape[1] != self.k or up.shape != (self.n, down.shape[0]):
            raise ValueError(f"adapter needs down [rank, {self.k}] and up [{self.n}, rank]")
        rank = down.shape[0]
        if not 1 <= rank <= self.max_rank:
            raise ValueError(f"adapter rank {rank} outside 1..{self.max_rank}")
        if down.dtype != self.dtype or up.dtype != self.dtype:
            raise ValueError("adapter matrices differ from the bank's dtype")
        scale = float(scale)  # before anything of the slot changes
        self.down[slot, :rank].copy_(down)
        self.down[slot, rank:].zero_()
        self.up[slot, :, :rank].copy_(up)
        self.up[slot, :, rank:].zero_()  # the kernel multiplies whole groups of 8 ranks
        self.scales[slot].fill_(scale)
        self.ranks[slot].fill_(rank)

    def clear(self, slot: int) -> None:
        """Empty a slot: its rows pass through."""
        self.ranks[self._slot(slot)].fill_(0)


def _table(ctype, values):
    return (ctype * len(values))(*values)


class _AdapterLaunch:
    """One bound cubic_adapters call; the argument tables are built once."""

    def __init__(self, x: Tensor, banks: tuple, row_slots: Tensor, bases: tuple, outputs: tuple,
                 workspace: Tensor):
        c = _native.ctypes
        self.x, self.banks, self.row_slots = x, banks, row_slots
        self.bases, self.outputs, self.workspace = bases, outputs, workspace
        self._operands = (x, row_slots, *bases, *outputs)
        # the banks' memory is held, so that no other tensor can come to its addresses
        self._held = tuple(t.untyped_storage() for b in banks for t in (b.down, b.up, b.scales, b.ranks))
        self.identity, self._addresses = self._identity(), self._bank_addresses()
        ptrs = lambda ts: _table(c.c_void_p, [t.data_ptr() for t in ts])
        # (the row stride of a single row means nothing: a row, or at least that, then)
        self._args = (
            x.data_ptr(), x.stride(0) if x.shape[0] > 1 else x.shape[1], row_slots.data_ptr(), x.shape[0], x.shape[1], banks[0].slots,
            len(banks), _table(c.c_int64, [b.n for b in banks]), _table(c.c_int, [b.capacity for b in banks]),
            ptrs([b.down for b in banks]), ptrs([b.up for b in banks]), ptrs([b.scales for b in banks]),
            ptrs([b.ranks for b in banks]), ptrs(bases), _table(c.c_int64, [max(b.stride(0), b.shape[1]) for b in bases]),
            ptrs(outputs), _table(c.c_int64, [max(y.stride(0), y.shape[1]) for y in outputs]), DTYPE_IDS[x.dtype],
            workspace.data_ptr(), workspace.numel())

    def _identity(self):
        return [(t.data_ptr(), t.shape, t.stride(), t.dtype) for t in self._operands]

    def _bank_addresses(self):
        return [(b.down.data_ptr(), b.up.data_ptr(), b.scales.data_ptr(), b.ranks.data_ptr()) for b in self.banks]

    def validate(self) -> None:
        if self._identity() != self.identity or self._bank_addresses() != self._addresses:
            raise ValueError("adapter launch operands changed after binding")

    def __call__(self, stream: int) -> None:
        _native.call("cubic_adapters", *self._args, stream)


def _overlap(a: Tensor, b: Tensor) -> bool:
    """Whether two row-major matrices share memory; column slices of one
    matrix (q, k, v of a fused output) interleave without sharing any."""
    size, stride = a.element_size(), a.stride(0) * a.element_size()
    extent = lambda t: ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size()
    a0, b0 = a.data_ptr(), b.data_ptr()
    if a0 + extent(a) <= b0 or b0 + extent(b) <= a0:
        return False
    if a.stride(0) != b.stride(0) or size != b.element_size() or min(a.shape[0], b.shape[0]) < 2:
        return True
    apart = (b0 - a0) % stride
    return apart < a.shape[1] * size or apart + b.shape[1] * size > stride


def bind_adapters(x: Tensor, banks: Sequence[AdapterBank] | AdapterBank, row_slots: Tensor,
                  outputs: Sequence[Tensor] | Tensor, *,
                  bases: Sequence[Tensor] | Tensor | None = None) -> PackedOperatorBinding:
    """Bind ``outputs[j] = bases[j] + adapter of banks[j]`` for rows of ``x``.

    ``row_slots`` int32 [m] names each row's slot; a number outside the bank
    (-1 by convention) or an empty slot means none.  ``bases`` None adds to the
    outputs in place.  Matrices may have padded rows (a row stride); the
    binding owns its workspace, so launches of one binding must not overlap.
    """
    single = isinstance(banks, AdapterBank)
    listed = lambda v: (v,) if isinstance(v, Tensor) else tuple(v)
    banks = (banks,) if single else tuple(banks)
    outputs = listed(outputs)
    bases = outputs if bases is None else listed(bases)
    if not 1 <= len(banks) <= MAX_GROUP_MEMBERS or len(outputs) != len(banks) or len(bases) != len(banks):
        raise ValueError(f"adapters need 1..{MAX_GROUP_MEMBERS} banks with one base and one output each")
    if any(not isinstance(b, AdapterBank) for b in banks):
        raise TypeError("adapters must be AdapterBank objects")
    for bank in banks:
        bank.check()
    tensors = (x, row_slots, *bases, *outputs)
    if any(not isinstance(t, Tensor) for t in tensors):
        raise TypeError("adapter operands must be tensors")
    if x.dtype not in DTYPE_IDS or x.device.type != "cuda":
        raise ValueError("adapters require CUDA FP16/BF16 activations")
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("adapters must be bound before graph capture")
    if any(t.device != x.device for t in tensors) or any(b.down.device != x.device for b in banks):
        raise ValueError("adapter operands must be on one CUDA device")
    if x.ndim != 2 or min(x.shape) < 1 or x.stride(1) != 1 or x.data_ptr() % 16 or \
            (x.shape[0] > 1 and (x.stride(0) < x.shape[1] or x.stride(0) % 8)):
        raise ValueError("adapters require positive 16-byte aligned [M,K] activations")
    m, k = x.shape
    if row_slots.dtype != torch.int32 or row_slots.shape != (m,) or not row_slots.is_contiguous():
        raise ValueError("adapter row slots must be a contiguous int32 [M] tensor")
    for bank, base, y in zip(banks, bases, outputs):
        if bank.k != k or bank.dtype != x.dtype or bank.slots != banks[0].slots:
            raise ValueError("adapter banks differ from the activations in K, dtype or slot count")
        for t in (base, y):
            if t.shape != (m, bank.n) or t.dtype != x.dtype or (t.stride(1) != 1 and bank.n > 1) or \
                    (t.stride(0) < bank.n and m > 1):
                raise ValueError("adapter base or output has an invalid ABI")
    bank_tensors = [t.view(t.shape[0], -1) for b in banks for t in (b.down, b.up)]
    bank_tensors += [t.view(1, -1) for b in banks for t in (b.ranks, b.scales)]
    for j, y in enumerate(outputs):
        others = [x, row_slots.view(1, -1), *bank_tensors, *outputs[:j], *outputs[j + 1:]]
        others += [b for i, b in enumerate(bases) if not (i == j and b.data_ptr() == y.data_ptr()
                                                           and b.stride() == y.stride())]
        if any(_overlap(y, t) for t in others):
            raise ValueError("adapter output must not alias its operands")
    ranks = _table(_native.ctypes.c_int, [b.capacity for b in banks])
    nbytes = _native.lib().cubic_adapters_workspace_bytes(m, k, len(banks), ranks)
    if nbytes < 0:
        raise ValueError("adapter geometry not admitted")
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    launch = _AdapterLaunch(x, banks, row_slots, bases, outputs, workspace)
    return PackedOperatorBinding(outputs[0] if single else outputs, (launch,), scratch=(workspace,))
