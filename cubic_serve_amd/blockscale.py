"""Block-scaled 8-bit linears: e4m3 weights with a scale for each 128 x 128 block,
e4m3 activations with a scale for each row and 128 columns, and what makes such
activations (row norms with the residual's addition, gated activations).

  bind_norm         h = x + residual, y = h (offset + weight) / sqrt(mean(h^2) + eps),
                    in 16 bits and / or as BlockScaledActivations
  bind_quantize     x, or silu(gate) * x, as BlockScaledActivations
  bind_block_linear y = x w^T of BlockScaledActivations and BlockScaledMatrix, in
                    bf16, fp16 or fp32; a group shares x in one launch

``PackedLinearOperators`` has them as methods.  Bindings check their operands at
bind time, enqueue on the current stream and allocate nothing at launch.  No
counterpart in the reference's Cubic path.  The kernels are cubic_row_norm,
cubic_quantize_rows and cubic_block_gemm; there is no eager fallback.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import torch
from torch import Tensor

from . import _native
from .adapters import _overlap
from .linear import DTYPE_IDS, MAX_GROUP_MEMBERS, PackedOperatorBinding, operand_identity

BLOCK = 128            # columns (and rows of a weight) that share a scale
E4M3 = torch.float8_e4m3fn
TOP = 448.0            # the largest e4m3 value
SMALLEST = 2.0 ** -96  # a group's largest magnitude counts as at least this
OUTPUT_IDS = {**DTYPE_IDS, torch.float32: 2}


def _blocks(size: int) -> int:
    return (size + BLOCK - 1) // BLOCK


def _row_major(t: Tensor) -> bool:
    """A matrix of contiguous rows at a stride of at least their length."""
    return (t.ndim == 2 and min(t.shape) >= 1 and (t.stride(1) == 1 or t.shape[1] == 1)
            and (t.stride(0) >= t.shape[1] or t.shape[0] == 1))


def _apart(scales: Tensor) -> bool:
    """Whether the [rows, groups] scales have places of their own."""
    (rows, groups), (row, group) = scales.shape, scales.stride()
    return ((rows == 1 or row >= 1) and (groups == 1 or group >= 1)
            and (rows == 1 or groups == 1 or row > (groups - 1) * group or group > (rows - 1) * row))


@dataclass(frozen=True, slots=True)
class BlockScaledActivations:
    """``values`` e4m3 [m, k] (rows may be padded) that stand for values * scales,
    ``scales`` float32 [m, ceil(k / 128)] of any positive strides."""

    values: Tensor
    scales: Tensor

    def __post_init__(self):
        self.check()

    def check(self) -> None:
        """Whether the scales are those of the values' extents, which a launch reads
        (a tensor may have been given other memory since)."""
        if not isinstance(self.values, Tensor) or not isinstance(self.scales, Tensor):
            raise TypeError("block-scaled activations are two tensors")
        if self.values.dtype is not E4M3 or not _row_major(self.values):
            raise ValueError("block-scaled activations need row-major float8_e4m3fn [M, K] values")
        if (self.scales.dtype is not torch.float32
                or self.scales.shape != (self.values.shape[0], _blocks(self.values.shape[1]))
                or not _apart(self.scales) or self.scales.device != self.values.device):
            raise ValueError("block-scaled activations need float32 [M, ceil(K / 128)] scales on the values' device")

    @classmethod
    def empty(cls, m: int, k: int, device: torch.device | str = "cuda") -> "BlockScaledActivations":
        """Buffers for ``m`` rows: rows of whole 16 bytes, a block's scales of all rows side by side."""
        if type(m) is not int or type(k) is not int or m < 1 or k < 1:
            raise ValueError("block-scaled activations need positive extents")
        values = torch.empty((m, (k + 15) // 16 * 16), dtype=E4M3, device=device)
        return cls(values[:, :k], torch.empty((_blocks(k), m), dtype=torch.float32, device=device).t())

    def dequantize(self) -> Tensor:
        """The values it stands for, float32."""
        return self.values.float() * self.scales.repeat_interleave(BLOCK, 1)[:, :self.values.shape[1]]


@dataclass(frozen=True, slots=True, eq=False)
class BlockScaledMatrix:
    """A weight: ``values`` e4m3 [n, k], ``scales`` float32 [ceil(n / 128), ceil(k / 128)],
    which multiply (checkpoints call them inverse scales)."""

    values: Tensor
    scales: Tensor

    def __post_init__(self):
        self.check()

    def check(self) -> None:
        """As BlockScaledActivations.check."""
        if not isinstance(self.values, Tensor) or not isinstance(self.scales, Tensor):
            raise TypeError("a block-scaled matrix is two tensors")
        if self.values.dtype is not E4M3 or not _row_major(self.values):
            raise ValueError("a block-scaled matrix needs row-major float8_e4m3fn [N, K] values")
        if (self.scales.dtype is not torch.float32
                or self.scales.shape != tuple(_blocks(d) for d in self.values.shape)
                or not self.scales.is_contiguous() or self.scales.device != self.values.device):
            raise ValueError("a block-scaled matrix needs contiguous float32 [ceil(N / 128), ceil(K / 128)] "
                             "scales on the values' device")

    @property
    def shape(self) -> tuple[int, int]:
        return tuple(self.values.shape)

    @property
    def device(self) -> torch.device:
        return self.values.device

    def to(self, device: torch.device | str) -> "BlockScaledMatrix":
        return BlockScaledMatrix(self.values.to(device), self.scales.to(device))

    def dequantize(self) -> Tensor:
        """The values it stands for, float32."""
        n, k = self.shape
        spread = self.scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        return self.values.float() * spread


@torch.no_grad()
def quantize_block_scaled(weight: Tensor) -> BlockScaledMatrix:
    """A matrix's nearest e4m3 values under each block's scale, the largest magnitude
    at 448 (load time, on the weight's device)."""
    if weight.ndim != 2 or min(weight.shape) < 1 or not weight.is_floating_point():
        raise ValueError("block scaling needs a positive floating-point [N, K] matrix")
    n, k = weight.shape
    values = torch.empty((n, k), dtype=E4M3, device=weight.device)
    scales = torch.empty((_blocks(n), _blocks(k)), dtype=torch.float32, device=weight.device)
    for row in range(0, n, 32 * BLOCK):  # bounds the 32-bit copy
        part = weight[row:row + 32 * BLOCK].float()
        rows = part.shape[0]
        tiles = torch.nn.functional.pad(part, (0, _blocks(k) * BLOCK - k, 0, _blocks(rows) * BLOCK - rows))
        tiles = tiles.view(_blocks(rows), BLOCK, _blocks(k), BLOCK)
        top = tiles.abs().amax((1, 3)).clamp_min(SMALLEST)
        scales[row // BLOCK:row // BLOCK + _blocks(rows)] = top / TOP
        scaled = (tiles * (TOP / top)[:, None, :, None]).view(_blocks(rows) * BLOCK, -1)
        values[row:row + rows] = scaled[:rows, :k].to(E4M3)
    return BlockScaledMatrix(values, scales)


# --------------------------------------------------------------------------- #
# bindings
# --------------------------------------------------------------------------- #
class _Launch:
    """One bound C call and the operands it came from.

    Addresses, extents and strides are those at bind time; a launch looks whether every
    operand still has them (1.6 us of the host's time for six).  Their memory is held, so no
    other tensor comes to it.
    """

    def __init__(self, name: str, operands: Sequence[Tensor], args: tuple, held: tuple = ()):
        self.held = (held, tuple(t.untyped_storage() for t in operands))
        with torch.cuda.device(operands[0].device):
            self._call = _native.BoundCall(name, *args)
        self._operands = tuple(operands)
        self._identity = operand_identity(self._operands)

    def validate(self) -> None:
        if operand_identity(self._operands) != self._identity:
            raise ValueError("packed launch operands changed after binding")

    def __call__(self, stream: int) -> None:
        self._call.launch(stream)


def _stride(t: Tensor) -> int:
    return max(t.stride(0), t.shape[1])  # a single row's stride means nothing


def _extent(t: Tensor) -> tuple[int, int]:
    size = t.element_size()
    return t.data_ptr(), t.data_ptr() + size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _shares(a: Tensor, b: Tensor) -> bool:
    """Whether two operands may share memory (interleaved columns of one matrix do not)."""
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    if a1 <= b0 or b1 <= a0:
        return False
    return _overlap(a, b) if _row_major(a) and _row_major(b) else True


def _same(a: Tensor, b: Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.dtype is b.dtype and (a.shape[0] == 1 or a.stride(0) == b.stride(0))


def _check_apart(outputs: Sequence[Tensor], inputs: Sequence[Tensor], in_place: Sequence[Tensor] = ()) -> None:
    """Outputs must not share memory with each other or an input, but for the
    inputs of ``in_place``, which an output may be as a whole."""
    for i, y in enumerate(outputs):
        if any(_shares(y, t) for t in (*outputs[:i], *inputs)) or any(_shares(y, t) and not _same(y, t) for t in in_place):
            raise ValueError("bound operator output must not alias its operands")


def _rows(t: Tensor | None, shape: tuple, dtype: torch.dtype, device: torch.device, what: str) -> None:
    if t is None:
        return
    if not isinstance(t, Tensor):
        raise TypeError(f"{what} must be a tensor")
    if t.shape != shape or t.dtype is not dtype or t.device != device or not _row_major(t):
        raise ValueError(f"{what} must be row-major {dtype} {list(shape)} on {device}")


def _activations(x: Tensor, what: str) -> None:
    if not isinstance(x, Tensor):
        raise TypeError(f"{what} must be a tensor")
    if x.dtype not in DTYPE_IDS or x.device.type != "cuda":
        raise ValueError(f"{what} requires CUDA FP16/BF16 activations")
    if not _row_major(x):
        raise ValueError(f"{what} requires positive row-major [M, K] activations")


def _quantized(q: BlockScaledActivations | None, shape: tuple, device: torch.device) -> tuple:
    """(operands, arguments) of an 8-bit output."""
    if q is None:
        return (), (None, 0, None, 0, 0)
    if not isinstance(q, BlockScaledActivations):
        raise TypeError("an 8-bit output must be BlockScaledActivations")
    q.check()
    if q.values.shape != shape or q.values.device != device:
        raise ValueError(f"an 8-bit output must be {list(shape)} on {device}")
    return (q.values, q.scales), (q.values.data_ptr(), _stride(q.values), q.scales.data_ptr(), *q.scales.stride())


def bind_norm(x: Tensor, weight: Tensor, *, epsilon: float, weight_offset: float = 0.0,
              residual: Tensor | None = None, residual_output: Tensor | None = None,
              output: Tensor | None = None, quantized: BlockScaledActivations | None = None) -> PackedOperatorBinding:
    """Bind ``y = h (weight_offset + weight) / sqrt(mean(h^2) + epsilon)``, ``h = x + residual``.

    ``output`` takes y in the inputs' type, ``quantized`` in 8 bits; one of them at
    least.  ``residual_output`` takes h; it may be the residual or x itself, and
    ``output`` too.  Everything is computed in 32 bits from h before its rounding.
    """
    _activations(x, "row norm")
    shape, device = tuple(x.shape), x.device
    _rows(residual, shape, x.dtype, device, "row norm residual")
    _rows(residual_output, shape, x.dtype, device, "row norm residual output")
    _rows(output, shape, x.dtype, device, "row norm output")
    if not isinstance(weight, Tensor):
        raise TypeError("row norm weight must be a tensor")
    if weight.shape != shape[1:] or weight.dtype is not x.dtype or weight.device != device or not weight.is_contiguous():
        raise ValueError(f"row norm weight must be contiguous {x.dtype} [{shape[1]}] on {device}")
    if output is None and quantized is None:
        raise ValueError("row norm needs an output")
    eight, eight_args = _quantized(quantized, shape, device)
    inputs = [t for t in (x, residual) if t is not None]
    outputs = [t for t in (residual_output, output) if t is not None]
    _check_apart((*outputs, *eight), [weight], inputs)
    given = lambda t: (None, 0) if t is None else (t.data_ptr(), _stride(t))
    args = (*given(x), *given(residual), weight.data_ptr(), *shape, DTYPE_IDS[x.dtype], float(epsilon),
            float(weight_offset), *given(output), *given(residual_output), *eight_args)
    launch = _Launch("cubic_row_norm", (*inputs, weight, *outputs, *eight), args)
    return _binding((output, quantized, residual_output), launch, device)


def bind_quantize(x: Tensor, quantized: BlockScaledActivations, *, gate: Tensor | None = None) -> PackedOperatorBinding:
    """Bind x, or ``silu(gate) * x``, to 8 bits; gate and x may be columns of one matrix."""
    _activations(x, "quantization")
    shape, device = tuple(x.shape), x.device
    _rows(gate, shape, x.dtype, device, "quantization gate")
    if quantized is None:
        raise TypeError("an 8-bit output must be BlockScaledActivations")
    eight, eight_args = _quantized(quantized, shape, device)
    inputs = [t for t in (x, gate) if t is not None]
    _check_apart(eight, inputs)
    args = (x.data_ptr(), _stride(x), *((None, 0) if gate is None else (gate.data_ptr(), _stride(gate))), *shape,
            DTYPE_IDS[x.dtype], *eight_args)
    return _binding((quantized,), _Launch("cubic_quantize_rows", (*inputs, *eight), args), device)


def _binding(results: Sequence, launch: _Launch, device: torch.device, scratch: tuple = ()) -> PackedOperatorBinding:
    given = tuple(r for r in results if r is not None)
    return PackedOperatorBinding(given[0] if len(given) == 1 else given, (launch,), scratch=scratch, device=device)


def prepare_block_matrix(weight: BlockScaledMatrix, device: torch.device | None = None) -> tuple[Tensor, Tensor]:
    """The values in the order in which the products read them, and the scales
    (load time, allocates)."""
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("block-scaled weights require cold preparation before capture")
    weight.check()
    device = torch.device(device) if device is not None else weight.device
    values = weight.values.to(device)
    n, k = weight.shape
    nbytes = _native.lib().cubic_block_prepared_bytes(n, k)
    if nbytes < 0:
        raise ValueError("block-scaled matrix geometry not admitted")
    with torch.cuda.device(device):
        prepared = torch.empty(nbytes, dtype=torch.uint8, device=device)
        scales = weight.scales.to(device, copy=True)
        _native.call("cubic_block_prepare", values.data_ptr(), _stride(values), n, k, prepared.data_ptr(),
                     _native.stream_of(device))
        torch.cuda.current_stream(device).synchronize()
    return prepared, scales


def bind_block_linear_group(operators, x: BlockScaledActivations, weights: Sequence[BlockScaledMatrix],
                            outputs: Sequence[Tensor]) -> PackedOperatorBinding:
    """Bind ``outputs[j] = x weights[j]^T`` in one launch.

    Outputs are bf16, fp16 or fp32 (one type for all) and may have padded rows.  Sums are
    in 32 bits for fp32; for 16-bit outputs the matrix instruction adds each eight products of
    consecutive columns at 14 bits below the largest, at most 7 * 2^-13 of the eight's largest
    |x| times its largest |w| off (1.5e-5 of y for normal operands).
    K has to be a multiple of 16, x 16-byte aligned with rows of whole 16 bytes.
    Weights are laid out as they are now (bindings of the same values share the layout);
    after a change to one, bind again.
    The binding owns its workspace, cleared on the current stream: a launch on
    another one has to follow it, and launches of one binding must not overlap.
    """
    weights, outputs = tuple(weights), tuple(outputs)
    if not 1 <= len(weights) <= MAX_GROUP_MEMBERS or len(weights) != len(outputs):
        raise ValueError(f"block-scaled linear needs 1..{MAX_GROUP_MEMBERS} weights with one output each")
    if not isinstance(x, BlockScaledActivations) or any(not isinstance(w, BlockScaledMatrix) for w in weights):
        raise TypeError("block-scaled linear requires BlockScaledActivations and BlockScaledMatrix")
    if any(not isinstance(y, Tensor) for y in outputs):
        raise TypeError("block-scaled linear outputs must be tensors")
    for operand in (x, *weights):
        operand.check()
    values, device = x.values, x.values.device
    m, k = values.shape
    if device.type != "cuda":
        raise ValueError("block-scaled linear requires CUDA activations")
    if k % 16 or values.data_ptr() % 16 or (m > 1 and values.stride(0) % 16):
        raise ValueError("block-scaled linear requires 16-byte aligned activations with K % 16 == 0")
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("block-scaled linears must be bound before graph capture")
    for w, y in zip(weights, outputs):
        if w.shape[1] != k:
            raise ValueError("bound linear weight K differs")
        if w.device != device and w.device.type != "cpu":
            raise ValueError("linear weights and activations must share one device")
        if (y.shape != (m, w.shape[0]) or y.dtype not in OUTPUT_IDS or y.dtype is not outputs[0].dtype
                or y.device != device or not _row_major(y)):
            raise ValueError("bound linear output has an invalid ABI")
    prepared = [operators.prepared_block(w, device) for w in weights]
    _check_apart(outputs, [values, x.scales, *(t for pair in prepared for t in pair)])
    c = _native.ctypes
    table = lambda ctype, items: (ctype * len(items))(*items)
    widths = table(c.c_int64, [w.shape[0] for w in weights])
    nbytes = _native.lib().cubic_block_gemm_workspace_bytes(m, k, len(weights), widths)
    if nbytes < 0:
        raise ValueError("block-scaled linear geometry not admitted")
    workspace = torch.zeros(nbytes, dtype=torch.uint8, device=device)
    args = (values.data_ptr(), _stride(values), x.scales.data_ptr(), *x.scales.stride(), m, k, len(weights), widths,
            table(c.c_void_p, [p.data_ptr() for p, _ in prepared]), table(c.c_void_p, [s.data_ptr() for _, s in prepared]), table(c.c_void_p, [y.data_ptr() for y in outputs]),
            table(c.c_int64, [_stride(y) for y in outputs]), OUTPUT_IDS[outputs[0].dtype], workspace.data_ptr(), nbytes)
    launch = _Launch("cubic_block_gemm", (values, x.scales, *outputs), args, held=(weights, prepared, workspace))
    return _binding(outputs, launch, device, scratch=(workspace,) if nbytes else ())
