"""GPU: row norms and 8-bit activations against their formulas in 64 bits.

Tolerances.  h = x + r is rounded once (2^-24), the mean of squares is summed by
at most 32 additions per thread, 6 in the wave and 4 over the waves, its root halves
that, and three products and the weights' offset follow: at most 2^-18 of y in all
(u(y)); y in 16 bits adds half a step of its type, a 16-bit sum too.  A scale is off by u(y)
and its division, 2^-17 in all.  An e4m3 value is off by half a step, 2^-4 of it
(2^-10 below 2^-6), from a value that is off by 2^-16.  silu(g): the exponent t is off
by 2^-24 of 1 (its rest is added), exp2 and the reciprocal by 2^-22 each: within
u(y), also where exp(-g) is past the 32-bit numbers.
"""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import blockscale, linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16 = torch.bfloat16, torch.float16
HALF_STEP = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}
LEAST = {BF16: 2.0 ** -134, FP16: 2.0 ** -25}  # half a step below the normal numbers
U = 2.0 ** -18
OPS = linear.PackedLinearOperators()


def rows(m, k, dtype, seed, scale=1.0, pad=0):
    """[m, k] of N(0, scale) in rows of k + pad."""
    gen = torch.Generator().manual_seed(seed)
    whole = (torch.randn((m, k + pad), generator=gen) * scale).to(dtype).to(DEV)
    return whole[:, :k]


def norm_exact(x, r, w, eps, offset):
    h = x.double() + (r.double() if r is not None else 0)
    return h, h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * (offset + w.double())


def near16(got, want, what=""):
    bound = want.abs() * (HALF_STEP[got.dtype] + U) + LEAST[got.dtype]
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (what, (off / bound).max().item())


def near8(q, want):
    """Values and scales against the exact y."""
    values, scales = q.values.double(), q.scales.double()
    m, k = want.shape
    blocks = (k + 127) // 128
    padded = torch.nn.functional.pad(want, (0, blocks * 128 - k)).view(m, blocks, 128)
    top = padded.abs().amax(2).clamp_min(2.0 ** -96)
    assert ((scales - top / 448).abs() <= top / 448 * 2.0 ** -17).all()
    v = want * (448 / top).repeat_interleave(128, 1)[:, :k]
    bound = torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + v.abs() * 2.0 ** -16
    off = (values - v).abs()
    assert (off <= bound).all(), (off / bound).max().item()


SHAPES = [(1, 1), (3, 7), (5, 8), (2, 127), (4, 128), (3, 129), (7, 520), (2, 1024), (5, 1025), (1, 4096),
          (33, 2056), (2, 8192), (600, 8200), (3, 16384), (2, 20003), (2, 32768), (2, 32769), (1, 70000)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k", SHAPES)
def test_norm(m, k, dtype):
    print(f"norm m={m} k={k} {dtype}", flush=True)
    x, r, w = rows(m, k, dtype, 1), rows(m, k, dtype, 2, 3.0), rows(1, k, dtype, 3)[0].contiguous()
    y, s = torch.empty((m, k), dtype=dtype, device=DEV), torch.empty((m, k), dtype=dtype, device=DEV)
    q = blockscale.BlockScaledActivations.empty(m, k, DEV)
    for residual in (r, None):
        OPS.bind_norm(x, w, epsilon=1e-5, residual=residual, residual_output=s, output=y, quantized=q).launch()
        h, want = norm_exact(x, residual, w, 1e-5, 0.0)
        near16(s, h, "sum")
        near16(y, want, "y")
        near8(q, want)


@pytest.mark.parametrize("m,k", [(3, 100), (2, 1024), (9, 2056), (3, 40000)])
def test_norm_in_place_padded_offset(m, k):
    """Rows at strides that no vector fits, columns of one matrix, outputs over their inputs."""
    print(f"norm in place m={m} k={k}", flush=True)
    whole = rows(m, 2 * k + 3, BF16, 4, pad=2)
    x, r = whole[:, 1:1 + k], whole[:, k + 2:2 * k + 2]
    w = rows(1, k + 1, BF16, 5)[0][1:]
    h, want = norm_exact(x, r, w, 1e-6, 1.0)
    around = whole.clone()
    q = blockscale.BlockScaledActivations(torch.zeros((m, k + 5), dtype=blockscale.E4M3, device=DEV)[:, 3:3 + k],
                                          torch.zeros((m, (k + 127) // 128 + 1), device=DEV)[:, 1:])
    OPS.bind_norm(x, w, epsilon=1e-6, weight_offset=1.0, residual=r, residual_output=r, output=x, quantized=q).launch()
    near16(x, want)
    near16(r, h)
    near8(q, want)
    for c in (0, k + 1, 2 * k + 2):  # what lies between the columns
        assert torch.equal(whole[:, c], around[:, c])


def test_norm_values_at_the_edges():
    k = 384
    x = rows(6, k, FP16, 6)
    x[0] = 0
    x[1, :128] = 0                      # a group of zeros beside others
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4] = 2.0 ** -24                   # the least numbers
    w = torch.ones(k, dtype=FP16, device=DEV)
    q, y = blockscale.BlockScaledActivations.empty(6, k, DEV), torch.empty_like(x)
    OPS.bind_norm(x, w, epsilon=1e-6, output=y, quantized=q).launch()
    _, want = norm_exact(x, None, w, 1e-6, 0.0)
    assert not y[0].any() and not q.values[0].float().any() and torch.isfinite(q.scales[:2]).all()
    assert not q.values[1, :128].float().any()
    assert torch.isnan(y[2]).all() and torch.isnan(q.dequantize()[2]).all()
    assert torch.isnan(y[3, 7]) and not y[3, :7].any()  # inf / inf, and finite / inf
    for r in (1, 4, 5):
        near16(y[r:r + 1], want[r:r + 1])
    near8(blockscale.BlockScaledActivations(q.values[4:], q.scales[4:]), want[4:])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 120), (4, 128), (9, 136), (2, 777), (70, 2048), (3, 2056), (129, 4104), (2, 20001)])
def test_quantize(m, k, dtype):
    print(f"quantize m={m} k={k} {dtype}", flush=True)
    both = rows(m, 2 * k, dtype, 7, 3.0)
    gate, up = both[:, :k], both[:, k:]
    q = blockscale.BlockScaledActivations.empty(m, k, DEV)
    OPS.bind_quantize(up, q).launch()
    near8(q, up.double())
    OPS.bind_quantize(up, q, gate=gate).launch()
    g = gate.double()
    near8(q, g / (1 + torch.exp(-g)) * up.double())


def test_quantize_values_at_the_edges():
    k = 256
    up, gate = torch.ones((5, k), dtype=BF16, device=DEV), torch.ones((5, k), dtype=BF16, device=DEV)
    gate[0] = torch.linspace(-200, 200, k)      # exp(-g) overflows on one side and vanishes on the other
    up[1, 3] = float("nan")                     # its group, not the next
    up[2, 130] = float("-inf")
    up[3] = torch.finfo(BF16).max
    up[4] = torch.finfo(BF16).tiny
    q = blockscale.BlockScaledActivations.empty(5, k, DEV)
    OPS.bind_quantize(up, q, gate=gate).launch()
    g = gate.double()
    near8(blockscale.BlockScaledActivations(q.values[:1], q.scales[:1]), (g / (1 + torch.exp(-g)) * up.double())[:1])
    got = q.dequantize()
    assert torch.isnan(got[1, :128]).all() and torch.isfinite(got[1, 128:]).all()
    assert torch.isnan(got[2, 128:]).all() and torch.isfinite(got[2, :128]).all()
    assert torch.isfinite(got[3]).all() and (got[3] > 0).all()
    assert torch.isfinite(got[4]).all() and (q.scales[4].double() == 2.0 ** -96 / 448).logical_or(
        (q.scales[4].double() - 2.0 ** -96 / 448).abs() <= 2.0 ** -96 / 448 * 2.0 ** -23).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k", [(3, 5), (5, 8), (4, 135), (2, 1032), (6, 4104), (2, 9161), (2, 33000)])
def test_any_alignment(m, k, dtype):
    """Operands that begin at any element, in rows of odd strides, whose neighbours stay as they are."""
    print(f"alignment m={m} k={k} {dtype}", flush=True)

    def inside(offset, pad, kind=dtype):
        whole = torch.full((m, k + pad), 7.0, device=DEV).to(kind)
        return whole, whole[:, offset:offset + k]

    x, r = rows(m, k, dtype, 41, pad=3), inside(1, 5)[1].copy_(rows(m, k, dtype, 42))
    w = rows(1, k + 1, dtype, 43)[0, 1:]
    (all_y, y), (all_s, s), (all_q, values) = inside(3, 4), inside(5, 7), inside(1, 2, blockscale.E4M3)
    q = blockscale.BlockScaledActivations(values, torch.empty((m, (k + 127) // 128), device=DEV))
    OPS.bind_norm(x, w, epsilon=1e-5, residual=r, residual_output=s, output=y, quantized=q).launch()
    h, want = norm_exact(x, r, w, 1e-5, 0.0)
    near16(s, h, "sum")
    near16(y, want, "y")
    near8(q, want)
    for whole, part in ((all_y, 3), (all_s, 5), (all_q, 1)):
        assert (whole[:, :part].float() == 7).all() and (whole[:, part + k:].float() == 7).all()
    OPS.bind_quantize(x, q, gate=r).launch()
    g = r.double()
    near8(q, g / (1 + torch.exp(-g)) * x.double())
    assert (all_q[:, :1].float() == 7).all() and (all_q[:, 1 + k:].float() == 7).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k", [(131200, 128), (33000, 520), (16500, 1017), (4200, 4097), (2100, 8200), (520, 32768), (250, 70001)])
def test_outputs_past_the_caches(m, k, dtype):
    print(f"large m={m} k={k} {dtype}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(51)
    x, r = (torch.randn((m, k), generator=gen, device=DEV).to(dtype) for _ in range(2))
    w = rows(1, k, dtype, 52)[0].contiguous()
    y, s = torch.empty_like(x), torch.empty_like(x)
    q = blockscale.BlockScaledActivations.empty(m, k, DEV)
    OPS.bind_norm(x, w, epsilon=1e-5, residual=r, residual_output=s, output=y, quantized=q).launch()
    h, want = norm_exact(x, r, w, 1e-5, 0.0)
    near16(s, h, "sum")
    near16(y, want, "y")
    near8(q, want)
    OPS.bind_quantize(x, q, gate=r).launch()
    g = r.double()
    near8(q, g / (1 + torch.exp(-g)) * x.double())


def test_gates_far_below_zero():
    """silu(g) is below the 32-bit numbers, its product with x is not.  (Products by powers of two, exact, and
    silu's error as above: u(y).)"""
    gate = torch.linspace(-170, -60, 23)[:, None].repeat(1, 128).to(BF16).to(DEV)
    gate[:, 1::2] += 3
    gate[0, 0::2], gate[1] = 3.3e38, -3.3e38
    for x in (2.0 ** 127, 2.0 ** 40, 1.0):
        up = torch.full_like(gate, x)
        up[0] = 1.0
        q = blockscale.BlockScaledActivations.empty(*gate.shape, DEV)
        OPS.bind_quantize(up, q, gate=gate).launch()
        g = gate.double()
        near8(q, g / (1 + torch.exp(-g)) * up.double())


def test_rows_that_lie_far_apart():
    """The second row starts past 2^31 elements of the first."""
    k, stride = 200, (1 << 31) + 16
    whole = torch.empty(stride + k, dtype=BF16, device=DEV)
    x = whole.as_strided((2, k), (stride, 1))
    x.copy_(rows(2, k, BF16, 8))
    y, q = torch.empty((2, k), dtype=BF16, device=DEV), blockscale.BlockScaledActivations.empty(2, k, DEV)
    w = torch.ones(k, dtype=BF16, device=DEV)
    _, want = norm_exact(x, None, w, 1e-6, 0.0)
    OPS.bind_norm(x, w, epsilon=1e-6, output=y, quantized=q).launch()
    near16(y, want)
    near8(q, want)
    OPS.bind_quantize(x, q).launch()
    near8(q, x.double())


def test_many_short_rows():
    """More rows than workgroups of one launch: a head's norm over many tokens."""
    m, k = (1 << 20) + 5, 64
    gen = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn((m, k), generator=gen, device=DEV).to(BF16)
    y, q, w = torch.empty_like(x), blockscale.BlockScaledActivations.empty(m, k, DEV), torch.ones(k, dtype=BF16, device=DEV)
    OPS.bind_norm(x, w, epsilon=1e-6, output=y, quantized=q).launch()
    _, want = norm_exact(x, None, w, 1e-6, 0.0)
    near16(y, want)
    near8(q, want)
    OPS.bind_quantize(x, q).launch()
    near8(q, x.double())


def test_captured_and_replayed_on_another_stream():
    m, k = 40, 2056
    x, r, w = rows(m, k, BF16, 10), rows(m, k, BF16, 11), rows(1, k, BF16, 12)[0].contiguous()
    y, s = torch.empty((m, k), dtype=BF16, device=DEV), torch.empty((m, k), dtype=BF16, device=DEV)
    q = blockscale.BlockScaledActivations.empty(m, k, DEV)
    norm = OPS.bind_norm(x, w, epsilon=1e-6, residual=r, residual_output=s, output=y)
    quantize = OPS.bind_quantize(y, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm.launch(), quantize.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm.launch(), quantize.launch()
    for turn in range(3):
        x.copy_(rows(m, k, BF16, 20 + turn))
        y.zero_(), s.zero_(), q.scales.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone(), s.clone(), q.values.float(), q.scales.clone()
        norm.launch(), quantize.launch()
        torch.cuda.synchronize()
        for a, b in zip(got, (y, s, q.values.float(), q.scales)):
            assert torch.equal(a, b)
        near16(y, norm_exact(x, r, w, 1e-6, 0.0)[1])
        near8(q, y.double())


def test_operands_changed_after_binding():
    x, w = rows(2, 64, BF16, 13), torch.ones(64, dtype=BF16, device=DEV)
    y = torch.empty_like(x)
    binding = OPS.bind_norm(x, w, epsilon=1e-6, output=y)
    y.resize_((2, 32))
    with pytest.raises(ValueError, match="changed after binding"):
        binding.launch()


def test_refusals():
    x, w = rows(4, 64, BF16, 14), torch.ones(64, dtype=BF16, device=DEV)
    y, q = torch.empty_like(x), blockscale.BlockScaledActivations.empty(4, 64, DEV)
    bad = [(dict(x=x.float()), "FP16/BF16"), (dict(x=x.t()), "row-major"), (dict(weight=w.half()), "weight"),
           (dict(weight=w[:63]), "weight"), (dict(output=None), "output"), (dict(output=y.half()), "output"),
           (dict(residual=x[:3]), "residual"), (dict(residual_output=y), "alias"), (dict(output=x[:, :1].expand(4, 64)), "output"),
           (dict(quantized=blockscale.BlockScaledActivations.empty(4, 65, DEV)), "8-bit"), (dict(epsilon=float("nan")), "epsilon"),
           (dict(epsilon=-1.0), "epsilon"), (dict(weight_offset=float("inf")), "epsilon|offset")]
    for change, match in bad:
        args = dict(x=x, weight=w, output=y, epsilon=1e-6) | change
        with pytest.raises(ValueError, match=match):
            OPS.bind_norm(args.pop("x"), args.pop("weight"), **args).launch()
    big = torch.empty((5, 64), dtype=BF16, device=DEV)
    with pytest.raises(ValueError, match="alias"):  # a row below its input
        OPS.bind_norm(big[:4], w, epsilon=1e-6, output=big[1:])
    with pytest.raises(ValueError, match="alias"):
        OPS.bind_quantize(x, blockscale.BlockScaledActivations(x.view(torch.uint8).view(blockscale.E4M3)[:, :64], q.scales))
    with pytest.raises(TypeError):
        OPS.bind_quantize(x, y)
    with pytest.raises(ValueError, match="gate"):
        OPS.bind_quantize(x, q, gate=x[:, :63])


def transposed(t):
    t.t_()


def narrowed(t):
    t.as_strided_((t.shape[0] // 2, 2 * t.shape[1]), (t.stride(0), 1)) if t.stride(0) >= 2 * t.shape[1] else t.as_strided_(
        (2 * t.shape[0], t.shape[1] // 2), (t.shape[1] // 2, 1))


def retyped(t):
    t.data = t.view({BF16: FP16, torch.float32: torch.int32, blockscale.E4M3: torch.uint8}[t.dtype])


@pytest.mark.parametrize("name,change", [(name, change) for name in ("x", "residual", "output", "values", "scales")
                                         for change in (transposed, narrowed, retyped) if (name, change) != ("scales", narrowed)])
def test_operands_with_another_layout_after_binding(name, change):
    """The same memory and number of elements, read another way."""
    k = 64
    t = {n: torch.ones((k, k), dtype=BF16, device=DEV) for n in ("x", "residual", "output")}
    t["values"], t["scales"] = torch.zeros((k, k), dtype=blockscale.E4M3, device=DEV), torch.zeros((k, 4), device=DEV)[:, :1]
    w = torch.ones(k, dtype=BF16, device=DEV)
    bindings = (OPS.bind_norm(t["x"], w, epsilon=1e-6, residual=t["residual"], output=t["output"],
                              quantized=blockscale.BlockScaledActivations(t["values"], t["scales"])),
                OPS.bind_quantize(t["x"], blockscale.BlockScaledActivations(t["values"], t["scales"]), gate=t["residual"]))
    change(t[name])
    for binding in bindings[:1] if name == "output" else bindings:
        with pytest.raises(ValueError, match="changed after binding"):
            binding.launch()


@pytest.mark.parametrize("k", [1 << 24, (1 << 21) + 8, 1 << 17])
def test_norm_of_the_longest_rows(k):
    """Equal squares of 1 + 2^-6 + 2^-14, whose last part a plain running sum loses from 2^10 on; a thread of a row that is
    read twice adds 8 squares, and these eights with the rounding carried over, so the bound above holds at any length."""
    x = torch.full((2, k), 1 + 2.0 ** -7, dtype=BF16, device=DEV)
    x[1] = rows(1, k, BF16, 61)[0]
    w = torch.ones(k, dtype=BF16, device=DEV)
    y, q = torch.empty_like(x), blockscale.BlockScaledActivations.empty(2, k, DEV)
    for value in (float("inf"), float("nan")):  # finite / inf, inf / inf
        other = x.clone()
        other[0, 5] = value
        OPS.bind_norm(other, w, epsilon=1e-6, output=y).launch()
        assert torch.isnan(y[0, 5]) and ((y[0] == 0).sum() == k - 1 if value > 0 else torch.isnan(y[0]).all())
        near16(y[1:], norm_exact(other[1:], None, w, 1e-6, 0.0)[1])
    OPS.bind_norm(x, w, epsilon=1e-6, output=y, quantized=q).launch()
    _, want = norm_exact(x, None, w, 1e-6, 0.0)
    near16(y, want)
    near8(q, want)


@pytest.mark.parametrize("k", [100, 1000, 4096, 10000, 20003, 70000])
def test_squares_that_leave_the_32_bit_numbers(k):
    """Rows whose squares are past 2^128, or below 2^-126 under an epsilon that is as small; beside them ordinary rows,
    rows of zeros, one large number among ordinary ones.  Scaling by a power of two rounds nothing but numbers that it takes
    below 2^-126 (below 2^-46 in a row past 2^52, whose y is under 2^-98; none here), so u(y) holds."""
    x = rows(8, k, BF16, 71)
    for row, scale in enumerate((2.0 ** 100, 2.0 ** 70, 2.0 ** -70, 2.0 ** -110, 1.0, 2.0 ** -60, 1.0, 0.0)):
        x[row] *= scale
    x[6, k // 2] = 3e38
    r, w = torch.zeros_like(x), (1 + 0.1 * rows(1, k, BF16, 72)[0]).to(BF16)
    r[:5] = x[:5].flip(1) * 0.5
    y, s, q = torch.empty_like(x), torch.empty_like(x), blockscale.BlockScaledActivations.empty(8, k, DEV)
    for epsilon in (0.0, 1e-38, 2.0 ** -90, 1e-6):
        OPS.bind_norm(x, w, epsilon=epsilon, residual=r, residual_output=s, output=y, quantized=q).launch()
        h, want = norm_exact(x, r, w, torch.tensor(epsilon, dtype=torch.float32).double().item(), 0.0)
        near16(s, h, "sum")
        some = 8 if epsilon else 7  # 0 / sqrt(0) is no number
        near16(y[:some], want[:some], epsilon)
        near8(blockscale.BlockScaledActivations(q.values[:some], q.scales[:some]), want[:some])
        if not epsilon:
            assert torch.isnan(y[7]).all()
