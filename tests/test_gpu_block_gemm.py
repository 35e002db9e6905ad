"""GPU: block-scaled products against their formula in 64 bits.

Tolerance.  The matrix instruction adds eight products of consecutive k at a time, at
14 bits: with 2^E the largest product of the exponents' powers among them, what lies
below 2^(E - 13) of a product is cut.  (2^16 + 2^e over two places of eight keeps 2^e down
to e = 3 and loses it from e = 2 on; over two places of different eights down to e = -7.)  The
largest product's last bit is 2^(E - 6), so it is whole; each of the other seven is off by
less than 2^(E - 13), at most 2^-13 of the largest: 7 * 2^-13 of (largest |x| of the
eight) (largest |w| of the eight) bounds that.  The sums of eight are then added in 32
bits; were each addition truncated, 16 of them are off by 2^-19 of the sum of
magnitudes.  The scale is rounded, one addition per block and per wave follows, 2^-24 each,
and y is rounded once to its type.  Whole numbers whose products all lie above the cut
have exact sums, and those are compared for equality.
"""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import blockscale, linear
from test_blockscale_host import plan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = blockscale.E4M3
HALF_STEP = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}
LEAST = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -150}


def activations(m, k, seed, column_major=True, pad=0):
    """Random values and scales, rows at a stride of k + pad."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    values = (torch.randn((m, k + pad), generator=gen, device=DEV) * 60).to(E4M3)[:, :k]
    blocks = (k + 127) // 128
    scales = 0.01 + torch.rand((blocks, m), generator=gen, device=DEV)
    return blockscale.BlockScaledActivations(values, scales.t() if column_major else scales.t().contiguous())


def matrix(n, k, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    values = (torch.randn((n, k), generator=gen, device=DEV) * 60).to(E4M3)
    scales = 0.01 + torch.rand(((n + 127) // 128, (k + 127) // 128), generator=gen, device=DEV)
    return blockscale.BlockScaledMatrix(values, scales)


def wide(q):
    s = q.scales.double()
    if isinstance(q, blockscale.BlockScaledMatrix):
        s = s.repeat_interleave(128, 0)[:q.values.shape[0]]
    return q.values.double() * s.repeat_interleave(128, 1)[:, :q.values.shape[1]]


def largest_of_eight(a):
    """[rows, ceil(k / 8)] largest magnitudes of eight consecutive columns."""
    a = torch.nn.functional.pad(a.abs(), (0, -a.shape[1] % 8))
    return a.view(a.shape[0], -1, 8).amax(2)


def check(x, w, y, what=""):
    a, b = wide(x), wide(w)
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    cut = largest_of_eight(a) @ largest_of_eight(b).t()
    blocks = (x.values.shape[1] + 127) // 128
    bound = cut * 7 * 2.0 ** -13 + size * (2.0 ** -19 + (blocks + 20) * 2.0 ** -24) + want.abs() * HALF_STEP[y.dtype] + LEAST[y.dtype]
    off = (y.double() - want).abs()
    # past its largest number a type has the infinity of that sign
    over = torch.isinf(y) & (want.abs() + bound >= torch.finfo(y.dtype).max) & (y.sign() == want.sign())
    assert ((off <= bound) | over).all(), (what, (off / bound)[~over].max().item())


def product(x, weights, dtype=BF16, pad=0):
    m = x.values.shape[0]
    ys = [torch.full((m, w.shape[0] + pad), 7.0, dtype=dtype, device=DEV) for w in weights]
    linear.PackedLinearOperators().bind_block_linear_group(x, weights, [y[:, :w.shape[0]] for y, w in zip(ys, weights)]).launch()
    torch.cuda.synchronize()
    for y, w in zip(ys, weights):
        assert (y[:, w.shape[0]:] == 7).all()
    return [y[:, :w.shape[0]] for y, w in zip(ys, weights)]


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 130, 257])
@pytest.mark.parametrize("n,k", [(1, 16), (16, 128), (17, 144), (129, 256), (520, 2064), (1001, 1104)])
def test_product(m, n, k):
    print(f"block gemm m={m} n={n} k={k}", flush=True)
    x, w = activations(m, k, 1, column_major=m % 2 == 0, pad=16 * (m % 3)), matrix(n, k, 2)
    for dtype in (BF16, FP32):
        y, = product(x, [w], dtype, pad=m % 4)
        check(x, w, y, dtype)


@pytest.mark.parametrize("m", [1, 5, 40, 100, 300, 1500])
def test_group(m):
    """Members of any widths in one launch equal their own launches, bit for bit."""
    print(f"block gemm group m={m}", flush=True)
    k = 1168
    x = activations(m, k, 3)
    ws = [matrix(n, k, 4 + n) for n in (1000, 24, 1, 392, 128, 3000, 129, 77)]
    ys = product(x, ws, BF16)
    for w, y in zip(ws, ys):
        check(x, w, y)


@pytest.mark.parametrize("m,n,k", [(3, 5000, 4096), (64, 40000, 1024), (200, 33000, 512), (700, 2048, 8192), (1111, 3333, 1040), (2048, 1536, 2048),
                                   (64, 1024, 8192), (20, 3000, 12272), (100, 500, 6000), (17, 130, 4224)])
def test_larger(m, n, k):
    print(f"block gemm m={m} n={n} k={k}", flush=True)
    x, w = activations(m, k, 5), matrix(n, k, 6)
    y, = product(x, [w], FP16 if m == 200 else BF16)
    check(x, w, y)


@pytest.mark.parametrize("m", [1, 9, 17, 48, 80, 200, 513])
@pytest.mark.parametrize("n,k", [(1, 16), (17, 144), (300, 2096), (1000, 256), (2100, 1040), (700, 4400)])
def test_integers_are_exact(m, n, k):
    """Whole numbers and scales of powers of two: every sum is exact in 32 bits, no product cut."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    ints = lambda rows: torch.randint(-15, 16, (rows, k), generator=gen, device=DEV).float().to(E4M3)
    blocks = (k + 127) // 128
    power = lambda *shape: 2.0 ** torch.randint(0, 2, shape, generator=gen, device=DEV).float()
    x = blockscale.BlockScaledActivations(ints(m), power(m, blocks))
    w = blockscale.BlockScaledMatrix(ints(n), power((n + 127) // 128, blocks))
    y, = product(x, [w], FP32)
    assert torch.equal(y.double(), wide(x) @ wide(w).t())


@pytest.mark.parametrize("m,n,k", [(50, 65000, 4864), (128, 65000, 4864), (1, 66001, 4864), (7, 66001, 4864), (3, 20000, 16400)])
def test_weights_larger_than_the_cache(m, n, k):
    print(f"block gemm m={m} n={n} k={k}", flush=True)
    x, w = activations(m, k, 31, column_major=m == 50), matrix(n, k, 32)
    y, = product(x, [w], BF16)
    check(x, w, y)


@pytest.mark.parametrize("m,ns", [(200, [8100]), (1000, [8100]), (2050, [4000, 2001])])
@pytest.mark.parametrize("k", [16, 144, 272, 512, 528, 768, 784, 1168])
def test_every_number_of_blocks(m, ns, k):
    """Tiles of 128, 256 and 256 columns by 64, 128 and 256 rows go through K in rounds of three and four blocks."""
    print(f"block gemm m={m} ns={ns} k={k}", flush=True)
    x, ws = activations(m, k, 21, column_major=k % 32 == 0, pad=16 * (k % 3)), [matrix(n, k, 22 + n) for n in ns]
    for w, y in zip(ws, product(x, ws, BF16, pad=k % 5)):
        check(x, w, y)


@pytest.mark.parametrize("m", [2, 70, 400])
def test_values_at_the_edges(m):
    k, n = 272, 140
    x, w = activations(m, k, 8), matrix(n, k, 9)
    x.values[0] = 0
    x.scales[1, 1] = 0.0                  # a block under a scale of 0
    clean, = product(x, [w], FP32)
    check(x, w, clean)
    assert not clean[0].any()
    x.values[1, 200] = float("nan")       # one row
    y, = product(x, [w], FP32)
    assert torch.isnan(y[1]).all() and torch.equal(y[0], clean[0]) and torch.equal(y[2:], clean[2:])
    x, w = activations(m, k, 8), matrix(n, k, 9)
    w.values[3, 271] = float("nan")       # one column, the last of a short block
    w.scales[1, 0] = float("inf")         # the columns of a block
    y, = product(x, [w], FP32)
    assert torch.isnan(y[:, 3]).all() and not torch.isnan(y[:, :3]).any() and not torch.isfinite(y[:, 128:]).any()


def test_columns_past_k_are_not_read_as_numbers():
    """Rows whose padding holds NaN, K inside a block."""
    for m in (3, 90, 600):
        x = activations(m, 400, 10, pad=112)
        whole = x.values._base if x.values._base is not None else x.values
        whole[:, 400:] = float("nan")
        w = matrix(96, 400, 11)
        y, = product(x, [w])
        check(x, w, y)


@pytest.mark.parametrize("m", [4, 64, 300])
def test_rows_do_not_depend_on_their_neighbours(m):
    x, w = activations(m, 1024, 12), matrix(2000, 1024, 13)
    y, = product(x, [w])
    order = torch.randperm(m, generator=torch.Generator().manual_seed(1)).to(DEV)
    moved = blockscale.BlockScaledActivations(x.values.view(torch.uint8)[order].view(E4M3), x.scales[order])
    z, = product(moved, [w])
    assert torch.equal(z, y[order])


def test_captured_replayed_and_concurrent():
    m, n, k = 30, 3000, 4112  # K in parts that meet in the workspace
    x, w = activations(m, k, 14), matrix(n, k, 15)
    ops = linear.PackedLinearOperators()
    y, z = (torch.empty((m, n), dtype=BF16, device=DEV) for _ in range(2))
    one, two = ops.bind_block_linear(x, w, y), ops.bind_block_linear(x, w, z)
    assert len(ops.prepared_weights) == 1 and one.scratch and one.scratch[0].data_ptr() != two.scratch[0].data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):  # two launches at once
        one.launch()
        with torch.cuda.stream(side):
            two.launch()
    torch.cuda.synchronize()
    check(x, w, y)
    assert torch.equal(y, z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.launch()
    for turn in range(3):
        other = activations(m, k, 20 + turn)
        x.values.copy_(other.values), x.scales.copy_(other.scales)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(x, w, y)
        two.launch()
        torch.cuda.synchronize()
        assert torch.equal(y, z)
    assert not one.scratch[0][:4 * ((n + 63) // 64)].any()  # the counters


def test_weights_changed_later_are_prepared_again():
    x, w = activations(4, 256, 16), matrix(64, 256, 17)
    ops = linear.PackedLinearOperators()
    y = torch.empty((4, 64), dtype=FP32, device=DEV)
    ops.bind_block_linear(x, w, y).launch()
    check(x, w, y)
    w.values.copy_(matrix(64, 256, 18).values)
    w.scales.mul_(2)
    ops.bind_block_linear(x, w, y).launch()
    check(x, w, y)


def test_norm_quantize_product_chain():
    """norm -> q, k, v; gate and up -> gated activations -> down, as a layer has them."""
    m, hidden, inter = 21, 512, 1040
    gen = torch.Generator(device=DEV).manual_seed(19)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    x, r = normal(m, hidden).to(BF16), normal(m, hidden).to(BF16)
    weight = (1 + 0.1 * normal(hidden)).to(BF16)
    gate_up = [blockscale.quantize_block_scaled(normal(inter, hidden) * 0.05) for _ in range(2)]
    down = blockscale.quantize_block_scaled(normal(hidden, inter) * 0.05)
    ops = linear.PackedLinearOperators()
    a, b = blockscale.BlockScaledActivations.empty(m, hidden, DEV), blockscale.BlockScaledActivations.empty(m, inter, DEV)
    both, y = torch.empty((m, 2 * inter), dtype=BF16, device=DEV), torch.empty((m, hidden), dtype=BF16, device=DEV)
    gate, up = both[:, :inter], both[:, inter:]
    for binding in (ops.bind_norm(x, weight, epsilon=1e-6, residual=r, residual_output=r, quantized=a),
                    ops.bind_block_linear_group(a, gate_up, (gate, up)), ops.bind_quantize(up, b, gate=gate),
                    ops.bind_block_linear(b, down, y)):
        binding.launch()
    torch.cuda.synchronize()
    check(a, gate_up[0], gate)
    check(a, gate_up[1], up)
    check(b, down, y)


def test_refusals():
    ops = linear.PackedLinearOperators()
    x, w = activations(4, 256, 21), matrix(64, 256, 22)
    y = torch.empty((4, 64), dtype=BF16, device=DEV)
    bad = [(activations(4, 250, 23, pad=6), matrix(64, 250, 24), y, "K % 16"), (x, matrix(64, 272, 24), y, "K differs"),
           (activations(4, 256, 23, pad=8), w, y, "16-byte"), (x, w, y[:3], "ABI"), (x, w, y.double(), "ABI"), (x, w, y.t(), "ABI")]
    for a, b, c, match in bad:
        with pytest.raises(ValueError, match=match):
            ops.bind_block_linear(a, b, c)
    with pytest.raises(ValueError, match="alias"):
        ops.bind_block_linear_group(x, (w, w), (y, y))
    with pytest.raises(ValueError, match="ABI"):
        ops.bind_block_linear_group(x, (w, w), (y, torch.empty((4, 64), device=DEV)))
    with pytest.raises(ValueError, match="weights"):
        ops.bind_block_linear_group(x, (w,) * 9, (y,) * 9)
    with pytest.raises(TypeError):
        ops.bind_block_linear(x.values, w, y)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="before graph capture"):
            ops.bind_block_linear(x, w, y)


def test_weights_written_past_autograd_are_prepared_again():
    """Through .data, into an inference tensor: no version counts these."""
    x, w = activations(4, 256, 41), matrix(64, 256, 42)
    ops = linear.PackedLinearOperators()
    y = torch.empty((4, 64), dtype=FP32, device=DEV)
    ops.bind_block_linear(x, w, y).launch()
    other = matrix(64, 256, 43)
    for change in (lambda: w.values.data.copy_(other.values), lambda: w.scales.data.mul_(2),
                   lambda: setattr(w.values, "data", matrix(64, 256, 44).values), lambda: setattr(w.scales, "data", w.scales * 3)):
        change()
        ops.bind_block_linear(x, w, y).launch()
        check(x, w, y)
        assert len(ops.prepared_weights) == 1
    with torch.inference_mode():
        w = matrix(64, 256, 45)
        ops.bind_block_linear(x, w, y).launch()
        w.values.copy_(other.values)
        w.scales.mul_(0.5)
        ops.bind_block_linear(x, w, y).launch()
    check(x, w, y)


@pytest.mark.parametrize("m,n,k", [(1, 300, 272), (3, 17000, 400), (8, 33000, 144), (9, 300, 1168), (64, 4000, 4112), (100, 1000, 2064),
                                   (300, 12000, 272), (1000, 8192, 144), (2050, 4000, 528), (1, 66001, 4864), (60, 65000, 4864), (130, 520, 16)])
def test_outputs_in_32_bits_hold_every_product(m, n, k):
    """Products of 1 to 2^16 beside each other, large ones that cancel among them; whole sums below 2^24, which
    additions in 32 bits leave exact in any order.  (Per eight: 256 * 256, its negative, six of 1 to 225.)"""
    print(f"block gemm in 32 bits m={m} n={n} k={k}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(51)
    ints = lambda rows: torch.randint(-15, 16, (rows, k), generator=gen, device=DEV).float()
    a, b = ints(m), ints(n)
    a[:, 2::8], a[:, 5::8] = 256.0, -256.0
    b[:, 2::8] = b[:, 5::8] = 256.0
    blocks = (k + 127) // 128
    # (magnitudes: 16 * 2 * 2^16 + 96 * 225 in a block, under 2^22; the large ones cancel in pairs)
    x = blockscale.BlockScaledActivations(a.to(E4M3), torch.ones((m, blocks), device=DEV))
    w = blockscale.BlockScaledMatrix(b.to(E4M3), torch.full(((n + 127) // 128, blocks), 0.5, device=DEV))
    y, = product(x, [w], FP32, pad=m % 4)
    want = torch.cat([wide(x) @ part.t() for part in wide(w).split(8192)], 1)
    assert torch.equal(y.double(), want)


def check32(x, w, y):
    """In 32 bits: 128 products of a block, each exact, added in any order (127 additions, truncated: 2^-23 of the block's
    magnitudes each), scaled, and added to the sum block by block and wave by wave, at most blocks + 20 roundings of 2^-24."""
    a, b = wide(x), wide(w)
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    blocks = (x.values.shape[1] + 127) // 128
    bound = size * (127 * 2.0 ** -23 + (blocks + 20) * 2.0 ** -24) + want.abs() * 2.0 ** -24 + LEAST[FP32]
    off = (y.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()
    # Errors add at random: 128 of 2^-24 of partial sums near size / sqrt(128) are 2^-24 of size, a 250th of the bound.
    assert off.square().mean().sqrt() <= 0.01 * bound.square().mean().sqrt()


@pytest.mark.parametrize("m,n,k", [(1, 1000, 4096), (7, 20011, 1104), (33, 3000, 2064), (64, 40000, 1024), (512, 4096, 4096), (1111, 3333, 1040),
                                   (700, 9000, 8192), (64, 1024, 8192)])
def test_outputs_in_32_bits(m, n, k):
    x, w = activations(m, k, 53), matrix(n, k, 54)
    y, = product(x, [w], FP32)
    check32(x, w, y)


STREAM, T64, T128, T256, WIDE, PAIRED = range(6)  # kernels of cubic_block_gemm_launch_plan
OUTPUT_IDS = {BF16: 0, FP16: 1, FP32: 2}


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,n,k,kernel,split", [
    (5, 640, 1040, STREAM, 1), (100, 1024, 1040, T64, 1), (1000, 2048, 528, T128, 1), (1000, 8192, 528, T256, 1), (2000, 8192, 272, WIDE, 1),
    (100, 1024, 2064, PAIRED, 1), (100, 1024, 4112, PAIRED, 4),
    # weights that are read past the cache
    (5, 66048, 4864, T128, 1), (50, 65024, 4864, T128, 1), (120, 65024, 4864, T256, 1)])
def test_every_kernel_writes_whole_lines(m, n, k, kernel, split, dtype):
    """Rows of y that are whole lines of 128 bytes, in each type, through each kernel; the rows behind the last stay as they were."""
    print(f"block gemm lines m={m} n={n} k={k} {dtype}", flush=True)
    took = plan(m, k, [n], OUTPUT_IDS[dtype])[1:]
    assert took == (T256 if kernel == WIDE and dtype is FP32 else kernel, split)
    x, w = activations(m, k, 61, column_major=m % 2 == 0), matrix(n, k, 62)
    y = torch.full((m + 3, n), 7.0, dtype=dtype, device=DEV)
    linear.PackedLinearOperators().bind_block_linear(x, w, y[:m]).launch()
    torch.cuda.synchronize()
    assert y.data_ptr() % 128 == 0 and n * y.element_size() % 128 == 0
    assert (y[m:] == 7).all()
    check(x, w, y[:m], dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("m,k,ns", [(1, 1168, (1000, 24, 1, 392)), (5, 2064, (9000, 8000)), (40, 1168, (1000, 24, 392, 128)), (100, 1936, (1000, 24, 129, 77)),
                                    (40, 4240, (1000, 520, 77)), (300, 528, (3000, 2048)), (1000, 272, (8192, 1024)), (300, 4240, (1000, 24, 3000)),
                                    (2000, 272, (8192, 333))])
def test_members_of_a_group_and_their_own_launches(m, k, ns, dtype):
    """Through the same order of sums they are equal bit for bit: kernels that go through K in order, or the same one with
    the same partitions.  (A group of many columns may take another order than a narrow member by itself.)"""
    print(f"block gemm members m={m} k={k} ns={ns} {dtype}", flush=True)
    order = lambda widths: (lambda need, kernel, split: (kernel if kernel in (STREAM, PAIRED) else None, split))(*plan(m, k, widths, OUTPUT_IDS[dtype]))
    x, ws = activations(m, k, 63), [matrix(n, k, 64 + n) for n in ns]
    equal = 0
    for w, y in zip(ws, product(x, ws, dtype)):
        check(x, w, y)
        if order(ns) == order([w.shape[0]]):
            assert torch.equal(y, product(x, [w], dtype)[0])
            equal += 1
    assert equal or order(ns)[0] is None


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_every_code(dtype):
    """Each of the 256 codes times 1, the numbers below the normal ones among them: exact in every type."""
    codes = torch.arange(256, dtype=torch.uint8, device=DEV)
    values = torch.zeros((256, 256), dtype=torch.uint8, device=DEV)
    values[codes.long(), codes.long()] = codes
    w = blockscale.BlockScaledMatrix(torch.ones((20, 256), device=DEV).to(E4M3), torch.ones((1, 2), device=DEV))
    want = codes.view(E4M3).double()[:, None].expand(256, 20)
    for m in (8, 40, 256):  # few rows, tiles
        for first in range(0, 256 - m + 1, m):
            x = blockscale.BlockScaledActivations(values[first:first + m].view(E4M3), torch.ones((m, 2), device=DEV))
            y, = product(x, [w], dtype)
            assert torch.equal(y.double().nan_to_num(1e9), want[first:first + m].nan_to_num(1e9))
    # as weights, one code a column
    w = blockscale.BlockScaledMatrix(values.view(E4M3), torch.ones((2, 2), device=DEV))
    for m in (3, 70):
        x = blockscale.BlockScaledActivations(torch.ones((m, 256), device=DEV).to(E4M3), torch.ones((m, 2), device=DEV))
        y, = product(x, [w], dtype)
        assert torch.equal(y.double().nan_to_num(1e9), want[:, 0].expand(m, 256).nan_to_num(1e9))
