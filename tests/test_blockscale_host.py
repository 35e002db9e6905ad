"""CPU: block-scaled types, quantisation of weights, and what the C entries refuse
before anything is launched."""
from __future__ import annotations

import pytest
import torch

from cubic_serve_amd import _native, blockscale, linear

E4M3 = blockscale.E4M3


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 257), (4100, 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantized_matrix_is_within_half_a_step(n, k, dtype):
    w = (torch.randn((n, k), generator=torch.Generator().manual_seed(1)) * 0.1).to(dtype)
    w[:, 0] = 0
    m = blockscale.quantize_block_scaled(w)
    assert m.shape == (n, k) and m.scales.shape == ((n + 127) // 128, (k + 127) // 128)
    scale = m.scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    v = w.double() / scale
    # half a step of e4m3, and three roundings in 32 bits (top / 448, 448 / top, their product)
    bound = torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + v.abs() * 2.0 ** -21
    assert ((m.values.double() - v).abs() <= bound).all()
    assert torch.equal(m.dequantize(), m.values.float() * scale.float())


def test_quantized_matrix_of_zeros():
    m = blockscale.quantize_block_scaled(torch.zeros((130, 130)))
    assert not m.values.float().any() and torch.isfinite(m.scales).all() and (m.scales > 0).all()


def test_types_check_their_tensors():
    v, s = torch.zeros((4, 256), dtype=E4M3), torch.ones((4, 2))
    q = blockscale.BlockScaledActivations(v, s)
    assert torch.equal(q.dequantize(), torch.zeros((4, 256)))
    blockscale.BlockScaledActivations(v, torch.ones((2, 4)).t())
    for values, scales in ((v.float(), s), (v, s.double()), (v, s[:, :1]), (v, s[:1].expand(4, 2)), (v.t(), s), (v[0], s)):
        with pytest.raises(ValueError):
            blockscale.BlockScaledActivations(values, scales)
    blockscale.BlockScaledMatrix(v, torch.ones((1, 2)))
    for values, scales in ((v, s), (v, torch.ones((1, 2)).double()), (v.float(), torch.ones((1, 2))),
                           (v, torch.ones((2, 1)).expand(2, 2)[:1].t())):
        with pytest.raises(ValueError):
            blockscale.BlockScaledMatrix(values, scales)
    with pytest.raises(TypeError):
        blockscale.BlockScaledActivations(v, None)
    for m, k in ((0, 4), (4, 0), (2.0, 4)):
        with pytest.raises(ValueError):
            blockscale.BlockScaledActivations.empty(m, k, "cpu")
    e = blockscale.BlockScaledActivations.empty(3, 130, "cpu")
    assert e.values.shape == (3, 130) and e.values.stride(0) == 144 and e.scales.stride() == (1, 3)
    for bad in (torch.zeros(4), torch.zeros((0, 4)), torch.zeros((2, 2), dtype=torch.int32)):
        with pytest.raises(ValueError):
            blockscale.quantize_block_scaled(bad)


def test_bindings_need_a_gpu():
    ops = linear.PackedLinearOperators()
    x, w = torch.zeros((2, 64), dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    q = blockscale.BlockScaledActivations.empty(2, 64, "cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ops.bind_norm(x, w, epsilon=1e-6, output=x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.bind_quantize(x, q)
    with pytest.raises(ValueError, match="CUDA"):
        ops.bind_block_linear(q, blockscale.BlockScaledMatrix(torch.zeros((4, 64), dtype=E4M3), torch.ones((1, 1))), x)


def norm(**change):
    a = dict(x=16, ldx=64, r=None, ldr=0, w=16, m=2, k=64, dtype=0, eps=1e-6, off=0.0, y=16, ldy=64, s=None, lds=0,
             q=None, ldq=0, sc=None, row=0, group=0, bound=None, stream=None) | change
    return _native.call("cubic_row_norm", *a.values())


@pytest.mark.parametrize("change,match", [
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"), (dict(k=0), "k="), (dict(k=(1 << 24) + 1), "k="),
    (dict(m=0), "m="), (dict(m=1 << 31), "m="), (dict(dtype=2), "dtype"), (dict(ldx=63), "row stride"), (dict(ldy=63), "row stride"),
    (dict(r=16, ldr=63), "row stride"), (dict(eps=-1.0), "epsilon"), (dict(eps=float("nan")), "epsilon"),
    (dict(off=float("inf")), "epsilon"), (dict(x=17), "aligned"), (dict(w=17), "aligned"), (dict(q=16, ldq=64), "scales"),
    (dict(q=16, ldq=64, sc=18, row=1, group=2), "scales"), (dict(q=16, ldq=64, sc=16, row=0, group=1), "overlap"),
    (dict(q=16, ldq=256, sc=16, row=1, group=1, k=256, ldx=256, ldy=256), "overlap")])
def test_norm_entry_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        norm(**change)


@pytest.mark.parametrize("change,match", [
    (dict(q=None), "null"), (dict(x=None), "null"), (dict(k=0), "k="), (dict(m=0), "m="), (dict(ldg=3, g=16), "row stride"),
    (dict(ldq=63), "row stride"), (dict(dtype=7), "dtype"), (dict(sc=None), "scales")])
def test_quantize_entry_refuses(change, match):
    a = dict(x=16, ldx=64, g=None, ldg=0, m=2, k=64, dtype=0, q=16, ldq=64, sc=16, row=1, group=2, bound=None, stream=None) | change
    with pytest.raises(ValueError, match=match):
        _native.call("cubic_quantize_rows", *a.values())


@pytest.mark.parametrize("change,match", [
    (dict(x=None), "null"), (dict(sx=None), "null"), (dict(members=0), "members"), (dict(members=9), "members"), (dict(out=3), "dtype"),
    (dict(m=0), "extents"), (dict(m=1 << 21), "extents"), (dict(k=0), "extents"), (dict(k=1 << 21), "extents"),
    (dict(k=72), "k % 16"), (dict(ldx=120), "row stride"), (dict(ldx=1 << 24), "row stride"), (dict(x=24), "alignment"),
    (dict(row=0), "scale strides"), (dict(k=256, ldx=256, group=0), "scale strides"), (dict(n=0), "width"), (dict(n=(1 << 24) + 1), "width"),
    (dict(w=24), "misaligned"), (dict(w=None), "null operand of"), (dict(y=None), "null operand of"), (dict(y=17), "misaligned"),
    (dict(ldy=63), "leading dimension")])
def test_block_gemm_entry_refuses(change, match):
    a = dict(x=16, ldx=128, sx=16, row=1, group=2, m=2, k=128, members=1, n=64, w=16, sw=16, y=16, ldy=64, out=0) | change
    c = _native.ctypes
    one = lambda ctype, v: (ctype * 1)(v)
    with pytest.raises(ValueError, match=match):
        _native.call("cubic_block_gemm", a["x"], a["ldx"], a["sx"], a["row"], a["group"], a["m"], a["k"], a["members"],
                     one(c.c_int64, a["n"]), one(c.c_void_p, a["w"]), one(c.c_void_p, a["sw"]), one(c.c_void_p, a["y"]),
                     one(c.c_int64, a["ldy"]), a["out"], 16, 1 << 30, None, None)


def test_block_prepare_entry():
    lib = _native.lib()
    assert lib.cubic_block_prepared_bytes(16, 128) == 128 * 128
    assert lib.cubic_block_prepared_bytes(129, 129) == 4 * 128 * 128
    for n, k in ((0, 1), (1, 0), ((1 << 24) + 1, 1), (1, (1 << 20) + 1)):
        assert lib.cubic_block_prepared_bytes(n, k) == -1
        with pytest.raises(ValueError):
            _native.call("cubic_block_prepare", 16, 1 << 21, n, k, 16, None)
    for args in ((None, 128, 4, 128, 16), (16, 127, 4, 128, 16), (16, 128, 4, 128, 24), (16, 128, 4, 128, None)):
        with pytest.raises(ValueError):
            _native.call("cubic_block_prepare", *args, None)


def test_block_gemm_workspace():
    c, lib = _native.ctypes, _native.lib()
    need = lambda m, k, *ns: lib.cubic_block_gemm_workspace_bytes(m, k, len(ns), (c.c_int64 * len(ns))(*ns))
    assert need(1, 12288, 4096) == 0 and need(4096, 8192, 8192) == 0 and need(64, 2048, 4096) == 0
    # 64 tiles of 64 x 64 in four parts of K, and a counter each
    assert need(64, 12288, 4096) == 256 + 64 * 4 * 64 * 64 * 4
    assert need(0, 128, 64) == -1 and need(64, 0, 64) == -1 and need(64, 128, 0) == -1
    one = lambda ctype, v: (ctype * 1)(v)
    for workspace, nbytes, match in ((16, need(64, 12288, 4096) - 1, "workspace"), (None, 1 << 30, "aligned"), (24, 1 << 30, "aligned")):
        with pytest.raises(ValueError, match=match):
            _native.call("cubic_block_gemm", 16, 12288, 16, 96, 1, 64, 12288, 1, one(c.c_int64, 4096), one(c.c_void_p, 16),
                         one(c.c_void_p, 16), one(c.c_void_p, 16), one(c.c_int64, 4096), 0, workspace, nbytes, None, None)


def test_bound_calls():
    """A checked call is kept, not launched; what is no bound call is refused."""
    c, lib = _native.ctypes, _native.lib()
    nbytes = lib.cubic_bound_bytes()
    assert 0 < nbytes <= 4096
    memory = c.create_string_buffer(nbytes + 8)
    with pytest.raises(ValueError, match="not a bound call"):
        _native.call("cubic_launch_bound", c.addressof(memory), None)
    with pytest.raises(ValueError, match="not a bound call"):
        _native.call("cubic_launch_bound", None, None)
    assert norm(bound=c.addressof(memory)) == 0
    assert any(memory.raw)
    with pytest.raises(ValueError, match="aligned to 8"):
        norm(bound=c.addressof(memory) + 4)
    with pytest.raises(ValueError, match="epsilon"):
        norm(eps=-1.0, bound=c.addressof(memory))


def test_layouts_follow_their_weights(monkeypatch):
    """Writes that neither a version nor an address shows; one layout is kept per weight, and shared while it holds."""
    monkeypatch.setattr(blockscale, "prepare_block_matrix", lambda w, device: (w.values.clone().view(torch.uint8), w.scales.clone()))
    ops, device = linear.PackedLinearOperators(), torch.device("cpu")
    make = lambda v: torch.full((4, 256), v).to(E4M3)
    w = blockscale.BlockScaledMatrix(make(1.0), torch.ones((1, 2)))
    first = ops.prepared_block(w, device)
    assert ops.prepared_block(w, device) is first

    def inference(t):
        with torch.inference_mode():
            return t.clone()

    def write(t):
        with torch.inference_mode():
            t.copy_(make(6.0))

    changes = [lambda: w.values.copy_(make(2.0)), lambda: w.values.data.copy_(make(3.0)),
               lambda: setattr(w.values, "data", make(4.0)), lambda: w.scales.data.fill_(5.0),
               lambda: setattr(w.scales, "data", torch.full((1, 2), 6.0)), lambda: w.scales.data.fill_(float("nan"))]
    for change in changes:
        change()
        values, scales = ops.prepared_block(w, device)
        assert torch.equal(values, w.values.view(torch.uint8)) and torch.equal(scales.nan_to_num(-1), w.scales.nan_to_num(-1))
        assert ops.prepared_block(w, device)[0] is values  # NaNs too are the same
        assert len(ops.prepared_weights) == 1
    w = blockscale.BlockScaledMatrix(inference(make(5.0)), inference(torch.ones((1, 2))))
    ops.prepared_block(w, device)
    write(w.values)
    assert torch.equal(ops.prepared_block(w, device)[0], w.values.view(torch.uint8))


def test_tensors_that_grew_after_their_check():
    """A launch would read scales past their end."""
    make = lambda m: blockscale.BlockScaledActivations(torch.zeros((m, 64), dtype=E4M3), torch.ones((m, 1)))
    weight = lambda: blockscale.BlockScaledMatrix(torch.zeros((4, 64), dtype=E4M3), torch.ones((1, 1)))
    ops, y = linear.PackedLinearOperators(), torch.zeros((2, 4))
    for grown, other in ((lambda q: q.values, (300, 64)), (lambda q: q.scales, (1, 3))):
        x, w = make(2), weight()
        grown(x).data = torch.zeros(other, dtype=grown(x).dtype)
        for refused in (lambda: ops.bind_block_linear(x, w, y), lambda: blockscale._quantized(x, tuple(x.values.shape), x.values.device)):
            with pytest.raises(ValueError, match="scales"):
                refused()
        x = make(2)
        grown(w).data = torch.zeros(other, dtype=grown(w).dtype)
        for refused in (lambda: ops.bind_block_linear(x, w, y), lambda: blockscale.prepare_block_matrix(w)):
            with pytest.raises(ValueError, match="scales"):
                refused()


def plan(m, k, ns, out=0):
    """(workspace, kernel, K partitions) of a launch."""
    c = _native.ctypes
    kernel, split = c.c_int(), c.c_int()
    need = _native.lib().cubic_block_gemm_launch_plan(m, k, len(ns), (c.c_int64 * len(ns))(*ns), out, c.byref(kernel), c.byref(split))
    return need, kernel.value, split.value


def test_launch_plans():
    lib, c = _native.lib(), _native.ctypes
    assert plan(1, 4096, [6144]) == (0, 0, 1) and plan(4096, 8192, [8192]) == (0, 4, 1)
    assert plan(64, 12288, [4096])[1:] == (5, 4)
    ns = (c.c_int64 * 1)(4096)
    assert lib.cubic_block_gemm_launch_plan(64, 12288, 1, ns, 0, None, None) == plan(64, 12288, [4096])[0]
    for bad in ((0, 128, 1, ns, 0), (64, 0, 1, ns, 0), (64, 128, 0, ns, 0), (64, 128, 9, ns, 0), (64, 128, 1, None, 0), (64, 128, 1, ns, 3),
                (64, 128, 1, (c.c_int64 * 1)(0), 0)):
        assert lib.cubic_block_gemm_launch_plan(*bad, None, None) == -1
    # one workspace serves every type of output, and 32-bit ones never take the tile without registers for them
    for m in (1, 8, 9, 64, 100, 257, 1000, 4096):
        for k in (128, 1792, 4096, 12288):
            for widths in ([1], [520, 1001], [4096], [8192, 1024], [24576], [151936]):
                need, _, split = plan(m, k, widths)
                assert all(plan(m, k, widths, out)[::2] == (need, split) for out in (1, 2)) and plan(m, k, widths, 2)[1] != 4
                assert lib.cubic_block_gemm_workspace_bytes(m, k, len(widths), (c.c_int64 * len(widths))(*widths)) == need
