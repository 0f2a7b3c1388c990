"""The packers of the block-scaled linears on the CPU, against the formats'
definitions written out, and what the wrappers refuse."""
import ctypes
import itertools
import math

import pytest
import torch

from taomate_amd import _native, kernels, quant

from .helpers import gen, randn

BF = torch.bfloat16
E4M3 = sorted({s * v for s in (1, -1) for v in
               [m / 8 * 2.0 ** -6 for m in range(8)]
               + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)]})


def test_8bit_rows_are_the_nearest_values_under_the_smallest_scale():
    x = randn((3, 5, 96), gen(1)) * torch.exp(4 * randn((96,), gen(2)))
    x[0, 0, :32] = 0
    x[0, 1, 0] = 448.0
    x[0, 1, 1:32] = 1.0
    x[0, 2, 32:64] = 449.0
    q = quant.quantize_mx(x)
    assert q.shape == x.shape and q.scales.shape == (1, 15, 4) and q.codes.dtype == torch.float8_e4m3fn
    grid = torch.tensor(E4M3, dtype=torch.float64)
    flat, codes = x.reshape(15, 3, 32).double(), q.codes.reshape(15, 3, 32).double()
    byte = q.scales.view(torch.uint8)[0]
    assert (byte[:, 3] == 0).all()
    for r in range(15):
        for b in range(3):
            top = flat[r, b].abs().max().item()
            k = -127 if top == 0 else max(-127, math.ceil(math.log2(top / 448)))
            assert byte[r, b] == k + 127
            t = flat[r, b] / 2.0 ** k
            best = (t[:, None] - grid).abs().min(1).values
            assert torch.equal((t - codes[r, b]).abs(), best)
    d = q.dequantize().reshape(15, 3, 32).double()
    assert torch.equal(d, codes * torch.exp2(byte[:, :3].double() - 127)[..., None])


def test_8bit_rows_of_odd_values():
    x = torch.zeros(4, 32)
    x[0, 0], x[0, 1], x[0, 2] = float("nan"), float("inf"), 3.0
    x[1] = float("-inf")
    x[2, 0], x[2, 1] = 2.0 ** -149, -0.0
    x[3, 0] = torch.finfo(torch.float32).max
    q = quant.quantize_mx(x)
    d = q.dequantize()
    assert d[0, :2].isnan().all() and d[0, 2] == 3.0 and (d[0, 3:] == 0).all() and d[1].isnan().all()
    assert q.scales.view(torch.uint8)[0, :, 0].tolist() == [120, 0, 0, 247] and (d[2] == 0).all()
    # the nearest code stands for 2^128, which float32 does not hold
    assert q.codes[3, 0].double() * 2.0 ** 120 == 2.0 ** 128 and d[3, 0].isinf()


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (3, 96, 32), (2, 192, 64), (5, 384, 128), (4, 160, 32)])
def test_4bit_weight(n, k, group):
    w = randn((n, k), gen(n + k))
    w[0, :group] = 0
    q = quant.quantize_group4(w, group)
    assert q.shape == (n, k) and q.group == group and q.codes.shape == (-(-n // 16), -(-k // 128), 4, 16, 16)
    s = (w.reshape(n, -1, group).abs().amax(-1) / 6).to(BF)
    assert q.scales.shape == (-(-n // 16), -(-k // 128), 16, 128 // group)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6])
    grid = torch.cat([grid, -grid]).double()
    t = w.double().reshape(n, -1, group)
    sd = s.double()[..., None]
    best = (t[..., None] - sd[..., None] * grid).abs().min(-1).values
    got = (q.dequantize().double().reshape(n, -1, group) - t).abs()
    assert (got <= best * (1 + 1e-6) + 1e-30).all()
    # the packed order, and zeros past the weight
    value = q.dequantize()
    assert value.shape == (n, k)
    table = [0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6]
    for (t, c, p, r, at), byte in zip(itertools.product(*map(range, q.codes.shape)), q.codes.flatten().tolist()):
        row, col = 16 * t + r, 128 * c + 32 * (at // 4) + 8 * p + 2 * (at % 4)
        for half, col in ((byte & 15, col), (byte >> 4, col + 1)):
            scale = float(q.scales[t, c, r, col % 128 // group])
            if row < n and col < k:
                assert scale == float(s[row, col // group]) and float(value[row, col]) == table[half] * scale
            else:
                assert half == 0 and (row < n and col // group < k // group or scale == 0)


def test_4bit_ties_go_to_the_even_code():
    w = torch.zeros(1, 32)
    w[0, :9] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -2.5])
    assert quant.quantize_group4(w).dequantize()[0, :9].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -2.0]


def test_no_rows():
    q = quant.quantize_mx(torch.empty(0, 2, 96))
    assert q.shape == (0, 2, 96) and q.scales.shape == (1, 0, 4) and q.dequantize().shape == (0, 2, 96)
    w = quant.quantize_group4(torch.empty(0, 160))
    assert w.shape == (0, 160) and w.group == 32 and w.dequantize().shape == (0, 160)


def test_packers_refuse():
    with pytest.raises(ValueError, match="multiple of 32"):
        quant.quantize_mx(torch.zeros(2, 48))
    with pytest.raises(TypeError):
        quant.quantize_mx(torch.zeros(2, 32, dtype=torch.int32))
    with pytest.raises(ValueError, match="group must be"):
        quant.quantize_group4(torch.zeros(2, 32), 16)
    with pytest.raises(ValueError, match="multiple of 64"):
        quant.quantize_group4(torch.zeros(2, 96), 64)
    with pytest.raises(ValueError, match="not finite"):
        quant.quantize_group4(torch.full((2, 32), float("inf")))
    with pytest.raises(ValueError, match="groups must be"):
        quant.Group4Weight.from_codes(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 2, dtype=BF))


def test_wrappers_refuse_on_the_host():
    """What never reaches the library: CPU tensors and wrong objects."""
    rows = quant.quantize_mx(torch.zeros(4, 64))
    w4 = quant.quantize_group4(torch.zeros(8, 64))
    for call in (lambda: kernels.adaln_mx(torch.zeros(1, 4, 64, dtype=BF)),
                 lambda: kernels.mx_linear(rows, rows),
                 lambda: kernels.group4_linear(torch.zeros(1, 64, dtype=BF), w4)):
        with pytest.raises(ValueError, match="device tensors"):
            call()
    with pytest.raises(TypeError, match="expected 8 arguments"):
        _native.host().mx_linear(rows.codes)


def test_a_scale_that_is_not_a_number():
    """E8M0's byte 255 is NaN: so is what its block stands for, and nothing else."""
    q = quant.quantize_mx(torch.ones(3, 96))
    q.scales.view(torch.uint8)[0, 1, 2] = 255
    v = q.dequantize()
    assert v[1, 64:].isnan().all() and v.isnan().sum() == 32


def test_packing_leaves_its_input():
    """A weight of whole tiles is not padded: the packed tensors must still be their own."""
    for n, group in ((16, 128), (16, 32), (32, 64)):
        codes = torch.randint(0, 256, (n, 64), dtype=torch.uint8)
        scales = torch.rand(n, 128 // group).to(BF)
        w = quant.Group4Weight.from_codes(codes, scales)
        was = w.dequantize()
        codes.zero_()
        scales.zero_()
        assert torch.equal(w.dequantize(), was) and was.any()


P = ctypes.c_void_p(4096)   # never read: each call below is refused before a launch
BIG = 1 << 30


def _adaln_mx(B, L, C, x_out=None, xo=(0, 0), eps=1e-6, y=P):
    _native.call("ltx_adaln_mx", B, L, C, P, L * C, C, y, L * C, C, None, 0, 0, x_out, *xo, None, 0, 0, None, 0, 0, eps,
                 P, P, None)


def _mx_linear(M, N, K, y_ls=None, y_scales=None, act=0, a=P):
    _native.call("ltx_mx_linear", M, N, K, a, P, P, P, None, act, P, N if y_ls is None else y_ls, y_scales, None)


def _group4_linear(M, N, K, group=32, y_ls=None, x_ls=None, x=P):
    _native.call("ltx_group4_linear", M, N, K, group, x, K if x_ls is None else x_ls, 0, P, P, None, P,
                 N if y_ls is None else y_ls, None)


@pytest.mark.parametrize("match,call", [
    ("multiple of 32", lambda: _adaln_mx(1, 1, 40)),
    ("multiple of 32", lambda: _adaln_mx(1, 1, 8224)),
    ("too many rows", lambda: _adaln_mx(1, 1 << 23, 32)),
    ("too many rows", lambda: _adaln_mx(1 << 20, 1 << 12, 32)),
    ("x_out without", lambda: _adaln_mx(1, 1, 32, P, y=None)),
    ("rows of x_out overlap", lambda: _adaln_mx(2, 3, 64, P, (0, 64))),
    ("rows of x_out overlap", lambda: _adaln_mx(2, 3, 64, P, (192, 0))),
    ("null pointer", lambda: _mx_linear(1, 32, 32, a=None)),
    ("16-byte aligned", lambda: _mx_linear(1, 32, 32, a=ctypes.c_void_p(4104))),
    ("bad M or N", lambda: _mx_linear(BIG, 32, 32)),
    ("too large", lambda: _mx_linear(BIG - 1, BIG - 1, 32)),
    ("too large", lambda: _mx_linear(BIG - 1, 1 << 20, 4096, act=1)),
    ("too large", lambda: _mx_linear(1 << 20, BIG - 32, 4096, y_scales=P)),
    ("rows of y overlap", lambda: _mx_linear(2, 64, 32, 63)),
    ("multiple of 32", lambda: _mx_linear(2, 40, 32, y_scales=P)),
    ("K must be", lambda: _mx_linear(2, 32, (1 << 20) + 32)),
    ("rows of y overlap", lambda: _group4_linear(2, 64, 32, y_ls=63)),
    ("16-byte aligned", lambda: _group4_linear(2, 64, 32, x_ls=36)),
    ("M must be", lambda: _group4_linear(17, 64, 32)),
    ("group must be", lambda: _group4_linear(2, 64, 32, group=16)),
    ("K must be", lambda: _group4_linear(2, 64, 4128)),
])
def test_entry_points_refuse(match, call):
    with pytest.raises(_native.NativeCallError, match=match):
        call()


@pytest.mark.parametrize("B,L,C,bs,ls", [(2, 2, 64, 64, 64), (2, 3, 64, 128, 64), (2, 3, 64, 184, 64), (3, 2, 64, 64, 128),
                                         (3, 2, 64, 64, 184), (2, 2, 64, 96, 64), (4, 4, 32, 64, 64)])
def test_rows_of_x_out_that_overlap_across_samples(B, L, C, bs, ls):
    """Two workgroups would store to one address."""
    at = sorted(b * bs + l * ls for b in range(B) for l in range(L))
    assert any(q - p < C for p, q in zip(at, at[1:]))
    with pytest.raises(_native.NativeCallError, match="rows of x_out overlap"):
        _adaln_mx(B, L, C, P, (bs, ls))


@pytest.mark.parametrize("B,L,C,bs,ls", [(2, 3, 64, 192, 64), (2, 3, 64, 64, 128), (2, 3, 64, 72, 136), (1, 3, 64, 0, 64),
                                         (3, 1, 64, 64, 0), (1, 1, 64, 0, 0), (2, 2, 64, 1 << 60, 64)])
def test_rows_of_x_out_side_by_side(B, L, C, bs, ls):
    """Refused for the alignment of its x only, which is looked at last."""
    odd = ctypes.c_void_p(4104)
    with pytest.raises(_native.NativeCallError, match="16-byte aligned"):
        _native.call("ltx_adaln_mx", B, L, C, odd, L * C, C, P, L * C, C, None, 0, 0, P, bs, ls, None, 0, 0, None, 0, 0, 1e-6,
                     P, P, None)


def _calls_that_want_gradients(x, make):
    """Each public call with one tensor of each kind made by ``make``."""
    rows, w4 = quant.quantize_mx(torch.zeros(4, 64)), quant.quantize_group4(torch.zeros(8, 64))
    bias, big = torch.zeros(8, dtype=BF), x.new_zeros(4, 4)
    return [lambda: kernels.adaln_mx(make(x)), lambda: kernels.adaln_mx(x, y=make(x)),
            lambda: kernels.adaln_mx(x, y=x, gate=make(x)), lambda: kernels.adaln_mx(x, y=x, x_out=make(x)),
            lambda: kernels.adaln_mx(x, scale=make(x), shift=x), lambda: kernels.adaln_mx(x, scale=x, shift=make(x)),
            lambda: kernels.mx_linear(rows, rows, make(bias[:4])), lambda: kernels.mx_linear(rows, rows, out=make(big)),
            lambda: kernels.group4_linear(make(x[0]), w4), lambda: kernels.group4_linear(x[0], w4, make(bias))]


def test_tensors_that_want_gradients_are_refused():
    """The results have no history: a gradient would be lost without a word."""
    x = torch.zeros(1, 4, 64, dtype=BF)
    calls = _calls_that_want_gradients(x, lambda t: t.clone().requires_grad_())
    for call in calls:
        with pytest.raises(RuntimeError, match="computes no gradients"):
            call()
    for call in calls:
        with torch.no_grad(), pytest.raises(ValueError, match="device tensors"):
            call()
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        for call in _calls_that_want_gradients(x, lambda t: torch.autograd.forward_ad.make_dual(t, t)):
            with pytest.raises(RuntimeError, match="computes no gradients"):
                call()


@pytest.mark.parametrize("top", [6e-38, 6e-39, 3e-40, 2.0 ** -133, 2.0 ** -149, 1.2e-38])
def test_4bit_weights_near_the_smallest_scales(top):
    """Scales below 2^-126, which bf16 holds to 2^-133: each value is still the nearest."""
    w = (torch.linspace(-1, 1, 32, dtype=torch.float64) * top).to(torch.float32)[None]
    q = quant.quantize_group4(w)
    s = (w.abs().amax() / 6).to(BF)
    assert q.scales[0, 0, 0, 0] == s
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    best = (w.double().abs()[..., None] - s.double() * grid).abs().amin(-1)
    # the value that a code stands for is a product in float32, to half of 2^-149
    assert ((q.dequantize().double() - w.double()).abs() <= best + 2.0 ** -150).all()


def _tile(M, N, K, quantized):
    tile = _native.i64_array([0] * 5)
    _native.call("ltx_mx_linear_tile", M, N, K, int(quantized), ctypes.cast(tile, ctypes.c_void_p))
    return tuple(tile)


def test_the_size_lists_reach_every_tile():
    """The GPU tests' sizes run every tile that a bf16 and an 8-bit result can take, and the long ones."""
    from .test_gpu_mx_linear import TILES, TILES_OF_48
    for quantized in (False, True):
        seen = {}
        for M, K, N in TILES + TILES_OF_48:
            rows, cols, groups, at, count = _tile(M, N // 32 * 32 if quantized else N, K, quantized)
            assert seen.setdefault(at, (rows, cols, groups)) == (rows, cols, groups)
        assert sorted(seen) == list(range(count)) and len(set(seen.values())) == count == 11
        assert ((16, 32, 8) in seen.values()) == quantized and ((16, 16, 8) in seen.values()) == (not quantized)
    assert _tile(2304, 16384, 4096, True)[:2] == (192, 256) and _tile(1, 40, 32, False)[:2] == (16, 16)


@pytest.mark.parametrize("match,call", [
    ("null pointer", lambda: _native.call("ltx_mx_linear_tile", 1, 32, 32, 0, None)),
    ("bad M or N", lambda: _tile(-1, 32, 32, False)),
    ("K must be", lambda: _tile(1, 32, 33, False)),
    ("empty or too large", lambda: _tile(0, 32, 32, False)),
    ("empty or too large", lambda: _tile(BIG - 1, BIG - 1, 32, True)),
])
def test_the_tile_query_refuses(match, call):
    with pytest.raises(_native.NativeCallError, match=match):
        call()
