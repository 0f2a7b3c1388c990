"""ltx_group4_linear against float64: every row count, K at and around the
128-column chunks, N around the 16-row tiles, every group, SiLU and bias."""
import pytest
import torch

from taomate_amd import _native as N
from taomate_amd import kernels, quant

from .helpers import gen, randn

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _weight(n, k, group, g):
    return quant.quantize_group4(randn((n, k), g) * torch.exp(randn((n, 1), g)) / k ** 0.5, group)


def _to(w, dev):
    return quant.Group4Weight(w.codes.to(dev), w.scales.to(dev), w.rows, w.columns)


def check(x, w, b, silu, y):
    xd = x.double()
    # float32 sums of K products: within 2^-20 of the magnitudes; the result's rounding, half a bf16 step
    extra = 0.0
    if silu:
        xd = xd * torch.sigmoid(xd)
        extra = 2.0 ** -8    # SiLU rounded to bf16
    wd = w.dequantize().double()
    ref = xd @ wd.t() + (0 if b is None else b.double())
    mag = xd.abs() @ wd.abs().t() + (0 if b is None else b.double().abs())
    assert y.shape == ref.shape and y.dtype == BF
    assert ((y.double().cpu() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1.01 * (2.0 ** -20 + extra) * mag).all()


@pytest.mark.parametrize("silu", [False, True], ids=["plain", "silu"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,chunks,n", [(1, 1, 1), (2, 3, 17), (3, 2, 16), (4, 5, 40), (5, 4, 33), (7, 9, 300),
                                        (8, 32, 130), (9, 8, 64), (15, 12, 47), (16, 32, 100), (2, 16, 4099)])
def test_group4_linear(dev, M, chunks, n, group, silu):
    g = gen(M * n + chunks + group)
    k = group * chunks if group * chunks <= 4096 else 4096
    x, w = randn((M, k), g, BF), _weight(n, k, group, g)
    b = randn((n,), g, BF) if n % 2 else None
    y = kernels.group4_linear(x.to(dev), _to(w, dev), None if b is None else b.to(dev), silu=silu)
    check(x, w, b, silu, y)


def test_strided_rows(dev):
    g = gen(5)
    big = randn((5, 512), g, BF)
    w = _weight(48, 256, 64, g)
    y = kernels.group4_linear(big.to(dev)[1:4, 128:384], _to(w, dev))
    check(big[1:4, 128:384], w, None, False, y)


def test_rows_do_not_meet(dev):
    """NaN and infinities in one row of x stay in that row of y."""
    g = gen(6)
    x, w = randn((4, 160), g, BF), _weight(70, 160, 32, g)
    clean = kernels.group4_linear(x.to(dev), _to(w, dev))
    x[1, 7], x[2, 3] = float("nan"), float("inf")
    y = kernels.group4_linear(x.to(dev), _to(w, dev))
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])
    assert y[1].isnan().all() and not y[2].isfinite().all()


def test_empty(dev):
    w = _to(_weight(16, 64, 32, gen(1)), dev)
    assert kernels.group4_linear(torch.empty(0, 64, dtype=BF, device=dev), w).shape == (0, 16)
    none = quant.Group4Weight(w.codes[:0], w.scales[:0], 0, 64)
    assert kernels.group4_linear(torch.empty(3, 64, dtype=BF, device=dev), none).shape == (3, 0)


def test_refusals(dev):
    w = _to(_weight(16, 64, 32, gen(1)), dev)
    x = torch.zeros(3, 64, device=dev, dtype=BF)
    with pytest.raises(N.NativeCallError, match="M must be"):
        kernels.group4_linear(torch.zeros(17, 64, device=dev, dtype=BF), w)
    with pytest.raises(N.NativeCallError, match="multiple of the group"):
        kernels.group4_linear(x, quant.Group4Weight(w.codes, w.scales[..., :1].contiguous(), 16, 64))   # groups of 128
    with pytest.raises(ValueError, match="group4_linear"):
        kernels.group4_linear(x, quant.Group4Weight(w.codes, w.scales.repeat(1, 1, 1, 2), 16, 64))   # groups of 16
    with pytest.raises(ValueError, match="group4_linear"):
        kernels.group4_linear(x, quant.Group4Weight(w.codes, w.scales, 17, 64))
    with pytest.raises(N.NativeCallError, match="16-byte aligned"):
        kernels.group4_linear(torch.zeros(3, 72, device=dev, dtype=BF)[:, 1:65], w)
    with pytest.raises(ValueError, match="group4_linear"):
        kernels.group4_linear(x[:, :32], w)
    with pytest.raises(ValueError, match="contiguous"):
        kernels.group4_linear(x, w, torch.zeros(15, device=dev, dtype=BF))
    with pytest.raises(TypeError):
        kernels.group4_linear(x.float(), w)


def test_one_row_expanded(dev):
    g = gen(7)
    x, w = randn((1, 256), g, BF), _weight(100, 256, 64, g)
    y = kernels.group4_linear(x.to(dev).expand(5, 256), _to(w, dev))
    assert torch.equal(y, kernels.group4_linear(x.to(dev), _to(w, dev)).expand(5, 100))


def test_a_long_weight(dev):
    """Codes past 2^32 bytes."""
    tiles, chunks = 70_000, 64 // 2
    codes = torch.empty(tiles, chunks, 4, 16, 16, dtype=torch.uint8, device=dev)
    g = torch.Generator(device=dev).manual_seed(3)
    for i in range(0, tiles, 10_000):
        codes[i:i + 10_000] = torch.randint(0, 256, (min(10_000, tiles - i), chunks, 4, 16, 16), generator=g, device=dev,
                                            dtype=torch.uint8)
    scales = torch.rand(tiles, chunks, 16, 1, generator=g, device=dev).to(BF)
    K = chunks * 128
    w = quant.Group4Weight(codes, scales, tiles * 16, K)
    x = torch.randn(2, K, generator=g, device=dev).to(BF)
    y = kernels.group4_linear(x, w)
    for t in (0, 32_767, 32_768, 65_536, tiles - 1):
        part = quant.Group4Weight(codes[t:t + 1].contiguous(), scales[t:t + 1].contiguous(), 16, K)
        check(x.cpu(), quant.Group4Weight(part.codes.cpu(), part.scales.cpu(), 16, K), None, False, y[:, t * 16:t * 16 + 16])


@pytest.mark.parametrize("M,K,n,group", [(1, 64, 5, 64), (3, 4096, 40, 32), (8, 2048, 300, 128), (9, 4096, 130, 64),
                                         (12, 160, 17, 32), (16, 32, 1, 32), (16, 4096, 4099, 128), (13, 1152, 9001, 32)])
def test_silu_is_not_rounded(dev, M, K, n, group):
    """Only the sums and the result's rounding: SiLU of |x| < 6 in float32 is within
    2^-20 (exp2's argument |x| 2^-23.4, exp2, reciprocal and product 1 ulp each), and
    what two bf16 hold of it within 2^-16 (each rounding leaves 2^-8 of what it rounds)."""
    g = gen(M + K + n)
    x, w = randn((M, K), g, BF).clamp(-6, 6), _weight(n, K, group, g)
    b = randn((n,), g, BF)
    y = kernels.group4_linear(x.to(dev), _to(w, dev), b.to(dev), silu=True).double().cpu()
    xd, wd = torch.nn.functional.silu(x.double()), w.dequantize().double()
    ref, mag = xd @ wd.t() + b.double(), xd.abs() @ wd.abs().t() + b.double().abs()
    assert ((y - ref).abs() <= 2.0 ** -8 * ref.abs() + 1.01 * (2.0 ** -16 + 2 * 2.0 ** -20) * mag).all()


@pytest.mark.parametrize("M", [4, 11])
def test_silu_of_infinities(dev, M):
    """+inf keeps its sign of the weights, NaN and -inf (0 * inf) are NaN, in their rows."""
    g = gen(M)
    x, w = randn((M, 128), g, BF), _weight(64, 128, 32, g)
    w = quant.quantize_group4(w.dequantize().abs() + 0.1 * w.dequantize().abs().amax(), 32)   # no code 0
    clean = kernels.group4_linear(x.to(dev), _to(w, dev), silu=True)
    x[0, 5], x[1, 7], x[M - 1, 9] = float("inf"), float("-inf"), float("nan")
    y = kernels.group4_linear(x.to(dev), _to(w, dev), silu=True)
    assert (w.dequantize()[:, 5] > 0).all() and (y[0] == float("inf")).all()
    assert y[1].isnan().all() and y[M - 1].isnan().all() and torch.equal(y[2:M - 1], clean[2:M - 1])


def check_unrounded(x, w, b, silu, y):
    """``check`` with SiLU(x) held to 2^-16 (two bf16 parts) + 2^-20 (its float32 steps), for |x| < 6."""
    xd, held = x.double(), 2.0 ** -20
    if silu:
        xd, held = torch.nn.functional.silu(xd), 2.0 ** -16 + 2 * 2.0 ** -20
    wd = w.dequantize().double()
    ref, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if b is not None:
        ref, mag = ref + b.double(), mag + b.double().abs()
    y = y.double()
    assert y.shape == ref.shape and ((y - ref).abs() <= 2.0 ** -8 * ref.abs() + 1.01 * held * mag).all()


# chunks of 128 columns that 1, 2, 4 and 8 waves share, whole and not, with the rows around the halves
UNROUNDED = [(1, 32, 1, 32), (2, 288, 17, 32), (8, 512, 40, 128), (9, 448, 33, 64), (16, 512, 300, 32),   # 1 wave
             (1, 544, 130, 32), (3, 576, 64, 64), (7, 640, 47, 128), (8, 1024, 100, 32), (9, 768, 515, 64),  # 2
             (12, 896, 31, 128), (16, 1024, 999, 64), (15, 992, 18, 32),
             (2, 1056, 50, 32), (8, 2048, 75, 64), (10, 1920, 20, 128), (16, 1600, 33, 64),   # 4
             (4, 2080, 41, 32), (8, 4096, 66, 128), (11, 4032, 19, 64), (16, 4096, 130, 32)]   # 8


@pytest.mark.parametrize("silu", [False, True], ids=["plain", "silu"])
@pytest.mark.parametrize("M,K,n,group", UNROUNDED)
def test_nothing_but_the_result_is_rounded(dev, M, K, n, group, silu):
    g = gen(3 * M + K + n)
    x, w = randn((M, K), g, BF).clamp(-5.96875, 5.96875), _weight(n, K, group, g)
    b = randn((n,), g, BF) if n % 2 else None
    y = kernels.group4_linear(x.to(dev), _to(w, dev), None if b is None else b.to(dev), silu=silu)
    check_unrounded(x, w, b, silu, y.cpu())


@pytest.mark.parametrize("M,silu", [(1, False), (2, True), (8, True), (9, True), (16, False)])
@pytest.mark.parametrize("K,group", [(64, 64), (512, 128), (544, 32), (1024, 64)])
@pytest.mark.parametrize("per", [1, 2, 4])
def test_several_rounds_of_short_rows(dev, per, K, group, M, silu):
    """Weights long enough that a workgroup takes 2, 3 and 5 rounds of tiles (and twice as many where
    the rows go by halves or one workgroup fills a CU): 512 workgroups of 8 tiles of 16 rows with one
    wave each, or of 4 with two.  Some workgroups have a round fewer than others."""
    n = per * 512 * (8 if K <= 512 else 4) * 16 + 5 * 16 + 3
    g = torch.Generator(device=dev).manual_seed(K + M + per)
    tiles, chunks = -(-n // 16), -(-K // 128)
    codes = torch.randint(0, 256, (n, K // 2), generator=g, device=dev, dtype=torch.uint8)
    scales = torch.rand(n, K // group, generator=g, device=dev).to(BF)
    w = quant.Group4Weight.from_codes(codes, scales)
    assert w.codes.shape[:2] == (tiles, chunks)
    x = torch.randn(M, K, generator=g, device=dev).clamp(-5.96875, 5.96875).to(BF)
    b = torch.randn(n, generator=g, device=dev).to(BF)
    check_unrounded(x, w, b, silu, kernels.group4_linear(x, w, b, silu=silu))
