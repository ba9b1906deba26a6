"""rmsnorm_quantize where its promises are narrow: the rows behind the last, and the scales counted rounding by rounding.

The roundings of an inverse scale, U = 2^-24 each, before any run.  The sum of squares of a row: a lane's four columns 3 (two products, of which one
is part of a multiply-add, and two additions), the 32 lanes 5, then the row's blocks: rows that a cluster holds, every eighth block to a lane, 3 more
between the lanes; longer rows, a warp's blocks one after the other, 8 warps, 8 CTAs.  All terms are positive, so the count bounds the
relative error.  The mean adds 2 (1 / K is rounded too), eps 1; the root halves it all and adds 1.5 of its own; the rounding of s = x + r counts once under the root
and once as the value.  Then the product with the weight, with 1 / rms, the reciprocal, the product with fp8_max and the second reciprocal: 5.
A reciprocal is a Newton step on the hardware's approximation (2^-22): its error is squared away, the last multiply-add rounds once.  The root's step has
a rounded product in it, half of whose error stays."""
import pytest

import fp8_quant_matmul_b200 as f

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"
U = 2.0 ** -24


def scale_roundings(K, long_rows, with_residual):
    blocks = K // 128
    if long_rows:
        squares = 3 + 5 + (blocks + 63) // 64 + 8 + 8
    else:
        squares = 3 + 5 + (blocks + 7) // 8 - 1 + 3
    return 0.5 * (squares + 3) + 1.5 + 5 + (2 if with_residual else 0)


@pytest.mark.parametrize("rows", [1, 5, 16, 17, 31])
@pytest.mark.parametrize("K", [256, 1152, 20480])
@pytest.mark.parametrize("xt,rt", [(BF16, None), (F32, None), (BF16, BF16), (F32, F32), (BF16, F32)], ids=lambda t: str(t).replace("torch.", ""))
def test_rows_behind_the_last_are_zero_bytes_whatever_the_weights(rows, K, xt, rt):
    g = torch.Generator().manual_seed(rows + K)
    x = torch.randn(rows, K, generator=g).to(xt).to(DEV)
    r = None if rt is None else torch.randn(rows, K, generator=g).to(rt).to(DEV)
    M = (rows + 15) // 16 * 16
    for special in ((), (float("nan"),), (float("inf"), float("-inf"))):
        w = torch.randn(K, generator=g)
        assert (w < 0).any()
        for i, v in enumerate(special):
            w[3 + 130 * i] = v
        q, sc = f.rmsnorm_quantize(x, w.to(DEV), residual=r)[:2]
        assert (q.view(K, M)[:, rows:] == 0).all()
        # 1 / (fp8_max / 1e-12): two reciprocals, a product and the constant's own rounding
        behind = sc.view(K // 128, M)[:, rows:].double()
        assert ((behind - 1e-12 / 448.0).abs() <= 4 * U * 1e-12 / 448.0).all()
        if not special:
            values = (x.double() + (0 if r is None else r.double()))
            values = values / torch.sqrt((values * values).mean(1, keepdim=True) + 1e-6) * w.to(DEV).double()
            inv = values.view(rows, K // 128, 128).abs().amax(2) / 448.0
            tol = scale_roundings(K, K > 16384, r is not None) * U
            assert ((sc.view(K // 128, M)[:, :rows].t().double() - inv).abs() <= tol * inv).all()
    f.last_device_status()


@pytest.mark.parametrize("K", [5248, 6144, 7168, 8192, 8320, 9216, 9344, 11264, 12288, 14336, 16384])
@pytest.mark.parametrize("rt", [None, BF16, F32], ids=lambda t: str(t).replace("torch.", ""))
def test_a_row_does_not_depend_on_how_many_there_are(K, rt):
    """The number of rows decides over how many CTAs of how many warps a row is spread; the order of its sums stays the same."""
    rows = 721
    g = torch.Generator().manual_seed(K)
    x = torch.randn(rows, K, generator=g).to(BF16).to(DEV)
    r = None if rt is None else torch.randn(rows, K, generator=g).to(rt).to(DEV)
    w = (1 + 0.3 * torch.randn(K, generator=g)).to(DEV)
    whole = f.rmsnorm_quantize(x, w, residual=r)
    M = 736
    values = x.double() + (0 if r is None else r.double())
    inv = (values / torch.sqrt((values * values).mean(1, keepdim=True) + 1e-6) * w.double()).view(rows, K // 128, 128).abs().amax(2) / 448.0
    assert ((whole[1].view(K // 128, M)[:, :rows].t().double() - inv).abs() <= scale_roundings(K, False, r is not None) * U * inv).all()
    for n in (1, 16, 241, 257, 369, 449, 529, 600):
        m = (n + 15) // 16 * 16
        part = f.rmsnorm_quantize(x[:n], w, residual=None if r is None else r[:n])
        assert torch.equal(part[0].view(K, m)[:, :n], whole[0].view(K, M)[:, :n]), n
        assert torch.equal(part[1].view(K // 128, m)[:, :n], whole[1].view(K // 128, M)[:, :n]), n
        if r is not None:
            assert torch.equal(part[2], whole[2][:n])
    f.last_device_status()


@pytest.mark.parametrize("fp8_max", [448.0, 240.0])
def test_reciprocals_of_many_magnitudes(fp8_max):
    """One value of 1 per block makes the mean 1 / 128 exactly, and the scale of a block its weight times sqrt(128): 1.5 roundings of the root, the product, and
    the two reciprocals with a product between."""
    KB = 128
    K = 128 * KB
    g = torch.Generator().manual_seed(1)
    for _ in range(8):
        x = torch.zeros(1, K, device=DEV)
        x[:, ::128] = 1.0
        w = torch.zeros(K)
        w[::128] = torch.exp(torch.empty(KB).uniform_(-25.0, 60.0, generator=g)) * (1 + torch.rand(KB, generator=g))
        w = w.to(DEV)
        _, sc = f.rmsnorm_quantize(x, w, eps=0.0, fp8_max=fp8_max)
        want = w[::128].double() * 128 ** 0.5 / fp8_max
        got = sc.view(KB, 16)[:, 0].double()
        assert ((got - want).abs() <= (1.5 + 1 + 3) * U * 1.001 * want).all(), float(((got - want).abs() / want).max() / U)


def test_roots_of_many_magnitudes():
    """Rows with one value v: the mean is v^2 / 128 with one rounding, eps adds one, the root's own 1.5; then the value over the root and as above."""
    rows, K = 4096, 128
    g = torch.Generator().manual_seed(2)
    v = torch.exp(torch.empty(rows).uniform_(-30.0, 40.0, generator=g)) * (1 + torch.rand(rows, generator=g))
    x = torch.zeros(rows, K)
    x[:, 5] = v
    for eps in (0.0, 1e-6, 3e5):
        _, sc = f.rmsnorm_quantize(x.to(DEV), torch.full((K,), 1e6, device=DEV), eps=eps)
        v64, e = v.double(), torch.tensor(eps, dtype=F32).double()
        want = (1e6 * v64 / torch.sqrt(v64 * v64 / 128 + e)).clamp(min=1e-12) / 448.0
        got = sc.cpu().double()
        # the weight of 1e6 is exact in fp32; its product with v rounds once
        assert ((got - want).abs() <= (1.0 + 1.5 + 1 + 1 + 3) * U * 1.001 * want).all(), (eps, float(((got - want).abs() / want).max() / U))


def test_the_scales_of_quantize_rowwise_within_their_roundings():
    """With a root of exactly 1 the norm hands its rows to the scaling of quantize_rowwise: the values of both are e4m3 steps of the same scales up to the
    counted roundings, and no byte is more than one step apart."""
    rows, K = 64, 1024
    g = torch.Generator().manual_seed(3)
    x = torch.randn(rows, K, generator=g).to(DEV)
    y = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6)
    a, s = f.rmsnorm_quantize(x, torch.ones(K, device=DEV))
    b, t = f.quantize_rowwise(y.float())
    tol = (scale_roundings(K, False, False) + 4) * U          # and y's own rounding and three of the other scale
    assert ((s.double() - t.double()).abs() <= tol * t.double()).all()
    # magnitudes of e4m3 bytes are in order: neighbouring values have neighbouring bytes
    assert ((a & 0x7F).int() - (b & 0x7F).int()).abs().max() <= 1
    assert (((a ^ b) & 0x80 == 0) | ((a & 0x7F) == 0) | ((b & 0x7F) == 0)).all()
