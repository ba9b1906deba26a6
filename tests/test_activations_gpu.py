"""The activations of the fused epilogues on their own: zero or exact sums, so that the argument is known to the bit.

What is allowed.  silu: the exponential's argument (57 at -40) is off by two roundings of 2^-24, times ln 2; two approximations of 2^-22 and five
products: below 2^-17 of the result.  gelu_tanh: the argument (57 at -7.4) is off by five: below 2^-16 of the result.  gelu: the formula 7.5e-8 of the
argument's magnitude, and of erfc's share of the result (all of it below 0) 2^-19: t is off by 2^-21.4, times 3.44, the largest logarithmic slope of the
polynomial, whose own roundings are 2^-21 and the exponential's 2^-22.  Below -3 that absolute bound says little, and the formula's error relative to the result is
held to what 7.1.26 has there in exact arithmetic, a tenth more, and the exponential's argument (26 at -6, two roundings).  A bf16 step is 2^-8 to 2^-7 of its value."""
import math

import pytest

import fp8_quant_matmul_b200 as f

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DEV = "cuda"
PAIR = 256 | f.TILE_PAIR
U = 2.0 ** -24
REACH = {"silu": -39.5, "gelu": -12.5, "gelu_tanh": -7.35}        # below it silu and gelu_tanh are less than 3e-16
ALLOWED = {"silu": 2.0 ** -17, "gelu_tanh": 2.0 ** -16}


def act64(x, name):
    if name == "silu":
        return x * torch.sigmoid(x)
    if name == "gelu":
        return x * 0.5 * torch.special.erfc(-x * math.sqrt(0.5))
    return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))


def allowed(x, want, name):
    """How far a result may be from `want` before it is rounded."""
    if name != "gelu":
        return ALLOWED[name] * want.abs()
    u = x.abs()
    tol = 7.5e-8 * u + 2.0 ** -19 * u * 0.5 * torch.special.erfc(u * math.sqrt(0.5)) + 2 * U * want.abs()
    # 7.1.26 in exact arithmetic, relative to erfc
    z = u * math.sqrt(0.5)
    t = 1 / (1 + 0.3275911 * z)
    poly = t * (0.254829592 + t * (-0.284496736 + t * (1.421413741 + t * (-1.453152027 + t * 1.061405429))))
    tail = (1.1 * (poly / torch.special.erfcx(z) - 1).abs() + 2.0 ** -19 + 0.72 * u * u * 2.0 ** -23) * want.abs()
    return torch.where(x < -3.0, torch.minimum(tol, tail), tol)


def arguments(name, n):
    lo = REACH[name]
    g = torch.Generator().manual_seed(n)
    x = torch.empty(n).uniform_(lo, -lo, generator=g)
    x[: n // 4] = torch.linspace(lo, 0, n // 4)
    x[n // 4: n // 2] = torch.empty(n // 4).uniform_(-6.0, 6.0, generator=g)
    x[-16:] = torch.exp(torch.linspace(-12, 0, 16)) * torch.tensor([1.0, -1.0]).repeat(8)
    return x


def one_by_one(n_blocks, M, gate, up):
    """Operands whose product is gate[b] in every column of block b, and up in the block's first column and 0 in the others; row 0, the others zeros."""
    K, N = 128, 128 * n_blocks
    A = torch.zeros(K, M, dtype=torch.uint8)
    A[0, 0] = 0x38                                                # 1.0
    G = torch.zeros(K, N, dtype=torch.uint8)
    G[0] = 0x38
    P = torch.zeros(K, N, dtype=torch.uint8)
    P[0, ::128] = 0x38
    return [t.flatten().to(DEV) for t in (A, G, P, torch.ones(M), gate.float(), torch.full((n_blocks,), up))] + [N, K]


@pytest.mark.parametrize("act", sorted(REACH))
@pytest.mark.parametrize("M,kw", [(16, {}), (64, {}), (144, dict(splits=1, tile_n=256)), (144, dict(splits=1, tile_n=PAIR))], ids=str)
def test_in_32_bits(act, M, kw):
    # the inverse scale of a block is its only value over 448, in fp32: 4 roundings on top of the product with 2^80, which is exact
    n, up = 512, 2.0 ** 80
    x = arguments(act, n)
    A, G, P, a_s, g_s, p_s, N, K = one_by_one(n, M, x, up)
    _, sc = f.gemm_gated(A, G, P, a_s, g_s, p_s, M=M, N=N, K=K, activation=act, quantize=True, **kw)
    f.last_device_status()
    got = sc.view(n, M)[:, 0].cpu().double() * 448.0 / up
    want = act64(x.double(), act).abs().clamp(min=1e-12 / up)          # the scale's lower bound, which an argument of 0 meets
    tol = allowed(x.double(), want, act) + 5 * U * want
    worst = ((got - want).abs() / tol).argmax()
    assert ((got - want).abs() <= tol).all(), (float(x[worst]), float(got[worst]), float(want[worst]))


@pytest.mark.parametrize("act", sorted(REACH))
@pytest.mark.parametrize("M,splits,tile", [(16, 1, f.SMALL_M), (64, 2, f.SMALL_M), (144, 1, 128), (144, 1, PAIR), (144, 2, 128)])
def test_the_tail_in_bf16(act, M, splits, tile):
    # zero sums: the argument is the bias.  Half a bf16 step is at most 2^-8 of the value
    N, K = 4096, 256
    A, a_s = torch.zeros(M * K, dtype=torch.uint8, device=DEV), torch.ones(M * 2, device=DEV)
    B, b_s = torch.full((N * K,), 0x38, dtype=torch.uint8, device=DEV), torch.ones(N // 128 * 2, device=DEV)
    x = torch.linspace(REACH[act], 0.0, N)
    C = f.gemm_bias_act(A, B, a_s, b_s, M=M, N=N, K=K, bias=x.to(DEV), activation=act, splits=splits, tile_n=tile).cpu().double()
    want = act64(x.double(), act)
    tol = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * allowed(x.double(), want, act)
    worst = ((C - want).abs() / tol.clamp(min=1e-300)).amax(0).argmax()
    assert ((C - want).abs() <= tol).all(), (float(x[worst]), float(C[0, worst]), float(want[worst]))
