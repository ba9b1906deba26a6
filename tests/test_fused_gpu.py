"""gemm_bias_act and gemm_gated against the formulas in 64 bits, for every kernel they can run on.

Tolerances, before any run.  A sum of K products in fp32 (the tensor core's accumulation, one multiply-add per K block, the partial sums of up
to 8 CTAs) is off by at most (K + K / 128 + 8) 2^-24 of the sum of magnitudes; the bias adds one rounding.  The activations have slopes
below 1.13 and are computed to 2^-19 of their argument (two approximations of 2^-22, an argument rounded a few times whose error
the exponential multiplies by at most 20 before the result is below 2^-19 of x; erf 7.5e-8).  A product of two adds its factors' errors.
bf16: half a step, 2^-8 of the value.  8 bits: half a step of e4m3 (2^-4 of the value's binade, 2^-10 below 2^-6); the scale is as far off as
the largest element of its group, and 4 roundings."""
import math
import os
import subprocess
import sys

import pytest

import fp8_quant_matmul_b200 as f

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
DEV = "cuda"
PAIR = 256 | f.TILE_PAIR
U = 2.0 ** -24
ACT_ERR = 2.0 ** -19
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def operand(rows, K, seed, rows_per_group, std=1.0, live=None):
    """Column-major bytes, inverse scales and the [rows, K] float64 values; rows from `live` on are zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g) * torch.exp(0.5 * torch.randn(K, generator=g)) * std
    if live is not None:
        x[live:] = 0
    pad = -rows % rows_per_group
    b = torch.nn.functional.pad(x, (0, 0, 0, pad)).view((rows + pad) // rows_per_group, rows_per_group, K // 128, 128)
    inv = b.abs().amax((1, 3), keepdim=True).clamp(min=1e-12) / 448.0
    q = (b / inv).clamp(-448, 448).view(rows + pad, K)[:rows].to(FP8)
    inv = inv.view(-1, K // 128)
    values = q.double() * inv.double().repeat_interleave(rows_per_group, 0)[:rows].repeat_interleave(128, 1)
    return q.view(torch.uint8).t().contiguous().flatten().to(DEV), inv.t().contiguous().flatten().to(DEV), values.to(DEV)


def product(A, B):
    """(product, bound of its error) in float64."""
    K = A.shape[1]
    return A @ B.t(), (K + K // 128 + 9) * U * (A.abs() @ B.abs().t())


def act64(x, name):
    if name == "relu":
        return x.clamp(min=0)
    if name == "silu":
        return x * torch.sigmoid(x)
    if name == "gelu":
        return x * torch.special.ndtr(x)
    if name == "gelu_tanh":
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
    return x


def activated(x, err, name):
    y = act64(x, name)
    return y, 1.13 * err + (0 if name in ("none", "relu") else ACT_ERR * x.abs())


def close_bf16(got, want, err):
    d = (got.double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + 1.01 * err + 1e-30
    assert got.isfinite().all()
    assert (d <= tol).all(), float((d / tol).max())


# (M, rows, N, K, splits, tile_n): the library's choices, then every kernel by name
SHAPES = [
    (16, 1, 16, 128, 0, 0), (16, 3, 208, 384, 0, 0), (16, 16, 1536, 7168, 0, 0), (32, 20, 144, 1024, 0, 0), (64, 49, 400, 2304, 0, 0),
    (64, 64, 272, 640, 1, f.SMALL_M), (48, 33, 528, 1152, 3, f.SMALL_M), (32, 31, 128, 1024, 8, f.SMALL_M),
    (80, 77, 320, 512, 0, 0), (272, 257, 1040, 1664, 0, 0),
    (144, 130, 272, 128, 1, 128), (400, 399, 336, 640, 1, 128), (208, 200, 48, 256, 1, 128), (2064, 2051, 1552, 384, 1, 128),
    (144, 130, 272, 128, 1, PAIR), (528, 513, 784, 896, 1, PAIR), (272, 270, 80, 384, 1, PAIR), (2064, 2051, 1552, 384, 1, PAIR),
    (144, 130, 272, 384, 2, 128), (272, 257, 400, 1152, 8, 128), (144, 144, 528, 896, 5, 256), (272, 260, 144, 384, 3, 256),
]
EXTRAS = [("none", None, False), ("relu", F32, False), ("silu", BF16, True), ("gelu", F32, True), ("gelu_tanh", None, True)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act,bias_type,with_residual", EXTRAS, ids=[e[0] for e in EXTRAS])
def test_bias_activation_residual(shape, act, bias_type, with_residual):
    M, rows, N, K, splits, tile = shape
    A, a_s, Av = operand(M, K, M + N, 1, live=rows)
    B, b_s, Bv = operand(N, K, N + K, 128, std=2 * K ** -0.5)
    g = torch.Generator().manual_seed(7)
    bias = None if bias_type is None else torch.randn(N, generator=g).to(bias_type).to(DEV)
    wide = torch.randn(rows, N + 24, generator=g).to(BF16).to(DEV)
    residual = wide[:, 8:8 + N] if with_residual else None
    C = f.gemm_bias_act(A, B, a_s, b_s, M=M, N=N, K=K, rows=rows, bias=bias, activation=act, residual=residual, splits=splits, tile_n=tile)
    f.last_device_status()
    x, err = product(Av[:rows], Bv)
    if bias is not None:
        x = x + bias.double()
        err = err + U * x.abs()
    y, err = activated(x, err, act)
    if residual is not None:
        y = y + residual.double()
        err = err + U * y.abs()
    assert C.shape == (rows, N)
    close_bf16(C, y, err)


@pytest.mark.parametrize("M,N,K,splits,tile", [(32, 400, 1024, 0, 0), (64, 272, 640, 1, f.SMALL_M), (272, 528, 896, 1, 128), (528, 784, 896, 1, PAIR),
                                               (272, 400, 1152, 4, 128), (144, 528, 896, 3, 256)])
def test_without_extras_it_is_the_product_bit_for_bit(M, N, K, splits, tile):
    A, a_s, _ = operand(M, K, 1, 1)
    B, b_s, _ = operand(N, K, 2, 128)
    path = f.PATH_AUTO if tile in (0, f.SMALL_M) else (f.PATH_MN_SMALL if splits > 1 else f.PATH_MN_LARGE)
    want = f.gemm(A, B, a_s, b_s, M=M, N=N, K=K, path=path, splits=splits, tile_n=tile)
    got = f.gemm_bias_act(A, B, a_s, b_s, M=M, N=N, K=K, splits=splits, tile_n=tile)
    assert torch.equal(want.view(torch.int16), got.view(torch.int16))


@pytest.mark.parametrize("M,rows,N,K,splits,tile", [(16, 5, 400, 1024, 0, 0), (64, 50, 272, 640, 1, f.SMALL_M), (272, 259, 528, 896, 1, 128),
                                                    (528, 515, 784, 896, 1, PAIR), (272, 258, 400, 1152, 4, 128)])
def test_residual_in_place_and_nothing_behind_the_last_row(M, rows, N, K, splits, tile):
    A, a_s, _ = operand(M, K, 3, 1)
    B, b_s, _ = operand(N, K, 4, 128)
    buf = torch.randn(M + 2, N, generator=torch.Generator().manual_seed(5)).to(BF16).to(DEV)
    before = buf.clone()
    kw = dict(M=M, N=N, K=K, rows=rows, activation="silu", splits=splits, tile_n=tile)
    apart = f.gemm_bias_act(A, B, a_s, b_s, residual=before[1:1 + rows], **kw)
    C = buf[1:1 + rows]
    assert f.gemm_bias_act(A, B, a_s, b_s, C=C, residual=C, **kw) is C
    torch.cuda.synchronize()
    assert torch.equal(apart.view(torch.int16), C.view(torch.int16))
    assert torch.equal(buf[:1], before[:1]) and torch.equal(buf[1 + rows:], before[1 + rows:])


# (M, rows, N, K, splits, tile_n, fp8)
GATED = [
    (16, 1, 128, 128, 0, 0), (16, 7, 512, 7168, 0, 0), (16, 16, 384, 640, 1, f.SMALL_M), (32, 18, 256, 1024, 3, f.SMALL_M),
    (48, 48, 640, 1152, 0, 0), (64, 50, 384, 2304, 8, f.SMALL_M), (64, 64, 128, 256, 2, f.SMALL_M),
    (80, 70, 256, 512, 0, 0), (208, 193, 384, 1664, 0, 0),
    (144, 130, 256, 128, 1, 256), (400, 390, 384, 640, 1, 256), (2064, 2051, 2560, 256, 1, 256),
    (144, 130, 256, 128, 1, PAIR), (528, 513, 640, 896, 1, PAIR), (272, 260, 128, 384, 1, PAIR), (2064, 2051, 2560, 256, 1, PAIR), (1040, 1033, 2432, 384, 1, PAIR),
    (144, 130, 256, 384, 2, 256), (272, 257, 384, 1152, 8, 256), (144, 144, 512, 896, 5, 256), (80, 66, 128, 1664, 7, 256),
]


def gated_want(Av, Gv, Uv, act):
    g, eg = product(Av, Gv)
    u, eu = product(Av, Uv)
    a, ea = activated(g, eg, act)
    h = a * u
    return h, a.abs() * eu + u.abs() * ea + ea * eu + 2 * U * h.abs()


def gated_operands(M, rows, N, K):
    A, a_s, Av = operand(M, K, M + 1, 1, live=rows)
    G, g_s, Gv = operand(N, K, N + 2, 128, std=2 * K ** -0.5)
    P, p_s, Pv = operand(N, K, N + 3, 128, std=K ** -0.5)
    return (A, G, P, a_s, g_s, p_s), (Av, Gv, Pv)


@pytest.mark.parametrize("shape", GATED, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_in_8_bits(shape, act):
    M, rows, N, K, splits, tile = shape
    args, values = gated_operands(M, rows, N, K)
    q, sc = f.gemm_gated(*args, M=M, N=N, K=K, activation=act, quantize=True, splits=splits, tile_n=tile)
    f.last_device_status()
    h, err = gated_want(*values, act)
    blocks = h.view(M, N // 128, 128)
    amax = blocks.abs().amax(2)
    inv = amax.clamp(min=1e-12) / 448.0
    e_inv = err.view(M, N // 128, 128).amax(2) / 448.0 + 4 * U * inv
    got_inv = sc.view(N // 128, M).t().double()
    assert ((got_inv - inv).abs() <= 1.01 * e_inv).all()
    got = q.view(FP8).view(N, M).t().double()
    # the bytes against the exact value over the scale that was stored, which has been checked
    exact = (blocks / got_inv[:, :, None]).view(M, N)
    half_step = torch.exp2(torch.floor(torch.log2(exact.abs().clamp(min=2.0 ** -6)))) * 2.0 ** -4
    tol = half_step + (1.01 * err.view(M, N // 128, 128) / got_inv[:, :, None]).view(M, N) + 2.0 ** -20 * exact.abs()
    assert ((got - exact).abs() <= tol).all(), float(((got - exact).abs() / tol).max())
    assert (got[rows:] == 0).all()


@pytest.mark.parametrize("shape", GATED + [(16, 5, 48, 384, 0, 0), (64, 40, 336, 896, 4, f.SMALL_M), (272, 270, 208, 640, 1, 256),
                                           (528, 520, 80, 640, 1, PAIR), (400, 399, 1552, 256, 1, PAIR), (272, 270, 208, 640, 3, 256), (1040, 1037, 1552, 3200, 0, 0)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", ["gelu_tanh", "relu", "none"])
def test_gated_in_bf16(shape, act):
    M, rows, N, K, splits, tile = shape
    args, (Av, Gv, Pv) = gated_operands(M, rows, N, K)
    buf = torch.full((rows + 2, N), 7.0, dtype=BF16, device=DEV)
    H = f.gemm_gated(*args, M=M, N=N, K=K, activation=act, rows=rows, splits=splits, tile_n=tile, H=buf[1:1 + rows])
    f.last_device_status()
    h, err = gated_want(Av[:rows], Gv, Pv, act)
    close_bf16(H, h, err)
    assert (buf[0] == 7.0).all() and (buf[-1] == 7.0).all()


@pytest.mark.parametrize("M,splits,tile", [(32, 2, f.SMALL_M), (144, 1, PAIR), (144, 1, 256), (144, 3, 256)])
def test_gated_fp8_max_zeros_and_nan(M, splits, tile):
    N, K = 256, 384
    (A, G, P, a_s, g_s, p_s), values = gated_operands(M, M - 3, N, K)
    A.view(K, M)[5, 2] = 0x7F                                            # a NaN in row 2
    q, sc = f.gemm_gated(A, G, P, a_s, g_s, p_s, M=M, N=N, K=K, quantize=True, fp8_max=240.0, splits=splits, tile_n=tile)
    q, sc = q.view(N, M).t(), sc.view(N // 128, M).t()
    assert ((q[2] & 0x7F) == 0x7F).all() and sc[2].isnan().all()
    ok = [m for m in range(M) if m != 2]
    v = q[ok].contiguous().view(FP8).float()
    assert v.isfinite().all() and v.abs().max() == 240.0
    assert (v[-3:] == 0).all() and sc[ok].isfinite().all()
    # each group's largest element sits at fp8_max, up to its rounding
    assert (v[:-3].view(len(ok) - 3, 2, 128).abs().amax(2) >= 224.0).all()


def test_the_same_call_gives_the_same_bits_on_two_streams_and_in_a_graph():
    cases = []
    for M, N, K, kw in [(16, 512, 2304, {}), (208, 384, 1664, {}), (528, 640, 896, {})]:
        args, _ = gated_operands(M, M, N, K)
        B, b_s, _ = operand(K, N, 9, 128)
        r = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)

        def block(M=M, N=N, K=K, args=args, B=B, b_s=b_s, r=r):
            q, sc = f.gemm_gated(*args, M=M, N=N, K=K, quantize=True)
            return f.gemm_bias_act(q, B, sc, b_s, M=M, N=K, K=N, residual=r)
        cases.append((block, block()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append([b() for b, _ in cases])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [b() for b, _ in cases]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    f.last_device_status()
    for out in outs + [captured]:
        for o, (_, want) in zip(out, cases):
            assert torch.equal(o.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_a_feed_forward_block(rows):
    """x -> norm -> gate, up, activation, product -> down projection + the residual stream: three launches, against the same run in 64 bits on the
    quantised operands each step was given."""
    K, F, M = 1024, 512, (rows + 15) // 16 * 16
    g = torch.Generator().manual_seed(rows)
    x, stream = (torch.randn(rows, K, generator=g).to(BF16).to(DEV) for _ in range(2))
    w = (1 + 0.1 * torch.randn(K, generator=g)).to(BF16).to(DEV)
    Wg, Wu = ((torch.randn(F, K, generator=g) * K ** -0.5).to(DEV) for _ in range(2))
    Wd = (torch.randn(K, F, generator=g) * F ** -0.5).to(DEV)
    (G, g_s), (P, p_s), (D, d_s) = (f.quantize_block(t) for t in (Wg, Wu, Wd))
    before = f.launch_count()
    q, sc, s = f.rmsnorm_quantize(x, w, residual=stream)
    hq, hs = f.gemm_gated(q, G, P, sc, g_s, p_s, M=M, N=F, K=K, quantize=True)
    y = f.gemm_bias_act(hq, D, hs, d_s, M=M, N=K, K=F, rows=rows, residual=s)
    assert f.launch_count() - before == 3
    f.last_device_status()

    def values(b, inv, R, C, group):
        sv = inv.double().view(C // 128, -1).t().repeat_interleave(group, 0)[:R].repeat_interleave(128, 1)
        return b.view(FP8).view(C, R).t().double() * sv
    h, _ = gated_want(values(q, sc, M, K, 1), values(G, g_s, F, K, 128), values(P, p_s, F, K, 128), "silu")
    hv = values(hq, hs, M, F, 1)
    assert ((hv - h).abs() <= h.view(M, F // 128, 128).abs().amax(2).repeat_interleave(128, 1) * 2.0 ** -4 * 1.001).all()
    out, err = product(hv[:rows], values(D, d_s, K, F, 128))
    out = out + s.double()
    close_bf16(y, out, err + U * out.abs())
    # and what the block computes without any quantisation: e4m3 operands (3 mantissa bits, errors that average out) in two products
    xs = x.double() + stream.double()
    n = xs / torch.sqrt((xs * xs).mean(1, keepdim=True) + 1e-6) * w.double()
    gd = n @ Wg.double().t()
    plain = (gd * torch.sigmoid(gd) * (n @ Wu.double().t())) @ Wd.double().t()
    assert ((y.double() - s.double()) - plain).norm() <= 0.1 * plain.norm()


@pytest.mark.parametrize("act,want", [
    ("none", lambda x: x),
    ("relu", lambda x: 0.0 if x < 0 else x),
    ("silu", lambda x: x if x > 0 else 0.0),
    ("gelu", lambda x: x if x > 0 else 0.0),
    ("gelu_tanh", lambda x: x if x > 0 else 0.0)])
@pytest.mark.parametrize("M,splits,tile", [(16, 1, f.SMALL_M), (64, 2, f.SMALL_M), (144, 1, 128), (144, 1, PAIR), (144, 2, 128)])
def test_extreme_arguments_of_the_activations(act, want, M, splits, tile):
    # sums are 0, so that the argument is the bias: infinities, NaN and magnitudes at which squares and exponentials overflow, each beside an
    # ordinary value that must not be touched
    N, K = 272, 256
    A, a_s, _ = operand(M, K, 1, 1)
    A.zero_()
    B, b_s, _ = operand(N, K, 2, 128)
    values = [float("inf"), 1.5, float("-inf"), 1.5, float("nan"), 1.5, 1e30, 1.5, -1e30, 1.5, 3e38, 1.5, -3e38, 1.5, -50.0, 1.5]
    bias = torch.tensor((values * 17)[:N], device=DEV)
    C = f.gemm_bias_act(A, B, a_s, b_s, M=M, N=N, K=K, bias=bias, activation=act, splits=splits, tile_n=tile).double()
    ordinary = float(act64(torch.tensor(1.5, dtype=torch.float64), act))
    for j, v in enumerate(values):
        got = C[:, j::16]
        if v == 1.5:
            assert ((got - ordinary).abs() <= 2.0 ** -8 * ordinary).all()
        elif v != v:
            assert got.isnan().all()
        elif act == "none" or want(v) != 0.0:
            assert (got == torch.tensor(want(v), dtype=torch.float64).to(BF16).double()).all(), (v, got[0, 0])
        else:
            assert (got.abs() <= 1e-15).all(), (v, got[0, 0])           # the tail: below 40 * 2^-57


def test_offsets_beyond_32_bits():
    # C and the residual of 2.2e9 elements, the A operand of a wide product of 2.2e9 bytes: the last rows and columns are where they belong
    M, N, K = 270336, 8192, 128
    g = torch.Generator(device=DEV).manual_seed(1)
    A = torch.randint(0x20, 0x40, (M * K,), dtype=torch.uint8, device=DEV, generator=g)
    a_s = torch.rand(M, device=DEV, generator=g)
    B, b_s, Bv = operand(N, K, 3, 128)
    R = torch.randn(M, N, device=DEV, generator=g, dtype=BF16)
    C = f.gemm_bias_act(A, B, a_s, b_s, M=M, N=N, K=K, residual=R, activation="relu")
    q, sc = f.gemm_gated(A, B, B, a_s, b_s, b_s, M=M, N=N, K=K, activation="none", quantize=True)
    f.last_device_status()
    rows = torch.tensor([0, 1, M // 2 + 3, M - 17, M - 1], device=DEV)
    Av = A.view(FP8).view(K, M)[:, rows].t().double() * a_s[rows, None].double()
    x, err = product(Av, Bv)
    y = x.clamp(min=0) + R[rows].double()
    close_bf16(C[rows], y, 1.13 * err + U * y.abs())
    h = (x * x).view(len(rows), N // 128, 128)
    inv = sc.view(N // 128, M)[:, rows].t().double()
    assert ((inv - h.amax(2) / 448.0).abs() <= 1e-5 * inv).all()
    got = q.view(FP8).view(N, M)[:, rows].t().double().view(len(rows), N // 128, 128)
    assert ((got * inv[:, :, None] - h).abs() <= h.amax(2, keepdim=True) * 2.0 ** -4 * 1.001).all()



@pytest.mark.parametrize("splits", [2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("M,rows", [(80, 67), (128, 128), (272, 257)])
def test_every_number_of_splits(splits, M, rows):
    """The shares of a tile's rows are of other sizes and start at other places for each; nothing around the results is touched."""
    N, K = 256, 1152
    (A, G, P, a_s, g_s, p_s), (Av, Gv, Pv) = gated_operands(M, rows, N, K)
    pad, stream = 256, torch.cuda.current_stream().cuda_stream
    q = torch.full((M * N + 2 * pad,), 0xAB, dtype=torch.uint8, device=DEV)
    sc = torch.full((M * 2 + 2 * pad,), -7.0, device=DEV)
    rc = f.lib().fp8bs_gemm_gated(A.data_ptr(), G.data_ptr(), P.data_ptr(), a_s.data_ptr(), g_s.data_ptr(), p_s.data_ptr(), q[pad:].data_ptr(), sc[pad:].data_ptr(),
                                  M, N, K, rows, f.ACTIVATIONS["silu"], 448.0, splits, 256, stream)
    assert rc == 0
    f.last_device_status()
    for buf, n, fill in ((q, M * N, 0xAB), (sc, M * 2, -7.0)):
        assert (buf[:pad] == fill).all() and (buf[pad + n:] == fill).all()
    h, err = gated_want(Av, Gv, Pv, "silu")
    inv = sc[pad:pad + M * 2].view(2, M).t().double()
    amax, e = (v.view(M, 2, 128).abs().amax(2) for v in (h, err))
    assert ((inv - amax.clamp(min=1e-12) / 448.0).abs() <= 1.01 * e / 448.0 + 4 * U * inv).all()
    exact = (h.view(M, 2, 128) / inv[:, :, None]).view(M, N)
    got = q[pad:pad + M * N].view(FP8).view(N, M).t().double()
    half_step = torch.exp2(torch.floor(torch.log2(exact.abs().clamp(min=2.0 ** -6)))) * 2.0 ** -4
    assert ((got - exact).abs() <= half_step + (1.01 * err.view(M, 2, 128) / inv[:, :, None]).view(M, N) + 2.0 ** -20 * exact.abs()).all()
    H = torch.full((rows + 1, N), 7.0, dtype=BF16, device=DEV)
    f.gemm_gated(A, G, P, a_s, g_s, p_s, M=M, N=N, K=K, rows=rows, H=H[:rows], splits=splits, tile_n=256)
    close_bf16(H[:rows], h[:rows], err[:rows])
    assert (H[rows] == 7.0).all()
    product_of_one, e1 = product(Av, Gv)
    for tile in (128, 256):
        C = torch.full((rows + 1, N), 7.0, dtype=BF16, device=DEV)
        f.gemm_bias_act(A, G, a_s, g_s, C[:rows], M=M, N=N, K=K, rows=rows, splits=splits, tile_n=tile)
        close_bf16(C[:rows], product_of_one[:rows], e1[:rows])
        assert (C[rows] == 7.0).all()


def test_one_matrix_in_both_places():
    """The same tensor as both weights of the gated product, in two calls on two streams at once."""
    M, N, K = 272, 256, 640
    (A, G, _, a_s, g_s, _), (Av, Gv, _) = gated_operands(M, M, N, K)
    h, err = gated_want(Av, Gv, Gv, "relu")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(f.gemm_gated(A, G, G, a_s, g_s, g_s, M=M, N=N, K=K, activation="relu", splits=1 + i % 3))
    torch.cuda.synchronize()
    for H in outs:
        close_bf16(H, h, err)



def test_side_by_side_on_four_streams_the_bits_stay_the_same():
    """The norm and every kind of fused kernel at once, so that each is held up by others at changing places."""
    def norm(rows, K, xt, rt):
        x = torch.randn(rows, K, device=DEV).to(xt)
        r = None if rt is None else torch.randn(rows, K, device=DEV).to(rt)
        w = torch.rand(K, device=DEV)
        return lambda: f.rmsnorm_quantize(x, w, residual=r)

    def gated(M, N, K, **kw):
        args, _ = gated_operands(M, M, N, K)
        return lambda: f.gemm_gated(*args, M=M, N=N, K=K, quantize=True, **kw)

    def act(M, N, K, **kw):
        (A, B, _, a_s, b_s, _), _ = gated_operands(M, M, N, K)
        bias, R = torch.randn(N, device=DEV), torch.randn(M, N, device=DEV).to(BF16)
        return lambda: (f.gemm_bias_act(A, B, a_s, b_s, M=M, N=N, K=K, bias=bias, activation="gelu", residual=R, **kw),)

    jobs = [norm(2048, 2048, F32, None), norm(1000, 7168, BF16, BF16), norm(3000, 512, BF16, None), norm(777, 4608, F32, F32), norm(40, 20480, F32, BF16),
            gated(272, 512, 1152, splits=3, tile_n=256), gated(64, 1024, 1024), gated(1040, 768, 512), act(1040, 1552, 384, tile_n=PAIR),
            act(528, 1040, 640, tile_n=128, splits=1), act(272, 528, 1024, splits=2, tile_n=128)]
    first = [job() for job in jobs]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for round_of_calls in range(10):
        outs = []
        for i, job in enumerate(jobs * 3):
            with torch.cuda.stream(streams[(i + round_of_calls) % 4]):
                outs.append((i % len(jobs), job()))
        torch.cuda.synchronize()
        for i, out in outs:
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(first[i], out)), i
    f.last_device_status()


FIRST_CALLS = """
import torch, fp8_quant_matmul_b200 as f
K, N = 256, 256
one = torch.ones(4096, device="cuda")
A, B = (torch.full((n * K,), 0x38, dtype=torch.uint8, device="cuda") for n in (160, N))       # ones
f.gemm(A, B, one, one, M=16, N=N, K=K)
torch.cuda.synchronize()
outs = []
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    for M in (16, 160):
        for splits in (0, 2):
            outs.append(f.gemm_bias_act(A, B, one, one, M=M, N=N, K=K, activation="relu", splits=splits))
            outs.append(f.gemm_gated(A, B, B, one, one, one, M=M, N=N, K=K, activation="none", splits=splits))
            outs.append(f.gemm_gated(A, B, B, one, one, one, M=M, N=N, K=K, activation="none", quantize=True, splits=splits)[1])
g.replay()
f.last_device_status()
for i in range(0, len(outs), 3):
    assert (outs[i] == 256).all() and (outs[i + 1] == 65536).all() and torch.allclose(outs[i + 2], one[:1] * 65536 / 448)
print("captured")
"""


def test_the_first_fused_calls_of_a_process_may_be_captured():
    """A process of its own: each kernel is set up by the first call that uses it, here under capture."""
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout + done.stderr
