"""rmsnorm_quantize against the formula in 64 bits.

Tolerances, before any run.  s = x + r is one rounding of fp32, y = s * rstd * w three more on top of the error of rstd, half that
of the mean of squares: a square, sums over a lane's 4 columns, 32 lanes, 16 warps one after the other, 8 CTAs one after the other,
and one more addition per 8192 columns where a warp walks several blocks, the mean and eps: 1 + 2 + 5 + 16 + 8 + 2 + 3 = 37, 18.5 after
the root, which adds one.  The product with w, with rstd, the reciprocal, the scale and the inverse scale add one each: 24 roundings
of 2^-24 and the one of s bound the scales (SCALE_TOL: 26, counted up).  A byte is the value times scale, with three more, rounded to e4m3 once: at most half a step (2^-4 of the value's binade, 2^-10 below 2^-6) from the exact product,
and those 32 roundings (VALUE_TOL) of its value."""
import itertools

import pytest

import fp8_quant_matmul_b200 as f

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SCALE_TOL = 26 * 2.0 ** -24
VALUE_TOL = 32 * 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def make(rows, K, xt, rt, wt, seed, wide=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, wide or K, generator=g) * torch.exp(torch.randn(wide or K, generator=g))).to(xt).to(DEV)[:, (wide - K if wide else 0):]
    r = None if rt is None else (3 * torch.randn(rows, wide or K, generator=g)).to(rt).to(DEV)[:, :K]
    w = (1 + 0.3 * torch.randn(K, generator=g)).to(wt).to(DEV)
    return x, w, r


def want(x, w, r, eps, fp8_max):
    """(values before the rounding to 8 bits, inverse scales, sums), float64, rows padded to 16."""
    s = x.double() + (0 if r is None else r.double())
    rows, K = s.shape
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + eps) * w.double()
    M = (rows + 15) // 16 * 16
    full = torch.zeros(M, K, dtype=torch.float64, device=DEV)
    full[:rows] = y
    b = full.view(M, K // 128, 128)
    inv = b.abs().amax(2).clamp(min=1e-12) / fp8_max
    return (b / inv[:, :, None]).view(M, K), inv, s


def check(q, scales, values, inv):
    M, K = values.shape
    got = q.view(torch.float8_e4m3fn).view(K, M).t().double()
    assert ((scales.view(K // 128, M).t().double() - inv).abs() <= SCALE_TOL * inv).all()
    half_step = torch.exp2(torch.floor(torch.log2(values.abs().clamp(min=2.0 ** -6)))) * 2.0 ** -4
    assert ((got - values).abs() <= half_step + VALUE_TOL * values.abs()).all()


def check_sum(out, s):
    assert ((out.double() - s).abs() <= s.abs() * torch.finfo(out.dtype).eps / 2 * (1 + 2.0 ** -12) + 2.0 ** -24 * s.abs()).all()


SHAPES = [(1, 128), (1, 7168), (3, 384), (15, 1024), (16, 1152), (17, 2304), (40, 512), (333, 896), (2049, 1664), (7, 6272), (64, 8192), (5, 8320), (18, 14336), (18, 16384), (33, 20480), (19, 13312), (50, 5504)]


@pytest.mark.parametrize("rows,K", SHAPES)
@pytest.mark.parametrize("xt,rt", [(BF16, None), (F32, None), (BF16, BF16), (F32, F32)], ids=lambda t: str(t).replace("torch.", ""))
def test_against_64_bits(rows, K, xt, rt):
    x, w, r = make(rows, K, xt, rt, xt, seed=rows + K)
    out = f.rmsnorm_quantize(x, w, residual=r, eps=1e-5)
    values, inv, s = want(x, w, r, 1e-5, 448.0)
    check(out[0], out[1], values, inv)
    assert len(out) == (2 if r is None else 3)
    if r is not None:
        assert out[2].dtype is rt
        check_sum(out[2], s)


@pytest.mark.parametrize("xt,rt,wt", [t for t in itertools.product((BF16, F32), (None, BF16, F32), (BF16, F32))],
                         ids=lambda t: str(t).replace("torch.", ""))
def test_every_mix_of_types_on_column_slices(xt, rt, wt):
    x, w, r = make(50, 640, xt, rt, wt, seed=5, wide=648)
    assert not x.is_contiguous()
    out = f.rmsnorm_quantize(x, w, residual=r, eps=0.0, fp8_max=240.0)
    values, inv, s = want(x, w, r, 0.0, 240.0)
    check(out[0], out[1], values, inv)
    assert out[0].view(torch.float8_e4m3fn).float().abs().max() <= 240.0
    if r is not None:
        check_sum(out[2], s)


@pytest.mark.parametrize("K", [768, 9216, 17408])
@pytest.mark.parametrize("which", ["residual", "x"])
def test_the_sum_in_place(K, which):
    x, w, r = make(37, K, BF16, BF16, BF16, seed=9)
    a = f.rmsnorm_quantize(x, w, residual=r)
    target = r if which == "residual" else x
    b = f.rmsnorm_quantize(x, w, residual=r, residual_out=target)
    assert b[2] is target
    for p, q in zip(a, b):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))     # and the same call gives the same bits


def test_writes_nothing_but_its_outputs():
    rows, K, pad = 21, 384, 64
    x, w, r = make(rows, K, BF16, F32, F32, seed=11)
    M = 32
    q = torch.full((M * K + 2 * pad,), 0xAB, dtype=torch.uint8, device=DEV)
    sc = torch.full((M * 3 + 2 * pad,), -7.0, device=DEV)
    ro = torch.full((rows * K + 2 * pad,), -7.0, device=DEV)
    rc = f.lib().fp8bs_rmsnorm_quantize(x.data_ptr(), 1, K, r.data_ptr(), 0, K, ro[pad:].data_ptr(), w.data_ptr(), 0, q[pad:].data_ptr(),
                                        sc[pad:].data_ptr(), rows, K, 1e-6, 448.0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    for t, n, fill in ((q, M * K, 0xAB), (sc, M * 3, -7.0), (ro, rows * K, -7.0)):
        assert (t[:pad] == fill).all() and (t[pad + n:] == fill).all()
    values, inv, s = want(x, w, r, 1e-6, 448.0)
    check(q[pad:pad + M * K], sc[pad:pad + M * 3], values, inv)
    assert (q[pad:pad + M * K].view(K, M)[:, rows:] == 0).all()          # rows behind the last: zeros, of either sign none
    check_sum(ro[pad:pad + rows * K].view(rows, K), s)


def test_zeros_nan_and_infinity_stay_in_their_rows():
    rows, K = 20, 512
    x, w, _ = make(rows, K, F32, None, F32, seed=13)
    x[2] = 0.0
    x[5, 130] = float("nan")
    x[7, 300] = float("inf")
    x[19, 0] = float("-inf")
    q, sc = f.rmsnorm_quantize(x, w)
    M = 32
    q, sc = q.view(K, M).t(), sc.view(K // 128, M).t()
    nan = (q & 0x7F) == 0x7F
    assert ((q[2] & 0x7F) == 0).all() and sc[2].isfinite().all()
    assert nan[5].all() and sc[5].isnan().all()
    for row, block in ((7, 2), (19, 0)):                                 # 1 / inf = 0: the other blocks are zero
        hit = torch.zeros(K // 128, dtype=torch.bool, device=DEV)
        hit[block] = True
        assert torch.equal(sc[row].isnan(), hit)
        assert torch.equal(nan[row].view(-1, 128), hit[:, None].expand(-1, 128))
        assert ((q[row].view(-1, 128)[~hit] & 0x7F) == 0).all()
    good = [i for i in range(rows) if i not in (5, 7, 19)]
    values, inv, _ = want(x[good], w, None, 1e-6, 448.0)
    n = len(good)
    got = q[good].contiguous().view(torch.float8_e4m3fn).double()
    half_step = torch.exp2(torch.floor(torch.log2(values[:n].abs().clamp(min=2.0 ** -6)))) * 2.0 ** -4
    assert ((got - values[:n]).abs() <= half_step + VALUE_TOL * values[:n].abs()).all()


def test_streams_and_a_replayed_graph():
    x, w, r = make(130, 1536, BF16, BF16, BF16, seed=17)
    base = f.rmsnorm_quantize(x, w, residual=r)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(f.rmsnorm_quantize(x, w, residual=r))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = f.rmsnorm_quantize(x, w, residual=r)
    x2 = x.clone()
    x.mul_(2)
    graph.replay()
    want2 = f.rmsnorm_quantize(2 * x2, w, residual=r)
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(o, base))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(captured, want2))
    f.last_device_status()


def test_feeds_the_product():
    rows, K, N = 45, 1024, 384
    x, w, r = make(rows, K, BF16, BF16, BF16, seed=19)
    g = torch.Generator().manual_seed(20)
    W = (torch.randn(N, K, generator=g) * K ** -0.5).to(DEV)
    q, sc, _ = f.rmsnorm_quantize(x, w, residual=r)
    Bq, Bs = f.quantize_block(W)
    C = f.gemm(q, Bq, sc, Bs, M=48, N=N, K=K)
    A = q.view(torch.float8_e4m3fn).view(K, 48).t().double() * sc.double().view(K // 128, 48).t().repeat_interleave(128, 1)
    Bv = Bq.view(torch.float8_e4m3fn).view(K, N).t().double() * Bs.double().view(K // 128, N // 128).t().repeat_interleave(128, 1).repeat_interleave(128, 0)
    ref = A @ Bv.t()
    # bf16's half step, and K + K / 128 fp32 roundings of the sum of magnitudes
    assert ((C.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (K + 8) * 2.0 ** -24 * (A.abs() @ Bv.abs().t())).all()
    assert (C[rows:] == 0).all()


def test_offsets_beyond_32_bits():
    # 2.2e9 elements, in a slice of rows that are wider still
    rows, K, wide = 264000, 8192, 8320
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(rows, wide, device=DEV, generator=g, dtype=BF16)[:, 64:64 + K]
    r = torch.randn(rows, K, device=DEV, generator=g, dtype=BF16)
    w = torch.ones(K, device=DEV)
    pick = torch.tensor([0, 15, 16, rows // 2, rows - 33, rows - 1], device=DEV)
    values, inv, s = want(x[pick], w, r[pick], 1e-6, 448.0)
    q, sc, out = f.rmsnorm_quantize(x, w, residual=r, residual_out=r)
    n = len(pick)
    check_sum(out[pick], s)
    got_inv = sc.view(K // 128, rows)[:, pick].t().double()
    assert ((got_inv - inv[:n]).abs() <= SCALE_TOL * inv[:n]).all()
    got = q.view(torch.float8_e4m3fn).view(K, rows)[:, pick].t().double()
    half_step = torch.exp2(torch.floor(torch.log2(values[:n].abs().clamp(min=2.0 ** -6)))) * 2.0 ** -4
    assert ((got - values[:n]).abs() <= half_step + VALUE_TOL * values[:n].abs()).all()


def test_groups_at_odd_places_and_unaligned_bytes():
    # 16 rows of a column leave together with the 16 before them where both lie in one aligned 32 bytes: every start and every number of
    # groups, with outputs that begin on 16 but not on 32 bytes
    K = 256
    for rows in (16, 32, 48, 1000, 5000, 5016):
        for lead in (0, 16):
            x, w, r = make(rows, K, BF16, None, BF16, seed=rows)
            M = (rows + 15) // 16 * 16
            buf = torch.zeros(M * K + 64, dtype=torch.uint8, device=DEV)
            q = buf[lead:lead + M * K]
            sc = torch.zeros(M * K // 128, device=DEV)
            assert q.data_ptr() % 32 == lead
            assert f.lib().fp8bs_rmsnorm_quantize(x.data_ptr(), 1, K, None, 0, 0, None, w.data_ptr(), 1, q.data_ptr(), sc.data_ptr(), rows, K, 1e-6, 448.0,
                                                  torch.cuda.current_stream().cuda_stream) == 0
            values, inv, _ = want(x, w, None, 1e-6, 448.0)
            check(q, sc, values, inv)
            assert (buf[:lead] == 0).all() and (buf[lead + M * K:] == 0).all()


def test_the_first_call_of_a_shape_may_be_captured():
    """Shapes that no other test here uses: what the library asks the driver about them is asked under capture."""
    f.rmsnorm_quantize(torch.ones(16, 128, device="cuda"), torch.ones(128, device="cuda"))
    for K, xt in ((128 * 13, F32), (128 * 97, BF16)):
        x = torch.randn(37, K, device="cuda", generator=torch.Generator("cuda").manual_seed(K)).to(xt)
        w = torch.ones(K, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            q, s = f.rmsnorm_quantize(x, w)
        g.replay()
        torch.cuda.synchronize()
        q2, s2 = f.rmsnorm_quantize(x, w)
        assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("K", [1280, 20480])
def test_x_is_its_own_residual(K):
    x, w, _ = make(45, K, F32, None, F32, seed=21)
    values, inv, s = want(x, w, x, 1e-6, 448.0)
    a = f.rmsnorm_quantize(x, w, residual=x)
    check(a[0], a[1], values, inv)
    b = f.rmsnorm_quantize(x, w, residual=x, residual_out=x)             # all three one tensor
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))
    check_sum(x, s)


@pytest.mark.parametrize("xt,rt", [(F32, None), (BF16, None), (F32, F32), (BF16, BF16)], ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("K", [384, 2048, 4736])
def test_many_rounds_give_the_same_bits(K, xt, rt):
    """Many groups of rows per cluster, inputs that stay in L2: a box must not be filled again before its rows are in registers."""
    rows = 8000 * 2048 // max(K, 2048)
    x, w, r = make(rows, K, xt, rt, xt, seed=K + 1)
    values, inv, s = want(x, w, r, 1e-6, 448.0)
    first = f.rmsnorm_quantize(x, w, residual=r)
    check(first[0], first[1], values, inv)
    for _ in range(12):
        again = f.rmsnorm_quantize(x, w, residual=r)
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(first, again))
    f.last_device_status()


def test_the_pitch_of_a_single_row_does_not_matter():
    K = 640
    x, w, r = make(1, K, BF16, F32, F32, seed=31)
    a = f.rmsnorm_quantize(x, w, residual=r)
    q, sc, ro = torch.empty_like(a[0]), torch.empty_like(a[1]), torch.empty_like(a[2])
    rc = f.lib().fp8bs_rmsnorm_quantize(x.data_ptr(), 1, 1 << 50, r.data_ptr(), 0, 1 << 50, ro.data_ptr(), w.data_ptr(), 0, q.data_ptr(), sc.data_ptr(), 1, K, 1e-6, 448.0,
                                        torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert all(torch.equal(p.view(torch.uint8), o.view(torch.uint8)) for p, o in zip(a, (q, sc, ro)))
