"""What gemm_bias_act and gemm_gated refuse, in the binding and in the library, before anything is launched.  Runs without a GPU."""
import ctypes

import pytest

import fp8_quant_matmul_b200 as f
from fp8_quant_matmul_b200 import api

torch = pytest.importorskip("torch")
PAIR = 256 | f.TILE_PAIR


def p(v):
    return ctypes.c_void_p(v) if v else None


def bias_act(A=0x1000, B=0x2000, a=0x3000, b=0x4000, C=0x500000, M=128, N=256, K=512, rows=128, bias=0x6000, bb=0, act=0, r=0x7000, ldr=256, splits=0,
             tile=0):
    return f.lib().fp8bs_gemm_bias_act(p(A), p(B), p(a), p(b), p(C), M, N, K, rows, p(bias), bb, act, p(r), ldr, splits, tile, None)


def gated(A=0x1000, G=0x2000, U=0x2800, a=0x3000, g=0x4000, u=0x4800, H=0x5000, s=0x6000, M=128, N=256, K=512, rows=128, act=2, fp8_max=448.0, splits=0,
          tile=0):
    return f.lib().fp8bs_gemm_gated(p(A), p(G), p(U), p(a), p(g), p(u), p(H), p(s), M, N, K, rows, act, fp8_max, splits, tile, None)


@pytest.mark.parametrize("kw,code", [
    (dict(A=0), -1), (dict(B=0), -1), (dict(a=0), -1), (dict(b=0), -1), (dict(C=0), -1),
    (dict(M=0, rows=0), -2), (dict(N=0), -2), (dict(K=100), -2), (dict(M=120, rows=120), -3), (dict(N=200), -3), (dict(rows=0), -2), (dict(rows=129), -2),
    (dict(A=0x1008), -3), (dict(B=0x2001), -3), (dict(C=0x5002), -3), (dict(a=0x3004), -3), (dict(b=0x4002), -3), (dict(bias=0x6004), -3),
    (dict(r=0x7008), -3), (dict(ldr=260), -3), (dict(ldr=248), -5),
    (dict(r=0x500000, ldr=512), -5), (dict(r=0x500010), -5), (dict(r=0x4fffe0), -5), (dict(r=0x500000 - 127 * 1024 - 512 + 16, ldr=512), -5),
    (dict(act=-1), -5), (dict(act=5), -5), (dict(splits=-1), -5), (dict(splits=5), -5), (dict(K=2048, splits=9), -5),
    (dict(tile=192), -5), (dict(tile=256, splits=1), -5), (dict(tile=PAIR, splits=2), -5), (dict(tile=128 | f.TILE_PAIR), -5),
    (dict(tile=f.SMALL_M), -5), (dict(tile=f.SMALL_M | 256, M=64, rows=64), -5), (dict(tile=128 | f.SPLIT_WORKSPACE), -5), (dict(tile=f.STREAM_K), -5),
    (dict(tile=256 | f.SHORT_K, K=256), -5),
], ids=lambda v: str(v).replace(" ", "") if isinstance(v, dict) else "")
def test_bias_act_refuses(kw, code):
    before = f.launch_count()
    assert bias_act(**kw) == code
    assert f.launch_count() == before


@pytest.mark.parametrize("kw,code", [
    (dict(A=0), -1), (dict(G=0), -1), (dict(U=0), -1), (dict(a=0), -1), (dict(g=0), -1), (dict(u=0), -1), (dict(H=0), -1),
    (dict(K=0), -2), (dict(K=130), -2), (dict(N=208), -2), (dict(s=0, N=200), -3), (dict(rows=0), -2), (dict(rows=200), -2), (dict(M=100, rows=1), -3),
    (dict(U=0x2808), -3), (dict(H=0x5004), -3), (dict(s=0x6002), -3), (dict(u=0x4801), -3),
    (dict(act=9), -5), (dict(fp8_max=0.0), -5), (dict(fp8_max=500.0), -5), (dict(fp8_max=float("nan")), -5),
    (dict(tile=128), -5), (dict(tile=PAIR, splits=3), -5), (dict(splits=8), -5), (dict(tile=f.SMALL_M), -5),
], ids=lambda v: str(v).replace(" ", "") if isinstance(v, dict) else "")
def test_gated_refuses(kw, code):
    before = f.launch_count()
    assert gated(**kw) == code
    assert f.launch_count() == before


def test_without_a_device_valid_calls_are_an_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for kw in (dict(), dict(tile=128), dict(tile=PAIR), dict(splits=2, tile=256), dict(M=64, rows=60, tile=f.SMALL_M), dict(M=16, rows=1, r=0, ldr=0, bias=0)):
        assert bias_act(**kw) == -6
    # the residual is C, or lies in front of it or behind it
    for kw in (dict(r=0x500000), dict(r=0x500000, ldr=512, rows=1), dict(r=0x500000 + 0x10000), dict(r=0x500000 - 0x10000)):
        assert bias_act(**kw) == -6
    for kw in (dict(), dict(tile=256), dict(tile=PAIR), dict(splits=3), dict(s=0, N=208, fp8_max=0.0), dict(M=16, rows=2, splits=4)):
        assert gated(**kw) == -6


class Fake:
    """As much of a CUDA tensor as an argument check looks at."""
    is_cuda = True

    def __init__(self, n, size, dtype=torch.uint8, shape=None, index=0, contiguous=True):
        self.n, self.size, self.dtype, self.shape, self.index, self.contiguous = n, size, dtype, shape or (n,), index, contiguous

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return self.contiguous

    def numel(self):
        return self.n

    def element_size(self):
        return self.size

    def stride(self, i):
        return (self.shape[1], 1)[i] if len(self.shape) == 2 else 1


def operands(**other):
    t = dict(A=Fake(32 * 256, 1), B=Fake(64 * 256, 1), a_scale=Fake(64, 4), b_scale=Fake(2, 4))
    t.update(other)
    return [t[k] for k in ("A", "B", "a_scale", "b_scale")]


@pytest.mark.parametrize("other", [dict(A=Fake(32 * 256 - 1, 1)), dict(B=Fake(64, 1)), dict(B=Fake(64 * 256, 1, index=1)), dict(a_scale=Fake(64, 2)),
                                   dict(b_scale=Fake(1, 4)), dict(B=Fake(64 * 256, 1, contiguous=False)), dict(a_scale=Fake(64, 4, index=-1))])
def test_binding_checks_the_operands(other):
    with pytest.raises(ValueError):
        f.gemm_bias_act(*operands(**other), M=32, N=64, K=256)
    A, B, a, b = operands(**other)
    with pytest.raises(ValueError):
        f.gemm_gated(A, B, B, a, b, b, M=32, N=64, K=256)


@pytest.mark.parametrize("kw", [dict(activation="swish"), dict(rows=33), dict(rows=0), dict(M=None), dict(bias=Fake(64, 2, torch.float16)),
                                dict(bias=Fake(63, 4, torch.float32)), dict(bias=Fake(64, 4, torch.float32, index=1)),
                                dict(residual=Fake(32 * 64, 4, torch.float32, (32, 64))), dict(residual=Fake(31 * 64, 2, torch.bfloat16, (31, 64))),
                                dict(C=Fake(32 * 64, 2, torch.bfloat16, (32, 64), contiguous=False)), dict(C=Fake(32 * 64, 4, torch.float32, (32, 64)))])
def test_binding_checks_the_rest(kw):
    before = f.launch_count()
    with pytest.raises(ValueError):
        f.gemm_bias_act(*operands(), **{**dict(M=32, N=64, K=256), **kw})
    assert f.launch_count() == before


def test_binding_refuses_cpu_tensors():
    z, s = torch.zeros(16 * 128, dtype=torch.uint8), torch.ones(16)
    with pytest.raises(RuntimeError):
        f.gemm_bias_act(z, z, s, s, M=16, N=16, K=128)
    with pytest.raises(RuntimeError):
        f.gemm_gated(z, z, z, s, s, s, M=16, N=16, K=128)


def test_a_call_for_another_device_is_made_with_that_device_current(monkeypatch):
    """The library launches on the current device; the binding makes the tensors' device current around the call."""
    seen, current = [], [0]

    class On:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.was, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.was

    class Lib:
        def fp8bs_anything(self, *args):
            seen.append((current[0], args))
            return 0

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(api, "_stream", lambda index: 100 + index)
    monkeypatch.setattr(api, "lib", lambda: Lib())
    api._call("fp8bs_anything", 0, 1)
    api._call("fp8bs_anything", 1, 2)
    assert seen == [(0, (1, 100)), (1, (2, 101))] and current == [0]
