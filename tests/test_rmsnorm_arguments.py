"""What rmsnorm_quantize refuses, in the binding and in the library, before anything is launched.  Runs without a GPU."""
import ctypes

import pytest

import fp8_quant_matmul_b200 as f

torch = pytest.importorskip("torch")


def test_binding_refuses_cpu_tensors():
    before = f.launch_count()
    with pytest.raises(ValueError):
        f.rmsnorm_quantize(torch.zeros(4, 256), torch.ones(256))
    assert f.launch_count() == before


def c_call(X=0x1000, xb=1, ldx=256, r=0x2000, rb=1, ldr=256, ro=0x3000, w=0x4000, wb=1, A=0x5000, s=0x6000, rows=4, K=256, eps=1e-6,
           fp8_max=448.0):
    p = lambda v: ctypes.c_void_p(v) if v else None
    return f.lib().fp8bs_rmsnorm_quantize(p(X), xb, ldx, p(r), rb, ldr, p(ro), p(w), wb, p(A), p(s), rows, K, eps, fp8_max, None)


@pytest.mark.parametrize("kw,code", [
    (dict(X=0), -1), (dict(w=0), -1), (dict(A=0), -1), (dict(s=0), -1), (dict(ro=0), -1),
    (dict(rows=0), -2), (dict(rows=-1), -2), (dict(K=0), -2), (dict(K=200), -2), (dict(rows=0x7fffffff), -2),
    (dict(ldx=128), -5), (dict(ldr=252), -5), (dict(ldx=260), -3), (dict(ldr=257), -3), (dict(ldx=258, xb=0), -3),
    (dict(X=0x1004), -3), (dict(X=0x1008, xb=0), -3), (dict(r=0x2002), -3), (dict(ro=0x3008, rb=0), -3), (dict(w=0x4004), -3),
    (dict(A=0x5008), -3), (dict(s=0x6002), -3),
    # the sum over the residual or X, but not element on element: other pitches, types, places
    (dict(ro=0x2000, ldr=512), -5), (dict(ro=0x1000, ldx=512), -5), (dict(ro=0x1000, xb=0), -5), (dict(ro=0x1000, rb=0, ldr=256, r=0x8000), -5),
    (dict(ro=0x2010), -5), (dict(ro=0x17f0), -5), (dict(ro=0x27f0), -5),
    (dict(fp8_max=0.0), -5), (dict(fp8_max=449.0), -5), (dict(fp8_max=float("nan")), -5), (dict(eps=-1.0), -5), (dict(eps=float("nan")), -5),
], ids=lambda v: str(v).replace(" ", "") if isinstance(v, dict) else "")
def test_library_refuses(kw, code):
    before = f.launch_count()
    assert c_call(**kw) == code
    assert f.launch_count() == before


def test_without_a_device_it_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert c_call() == -6
    assert c_call(r=0, ro=0, ldr=0) == -6          # no residual: its arguments are not looked at
    assert c_call(ro=0x2000) == -6 and c_call(ro=0x1000) == -6 and c_call(ro=0x1000, ldx=512, rows=1) == -6       # in place
    assert c_call(ro=0x2800) == -6 and c_call(ro=0x1800) == -6                                                     # side by side
