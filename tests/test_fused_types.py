"""The types of the operands of gemm_bias_act and gemm_gated: bytes of another format, or scales that are not fp32, are refused before
anything is launched.  Runs without a GPU."""
import pytest

import fp8_quant_matmul_b200 as f
from fp8_quant_matmul_b200 import api

torch = pytest.importorskip("torch")
M, N, K = 32, 64, 256


class OnDevice(torch.Tensor):
    """A tensor that says it is on device 0."""
    is_cuda = True

    def get_device(self):
        return 0


def on_device(n, dtype):
    size = torch.empty(0, dtype=dtype).element_size()
    return torch.zeros(n * size, dtype=torch.uint8).view(dtype).as_subclass(OnDevice)


GOOD = dict(A=(M * K, torch.uint8), B=(N * K, torch.uint8), up=(N * K, torch.float8_e4m3fn), a=(M * K // 128, torch.float32),
            b=(K // 128, torch.float32), u=(K // 128, torch.float32))


def operands(**dtypes):
    return {k: on_device(n, dtypes.get(k, t)) for k, (n, t) in GOOD.items()}


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(api, "_call", lambda name, index, *args: seen.append(name))
    return seen


def bias_act(t):
    f.gemm_bias_act(t["A"], t["B"], t["a"], t["b"], C=on_device(M * N, torch.bfloat16).view(M, N), M=M, N=N, K=K)


def gated(t):
    f.gemm_gated(t["A"], t["B"], t["up"], t["a"], t["b"], t["u"], M=M, N=N, K=K, H=on_device(M * N, torch.bfloat16).view(M, N))


@pytest.mark.parametrize("which,dtype", [("A", t) for t in (torch.uint8, torch.float8_e4m3fn)] + [("B", t) for t in (torch.uint8, torch.float8_e4m3fn)])
def test_both_types_of_bytes_are_taken(calls, which, dtype):
    t = operands(**{which: dtype})
    bias_act(t)
    gated(t)
    assert calls == ["fp8bs_gemm_bias_act", "fp8bs_gemm_gated"]


@pytest.mark.parametrize("which,dtype", [(w, t) for w in ("A", "B") for t in (torch.int8, torch.bool, torch.float8_e4m3fnuz, torch.float8_e5m2)]
                         + [(w, t) for w in ("a", "b") for t in (torch.int32, torch.uint8, torch.bfloat16, torch.float64)], ids=str)
def test_other_types_are_refused(calls, which, dtype):
    t = operands(**{which: dtype})
    with pytest.raises(ValueError, match="e4m3fn"):
        bias_act(t)
    with pytest.raises(ValueError, match="e4m3fn"):
        gated(t)
    assert calls == []


@pytest.mark.parametrize("which,dtype", [("up", torch.float8_e5m2), ("up", torch.int8), ("u", torch.int32), ("u", torch.float16)], ids=str)
def test_of_the_second_matrix_too(calls, which, dtype):
    with pytest.raises(ValueError, match="e4m3fn"):
        gated(operands(**{which: dtype}))
    assert calls == []
