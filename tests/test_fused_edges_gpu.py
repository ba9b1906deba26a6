"""Corners of gemm_bias_act and gemm_gated that the header allows."""
import pytest

import fp8_quant_matmul_b200 as f

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DEV = "cuda"
PAIR = 256 | f.TILE_PAIR


@pytest.mark.parametrize("M,splits,tile", [(16, 1, f.SMALL_M), (16, 2, f.SMALL_M), (144, 1, 128), (144, 1, PAIR), (144, 2, 128), (144, 2, 256)])
def test_the_pitch_of_a_single_row_does_not_matter(M, splits, tile):
    N, K = 272, 256
    g = torch.Generator().manual_seed(M)
    A = torch.randint(0x20, 0x40, (M * K,), dtype=torch.uint8, generator=g).to(DEV)
    B = torch.randint(0x20, 0x40, (N * K,), dtype=torch.uint8, generator=g).to(DEV)
    a_s, b_s = torch.rand(M * 2, generator=g).to(DEV), torch.rand(3 * 2, generator=g).to(DEV)
    R = torch.randn(1, N, generator=g).to(torch.bfloat16).to(DEV)
    want = f.gemm_bias_act(A, B, a_s, b_s, M=M, N=N, K=K, rows=1, residual=R, splits=splits, tile_n=tile)
    C = torch.full((3, N), 7.0, dtype=torch.bfloat16, device=DEV)
    rc = f.lib().fp8bs_gemm_bias_act(A.data_ptr(), B.data_ptr(), a_s.data_ptr(), b_s.data_ptr(), C[1:].data_ptr(), M, N, K, 1, None, 0, 0, R.data_ptr(), 1 << 50,
                                     splits, tile, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    f.last_device_status()
    assert torch.equal(C[1:2].view(torch.int16), want.view(torch.int16))
    assert (C[0] == 7.0).all() and (C[2] == 7.0).all()
