"""Products of few rows against so many weight tiles that three CTAs share an SM: 297 to 444 tiles on 148 SMs."""

import pytest
import torch

from olmo_core_b200.ops import fp8_block as fb

pytestmark = pytest.mark.gpu
U_BF16, U_F32 = 2.0 ** -8, 2.0 ** -24  # half a step, relative


def _rand(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


def _assert_product(out, a, b):
    """K roundings of the fp32 sum, one of the result to bf16; ``a [M, K]``, ``b [N, K]`` fp64."""
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    assert ((out.double().cpu() - want).abs() <= (a.shape[1] + 4) * U_F32 * size + U_BF16 * want.abs()).all()


@pytest.mark.parametrize("M", [1, 3, 16])
@pytest.mark.parametrize("K", [130, 640])
def test_dense(M, K):
    N = 297 * 128 - 3
    x, (wq, sw) = _rand((M, K), 1).cuda(), fb.quantize_block_tiles(_rand((N, K), 2).cuda())
    w = fb.dequantize_block_tiles(wq, sw).double().cpu()
    xq, sx = fb.quantize_block_rows(x)
    first = fb.gemm_fp8_block(xq, sx, wq, sw)
    _assert_product(first, fb.dequantize_block_rows(xq, sx).double().cpu(), w)
    assert torch.equal(fb.fp8_block_matmul(x, wq, sw), first)  # quantised inside: the same bits
    for _ in range(3):
        assert torch.equal(fb.gemm_fp8_block(xq, sx, wq, sw), first)


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("K,N", [(130, 1000), (1160, 1000)])
@pytest.mark.parametrize("sizes", ["even", "uneven"])
def test_grouped(sizes, K, N, trans_b):
    # 128 rows in all, which fall evenly on 64 (1 - e^-2) = 55.3 groups: 443 of the 444 tiles that three CTAs per SM take at once
    G, before, after = 64, 2, 3
    n = [2] * 59 + [1] * 5 if sizes == "even" else [0, 5, 1, 0, 17, 2, 0, 33, 3, 0, 0, 62] + [0] * 52
    assert before + sum(n) + after == 128
    bounds = [before]
    for m in n:
        bounds.append(bounds[-1] + m)
    x = _rand((bounds[-1] + after, K), 3).cuda()
    wq, sw = fb.quantize_block_tiles(_rand((G, N, K) if trans_b else (G, K, N), 4).cuda())
    offsets = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    xq, sx = fb.quantize_block_rows(x)
    out = torch.full((x.shape[0], N), 7.0, dtype=torch.bfloat16, device="cuda")
    fb.grouped_gemm_fp8_block(xq, sx, wq, sw, offsets, trans_b=trans_b, out=out)
    a = fb.dequantize_block_rows(xq, sx).double().cpu()
    inside = fb.fp8_block_grouped_matmul(x, wq, sw, offsets, trans_b=trans_b)
    for g in range(G):
        rows = slice(bounds[g], bounds[g + 1])
        if n[g]:
            b = fb.dequantize_block_tiles(wq[g], sw[g]).double().cpu()
            _assert_product(out[rows], a[rows], b if trans_b else b.t())
            assert torch.equal(inside[rows], out[rows])
    assert (out[:before] == 7).all() and (out[bounds[-1]:] == 7).all()
