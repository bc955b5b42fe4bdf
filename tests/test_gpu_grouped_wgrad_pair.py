"""Weight gradients of groups of rows on CTA pairs: element-wise against fp64, with everything outside a group poisoned."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _offsets(sizes):
    return torch.tensor([0] + sizes, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


@pytest.mark.parametrize("sizes", [[320], [257], [0, 0, 1030, 5], [640, 128, 64], [1900, 0, 333, 7, 1, 63, 65], [9000, 0, 17, 4500, 129] + [40] * 40, [11] * 299 + [90000]])
@pytest.mark.parametrize("M,N", [(136, 264), (256, 256), (520, 768)])
@pytest.mark.parametrize("form", ["bf16", "fp32", "accumulate"])
def test_against_fp64_and_the_single_cta_kernel(sizes, M, N, form):
    from olmo_core_b200.ops import _lib
    from olmo_core_b200.ops.gemm import grouped_gemm_wgrad

    gen = torch.Generator().manual_seed(len(sizes) + M)
    G, rows = len(sizes), sum(sizes)
    a, b = (torch.randn(rows + 70, n, generator=gen).to("cuda", torch.bfloat16) for n in (M, N))
    a[rows:], b[rows:] = float("nan"), float("inf")  # behind the last group
    base = torch.randn(G * M, N, generator=gen).cuda()
    offsets = _offsets(sizes)

    def run():
        out = base.clone() if form == "accumulate" else torch.full(
            (G * M, N), float("nan"), device="cuda", dtype=torch.bfloat16 if form == "bf16" else torch.float32)
        grouped_gemm_wgrad(a, b, offsets, out, accumulate=form == "accumulate")
        _lib.check_device_status()
        return out

    out = run()
    bounds = offsets.tolist()
    for g, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
        x, y = a[lo:hi].double(), b[lo:hi].double()
        want, size = x.t() @ y, x.abs().t() @ y.abs()
        got = out[g * M:(g + 1) * M].double()
        if form == "accumulate":
            want = want + base[g * M:(g + 1) * M].double()
            size = size + base[g * M:(g + 1) * M].double().abs()
        # sixteen products join the fp32 sum at a time; a product or sum that is cut off loses less than 2^-22 of the whole
        bound = ((hi - lo) / 16 + 17) * 2.0 ** -22 * size + (2.0 ** -8 * want.abs() if form == "bf16" else 0.0)
        assert bool(((got - want).abs() <= bound).all()), f"group {g}"
    assert torch.equal(out, run())
    old = _lib.lib().ocb_gemm_set_pair_mode(0)
    try:
        assert torch.equal(out, run())  # the same sums in the same order
    finally:
        _lib.lib().ocb_gemm_set_pair_mode(old)


def test_poisoned_neighbours_stay_out():
    from olmo_core_b200.ops.gemm import grouped_gemm_wgrad

    sizes = [30, 1100, 64, 1, 200]
    offsets = _offsets(sizes)
    a = torch.randn(sum(sizes), 256, device="cuda", dtype=torch.bfloat16)
    b = torch.randn(sum(sizes), 320, device="cuda", dtype=torch.bfloat16)
    bounds = offsets.tolist()
    clean = torch.empty(5 * 256, 320, device="cuda")
    grouped_gemm_wgrad(a, b, offsets, clean, accumulate=False)
    for g in range(5):
        for poison_a, poison_b in ((True, False), (False, True), (True, True)):
            pa, pb = a.clone(), b.clone()
            if poison_a:
                pa[bounds[g]:bounds[g + 1]] = float("nan")
            if poison_b:
                pb[bounds[g]:bounds[g + 1]] = float("inf")
            out = torch.empty(5 * 256, 320, device="cuda")
            grouped_gemm_wgrad(pa, pb, offsets, out, accumulate=False)
            keep = torch.ones(5, dtype=torch.bool, device="cuda")
            keep[g] = False
            assert torch.equal(out.view(5, -1)[keep], clean.view(5, -1)[keep])
