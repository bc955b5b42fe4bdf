"""Ops that launch from C++ (torch.ops.ocb_native) keep to what holds for every launcher: counted, ranged, refusals as KernelError."""

import pytest
import torch

from olmo_core_b200.ops import _lib
from olmo_core_b200.ops import fp8_block as fb
from olmo_core_b200.ops.moe import route

pytestmark = pytest.mark.gpu


def _leaf(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(1)).bfloat16().cuda().requires_grad_(True)


OFFSETS = [0, 30, 64]
# (forward, entry points of the forward and of the backward pass)
CALLS = {
    "route": (lambda: route(_leaf(64, 32).float(), 4)[0], ["ocb_moe_route"], ["ocb_moe_route_grad"]),
    "linear": (lambda: fb.fp8_block_linear(_leaf(64, 128), _leaf(48, 128)),
               ["ocb_quantize_block_fp8", "ocb_linear_block_fp8"], ["ocb_linear_block_fp8", "ocb_gemm_block_fp8"]),
    "linear, bf16 weight gradient": (lambda: fb.fp8_block_linear(_leaf(64, 128), _leaf(48, 128), wgrad_high_precision=True),
                                     ["ocb_quantize_block_fp8", "ocb_linear_block_fp8"], ["ocb_linear_block_fp8", "ocb_gemm_bf16"]),
    "experts": (lambda: fb.fp8_block_grouped_linear(_leaf(64, 128), _leaf(96, 128), torch.tensor(OFFSETS, dtype=torch.int32).cuda()),
                ["ocb_quantize_block_fp8", "ocb_linear_block_fp8"], ["ocb_linear_block_fp8", "ocb_grouped_gemm_bf16"]),
    "kept weight": (lambda: fb.fp8_block_matmul(_leaf(64, 128), *fb.quantize_block_tiles(_leaf(48, 128).detach())),
                    ["ocb_quantize_block_fp8", "ocb_linear_block_fp8"], []),
}


@pytest.mark.parametrize("name", CALLS)
def test_launches_are_counted_both_ways(name):
    forward, there, back = CALLS[name]
    before = _lib.launch_count
    y = forward()
    assert _lib.launch_count == before + len(there)
    if back:
        y.sum().backward()
        assert _lib.launch_count == before + len(there) + len(back)


def test_a_refused_launch_is_a_kernel_error():
    with pytest.raises(_lib.KernelError, match="ocb_moe_route failed with code -1"):
        _lib.native().route.default(torch.zeros(2, 4, device="cuda"), 9, False, None, 1, 1, 0)
    x = torch.zeros(2, 4, device="cuda", requires_grad=True)
    with pytest.raises(_lib.KernelError, match="ocb_moe_route failed with code -1"):
        _lib.native().route.default(x, 9, False, None, 1, 1, 0)


def test_a_launch_refused_in_a_backward_pass_is_a_kernel_error():
    x, w = _leaf(64, 128), _leaf(48, 128)
    native = _lib.native()
    # through the op itself: a bf16 weight gradient whose width is no multiple of 8, which the Python form refuses beforehand
    narrow, w = x[:, :124].contiguous(), w[:, :124].contiguous()
    y = native.block_linear.default(narrow, w, w.detach(), None, None, True, _lib.status_buffer(x.device).data_ptr())
    with pytest.raises(_lib.KernelError, match="ocb_gemm_bf16 failed with code"):
        y.sum().backward()


@pytest.mark.parametrize("name", CALLS)
def test_ranges_surround_the_launchers_both_ways(name, monkeypatch):
    forward, there, back = CALLS[name]
    forward()
    seen, depth = [], [0]

    def push(what):
        seen.append(what)
        depth[0] += 1

    def pop():
        depth[0] -= 1

    monkeypatch.setattr(torch.cuda.nvtx, "range_push", push)
    monkeypatch.setattr(torch.cuda.nvtx, "range_pop", pop)
    _lib.set_nvtx(True)
    try:
        y = forward()
        assert seen == there and depth == [0]
        if back:
            y.sum().backward()
            assert seen == there + back and depth == [0]
    finally:
        _lib.set_nvtx(False)
    count = len(seen)
    forward()
    assert len(seen) == count
