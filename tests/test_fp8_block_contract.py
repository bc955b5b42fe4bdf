"""What the block-scaled layers check before they launch, and how they behave inside autograd."""

import pytest
import torch

from olmo_core_b200.ops import fp8_block as fb

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _rand(shape, seed, device, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).bfloat16().to(device)


def _bad_main_grads(n, k, device):
    """(main_grad, what the message says) that do not fit a weight of n x k."""
    yield torch.zeros(n - 8, k, device=device), "does not fit"
    yield torch.zeros(n, k - 8, device=device), "does not fit"
    yield torch.zeros(k, n, device=device).t(), "does not fit"
    yield torch.zeros(1, k, device=device).expand(n, k), "does not fit"
    yield torch.zeros(n, k, dtype=torch.float64, device=device), "must be float32"
    if device == "cuda":
        yield torch.zeros(n, k), "must be float32 on"


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hp", [False, True])
def test_linear_refuses_a_main_grad_that_does_not_fit(hp, device):
    x, w = _rand((16, 64), 1, device), torch.nn.Parameter(_rand((48, 64), 2, device))
    for bad, text in _bad_main_grads(48, 64, device):
        w.main_grad = bad
        with pytest.raises(ValueError, match=text):
            fb.fp8_block_linear(x, w, wgrad_high_precision=hp)
        with torch.no_grad():  # nothing is going to be written
            assert fb.fp8_block_linear(x, w).shape == (16, 48)
    wide = torch.zeros(48, 72, device=device)
    w.main_grad = wide[:, :64]  # rows apart are fine
    fb.fp8_block_linear(x, w, wgrad_high_precision=hp).sum().backward()
    assert wide[:, :64].abs().sum() > 0 and (wide[:, 64:] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_experts_refuse_a_main_grad_that_does_not_fit(device):
    x, w = _rand((16, 64), 3, device), torch.nn.Parameter(_rand((2 * 48, 64), 4, device))
    offsets = torch.tensor([0, 5, 16], dtype=torch.int32, device=device)
    for bad, text in [*_bad_main_grads(96, 64, device), (torch.zeros(96, 72, device=device)[:, :64], "contiguous")]:
        w.main_grad = bad
        with pytest.raises(ValueError, match=text):
            fb.fp8_block_grouped_linear(x, w, offsets)
    w.main_grad = torch.zeros(2, 48, 64, device=device)
    fb.fp8_block_grouped_linear(x, w, offsets).sum().backward()
    assert w.main_grad.abs().sum() > 0


@pytest.mark.gpu
def test_kept_weights_of_another_size_are_refused():
    from olmo_core_b200.ops import _lib

    native, status = _lib.native(), _lib.status_buffer(torch.device("cuda", 0)).data_ptr()
    x, w = _rand((16, 64), 5, "cuda"), _rand((48, 64), 6, "cuda")
    offsets = torch.tensor([0, 5, 16], dtype=torch.int32, device="cuda")
    tiles = native.block_tile_buffer(w, 1)
    native.block_linear(x, w, w, tiles, None, False, status)
    for bad in (tiles[:-4], tiles.cpu(), tiles.view(torch.int32), native.block_tile_buffer(_rand((40, 64), 7, "cuda"), 1)):
        with pytest.raises(ValueError, match="kept 8-bit form"):
            native.block_linear(x, w, w, bad, None, False, status)
        with pytest.raises(ValueError, match="kept 8-bit form"):
            native.block_grouped_linear(x, w, w, offsets, bad, None, True, status)


def test_kernels_that_start_early_use_no_read_only_loads():
    """A kernel under programmatic dependent launch lives while its inputs are still written: the read-only path is not for it."""
    import re

    from olmo_core_b200.ops.build import CSRC_DIR

    early = [f for f in sorted(CSRC_DIR.glob("*.cu")) if "previous_kernel_done()" in f.read_text()]
    assert {f.name for f in early} == {"block_quant_sm100.cu", "gemm_block_fp8_sm100.cu"}
    for f in [*early, CSRC_DIR / "block_quant.cuh"]:
        code = re.sub(r"//[^\n]*", "", f.read_text())
        assert not re.search(r"__ldg|ld\.global\.nc|__restrict__|__ldcs|__ldca", code), f.name


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("constant", [False, True])
def test_layers_refuse_a_second_derivative(constant, grouped, device):
    x, w = _rand((16, 64), 8, device).requires_grad_(True), _rand((48, 64), 9, device).requires_grad_(True)
    offsets = torch.tensor([0, 5, 16], dtype=torch.int32, device=device)
    dy = _rand((16, 24 if grouped else 48), 10, device).requires_grad_(not constant)

    def grads(**kwargs):
        y = fb.fp8_block_grouped_linear(x, w, offsets) if grouped else fb.fp8_block_linear(x, w)
        return torch.autograd.grad(y, (x, w), dy, **kwargs)

    first = grads(create_graph=True)
    for a, b in zip(first, grads()):
        assert torch.equal(a, b)
    for g in first:
        with pytest.raises(RuntimeError, match="no second derivative"):
            (g.float().square().sum() + x.float().sum()).backward(retain_graph=True)
    x.float().square().sum().backward()  # a graph that does not pass through them is none of their business


@pytest.mark.gpu
def test_more_rows_and_matrices_than_a_grid_has_ctas_along_an_axis():
    rows = 65535 * 128 + 300  # 65538 tiles
    x = torch.randn(rows, 8, generator=torch.Generator(device="cuda").manual_seed(11), device="cuda").bfloat16()
    last = 65535 * 128 - 128  # the last tile of the first launch, and those behind it
    q, s = fb.quantize_block_rows(x)
    want_q, want_s = fb.quantize_block_rows(x[last:].cpu())
    assert torch.equal(q[last:].cpu(), want_q) and torch.equal(s[:, last:].cpu(), want_s)
    q, s = fb.quantize_block_columns(x)
    want_q, want_s = fb.quantize_block_columns(x[last:].cpu())
    assert torch.equal(q[last:].cpu(), want_q) and torch.equal(s[last // 128:].cpu(), want_s)
    qr, sr, qc, sc = fb.quantize_block_rows_columns(x)
    assert torch.equal(qc, q) and torch.equal(sc, s)
    q, s = fb.quantize_block_tiles(x)
    want_q, want_s = fb.quantize_block_tiles(x[last:].cpu())
    assert torch.equal(q[last:].cpu(), want_q) and torch.equal(s[last // 128:].cpu(), want_s)
    stack = x[:65540 * 2].view(65540, 2, 8)
    q, s = fb.quantize_block_tiles(stack)
    want_q, want_s = fb.quantize_block_tiles(stack.cpu())
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)


@pytest.mark.gpu
def test_linear_step_over_more_rows_than_one_launch_quantises():
    rows = 65535 * 128 + 300
    x = torch.randn(rows, 16, generator=torch.Generator(device="cuda").manual_seed(12), device="cuda").bfloat16().requires_grad_(True)
    w = _rand((24, 16), 13, "cuda").requires_grad_(True)
    dy = torch.zeros(rows, 24, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 65535 * 128 - 1, 65535 * 128, rows - 1], device="cuda")
    dy[at] = _rand((4, 24), 14, "cuda")
    y = fb.fp8_block_linear(x, w)
    y.backward(dy)
    few = x.detach()[at].requires_grad_(True)
    w2 = w.detach().clone().requires_grad_(True)
    yf = fb.fp8_block_linear(few, w2)
    yf.backward(dy[at])
    assert torch.equal(y[at], yf) and torch.equal(x.grad[at], few.grad)
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert (x.grad[rest] == 0).all()
    # the column blocks of both operands differ from those of the four rows alone, so the weight gradient is compared as numbers:
    # a product of two values off by half an e4m3 step each (2^-4)
    want = dy[at].double().t() @ x.detach()[at].double()
    bound = (2 * 2.0 ** -4 + 2.0 ** -8 + 2.0 ** -8) * (dy[at].double().abs().t() @ x.detach()[at].double().abs()) + 2.0 ** -8 * want.abs()
    floor = 2.0 ** -10 * x.detach().abs().max().double() * dy.abs().max().double() * 4  # codes below 2^-6 are off by 2^-10 of the scale
    assert ((w.grad.double() - want).abs() <= bound + 8 * floor).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_experts_marked_for_8_bits_run_in_8_bits(dtype, device):
    """On the CPU and for fp32 activations too, as the dense layers do."""
    from olmo_core_b200.float8 import BlockFloat8LinearConfig, Float8Config
    from olmo_core_b200.nn.moe.mlp import DroplessMoEMLP
    from olmo_core_b200.ops.elementwise import swiglu

    torch.manual_seed(0)
    mlp = DroplessMoEMLP(d_model=72, hidden_size=136, num_experts=3, dtype=dtype, init_device="cpu").to(device)
    Float8Config(block=BlockFloat8LinearConfig(), cache_weight_casts=True).apply_float8_linear(torch.nn.Sequential(mlp))
    x = _rand((40, 72), 15, device).to(dtype).requires_grad_(True)
    sizes = [13, 0, 27]
    y = mlp(x, sizes)
    assert y.dtype == dtype and set(mlp.float8["weight_cache"]) == {"w1", "w2", "w3"}
    offsets = torch.tensor([0, 13, 13, 40], dtype=torch.int32, device=device)
    a, b = (fb.fp8_block_grouped_linear(x, w, offsets).to(dtype) for w in (mlp.w1, mlp.w3))
    want = fb.fp8_block_grouped_linear(swiglu(a, b), mlp.w2, offsets, trans_b=False).to(dtype)
    assert torch.equal(y, want)
    y.float().square().sum().backward()
    assert x.grad.dtype == dtype and all(p.grad is not None and torch.isfinite(p.grad).all() for p in (mlp.w1, mlp.w2, mlp.w3))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grouped", [False, True])
def test_the_backward_pass_uses_the_main_grad_of_its_own_time(grouped, device):
    x, w = _rand((16, 64), 16, device), torch.nn.Parameter(_rand((48, 64), 17, device).float())
    offsets = torch.tensor([0, 5, 16], dtype=torch.int32, device=device)

    def forward():
        return (fb.fp8_block_grouped_linear(x, w, offsets) if grouped else fb.fp8_block_linear(x, w)).float().sum()

    forward().backward()
    want = w.grad
    w.grad, w.grad_added_to_main_grad = None, False
    y = forward()  # attached after the forward pass: an ordinary gradient
    w.main_grad = first = torch.zeros(48, 64, device=device)
    y.backward()
    assert torch.equal(w.grad, want) and not w.grad_added_to_main_grad and (first == 0).all()
    w.grad = None
    forward().backward()
    assert w.grad is None and w.grad_added_to_main_grad and torch.equal(first, want)
    w.grad_added_to_main_grad = False
    y = forward()  # replaced
    assert not w.grad_added_to_main_grad
    w.main_grad = second = torch.zeros(48, 64, device=device)
    y.backward()
    assert w.grad is None and w.grad_added_to_main_grad and torch.equal(second, want) and torch.equal(first, want)
    y = forward()  # replaced by one that does not fit
    w.main_grad = torch.zeros(40, 64, device=device)
    with pytest.raises(ValueError, match="does not fit"):
        y.backward()
    w.main_grad = second
    w.grad_added_to_main_grad = False
    y = forward()  # taken away
    del w.main_grad
    y.backward()
    assert torch.equal(w.grad, want) and torch.equal(second, want) and not w.grad_added_to_main_grad


@pytest.mark.parametrize("device", DEVICES)
def test_layer_refuses_shapes_that_are_no_matrix_product(device):
    x, w = _rand((4, 64), 18, device), _rand((48, 64), 19, device)
    for bad in ((x, w[0]), (x, w.view(2, 24, 64)), (x[0, 0], w), (x[0, 0], w[0])):
        with pytest.raises(ValueError, match="takes x"):
            fb.fp8_block_linear(*bad)
    q, s = fb.quantize_block_tiles(w)
    with pytest.raises(ValueError, match="features"):
        fb.fp8_block_matmul(x[0, 0], q, s)
    for shape in ((64,), (4, 64), (2, 2, 64), (0, 64), (2, 0, 64)):
        assert fb.fp8_block_linear(_rand(shape, 20, device), w).shape == (*shape[:-1], 48)
        assert fb.fp8_block_matmul(_rand(shape, 20, device), q, s).shape == (*shape[:-1], 48)
