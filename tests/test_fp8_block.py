"""e4m3 products with one scale per block of 128: quantisers, dense and grouped products, layers; against fp64 arithmetic."""

import pytest
import torch

from olmo_core_b200.ops import fp8_block as fb

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U_BF16, U_F32 = 2.0 ** -8, 2.0 ** -24  # half a rounding step, relative


def _rand(shape, seed, device, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * std
    x = x * torch.exp(2 * torch.randn(shape[:-1] + (1,), generator=g))  # rows of very different magnitude
    return x.to(torch.bfloat16).to(device)


def _blocks_fp64(x, rows, cols):
    """(codes as fp64 values, scale of every element) of a matrix quantised over blocks of rows x cols, element by element."""
    x = x.double().cpu()
    R, C = x.shape
    q, s = torch.zeros_like(x), torch.ones_like(x)
    grid = torch.arange(0, 127, dtype=torch.float64)
    e, m = (grid // 8), grid % 8
    values = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7))  # the 127 magnitudes of e4m3
    for r in range(0, R, rows):
        for c in range(0, C, cols):
            b = x[r:r + rows, c:c + cols]
            top = b.abs().max().item()
            scale = 1.0
            if top > 0:
                scale = 2.0 ** -126
                while top / scale > 448:
                    scale *= 2
            v = (b / scale).abs()
            hi = torch.searchsorted(values, v.contiguous()).clamp(max=126)
            lo = (hi - 1).clamp(min=0)
            up, down = values[hi] - v, v - values[lo]
            pick = torch.where(up < down, hi, torch.where(up > down, lo, torch.where(hi % 2 == 0, hi, lo)))
            q[r:r + rows, c:c + cols] = torch.sign(b) * values[pick]
            s[r:r + rows, c:c + cols] = scale
    return q, s


def _val(q):
    return q.view(torch.float8_e4m3fn).double().cpu()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("R,C", [(1, 1), (3, 130), (128, 128), (129, 257), (260, 100)])
def test_quantisers_are_exact(R, C, device):
    x = _rand((R, C), 0, device)
    x.view(-1)[:: 7] = 0
    if R > 2:
        x[2] = 0  # blocks of zeros
        x[0, 0] = 3e-39  # a subnormal
    for fn, deq, rows, cols in ((fb.quantize_block_rows, fb.dequantize_block_rows, 1, 128),
                                (fb.quantize_block_columns, fb.dequantize_block_columns, 128, 1),
                                (fb.quantize_block_tiles, fb.dequantize_block_tiles, 128, 128)):
        q, s = fn(x)
        want_q, want_s = _blocks_fp64(x, rows, cols)
        assert q.shape == x.shape and q.dtype == torch.uint8 and s.dtype == torch.float32
        assert torch.equal(_val(q), want_q)
        assert torch.equal(deq(q, s).double().cpu(), (want_q * want_s).float().double())
    q, s, qc, sc = fb.quantize_block_rows_columns(x)
    for a, b in zip((q, s, qc, sc), fb.quantize_block_rows(x) + fb.quantize_block_columns(x)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_quantiser_borders(device):
    # 448 fits with scale 1, the next bf16 value above does not; ties go to the even code; the largest finite value fits
    x = torch.zeros(5, 128, dtype=torch.bfloat16)
    x[0, 0], x[1, 0], x[2, 0] = 448.0, 450.0, torch.finfo(torch.bfloat16).max
    x[3, :4] = torch.tensor([256.0, 17.0, 19.0, 21.0])  # steps of 2 in [16, 32): 17 -> 16, 19 -> 20, 21 -> 20
    x[4, 0], x[4, 1] = float("inf"), float("nan")
    q, s = fb.quantize_block_rows(x.to(device))
    v, s = _val(q), s.cpu()
    assert s[0].tolist()[:4] == [1.0, 2.0, 2.0 ** 120, 1.0]
    assert v[0, 0] == 448 and v[1, 0] == 224 and v[3, :4].tolist() == [256.0, 16.0, 20.0, 20.0]
    assert v[4, :2].isnan().all() and (v[4, 2:] == 0).all() and torch.isfinite(s).all()


@pytest.mark.parametrize("device", DEVICES)
def test_quantisers_take_strided_input_and_stacks(device):
    big = _rand((300, 401), 3, device)
    for x in (big[1:, 3:200], big.t()[:130, :77], big[::2]):
        for fn in (fb.quantize_block_rows, fb.quantize_block_columns, fb.quantize_block_tiles):
            for a, b in zip(fn(x), fn(x.contiguous())):
                assert torch.equal(a, b)
    w = _rand((3, 200, 150), 4, device)
    q, s = fb.quantize_block_tiles(w)
    for g in range(3):
        qg, sg = fb.quantize_block_tiles(w[g])
        assert torch.equal(q[g], qg) and torch.equal(s[g], sg)


def _operand(shape, seed, form, device):
    """(codes, scales, fp64 values); scales other than the ones that fit the codes."""
    x = _rand(shape, seed, device)
    fn, deq = {"rows": (fb.quantize_block_rows, fb.dequantize_block_rows),
               "columns": (fb.quantize_block_columns, fb.dequantize_block_columns),
               "tiles": (fb.quantize_block_tiles, fb.dequantize_block_tiles)}[form]
    q, s = fn(x)
    g = torch.Generator().manual_seed(seed + 1)
    s = s * torch.exp2(torch.randint(-6, 7, s.shape, generator=g).float()).to(device)
    expand = {"rows": lambda: s.t().repeat_interleave(128, 1)[:, : shape[1]],
              "columns": lambda: s.repeat_interleave(128, 0)[: shape[0]],
              "tiles": lambda: s.repeat_interleave(128, 0)[: shape[0]].repeat_interleave(128, 1)[:, : shape[1]]}[form]()
    return q, s, _val(q) * expand.double().cpu()


def _assert_product(out, a, b, base=None):
    """|error| of a dot product of K terms summed in fp32: K roundings of partial sums, one of the scaled block, one at the
    end; ``a [M, K]``, ``b [N, K]`` fp64."""
    K = a.shape[1]
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    if base is not None:
        ref, mag = ref + base, mag + base.abs()
    bound = (K + 4) * U_F32 * mag + (U_BF16 if out.dtype == torch.bfloat16 else U_F32) * ref.abs() + 1e-38
    err = (out.double().cpu() - ref).abs()
    assert (err <= bound).all(), (err / bound).max()


SHAPES = [(1, 1, 1), (1, 300, 520), (7, 128, 128), (100, 257, 129), (128, 256, 256), (129, 1001, 2050), (300, 40, 1000),
          (520, 513, 384), (16, 640, 1500), (33, 200, 260), (64, 130, 2000), (2560, 2050, 300)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("trans_a,trans_b,b_tiles", [(False, True, True), (False, False, True), (True, False, False),
                                                     (False, True, False), (True, True, True)])
def test_product(M, N, K, trans_a, trans_b, b_tiles, device):
    aq, sa, a = _operand((K, M) if trans_a else (M, K), 5, "columns" if trans_a else "rows", device)
    bform = "tiles" if b_tiles else ("rows" if trans_b else "columns")
    bq, sb, b = _operand((N, K) if trans_b else (K, N), 6, bform, device)
    a, b = a.t() if trans_a else a, b if trans_b else b.t()
    kw = dict(trans_a=trans_a, trans_b=trans_b, b_tiles=b_tiles)
    out = fb.gemm_fp8_block(aq, sa, bq, sb, **kw)
    assert out.dtype == torch.bfloat16
    _assert_product(out, a, b)
    _assert_product(fb.gemm_fp8_block(aq, sa, bq.view(torch.float8_e4m3fn), sb, out_dtype=torch.float32, **kw), a, b)
    base = torch.randn(M, N)
    wide = torch.full((M, N + 3), 7.0, device=device)
    acc = wide[:, 1:N + 1]
    acc.copy_(base)
    fb.gemm_fp8_block(aq, sa, bq, sb, out=acc, accumulate=True, **kw)
    _assert_product(acc, a, b, base.double())
    assert (wide[:, 0] == 7).all() and (wide[:, N + 1:] == 7).all()  # nothing beside the output is touched


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 1024, 4096), (640, 768, 512), (2048, 1000, 1160), (4096, 2304, 512)])
def test_product_repeats_bit_for_bit_and_replays(M, N, K):
    aq, sa, a = _operand((M, K), 7, "rows", "cuda")
    bq, sb, b = _operand((N, K), 8, "tiles", "cuda")
    first = fb.gemm_fp8_block(aq, sa, bq, sb)
    _assert_product(first, a, b)
    for _ in range(5):
        assert torch.equal(first, fb.gemm_fp8_block(aq, sa, bq, sb))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = fb.gemm_fp8_block(aq, sa, bq, sb)
            graphs.append((graph, out))
        for graph, out in graphs:
            graph.replay()
    side.synchronize()
    for _, out in graphs:
        assert torch.equal(first, out)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [3.0, 0.0, -2.0, float("inf"), float("nan"), 1e-40])
def test_scales_that_are_no_powers_of_two_show_as_nan(bad, device):
    aq, sa, a = _operand((140, 300), 27, "rows", device)
    bq, sb, b = _operand((200, 300), 28, "tiles", device)
    sa[1, 7], sb[1, 2] = bad, bad
    out = fb.gemm_fp8_block(aq, sa, bq, sb)
    assert out[7].isnan().all() and out[:, 128:].isnan().all()
    keep = [i for i in range(140) if i != 7]
    _assert_product(out[keep, :128], a[keep], b[:128])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 300, 520), (2, 700, 1536), (16, 129, 2050), (15, 2000, 130), (17, 64, 300), (0, 40, 256)])
def test_kept_weight_product_of_few_tokens(M, N, K, device):
    """Few rows are quantised inside the product: the same bits as quantising them first."""
    wide = _rand((M, K + 9), 33, device)
    wq, sw, w = _operand((N, K), 34, "tiles", device)
    for x in (wide[:, :K], wide[:, 3:K + 3], wide[:, 8:K + 8].contiguous()):
        y = fb.fp8_block_matmul(x, wq, sw)
        q, s = fb.quantize_block_rows(x)
        assert torch.equal(y, fb.gemm_fp8_block(q, s, wq, sw))
    bias = torch.ones(N, device=device)
    assert torch.equal(fb.fp8_block_matmul(x.view(M, 1, K), wq, sw, bias)[:, 0], y + 1)
    if M:
        x = x.clone()
        x[0, K // 2], x[-1, 0] = float("inf"), float("nan")
        assert fb.fp8_block_matmul(x, wq, sw)[[0, -1]].isnan().all()


GROUPS = [[128, 256, 128], [100, 0, 333, 7, 1], [0, 0, 5], [1, 1, 2, 0, 1, 3, 1, 1], [20, 0, 17, 3] * 10, [0] * 40 + [50, 33] + [0] * 3, [1000, 37, 0, 0, 513, 64, 65, 2]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sizes", GROUPS)
@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("K,N", [(256, 512), (320, 264), (130, 77)])
def test_grouped_product(sizes, trans_b, K, N, device):
    G, before, after = len(sizes), 3, 5
    R = sum(sizes) + before + after  # rows in front of the first group and behind the last belong to nobody
    aq, sa, a = _operand((R, K), 9, "rows", device)
    w = _rand((G, N, K) if trans_b else (G, K, N), 10, device)
    bq, sb = fb.quantize_block_tiles(w)
    bounds = [before]
    for n in sizes:
        bounds.append(bounds[-1] + n)
    out = torch.full((R, N), 7.0, dtype=torch.bfloat16, device=device)
    fb.grouped_gemm_fp8_block(aq, sa, bq, sb, torch.tensor(bounds, dtype=torch.int32, device=device), trans_b=trans_b, out=out)
    for g in range(G):
        lo, hi = bounds[g], bounds[g + 1]
        b = fb.dequantize_block_tiles(bq[g], sb[g]).double().cpu()
        if hi > lo:
            _assert_product(out[lo:hi], a[lo:hi], b if trans_b else b.t())
    assert (out[:before] == 7).all() and (out[bounds[-1]:] == 7).all()


def _assert_layer(x, w, g, y, dx, dw, hp):
    """The three products of the layer on operands quantised in fp64."""
    q = {n: (lambda t: t[0] * t[1])(_blocks_fp64(t, r, c)) for n, t, r, c in (
        ("x", x, 1, 128), ("w", w, 128, 128), ("g", g, 1, 128), ("xc", x, 128, 1), ("gc", g, 128, 1))}
    _assert_product(y, q["x"], q["w"])
    _assert_product(dx, q["g"], q["w"].t())
    if hp:
        _assert_product(dw, g.double().cpu().t(), x.double().cpu().t())
    else:
        _assert_product(dw, q["gc"].t(), q["xc"].t())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,N,K,hp", [(1, 24, 40, False), (130, 75, 201, False), (257, 264, 136, True), (300, 129, 520, False)])
def test_linear_gradients(M, N, K, hp, device):
    x, w, g = _rand((M, K), 11, device), _rand((N, K), 12, device, 0.1), _rand((M, N), 13, device)
    x.requires_grad_(True), w.requires_grad_(True)
    y = fb.fp8_block_linear(x.view(1, M, K), w, wgrad_high_precision=hp)
    assert y.shape == (1, M, N)
    y.backward(g.view(1, M, N))
    _assert_layer(x.detach(), w.detach(), g, y.detach()[0], x.grad, w.grad, hp)


@pytest.mark.parametrize("device", DEVICES)
def test_linear_main_grad_cache_and_frozen_operands(device):
    M, N, K = 200, 136, 264
    x, w, g = _rand((M, K), 14, device), torch.nn.Parameter(_rand((N, K), 15, device, 0.1).float()), _rand((M, N), 16, device)
    wide = fb.fp8_block_linear(x, w)
    dw, = torch.autograd.grad(wide, w, g)
    assert dw.dtype == torch.float32
    w.main_grad = torch.ones(N, K, device=device)
    cache = {}
    y = fb.fp8_block_linear(x, w, weight_cache=cache)
    assert torch.equal(y, wide) and set(cache) == {"block_tiles"}
    y.backward(g)
    assert w.grad is None
    torch.testing.assert_close(w.main_grad, dw + 1, rtol=4 * U_F32, atol=4 * U_F32)  # one more addition
    held = cache["block_tiles"][1]
    fb.fp8_block_linear(x, w, weight_cache=cache)
    assert cache["block_tiles"][1] is held
    del w.main_grad
    w.requires_grad_(False)
    x.requires_grad_(True)
    y = fb.fp8_block_linear(x, w)
    dx, = torch.autograd.grad(y, x, g)
    assert dx.shape == x.shape and torch.equal(y.detach(), wide.detach())
    assert torch.equal(fb.fp8_block_matmul(x.detach(), *fb.quantize_block_tiles(w)), wide.detach())
    none = fb.fp8_block_linear(x.detach()[:0], w)
    assert none.shape == (0, N)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hp", [False, True])
def test_linear_takes_broadcast_gradients_and_strided_input(hp, device):
    wide = _rand((40, 150), 30, device)
    w = _rand((72, 136), 31, device, 0.1).requires_grad_(True)
    for g in (torch.ones((), dtype=torch.bfloat16, device=device).expand(40, 72), _rand((1, 72), 32, device).expand(40, 72)):
        x = wide[:, 5:141].detach().requires_grad_(True)
        y = fb.fp8_block_linear(x, w, wgrad_high_precision=hp)
        dx, dw = torch.autograd.grad(y, (x, w), g)
        want = torch.autograd.grad(fb.fp8_block_linear(x.detach().clone().requires_grad_(True), w, wgrad_high_precision=hp), w, g.contiguous())
        assert torch.equal(dw, want[0])
        _assert_layer(x.detach(), w.detach(), g.contiguous(), y.detach(), dx, dw, hp)


@pytest.mark.parametrize("device", DEVICES)
def test_linear_gradient_against_differences(device):
    """Inputs that e4m3 holds exactly leave only the products, which are linear: differences of the output equal the gradient."""
    g = torch.Generator().manual_seed(17)
    x = torch.randint(-8, 9, (5, 256), generator=g).bfloat16().to(device).requires_grad_(True)
    w = torch.randint(-8, 9, (136, 256), generator=g).bfloat16().to(device)
    c = torch.randint(-2, 3, (5, 136), generator=g).bfloat16().to(device)
    x.data[:, ::128] = 8  # every block keeps its scale when another element moves
    y = fb.fp8_block_linear(x, w)
    dx, = torch.autograd.grad(y, x, c)
    for r, k in ((0, 3), (2, 130), (4, 255)):
        up = x.detach().clone()
        up[r, k] = 1.0 - up[r, k]
        step = (up[r, k] - x.detach()[r, k]).item()
        hi = fb.gemm_fp8_block(*fb.quantize_block_rows(up), *fb.quantize_block_tiles(w), out_dtype=torch.float32)
        lo = fb.gemm_fp8_block(*fb.quantize_block_rows(x.detach()), *fb.quantize_block_tiles(w), out_dtype=torch.float32)
        want = ((hi - lo).double() * c.double()).sum().item() / step
        assert abs(dx[r, k].item() - want) <= U_BF16 * abs(want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("sizes", [[100, 0, 133, 7, 1], [1, 2, 0, 1], [0, 21, 3, 0, 1, 1, 0, 9]])
def test_grouped_linear_gradients(sizes, trans_b, device):
    G, K, N = len(sizes), 136, 72
    R = sum(sizes)
    x, g = _rand((R, K), 18, device), _rand((R, N), 19, device)
    w = _rand((G, N, K) if trans_b else (G, K, N), 20, device, 0.1)
    flat = w.reshape(-1, w.shape[-1]).clone().requires_grad_(True)
    offsets = torch.tensor([0] + sizes, dtype=torch.int32).cumsum(0).to(torch.int32).to(device)
    x.requires_grad_(True)
    y = fb.fp8_block_grouped_linear(x, flat, offsets, trans_b=trans_b)
    y.backward(g)
    dw = flat.grad.view(w.shape)
    for i in range(G):
        lo, hi = int(offsets[i]), int(offsets[i + 1])
        if hi == lo:
            assert (dw[i] == 0).all()
            continue
        wi, dwi = (w[i], dw[i]) if trans_b else (w[i].t().contiguous(), dw[i].t())
        _assert_layer(x.detach()[lo:hi], wi, g[lo:hi], y.detach()[lo:hi], x.grad[lo:hi], dwi, True)
    q, s = fb.quantize_block_tiles(w)
    assert torch.equal(fb.fp8_block_grouped_matmul(x.detach(), q, s, offsets, trans_b=trans_b), y.detach())
    xq, xs = fb.quantize_block_rows(x.detach())  # few rows per group are quantised inside the product: the same bits
    assert torch.equal(fb.grouped_gemm_fp8_block(xq, xs, q, s, offsets, trans_b=trans_b), y.detach())


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    aq, sa = fb.quantize_block_rows(_rand((10, 200), 21, device))
    bq, sb = fb.quantize_block_tiles(_rand((30, 200), 22, device))
    ok = dict(a_q=aq, a_s=sa, b_q=bq, b_s=sb)
    fb.gemm_fp8_block(**ok)
    for change, text in (
        (dict(a_q=aq[0]), "dimensions"), (dict(a_q=aq.float()), "e4m3 bytes"), (dict(b_q=bq[:, :100]), "inner dimensions"),
        (dict(a_s=sa.t()), "shape"), (dict(b_s=sb.double()), "float32"), (dict(b_s=sb[:, :1]), "shape"),
        (dict(b_tiles=False), "shape"), (dict(accumulate=True), "needs an output"),
        (dict(out=torch.empty(10, 31, device=device)), "expected"), (dict(out_dtype=torch.float16), "writes"),
        (dict(out=torch.empty(10, 30, dtype=torch.bfloat16, device=device), accumulate=True), "writes"),
        (dict(out=torch.empty(30, 10, device=device).t()), "contiguous"),
    ):
        with pytest.raises(ValueError, match=text):
            fb.gemm_fp8_block(**{**ok, **change})
    if device == "cuda":
        for bad in (aq.contiguous()[:, 1:], torch.empty(10, 200, dtype=torch.uint8, device=device), aq.t().contiguous().t()):
            with pytest.raises(ValueError, match="16-byte"):
                fb.gemm_fp8_block(bad, sa[: (bad.shape[1] + 127) // 128], bq[:, : bad.shape[1]], sb)
        with pytest.raises(ValueError, match="is on"):
            fb.gemm_fp8_block(aq, sa.cpu(), bq, sb)
    wq, ws = fb.quantize_block_tiles(_rand((2, 30, 200), 23, device))
    off = torch.tensor([0, 4, 10], dtype=torch.int32, device=device)
    for change, text in ((dict(offsets=off.long()), "int32"), (dict(offsets=off[:2]), "int32"), (dict(b_q=wq[0]), "dimensions"),
                         (dict(b_s=ws[:1]), "shape"), (dict(out=torch.empty(10, 30, device=device)), "bfloat16")):
        with pytest.raises(ValueError, match=text):
            fb.grouped_gemm_fp8_block(**{**dict(a_q=aq, a_s=sa, b_q=wq, b_s=ws, offsets=off), **change})
    with pytest.raises(ValueError, match="features"):
        fb.fp8_block_linear(_rand((4, 100), 24, device), _rand((8, 104), 25, device))
    with pytest.raises(ValueError, match="stack"):
        fb.fp8_block_grouped_linear(_rand((10, 104), 24, device), _rand((9, 104), 25, device), off)
    with pytest.raises(ValueError, match="multiples of 8"):
        fb.fp8_block_grouped_linear(_rand((10, 100), 24, device), _rand((20, 100), 25, device), off)
    with pytest.raises(ValueError, match="dimensions"):
        fb.quantize_block_rows(_rand((2, 3, 4), 26, device))


@pytest.mark.parametrize("device", DEVICES)
def test_dimensions_beyond_32_bits_are_refused(device):
    long = torch.zeros(1, 1, dtype=torch.bfloat16, device=device).expand(2 ** 31 - 100, 1)  # no memory behind it
    w, codes = torch.ones(8, 1, dtype=torch.bfloat16, device=device), torch.zeros(1, 16, dtype=torch.uint8, device=device)
    q, s = fb.quantize_block_tiles(w)
    for call in (lambda: fb.quantize_block_rows(long), lambda: fb.quantize_block_columns(long), lambda: fb.quantize_block_tiles(long),
                 lambda: fb.gemm_fp8_block(codes.expand(2 ** 31 - 100, 16), s, q, s), lambda: fb.fp8_block_matmul(long, q, s),
                 lambda: fb.fp8_block_linear(long, w), lambda: fb.fp8_block_linear(w, long)):
        with pytest.raises(ValueError, match="too large|no dimension above"):
            call()
