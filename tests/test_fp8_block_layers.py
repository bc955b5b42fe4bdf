"""Block-scaled e4m3 layers and expert routing together: configuration, mixtures, generation and a training step."""

import pytest
import torch

from olmo_core_b200.exceptions import OLMoConfigurationError
from olmo_core_b200.float8 import AOMXLinearConfig, BlockFloat8LinearConfig, Float8Config, refresh_float8_scales
from olmo_core_b200.nn.feed_forward import Linear
from olmo_core_b200.nn.moe import MoEConfig, MoERouterConfig, MoEType
from olmo_core_b200.nn.moe.router import MoERouterGatingFunction
from olmo_core_b200.nn.transformer import TransformerConfig
from olmo_core_b200.ops import fp8_block as fb

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(device, **kwargs):
    torch.manual_seed(0)
    return TransformerConfig.olmo2_30M(vocab_size=512, n_layers=2, **kwargs).build(init_device="cpu").to(device, torch.bfloat16)


@pytest.mark.parametrize("device", DEVICES)
def test_config_marks_layers_and_they_run_the_block_kernels(device):
    model = _model(device)
    config = Float8Config(block=BlockFloat8LinearConfig(), cache_weight_casts=True, modules_to_ignore=["*.feed_forward.w2"])
    model.apply_fp8(config)
    marked = {n: m for n, m in model.named_modules() if getattr(m, "float8", None) is not None}
    assert marked and all(isinstance(m, Linear) for m in marked.values())
    assert not any(n.startswith("lm_head") or n.endswith("feed_forward.w2") for n in marked)
    ids = torch.randint(0, 512, (2, 48), device=device)
    out = model(ids)
    out.float().square().mean().backward()
    assert torch.isfinite(out).all()
    for m in marked.values():
        assert m.weight.grad is not None and torch.isfinite(m.weight.grad).all() and m.weight.grad.abs().sum() > 0
        assert set(m.float8["weight_cache"]) == {"block_tiles"}
        x = torch.randn(5, m.in_features, device=device, dtype=torch.bfloat16)
        assert torch.equal(m(x), fb.fp8_block_linear(x, m.weight, m.bias))
    with torch.no_grad():
        next(iter(marked.values())).weight.mul_(2.0)  # a changed weight drops its kept form, also without the hook
    name, m = next(iter(marked.items()))
    x = torch.randn(5, m.in_features, device=device, dtype=torch.bfloat16)
    assert torch.equal(m(x), fb.fp8_block_linear(x, m.weight, m.bias))
    refresh_float8_scales(model)
    assert all(not m.float8["weight_cache"] for m in marked.values())


def test_config_refusals_and_serialised_form():
    with pytest.raises(OLMoConfigurationError, match="at most one"):
        Float8Config(block=BlockFloat8LinearConfig(), ao_mx=AOMXLinearConfig())
    config = Float8Config(block=BlockFloat8LinearConfig(wgrad_high_precision=True))
    assert Float8Config.from_dict(config.as_config_dict()) == config
    lin = torch.nn.Sequential(Linear(36, 44, False, torch.float32, "cpu"), Linear(40, 48, False, torch.float32, "cpu"))
    config.apply_float8_linear(lin)  # a bf16 weight gradient needs widths that are multiples of 8
    assert getattr(lin[0], "float8", None) is None and lin[1].float8["block"].wgrad_high_precision


@pytest.mark.parametrize("device", DEVICES)
def test_cache_made_under_inference_mode_serves_training(device):
    lin = Linear(64, 48, False, torch.bfloat16, "cpu").to(device)
    Float8Config(block=BlockFloat8LinearConfig(), cache_weight_casts=True).apply_float8_linear(torch.nn.Sequential(lin))
    x = torch.randn(7, 64, device=device, dtype=torch.bfloat16)
    with torch.inference_mode():
        first = lin(x).clone()
    y = lin(x)
    y.sum().backward()
    assert torch.equal(first, y) and lin.weight.grad is not None


def _quantized(t, rows, cols):
    q, s = fb._emulate_block_quantize(t.cpu().bfloat16(), rows, cols)
    s = s.repeat_interleave(rows, 0)[: t.shape[0]].repeat_interleave(cols, 1)[:, : t.shape[1]]
    return q.view(torch.float8_e4m3fn).double() * s.double()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 200, 3000])
def test_mixture_of_experts_block_in_8_bits(tokens):
    """Routing with bias and groups, sorting, experts in 8 bits, weighted sum: against the same chain in fp64."""
    torch.manual_seed(1)
    E, d, h, k = 16, 136, 200, 4
    moe = MoEConfig(name=MoEType.dropless, num_experts=E, hidden_size=h, router=MoERouterConfig(
        top_k=k, n_groups=4, top_k_groups=2, bias_gamma=1e-3, normalize_expert_weights=1.0,
        gating_function=MoERouterGatingFunction.sigmoid)).build(d, init_device="cpu").to("cuda")
    moe.router.score_bias.uniform_(-0.1, 0.1)
    moe.experts.to(torch.bfloat16)
    Float8Config(block=BlockFloat8LinearConfig()).apply_float8_linear(moe)
    assert moe.experts.mlp.float8 is not None
    x = torch.randn(1, tokens, d, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = moe(x)
    g = torch.randn_like(out)
    out.backward(g)
    assert torch.isfinite(x.grad).all()
    assert all(torch.isfinite(p.grad).all() for p in moe.parameters())

    weights, experts, _, _ = moe.router(x.detach())
    w1, w2, w3 = (w.detach().cpu().view(E, h, d) for w in (moe.experts.mlp.w1, moe.experts.mlp.w2, moe.experts.mlp.w3))
    want = torch.zeros(tokens, d, dtype=torch.float64)
    xq = _quantized(x.detach()[0], 1, 128)
    for e in range(E):
        t, j = (experts[0].cpu() == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        a = (xq[t] @ _quantized(w1[e], 128, 128).t()).bfloat16()
        b = (xq[t] @ _quantized(w3[e], 128, 128).t()).bfloat16()
        act = (torch.nn.functional.silu(a.double()) * b.double()).bfloat16()
        y = (_quantized(act, 1, 128) @ _quantized(w2[e], 128, 128)).bfloat16()
        want[t] += weights[0].detach().cpu().double()[t, j, None] * y.double()
    # roundings to bf16 of the experts' result and of the sum: 2 x 2^-8 at most. A bf16 rounding of a, b or the activation falls
    # the other way for fewer than one element in a hundred (fp32 against fp64 sums), which moves its 8-bit code by a step of 2^-3
    # at most: sqrt(0.01) 2^-3 = 2^-6.3 of the norm.
    err = (out.detach()[0].double().cpu() - want).norm() / want.norm()
    assert err <= 2 * 2.0 ** -8 + 2.0 ** -6


@pytest.mark.parametrize("device", DEVICES)
def test_generation_with_weights_in_8_bits(device):
    from olmo_core_b200.generate.generation_module.config import GenerationConfig
    from olmo_core_b200.generate.generation_module.transformer import TransformerGenerationModule

    model = _model(device)
    module = TransformerGenerationModule(
        model, GenerationConfig(max_new_tokens=6, do_sample=False, use_cache=True, pad_token_id=0, eos_token_id=511),
        float8_config=Float8Config(block=BlockFloat8LinearConfig()), device=torch.device(device))
    ids = torch.randint(1, 500, (2, 9), device=device)
    first, _, _ = module.generate_batch(ids, log_timing=False)
    caches = [m.float8["weight_cache"] for m in model.modules() if getattr(m, "float8", None) is not None]
    assert caches and all(set(c) == {"block_tiles"} for c in caches)
    again, _, _ = module.generate_batch(ids, log_timing=False)
    assert torch.equal(first, again) and first.shape[0] == 2


@pytest.mark.gpu
def test_training_steps_with_block_layers():
    from olmo_core_b200.config import DType
    from olmo_core_b200.optim import AdamWConfig
    from olmo_core_b200.train.train_module import TransformerDataParallelConfig, TransformerTrainModuleConfig

    device = torch.device("cuda", 0)
    model = TransformerConfig.olmo2_30M(vocab_size=1024, n_layers=2).build(init_device="meta")
    module = TransformerTrainModuleConfig(
        rank_microbatch_size=2 * 128, max_sequence_length=128, optim=AdamWConfig(lr=1e-3), max_grad_norm=1.0,
        float8_config=Float8Config(block=BlockFloat8LinearConfig(), cache_weight_casts=True),
        dp_config=TransformerDataParallelConfig(name="fsdp", param_dtype=DType.bfloat16)).build(model, device=device)
    ids = torch.randint(0, 1024, (4, 128))
    for _ in range(2):
        module.zero_grads()
        module.train_batch({"input_ids": ids})
        grads = [p.main_grad for p in model.parameters() if getattr(p, "main_grad", None) is not None]
        assert grads and all(torch.isfinite(t).all() for t in grads)
        module.optim_step()
        assert torch.isfinite(module.latest_ce_loss)


@pytest.mark.parametrize("device", DEVICES)
def test_experts_main_grad_and_cache(device):
    G, K, N, sizes = 5, 72, 136, [20, 0, 33, 1, 140]
    g = torch.Generator().manual_seed(3)
    x = torch.randn(sum(sizes), K, generator=g).bfloat16().to(device).requires_grad_(True)
    w = torch.nn.Parameter((torch.randn(G * N, K, generator=g) * 0.1).to(device))
    offsets = torch.tensor([0] + sizes, dtype=torch.int32).cumsum(0).to(torch.int32).to(device)
    dy = torch.randn(sum(sizes), N, generator=g).bfloat16().to(device)
    y = fb.fp8_block_grouped_linear(x, w, offsets)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dw.dtype == torch.float32 and dw.shape == w.shape
    w.main_grad, w.grad_added_to_main_grad = torch.ones(G * N, K, device=device), False
    cache = {}
    for n in (1, 2):
        again = fb.fp8_block_grouped_linear(x, w, offsets, weight_cache=cache)
        assert torch.equal(again, y) and set(cache) == {"block_tiles"}
        x.grad = None
        again.backward(dy)
        assert w.grad is None and w.grad_added_to_main_grad and torch.equal(x.grad, dx)
        # one more fp32 addition per pass
        torch.testing.assert_close(w.main_grad, n * dw + 1, rtol=4 * 2.0 ** -24 * n, atol=4 * 2.0 ** -24 * n)
    with torch.no_grad():
        none = fb.fp8_block_grouped_linear(x[:0], w, torch.zeros(G + 1, dtype=torch.int32, device=device))
    assert none.shape == (0, N)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [5, 300])
def test_training_step_in_a_graph_and_on_other_streams(tokens):
    """Linear layer, experts and routing forward and backward: captured and replayed, and on two streams at once."""
    from olmo_core_b200.ops.moe import route

    g = torch.Generator().manual_seed(4)

    def make(seed):
        g.manual_seed(seed)
        x = torch.randn(tokens, 264, generator=g).bfloat16().cuda().requires_grad_(True)
        w = (torch.randn(136, 264, generator=g) * 0.1).bfloat16().cuda().requires_grad_(True)
        we = (torch.randn(4 * 136, 264, generator=g) * 0.1).bfloat16().cuda().requires_grad_(True)
        logits = torch.randn(tokens, 32, generator=g).cuda().requires_grad_(True)
        dy = torch.randn(tokens, 136, generator=g).bfloat16().cuda()
        offsets = torch.tensor([0, tokens // 3, tokens // 2, tokens // 2, tokens], dtype=torch.int32, device="cuda")
        return x, w, we, logits, dy, offsets

    def step(x, w, we, logits, dy, offsets):
        y = fb.fp8_block_linear(x, w)
        ye = fb.fp8_block_grouped_linear(x, we, offsets)
        weights, experts, scores, counts = route(logits, 4, gating="sigmoid", n_groups=4, top_k_groups=2, normalize=1)
        grads = torch.autograd.grad((y, ye, weights, scores), (x, w, we, logits), (dy, dy, weights.detach(), scores.detach()))
        return [t.detach() for t in (y, ye, weights, experts, scores, counts, *grads)]

    states = [make(1), make(2)]
    want = [step(*s) for s in states]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    got = []
    for stream, s in zip(streams, states):  # nothing waits between the two
        with torch.cuda.stream(stream):
            for _ in range(3):
                out = step(*s)
            got.append(out)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs = []
    for stream, s in zip(streams, states):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(*s)
        graphs.append((graph, out))
    for _ in range(2):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for a, (_, b) in zip(want, graphs):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("device", DEVICES)
def test_layers_and_routing_under_activation_checkpointing(device):
    from torch.utils.checkpoint import checkpoint

    from olmo_core_b200.ops import fp8_block as fb
    from olmo_core_b200.ops.moe import route

    gen = torch.Generator().manual_seed(3)
    x, w, wr = (torch.randn(*shape, generator=gen).to(device, torch.bfloat16) for shape in ((200, 64), (64, 64), (8, 64)))

    def block(x, w, wr):
        h = fb.fp8_block_linear(x, w)
        weights, experts, _, _ = route((h @ wr.t()).float(), 2, normalize=1)
        return (h.float() * weights.gather(1, experts.argsort(1)).sum(1, keepdim=True)).sum()

    grads = []
    for wrapped in (False, True):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, wr)]
        loss = checkpoint(block, *leaves, use_reentrant=False) if wrapped else block(*leaves)
        loss.backward()
        grads.append([loss.detach()] + [t.grad for t in leaves])
    for a, b in zip(*grads):
        assert torch.equal(a, b)
