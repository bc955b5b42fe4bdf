"""Routing: derivatives beyond the first gradient (second order, forward mode, torch.func transforms), accuracy, and rows of NaN."""

import pytest
import torch

from olmo_core_b200.ops.moe import _route_reference, route

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
OPTIONS = [dict(gating=gating, normalize=normalize, n_groups=groups, top_k_groups=max(1, groups // 2), biased=biased)
           for gating in ("softmax", "sigmoid") for normalize in (None, 1, 2) for groups, biased in ((1, False), (4, True))]
# fp32 sums of 32 terms of size one, a few operations deep on either side: 2^-24 times a hundred
TOLERANCE = dict(rtol=1e-5, atol=1e-5)


def _case(options, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    options = dict(options)
    x = torch.randn(9, 32, generator=g).to(device)
    options["score_bias"] = (torch.randn(32, generator=g) * 0.1).to(device) if options.pop("biased") else None
    d_weights, d_scores = torch.randn(9, 4, generator=g).to(device), torch.randn(9, 32, generator=g).to(device)
    return x, options, d_weights, d_scores


def _exact(x, experts, options):
    """weights and scores of the experts that were chosen, in fp64."""
    x = x.double()
    scores = x.softmax(-1) if options["gating"] == "softmax" else torch.sigmoid(x) + 1e-7
    weights = scores.gather(1, experts)
    return weights if options["normalize"] is None else weights / weights.norm(p=options["normalize"], dim=1, keepdim=True), scores


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("options", OPTIONS)
def test_second_order(options, device):
    x, options, dw, ds = _case(options, device)
    results = []
    for exact in (False, True):
        leaf = x.clone().requires_grad_(True)
        a, b = dw.clone().requires_grad_(True), ds.clone().requires_grad_(True)
        weights, experts, scores, _ = route(leaf, 4, **options)
        if exact:
            weights, scores = _exact(leaf, experts, options)
            a, b = a.double().detach().requires_grad_(True), b.double().detach().requires_grad_(True)
        (first,) = torch.autograd.grad((weights, scores), leaf, (a, b), create_graph=True)
        assert first.requires_grad
        loss = first.square().sum() + (first * x).sum() + weights.square().sum()
        results.append([first.detach(), *torch.autograd.grad(loss, (leaf, a, b))])
    for got, want in zip(*results):
        torch.testing.assert_close(got.double(), want.double(), **TOLERANCE)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", [0, 2])
def test_second_order_of_one_output_and_in_bf16(which, device):
    x, options, _, _ = _case(OPTIONS[1], device)
    leaf = x.bfloat16().requires_grad_(True)
    out = route(leaf, 4, **options)
    (first,) = torch.autograd.grad(out[which].square().sum(), leaf, create_graph=True)
    (second,) = torch.autograd.grad(first.float().square().sum(), leaf)
    assert first.dtype == second.dtype == torch.bfloat16
    first_of = torch.func.grad(lambda t: _exact(t, out[1], options)[which // 2].square().sum())
    exact = x.bfloat16().double()
    first, hessian = first_of(exact), torch.func.jacrev(first_of)(exact)
    want = (hessian * 2 * first).sum((2, 3))
    # the first gradient and the gradient that reaches it are rounded to bf16 (2^-8 each), and so is the result
    bound = (hessian.abs() * 4 * 2.0 ** -8 * first.abs()).sum((2, 3)) + 2.0 ** -8 * want.abs() + 1e-5
    assert ((second.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode(options, needs_grad, device):
    import torch.autograd.forward_ad as fwd

    x, options, _, _ = _case(options, device)
    tangent = torch.randn(9, 32, generator=torch.Generator().manual_seed(5)).to(device)
    with fwd.dual_level():
        weights, experts, scores, counts = route(fwd.make_dual(x.clone().requires_grad_(needs_grad), tangent), 4, **options)
        got = [fwd.unpack_dual(t).tangent for t in (weights, scores)]
        want = [fwd.unpack_dual(t).tangent for t in _exact(fwd.make_dual(x.double(), tangent.double()), experts, options)]
    assert all(t is not None for t in got)
    for a, b in zip(got, want):
        torch.testing.assert_close(a.double(), b, **TOLERANCE)
    plain = route(x, 4, **options)
    assert torch.equal(plain[1], experts) and torch.equal(plain[3], counts)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("options", OPTIONS[:2] + OPTIONS[-2:])
def test_func_transforms(options, device):
    x, options, dw, ds = _case(options, device)

    def loss(t):
        weights, _, scores, _ = route(t, 4, **options)
        return (weights * dw).sum() + (scores * ds).sum()

    leaf = x.clone().requires_grad_(True)
    loss(leaf).backward()
    torch.testing.assert_close(torch.func.grad(loss)(x), leaf.grad, **TOLERANCE)
    _, along = torch.func.jvp(loss, (x,), (dw.sum() * ds,))
    torch.testing.assert_close(along, (leaf.grad * dw.sum() * ds).sum(), rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
def test_router_module_second_order(gating, device):
    from olmo_core_b200.nn.moe.router import MoERouterConfig, MoERouterGatingFunction

    router = MoERouterConfig(top_k=2, gating_function=MoERouterGatingFunction(gating)).build(16, 8).to(device)
    x = torch.randn(1, 5, 16, generator=torch.Generator().manual_seed(1)).to(device).requires_grad_(True)
    weights, _, _, _ = router(x)
    (first,) = torch.autograd.grad(weights.square().sum(), x, create_graph=True)
    penalty = first.square().sum() + x.sum()  # another term carries a graph of its own
    (got,) = torch.autograd.grad(penalty, router.weight)
    assert got.abs().sum() > 0
    logits = router.get_expert_logits(x).view(5, 8)
    want_weights, _, _, _ = _route_reference(logits, 2, gating, None, 1, 1, 0)
    (first,) = torch.autograd.grad(want_weights.square().sum(), x, create_graph=True)
    (want,) = torch.autograd.grad(first.square().sum() + x.sum(), router.weight)
    torch.testing.assert_close(got, want, **TOLERANCE)


@pytest.mark.gpu
def test_the_kernels_op_itself_refuses_tangents():
    import torch.autograd.forward_ad as fwd

    from olmo_core_b200.ops import _lib

    x = torch.randn(3, 8, device="cuda")
    for needs_grad in (False, True):
        with fwd.dual_level(), pytest.raises(RuntimeError, match="tangents"):
            _lib.native().route.default(fwd.make_dual(x.clone().requires_grad_(needs_grad), x), 2, False, None, 1, 1, 0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("biased", [False, True])
def test_scores_weights_and_gradients_keep_their_relative_accuracy(biased, device):
    """Sigmoid scores over many magnitudes, with U = 2^-24 per rounding: the exponential 4 U (two steps), three more operations;
    weights: twice that, a sum of 4 and a division; gradient p (1 - p) = z / (1 + z)^2: 4 U of z, 2 (1 + 2) of 1 + z, four more."""
    U = 2.0 ** -24
    x = torch.linspace(-25, 25, 64 * 500).view(500, 64)[:, torch.randperm(64, generator=torch.Generator().manual_seed(2))].to(device)
    bias = torch.zeros(64, device=device) if biased else None
    leaf = x.clone().requires_grad_(True)
    weights, experts, scores, _ = route(leaf, 4, gating="sigmoid", score_bias=bias, normalize=1)
    d = torch.randn(500, 64, generator=torch.Generator().manual_seed(3)).to(device)
    (grad,) = torch.autograd.grad(scores, leaf, d)
    xd = x.double()
    want = torch.sigmoid(xd) + 1e-7
    assert ((scores.double() - want).abs() <= 8 * U * want).all()
    chosen = want.gather(1, experts)
    chosen = chosen / chosen.sum(1, keepdim=True)
    assert ((weights.double() - chosen).abs() <= 24 * U * chosen).all()
    if device == "cuda":  # the tensor form takes 1 - p as it comes
        slope = d.double() * torch.sigmoid(xd) * torch.sigmoid(-xd)
        assert ((grad.double() - slope).abs() <= 16 * U * slope.abs()).all()
    soft = route(x, 4, score_bias=bias)[2].double()
    want = xd.softmax(-1)
    # the difference to the maximum is rounded once (half a step of numbers up to 64: 32 U of the exponential), the exponential 4 U;
    # the same for the terms of the sum, whose own additions are 6 deep; reciprocal and product
    assert ((soft - want).abs() <= (2 * (32 + 4) + 8 + 3) * U * want).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("groups", [1, 4])
def test_a_row_of_nan_and_masked_logits_ranks_like_nan(groups, device):
    """Softmax scores of such a row are all NaN, so no expert is ahead of another, whatever the bias."""
    x = torch.randn(3, 16, generator=torch.Generator().manual_seed(6))
    x[1] = float("-inf")
    x[1, 5] = float("nan")
    bias = torch.linspace(-1, 1, 16)
    options = dict(score_bias=bias.to(device), n_groups=groups, top_k_groups=max(1, groups // 2))
    weights, experts, scores, _ = route(x.to(device), 4, **options)
    assert scores[1].isnan().all() and weights[1].isnan().all() and experts[1].tolist() == [0, 1, 2, 3]
    for t in (0, 2):
        alone = route(x[t:t + 1].to(device), 4, **options)
        assert torch.equal(alone[1][0], experts[t]) and torch.equal(alone[0][0], weights[t])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
def test_a_router_with_its_own_choice_is_asked_with_groups_too(gating, device):
    from olmo_core_b200.nn.moe.router import MoELinearRouter, MoERouterGatingFunction

    class Last(MoELinearRouter):
        def get_top_k(self, scores):
            indices = torch.arange(6, 8, device=scores.device).expand(*scores.shape[:-1], 2)
            return scores.gather(-1, indices), indices

    router = Last(d_model=16, num_experts=8, top_k=2, n_groups=4, top_k_groups=2, normalize_expert_weights=1.0,
                  gating_function=MoERouterGatingFunction(gating)).to(device)
    x = torch.randn(2, 3, 16, generator=torch.Generator().manual_seed(5)).to(device)
    weights, experts, counts, _ = router(x)
    assert experts.flatten().tolist() == [6, 7] * 6 and counts.flatten().tolist() == [0] * 6 + [6, 6]
    torch.testing.assert_close(weights.sum(-1), torch.ones(2, 3, device=device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("normalize", [1, 2])
@pytest.mark.parametrize("create_graph", [False, True])
def test_chosen_experts_without_any_weight_have_finite_gradients(create_graph, normalize, device):
    """The bias opens a group whose experts are all masked for the token: its weights are zero, and their gradient counts for nothing."""
    x = torch.randn(3, 8, generator=torch.Generator().manual_seed(7))
    x[1, 4:] = float("-inf")
    bias = torch.tensor([0.0] * 4 + [5.0] * 4)
    leaf = x.to(device).requires_grad_(True)
    weights, experts, scores, _ = route(leaf, 2, score_bias=bias.to(device), n_groups=2, top_k_groups=1, normalize=normalize)
    assert (weights[1] == 0).all() and experts[1].tolist() == [4, 5]
    dw, ds = torch.randn(3, 2, generator=torch.Generator().manual_seed(8)).to(device), torch.randn(3, 8, generator=torch.Generator().manual_seed(9)).to(device)
    (grad,) = torch.autograd.grad((weights, scores), leaf, (dw, ds), create_graph=create_graph)
    assert torch.isfinite(grad).all()
    s = x[1].to(device).double().softmax(0)
    want = s * (ds[1].double() - (s * ds[1].double()).sum())
    assert (grad[1].detach().double() - want).abs().max() <= 16 * 2.0 ** -24 * ds[1].abs().max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("normalize", [1, 2])
@pytest.mark.parametrize("create_graph", [False, True])
def test_small_scores_are_normalised_like_large_ones(create_graph, normalize, device):
    """Logits 30 to 82 below the best ones: the squares of their scores leave fp32 long before they do. Where all chosen scores are below
    2^-120 = e^-83.2 (a gap of 82 and a sum of four: e^-82 / 4 = e^-83.4) weights are zero."""
    U = 2.0 ** -24
    gaps = torch.tensor([30.0, 45.0, 60.0, 75.0, 82.0, 85.0, 120.0])
    x = torch.randn(7, 8, generator=torch.Generator().manual_seed(10)) * 0.25
    x[:, 4:] -= gaps[:, None]
    bias = torch.tensor([0.0] * 4 + [5.0] * 4)  # opens the group of the small ones
    leaf = x.to(device).requires_grad_(True)
    weights, experts, scores, _ = route(leaf, 3, score_bias=bias.to(device), n_groups=2, top_k_groups=1, normalize=normalize)
    assert (experts >= 4).all()
    dw = torch.randn(7, 3, generator=torch.Generator().manual_seed(11)).to(device)
    (grad,) = torch.autograd.grad(weights, leaf, dw, create_graph=create_graph)
    exact = x.to(device).double().requires_grad_(True)
    chosen = exact.softmax(-1).gather(1, experts)
    want = chosen / chosen.norm(p=normalize, dim=1, keepdim=True)
    (slope,) = torch.autograd.grad(want, exact, dw.double())
    # the exponential of a difference of up to 128, rounded to 64 U of it, twice; weights and gradients are of size one
    tolerance = (2 * 64 + 64) * U
    some = chosen.amax(1) >= 2.0 ** -120
    assert some.tolist() == [True] * 4 + [False] * 3
    assert (weights[some].double() - want[some]).abs().max() <= tolerance
    assert (grad[some].detach().double() - slope[some]).abs().max() <= 8 * tolerance * dw.abs().max()
    assert (weights[~some] == 0).all() and (grad[~some] == 0).all()
