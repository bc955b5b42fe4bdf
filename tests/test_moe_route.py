"""Routing of tokens to experts: scores, bias, groups, top-k, normalised weights and the gradient, against fp64 arithmetic."""

import pytest
import torch

from olmo_core_b200.ops.moe import route

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24  # half a step of fp32, relative


def _want(x, k, gating, bias, n_groups, top_groups, normalize):
    """Straight from the definition, token by token, in fp64: (weights, experts, scores, counts)."""
    x = x.detach().double().cpu()
    n, e = x.shape
    weights, experts, counts = torch.zeros(n, k, dtype=torch.float64), torch.zeros(n, k, dtype=torch.long), torch.zeros(e, dtype=torch.int32)
    scores = torch.zeros(n, e, dtype=torch.float64)
    for t in range(n):
        if gating == "softmax":
            top = x[t].max()
            if top > float("-inf"):
                z = (x[t] - top).exp()
                scores[t] = z / z.sum()
        else:
            scores[t] = torch.sigmoid(x[t]) + 1e-7
        rank = scores[t] if bias is not None else x[t]
        if bias is not None:
            rank = rank + bias.double().cpu()
        ids = list(range(e))
        if n_groups > 1:
            size = e // n_groups
            r = scores[t] + (bias.double().cpu() if bias is not None else 0.0)
            value = [sum(sorted(r[g * size:(g + 1) * size].tolist(), reverse=True)[:2]) for g in range(n_groups)]
            kept = sorted(range(n_groups), key=lambda g: (-value[g], g))[:top_groups]
            ids = [i for i in ids if i // size in kept]
        chosen = sorted(ids, key=lambda i: (-rank[i].item(), i))[:k]
        experts[t] = torch.tensor(chosen)
        w = scores[t][experts[t]]
        if normalize:
            norm = w.sum() if normalize == 1 else w.square().sum().sqrt()
            w = w / norm if norm > 0 else torch.zeros_like(w)
        weights[t] = w
        for i in chosen:
            counts[i] += 1
    return weights, experts, scores, counts


def _score_bound(e):
    """Relative error of an fp32 score: exponential (2 + 1.173 |x| steps of 2^-23, |x| < 64 after subtracting the maximum), a
    sum of e terms, reciprocal, product."""
    return (2 * (2 + 1.173 * 64) + e + 4) * U


def _check(x, k, gating, bias, n_groups, top_groups, normalize, device):
    w, i, s, c = route(x.to(device), k, gating=gating, score_bias=None if bias is None else bias.to(device), n_groups=n_groups,
                       top_k_groups=top_groups, normalize=normalize)
    ww, wi, ws, wc = _want(x, k, gating, bias, n_groups, top_groups, normalize)
    assert w.dtype == s.dtype == torch.float32 and i.dtype == torch.int64 and c.dtype == torch.int32
    assert torch.equal(i.cpu(), wi)
    assert torch.equal(c.cpu(), wc)
    b = _score_bound(x.shape[1])
    torch.testing.assert_close(s.double().cpu(), ws, rtol=b, atol=2.0 ** -149)
    torch.testing.assert_close(w.double().cpu(), ww, rtol=2 * b + 40 * U, atol=2.0 ** -149)


def _logits(n, e, seed, dtype=torch.float32, std=1.5):
    return (torch.randn(n, e, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _bias(e, seed):
    return torch.randint(-100, 101, (e,), generator=torch.Generator().manual_seed(seed)).float() * 1e-3


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,e,k,groups,top_groups", [(1, 1, 1, 1, 1), (3, 7, 7, 1, 1), (65, 32, 2, 1, 1), (200, 64, 8, 1, 1),
                                                     (70, 100, 5, 4, 2), (300, 256, 8, 8, 4), (17, 48, 6, 16, 3), (9, 1024, 32, 32, 5),
                                                     (40, 31, 3, 31, 7), (33, 300, 12, 3, 1)])
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("normalize", [None, 1, 2])
def test_route(n, e, k, groups, top_groups, gating, biased, normalize, device):
    _check(_logits(n, e, 1), k, gating, _bias(e, 2) if biased else None, groups, top_groups, normalize, device)


@pytest.mark.parametrize("device", DEVICES)
def test_route_bf16_logits_many_tokens_and_strides(device):
    # bf16 logits repeat: ties go to the lower expert
    x = _logits(3000, 40, 3, torch.bfloat16)
    _check(x, 4, "softmax", None, 1, 1, None, device)
    wide = _logits(50, 90, 4)
    _check(wide[:, 10:74], 6, "sigmoid", _bias(64, 5), 4, 2, 1, device)
    _check(wide.t(), 6, "softmax", None, 2, 1, 1, device)
    w, i, s, c = route(x[:0].to(device), 4)
    assert w.shape == (0, 4) and s.shape == (0, 40) and (c == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_ties_masks_and_extremes(gating, groups, top_groups, biased, device):
    x = _logits(8, 32, 6)
    x[0] = 0.0  # every expert the same
    x[1] = float("-inf")  # nothing to choose from
    x[2, 5:] = float("-inf")  # five experts left
    x[3, ::2] = torch.finfo(torch.float32).min  # masked with the type's lowest value
    x[4] = torch.finfo(torch.float32).min
    x[5] = 1.0 + 2.0 ** -23 * torch.arange(32)  # scores that fp32 cannot tell apart
    x[6] = torch.where(torch.arange(32) < 16, 30.0, 20.0)  # saturated sigmoids
    x[7] *= 40
    bias = torch.zeros(32) if biased else None
    _check(x, 6, gating, bias, groups, top_groups, 1, device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("biased", [False, True])
def test_route_takes_zeros_of_both_signs_for_equal(gating, groups, biased, device):
    x = torch.zeros(3, 32)
    x[0, ::2] = -0.0
    x[1, :16] = -0.0
    x[2, 5] = -0.0
    _check(x, 6, gating, torch.full((32,), -0.0) if biased else None, groups, 2 if groups > 1 else 1, 1, device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_with_nan_and_infinity_stays_in_range(gating, groups, device):
    x = _logits(5, 32, 7)
    x[0] = float("nan")
    x[1, 3] = float("nan")
    x[2, 4:9] = float("inf")
    x[3, 20] = -float("nan")
    w, i, s, c = route(x.to(device), 4, gating=gating, n_groups=groups, top_k_groups=max(1, groups // 2), normalize=1)
    assert (i >= 0).all() and (i < 32).all() and c.sum() == 20
    assert all(len(set(row)) == 4 for row in i.tolist())
    if groups == 1 or gating == "sigmoid":  # NaN ranks above every number; one NaN makes all softmax scores (and groups) NaN
        assert i[1, 0] == 3 and i[3, 0] == 20
    ww, wi, ws, _ = _want(x[4:], 4, gating, None, groups, max(1, groups // 2), 1)
    assert torch.equal(i[4:].cpu(), wi)  # the other tokens do not notice
    torch.testing.assert_close(w[4:].double().cpu(), ww, rtol=1e-4, atol=0)


def _grads(x, k, dw, ds, device, dtype=torch.float32, **options):
    x = x.to(device).requires_grad_(True)
    w, i, s, _ = route(x, k, **options)
    outs, gs = [], []
    if dw is not None:
        outs.append(w), gs.append(dw.to(device))
    if ds is not None:
        outs.append(s), gs.append(ds.to(device))
    return torch.autograd.grad(outs, x, gs)[0], i.cpu()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,e,k,groups", [(1, 4, 1, 1), (65, 64, 8, 1), (33, 100, 12, 4), (7, 1024, 32, 8)])
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [None, 1, 2])
@pytest.mark.parametrize("which", ["both", "weights", "scores"])
def test_route_gradient(n, e, k, groups, gating, normalize, which, device):
    x = _logits(n, e, 8)
    g = torch.Generator().manual_seed(9)
    dw = torch.randn(n, k, generator=g) if which != "scores" else None
    ds = torch.randn(n, e, generator=g) * 0.1 if which != "weights" else None
    got, i = _grads(x, k, dw, ds, device, gating=gating, n_groups=groups, normalize=normalize)
    xd = x.double().requires_grad_(True)
    s = xd.softmax(-1) if gating == "softmax" else torch.sigmoid(xd) + 1e-7
    w = s.gather(1, i)
    if normalize:
        w = w / w.norm(p=normalize, dim=-1, keepdim=True)
    total = (0.0 if dw is None else (w * dw.double()).sum()) + (0.0 if ds is None else (s * ds.double()).sum())
    want, = torch.autograd.grad(total, xd)
    # every addend of a logit's gradient is a product of scores (or 1 / norm) and upstream gradients: relative errors of a few
    # scores on the size of the largest addend, which the row's upstream gradients and its largest weight bound
    size = torch.zeros(n, 1, dtype=torch.float64)
    if dw is not None:
        size += dw.double().abs().sum(1, keepdim=True) * (2.0 if normalize else 1.0)
    if ds is not None:
        size += ds.double().abs().max(1, keepdim=True)[0] * (2.0 if gating == "softmax" else 1.0)
    assert ((got.double().cpu() - want).abs() <= 4 * _score_bound(e) * size).all()


@pytest.mark.parametrize("device", DEVICES)
def test_route_gradient_against_differences_and_bf16(device):
    x = _logits(4, 24, 10)
    g = torch.Generator().manual_seed(11)
    dw, ds = torch.randn(4, 3, generator=g).double(), torch.randn(4, 24, generator=g).double()
    options = dict(gating="sigmoid", n_groups=4, top_k_groups=2, normalize=1, score_bias=_bias(24, 12).to(device))
    got, i = _grads(x, 3, dw.float(), ds.float(), device, **options)

    def value(t):
        w, idx, s, _ = _want(t, 3, "sigmoid", _bias(24, 12), 4, 2, 1)
        assert torch.equal(idx, i)  # the choice does not move with these steps
        return ((w * dw).sum() + (s * ds).sum()).item()

    h = 1e-5
    for t, e in ((0, 0), (1, int(i[1, 0])), (2, int(i[2, 2])), (3, 23)):
        step = torch.zeros(4, 24, dtype=torch.float64)
        step[t, e] = h
        want = (value(x.double() + step) - value(x.double() - step)) / (2 * h)
        # second-order term of the central difference (third derivatives are below 100 here) and the fp64 rounding of it
        assert abs(got[t, e].item() - want) <= 100 * h * h + 1e-9 + 1e-4 * max(1.0, abs(want)) * 0.1
    xb = x.bfloat16()
    gb, ib = _grads(xb, 3, dw.float(), ds.float(), device, **options)
    gf, _ = _grads(xb.float(), 3, dw.float(), ds.float(), device, **options)
    assert gb.dtype == torch.bfloat16
    torch.testing.assert_close(gb, gf.bfloat16(), rtol=2.0 ** -7, atol=1e-9)


@pytest.mark.gpu
def test_route_repeats_and_replays_in_two_graphs():
    x = _logits(2000, 256, 13).cuda()
    bias = _bias(256, 14).cuda()
    call = lambda: route(x, 8, gating="sigmoid", score_bias=bias, n_groups=8, top_k_groups=4, normalize=1)  # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = call()
            graphs.append((graph, out))
        for _ in range(2):
            for graph, _ in graphs:
                graph.replay()
    side.synchronize()
    for _, out in graphs:
        for a, b in zip(first, out):
            assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_route_refusals(device):
    x = _logits(4, 32, 15).to(device)
    for args, kwargs, text in (((x[0], 2), {}, "logits"), ((x.double(), 2), {}, "logits"), ((x, 0), {}, "choose"),
                               ((x, 33), {}, "choose"), ((x, 9), dict(n_groups=4, top_k_groups=1), "choose"),
                               ((x, 2), dict(gating="tanh"), "gating"), ((x, 2), dict(n_groups=5), "groups"),
                               ((x, 2), dict(n_groups=4, top_k_groups=5), "groups"), ((x, 2), dict(normalize=3), "normalize"),
                               ((x, 2), dict(score_bias=torch.zeros(31, device=device)), "score_bias"),
                               ((x, 2), dict(score_bias=torch.zeros(32, device=device, dtype=torch.bfloat16)), "score_bias")):
        with pytest.raises(ValueError, match=text):
            route(*args, **kwargs)
    if device == "cuda":
        with pytest.raises(ValueError, match="1024"):
            route(torch.zeros(2, 1025, device=device), 2)
        with pytest.raises(ValueError, match="score_bias"):
            route(x, 2, score_bias=torch.zeros(32))


@pytest.mark.parametrize("device", DEVICES)
def test_a_router_with_its_own_choice_is_asked(device):
    from olmo_core_b200.nn.moe.router import MoELinearRouter, MoERouterGatingFunction

    class Last(MoELinearRouter):
        def get_top_k(self, scores):
            indices = torch.arange(6, 8, device=scores.device).expand(*scores.shape[:-1], 2)
            return scores.gather(-1, indices), indices

    router = Last(d_model=16, num_experts=8, top_k=2, gating_function=MoERouterGatingFunction.sigmoid).to(device)
    _, experts, counts, _ = router(_logits(6, 16, 5).view(2, 3, 16).to(device))
    assert experts.flatten().tolist() == [6, 7] * 6 and counts.flatten().tolist() == [0] * 6 + [6, 6]


@pytest.mark.gpu
def test_what_the_kernels_entry_refuses_is_an_exception():
    from olmo_core_b200.ops import _lib

    with pytest.raises(RuntimeError, match="ocb_moe_route failed with code -1"):
        _lib.native().route.default(torch.zeros(2, 4, device="cuda"), 9, False, None, 1, 1, 0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
def test_router_module_with_groups_and_bias(gating, device):
    from olmo_core_b200.exceptions import OLMoConfigurationError
    from olmo_core_b200.nn.moe.router import MoERouterConfig, MoERouterGatingFunction

    config = MoERouterConfig(top_k=4, n_groups=4, top_k_groups=2, bias_gamma=1e-3, normalize_expert_weights=1.0,
                             gating_function=MoERouterGatingFunction(gating))
    router = config.build(48, 32, lb_loss_weight=0.01, z_loss_weight=1e-3).to(device)
    router.score_bias.copy_(_bias(32, 16))
    x = _logits(2 * 25, 48, 17).view(2, 25, 48).to(device).requires_grad_(True)
    weights, experts, counts, aux = router(x)
    logits = router.get_expert_logits(x.detach()).view(50, 32)
    want = _want(logits, 4, gating, router.score_bias, 4, 2, 1)
    assert torch.equal(experts.cpu().view(50, 4), want[1]) and torch.equal(counts.cpu().int(), want[3])
    torch.testing.assert_close(weights.double().cpu().view(50, 4), want[0], rtol=1e-4, atol=0)
    (weights.square().sum() + aux).backward()
    assert torch.isfinite(x.grad).all() and torch.isfinite(router.weight.grad).all() and router.weight.grad.abs().sum() > 0
    router.post_batch()
    assert not torch.equal(router.score_bias.cpu(), _bias(32, 16))
    for bad in (dict(n_groups=5), dict(n_groups=4, top_k_groups=5), dict(n_groups=8, top_k_groups=1, top_k=5),
                dict(n_groups=4, uniform_expert_assignment=True)):
        with pytest.raises(OLMoConfigurationError):
            MoERouterConfig(**bad).build(48, 32)
