"""
Measured cases of two operator families of the mixture-of-experts and 8-bit training / serving paths.

* Routing (``olmo_core_b200.ops.moe.route``): the scores of a router (softmax or sigmoid), an optional selection bias per
  expert, optional selection of expert groups before experts, the top-k experts, renormalised weights, tokens per expert,
  and the gradient of the logits.
* Products of e4m3 operands with one power-of-two scale per block of 128 (``olmo_core_b200.ops.fp8_block``): the serving
  product over a weight that is kept in 8 bits, the training step of a linear layer (output, input gradient, weight
  gradient), and the same two for the experts of a mixture (rows sorted by expert, group boundaries on the device).

Blocks: an operand that is scaled "by rows" has one scale per 128 elements of each row, "by columns" one per 128 elements
of each column, a weight one per 128 x 128 tile. A scale is the smallest power of two that brings its block's largest
magnitude to 448 (the largest e4m3 value) or below, and 1 for a block of zeros; elements are rounded to the nearest e4m3
value, ties to even. Dividing by a power of two is exact, so what a block is quantised to does not depend on the arithmetic.
"""

import math

import torch

own = False

BLOCK = 128


# ---------------------------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one decoding step of one conversation: the routing of a single token, where only latency counts
        dict(name="route 1 token of 64", op="route", tokens=1, experts=64, top_k=8, gating="softmax", biased=False, groups=1,
             top_groups=1, normalize=0, train=False),
        # a training micro-batch through the router of a 64-expert model: softmax scores, top 8, auxiliary-loss gradient
        dict(name="route step softmax 64", op="route", tokens=16384, experts=64, top_k=8, gating="softmax", biased=False,
             groups=1, top_groups=1, normalize=0, train=True),
        # a large mixture balanced by a selection bias, groups of experts selected first, odd token count
        dict(name="route step grouped 256", op="route", tokens=8191, experts=256, top_k=8, gating="sigmoid", biased=True,
             groups=8, top_groups=4, normalize=1, train=True),
        # decoding: one token against an MLP projection of a 7B model kept in 8 bits (bound by the weight's bytes)
        dict(name="product 1 token", op="product", tokens=1, features=4096, outputs=11008),
        # a small batch of prompts with odd sizes: nothing is a multiple of a tile or of a block
        dict(name="product 77 odd", op="product", tokens=77, features=2050, outputs=1001),
        # a long prompt through the same projection (bound by the tensor cores)
        dict(name="product 8192", op="product", tokens=8192, features=4096, outputs=11008),
        # training step of a small model's projection on a ragged micro-batch
        dict(name="linear step 1000", op="linear", tokens=1000, features=768, outputs=2048),
        # training step of the 7B projection: output, input gradient and weight gradient
        dict(name="linear step 8192", op="linear", tokens=8192, features=4096, outputs=11008),
        # decoding 16 sequences through the experts' up-projections: two rows an expert, bound by the weights' bytes
        dict(name="experts 128 rows", op="experts", rows=128, experts=64, features=2048, outputs=1024, skew=0.3),
        # a long prompt through the experts
        dict(name="experts 65536 rows", op="experts", rows=65536, experts=64, features=2048, outputs=1024, skew=0.3),
        # training micro-batch through the experts' down-projection, uneven load with experts that get nothing
        dict(name="experts step 32768", op="experts_step", rows=32768, experts=64, features=1024, outputs=2048, skew=0.6),
    ]


def _between(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route", "product", "linear", "experts", "experts_step"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        experts = groups * _between(rng, 4, 384 // groups)
        top_groups = rng.randint(max(1, groups // 4), groups)
        return dict(op=op, tokens=_between(rng, 1, 16384), experts=experts,
                    top_k=rng.randint(1, min(12, top_groups * (experts // groups))), gating=rng.choice(["softmax", "sigmoid"]),
                    biased=rng.random() < 0.5, groups=groups, top_groups=top_groups, normalize=rng.choice([0, 1, 2]),
                    train=rng.random() < 0.6)
    if op in ("product", "linear"):
        return dict(op=op, tokens=_between(rng, 1, 8192), features=_between(rng, 100, 4096), outputs=_between(rng, 100, 11008))
    # expert matrices keep widths that are multiples of 16, as every configuration of them has
    return dict(op=op, rows=_between(rng, 8, 32768), experts=_between(rng, 4, 128), features=16 * _between(rng, 16, 128),
                outputs=16 * _between(rng, 16, 128), skew=rng.choice([0.0, 0.3, 0.6]))


# --------------------------------------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 31))


def _normal(shape, g, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _activations(shape, g):
    """Token activations: a spread of magnitudes over the tokens and a few channels much larger than the others."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    x *= torch.exp(0.5 * torch.randn((shape[0], 1), generator=g, device="cuda"))
    x *= 1.0 + 20.0 * (torch.rand((1, shape[1]), generator=g, device="cuda") < 0.01)
    return x.to(torch.bfloat16)


def _offsets(rows, experts, skew, seed):
    """Row boundaries of the experts ``[experts + 1]`` (int32) and the largest group; ``skew``: spread of the log-load."""
    g = torch.Generator().manual_seed(int(seed) % (1 << 31))
    load = torch.softmax(2.0 * skew * torch.randn(experts, generator=g), 0)
    sizes = torch.bincount(torch.multinomial(load, rows, replacement=True, generator=g), minlength=experts)
    offsets = torch.zeros(experts + 1, dtype=torch.int32)
    offsets[1:] = sizes.cumsum(0)
    return offsets.cuda(), int(sizes.max())


def _kept_weight(shape, g):
    """A weight as a serving program keeps it: e4m3 codes (rows start on 16-byte boundaries) and a scale per tile."""
    codes, scales = _tiles(_normal(shape, g, shape[-1] ** -0.5))
    *lead, n, k = shape
    held = torch.zeros(*lead, n, (k + 15) // 16 * 16, dtype=torch.uint8, device="cuda")[..., :k]
    held.copy_(codes.to(torch.float8_e4m3fn).view(torch.uint8))
    return held.view(torch.float8_e4m3fn), scales


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    s = dict(case)
    if op == "route":
        n, e, k = case["tokens"], case["experts"], case["top_k"]
        s["logits"] = _normal((n, e), g, 1.5, torch.float32)
        # the bias moves in equal steps, one per training step and expert
        s["bias"] = torch.randint(-100, 101, (e,), generator=g, device="cuda").float() * 1e-3 if case["biased"] else None
        if case["train"]:
            s["logits"].requires_grad_(True)
            s["d_weights"] = _normal((n, k), g, 1.0, torch.float32)
            s["d_scores"] = _normal((n, e), g, 0.01, torch.float32)
    elif op == "product":
        s["x"] = _activations((case["tokens"], case["features"]), g)
        s["codes"], s["scales"] = _kept_weight((case["outputs"], case["features"]), g)
    elif op == "linear":
        s["x"] = _activations((case["tokens"], case["features"]), g).requires_grad_(True)
        s["weight"] = _normal((case["outputs"], case["features"]), g, case["features"] ** -0.5).requires_grad_(True)
        s["dy"] = _normal((case["tokens"], case["outputs"]), g, 1e-3)
    else:
        e, k, n = case["experts"], case["features"], case["outputs"]
        s["x"] = _activations((case["rows"], k), g)
        s["offsets"], s["most"] = _offsets(case["rows"], e, case["skew"], seed)
        if op == "experts":
            s["codes"], s["scales"] = _kept_weight((e, n, k), g)
        else:
            s["x"].requires_grad_(True)
            s["weight"] = _normal((e * n, k), g, k ** -0.5).requires_grad_(True)
            s["dy"] = _normal((case["rows"], n), g, 1e-3)
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms


def _scale_of(amax):
    """Smallest power of two with ``amax / scale <= 448 = 0.875 * 2^9``; 1 where the block is all zeros."""
    mantissa, exponent = torch.frexp(amax)
    exponent = exponent - 9 + (mantissa > 0.875).int()
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), exponent), torch.ones_like(amax))


def _codes(blocks, scale):
    return (blocks / scale).to(torch.float8_e4m3fn).float()


def _padded(x, rows, cols):
    """``x [..., R, C]`` in fp32 with zeros up to whole blocks of ``rows x cols``."""
    r, c = x.shape[-2:]
    return torch.nn.functional.pad(x.float(), (0, -c % cols, 0, -r % rows))


def _by_rows(x):
    """Values of ``x [R, C]`` after quantisation with a scale per 128 elements of each row."""
    b = _padded(x, 1, BLOCK).view(x.shape[0], -1, BLOCK)
    s = _scale_of(b.abs().amax(-1, keepdim=True))
    return (_codes(b, s) * s).view(x.shape[0], -1)[:, : x.shape[1]]


def _by_columns(x):
    """Values of ``x [R, C]`` after quantisation with a scale per 128 elements of each column."""
    b = _padded(x, BLOCK, 1).view(-1, BLOCK, x.shape[1])
    s = _scale_of(b.abs().amax(1, keepdim=True))
    return (_codes(b, s) * s).view(-1, x.shape[1])[: x.shape[0]]


def _tiles(w):
    """Codes of ``w [..., N, K]`` as fp32 values and the scale of each 128 x 128 tile ``[..., ceil(N/128), ceil(K/128)]``."""
    *lead, n, k = w.shape
    p = _padded(w, BLOCK, BLOCK)
    b = p.view(*lead, p.shape[-2] // BLOCK, BLOCK, p.shape[-1] // BLOCK, BLOCK)
    s = _scale_of(b.abs().amax((-3, -1), keepdim=True))
    return _codes(b, s).view(p.shape)[..., :n, :k], s.squeeze(-1).squeeze(-2)


def _spread(scales, n, k):
    """The scale of every element of a weight of ``n x k``."""
    return scales.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _by_tiles(w):
    codes, scales = _tiles(w)
    return codes * _spread(scales, *w.shape[-2:])


def _slots(s):
    """Where row ``r`` of the sorted rows sits in an ``[experts, most]`` layout: ``(expert, slot)``."""
    rows = torch.arange(s["rows"], device="cuda")
    expert = torch.searchsorted(s["offsets"][1:].long(), rows, right=True)
    return expert, rows - s["offsets"].long()[expert]


def _spread_rows(x, s, at):
    out = x.new_zeros(s["experts"], s["most"], x.shape[-1])
    out[at] = x
    return out


def _plain_route(s):
    logits, k = s["logits"].detach(), s["top_k"]
    n, e = logits.shape
    # what is selected is decided in 64 bits: scores of two experts can be closer than 32 bits tell apart
    fine = logits.double()
    if s["gating"] == "softmax":
        ex = torch.exp(logits - logits.amax(-1, keepdim=True))
        scores = ex / ex.sum(-1, keepdim=True)
        ex = torch.exp(fine - fine.amax(-1, keepdim=True))
        rank = ex / ex.sum(-1, keepdim=True)
    else:
        scores = 1.0 / (1.0 + torch.exp(-logits)) + 1e-7
        rank = 1.0 / (1.0 + torch.exp(-fine)) + 1e-7
    if s["bias"] is not None:
        rank = rank + s["bias"].double()
    if s["groups"] > 1:
        # a group counts as much as its two best experts together
        by_group = rank.view(n, s["groups"], -1)
        best = by_group.sort(dim=-1, descending=True)[0][..., :2].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True)[1][:, : s["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        rank = torch.where(open_[..., None], by_group, torch.full_like(by_group, -math.inf)).view(n, e)
    chosen = rank.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    picked = scores.gather(1, chosen)
    weights, norm = picked, None
    if s["normalize"]:
        norm = picked.sum(-1, keepdim=True) if s["normalize"] == 1 else picked.square().sum(-1, keepdim=True).sqrt()
        weights = picked / norm
    counts = torch.bincount(chosen.reshape(-1), minlength=e).to(torch.int32)
    if not s["train"]:
        return weights, chosen, scores, counts
    d_picked = s["d_weights"]
    if norm is not None:
        along = (d_picked * weights).sum(-1, keepdim=True)
        d_picked = (d_picked - along * (weights if s["normalize"] == 2 else 1.0)) / norm
    d = s["d_scores"].scatter_add(1, chosen, d_picked)
    if s["gating"] == "softmax":
        d_logits = scores * (d - (d * scores).sum(-1, keepdim=True))
    else:
        p = scores - 1e-7
        d_logits = d * p * (1.0 - p)
    return weights, chosen, scores, counts, d_logits


def _plain_product(s):
    w = s["codes"].float() * _spread(s["scales"], s["outputs"], s["features"])
    return (_by_rows(s["x"]) @ w.t()).to(torch.bfloat16)


def _plain_linear(s):
    x, w, dy = s["x"].detach(), s["weight"].detach(), s["dy"]
    wq = _by_tiles(w)
    y = _by_rows(x) @ wq.t()
    dx = _by_rows(dy) @ wq
    dw = _by_columns(dy).t() @ _by_columns(x)
    return y.to(torch.bfloat16), dx.to(torch.bfloat16), dw.to(torch.bfloat16)


def _plain_experts(s):
    w = s["codes"].float() * _spread(s["scales"], s["outputs"], s["features"])
    at = _slots(s)
    return torch.bmm(_spread_rows(_by_rows(s["x"]), s, at), w.transpose(1, 2))[at].to(torch.bfloat16)


def _plain_experts_step(s):
    # the weight gradient of the experts is taken from the unquantised rows
    x, dy, e = s["x"].detach(), s["dy"], s["experts"]
    w = _by_tiles(s["weight"].detach().view(e, s["outputs"], s["features"]))
    at = _slots(s)
    y = torch.bmm(_spread_rows(_by_rows(x), s, at), w.transpose(1, 2))[at]
    dx = torch.bmm(_spread_rows(_by_rows(dy), s, at), w)[at]
    dw = torch.bmm(_spread_rows(dy.float(), s, at).transpose(1, 2), _spread_rows(x.float(), s, at))
    return y.to(torch.bfloat16), dx.to(torch.bfloat16), dw.view(-1, s["features"]).to(torch.bfloat16)


_PLAIN = {"route": _plain_route, "product": _plain_product, "linear": _plain_linear, "experts": _plain_experts,
          "experts_step": _plain_experts_step}


# -------------------------------------------------------------------------------------------------- the framework's calls


def _own_route(s):
    from olmo_core_b200.ops.moe import route

    weights, chosen, scores, counts = route(s["logits"], s["top_k"], gating=s["gating"], score_bias=s["bias"],
                                            n_groups=s["groups"], top_k_groups=s["top_groups"],
                                            normalize=s["normalize"] or None)
    if not s["train"]:
        return weights, chosen, scores, counts
    (d_logits,) = torch.autograd.grad((weights, scores), s["logits"], (s["d_weights"], s["d_scores"]))
    return weights.detach(), chosen, scores.detach(), counts, d_logits


def _own_product(s):
    from olmo_core_b200.ops.fp8_block import fp8_block_matmul

    return fp8_block_matmul(s["x"], s["codes"], s["scales"])


def _own_linear(s):
    from olmo_core_b200.ops.fp8_block import fp8_block_linear

    y = fp8_block_linear(s["x"], s["weight"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
    return y.detach(), dx, dw


def _own_experts(s):
    from olmo_core_b200.ops.fp8_block import fp8_block_grouped_matmul

    return fp8_block_grouped_matmul(s["x"], s["codes"], s["scales"], s["offsets"])


def _own_experts_step(s):
    from olmo_core_b200.ops.fp8_block import fp8_block_grouped_linear

    y = fp8_block_grouped_linear(s["x"], s["weight"], s["offsets"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
    return y.detach(), dx, dw


_OWN = {"route": _own_route, "product": _own_product, "linear": _own_linear, "experts": _own_experts,
        "experts_step": _own_experts_step}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------------ work


def work(case):
    op = case["op"]
    if op == "route":
        n, e, k = case["tokens"], case["experts"], case["top_k"]
        # logits in, scores, weights (4 bytes), expert ids (8 bytes) and counts out; the gradient reads the logits' scores
        # again together with d_scores and d_weights and writes d_logits
        size = n * (8 * e + 12 * k) + 4 * e
        if case["train"]:
            size += n * (12 * e + 12 * k)
        return {"bytes": size, "flops": n * (8 * e + 2 * k * e) * (2 if case["train"] else 1)}
    k, n = case["features"], case["outputs"]
    tiles = -(-n // BLOCK) * -(-k // BLOCK)
    if op == "product":
        m = case["tokens"]
        return {"bytes": 2 * m * k + n * k + 4 * tiles + 2 * m * n, "flops": 2 * m * n * k}
    if op == "linear":
        m = case["tokens"]
        return {"bytes": 2 * (2 * m * k + 2 * m * n + 2 * n * k), "flops": 6 * m * n * k}
    m, e = case["rows"], case["experts"]
    used = min(m, e)  # an expert without rows is not read
    if op == "experts":
        return {"bytes": 2 * m * k + used * (n * k + 4 * tiles) + 2 * m * n, "flops": 2 * m * n * k}
    return {"bytes": 2 * (2 * m * k + 2 * m * n + used * n * k + e * n * k), "flops": 6 * m * n * k}


# ----------------------------------------------------------------------------------------------------------------- exact


def _e4m3(v):
    """Nearest e4m3 value (ties to even) of every element, in 64 bits: steps of 2^(exponent - 3), exponents from -6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0) - 3.0)
    return torch.round(v / step) * step


def _exact_blocks(x, rows, cols):
    """``x`` quantised over blocks of ``rows x cols`` and multiplied out again, in 64 bits."""
    r, c = x.shape
    out = torch.zeros(-(-r // rows) * rows, -(-c // cols) * cols, dtype=torch.float64, device=x.device)
    out[:r, :c] = x.detach().double()
    b = out.view(out.shape[0] // rows, rows, out.shape[1] // cols, cols)
    top = b.abs().amax(dim=(1, 3), keepdim=True)
    scale = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top / 448.0))), torch.ones_like(top))
    return (_e4m3(b / scale) * scale).view(out.shape)[:r, :c]


def _exact_kept(codes, scales):
    n, k = codes.shape
    at_n, at_k = torch.arange(n, device="cuda") // BLOCK, torch.arange(k, device="cuda") // BLOCK
    return codes.double() * scales.double()[at_n][:, at_k]


def _exact_route(s):
    x = s["logits"].detach().double()
    n, e = x.shape
    if s["gating"] == "softmax":
        scores = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
    else:
        scores = torch.special.expit(x) + 1e-7
    key = scores if s["bias"] is None else scores + s["bias"].double()
    if s["groups"] > 1:
        size = e // s["groups"]
        first = key.view(n, s["groups"], size)
        value = first.max(-1)[0]
        if size > 1:
            value = value + first.kthvalue(size - 1, dim=-1)[0]
        # a group stays when fewer than top_groups others are ahead of it (an equal one is ahead when it comes first)
        ahead = (value[:, None, :] > value[:, :, None]).double()
        index = torch.arange(s["groups"], device="cuda")
        ahead += ((value[:, None, :] == value[:, :, None]) & (index[None, None, :] < index[None, :, None])).double()
        stays = (ahead.sum(-1) < s["top_groups"]).repeat_interleave(size, dim=1)
        key = key.masked_fill(~stays, -math.inf)
    chosen = torch.argsort(-key, dim=1, stable=True)[:, : s["top_k"]]
    picked = scores.gather(1, chosen)
    norm = torch.ones(n, 1, dtype=torch.float64, device="cuda")
    if s["normalize"]:
        norm = picked.pow(s["normalize"]).sum(1, keepdim=True).pow(1.0 / s["normalize"])
    weights = picked / norm
    hot = torch.zeros(n, e, dtype=torch.float64, device="cuda").scatter_(1, chosen, 1.0)
    out = [weights, None, scores, None]
    if s["train"]:
        # by the chain rule, over the full width: w_j = s_j hot_j / norm(s), then s(x)
        g = torch.zeros(n, e, dtype=torch.float64, device="cuda").scatter_(1, chosen, s["d_weights"].double())
        d = s["d_scores"].double()
        if s["normalize"]:
            w = scores * hot / norm
            d_norm = -(g * w).sum(1, keepdim=True) / norm  # d L / d norm
            d = d + g / norm + d_norm * (hot if s["normalize"] == 1 else w)
        else:
            d = d + g
        if s["gating"] == "softmax":
            out.append(scores * d - scores * (scores * d).sum(1, keepdim=True))
        else:
            out.append(d * torch.special.expit(x) * torch.special.expit(-x))
    return tuple(out)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "route":
        return _exact_route(s)
    if op == "product":
        return _exact_blocks(s["x"], 1, BLOCK) @ _exact_kept(s["codes"], s["scales"]).t()
    if op == "linear":
        x, w, dy = s["x"].detach(), _exact_blocks(s["weight"], BLOCK, BLOCK), s["dy"]
        return (_exact_blocks(x, 1, BLOCK) @ w.t(), _exact_blocks(dy, 1, BLOCK) @ w,
                _exact_blocks(dy, BLOCK, 1).t() @ _exact_blocks(x, BLOCK, 1))
    bounds, n, k = s["offsets"].tolist(), s["outputs"], s["features"]
    x = s["x"].detach()
    y = torch.zeros(s["rows"], n, dtype=torch.float64, device="cuda")
    dx = torch.zeros(s["rows"], k, dtype=torch.float64, device="cuda")
    dw = torch.zeros(s["experts"] * n, k, dtype=torch.float64, device="cuda")
    for i, (a, b) in enumerate(zip(bounds[:-1], bounds[1:])):
        if b == a:
            continue
        if op == "experts":
            y[a:b] = _exact_blocks(x[a:b], 1, BLOCK) @ _exact_kept(s["codes"][i], s["scales"][i]).t()
            continue
        w = _exact_blocks(s["weight"][i * n:(i + 1) * n], BLOCK, BLOCK)
        y[a:b] = _exact_blocks(x[a:b], 1, BLOCK) @ w.t()
        dx[a:b] = _exact_blocks(s["dy"][a:b], 1, BLOCK) @ w
        dw[i * n:(i + 1) * n] = s["dy"][a:b].double().t() @ x[a:b].double()
    return y if op == "experts" else (y, dx, dw)
