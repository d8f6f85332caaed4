"""Cases, plain forms and 64-bit values of the expert-block operators.

Four kinds of case: ``route`` (top-k router with its balance loss, z loss and per-expert counts), ``dispatch`` (token rows
sorted by expert), ``combine`` (expert rows weighted back into tokens) and ``norm`` (RMS norms after and before a block,
fused with the block's gate and the residual scale).  ``train`` cases run the operator forward and backward, the others
forward only.
"""

import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-6


def listed():
    return [
        # a router asked for one token: nothing but latency
        dict(name="route 1x8", kind="route", tokens=1, experts=8, top_k=2, dtype="bf16", bias=False, closed=0,
             padding=0.0, normalize=True, train=False),
        # a padded batch of odd length, an odd number of experts, two of them closed by -inf logits
        dict(name="route 5003x60 padded", kind="route", tokens=5003, experts=60, top_k=4, dtype="fp16", bias=True,
             closed=2, padding=0.2, normalize=False, train=True),
        # a training step's router with many small experts and the selection bias of loss-free balancing
        dict(name="route 131072x256", kind="route", tokens=131072, experts=256, top_k=8, dtype="fp32", bias=True, closed=0,
             padding=0.0, normalize=True, train=True),
        # sorting a handful of tokens at the width of DiT-XL/2
        dict(name="dispatch 16x1152", kind="dispatch", tokens=16, experts=8, top_k=2, width=1152, dtype="bf16",
             padding=0.0, train=False),
        # odd sizes: rows that are no multiple of 16 bytes, dropped tokens
        dict(name="dispatch 5003x771 dropped", kind="dispatch", tokens=5003, experts=60, top_k=3, width=771, dtype="fp16",
             padding=0.2, train=True),
        # a training step's exchange, four experts a token
        dict(name="dispatch 32768x2048", kind="dispatch", tokens=32768, experts=128, top_k=4, width=2048, dtype="bf16",
             padding=0.0, train=True),
        # joining a few tokens of a ragged batch, in fp32
        dict(name="combine 77x1000", kind="combine", tokens=77, experts=16, top_k=2, width=1000, dtype="fp32", padding=0.1,
             train=False),
        # a DiT-XL/2 microbatch (128 images of 256 tokens), two experts a token
        dict(name="combine 32768x1152", kind="combine", tokens=32768, experts=16, top_k=2, width=1152, dtype="bf16",
             padding=0.0, train=True),
        # one token of a wide model between two blocks
        dict(name="norm 1x4096", kind="norm", batch=1, tokens=1, width=4096, stream="bf16", branch="bf16", weights=True,
             sample=False, post=True, pre=True, residual=1.0, train=False),
        # a DiT-XL/2 microbatch: fp32 stream under autocast, per-sample gate and scale
        dict(name="norm 128x256x1152", kind="norm", batch=128, tokens=256, width=1152, stream="fp32", branch="bf16",
             weights=True, sample=True, post=True, pre=True, residual=1.0, train=True),
        # odd width: no row but the first starts on a 16-byte boundary; the last norm of a model has no next one
        dict(name="norm 7x1025x1001", kind="norm", batch=7, tokens=1025, width=1001, stream="fp16", branch="fp16",
             weights=True, sample=True, post=True, pre=False, residual=0.5, train=True),
        # long sequences of a wide model, weights only, a scaled residual
        dict(name="norm 4x8192x4096", kind="norm", batch=4, tokens=8192, width=4096, stream="bf16", branch="bf16",
             weights=True, sample=False, post=True, pre=True, residual=1.4, train=True),
    ]


def _spread(rng, low, high):
    """A whole number between two, spread over its logarithm; one in three made odd."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.34:
        n |= 1
    return max(low, min(high, n))


def _width(rng, low, high):
    """A width: mostly a multiple of 64, sometimes of 8, sometimes anything."""
    step = rng.choice((64, 64, 64, 8, 1))
    return max(low, min(high, max(1, round(_spread(rng, low, high) / step)) * step))


def draw(rng):
    kind = rng.choice(("route", "dispatch", "combine", "norm"))
    train = rng.random() < 0.7
    if kind == "norm":
        width = _width(rng, 64, 8192)
        tokens = _spread(rng, 1, 8192)
        batch = _spread(rng, 1, max(1, min(256, (1 << 26) // (width * tokens))))
        branch = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        post = rng.random() < 0.85
        return dict(kind="norm", batch=batch, tokens=tokens, width=width, stream=rng.choice((branch, "fp32")),
                    branch=branch, weights=rng.random() < 0.7, sample=rng.random() < 0.5, post=post,
                    pre=not post or rng.random() < 0.8, residual=rng.choice((1.0, 0.5, 1.25)) if post else 1.0, train=train)
    experts = _spread(rng, 4, 256)
    top_k = rng.randint(1, min(8, experts // 2))
    common = dict(kind=kind, experts=experts, top_k=top_k, padding=rng.choice((0.0, 0.0, 0.1, 0.3)), train=train)
    if kind == "route":
        return dict(common, tokens=_spread(rng, 1, min(131072, (1 << 25) // experts)), dtype=rng.choice(("fp32", "bf16", "fp16")),
                    bias=rng.random() < 0.5, closed=rng.choice((0, 0, experts // 4)), normalize=rng.random() < 0.7)
    width = _width(rng, 64, 4096)
    return dict(common, tokens=_spread(rng, 1, max(1, min(32768, (1 << 28) // (width * top_k * 4)))), width=width,
                dtype=rng.choice(("fp32", "bf16", "bf16", "fp16")))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _rand(g, shape):
    return torch.rand(shape, generator=g, device="cuda")


def _choices(g, case):
    """Expert choices as a router leaves them: distinct within a token, some experts liked more than others, -1 dropped."""
    taste = _randn(g, (case["tokens"], case["experts"])) + 0.7 * _randn(g, (case["experts"],))
    indices = taste.topk(case["top_k"], dim=1).indices.to(torch.int32)
    if case["padding"]:
        indices = torch.where(_real(g, case)[:, None], indices, indices.new_tensor(-1))
    return indices


def _real(g, case):
    """Which tokens of a padded batch are real ones; the first is."""
    return (_rand(g, (case["tokens"],)) >= case["padding"]).index_fill_(0, torch.zeros(1, dtype=torch.long, device="cuda"), True)


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["kind"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        logits = 1.5 * _randn(g, (t, e)) + 0.5 * _randn(g, (e,))
        if case["closed"]:
            logits[:, torch.randperm(e, generator=g, device="cuda")[:case["closed"]]] = -math.inf
        state["logits"] = logits.to(_TYPES[case["dtype"]]).requires_grad_(case["train"])
        state["bias"] = 0.3 * _randn(g, (e,)) if case["bias"] else None
        state["mask"] = _real(g, case) if case["padding"] else None
        if case["train"]:
            # the mean over tokens, the small factors of the two losses, and the loss scale of fp16 training
            scale = 1024.0 if case["dtype"] == "fp16" else 1.0
            state["grads"] = (_randn(g, (t, k)) * (scale / t), torch.full((), 0.01 * scale, device="cuda"),
                              torch.full((), 0.001 * scale, device="cuda"))
        return state
    if case["kind"] == "norm":
        b, n, d = case["batch"], case["tokens"], case["width"]
        stream, branch = _TYPES[case["stream"]], _TYPES[case["branch"]]
        leaves = {"x": (2.0 * _randn(g, (b, n, d))).to(stream)}
        if case["post"]:
            leaves["y"] = _randn(g, (b, n, d), branch)
            if case["weights"]:
                leaves["weight"] = 1 + 0.2 * _randn(g, (d,))
            if case["sample"]:
                leaves["gate"] = (0.5 * _randn(g, (b, d))).to(branch)
        if case["pre"]:
            if case["weights"]:
                leaves["next_weight"] = 1 + 0.2 * _randn(g, (d,))
            if case["sample"]:
                leaves["next_scale"] = (0.3 * _randn(g, (b, d))).to(branch)
        if case["train"]:
            for leaf in leaves.values():
                leaf.requires_grad_(True)
            grads = []
            if case["post"]:
                grads.append(_randn(g, (b, n, d), stream))
            if case["pre"]:
                grads.append(_randn(g, (b, n, d), branch))
            state["grads"] = grads
        state["leaves"] = leaves
        return state
    dtype = _TYPES[case["dtype"]]
    t, k, d = case["tokens"], case["top_k"], case["width"]
    state["indices"] = _choices(g, case)
    if case["kind"] == "dispatch":
        state["x"] = _randn(g, (t, d), dtype).requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = _randn(g, (t * k, d), dtype)
        return state
    # the plan of the dispatch before it is at hand
    state["offsets"], state["positions"], used, _ = _sorted(state["indices"], case["experts"])
    rows = _randn(g, (t * k, d), dtype)
    state["rows"] = torch.where(used[:, None], rows, torch.zeros_like(rows)).requires_grad_(case["train"])
    weights = torch.softmax(_randn(g, (t, k)), dim=1)
    state["weights"] = weights.requires_grad_(case["train"])
    if case["train"]:
        state["grad"] = _randn(g, (t, d), dtype)
    return state


def run(state):
    return {"route": _route, "dispatch": _dispatch, "combine": _combine, "norm": _norm}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------------- router
def _route(state):
    case, logits = state["case"], state["logits"]
    if own:
        from viola_b200 import nn
        out = nn.route_tokens(logits, case["top_k"], bias=state["bias"], mask=state["mask"], normalize=case["normalize"])
        weights, indices, counts, balance, z = out
    else:
        weights, indices, counts, balance, z = _route_plain(case, logits, state["bias"], state["mask"])
    result = dict(weights=weights, indices=indices, counts=counts, balance=balance, z=z)
    if case["train"]:
        result["dlogits"], = torch.autograd.grad([weights, balance, z], [logits], list(state["grads"]))
    return result


def _route_plain(case, logits, bias, mask):
    experts, k = case["experts"], case["top_k"]
    live = torch.ones(logits.shape[0], dtype=torch.bool, device=logits.device) if mask is None else mask
    values = torch.where(live[:, None], logits.float(), torch.zeros((), device=logits.device))
    key = values.detach() if bias is None else values.detach() + bias
    indices = key.sort(dim=1, descending=True, stable=True).indices[:, :k]
    top = values.detach().amax(1, keepdim=True)
    e = torch.exp(values - top)
    total = e.sum(1, keepdim=True)
    p = e / total
    lse = (top + torch.log(total))[:, 0]
    chosen = p.gather(1, indices)
    if case["normalize"]:
        chosen = chosen / chosen.sum(1, keepdim=True)
    weights = chosen * live[:, None]
    indices = torch.where(live[:, None], indices, torch.full_like(indices, -1))
    counts = (indices.reshape(-1, 1) == torch.arange(experts, device=logits.device)).sum(0) if indices.numel() * experts < 1 << 24 \
        else torch.bincount(indices.reshape(-1) + 1, minlength=experts + 1)[1:]
    tokens = live.sum().clamp_min(1)
    share = counts.float() / counts.sum().clamp_min(1)
    mean_p = (p * live[:, None]).sum(0) / tokens
    balance = experts * (share * mean_p).sum()
    z = (torch.where(live, lse, torch.zeros_like(lse)) ** 2).sum() / tokens
    return weights, indices.to(torch.int32), counts.to(torch.int32), balance, z


def _route_exact(case, state):
    l = state["logits"].detach().double()
    t, experts = l.shape
    k, mask = case["top_k"], state["mask"]
    live = torch.ones(t, dtype=torch.bool, device=l.device) if mask is None else mask
    key = state["logits"].detach().float()              # the selection key is defined as a 32-bit sum
    key = key + state["bias"] if state["bias"] is not None else key
    order = torch.argsort(-key, dim=1, stable=True)[:, :k]
    picked = torch.zeros(t, experts, dtype=torch.bool, device=l.device).scatter_(1, order, True) & live[:, None]
    p = torch.softmax(l, dim=1) * live[:, None]
    lse = torch.logsumexp(l, dim=1) * live
    n = max(1, int(live.sum()))
    counts = picked.sum(0)
    share = counts.double() / max(1, int(counts.sum()))
    q = p * picked
    if case["normalize"]:
        q = q / q.sum(1, keepdim=True).clamp_min(torch.finfo(torch.float64).tiny)
    result = dict(weights=q.gather(1, order), indices=torch.where(live[:, None], order, -1).to(torch.int32),
                  counts=counts.to(torch.int32), balance=experts * (share * p.sum(0)).sum() / n, z=(lse * lse).sum() / n)
    if case["train"]:
        dw, db, dz = (v.double() for v in state["grads"])
        g = torch.zeros_like(p).scatter_(1, order, dw) * picked
        grad = (q if case["normalize"] else p) * (g - (q * g).sum(1, keepdim=True))
        grad += db * experts / n * p * (share - (p * share).sum(1, keepdim=True))
        grad += dz * 2 / n * lse[:, None] * p
        result["dlogits"] = grad
    return result


# ------------------------------------------------------------------------------------------------ dispatch and combine
def _sorted(indices, experts):
    """Offsets [experts + 1], position of every choice (or -1), which sorted rows are used, and their choices."""
    flat = indices.reshape(-1).long()
    bins = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    counts = torch.zeros(experts + 1, dtype=torch.long, device=flat.device).scatter_add_(0, bins, torch.ones_like(bins))
    offsets = torch.cat([counts.new_zeros(1), counts[:experts].cumsum(0)])
    order = bins.sort(stable=True).indices
    rank = torch.arange(flat.numel(), device=flat.device)
    positions = torch.empty_like(flat).scatter_(0, order, rank)
    positions = torch.where(bins < experts, positions, torch.full_like(positions, -1))
    return offsets.to(torch.int32), positions.to(torch.int32).view(indices.shape), rank < offsets[experts], order


def _dispatch(state):
    case, x = state["case"], state["x"]
    if own:
        from viola_b200 import nn
        plan = nn.plan_experts(state["indices"], case["experts"])
        rows = nn.dispatch_tokens(x, plan)
        result = dict(offsets=plan.offsets, positions=plan.positions, rows=rows)
        if case["train"]:
            result["dx"], = torch.autograd.grad([rows], [x], [state["grad"]])
        return result
    offsets, positions, used, order = _sorted(state["indices"], case["experts"])
    rows = torch.where(used[:, None], x.detach()[order // case["top_k"]], torch.zeros((), dtype=x.dtype, device=x.device))
    result = dict(offsets=offsets, positions=positions, rows=rows)
    if case["train"]:
        back = state["grad"].float()[positions.clamp_min(0).long()]
        result["dx"] = torch.where(positions[..., None] >= 0, back, back.new_zeros(())).sum(1).to(x.dtype)
    return result


def _dispatch_exact(case, state):
    indices, x = state["indices"].cpu(), state["x"].detach().cpu()
    flat = indices.reshape(-1)
    place = [torch.nonzero(flat == e)[:, 0] for e in range(case["experts"])]
    offsets = torch.tensor([0] + [len(v) for v in place]).cumsum(0)
    listing = torch.cat(place)
    positions = torch.full((flat.numel(),), -1, dtype=torch.long)
    positions[listing] = torch.arange(len(listing))
    rows = torch.zeros(flat.numel(), case["width"], dtype=torch.float64)
    rows[: len(listing)] = x.double()[listing // case["top_k"]]
    result = dict(offsets=offsets.to(torch.int32), positions=positions.to(torch.int32).view(indices.shape), rows=rows)
    if case["train"]:
        grad = state["grad"].cpu().double()
        result["dx"] = torch.zeros(case["tokens"], case["width"], dtype=torch.float64).index_add_(
            0, listing // case["top_k"], grad[: len(listing)])
    return result


def _combine(state):
    case, rows, weights = state["case"], state["rows"], state["weights"]
    if own:
        from viola_b200 import nn
        out = nn.combine_tokens(rows, weights, nn.ExpertPlan(state["offsets"], state["positions"]))
        result = dict(out=out)
        if case["train"]:
            result["drows"], result["dweights"] = torch.autograd.grad([out], [rows, weights], [state["grad"]])
        return result
    positions = state["positions"]
    taken = rows.detach().float()[positions.clamp_min(0).long()]
    factor = torch.where(positions >= 0, weights.detach(), torch.zeros_like(weights))[..., None]
    result = dict(out=(taken * factor).sum(1).to(rows.dtype))
    if case["train"]:
        grad = state["grad"].float()[:, None]
        result["dweights"] = torch.where(positions >= 0, (taken * grad).sum(2), torch.zeros_like(weights))
        # dropped choices write to a row behind the last, which is cut off
        spread = torch.zeros(rows.shape[0] + 1, rows.shape[1], dtype=rows.dtype, device=rows.device)
        at = torch.where(positions >= 0, positions, rows.shape[0]).long().reshape(-1)
        spread[at] = (factor * grad).to(rows.dtype).reshape(-1, rows.shape[1])
        result["drows"] = spread[:-1]
    return result


def _combine_exact(case, state):
    rows, weights, positions = (state[n].detach().double() for n in ("rows", "weights", "positions"))
    positions, k = positions.long(), case["top_k"]
    valid = (positions >= 0).double()
    out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device=rows.device)
    grad = state["grad"].double() if case["train"] else None
    drows, dweights = torch.zeros_like(rows), torch.zeros_like(weights)
    for j in range(k):
        at = positions[:, j].clamp_min(0)
        out += (weights[:, j] * valid[:, j])[:, None] * rows[at]
        if case["train"]:
            dweights[:, j] = torch.linalg.vecdot(grad, rows[at]) * valid[:, j]
            drows.index_add_(0, at, (weights[:, j] * valid[:, j])[:, None] * grad)
    return dict(out=out, drows=drows, dweights=dweights) if case["train"] else dict(out=out)


# ------------------------------------------------------------------------------------------------------------ norms
def _norm(state):
    case, leaves = state["case"], state["leaves"]
    if own:
        from viola_b200 import nn
        if case["post"]:
            outs = nn.rms_norm_residual(leaves["x"], leaves["y"], leaves.get("weight"), leaves.get("gate"),
                                        residual_scale=case["residual"], eps=EPS, next_norm=case["pre"],
                                        next_weight=leaves.get("next_weight"), next_scale=leaves.get("next_scale"))
            outs = list(outs) if case["pre"] else [outs]
        else:
            outs = [nn.rms_norm_modulate(leaves["x"], leaves.get("next_weight"), leaves.get("next_scale"), eps=EPS,
                                         dtype=_TYPES[case["branch"]])]
    else:
        outs = _norm_plain(case, leaves)
    names = (["out"] if case["post"] else []) + (["h"] if case["pre"] else [])
    result = dict(zip(names, outs))
    if case["train"]:
        grads = torch.autograd.grad(outs, list(leaves.values()), state["grads"])
        result.update(zip(("d" + n for n in leaves), grads))
    return result


def _unit(v):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)


def _norm_plain(case, leaves):
    x, outs = leaves["x"].float(), []
    if case["post"]:
        y = _unit(leaves["y"].float())
        if "weight" in leaves:
            y = y * leaves["weight"]
        if "gate" in leaves:
            y = y * leaves["gate"].float()[:, None]
        x = case["residual"] * x + y
        outs.append(x.to(leaves["x"].dtype))
    if case["pre"]:
        h = _unit(x)
        if "next_weight" in leaves:
            h = h * leaves["next_weight"]
        if "next_scale" in leaves:
            h = h * (1 + leaves["next_scale"].float())[:, None]
        outs.append(h.to(_TYPES[case["branch"]]))
    return outs


def _norm_exact(case, state):
    """Sample by sample, so that a few rows' worth of 64-bit values are held at a time."""
    v = {n: t.detach().double() for n, t in state["leaves"].items() if n not in ("x", "y")}
    x, y = state["leaves"]["x"].detach(), state["leaves"].get("y")
    b, n, d = x.shape
    ones = torch.ones(d, dtype=torch.float64, device=x.device)
    names = (["out"] if case["post"] else []) + (["h"] if case["pre"] else [])
    grads = dict(zip(names, state["grads"])) if case["train"] else {}
    result = {name: torch.empty(b, n, d, dtype=torch.float64, device=x.device) for name in names}
    if case["train"]:
        for name, leaf in state["leaves"].items():
            result["d" + name] = torch.zeros(leaf.shape, dtype=torch.float64, device=x.device)
    for i in range(b):
        w, g = v.get("weight", ones), (v["gate"][i] if "gate" in v else ones)
        w2, s2 = v.get("next_weight", ones), (1 + v["next_scale"][i] if "next_scale" in v else ones)
        u, dz, alpha = x[i].double(), 0.0, case["residual"]
        if case["post"]:
            yi = y[i].detach().double()
            ry = ((yi ** 2).sum(1, keepdim=True) / d + EPS) ** -0.5
            yh = yi * ry
            u = alpha * u + yh * (w * g)
            result["out"][i] = u
            dz = grads["out"][i].double() if case["train"] else 0.0
        if case["pre"]:
            ru = ((u ** 2).sum(1, keepdim=True) / d + EPS) ** -0.5
            uh = u * ru
            result["h"][i] = uh * (w2 * s2)
            if case["train"]:
                dh = grads["h"][i].double()
                column = (dh * uh).sum(0)
                if "next_weight" in v:
                    result["dnext_weight"] += column * s2
                if "next_scale" in v:
                    result["dnext_scale"][i] = column * w2
                t = dh * (w2 * s2)
                dz = dz + ru * (t - uh * ((t * uh).sum(1, keepdim=True) / d))
        if case["train"]:
            result["dx"][i] = (alpha if case["post"] else 1.0) * dz
            if case["post"]:
                column = (dz * yh).sum(0)
                if "weight" in v:
                    result["dweight"] += column * g
                if "gate" in v:
                    result["dgate"][i] = column * w
                t = dz * (w * g)
                result["dy"][i] = ry * (t - yh * ((t * yh).sum(1, keepdim=True) / d))
    return result


# -------------------------------------------------------------------------------------------------------- measures
def work(case):
    """Each input read once and each output written once."""
    if case["kind"] == "route":
        t, e, k, s = case["tokens"], case["experts"], case["top_k"], _BYTES[case["dtype"]]
        data = t * e * s + t * k * 8 + e * 4 + (t if case["padding"] else 0)
        if case["train"]:
            data += 2 * t * e * s + t * k * 8
        return {"bytes": data, "flops": t * e * (14 if case["train"] else 5)}
    if case["kind"] == "norm":
        elements = case["batch"] * case["tokens"] * case["width"]
        stream, branch = _BYTES[case["stream"]], _BYTES[case["branch"]]
        forward = (2 * stream + branch if case["post"] else stream) + (branch if case["pre"] else 0)
        # dx and what it comes from; y and dy; the stream again where both norms need it; the gradient of h
        backward = 2 * stream + (2 * branch if case["post"] else 0) + (branch if case["pre"] else 0)
        backward += stream if case["post"] and case["pre"] else 0
        return {"bytes": elements * (forward + (backward if case["train"] else 0)), "flops": elements * (30 if case["train"] else 8)}
    t, k, d, s = case["tokens"], case["top_k"], case["width"], _BYTES[case["dtype"]]
    one = t * d * s
    if case["kind"] == "dispatch":
        return {"bytes": one * (1 + k) * (2 if case["train"] else 1) + 8 * t * k, "flops": t * k * d if case["train"] else 0}
    return {"bytes": one * (1 + k) + 8 * t * k + (one * (1 + 2 * k) + 4 * t * k if case["train"] else 0),
            "flops": t * k * d * (5 if case["train"] else 2)}


def exact(case, seed):
    state = prepare(case, seed)
    return {"route": _route_exact, "dispatch": _dispatch_exact, "combine": _combine_exact, "norm": _norm_exact}[case["kind"]](case, state)
