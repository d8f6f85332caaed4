"""64-bit oracles of the expert-block operators, written from their definitions, and the tolerance the tests share.

Every oracle returns ``{name: (value, scale)}``: the value in 64 bits and the sum of the absolute values of the terms it
is made of (gradients: of the terms of the formula), which is what rounding errors of fp32 arithmetic are relative to.

A result computed in fp32 by sums of up to n terms in any order is off by at most n u * scale per sum, u = 2^-24; the
formulas here chain at most four sums (two norms forward, the two means of their backward) with a few products and an
exp, log, square root or division of at most 4 u each in between, so ``(4 n + 64) u * scale`` covers them to first order.
Storing it rounds by at most half a step, ``eps(dtype) / 2 * |value|`` (a subnormal: half the smallest number).
"""
import math

import torch


def tolerance(dtype, value, scale, terms):
    info = torch.finfo(dtype)
    return info.eps / 2 * value.abs() + info.smallest_normal * info.eps / 2 + (4 * terms + 64) * 2.0 ** -24 * scale


def assert_matches(actual, expected, terms, what=""):
    """``actual`` (a result in its dtype) against ``(value, scale)`` within the bound of the module docstring."""
    value, scale = (t.cpu().double() for t in expected)
    assert actual.shape == value.shape, (what, tuple(actual.shape), tuple(value.shape))
    got = actual.detach().cpu().double()
    bound = tolerance(actual.dtype, value, scale, terms)
    off = (got - value).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((off / bound.clamp_min(1e-300))[bad].max()), got[bad][:3], value[bad][:3])


def route(logits, top_k, *, bias=None, mask=None, normalize=True, dweights=None, dbalance=0.0, dz=0.0):
    """Token by token and choice by choice, in 64 bits (the selection key is the 32-bit sum it is defined as)."""
    tokens, experts = logits.shape
    l32, l = logits.detach().cpu().float(), logits.detach().cpu().double()
    key = l32 if bias is None else l32 + bias.detach().cpu().float()
    f64 = dict(dtype=torch.float64)
    weights, indices = torch.zeros(tokens, top_k, **f64), torch.full((tokens, top_k), -1, dtype=torch.int32)
    counts, p, lse = torch.zeros(experts, dtype=torch.int32), torch.zeros(tokens, experts, **f64), torch.zeros(tokens, **f64)
    live = []
    for t in range(tokens):
        if mask is not None and not bool(mask.cpu()[t]):
            continue
        ranked = sorted((e for e in range(experts) if float(key[t, e]) != -math.inf), key=lambda e: (-float(key[t, e]), e))
        chosen = ranked[:top_k]
        if not chosen:
            continue
        live.append(t)
        p[t] = torch.softmax(l[t], 0)
        lse[t] = torch.logsumexp(l[t], 0)
        total = float(p[t, chosen].sum()) if normalize else 1.0
        for j, e in enumerate(chosen):
            indices[t, j] = e
            weights[t, j] = torch.softmax(l[t, chosen], 0)[j] if normalize else p[t, e] / total
            counts[e] += 1
    n, choices = max(1, len(live)), max(1, int(counts.sum()))
    share = counts.double() / choices
    balance, z = experts * float((share * p.sum(0)).sum()) / n, float((lse * lse).sum()) / n
    result = dict(weights=(weights, weights.abs() * (1 + l.nan_to_num(0, 0, 0).abs().amax(1, keepdim=True))), indices=indices,
                  counts=counts, balance=(torch.tensor(balance, **f64), torch.tensor(abs(balance) * 4, **f64)),
                  z=(torch.tensor(z, **f64), torch.tensor(abs(z) * 4 + 1e-30, **f64)))
    if dweights is not None or dbalance or dz:
        grad, size = torch.zeros(tokens, experts, **f64), torch.zeros(tokens, experts, **f64)
        for t in live:
            sel = [e for e in indices[t].tolist() if e >= 0]
            if dweights is not None:
                g = dweights[t, :len(sel)].cpu().double()
                w = weights[t, :len(sel)]
                dot, dot_size = float((w * g).sum()), float((w * g).abs().sum())
                if normalize:
                    grad[t, sel] += w * (g - dot)
                    size[t, sel] += w * (g.abs() + dot_size)
                else:
                    grad[t, sel] += w * g
                    size[t, sel] += (w * g).abs()
                    grad[t] -= p[t] * dot
                    size[t] += p[t] * dot_size
            grad[t] += dbalance * experts / n * p[t] * (share - (p[t] * share).sum())
            size[t] += abs(dbalance) * experts / n * p[t] * (share + (p[t] * share).sum())
            grad[t] += dz * 2 / n * lse[t] * p[t]
            size[t] += abs(dz) * 2 / n * abs(lse[t]) * p[t]
            # p and the weights themselves carry the error of exp(l - max): relative to the spread of the logits
            size[t] *= 2 + float(l[t][l[t].isfinite()].abs().max())
        result["dlogits"] = (grad, size)
    return result


def plan(indices, experts):
    """Offsets and positions by walking the choices expert by expert."""
    flat = indices.reshape(-1).tolist()
    offsets, positions, row = [0], [-1] * len(flat), 0
    for e in range(experts):
        for at, chosen in enumerate(flat):
            if chosen == e:
                positions[at] = row
                row += 1
        offsets.append(row)
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(positions, dtype=torch.int32).view(indices.shape)


def combine(rows, weights, positions, dout=None):
    rows, weights, positions = rows.detach().cpu().double(), weights.detach().cpu().double(), positions.cpu()
    tokens, top_k = positions.shape
    out, size = torch.zeros(tokens, rows.shape[1], dtype=torch.float64), torch.zeros(tokens, rows.shape[1], dtype=torch.float64)
    drows, dweights, dsize = torch.zeros_like(rows), torch.zeros(tokens, top_k, dtype=torch.float64), torch.zeros(tokens, top_k, dtype=torch.float64)
    weights = weights.view(tokens, top_k)
    for t in range(tokens):
        for j in range(top_k):
            at = int(positions[t, j])
            if at < 0:
                continue
            out[t] += weights[t, j] * rows[at]
            size[t] += (weights[t, j] * rows[at]).abs()
            if dout is not None:
                g = dout[t].detach().cpu().double()
                drows[at] = weights[t, j] * g
                dweights[t, j] = (g * rows[at]).sum()
                dsize[t, j] = (g * rows[at]).abs().sum()
    result = dict(out=(out, size))
    if dout is not None:
        result.update(drows=(drows, drows.abs()), dweights=(dweights, dsize))
    return result


def block_norm(x, y, weight=None, gate=None, next_weight=None, next_scale=None, *, residual_scale=1.0, eps=1e-6, next_norm=True,
               dout=None, dh=None):
    """Values and term sizes of both norms and their gradients; ``x`` [batch, tokens, width], vectors [width] or [batch, width]."""
    def wide(v, shift=0.0):
        if v is None:
            return torch.ones(1, 1, 1, dtype=torch.float64)
        v = v.detach().cpu().double() + shift
        return v[None, None] if v.dim() == 1 else v[:, None]

    def back(value, v):
        return value.sum((0, 1)) if v.dim() == 1 else value.sum(1)

    n = x.shape[-1]
    u = x.detach().cpu().double()
    us = u.abs()
    result = {}
    w, g, w2, s2 = wide(weight), wide(gate), wide(next_weight), wide(next_scale, 1.0)
    if y is not None:
        yd = y.detach().cpu().double()
        ry = 1 / torch.sqrt((yd ** 2).mean(-1, keepdim=True) + eps)
        yh = yd * ry
        q = yh * w * g
        u, us = residual_scale * u + q, abs(residual_scale) * us + q.abs()
        result["out"] = (u, us)
    if next_norm:
        ru = 1 / torch.sqrt((u ** 2).mean(-1, keepdim=True) + eps)
        uh, uhs = u * ru, us * ru
        # an error of u that is relative to us changes ru by mean(u us) ru^2 of itself
        uhs = uhs + uh.abs() * (uh.abs() * uhs).mean(-1, keepdim=True)
        result["h"] = (uh * w2 * s2, uhs * (w2 * s2).abs())
    d = dout.detach().cpu().double() if dout is not None else torch.zeros_like(u)
    ds = d.abs()
    if next_norm and dh is not None:
        grad = dh.detach().cpu().double()
        if next_weight is not None:
            result["dnext_weight"] = back(grad * uh * s2, next_weight), back((grad * uhs * s2).abs(), next_weight)
        if next_scale is not None:
            result["dnext_scale"] = back(grad * uh * w2, next_scale), back((grad * uhs * w2).abs(), next_scale)
        t = grad * w2 * s2
        d = d + ru * (t - uh * (t * uh).mean(-1, keepdim=True))
        ds = ds + ru * (1 + uhs.square().mean(-1, keepdim=True)) * (t.abs() + uhs * (t.abs() * uhs).mean(-1, keepdim=True))
    if dout is not None or dh is not None:
        if y is not None:
            if weight is not None:
                result["dweight"] = back(d * yh * g, weight), back((ds * yh * g).abs(), weight)
            if gate is not None:
                result["dgate"] = back(d * yh * w, gate), back((ds * yh * w).abs(), gate)
            t, ts = d * w * g, ds * (w * g).abs()
            result["dy"] = (ry * (t - yh * (t * yh).mean(-1, keepdim=True)),
                            ry * (ts + yh.abs() * (ts * yh.abs()).mean(-1, keepdim=True)))
            d, ds = residual_scale * d, abs(residual_scale) * ds
        result["dx"] = (d, ds)
    return result


def route_batch(logits, top_k, *, bias=None, mask=None, normalize=True, dweights=None, dbalance=0.0, dz=0.0):
    """:func:`route` for many tokens at once: the same definitions and term sizes over whole tensors."""
    tokens, experts = logits.shape
    live = torch.ones(tokens, dtype=torch.bool) if mask is None else mask.cpu()
    l32 = torch.where(live[:, None], logits.detach().cpu().float(), -math.inf)
    key = l32 if bias is None else l32 + bias.detach().cpu().float()
    order = torch.argsort(-key, dim=1, stable=True)[:, :top_k]
    open_ = key.gather(1, order) != -math.inf
    live = live & open_[:, 0]
    l = torch.where(live[:, None], l32, 0.0).double()
    picked = torch.zeros(tokens, experts, dtype=torch.bool).scatter_(1, order, open_) & live[:, None]
    p = torch.softmax(l, 1) * live[:, None]
    lse = torch.logsumexp(l, 1) * live
    if normalize:
        w = torch.softmax(torch.where(picked, l, -math.inf), 1).nan_to_num(0) * picked
    else:
        w = p * picked
    counts = picked.sum(0)
    n, choices = max(1, int(live.sum())), max(1, int(counts.sum()))
    share = counts.double() / choices
    balance, z = experts * (share * p.sum(0)).sum() / n, (lse * lse).sum() / n
    weights, spread = w.gather(1, order) * open_, 1 + l.nan_to_num(0, 0, 0).abs().amax(1, keepdim=True)
    result = dict(weights=(weights, weights * spread), indices=torch.where(open_ & live[:, None], order, -1).to(torch.int32),
                  counts=counts.to(torch.int32), balance=(balance, balance.abs() * 4), z=(z, z.abs() * 4 + 1e-30))
    if dweights is not None or dbalance or dz:
        grad, size = torch.zeros_like(p), torch.zeros_like(p)
        if dweights is not None:
            g = torch.zeros_like(p).scatter_(1, order, dweights.cpu().double() * open_) * live[:, None]
            dot, dot_size = (w * g).sum(1, keepdim=True), (w * g).abs().sum(1, keepdim=True)
            over = w if normalize else p
            grad += w * g - over * dot
            size += (w * g).abs() + over * dot_size
        mean = (p * share).sum(1, keepdim=True)
        grad += dbalance * experts / n * p * (share - mean) + dz * 2 / n * lse[:, None] * p
        size += abs(dbalance) * experts / n * p * (share + mean) + abs(dz) * 2 / n * lse[:, None].abs() * p
        size *= 2 + torch.where(l.isfinite(), l, 0.0).abs().amax(1, keepdim=True)
        result["dlogits"] = (grad, size)
    return result


def combine_batch(rows, weights, positions, dout=None):
    """:func:`combine` for many tokens at once."""
    rows, weights, at = rows.detach().cpu().double(), weights.detach().cpu().double().view(positions.shape), positions.cpu().long()
    there = at >= 0
    factor, taken = weights * there, rows[at.clamp_min(0)] * there[..., None]
    terms = factor[..., None] * taken
    result = dict(out=(terms.sum(1), terms.abs().sum(1)))
    if dout is not None:
        g = dout.detach().cpu().double()[:, None]
        drows = torch.zeros_like(rows)
        drows[at[there]] = (factor[..., None] * g)[there]
        result.update(drows=(drows, drows.abs()), dweights=((g * taken).sum(2), (g * taken).abs().sum(2)))
    return result
