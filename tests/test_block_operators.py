"""Routing around the expert linear and the RMS norms around a block: values, gradients, edge cases and refusals.

Every case runs on the CPU path and, marked ``gpu``, on the kernels, against the 64-bit oracles of ``block_oracles.py``
within the bounds derived there; whole numbers have to be equal.
"""
import math

import pytest
import torch

import block_oracles as oracle
from viola_b200 import nn, ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(params=DEVICES)
def device(request):
    return request.param


def randn(seed, *shape, dtype=FP32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ------------------------------------------------------------------------------------------------------------ router
ROUTES = [  # tokens, experts, top_k, dtype, bias, padding, normalize, levels (0: continuous logits, else that many values)
    (1, 1, 1, FP32, False, 0, True, 0),
    (1, 8, 2, BF16, False, 0, True, 0),
    (300, 3, 2, FP32, True, 0.2, False, 0),
    (300, 4, 4, FP16, False, 0, True, 3),
    (150, 5, 3, BF16, True, 0, True, 2),
    (133, 8, 2, FP32, True, 0.3, False, 4),
    (70, 16, 5, BF16, False, 0.5, True, 0),
    (40, 17, 4, FP16, True, 0, False, 3),
    (33, 32, 32, FP32, False, 0, True, 0),
    (65, 60, 4, FP16, True, 0.2, False, 0),
    (37, 64, 6, BF16, True, 0, True, 5),
    (34, 100, 8, FP32, True, 0.1, True, 0),
    (35, 128, 1, BF16, False, 0, False, 0),
    (36, 256, 8, FP32, True, 0.2, True, 0),
    (5, 300, 7, FP16, False, 0, True, 4),
    (34, 512, 10, BF16, False, 0, True, 0),
    (3, 1000, 32, FP32, True, 0, False, 0),
    (33, 1024, 3, FP16, True, 0, True, 0),
]


def route_inputs(case, seed=0):
    tokens, experts, top_k, dtype, bias, padding, normalize, levels = case
    logits = 2.0 * randn(seed, tokens, experts)
    if levels:
        logits = (logits.clamp(-2, 2) * levels / 4).round()
    mask = None
    if padding:
        mask = torch.rand(tokens, generator=torch.Generator().manual_seed(seed + 1)) >= padding
        logits[~mask] = torch.tensor([math.nan, math.inf, -math.inf])[torch.arange(int((~mask).sum())) % 3][:, None]
    offset = (0.5 * randn(seed + 2, experts)).round(decimals=1) if bias else None
    grads = randn(seed + 3, tokens, top_k), 0.7, 0.3
    return logits.to(dtype), offset, mask, grads


@pytest.mark.parametrize("case", ROUTES, ids=str)
def test_route_values_and_gradients(case, device):
    tokens, experts, top_k, dtype, _, _, normalize, _ = case
    logits, bias, mask, (dw, db, dz) = route_inputs(case)
    expected = oracle.route(logits, top_k, bias=bias, mask=mask, normalize=normalize, dweights=dw, dbalance=db, dz=dz)
    leaf = logits.to(device).requires_grad_(True)
    out = nn.route_tokens(leaf, top_k, bias=None if bias is None else bias.to(device),
                          mask=None if mask is None else mask.to(device), normalize=normalize)
    assert torch.equal(out.indices.cpu(), expected["indices"]) and torch.equal(out.counts.cpu(), expected["counts"])
    terms = experts + tokens
    oracle.assert_matches(out.weights, expected["weights"], terms, "weights")
    oracle.assert_matches(out.balance_loss, expected["balance"], terms, "balance")
    oracle.assert_matches(out.z_loss, expected["z"], terms, "z")
    (out.weights * dw.to(device)).sum().add(db * out.balance_loss).add(dz * out.z_loss).backward()
    oracle.assert_matches(leaf.grad, expected["dlogits"], terms, "dlogits")
    # without a graph the same numbers come back
    again = nn.route_tokens(leaf.detach(), top_k, bias=None if bias is None else bias.to(device),
                            mask=None if mask is None else mask.to(device), normalize=normalize)
    for a, b in zip(out, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["weights", "balance", "z"])
def test_route_gradient_of_one_output(which, device):
    case = (70, 24, 3, FP32, True, 0.2, False, 0)
    logits, bias, mask, (dw, db, dz) = route_inputs(case, 5)
    only = dict(dweights=dw if which == "weights" else None, dbalance=db * (which == "balance"), dz=dz * (which == "z"))
    expected = oracle.route(logits, 3, bias=bias, mask=mask, normalize=False, **only)
    leaf = logits.to(device).requires_grad_(True)
    out = nn.route_tokens(leaf, 3, bias=bias.to(device), mask=mask.to(device), normalize=False)
    {"weights": (out.weights * dw.to(device)).sum(), "balance": db * out.balance_loss, "z": dz * out.z_loss}[which].backward()
    oracle.assert_matches(leaf.grad, expected["dlogits"], 94, which)


def test_route_gradient_against_differences(device):
    """Central differences of the 64-bit oracle along random directions; the choice is held by wide gaps of a bias."""
    tokens, experts, top_k = 20, 12, 3
    logits = randn(1, tokens, experts)
    bias = 50.0 * torch.arange(experts).float()
    dw, db, dz = randn(2, tokens, top_k), 1.3, 0.4

    def value(l):
        r = oracle.route(l, top_k, bias=bias, normalize=True)
        return float((r["weights"][0] * dw).sum() + db * r["balance"][0] + dz * r["z"][0])

    leaf = logits.to(device).requires_grad_(True)
    out = nn.route_tokens(leaf, top_k, bias=bias.to(device))
    ((out.weights * dw.to(device)).sum() + db * out.balance_loss + dz * out.z_loss).backward()
    for seed in range(3):
        v = randn(10 + seed, tokens, experts)
        step = 2.0 ** -7           # truncation step^2 / 6 * third derivative ~ 1e-5 of sums of order 10; the oracle is exact
        slope = (value(logits + step * v) - value(logits - step * v)) / (2 * step)
        assert abs(slope - float((leaf.grad.cpu() * v).sum())) < 2e-3


def test_route_rows_without_a_choice(device):
    """Closed experts, rows with nothing open, the type's lowest value, and fewer open experts than choices."""
    low = torch.finfo(FP32).min
    logits = torch.tensor([[0.0, 1.0, -math.inf, 2.0], [-math.inf] * 4, [low] * 4, [-math.inf, -math.inf, 5.0, -math.inf],
                           [low, -math.inf, low, 3.0]])
    expected = oracle.route(logits, 3, dweights=torch.ones(5, 3) * torch.tensor([1.0, 2.0, 3.0]), dbalance=1.0)
    leaf = logits.to(device).requires_grad_(True)
    out = nn.route_tokens(leaf, 3)
    assert out.indices.tolist() == [[3, 1, 0], [-1, -1, -1], [0, 1, 2], [2, -1, -1], [3, 0, 2]]
    assert out.indices.cpu().equal(expected["indices"]) and out.counts.cpu().equal(expected["counts"])
    torch.testing.assert_close(out.weights.cpu(), expected["weights"][0].float(), rtol=1e-6, atol=1e-7)
    assert out.weights[1].tolist() == [0, 0, 0] and out.weights[3].tolist() == [1, 0, 0]
    torch.testing.assert_close(out.balance_loss.cpu(), expected["balance"][0].float(), rtol=1e-6, atol=0)
    ((out.weights * torch.tensor([1.0, 2.0, 3.0], device=device)).sum() + out.balance_loss).backward()
    torch.testing.assert_close(leaf.grad.cpu(), expected["dlogits"][0].float(), rtol=1e-5, atol=1e-6)
    assert leaf.grad[1].tolist() == [0, 0, 0, 0]


def test_route_all_tokens_masked(device):
    logits = torch.full((40, 8), math.nan, device=device, requires_grad=True)
    out = nn.route_tokens(logits, 2, mask=torch.zeros(40, dtype=torch.bool, device=device))
    assert out.counts.tolist() == [0] * 8 and out.balance_loss.item() == 0 and out.z_loss.item() == 0
    assert (out.indices == -1).all() and (out.weights == 0).all()
    (out.weights.sum() + out.balance_loss + out.z_loss).backward()
    assert (logits.grad == 0).all()


def test_route_passes_nan_on_with_indices_in_range(device):
    logits = randn(0, 6, 8)
    logits[2, 5], logits[4, 1] = math.nan, math.inf
    out = nn.route_tokens(logits.to(device), 3, normalize=False)
    assert ((out.indices >= 0) & (out.indices < 8)).all() and out.indices[2, 0].item() == 5 and out.indices[4, 0].item() == 1
    assert out.weights[[2, 4]].isnan().any(1).all() and out.weights[[0, 1, 3, 5]].isfinite().all()
    assert out.balance_loss.isnan() and out.z_loss.isnan() | out.z_loss.isinf()


def test_route_with_an_infinite_bias(device):
    """+inf puts an expert first and -inf last, but neither opens a closed expert or a masked token."""
    logits = torch.tensor([[0.0, 1.0, 2.0, -math.inf], [5.0, 4.0, 3.0, 2.0], [0.0, 0.0, 0.0, 0.0]], device=device)
    bias = torch.tensor([math.inf, 0.0, -math.inf, math.inf], device=device)
    out = nn.route_tokens(logits, 3, bias=bias, mask=torch.tensor([True, True, False], device=device))
    assert out.indices.tolist() == [[0, 1, -1], [0, 3, 1], [-1, -1, -1]] and out.counts.tolist() == [2, 2, 0, 1]
    torch.testing.assert_close(out.weights[1].cpu(), torch.softmax(torch.tensor([5.0, 2.0, 4.0]), 0), rtol=1e-6, atol=0)


def test_route_shapes_strides_and_no_tokens(device):
    base = randn(3, 2, 7, 24, dtype=BF16).to(device)
    logits = base[..., ::2]                                    # strided columns
    out = nn.route_tokens(logits, 2)
    flat = nn.route_tokens(logits.reshape(14, 12).contiguous(), 2)
    assert out.weights.shape == (2, 7, 2) and out.indices.shape == (2, 7, 2)
    assert torch.equal(out.weights.view(14, 2), flat.weights) and torch.equal(out.balance_loss, flat.balance_loss)
    rows = randn(4, 5, 40).to(device)[:, 3:35]                 # rows that start off a 16-byte boundary
    assert torch.equal(nn.route_tokens(rows, 2).weights, nn.route_tokens(rows.contiguous(), 2).weights)
    empty = torch.empty(0, 12, device=device, requires_grad=True)
    out = nn.route_tokens(empty, 2)
    assert out.weights.shape == (0, 2) and out.counts.tolist() == [0] * 12 and out.balance_loss.item() == 0
    (out.weights.sum() + out.balance_loss).backward()
    assert empty.grad.shape == (0, 12)
    one = nn.route_tokens(randn(5, 12).to(device), 2)
    assert one.weights.shape == (2,)


def test_route_refusals(device):
    logits = torch.zeros(4, 8, device=device)
    for bad in (dict(top_k=0), dict(top_k=9), dict(top_k=2, bias=torch.zeros(7, device=device)),
                dict(top_k=2, mask=torch.zeros(3, dtype=torch.bool, device=device)),
                dict(top_k=2, mask=torch.zeros(4, device=device))):
        with pytest.raises(ValueError):
            nn.route_tokens(logits, **bad)
    with pytest.raises(TypeError):
        nn.route_tokens(logits.double(), 2)
    with pytest.raises(TypeError):
        nn.route_tokens(logits.int(), 2)
    with pytest.raises(ValueError):
        nn.route_tokens(torch.zeros(4, 1025, device=device), 2)
    with pytest.raises(ValueError):
        nn.route_tokens(torch.zeros(4, 64, device=device), 33)
    with pytest.raises(ValueError):
        nn.route_tokens(torch.zeros((), device=device), 1)


# ------------------------------------------------------------------------------------------------ dispatch and combine
PLANS = [(1, 1, 1), (1, 2, 8), (7, 3, 5), (300, 2, 4), (33, 8, 1024), (50, 32, 40), (1000, 5, 17)]   # tokens, top_k, experts


def choices(tokens, top_k, experts, dropped=0.2, seed=0):
    g = torch.Generator().manual_seed(seed)
    indices = torch.randint(0, experts, (tokens, top_k), generator=g)
    return torch.where(torch.rand(tokens, top_k, generator=g) < dropped, -1, indices)


@pytest.mark.parametrize("case", PLANS, ids=str)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_plan(case, dtype, device):
    indices = choices(*case).to(dtype)
    offsets, positions = oracle.plan(indices, case[2])
    plan = nn.plan_experts(indices.to(device), case[2])
    assert torch.equal(plan.offsets.cpu(), offsets) and torch.equal(plan.positions.cpu(), positions)


def test_plan_of_many_choices_crosses_blocks(device):
    """Several blocks with ragged ends, one expert that takes most of it, out-of-range values on both sides."""
    tokens, top_k, experts = 40001, 3, 9
    g = torch.Generator().manual_seed(1)
    indices = torch.randint(-2, experts + 2, (tokens, top_k), generator=g)
    indices[torch.rand(tokens, top_k, generator=g) < 0.6] = 4
    plan = nn.plan_experts(indices.to(device), experts)
    flat = indices.reshape(-1)
    bins = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.argsort(bins, stable=True)
    counts = torch.bincount(bins, minlength=experts + 1)[:experts]
    assert plan.offsets.tolist() == [0] + counts.cumsum(0).tolist()
    expected = torch.full_like(flat, -1)
    total = int(counts.sum())
    expected[order[:total]] = torch.arange(total)
    assert torch.equal(plan.positions.cpu().long().view(-1), expected)


def test_plan_without_choices(device):
    plan = nn.plan_experts(torch.full((5, 2), -1, dtype=torch.int32, device=device), 3)
    assert plan.offsets.tolist() == [0, 0, 0, 0] and (plan.positions == -1).all()
    plan = nn.plan_experts(torch.empty(0, 2, dtype=torch.int64, device=device), 3)
    assert plan.offsets.tolist() == [0, 0, 0, 0] and plan.positions.shape == (0, 2)


EXCHANGES = [  # tokens, top_k, experts, width, dtype
    (1, 1, 1, 1, FP32), (1, 2, 8, 1152, BF16), (5, 3, 4, 7, FP16), (40, 2, 8, 1000, BF16), (33, 4, 6, 771, FP16),
    (17, 8, 12, 260, FP32), (3, 32, 40, 66, BF16), (9, 2, 3, 4100, BF16), (6, 2, 3, 9001, FP32), (260, 1, 5, 64, FP16),
]


@pytest.mark.parametrize("case", EXCHANGES, ids=str)
def test_dispatch_values_and_gradients(case, device):
    tokens, top_k, experts, width, dtype = case
    indices = choices(tokens, top_k, experts)
    x = randn(0, tokens, width, dtype=dtype)
    _, positions = oracle.plan(indices, experts)
    plan = nn.plan_experts(indices.to(device), experts)
    leaf = x.to(device).requires_grad_(True)
    rows = nn.dispatch_tokens(leaf, plan)
    expected = torch.zeros(tokens * top_k, width, dtype=dtype)
    for t, j in (positions >= 0).nonzero().tolist():
        expected[positions[t, j]] = x[t]
    assert torch.equal(rows.cpu(), expected)               # the rows behind the last are zero
    grad = randn(1, tokens * top_k, width, dtype=dtype)
    rows.backward(grad.to(device))
    back = oracle.combine(grad, torch.ones(tokens, top_k), positions)["out"]
    oracle.assert_matches(leaf.grad, back, top_k, "dx")
    assert torch.equal(nn.dispatch_tokens(leaf.detach(), plan), rows)


@pytest.mark.parametrize("case", EXCHANGES, ids=str)
@pytest.mark.parametrize("weight_dtype", [FP32, BF16])
def test_combine_values_and_gradients(case, weight_dtype, device):
    tokens, top_k, experts, width, dtype = case
    indices = choices(tokens, top_k, experts, seed=2)
    _, positions = oracle.plan(indices, experts)
    plan = nn.plan_experts(indices.to(device), experts)
    rows = randn(3, tokens * top_k, width, dtype=dtype)
    rows[int(plan.offsets[-1]):] = math.nan                # nothing of these rows may be read
    weights = torch.rand(tokens, top_k, generator=torch.Generator().manual_seed(4)).to(weight_dtype)
    dout = randn(5, tokens, width, dtype=dtype)
    expected = oracle.combine(rows.nan_to_num(0), weights, positions, dout)
    leaf, wleaf = rows.to(device).requires_grad_(True), weights.to(device).requires_grad_(True)
    out = nn.combine_tokens(leaf, wleaf, plan)
    oracle.assert_matches(out, expected["out"], top_k, "out")
    out.backward(dout.to(device))
    oracle.assert_matches(leaf.grad, expected["drows"], 1, "drows")
    oracle.assert_matches(wleaf.grad, expected["dweights"], width, "dweights")
    assert torch.equal(nn.combine_tokens(leaf.detach(), wleaf.detach(), plan), out)
    # one gradient without the other
    only_rows, = torch.autograd.grad(nn.combine_tokens(leaf, wleaf.detach(), plan), leaf, dout.to(device))
    only_weights, = torch.autograd.grad(nn.combine_tokens(leaf.detach(), wleaf, plan), wleaf, dout.to(device))
    assert torch.equal(only_rows, leaf.grad) and torch.equal(only_weights, wleaf.grad)


def test_exchange_shapes_strides_and_no_tokens(device):
    indices = choices(10, 2, 3).view(2, 5, 2).to(device)
    plan = nn.plan_experts(indices, 3)
    base = randn(0, 2, 5, 96, dtype=BF16).to(device)
    for x in (base[..., :64], base[..., 3:67], base[..., ::2], base.transpose(0, 1).contiguous().transpose(0, 1)[..., :48]):
        leaf = x.detach().requires_grad_(True)
        rows = nn.dispatch_tokens(leaf, plan)
        assert torch.equal(rows, nn.dispatch_tokens(x.contiguous(), plan))
        out = nn.combine_tokens(rows, torch.ones(2, 5, 2, device=device), plan)
        assert out.shape == x.shape
        out.backward(torch.ones_like(out).transpose(0, 1).contiguous().transpose(0, 1))
        kept = (indices >= 0).sum(-1, keepdim=True)
        assert torch.equal(leaf.grad, kept.expand(x.shape).to(BF16))
    rows = randn(1, 21, 64, dtype=BF16).to(device)[1:]        # off the start of its storage
    weights = randn(2, 2, 2, 5).to(device).permute(1, 2, 0)   # not contiguous
    assert torch.equal(nn.combine_tokens(rows, weights, plan), nn.combine_tokens(rows.clone(), weights.contiguous(), plan))
    none = nn.plan_experts(torch.empty(0, 2, dtype=torch.int32, device=device), 3)
    x = torch.empty(0, 8, device=device, requires_grad=True)
    out = nn.combine_tokens(nn.dispatch_tokens(x, none), torch.empty(0, 2, device=device), none)
    assert out.shape == (0, 8)
    out.sum().backward()
    assert x.grad.shape == (0, 8)


def test_combine_skips_positions_out_of_range(device):
    """A plan is the caller's data: positions that name no row are passed over, not followed."""
    plan = nn.ExpertPlan(torch.tensor([0, 4, 9], dtype=torch.int32, device=device),
                         torch.tensor([[0, 7], [-5, 1], [3, 2 ** 31 - 1]], dtype=torch.int32, device=device))
    rows = torch.ones(6, 16, device=device, requires_grad=True)
    out = nn.combine_tokens(rows, torch.ones(3, 2, device=device), plan)
    assert out[:, 0].tolist() == [1, 1, 1]
    out.sum().backward()
    assert rows.grad[[0, 1, 3]].eq(1).all()
    assert nn.dispatch_tokens(torch.ones(3, 16, device=device), plan)[[0, 1, 3]].eq(1).all()


def test_exchange_refusals(device):
    indices = torch.zeros(4, 2, dtype=torch.int32, device=device)
    plan = nn.plan_experts(indices, 3)
    x, rows, weights = torch.zeros(4, 16, device=device), torch.zeros(8, 16, device=device), torch.ones(4, 2, device=device)
    for bad in (lambda: nn.plan_experts(indices, 0), lambda: nn.plan_experts(indices, 1025),
                lambda: nn.plan_experts(torch.zeros(4, 33, dtype=torch.int32, device=device), 3),
                lambda: nn.plan_experts(torch.zeros(4, 0, dtype=torch.int32, device=device), 3),
                lambda: nn.dispatch_tokens(x[:3], plan), lambda: nn.dispatch_tokens(x[:, :0], plan),
                lambda: nn.combine_tokens(rows[:7], weights, plan), lambda: nn.combine_tokens(rows, weights[:, :1], plan),
                lambda: nn.combine_tokens(rows.view(4, 2, 16), weights, plan),
                lambda: nn.dispatch_tokens(x, nn.ExpertPlan(plan.offsets.long(), plan.positions)),
                lambda: nn.dispatch_tokens(x, nn.ExpertPlan(plan.offsets, plan.positions.view(-1)))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: nn.plan_experts(indices.float(), 3), lambda: nn.dispatch_tokens(x.double(), plan),
                lambda: nn.combine_tokens(rows.double(), weights, plan), lambda: nn.combine_tokens(rows, weights.double(), plan)):
        with pytest.raises(TypeError):
            bad()


# ------------------------------------------------------------------------------------------------------------- norms
NORMS = [  # batch, tokens, width, stream, branch, weights, gate, scale, post, pre, residual
    (1, 1, 1, FP32, FP32, True, "shared", "shared", True, True, 1.0),
    (1, 1, 4096, BF16, BF16, True, None, None, True, True, 1.0),
    (3, 5, 64, BF16, BF16, True, "sample", "sample", True, True, 0.5),
    (2, 7, 72, FP32, BF16, True, "sample", "shared", True, True, 1.25),
    (4, 1, 1152, FP32, BF16, False, "sample", "sample", True, True, 1.0),
    (2, 33, 1152, FP32, FP16, True, "shared", "sample", True, True, -0.7),
    (7, 3, 1001, FP16, FP16, True, "sample", None, True, False, 0.5),
    (2, 9, 771, FP32, FP32, True, None, "sample", False, True, 1.0),
    (1, 300, 256, BF16, BF16, True, None, None, True, True, 1.0),
    (300, 2, 40, FP16, FP16, True, "sample", "sample", True, True, 1.0),
    (2, 3, 2056, FP32, BF16, True, "sample", "sample", True, True, 1.0),
    (1, 4, 8192, BF16, BF16, True, "shared", None, True, True, 1.4),
    (2, 2, 8200, FP32, FP32, True, "sample", "sample", True, True, 1.0),
    (1, 2, 2049, BF16, BF16, True, "sample", "sample", True, True, 1.0),
    (1, 3, 16384, FP16, FP16, True, "sample", "sample", True, True, 1.0),
    (1, 2, 16383, FP32, BF16, True, "shared", "shared", True, True, 1.0),
    (2, 40, 512, FP32, BF16, False, None, None, True, True, 1.0),
    (2, 40, 264, BF16, BF16, False, None, None, False, True, 1.0),
]


def norm_inputs(case, seed=0):
    batch, tokens, width, stream, branch, weights, gate, scale, post, pre, _ = case
    shape = {"shared": (width,), "sample": (batch, width)}
    v = dict(x=2 * randn(seed, batch, tokens, width), y=None, weight=None, gate=None, next_weight=None, next_scale=None)
    v["x"] = v["x"].to(stream)
    if post:
        v["y"] = randn(seed + 1, batch, tokens, width, dtype=branch)
        v["weight"] = 1 + 0.2 * randn(seed + 2, width) if weights else None
        v["gate"] = 0.5 * randn(seed + 3, *shape[gate]).to(branch) if gate else None
    if pre:
        v["next_weight"] = (1 + 0.2 * randn(seed + 4, width)).to(branch) if weights else None
        v["next_scale"] = 0.3 * randn(seed + 5, *shape[scale]).to(branch) if scale else None
    dout = randn(seed + 6, batch, tokens, width, dtype=stream) if post else None
    dh = randn(seed + 7, batch, tokens, width, dtype=branch) if pre else None
    return v, dout, dh


def call_norm(case, v, **kwargs):
    post, pre, residual = case[8:]
    if not post:
        return None, nn.rms_norm_modulate(v["x"], v["next_weight"], v["next_scale"], dtype=case[4], **kwargs)
    out = nn.rms_norm_residual(v["x"], v["y"], v["weight"], v["gate"], residual_scale=residual, next_norm=pre,
                               next_weight=v["next_weight"], next_scale=v["next_scale"], **kwargs)
    return out if pre else (out, None)


@pytest.mark.parametrize("case", NORMS, ids=str)
def test_norm_values_and_gradients(case, device):
    v, dout, dh = norm_inputs(case)
    batch, tokens, width = case[:3]
    expected = oracle.block_norm(**v, residual_scale=case[10], next_norm=case[9], dout=dout, dh=dh)
    leaves = {n: None if t is None else t.to(device).requires_grad_(True) for n, t in v.items()}
    out, h = call_norm(case, leaves)
    outs, grads = [], []
    for name, t, g in (("out", out, dout), ("h", h, dh)):
        if t is not None:
            oracle.assert_matches(t, expected[name], width, name)
            outs.append(t)
            grads.append(g.to(device))
    torch.autograd.backward(outs, grads)
    for name, leaf in leaves.items():
        if leaf is not None:
            assert leaf.grad.dtype == leaf.dtype
            oracle.assert_matches(leaf.grad, expected["d" + name], width + batch * tokens, "d" + name)
    plain = call_norm(case, {n: None if t is None else t.detach() for n, t in leaves.items()})
    for a, b in zip(plain, (out, h)):
        assert a is None and b is None or torch.equal(a, b)


@pytest.mark.parametrize("which", ["out", "h"])
def test_norm_gradient_of_one_output(which, device):
    case = (3, 5, 200, FP32, BF16, True, "sample", "sample", True, True, 0.8)
    v, dout, dh = norm_inputs(case, 3)
    only = dict(dout=dout if which == "out" else None, dh=dh if which == "h" else None)
    expected = oracle.block_norm(**v, residual_scale=0.8, **only)
    leaves = {n: t.to(device).requires_grad_(True) for n, t in v.items()}
    out, h = call_norm(case, leaves)
    (out if which == "out" else h).backward((dout if which == "out" else dh).to(device))
    for name, leaf in leaves.items():
        if "d" + name in expected and not (which == "out" and name.startswith("next")):
            oracle.assert_matches(leaf.grad, expected["d" + name], 215, "d" + name)
        else:
            assert leaf.grad is None or not leaf.grad.any()


def test_norm_gradient_against_differences(device):
    case = (2, 4, 24, FP32, FP32, True, "sample", "sample", True, True, 0.9)
    v, dout, dh = norm_inputs(case, 9)

    def value(inputs):
        r = oracle.block_norm(**inputs, residual_scale=0.9)
        return float((r["out"][0] * dout).sum() + (r["h"][0] * dh).sum())

    leaves = {n: t.to(device).requires_grad_(True) for n, t in v.items()}
    out, h = call_norm(case, leaves)
    torch.autograd.backward([out, h], [dout.to(device), dh.to(device)])
    for seed, name in enumerate(v):
        direction = randn(20 + seed, *v[name].shape)
        step = 2.0 ** -8             # truncation step^2 / 6 * third derivative ~ 1e-4 at most; the oracle is exact
        slope = (value({**v, name: v[name].double() + step * direction}) - value({**v, name: v[name].double() - step * direction})) / (2 * step)
        assert abs(slope - float((leaves[name].grad.cpu() * direction).sum())) < 5e-3 * max(1.0, abs(slope)), name


def test_norm_needs_only_what_is_asked(device):
    case = (3, 4, 136, BF16, BF16, True, "sample", "sample", True, True, 1.1)
    v, dout, dh = norm_inputs(case, 4)
    expected = oracle.block_norm(**v, residual_scale=1.1, dout=dout, dh=dh)
    full = {n: t.detach().to(device).requires_grad_(True) for n, t in v.items()}
    torch.autograd.backward(call_norm(case, full), [dout.to(device), dh.to(device)])
    for name in v:
        some = {n: t.detach().to(device).requires_grad_(n == name) for n, t in v.items()}
        reached = [(t, g.to(device)) for t, g in zip(call_norm(case, some), (dout, dh)) if t.requires_grad]
        torch.autograd.backward(*zip(*reached))
        oracle.assert_matches(some[name].grad, expected["d" + name], 136 + 12, name)
        assert device == "cpu" or torch.equal(some[name].grad, full[name].grad)
        assert all(t.grad is None for n, t in some.items() if n != name)


def test_norm_strides_views_and_broadcast_vectors(device):
    """Chunks of an adaLN projection, transposed and offset streams, expanded vectors: the same numbers as contiguous copies."""
    batch, tokens, width = 3, 6, 64
    ada = randn(0, batch, 6 * width, dtype=BF16).to(device)
    gate, scale = ada.chunk(6, -1)[2], ada.chunk(6, -1)[4]
    x = randn(1, tokens, batch, width).to(device).transpose(0, 1)
    y = randn(2, batch, tokens, width + 3, dtype=BF16).to(device)[..., 3:]
    w = randn(3, 2 * width).to(device)[::2]
    views, copies = [], []
    for make, store in ((lambda t: t, views), (lambda t: t.contiguous(), copies)):
        for g in (gate, gate[:1].expand(batch, width), gate[0]):
            leaves = [make(t).detach().requires_grad_(True) for t in (x, y, w, g, w, scale)]
            out, h = nn.rms_norm_residual(leaves[0], leaves[1], leaves[2], leaves[3], next_norm=True, next_weight=leaves[4],
                                          next_scale=leaves[5])
            (out.float().sum() + (h.float() * h.float()).sum()).backward()
            store += [out, h] + [t.grad for t in leaves]
    for a, b in zip(views, copies):
        assert torch.equal(a, b)
    flat = nn.rms_norm_modulate(x.reshape(-1, width)[0].contiguous())            # one vector
    assert flat.shape == (width,)
    per_row = nn.rms_norm_modulate(x.reshape(-1, width), scale=x.reshape(-1, width))  # a 2-D stream: one scale per row
    assert per_row.shape == (batch * tokens, width)


@pytest.mark.parametrize("width", [40, 250, 263, 1153])
@pytest.mark.parametrize("types", [(FP32, BF16), (FP16, FP16)])
def test_norm_rows_at_any_address(width, types, device):
    """Contiguous streams that begin anywhere in their storage, results and gradients included, next to untouched memory."""
    stream, branch = types
    for offset in (1, 2, 3, 6, 7):
        case = (2, 3, width, stream, branch, True, "sample", "sample", True, True, 0.75)
        v, dout, dh = norm_inputs(case, offset)
        expected = oracle.block_norm(**v, residual_scale=0.75, dout=dout, dh=dh)

        def moved(t):
            store = torch.full((t.numel() + 16,), math.nan, dtype=t.dtype, device=device)
            view = store[offset:offset + t.numel()].view(t.shape)
            view.copy_(t)
            return view

        leaves = {n: moved(t).requires_grad_(True) if n in ("x", "y") else t.to(device).requires_grad_(True) for n, t in v.items()}
        out, h = call_norm(case, leaves)
        torch.autograd.backward([out, h], [moved(dout), moved(dh)])
        for name, t in (("out", out), ("h", h)):
            oracle.assert_matches(t, expected[name], width, name)
        for name, leaf in leaves.items():
            oracle.assert_matches(leaf.grad, expected["d" + name], width + 6, "d" + name)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [8, 9, 24, 257, 519, 1031])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_norm_writes_its_rows_and_nothing_else(cols, dtype):
    """The C entry writes results at odd addresses: the bytes around them stay."""
    import ctypes

    class Vector(ctypes.Structure):
        _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int), ("pitch", ctypes.c_longlong)]

    class Norm(ctypes.Structure):
        _fields_ = [(n, ctypes.c_int) for n in ("rows", "cols", "tokens", "x_dtype", "y_dtype")] + [
            ("residual_scale", ctypes.c_float), ("eps", ctypes.c_float), ("x", ctypes.c_void_p), ("y", ctypes.c_void_p)] + [
            (n, Vector) for n in ("weight", "gate", "next_weight", "next_scale")] + [
            (n, ctypes.c_void_p) for n in ("out", "h", "ry", "ru")]

    ops.load()
    library = ctypes.CDLL(str(ops._LIB_PATH))
    rows, code = 5, {FP32: 0, BF16: 1}[dtype]
    x, y = randn(0, rows, cols, dtype=dtype).cuda(), randn(1, rows, cols, dtype=dtype).cuda()
    expected, following = nn.rms_norm_residual(x, y, next_norm=True)
    for offset in range(8):
        stores = [torch.full((rows * cols + 32,), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        views = [s[8 + offset:8 + offset + rows * cols] for s in stores]
        norm = Norm(rows, cols, rows, code, code, 1.0, 1e-6, x.data_ptr(), y.data_ptr(), *[Vector(None, 0, 0)] * 4,
                    views[0].data_ptr(), views[1].data_ptr(), None, None)
        assert library.vb_block_norm(ctypes.byref(norm), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        for store, view, wanted in zip(stores, views, (expected, following)):
            assert torch.equal(view.view(rows, cols), wanted)
            assert store[:8 + offset].eq(7).all() and store[8 + offset + rows * cols:].eq(7).all()


def test_norm_gradient_of_an_expanded_gate(device):
    """A gate broadcast over the batch outside gets the sum over the samples."""
    case = (4, 3, 48, FP32, FP32, True, "sample", None, True, False, 1.0)
    v, dout, _ = norm_inputs(case, 6)
    leaf = v["gate"][:1].to(device).requires_grad_(True)
    out = nn.rms_norm_residual(v["x"].to(device), v["y"].to(device), v["weight"].to(device), leaf.expand(4, 48))
    out.backward(dout.to(device))
    expected = oracle.block_norm(v["x"], v["y"], v["weight"], v["gate"][0], next_norm=False, dout=dout)["dgate"]
    oracle.assert_matches(leaf.grad[0], expected, 48 + 12 + 4, "gate")


def test_norm_zero_rows_and_extreme_values(device):
    x = torch.zeros(2, 3, 40, device=device, requires_grad=True)
    y = torch.zeros(2, 3, 40, device=device, requires_grad=True)
    out, h = nn.rms_norm_residual(x, y, next_norm=True)
    assert (out == 0).all() and (h == 0).all()
    (out + h).sum().backward()
    # by the formula: du = 1 + 1 / sqrt(eps), dx = du, dy = du / sqrt(eps)
    root = (1e-6) ** -0.5
    torch.testing.assert_close(x.grad, torch.full_like(x, 1 + root), rtol=1e-5, atol=0)
    torch.testing.assert_close(y.grad, torch.full_like(y, (1 + root) * root), rtol=1e-5, atol=0)
    big = torch.full((1, 1, 64), 3e4, dtype=FP16, device=device)          # squares overflow fp16, not fp32
    torch.testing.assert_close(nn.rms_norm_modulate(big), torch.ones_like(big), rtol=0, atol=0)
    bad = torch.ones(1, 2, 64, device=device)
    bad[0, 1, 3] = math.nan
    res = nn.rms_norm_modulate(bad)
    assert res[0, 0].isfinite().all() and res[0, 1].isnan().all()          # a row's NaN stays in its row


def test_norm_without_rows(device):
    for shape in ((0, 4, 32), (2, 0, 32)):
        x, y = (torch.empty(shape, device=device, requires_grad=True) for _ in range(2))
        w = torch.ones(32, device=device, requires_grad=True)
        gate = torch.ones(shape[0], 32, device=device, requires_grad=True)
        out, h = nn.rms_norm_residual(x, y, w, gate, next_norm=True, next_weight=w)
        assert out.shape == shape and h.shape == shape
        (out.sum() + h.sum()).backward()
        assert x.grad.shape == shape and w.grad.eq(0).all() and gate.grad.eq(0).all()


def test_norm_dtype_rules(device):
    x = torch.randn(2, 3, 32, device=device)
    assert nn.rms_norm_modulate(x).dtype == FP32 and nn.rms_norm_modulate(x, dtype=BF16).dtype == BF16
    assert nn.rms_norm_modulate(x.bfloat16()).dtype == BF16
    out, h = nn.rms_norm_residual(x, x.half(), next_norm=True)
    assert out.dtype == FP32 and h.dtype == FP16
    if device == "cuda":
        with torch.autocast("cuda", dtype=BF16):
            assert nn.rms_norm_modulate(x).dtype == BF16 and nn.rms_norm_modulate(x.half()).dtype == FP16


def test_norm_refusals(device):
    x, w = torch.zeros(2, 3, 32, device=device), torch.ones(32, device=device)
    for bad in (dict(weight=w[:31]), dict(weight=torch.ones(2, 32, device=device)), dict(gate=torch.ones(3, 32, device=device)),
                dict(gate=torch.ones(2, 3, 32, device=device)), dict(next_weight=w), dict(next_scale=w), dict(eps=0.0),
                dict(eps=math.nan), dict(eps=1e-60), dict(eps=math.inf), dict(residual_scale=math.inf), dict(residual_scale=math.nan),
                dict(residual_scale=-1e39), dict(residual_scale=w)):
        with pytest.raises(ValueError):
            nn.rms_norm_residual(x, x, **bad)
    for bad in (lambda: nn.rms_norm_residual(x, x[:1]), lambda: nn.rms_norm_modulate(torch.zeros(2, 16385, device=device)),
                lambda: nn.rms_norm_modulate(torch.zeros(2, 0, device=device)),
                lambda: nn.rms_norm_modulate(torch.zeros((), device=device))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: nn.rms_norm_residual(x.half(), x), lambda: nn.rms_norm_residual(x.double(), x.double()),
                lambda: nn.rms_norm_residual(x, x.double()), lambda: nn.rms_norm_residual(x, x.double(), next_norm=True),
                lambda: nn.rms_norm_residual(x, x, w.double()),
                lambda: nn.rms_norm_modulate(x.half(), dtype=FP32), lambda: nn.rms_norm_modulate(x, dtype=torch.float64)):
        with pytest.raises(TypeError):
            bad()


def test_operands_on_two_devices_are_refused():
    """The meta device stands for another GPU."""
    x, other = torch.zeros(4, 8), torch.zeros(4, 8, device="meta")
    plan = nn.plan_experts(torch.zeros(4, 2, dtype=torch.int32), 3)
    for bad in (lambda: nn.route_tokens(x, 2, bias=other[0]),
                lambda: nn.route_tokens(x, 2, mask=torch.zeros(4, dtype=torch.bool, device="meta")),
                lambda: nn.dispatch_tokens(other, plan), lambda: nn.combine_tokens(other.repeat(2, 1), torch.ones(4, 2), plan),
                lambda: nn.combine_tokens(x.repeat(2, 1), torch.ones(4, 2, device="meta"), plan),
                lambda: nn.rms_norm_residual(x, other), lambda: nn.rms_norm_modulate(x, other[0])):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------------------- with the expert linear
@pytest.mark.parametrize("scaling", ["current", "grouped"])
def test_expert_linear_leaves_zeros_behind_the_last_expert(scaling, device):
    layer = nn.GroupedLinear(3, 128, 256, scaling=scaling).to(device)
    offsets = torch.tensor([0, 5, 5, 140], dtype=torch.int32, device=device)
    x = randn(0, 300, 128, dtype=BF16).to(device).requires_grad_(True)
    dirt = torch.full((300, 256), math.nan, dtype=BF16, device=device)       # what the allocator may hand out again
    del dirt
    y = layer(x, offsets)
    assert y[140:].eq(0).all() and y[:140].isfinite().all() and y[:140].ne(0).any()
    y.backward(torch.ones_like(y))
    assert x.grad[140:].eq(0).all() and x.grad[:140].ne(0).any()


def test_expert_gemm_leaves_the_rest_of_a_given_result(device):
    codes, weights = randn(1, 40, 128).to(device), randn(2, 2, 64, 128).to(device)
    scale, offsets = torch.ones(1, device=device), torch.tensor([0, 7, 25], dtype=torch.int32, device=device)
    q, _ = ops.quantize(codes, scale)
    w, _ = ops.quantize(weights.view(128, 128), scale)
    out = torch.full((40, 64), 7.0, device=device)
    assert ops.expert_gemm(q, w.view(2, 64, 128), offsets, scale, scale, out_dtype=FP32, out=out) is out
    fresh = ops.expert_gemm(q, w.view(2, 64, 128), offsets, scale, scale, out_dtype=FP32)
    assert out[25:].eq(7).all() and fresh[25:].eq(0).all() and torch.equal(out[:25], fresh[:25])


def expert_block(x, logits, mask, first, second, weights, gate):
    """A block as a model has it: norm, experts, norm, gated residual, norm of the next block."""
    h = nn.rms_norm_modulate(x, weights[0])
    routing = nn.route_tokens(logits, 2, mask=mask)
    plan = nn.plan_experts(routing.indices, first.num_experts)
    rows = first(nn.dispatch_tokens(h, plan), plan.offsets)
    rows = second(torch.nn.functional.silu(rows), plan.offsets)
    y = nn.combine_tokens(rows, routing.weights, plan)
    out, following = nn.rms_norm_residual(x, y, weights[1], gate, residual_scale=0.9, next_norm=True, next_weight=weights[2])
    return out, following, routing


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", ["current", "grouped"])
@pytest.mark.parametrize("padded", [False, True])
def test_expert_block_matches_the_cpu_path(scaling, padded):
    """The operators together around FP8 expert linears, kernels against restatements.  Both sides quantise the same values
    up to rounding; a value on the border of two FP8 codes may fall on either side of it (a step of 2^-3 at most, for a
    share of about 2^-8 of the values), hence 2 % in the norm."""
    batch, tokens, width, hidden, experts = 2, 75, 128, 256, 5
    torch.manual_seed(0)
    first, second = nn.GroupedLinear(experts, width, hidden, scaling=scaling), nn.GroupedLinear(experts, hidden, width, scaling=scaling)
    mask = torch.rand(batch, tokens) < 0.7 if padded else None
    x, logits = torch.randn(batch, tokens, width).bfloat16(), torch.randn(batch, tokens, experts)
    if padded:
        logits[~mask] = math.nan
    weights, gate = [1 + 0.1 * torch.randn(width) for _ in range(3)], torch.randn(batch, width).bfloat16()
    grads = torch.randn(2, batch, tokens, width).bfloat16()
    results = []
    for device in ("cpu", "cuda"):
        a, b = first.to(device), second.to(device)
        a.zero_grad()
        b.zero_grad()
        leaves = [t.detach().to(device).requires_grad_(True) for t in (x, logits, *weights, gate)]
        # leave NaN in freed memory, which results that are not written would show
        dirt = [torch.full((4 * batch * tokens, hidden), math.nan, device=device) for _ in range(4)]
        del dirt
        out, following, routing = expert_block(leaves[0], leaves[1], None if mask is None else mask.to(device), a, b, leaves[2:5],
                                               leaves[5])
        loss = (out * grads[0].to(device)).float().sum() + (following * grads[1].to(device)).float().sum()
        (loss + 0.1 * routing.balance_loss + 0.01 * routing.z_loss).backward()
        results.append([t.detach().float().cpu() for t in (out, following, *(t.grad for t in leaves), a.weight.grad, b.weight.grad)])
        if padded:
            assert leaves[1].grad[~mask.to(device)].eq(0).all()
            torch.testing.assert_close(out[~mask.to(device)], 0.9 * leaves[0][~mask.to(device)], rtol=2 ** -7, atol=0)
    for i, (cpu, gpu) in enumerate(zip(*results)):
        assert gpu.isfinite().all(), i
        assert (gpu - cpu).norm() <= 0.02 * cpu.norm(), (i, float((gpu - cpu).norm() / cpu.norm()))


# ---------------------------------------------------------------------------------------------- graphs, streams, large sizes
def whole_pass(logits, x, y, weights, gate, mask):
    """Every operator forward and backward; leaves in, results and gradients out."""
    routing = nn.route_tokens(logits, 3, mask=mask)
    plan = nn.plan_experts(routing.indices, logits.shape[-1])
    rows = nn.dispatch_tokens(x, plan)
    z = nn.combine_tokens(rows * 1.5, routing.weights, plan).view(x.shape)
    out, h = nn.rms_norm_residual(y, z, weights, gate, next_norm=True, next_weight=weights)
    loss = out.sum() + (h * h).sum() + 0.1 * routing.balance_loss + 0.01 * routing.z_loss
    return [routing.indices, plan.offsets, plan.positions, rows.detach(), out.detach(), h.detach(),
            *torch.autograd.grad(loss, (logits, x, y, weights, gate))]


def pass_leaves(seed, batch=4, tokens=300, width=192, experts=40):
    return [randn(seed, batch * tokens, experts).cuda().requires_grad_(True),
            *(randn(seed + i, batch, tokens, width).cuda().requires_grad_(True) for i in (1, 2)),
            randn(seed + 3, width).cuda().requires_grad_(True), randn(seed + 4, batch, width).cuda().requires_grad_(True),
            (torch.rand(batch * tokens, generator=torch.Generator().manual_seed(seed)) < 0.8).cuda()]


@pytest.mark.gpu
def test_results_repeat_bit_for_bit():
    leaves = pass_leaves(0, batch=16, tokens=1000)
    first = whole_pass(*leaves)
    for _ in range(3):
        for a, b in zip(first, whole_pass(*leaves)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_graphs_share_nothing():
    """Two captured passes, replayed on new inputs, one after the other and on two streams at once."""
    torch.cuda.synchronize()
    captured = []
    for seed in (0, 50):
        leaves = pass_leaves(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            whole_pass(*leaves)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = whole_pass(*leaves)
        captured.append((graph, leaves, results))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for attempt in range(5):
        expected = []
        for i, (_, leaves, _) in enumerate(captured):
            fresh = pass_leaves(1000 + 100 * attempt + 10 * i)
            for leaf, value in zip(leaves, fresh):
                leaf.detach().copy_(value.detach())
            expected.append([t.clone() for t in whole_pass(*fresh)])
        torch.cuda.synchronize()
        for stream, (graph, _, _) in zip(streams, captured):
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for wanted, (_, _, results) in zip(expected, captured):
            for a, b in zip(wanted, results):
                assert torch.equal(a, b)
    captured.clear()


@pytest.mark.gpu
def test_two_streams_at_once():
    sets = [pass_leaves(7), pass_leaves(70)]
    expected = [whole_pass(*leaves) for leaves in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for stream, leaves, results in zip(streams, sets, got):
            with torch.cuda.stream(stream):
                results.append(whole_pass(*leaves))
    torch.cuda.synchronize()
    for wanted, results in zip(expected, got):
        for result in results:
            for a, b in zip(wanted, result):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    logits, x, y, weights, gate, mask = pass_leaves(3)
    out = nn.rms_norm_modulate(x, weights)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(out.sum(), x, create_graph=True)


@pytest.mark.gpu
def test_in_place_changes_of_saved_inputs_are_noticed():
    logits, x, y, weights, gate, mask = pass_leaves(4)
    values = x * 1.0
    out = nn.rms_norm_residual(values, y, weights, gate, next_norm=True)[1]
    values.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Buffers of more than 2^31 values: the last rows against the same rows alone."""
    tokens, top_k, width, last = 131200, 8, 2056, 37
    x = torch.randn(tokens, width, device="cuda", dtype=BF16)
    indices = torch.arange(top_k, device="cuda", dtype=torch.int32).repeat(tokens, 1)
    plan = nn.plan_experts(indices, top_k)
    assert tokens * top_k * width > 2 ** 31
    rows = nn.dispatch_tokens(x, plan)
    for e in (0, top_k - 1):
        assert torch.equal(rows[(e + 1) * tokens - last:(e + 1) * tokens], x[-last:])
    weights = torch.rand(tokens, top_k, device="cuda")
    small = nn.plan_experts(indices[:last], top_k)
    dout = torch.randn(tokens, width, device="cuda", dtype=BF16)
    rows, weights = rows.requires_grad_(True), weights.requires_grad_(True)
    out = nn.combine_tokens(rows, weights, plan)
    drows, dweights = torch.autograd.grad(out, (rows, weights), dout)
    tail = [t.detach().requires_grad_(True) for t in (nn.dispatch_tokens(x[-last:], small), weights[-last:])]
    tail_out = nn.combine_tokens(*tail, small)
    tail_grads = torch.autograd.grad(tail_out, tail, dout[-last:])
    assert torch.equal(out[-last:], tail_out)
    # few tokens are shared out to more warps each: two orders of the same sum, each off by at most n u * sum of |terms|
    terms = (dout[-last:].float().abs() * x[-last:].float().abs()).sum(1, keepdim=True)
    assert ((dweights[-last:] - tail_grads[1]).abs() <= 2 * width * 2.0 ** -24 * terms).all()
    assert torch.equal(drows[-last:], tail_grads[0][-last:])
    del rows, drows, out, x, dout, weights
    rows, width = 262200, 8200
    assert rows * width > 2 ** 31
    x = torch.randn(1, rows, width, device="cuda", dtype=BF16).requires_grad_(True)
    h = nn.rms_norm_modulate(x)
    dx, = torch.autograd.grad(h, x, h.detach())
    part = x.detach()[:, -last:].clone().requires_grad_(True)
    h_part = nn.rms_norm_modulate(part)
    assert torch.equal(h[:, -last:], h_part)
    assert torch.equal(dx[:, -last:], torch.autograd.grad(h_part, part, h_part.detach())[0])
    del x, h, dx
    tokens, experts = 2100000, 1024
    assert tokens * experts > 2 ** 31
    logits = torch.randn(tokens, experts, device="cuda", dtype=BF16)
    out, part = nn.route_tokens(logits, 2), nn.route_tokens(logits[-last:], 2)
    assert torch.equal(out.indices[-last:], part.indices) and torch.equal(out.weights[-last:], part.weights)
    assert int(out.counts.sum()) == 2 * tokens


@pytest.mark.gpu
def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    leaves = [t.detach().to("cuda:1").requires_grad_(t.requires_grad) for t in pass_leaves(11)]
    expected = whole_pass(*pass_leaves(11))
    for a, b in zip(expected, whole_pass(*leaves)):
        assert b.device.index == 1 and torch.equal(a.cpu(), b.cpu())


# ------------------------------------------------------------------------------------------------------- forward mode
def test_operators_refuse_tangents_before_anything_else():
    """The operators read values alone: a tangent is refused, whether or not a gradient is asked for.  Needs no GPU."""
    forward_ad = torch.autograd.forward_ad
    library = ops._ops()
    x, positions, offsets = torch.ones(4, 8), torch.zeros(4, 1, dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32)
    vector, rows = torch.ones(8), torch.ones(4, 8)
    calls = {
        "route": lambda t: library.route(t, 2, None, None, True),
        "dispatch": lambda t: library.expert_dispatch(t, positions, offsets),
        "combine rows": lambda t: library.expert_combine(t, torch.ones(4, 1), positions, offsets),
        "combine weights": lambda t: library.expert_combine(rows, t[:, :1], positions, offsets),
        "norm x": lambda t: library.block_norm(t, None, None, None, None, None, 1.0, 1e-6, 0),
        "norm y": lambda t: library.block_norm(x, t, None, None, None, None, 1.0, 1e-6, -1),
        "norm weight": lambda t: library.block_norm(x, x, t[0], None, None, None, 1.0, 1e-6, -1),
        "norm gate": lambda t: library.block_norm(x, x, vector, t[0], None, None, 1.0, 1e-6, -1),
        "norm next weight": lambda t: library.block_norm(x, None, None, None, t[0], None, 1.0, 1e-6, 0),
        "norm next scale": lambda t: library.block_norm(x, None, None, None, vector, t[0], 1.0, 1e-6, 0),
    }
    for name, call in calls.items():
        for wants_grad in (False, True):
            with forward_ad.dual_level():
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(forward_ad.make_dual(x.clone().requires_grad_(wants_grad), torch.ones_like(x)))
                    pytest.fail(name)


def test_tangents_reach_the_results_or_are_refused(device):
    """A result never comes back without the tangent of its inputs: on the CPU it has one, on the GPU the call is refused.
    The bias of the router moves the choice alone and has none to pass on."""
    forward_ad = torch.autograd.forward_ad
    x, vector = randn(0, 4, 8).to(device), randn(1, 8).to(device)
    weights = torch.rand(4, 2, generator=torch.Generator().manual_seed(2)).to(device)
    plan = nn.plan_experts(choices(4, 2, 3, dropped=0).to(device), 3)
    for primal, call in ((x, lambda t: nn.route_tokens(t, 2).weights), (x, lambda t: nn.dispatch_tokens(t, plan)),
                         (x.repeat(2, 1), lambda t: nn.combine_tokens(t, weights, plan)),
                         (weights, lambda t: nn.combine_tokens(x.repeat(2, 1), t, plan)),
                         (x, lambda t: nn.rms_norm_modulate(t)), (vector, lambda t: nn.rms_norm_modulate(x, t)),
                         (vector, lambda t: nn.rms_norm_modulate(x, scale=t)), (x, lambda t: nn.rms_norm_residual(x, t)),
                         (vector, lambda t: nn.rms_norm_residual(x, x, t)), (vector, lambda t: nn.rms_norm_residual(x, x, None, t))):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(primal, torch.ones_like(primal))
            if device == "cpu":
                assert forward_ad.unpack_dual(call(dual)).tangent is not None
            else:
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(dual)
    with forward_ad.dual_level():
        biased = nn.route_tokens(x, 2, bias=forward_ad.make_dual(vector, torch.ones_like(vector)))
        assert torch.equal(biased.indices, nn.route_tokens(x, 2, bias=vector).indices)


@pytest.mark.gpu
def test_tangents_of_gradients_are_refused():
    forward_ad = torch.autograd.forward_ad
    x = randn(0, 4, 8).cuda().requires_grad_(True)
    weights = torch.rand(4, 2, generator=torch.Generator().manual_seed(2)).cuda()
    plan = nn.plan_experts(choices(4, 2, 3, dropped=0).cuda(), 3)
    rows = randn(1, 8, 8).cuda().requires_grad_(True)
    for leaf, out in ((x, nn.route_tokens(x, 2).weights), (x, nn.dispatch_tokens(x, plan)),
                      (rows, nn.combine_tokens(rows, weights, plan)), (x, nn.rms_norm_modulate(x))):
        with forward_ad.dual_level():
            grad = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaf, grad)


# ----------------------------------------------------------------------------------- many rows to a group of the kernels
# Row groups of the norms' kernels take equal shares of consecutive rows: at most 148 blocks times those an SM holds times 8,
# 4, 2 or 1 rows at a time.  More rows than that put several to a group, and samples then begin and end inside one, cover it,
# or reach over many.
def check_many_rows(case, seed=0):
    """As :func:`test_norm_values_and_gradients`, on the GPU; every sum has the terms that are its own."""
    v, dout, dh = norm_inputs(case, seed)
    batch, tokens, width = case[:3]
    expected = oracle.block_norm(**v, residual_scale=case[10], next_norm=case[9], dout=dout, dh=dh)
    leaves = {n: None if t is None else t.cuda().requires_grad_(True) for n, t in v.items()}
    results = [(n, t, g) for n, t, g in zip(("out", "h"), call_norm(case, leaves), (dout, dh)) if t is not None]
    torch.autograd.backward([t for _, t, _ in results], [g.cuda() for _, _, g in results])
    for name, t, _ in results:
        oracle.assert_matches(t, expected[name], width, name)
    for name, leaf in leaves.items():
        if leaf is not None:
            rows = 0 if name in ("x", "y") else tokens if leaf.dim() == 2 else batch * tokens
            oracle.assert_matches(leaf.grad, expected["d" + name], width + rows, "d" + name)


MANY_NARROW_ROWS = [  # one warp a row, eight rows a block at a time
    (6500, 3, 256, BF16, BF16, True, "sample", "sample", True, True, 1.0),
    (400, 50, 136, FP32, BF16, True, "sample", "sample", True, True, 0.8),
    (23, 900, 40, FP16, FP16, True, "sample", "shared", True, True, 1.2),
    (7001, 3, 131, FP32, FP32, True, "shared", "sample", True, True, 1.0),
    (301, 67, 255, BF16, BF16, True, "sample", None, True, False, 0.5),
    (900, 23, 64, FP32, FP16, True, None, "sample", False, True, 1.0),
    (1, 20003, 72, FP32, BF16, True, "shared", "shared", True, True, 1.0),
    (20003, 1, 48, BF16, BF16, True, "sample", "sample", True, True, 1.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", MANY_NARROW_ROWS, ids=str)
def test_norm_many_narrow_rows(case):
    """With several samples the first use of a group's sums is behind no barrier where a row is one warp's."""
    check_many_rows(case)


# ------------------------------------------------------------------------------------------------- the largest row counts
@pytest.mark.parametrize("cols", [1, 40, 256, 1001, 1152, 16384])
def test_norm_workspace_at_the_largest_row_counts(cols):
    """The shares of a pass stop growing once every SM is full, up to the last row count that 31 bits hold.  Needs no GPU."""
    import ctypes

    ops.load()
    workspace = ctypes.CDLL(str(ops._LIB_PATH)).vb_block_norm_workspace
    workspace.restype = ctypes.c_longlong
    for shared in (True, False):                                   # one sample, or two
        full = workspace(1 << 20, cols, 1 << (20 if shared else 19))
        for rows in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 8, 2 ** 31 - 600, 2 ** 30):
            if shared or rows % 2 == 0:
                assert full > 0 and workspace(rows, cols, rows if shared else rows // 2) == full, rows


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2 ** 31 - 1, 2 ** 31 - 3000])
def test_norm_at_the_largest_row_counts(rows):
    """Every row of one value is written, forward and backward: x -> x / sqrt(x^2 + eps), dx = dh eps / (x^2 + eps)^(3/2)."""
    values = torch.tensor([-2.0, -1.0, -0.5, 0.25, 0.5, 1.0, 3.0], device="cuda")
    eps = 0.5                                                      # so that both results are far from zero
    x = values.to(BF16).repeat((rows + 6) // 7)[:rows].view(rows, 1).requires_grad_(True)
    h = nn.rms_norm_modulate(x, eps=eps)
    wanted = (values.double() / (values.double() ** 2 + eps).sqrt())
    slope = eps / (values.double() ** 2 + eps) ** 1.5
    dx, = torch.autograd.grad(h, x, torch.ones_like(h))
    for result, value in ((h.detach(), wanted), (dx, slope)):
        # sums of one term, a root and four products in fp32, 16 steps of 2^-24 at most (the slope: of terms three times its
        # size or less times a cancellation of 1 - uh^2 >= 1 / 19), and one rounding by 2^-8 of the value at most
        low, high = (value - (2.0 ** -8 + 2.0 ** -14) * value.abs()).float(), (value + (2.0 ** -8 + 2.0 ** -14) * value.abs()).float()
        low, high = torch.minimum(low, high), torch.maximum(low, high)
        for first in range(0, rows, 7 << 25):                      # a multiple of the seven values at a time
            part = result[first:first + (7 << 25), 0].float()
            whole = part[:part.numel() // 7 * 7].view(-1, 7)
            assert ((whole >= low) & (whole <= high)).all(), first
            rest = part[whole.numel():]
            assert ((rest >= low[:rest.numel()]) & (rest <= high[:rest.numel()])).all(), first


@pytest.mark.gpu
def test_route_counts_choices_past_31_bits():
    """2^31 choices and more: the balance loss divides by their number.  All tokens have the same logits (one row in memory), 16
    of 17 experts are chosen: counts_e = tokens for the 16, balance = 17 / 16 * (1 - p of the other)."""
    tokens, experts, top_k = 2 ** 27 + 5, 17, 16
    row = torch.linspace(-1.0, 1.0, experts).to(FP16)
    out = nn.route_tokens(row.cuda().expand(tokens, experts), top_k)
    assert out.counts.tolist() == [0] + [tokens] * 16 and tokens * top_k > 2 ** 31
    p = torch.softmax(row.double(), 0)
    # a lane adds the p of tokens / (592 blocks * 16 tokens a pass) of them, each addition off by 2^-24 of the sum at most
    off = (tokens / (592 * 16) + 700) * 2.0 ** -24
    assert abs(float(out.balance_loss) / (17 / 16 * float(1 - p[0])) - 1) < off
    assert abs(float(out.z_loss) / float(torch.logsumexp(row.double(), 0) ** 2) - 1) < off
    assert int(out.indices[-1].sum()) == sum(range(1, 17)) and abs(float(out.weights[-1].sum()) - 1) < 1e-6


# ---------------------------------------------------------------------------------------------------- counted launches
def test_launch_count_is_read_without_a_gpu():
    before = ops.launch_count
    ops._count(3)
    assert ops.launch_count == before + 3
    assert ops._ops().block_launches() >= 0 and not hasattr(ops, "launch_counts")


@pytest.mark.gpu
def test_launch_count_includes_the_block_operators():
    def launched(call):
        before = ops.launch_count
        result = call()
        return ops.launch_count - before, result

    def logits(tokens):
        return randn(0, tokens, 60).cuda().requires_grad_(True)

    assert launched(lambda: nn.route_tokens(logits(1), 2))[0] == 1                # one block: no finishing kernel
    count, routing = launched(lambda: nn.route_tokens(logits(5003), 4))
    assert count == 2
    assert launched(lambda: routing.z_loss.backward())[0] == 1
    assert launched(lambda: nn.plan_experts(routing.indices[:9], 60))[0] == 1
    count, plan = launched(lambda: nn.plan_experts(routing.indices, 60))
    assert count == 2
    x = randn(1, 5003, 64).cuda().requires_grad_(True)
    count, rows = launched(lambda: nn.dispatch_tokens(x, plan))
    assert count == 1 and launched(lambda: rows.backward(rows.detach(), retain_graph=True))[0] == 1
    count, out = launched(lambda: nn.combine_tokens(rows.detach().requires_grad_(True), routing.weights.detach(), plan))
    assert count == 1 and launched(lambda: out.backward(out.detach()))[0] == 1
    count, h = launched(lambda: nn.rms_norm_modulate(x))
    assert count == 1 and launched(lambda: h.backward(h.detach()))[0] == 1
    weight = torch.ones(64, device="cuda", requires_grad=True)
    count, h = launched(lambda: nn.rms_norm_modulate(x, weight))
    assert count == 1 and launched(lambda: h.backward(h.detach()))[0] == 2       # and the kernel of the vectors' sums
    assert launched(lambda: nn.route_tokens(torch.empty(0, 8, device="cuda"), 2))[0] == 1
    none = nn.plan_experts(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 3)
    assert launched(lambda: nn.dispatch_tokens(torch.empty(0, 64, device="cuda"), none))[0] == 0


@pytest.mark.parametrize("columns, out_dtype", [(64, FP32), (200, BF16), (68, BF16), (1152, BF16)])
def test_expert_gemm_clears_many_rows_behind_the_last_experts(columns, out_dtype, device):
    """More rows than the clearing warps take at a time, rows on and off 16 bytes, and nothing to clear."""
    rows, experts = 5003, 2
    q, _ = ops.quantize(randn(1, rows, 128).to(device), torch.ones(1, device=device))
    w, _ = ops.quantize(randn(2, experts * columns, 128).to(device), torch.ones(1, device=device))
    scale = torch.ones(1, device=device)
    results = []
    for used in (0, 17, 2600, rows):
        offsets = torch.tensor([0, used // 2, used], dtype=torch.int32, device=device)
        dirt = torch.full((rows, columns), math.nan, dtype=out_dtype, device=device)      # what the allocator may hand out again
        del dirt
        y = ops.expert_gemm(q, w.view(experts, columns, 128), offsets, scale, scale, out_dtype=out_dtype)
        assert y[used:].eq(0).all() and y[:used].isfinite().all() and y[:used].ne(0).any(1).all()
        results.append(y)
    assert torch.equal(results[2][:8], results[1][:8]) and torch.equal(results[2][2592:2600], results[3][2592:2600])


# --------------------------------------------------------------------------- shares of more than one row, token or block
MANY_ROWS = [  # batch, tokens, width, stream, branch, weights, gate, scale, post, pre, residual; 8 to 1 rows a block at a time
    (1500, 4, 264, BF16, BF16, True, "sample", "sample", True, True, 1.0),
    (1201, 5, 511, FP32, BF16, True, "sample", "sample", True, True, 0.7),
    (700, 5, 520, FP16, FP16, True, "shared", "sample", True, True, 1.0),
    (9, 401, 771, FP32, FP32, True, "sample", "sample", True, True, 1.1),
    (1000, 3, 1152, FP32, BF16, True, "sample", "sample", True, True, 1.0),
    (12, 251, 1152, BF16, BF16, True, "sample", "sample", True, True, 0.5),
    (2000, 1, 1152, BF16, BF16, True, "sample", "sample", True, True, 1.0),
    (1, 4001, 1152, FP32, BF16, True, "shared", "shared", True, True, 1.0),
    (64, 51, 1152, FP32, FP16, True, None, "sample", False, True, 1.0),
    (64, 51, 1152, FP32, BF16, True, "sample", None, True, False, 1.0),
    (7, 1025, 1001, FP16, FP16, True, "sample", None, True, False, 0.5),
    (150, 5, 2056, BF16, BF16, True, "sample", "sample", True, True, 1.0),
    (3, 251, 2049, FP32, BF16, False, "sample", "shared", True, True, 1.0),
    (60, 13, 4104, BF16, BF16, True, "sample", "sample", True, True, 1.0),
    (5, 125, 4099, FP16, FP16, True, "sample", "sample", True, True, 1.0),
    (45, 11, 8200, BF16, BF16, True, "sample", "sample", True, True, 1.0),
    (2, 211, 8201, FP32, BF16, True, "shared", "sample", True, True, 1.0),
    (7, 61, 16384, BF16, BF16, True, "sample", "sample", True, True, 1.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", MANY_ROWS, ids=str)
def test_norm_many_rows(case):
    check_many_rows(case)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [1, 3])
@pytest.mark.parametrize("case", [MANY_ROWS[0], MANY_ROWS[4], MANY_NARROW_ROWS[1]], ids=str)
def test_norm_many_rows_off_their_boundary(case, offset):
    """Aligned widths behind pointers that are not: every row is shifted by the same bytes."""
    v, dout, dh = norm_inputs(case, 5)
    batch, tokens, width = case[:3]
    expected = oracle.block_norm(**v, residual_scale=case[10], dout=dout, dh=dh)
    moved = {n: torch.cat([t.new_zeros(offset), t.reshape(-1)]).cuda()[offset:].view(t.shape) for n, t in v.items() if n in ("x", "y")}
    leaves = {n: moved.get(n, t.cuda()).requires_grad_(True) for n, t in v.items()}
    out, h = call_norm(case, leaves)
    torch.autograd.backward([out, h], [dout.cuda(), dh.cuda()])
    for name, t in (("out", out), ("h", h)):
        oracle.assert_matches(t, expected[name], width, name)
    for name, leaf in leaves.items():
        rows = 0 if name in ("x", "y") else tokens if leaf.dim() == 2 else batch * tokens
        oracle.assert_matches(leaf.grad, expected["d" + name], width + rows, "d" + name)


@pytest.mark.parametrize("case", ROUTES, ids=str)
def test_batched_route_oracle(case):
    """The two oracles of the router agree: only then does the one for many tokens stand for the other."""
    logits, bias, mask, (dw, db, dz) = route_inputs(case, 1)
    one = oracle.route(logits, case[2], bias=bias, mask=mask, normalize=case[6], dweights=dw, dbalance=db, dz=dz)
    many = oracle.route_batch(logits, case[2], bias=bias, mask=mask, normalize=case[6], dweights=dw, dbalance=db, dz=dz)
    assert torch.equal(one["indices"], many["indices"]) and torch.equal(one["counts"], many["counts"])
    for name in ("weights", "balance", "z", "dlogits"):
        torch.testing.assert_close(many[name][0], one[name][0], rtol=1e-11, atol=1e-14)


MANY_TOKENS = [  # tokens, experts, top_k, ... as above: more than 592 blocks take at a time, or than 256 blocks' sums a finishing thread
    (40003, 4, 2, FP32, False, 0.1, True, 3),
    (20011, 8, 2, BF16, True, 0, False, 0),
    (12011, 60, 4, FP16, True, 0.2, False, 0),
    (9973, 256, 8, FP32, True, 0, True, 0),
    (10007, 256, 3, BF16, False, 0.3, True, 6),
    (5003, 129, 20, FP16, True, 0.1, True, 0),
    (4999, 512, 8, FP32, False, 0, False, 0),
    (4801, 1024, 8, BF16, True, 0.1, True, 0),
    (2500, 1000, 32, FP32, True, 0, True, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", MANY_TOKENS, ids=str)
def test_route_many_tokens(case):
    tokens, experts, top_k, _, _, _, normalize, _ = case
    logits, bias, mask, (dw, db, dz) = route_inputs(case)
    expected = oracle.route_batch(logits, top_k, bias=bias, mask=mask, normalize=normalize, dweights=dw, dbalance=db, dz=dz)
    leaf = logits.cuda().requires_grad_(True)
    out = nn.route_tokens(leaf, top_k, bias=None if bias is None else bias.cuda(), mask=None if mask is None else mask.cuda(),
                          normalize=normalize)
    assert torch.equal(out.indices.cpu(), expected["indices"]) and torch.equal(out.counts.cpu(), expected["counts"])
    oracle.assert_matches(out.weights, expected["weights"], experts, "weights")
    # the losses' sums go through a lane's tokens (at most tokens / 4736), 5 exchanges, 8 warps, 19 of 592 blocks and 32 rows
    depth = experts + tokens // 4736 + 1 + 5 + 8 + 19 + 32
    oracle.assert_matches(out.balance_loss, expected["balance"], depth, "balance")
    oracle.assert_matches(out.z_loss, expected["z"], depth, "z")
    (out.weights * dw.cuda()).sum().add(db * out.balance_loss).add(dz * out.z_loss).backward()
    oracle.assert_matches(leaf.grad, expected["dlogits"], experts, "dlogits")


MANY_EXCHANGES = [  # tokens, top_k, experts, width, dtype: 2, 5 and 8 packs a lane, of 16 bytes and of one value, 1 to 8 warps a row
    (2400, 2, 16, 1152, BF16), (2500, 2, 8, 2048, BF16), (2400, 3, 9, 771, FP16), (3001, 2, 5, 145, FP32),
    (2400, 2, 8, 1000, FP32), (5001, 4, 7, 64, FP16), (2369, 1, 3, 4104, BF16), (2400, 2, 4, 2047, BF16),
]


@pytest.mark.parametrize("case", EXCHANGES, ids=str)
def test_batched_combine_oracle(case):
    tokens, top_k, experts, width, dtype = case
    _, positions = oracle.plan(choices(tokens, top_k, experts, seed=2), experts)
    rows, weights, dout = randn(3, tokens * top_k, width, dtype=dtype), randn(4, tokens, top_k), randn(5, tokens, width, dtype=dtype)
    one, many = oracle.combine(rows, weights, positions, dout), oracle.combine_batch(rows, weights, positions, dout)
    for name in one:
        torch.testing.assert_close(many[name], one[name], rtol=1e-12, atol=1e-14)


@pytest.mark.gpu
@pytest.mark.parametrize("case", MANY_EXCHANGES, ids=str)
@pytest.mark.parametrize("weight_dtype", [FP32, FP16])
def test_exchange_of_many_tokens(case, weight_dtype):
    tokens, top_k, experts, width, dtype = case
    indices = choices(tokens, top_k, experts, seed=2)
    plan = nn.plan_experts(indices.cuda(), experts)
    positions, last = plan.positions.cpu(), int(plan.offsets[-1])
    placed = positions >= 0
    assert int(placed.sum()) == last and torch.equal(positions[placed].long().sort().values, torch.arange(last))
    x = randn(0, tokens, width, dtype=dtype)
    leaf = x.cuda().requires_grad_(True)
    sent = nn.dispatch_tokens(leaf, plan)
    expected = torch.zeros(tokens * top_k, width, dtype=dtype)
    expected[positions[placed].long()] = x[placed.nonzero(as_tuple=True)[0]]
    assert torch.equal(sent.detach().cpu(), expected)
    grad = randn(1, tokens * top_k, width, dtype=dtype)
    sent.backward(grad.cuda())
    oracle.assert_matches(leaf.grad, oracle.combine_batch(grad, torch.ones(tokens, top_k), positions)["out"], top_k, "dx")
    rows = randn(3, tokens * top_k, width, dtype=dtype)
    rows[last:] = math.nan
    weights = torch.rand(tokens, top_k, generator=torch.Generator().manual_seed(4)).to(weight_dtype)
    dout = randn(5, tokens, width, dtype=dtype)
    expected = oracle.combine_batch(rows.nan_to_num(0), weights, positions, dout)
    leaf, wleaf = rows.cuda().requires_grad_(True), weights.cuda().requires_grad_(True)
    out = nn.combine_tokens(leaf, wleaf, plan)
    oracle.assert_matches(out, expected["out"], top_k, "out")
    out.backward(dout.cuda())
    oracle.assert_matches(leaf.grad, expected["drows"], 1, "drows")
    oracle.assert_matches(wleaf.grad, expected["dweights"], width, "dweights")
