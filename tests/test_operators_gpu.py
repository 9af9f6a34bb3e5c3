"""The operators around the grouped GEMM against their definitions in 64 bits, on the CPU: the router, the gated expert
layer for a few tokens, low-rank adapters.

Tolerances follow from how results are computed.  The router works in fp32: exp(x - top) is off by up to 2^-24 |x - top|
from the rounding of its argument and two units in the last place of its own, a sum over at most 1024 positive terms
and a quotient by less than 16 units; with |x - top| <= 64 that is below 1e-5 of a weight.  Gradients of the
logits are differences of such products: off by 1e-5 of the largest term they are made of.  A result in bfloat16 or
float16 is rounded once more, by 2^-8 or 2^-11 of itself (2^-25 absolute below float16's normal range).

The layers' products are sums in fp32 of n products of two-byte numbers, which are exact: off by at most n 2^-24 times the sum of the
terms' absolute values whatever the order (in matrix instructions too, which may round twice per step: 2 n 2^-24).  That
sum of absolute values is computed beside the reference.  What is handed from one product to the next is rounded to
twice the bits of the type (2^-16 of itself in bfloat16, 2^-21 in float16, there not below 2^-25), the gated activation's exponential and
quotient are off by 2^-20, and the result is rounded once.

Whole numbers are equal."""
import ctypes
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")
ROUNDING = {torch.float32: (0.0, 0.0), torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25)}


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from grouped_gemm import ops as _ops
    return _ops


def _announce(*what):
    print("[case]", *what, flush=True)


def _close(got, want, rtol, atol, what):
    """Every element within atol + rtol |want|; what is not finite in `want` alike in `got`.  atol may be a tensor."""
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    odd = ~torch.isfinite(want)
    both_inf = torch.isinf(want)
    assert torch.equal(got[both_inf], want[both_inf]), f"{what}: infinities differ"
    off = ((got - want).abs() - (atol + rtol * want.abs())).masked_fill(odd, 0.0)
    assert float(off.max()) <= 0.0, f"{what}: off by {float(off.max())} more than allowed"


# ------------------------------------------------------------------ router

def _route_reference(logits, k, score, normalize, weights_grad=None, mass_grad=None):
    """The router by its definition in 64 bits: a sort, its formulas and their derivatives."""
    x = logits.double()
    t, e = x.shape
    chosen = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    closed = (x == -INF).all(1, keepdim=True)
    safe = x.masked_fill(closed, 0.0)
    if score == "softmax":
        s = torch.softmax(safe, 1).masked_fill(closed, 0.0)
        slope = torch.ones_like(s)
    else:
        s = torch.sigmoid(x)
        slope = torch.sigmoid(-x)
    picked = s.gather(1, chosen)
    total = picked.sum(1, keepdim=True)
    share = torch.where(total == 0, torch.zeros_like(picked), picked / total)
    flat = chosen.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    out = dict(weights=share if normalize else picked, experts=chosen, batch_sizes=torch.bincount(flat, minlength=e),
               order=order, row_index=order // k, mass=s.sum(0))
    if weights_grad is not None or mass_grad is not None:
        g = weights_grad.double() if weights_grad is not None else torch.zeros(t, k, dtype=torch.float64)
        u = mass_grad.double().expand(t, e) if mass_grad is not None else torch.zeros_like(x)
        if not normalize:
            u = u.scatter_add(1, chosen, g)
        grad = s * (u - (u * s).sum(1, keepdim=True)) if score == "softmax" else s * slope * u
        if normalize:
            at = share * (g - (g * share).sum(1, keepdim=True)) * slope.gather(1, chosen)
            grad = grad.scatter_add(1, chosen, at)
        out["grad"] = grad
        out["grad_scale"] = u.abs().amax(1, keepdim=True) + g.abs().amax(1, keepdim=True)
    return out


def _check_route(ops, logits, k, score="softmax", normalize=True, with_mass=True, what=""):
    got = ops.route(logits.cuda(), k, score=score, normalize=normalize, with_mass=with_mass)
    want = _route_reference(logits, k, score, normalize)
    for name in ("experts", "batch_sizes", "order", "row_index"):
        assert torch.equal(getattr(got, name).cpu().long(), want[name]), (what, name)
    assert got.experts.dtype == got.order.dtype == got.row_index.dtype == torch.int32 and got.batch_sizes.dtype == torch.int64
    assert got.weights.dtype == torch.float32
    _close(got.weights, want["weights"], 1e-5, 1e-30, f"{what} weights")
    if with_mass:
        _close(got.mass, want["mass"], 1e-5, 1e-30, f"{what} mass")
    else:
        assert got.mass is None
    return got, want


# one token and none, sizes around a lane's, a group's and a workgroup's share, most experts and largest top_k
ROUTE_SHAPES = [(0, 8, 2), (1, 1, 1), (1, 64, 6), (3, 5, 5), (7, 37, 3), (33, 64, 8), (64, 65, 32), (65, 128, 17), (100, 129, 1),
                (513, 256, 8), (130, 257, 20), (77, 512, 10), (200, 1000, 32), (64, 1024, 32), (3000, 17, 4), (20001, 8, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", ROUTE_SHAPES)
def test_route_matches_its_definition(ops, shape, dtype):
    t, e, k = shape
    g = torch.Generator().manual_seed(t * 7 + e)
    logits = (torch.randn(t, e, generator=g) * 2).to(dtype)   # (two-byte logits: many equal ones)
    for score in ("softmax", "sigmoid"):
        for normalize in (True, False):
            _announce("route", shape, dtype, score, normalize)
            _check_route(ops, logits, k, score, normalize, what=f"{shape} {score} {normalize}")
    _check_route(ops, logits, k, with_mass=False, what=f"{shape}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("experts", [12, 200, 700])
def test_route_odd_values(ops, tokens, experts, dtype):
    """Closed experts, tokens that none is open to, equal logits, -0 and +0, infinities, NaN, the type's lowest value."""
    g = torch.Generator().manual_seed(experts)
    logits = torch.randn(tokens, experts, generator=g).to(dtype)
    logits[torch.rand(tokens, experts, generator=g) < 0.3] = -INF
    logits[0] = -INF
    logits[1] = -INF
    logits[1, 5] = 3.0                       # one open expert, fewer than are chosen
    logits[2] = 1.25                         # all equal
    logits[3] = 0.0
    logits[3, ::2] = -0.0                    # equal as well
    logits[4] = torch.finfo(dtype).min       # a mask of the lowest value instead of -inf
    logits[4, 7] = 2.0
    logits[5, 3] = float("nan")
    logits[6, 9] = INF
    logits[7] = torch.finfo(dtype).min
    for score in ("softmax", "sigmoid"):
        for normalize in (True, False):
            _announce("route odd values", tokens, experts, dtype, score, normalize)
            got = ops.route(logits.cuda(), 4, score=score, normalize=normalize, with_mass=True)
            want = _route_reference(logits, 4, score, normalize)
            for name in ("experts", "batch_sizes", "order", "row_index"):
                assert torch.equal(getattr(got, name).cpu().long(), want[name]), name
            # (row 7 under a normalized sigmoid: scores too small for 64 bits too, all alike)
            if score == "sigmoid" and normalize:
                want["weights"][7] = 0.25
            _close(got.weights, want["weights"], 1e-5, 1e-30, "weights")
            assert (got.weights[0] == 0).all()
            finite = torch.cat([logits[:5], logits[7:]])
            _check_route(ops, finite[:5], 4, score, normalize, what="finite rows")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts", [9, 100, 256, 600])
def test_route_nan_of_either_sign(ops, experts, dtype):
    """NaN of any sign and payload counts as one value above all others, ties by the lower index; other tokens do not notice."""
    g = torch.Generator().manual_seed(experts)
    logits = torch.randn(70, experts, generator=g).to(dtype)
    whole, least = (torch.int32, 0x80000000 - 2 ** 32) if dtype == torch.float32 else (torch.int16, 0x8000 - 2 ** 16)
    quiet = int(torch.tensor([float("nan")], dtype=dtype).view(whole)[0])
    bits = logits.view(whole)
    bits[3, 2] = quiet | least           # negative
    bits[3, 7] = quiet                   # positive
    bits[3, 8] = quiet | 1
    bits[10, experts - 1] = quiet | least | 1
    bits[11, :] = quiet | least
    logits[12, 4] = INF
    bits[12, 6] = quiet | least
    _announce("route NaN", experts, dtype)
    got = ops.route(logits.cuda(), 5, with_mass=False)
    want = _route_reference(logits, 5, "softmax", True)
    for name in ("experts", "batch_sizes", "order", "row_index"):
        assert torch.equal(getattr(got, name).cpu().long(), want[name]), name
    rest = torch.tensor([t for t in range(70) if t not in (3, 10, 11, 12)])
    _close(got.weights.cpu()[rest], want["weights"][rest], 1e-5, 1e-30, "weights")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 8, 2), (5, 64, 6), (70, 37, 3), (257, 256, 8), (90, 500, 32), (33, 1024, 5), (4099, 16, 4)])
def test_route_gradient_matches_its_formula(ops, shape, dtype):
    t, e, k = shape
    g = torch.Generator().manual_seed(e)
    logits = (torch.randn(t, e, generator=g) * 1.5).to(dtype)
    logits[0, : e // 2] = -INF
    if t > 2:
        logits[2] = -INF
    weights_grad, mass_grad = torch.randn(t, k, generator=g), torch.randn(e, generator=g)
    for score in ("softmax", "sigmoid"):
        for normalize in (True, False):
            for with_weights, with_mass in ((True, True), (True, False), (False, True)):
                _announce("route gradient", shape, dtype, score, normalize, with_weights, with_mass)
                x = logits.cuda().requires_grad_(True)
                r = ops.route(x, k, score=score, normalize=normalize, with_mass=with_mass)
                loss = 0.0
                if with_weights:
                    loss = loss + (r.weights * weights_grad.cuda()).sum()
                if with_mass:
                    loss = loss + (r.mass * mass_grad.cuda()).sum()
                loss.backward()
                want = _route_reference(logits, k, score, normalize, weights_grad if with_weights else None,
                                        mass_grad if with_mass else None)
                assert x.grad.dtype == dtype
                rtol, least = ROUNDING[dtype]
                _close(x.grad, want["grad"], 1e-5 + rtol, 1e-5 * want["grad_scale"] + least, f"{score} {normalize}")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [True, False])
def test_route_gradient_matches_differences(ops, score, normalize):
    """Central differences of the outputs, step h = 2^-6: the quotient is off by h^2 / 6 of a third derivative (at most 2 for
    these functions of one logit, times the gradients' sizes, 5e-5 each) and by two fp32 errors of the loss over 2 h."""
    g = torch.Generator().manual_seed(11)
    t, e, k, h = 4, 10, 3, 2.0 ** -6
    # well apart, so that no step changes which experts are chosen
    logits = torch.stack([torch.randperm(e, generator=g).float() * 0.25 for _ in range(t)])
    weights_grad, mass_grad = torch.randn(t, k, generator=g), torch.randn(e, generator=g)
    x = logits.cuda().requires_grad_(True)
    r = ops.route(x, k, score=score, normalize=normalize, with_mass=True)
    got, = torch.autograd.grad((r.weights, r.mass), x, (weights_grad.cuda(), mass_grad.cuda()))

    def loss(z):
        q = ops.route(z.cuda(), k, score=score, normalize=normalize, with_mass=True)
        return float((q.weights.cpu().double() * weights_grad).sum() + (q.mass.cpu().double() * mass_grad).sum())

    scale = float(weights_grad.abs().sum() + mass_grad.abs().sum())
    for i in range(t):
        for j in range(e):
            up, down = logits.clone(), logits.clone()
            up[i, j] += h
            down[i, j] -= h
            want = (loss(up) - loss(down)) / (2 * h)
            assert abs(float(got[i, j]) - want) <= scale * (h * h / 3 + 4 * 2.0 ** -22 / h), (i, j)


def test_route_refuses_forward_mode(ops):
    """A tangent is an error, not a result without one, with and without gradient mode; gradients in reverse go on as before."""
    x = torch.randn(6, 8, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        for leaf in (x, x.clone().requires_grad_(True)):
            dual = torch.autograd.forward_ad.make_dual(leaf, torch.randn_like(x))
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.route(dual, 2)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                ops.route(dual, 2, with_mass=True)
        ops.route(x, 2)


@pytest.mark.parametrize("parts", ["weights", "mass", "both"])
@pytest.mark.parametrize("normalize", [True, False])
def test_route_refuses_a_second_derivative(ops, normalize, parts):
    """With create_graph the gradient is the same, other terms of a loss have their second derivative, and one through the router's is an error."""
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(6, 6, device="cuda", generator=g).requires_grad_(True)
    x, at = torch.randn(5, 6, device="cuda", generator=g), torch.randn(5, 2, device="cuda", generator=g)

    def loss():
        r = ops.route(x @ w, 2, normalize=normalize, with_mass=True)
        weights, mass = (r.weights * at).sum(), r.mass.square().sum()
        return w.pow(3).sum() + {"weights": weights, "mass": mass, "both": weights + mass}[parts]

    want, = torch.autograd.grad(loss(), w)
    got, = torch.autograd.grad(loss(), w, create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(got.sum(), w)
    both = loss()
    cubes, = torch.autograd.grad(w.pow(3).sum() + 0 * both.detach(), w, create_graph=True)
    second, = torch.autograd.grad(cubes.sum(), w)
    assert torch.equal(second, 6 * w.detach())


def test_route_on_other_streams_and_in_a_graph(ops):
    """The same bits on another stream, on every call and in every replay of a captured one, with eager work in between."""
    logits = torch.randn(5000, 96, device="cuda").bfloat16()
    small = torch.randn(9, 96, device="cuda")
    want = [ops.route(logits, 6, with_mass=True), ops.route(small, 6, with_mass=True)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [ops.route(logits, 6, with_mass=True), ops.route(small, 6, with_mass=True)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [ops.route(logits, 6, with_mass=True), ops.route(small, 6, with_mass=True)]
    for _ in range(3):
        for r in captured:
            for part in r:
                part.zero_()
        graph.replay()
        eager = [ops.route(logits, 6, with_mass=True), ops.route(small, 6, with_mass=True)]
        torch.cuda.synchronize()
        for one in (again, captured, eager):
            for r, w in zip(one, want):
                for a, b in zip(r, w):
                    assert torch.equal(a, b)


def test_route_past_32_bits(ops):
    """More than 2^32 bytes and 2^31 elements of logits: the last tokens as in a call of their own, the order as a stable sort gives it."""
    tokens, experts, k = 8_500_000, 256, 4
    logits = torch.empty(tokens, experts, dtype=torch.bfloat16, device="cuda").normal_()
    assert logits.numel() > 2 ** 31
    _announce("route past 32 bits")
    got = ops.route(logits, k)
    alone = ops.route(logits[-1000:].contiguous(), k)
    assert torch.equal(got.weights[-1000:], alone.weights) and torch.equal(got.experts[-1000:], alone.experts)
    flat = got.experts.view(-1)
    order = torch.sort(flat, stable=True).indices.int()
    assert torch.equal(got.order, order) and torch.equal(got.row_index, order // k)
    assert torch.equal(got.batch_sizes, torch.bincount(flat, minlength=experts))
    del got, order, flat
    logits.requires_grad_(True)
    r = ops.route(logits, k)
    grad = torch.randn(tokens, k, device="cuda")
    full, = torch.autograd.grad((r.weights,), (logits,), (grad,))
    last = logits.detach()[-1000:].contiguous().requires_grad_(True)
    one, = torch.autograd.grad((ops.route(last, k).weights,), (last,), (grad[-1000:].contiguous(),))
    assert torch.equal(full[-1000:], one)


def test_route_refuses(ops):
    x = torch.zeros(4, 8, device="cuda")
    bad = [
        (lambda: ops.route(x.cpu(), 2), "GPU"), (lambda: ops.route(x[0], 2), "2-d"), (lambda: ops.route(x.double(), 2), "float32"),
        (lambda: ops.route(x, 0), "top_k"), (lambda: ops.route(x, 9), "top_k"), (lambda: ops.route(x.t(), 2), "contiguous"),
        (lambda: ops.route(x, 2, score="tanh"), "score"), (lambda: ops.route(torch.zeros(2, 1025, device="cuda"), 2), "at most"),
        (lambda: ops.route(torch.zeros(2, 64, device="cuda"), 33), "at most"),
    ]
    for call, message in bad:
        with pytest.raises(RuntimeError, match=message):
            call()


# ------------------------------------------------------------------ gated expert layer for a few tokens

HANDED_ON = {torch.bfloat16: (2.0 ** -16, 0.0), torch.float16: (2.0 ** -21, 2.0 ** -24)}


def _moe_reference(x, w13, w2, experts, weights, trans_b):
    """The layer in 64 bits, and by how much each element may be off before it is rounded."""
    t, hidden = x.shape
    num, ffn = w13.shape[0], w2.shape[2 if trans_b else 1]
    unit, least = HANDED_ON[x.dtype]
    out, off = torch.zeros(t, hidden, dtype=torch.float64), torch.zeros(t, hidden, dtype=torch.float64)
    for i in range(t):
        for j in range(experts.shape[1]):
            e, w = int(experts[i, j]), float(weights[i, j])
            if not 0 <= e < num:
                continue
            first, second = w13[e].double(), w2[e].double()
            if trans_b:
                first, second = first.t(), second.t()
            both = x[i].double() @ first
            err = (x[i].double().abs() @ first.abs()) * (2 * hidden * 2.0 ** -24)
            gate, up = both[:ffn], both[ffn:]
            s = torch.sigmoid(gate)
            h = gate * s * up
            # (the derivative of silu is at most 1.1)
            h_off = 1.1 * err[:ffn] * (up.abs() + err[ffn:]) + (gate * s).abs() * err[ffn:] + h.abs() * (unit + 2.0 ** -20) + least
            out[i] += w * (h @ second)
            off[i] += abs(w) * ((h_off @ second.abs()) + (h.abs() @ second.abs()) * ((2 * ffn + 64) * 2.0 ** -24))
    return out, off


def _moe_case(t, num, k, hidden, ffn, dtype, trans_b, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, hidden, generator=g).to(dtype)
    w13 = (torch.randn(num, hidden, 2 * ffn, generator=g) * hidden ** -0.5 * scale).to(dtype)
    w2 = (torch.randn(num, ffn, hidden, generator=g) * ffn ** -0.5).to(dtype)
    if trans_b:
        w13, w2 = w13.transpose(1, 2).contiguous(), w2.transpose(1, 2).contiguous()
    experts = torch.stack([torch.randperm(num, generator=g)[:k] for _ in range(t)]).to(torch.int32) if t else torch.zeros(0, k, dtype=torch.int32)
    weights = torch.rand(t, k, generator=g)
    return x, w13, w2, experts, weights


def _check_moe(ops, case, trans_b, what):
    x, w13, w2, experts, weights = case
    got = ops.moe_few_tokens(*(v.cuda() for v in case), trans_b=trans_b)
    assert got.dtype == x.dtype
    want, off = _moe_reference(x, w13, w2, experts, weights, trans_b)
    rtol, least = ROUNDING[x.dtype]
    _close(got, want, rtol, off * (1 + rtol) + least, what)
    return got


# tokens, experts, top_k, hidden, ffn: widths below a lane's, a tile's and a strip's share, depths that end inside a step and before one
MOE_SHAPES = [(1, 1, 1, 1, 1), (1, 4, 2, 8, 8), (1, 8, 2, 256, 512), (2, 3, 3, 5, 7), (3, 5, 2, 33, 9), (5, 8, 2, 100, 129),
              (1, 8, 8, 64, 1000), (7, 4, 1, 1021, 67), (16, 6, 3, 72, 200), (17, 2, 2, 130, 96), (33, 3, 2, 257, 65), (64, 4, 3, 95, 71),
              (64, 130, 8, 40, 33), (64, 1000, 1, 16, 24), (1, 2, 2, 2000, 2049), (4, 8, 2, 129, 1500), (0, 4, 2, 64, 64)]


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", MOE_SHAPES)
def test_moe_few_tokens_matches_its_definition(ops, shape, dtype, trans_b):
    _announce("moe few tokens", shape, dtype, trans_b)
    _check_moe(ops, _moe_case(*shape, dtype, trans_b, seed=sum(shape)), trans_b, f"{shape}")


@pytest.mark.parametrize("trans_b", [False, True])
def test_moe_few_tokens_odd_routing(ops, trans_b):
    """All tokens at one expert, an expert named twice by a token, numbers that name no expert, tokens without any."""
    for t in (3, 20, 64):
        case = list(_moe_case(t, 6, 4, 96, 136, torch.bfloat16, trans_b, seed=t))
        for name, experts in [
            ("one expert", torch.full((t, 4), 2)),
            ("none", torch.full((t, 4), -1)),
            ("past the end", torch.full((t, 4), 6)),
            ("largest", torch.full((t, 4), 2 ** 31 - 1)),
            ("some", torch.randint(-2, 8, (t, 4), generator=torch.Generator().manual_seed(t))),
        ]:
            _announce("moe odd routing", t, name, trans_b)
            case[3] = experts.to(torch.int32)
            got = _check_moe(ops, case, trans_b, name)
            if name in ("none", "past the end", "largest"):
                assert (got == 0).all()


@pytest.mark.parametrize("trans_b", [False, True])
def test_moe_few_tokens_reads_named_experts_only(ops, trans_b):
    """NaN in every expert that is not named, and behind every tensor, reaches no output."""
    x, w13, w2, experts, weights = _moe_case(5, 7, 2, 51, 43, torch.float16, trans_b, seed=3)
    named = set(experts.flatten().tolist())
    for e in range(7):
        if e not in named:
            w13[e], w2[e] = float("nan"), float("nan")

    def framed(t):   # between NaN, off the 16-byte boundary
        flat = torch.full((t.numel() + 67,), float("nan"), dtype=t.dtype, device="cuda")
        flat[33:33 + t.numel()] = t.flatten().cuda()
        return flat[33:33 + t.numel()].view(t.shape)

    got = ops.moe_few_tokens(framed(x), framed(w13), framed(w2), experts.cuda(), framed(weights), trans_b=trans_b)
    want, off = _moe_reference(x, w13, w2, experts, weights, trans_b)
    rtol, least = ROUNDING[x.dtype]
    _close(got, want, rtol, off * (1 + rtol) + least, "framed")


def test_moe_few_tokens_large_values(ops):
    """Gates far out on both sides: silu underflows to 0 on one and is the gate itself on the other; products past the
    type's range become infinities, not NaN."""
    x = torch.tensor([[1.0], [-1.0]], dtype=torch.bfloat16)
    w13 = torch.tensor([[[200.0, 3.0]], [[2.0 ** 100, 2.0 ** 60]]], dtype=torch.bfloat16)
    w2 = torch.ones(2, 1, 1, dtype=torch.bfloat16)
    experts, weights = torch.tensor([[0], [0]], dtype=torch.int32), torch.ones(2, 1)
    got = ops.moe_few_tokens(*(v.cuda() for v in (x, w13, w2, experts, weights))).cpu()
    assert float(got[0]) == 600.0 and float(got[1]) == 0.0
    got = ops.moe_few_tokens(x[:1].cuda(), w13.cuda(), w2.cuda(), experts[:1].cuda() + 1, weights[:1].cuda()).cpu()
    assert float(got) == INF


def _moe_reference_of_range(x, w13, w2, experts, weights, trans_b):
    """The layer in 64 bits, and by how much each element may be off where what is handed on keeps its bits whatever its size: 2^-16 of itself
    in bfloat16; in float16 2^-21 of itself and 2^-37 of the row's largest: its two halves are scaled by blocks, the largest to 2^14 at least (the
    lower one is off by up to 2^-25 there), and then to the row's largest (each off by the same once more, at most half of it again where the
    power of two is applied in two steps: 4 x 2^-25 of 2^14)."""
    t, hidden = x.shape
    ffn = w2.shape[2 if trans_b else 1]
    unit, of_largest = (2.0 ** -16, 0.0) if x.dtype == torch.bfloat16 else (2.0 ** -21, 2.0 ** -37)
    out, off = torch.zeros(t, hidden, dtype=torch.float64), torch.zeros(t, hidden, dtype=torch.float64)
    for i in range(t):
        for j in range(experts.shape[1]):
            e, w = int(experts[i, j]), float(weights[i, j])
            first, second = w13[e].double(), w2[e].double()
            if trans_b:
                first, second = first.t(), second.t()
            both = x[i].double() @ first
            err = (x[i].double().abs() @ first.abs()) * (2 * hidden * 2.0 ** -24)
            gate, up = both[:ffn], both[ffn:]
            s = torch.sigmoid(gate)
            h = gate * s * up
            h_off = 1.1 * err[:ffn] * (up.abs() + err[ffn:]) + (gate * s).abs() * err[ffn:] + h.abs() * (unit + 2.0 ** -20)
            h_off += h.abs().max() * of_largest
            out[i] += w * (h @ second)
            off[i] += abs(w) * ((h_off @ second.abs()) + (h.abs() @ second.abs()) * ((2 * ffn + 64) * 2.0 ** -24))
    return out, off


# one block of columns, parts of blocks, pieces of the depth, odd sizes, more rows than are taken at a time, rows that workgroups share
RANGE_SHAPES = [(1, 4, 2, 64, 24), (5, 8, 2, 100, 129), (2, 3, 2, 72, 2100), (33, 3, 2, 57, 65), (64, 4, 3, 95, 271), (64, 130, 8, 40, 33)]


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["large", "small", "mixed"])
@pytest.mark.parametrize("shape", RANGE_SHAPES)
def test_moe_few_tokens_activations_of_any_size(ops, shape, kind, dtype, trans_b):
    """Activations far past float16's largest number, far below its least, and of sizes 2^24 apart in one row, each made up for by the second
    weights: the result is an ordinary number, and has to be as exact as one."""
    t, num, k, hidden, ffn = shape
    x, w13, w2, experts, weights = _moe_case(t, num, k, hidden, ffn, torch.float32, False, seed=sum(shape))
    if kind == "large":     # gates and ups of 2^10 or so
        w13, w2 = w13 * 2.0 ** 10, w2 * 2.0 ** -14
    elif kind == "small":   # ... of 2^-12
        w13, w2 = w13 * 2.0 ** -12, w2 * 2.0 ** 12
    else:
        size = torch.randint(-6, 7, (ffn,), generator=torch.Generator().manual_seed(ffn)).double()
        w13 = (w13 * torch.exp2(torch.cat([size, size]))).float()
        w2 = (w2 * torch.exp2(-2 * size)[:, None]).float()
    if trans_b:
        w13, w2 = w13.transpose(1, 2), w2.transpose(1, 2)
    case = [v.to(dtype).contiguous() for v in (x, w13, w2)] + [experts, weights]
    _announce("moe activations of any size", shape, kind, dtype, trans_b)
    got = ops.moe_few_tokens(*(v.cuda() for v in case), trans_b=trans_b)
    want, off = _moe_reference_of_range(*case, trans_b)
    rtol, least = ROUNDING[dtype]
    assert float(want.abs().max()) < 3e4
    _close(got, want, rtol, off * (1 + rtol) + least, f"{shape} {kind}")


@pytest.mark.parametrize("trans_b", [False, True])
def test_moe_few_tokens_float16_past_its_largest_activation(ops, trans_b):
    """gate = up = 300: 90000 between the two products.  Against a small weight, one of zero, and one of the other sign."""
    x = torch.tensor([[1.0, 0.0], [0.0, 1.0]], dtype=torch.float16)
    w13 = torch.tensor([[[300.0, 300.0, 300.0, 300.0], [300.0, 300.0, -300.0, 300.0]]], dtype=torch.float16)   # gates | ups
    w2 = torch.tensor([[[2.0 ** -10, 0.0], [2.0 ** -11, 0.0]]], dtype=torch.float16)
    if trans_b:
        w13, w2 = w13.transpose(1, 2).contiguous(), w2.transpose(1, 2).contiguous()
    experts, weights = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1)
    got = ops.moe_few_tokens(*(v.cuda() for v in (x, w13, w2, experts, weights)), trans_b=trans_b).cpu().double()
    want = torch.tensor([[90000 * (2.0 ** -10 + 2.0 ** -11), 0.0], [-90000 * 2.0 ** -10 + 90000 * 2.0 ** -11, 0.0]], dtype=torch.float64)
    _close(got, want, 2.0 ** -11 + 2.0 ** -20, 2.0 ** -25, "past the largest")


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_few_tokens_infinite_weights(ops, dtype, trans_b):
    """An infinite weight of the second product gives an infinity of its sign, as its formula does, whatever is left of the activation in its lower
    half: nothing (600, 3), or something of either sign (silu(1) = 0.7310586, silu(2) = 1.7615942); other columns do not notice."""
    for gate, up in ((200.0, 3.0), (1.0, 1.0), (2.0, 1.0), (2.0, -1.0)):
        x = torch.ones(3, 1, dtype=dtype)
        w13 = torch.tensor([[[gate, up]]], dtype=dtype)
        w2 = torch.tensor([[[1.0, INF, -INF]]], dtype=dtype)
        x, w13, w2 = torch.cat([x, x, x], 1), torch.cat([w13, 0 * w13, 0 * w13], 1), w2   # (hidden is 3)
        if trans_b:
            w13, w2 = w13.transpose(1, 2).contiguous(), w2.transpose(1, 2).contiguous()
        experts, weights = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, 1)
        _announce("moe infinite weights", gate, up, dtype, trans_b)
        got = ops.moe_few_tokens(*(v.cuda() for v in (x, w13, w2, experts, weights)), trans_b=trans_b).cpu().double()
        h = gate / (1 + math.exp(-gate)) * up
        want = torch.tensor([[h, math.copysign(INF, h), math.copysign(INF, -h)]] * 3, dtype=torch.float64)
        rtol, least = ROUNDING[dtype]
        _close(got, want, rtol + 2.0 ** -15, least, "infinite weights")


@pytest.mark.parametrize("trans_b", [False, True])
def test_moe_few_tokens_bfloat16_largest_activation(ops, trans_b):
    """An activation between the largest bfloat16 and the largest float, which rounds up to an infinity: (2 - 2^-9) 2^127."""
    x = torch.ones(1, 2, dtype=torch.bfloat16)
    w13 = torch.tensor([[[(2 - 2.0 ** -7) * 2.0 ** 64, 2.0 ** 63], [0.75 * 2.0 ** 57, 0.0]]], dtype=torch.float64)
    w2 = torch.tensor([[[2.0 ** -100, 0.0]]], dtype=torch.bfloat16)
    w13 = w13.bfloat16()
    if trans_b:
        w13, w2 = w13.transpose(1, 2).contiguous(), w2.transpose(1, 2).contiguous()
    got = ops.moe_few_tokens(x.cuda(), w13.cuda(), w2.cuda(), torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.ones(1, 1).cuda(),
                             trans_b=trans_b).cpu().double()
    want = torch.tensor([[(2 - 2.0 ** -9) * 2.0 ** 27, 0.0]], dtype=torch.float64)
    _close(got, want, 2.0 ** -8 + 2.0 ** -15, 0.0, "largest")


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_few_tokens_infinite_activations(ops, dtype, trans_b):
    """An infinite activation gives infinities, NaN against a weight of zero, as its formula does; other tokens do not notice."""
    x, w13, w2, experts, weights = _moe_case(5, 3, 2, 40, 100, dtype, trans_b, seed=8)
    x[3] = 0
    x[3, 0] = INF
    for e in range(3):
        first, second = (w13[e].t(), w2[e].t()) if trans_b else (w13[e], w2[e])   # (views)
        first[0] = first[0].abs() + 0.125           # every gate and every up of token 3 infinite
        second[:, 5], second[:, 6], second[:, 7] = second[:, 5].abs() + 0.125, -second[:, 6].abs() - 0.125, 0.0
    _announce("moe infinite activations", dtype, trans_b)
    got = ops.moe_few_tokens(*(v.cuda() for v in (x, w13, w2, experts, weights)), trans_b=trans_b).cpu()
    x[3, 0] = 0
    want, off = _moe_reference(x, w13, w2, experts, weights, trans_b)
    rtol, least = ROUNDING[dtype]
    others = torch.tensor([0, 1, 2, 4])
    _close(got[others], want[others], rtol, (off * (1 + rtol) + least)[others], "other tokens")
    assert got[3, 5] == INF and got[3, 6] == -INF and torch.isnan(got[3, 7])
    assert not torch.isfinite(got[3]).any()


def test_moe_few_tokens_full_size_on_the_device(ops):
    """A large layer against 32-bit products on the device, every element (both sum in fp32: 4096 products of either sign,
    far within a rounding of the type)."""
    g = torch.Generator(device="cuda").manual_seed(5)
    for trans_b, t in ((False, 1), (True, 1), (False, 40), (True, 40)):
        x = torch.randn(t, 4096, device="cuda", generator=g).bfloat16()
        w13 = (torch.randn(8, 4096, 2 * 7168, device="cuda", generator=g) * 0.0156).bfloat16()
        w2 = (torch.randn(8, 7168, 4096, device="cuda", generator=g) * 0.0118).bfloat16()
        r = ops.route(torch.randn(t, 8, device="cuda", generator=g), 2)
        both = torch.matmul(x.float(), w13.float())   # (experts, tokens, 2 ffn)
        gate, up = both.chunk(2, dim=2)
        y = torch.matmul(torch.nn.functional.silu(gate) * up, w2.float())
        want = (y[r.experts.long(), torch.arange(t, device="cuda")[:, None]] * r.weights[..., None]).sum(1)
        if trans_b:
            w13, w2 = w13.transpose(1, 2).contiguous(), w2.transpose(1, 2).contiguous()
        _announce("moe full size", trans_b, t)
        got = ops.moe_few_tokens(x, w13, w2, r.experts, r.weights, trans_b=trans_b)
        off = (got.float() - want).abs() - (2.0 ** -8 * want.abs() + 1e-4 * want.abs().max())
        assert float(off.max()) <= 0.0


def test_moe_few_tokens_same_bits_on_streams_and_in_graphs(ops):
    cases = [[v.cuda() for v in _moe_case(t, 8, 2, 512, 4096, torch.bfloat16, True, seed=t)] for t in (1, 24)]
    want = [ops.moe_few_tokens(*c, trans_b=True) for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [ops.moe_few_tokens(*c, trans_b=True) for c in cases]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [ops.moe_few_tokens(*c, trans_b=True) for c in cases]
    for _ in range(4):
        for out in captured:
            out.zero_()
        graph.replay()
        eager = [ops.moe_few_tokens(*c, trans_b=True) for c in cases]
        torch.cuda.synchronize()
        for one in (again, captured, eager):
            for a, b in zip(one, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
# more than 64 slots (listed in any order), an expert's rows shared among workgroups in the second product, in the first one too (listed in their own)
@pytest.mark.parametrize("shape", [(24, 8, 4, 512, 1000), (64, 130, 8, 96, 200), (64, 4, 4, 1024, 2048), (64, 4, 4, 256, 512), (64, 3, 3, 129, 333)])
def test_moe_few_tokens_same_bits_of_many_slots(ops, shape, dtype, trans_b):
    """On every call, on another stream and in every replay, whatever the scratch held before."""
    case = [v.cuda() for v in _moe_case(*shape, dtype, trans_b, seed=sum(shape))]
    _announce("moe same bits", shape, dtype, trans_b)

    def poisoned():
        junk = [torch.full((n,), float("nan"), device="cuda") for n in (1 << 12, 1 << 16, 1 << 20, 1 << 21)]
        del junk

    want = ops.moe_few_tokens(*case, trans_b=trans_b)
    for _ in range(8):
        poisoned()
        assert torch.equal(ops.moe_few_tokens(*case, trans_b=trans_b), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.moe_few_tokens(*case, trans_b=trans_b)
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.moe_few_tokens(*case, trans_b=trans_b)
    for _ in range(4):
        captured.zero_()
        graph.replay()
        eager = ops.moe_few_tokens(*case, trans_b=trans_b)
        torch.cuda.synchronize()
        assert torch.equal(captured, want) and torch.equal(eager, want)


def test_moe_few_tokens_refuses(ops):
    x, w13, w2, experts, weights = (v.cuda() for v in _moe_case(2, 4, 2, 32, 48, torch.bfloat16, False, seed=1))

    def call(**kw):
        a = dict(x=x, w13=w13, w2=w2, experts=experts, weights=weights)
        a.update(kw)
        return ops.moe_few_tokens(**a)

    bad = [(dict(x=x.cpu()), "same GPU"), (dict(x=x[0]), "2-d"), (dict(x=x.float()), "bfloat16"), (dict(w13=w13[0]), "3-d"),
           (dict(w13=w13.half()), "element type"), (dict(w2=w2[:3]), "w2"), (dict(w2=w2[:, :47].contiguous()), "w2"),
           (dict(w13=w13[:, :, :95].contiguous()), "even"), (dict(w13=w13[:, :31].contiguous()), "contraction"),
           (dict(experts=experts.long()), "int32"), (dict(experts=experts[:1]), "int32"), (dict(weights=weights.half()), "float32"),
           (dict(weights=weights[:, :1]), "float32"), (dict(w13=w13.transpose(0, 1).contiguous().transpose(0, 1)), "contiguous"),
           (dict(x=x.repeat(40, 1), experts=experts.repeat(40, 1), weights=weights.repeat(40, 1)), "at most 64"),
           (dict(x=x.clone().requires_grad_(True)), "no gradient"), (dict(w2=w2.clone().requires_grad_(True)), "no gradient")]
    for kw, message in bad:
        with pytest.raises(RuntimeError, match=message):
            call(**kw)
    with torch.no_grad():   # (a model's parameters, in serving)
        call(w2=w2.clone().requires_grad_(True))


def test_moe_few_tokens_refuses_forward_mode(ops):
    case = [v.cuda() for v in _moe_case(2, 4, 2, 32, 48, torch.bfloat16, False, seed=1)]
    with torch.autograd.forward_ad.dual_level():
        for i in (0, 1, 2, 4):
            dual = list(case)
            dual[i] = torch.autograd.forward_ad.make_dual(case[i], torch.ones_like(case[i]))
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                ops.moe_few_tokens(*dual)


# ------------------------------------------------------------------ low-rank adapters

def _lora_reference(x, a, b, adapters, base, scales):
    """The adapters in 64 bits, and by how much each element may be off before it is rounded."""
    rows, hin = x.shape
    num, r, hout = a.shape[0], a.shape[1], b.shape[1]
    unit, least = HANDED_ON[x.dtype]
    out = base.double().clone() if base is not None else torch.zeros(rows, hout, dtype=torch.float64)
    off = torch.zeros(rows, hout, dtype=torch.float64)
    for n in range(num):
        at = torch.nonzero(adapters == n).squeeze(1)
        if at.numel() == 0:
            continue
        xs, an, bn = x[at].double(), a[n].double(), b[n].double()
        s = float(scales[n]) if scales is not None else 1.0
        v = xs @ an.t()
        # (float16's v is scaled to below 1, so that its lower half stays in range: relative to the row's largest)
        v_off = (xs.abs() @ an.abs().t()) * (2 * hin * 2.0 ** -24) + v.abs() * unit + v.abs().amax(1, keepdim=True) * least
        out[at] += s * (v @ bn.t())
        off[at] += abs(s) * (v_off @ bn.abs().t() + (v.abs() @ bn.abs().t()) * ((4 * r + 8) * 2.0 ** -24))
        off[at] += out[at].abs() * 2.0 ** -23
    return out, off


def _lora_case(rows, num, r, hin, hout, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hin, generator=g).to(dtype)
    a = (torch.randn(num, r, hin, generator=g) * hin ** -0.5).to(dtype)
    b = (torch.randn(num, hout, r, generator=g) * r ** -0.5).to(dtype)
    base = torch.randn(rows, hout, generator=g).to(dtype)
    scales = torch.rand(num, generator=g) * 2 - 1
    adapters = torch.randint(-1, num, (rows,), generator=g).to(torch.int32)
    return x, a, b, adapters, base, scales


def _check_lora(ops, case, what):
    x, a, b, adapters, base, scales = case
    cuda = [v.cuda() if v is not None else None for v in case]
    got = ops.lora(cuda[0], cuda[1], cuda[2], cuda[3], base=cuda[4], scales=cuda[5])
    assert got.dtype == x.dtype
    want, off = _lora_reference(*case)
    rtol, least = ROUNDING[x.dtype]
    _close(got, want, rtol, off * (1 + rtol) + least, what)
    untouched = ~((adapters >= 0) & (adapters < a.shape[0]))
    if base is not None:
        assert torch.equal(got.cpu()[untouched], base[untouched]), what
    else:
        assert (got.cpu()[untouched] == 0).all(), what
    return got


# rows, adapters, rank, hidden_in, hidden_out: parts of a window, of a tile, of a strip, of a step; several of each
LORA_SHAPES = [(0, 2, 8, 16, 16), (1, 1, 1, 1, 1), (1, 3, 16, 64, 256), (2, 2, 3, 5, 7), (5, 40, 8, 130, 300), (17, 2, 11, 257, 67),
               (64, 64, 16, 512, 200), (65, 1, 33, 100, 1030), (100, 5, 64, 1021, 129), (130, 3, 100, 72, 511), (200, 7, 256, 65, 90),
               (70, 300, 4, 640, 64), (1, 2, 65, 4096, 515), (400, 2, 16, 3000, 48), (1025, 9, 17, 63, 33)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", LORA_SHAPES)
def test_lora_matches_its_definition(ops, shape, dtype):
    _announce("lora", shape, dtype)
    _check_lora(ops, _lora_case(*shape, dtype, seed=sum(shape)), f"{shape}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lora_rows_in_any_order(ops, dtype):
    """Prompts (runs of one adapter), one adapter for all, none for any, every row another, numbers that name none."""
    rows, num = 150, 150
    x, a, b, _, base, scales = _lora_case(rows, num, 20, 88, 140, dtype, seed=9)
    g = torch.Generator().manual_seed(1)
    for name, adapters in [
        ("runs", torch.arange(rows) // 37), ("one", torch.full((rows,), 149)), ("none", torch.full((rows,), -1)),
        ("all different", torch.randperm(num, generator=g)), ("past the end", torch.full((rows,), num)),
        ("far out", torch.where(torch.arange(rows) % 3 == 0, 2 ** 31 - 1, -2 ** 31)), ("two in turn", torch.arange(rows) % 2),
    ]:
        for with_base, with_scales in ((True, True), (False, True), (True, False)):
            _announce("lora order", dtype, name, with_base, with_scales)
            _check_lora(ops, (x, a, b, adapters.to(torch.int32), base if with_base else None, scales if with_scales else None), name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [16, 32, 64, 128, 256])
def test_lora_whole_blocks_of_columns(ops, rank, dtype):
    """Ranks that fill their steps, blocks of 64 columns with and without a rest, several to a wave; also in place and off 16 bytes."""
    for rows, num, columns in ((3, 1, 64), (70, 2, 600), (21, 9, 1536), (150, 3, 2900)):
        _announce("lora whole blocks", rank, dtype, rows, num, columns)
        case = _lora_case(rows, num, rank, 96, columns, dtype, seed=rank + columns)
        x, a, b, adapters, base, scales = case
        got = _check_lora(ops, case, f"{rank} {columns}")
        _check_lora(ops, (x, a, b, adapters, None, scales), f"{rank} {columns}, no base")
        own = torch.empty(base.numel() + 3, dtype=dtype, device="cuda")[3:].view(base.shape)
        own.copy_(base)
        ops.lora(x.cuda(), a.cuda(), b.cuda(), adapters.cuda(), base=own, scales=scales.cuda(), c=own)
        assert torch.equal(own, got)


def _shifted(t, elements):
    """The same values `elements` behind a boundary of 16 bytes."""
    flat = torch.empty(t.numel() + 16, dtype=t.dtype, device="cuda")
    out = flat[elements:elements + t.numel()].view(t.shape)
    out.copy_(t)
    return out


def test_lora_past_32_bits(ops):
    """More than 2^32 bytes of base and out: windows at the end, in the middle and at the beginning as in calls of their own."""
    rows, num, rank, hin, hout = 600_001, 7, 16, 64, 4096
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, hin, device="cuda", generator=g).bfloat16()
    a = torch.randn(num, rank, hin, device="cuda", generator=g).bfloat16()
    b = torch.randn(num, hout, rank, device="cuda", generator=g).bfloat16()
    base = torch.empty(rows, hout, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    adapters = torch.randint(-1, num, (rows,), device="cuda", generator=g, dtype=torch.int32)
    assert base.numel() > 2 ** 31
    _announce("lora past 32 bits")
    got = ops.lora(x, a, b, adapters, base=base)
    for begin in (0, 64 * 4000, rows // 64 * 64 - 128):
        at = slice(begin, min(begin + 192, rows))
        assert torch.equal(got[at], ops.lora(x[at].contiguous(), a, b, adapters[at].contiguous(), base=base[at].contiguous()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_that_begin_on_any_element(ops, dtype):
    """Even sizes behind odd addresses, odd sizes behind either: the same bits as from a boundary."""
    for depth in (640, 641, 1000, 1027):
        x, a, b, adapters, base, scales = [v.cuda() for v in _lora_case(70, 3, 40, depth, 96, dtype, seed=depth)]
        w13 = torch.randn(4, 2 * 72, depth, device="cuda").mul_(depth ** -0.5).to(dtype)
        w2 = torch.randn(4, depth, 72, device="cuda").mul_(0.1).to(dtype)
        few, experts = x[:9].contiguous(), torch.randint(0, 4, (9, 2), dtype=torch.int32, device="cuda")
        weights = torch.rand(9, 2, device="cuda")
        want = ops.lora(x, a, b, adapters, base=base, scales=scales)
        want_few = ops.moe_few_tokens(few, w13, w2, experts, weights, trans_b=True)
        for at in ((1, 0), (0, 1), (1, 1), (2, 3)):
            _announce("rows on any element", dtype, depth, at)
            got = ops.lora(_shifted(x, at[0]), _shifted(a, at[1]), _shifted(b, at[0]), adapters, base=_shifted(base, at[1]), scales=scales)
            assert torch.equal(got, want)
            got = ops.moe_few_tokens(_shifted(few, at[0]), _shifted(w13, at[1]), _shifted(w2, at[0]), experts, weights, trans_b=True)
            assert torch.equal(got, want_few)


def test_lora_in_place_and_into_a_given_tensor(ops):
    case = [v.cuda() for v in _lora_case(90, 4, 12, 65, 333, torch.bfloat16, seed=4)]
    x, a, b, adapters, base, scales = case
    want = ops.lora(x, a, b, adapters, base=base, scales=scales)
    c = torch.full_like(base, float("nan"))
    assert ops.lora(x, a, b, adapters, base=base, scales=scales, c=c) is c and torch.equal(c, want)
    again = base.clone()
    ops.lora(x, a, b, adapters, base=again, scales=scales, c=again)
    assert torch.equal(again, want)


def test_lora_reads_named_adapters_only(ops):
    """NaN in adapters that no row names, and around every tensor (off the 16-byte boundary), reaches no output."""
    x, a, b, adapters, base, scales = _lora_case(40, 6, 13, 51, 77, torch.float16, seed=2)
    adapters = torch.where(adapters == 3, -1, adapters)
    a[3], b[3], scales[3] = float("nan"), float("nan"), float("nan")

    def framed(t):
        flat = torch.full((t.numel() + 67,), float("nan"), dtype=t.dtype, device="cuda")
        flat[33:33 + t.numel()] = t.flatten().cuda()
        return flat[33:33 + t.numel()].view(t.shape)

    c = framed(torch.zeros_like(base))
    got = ops.lora(framed(x), framed(a), framed(b), adapters.cuda(), base=framed(base), scales=framed(scales), c=c)
    rtol, least = ROUNDING[x.dtype]
    a[3], b[3], scales[3] = 0, 0, 0
    want, off = _lora_reference(x, a, b, adapters, base, scales)
    _close(got, want, rtol, off * (1 + rtol) + least, "framed")
    assert torch.isnan(c._base[:33]).all() and torch.isnan(c._base[33 + c.numel():]).all()


def test_lora_large_and_small_values(ops):
    """What lies between the two products may be larger than float16 holds, or far smaller; an infinite row stays one."""
    x = torch.full((3, 64), 1000.0, dtype=torch.float16)
    x[1] = 2.0 ** -20
    a = torch.full((1, 8, 64), 1000.0, dtype=torch.float16)           # v = 6.4e7, far past 65504
    b = torch.full((1, 40, 8), 2.0 ** -20, dtype=torch.float16)
    adapters, base = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 40, dtype=torch.float16)
    scales = torch.ones(1)
    _check_lora(ops, (x, a, b, adapters, base, scales), "large v")
    x[2, 5] = INF
    got = ops.lora(x.cuda(), a.cuda(), b.cuda(), adapters.cuda(), base=base.cuda()).cpu()
    assert torch.isinf(got[2]).all() and torch.isfinite(got[:2]).all()
    small = torch.full((1, 8, 64), 2.0 ** -24, dtype=torch.float16)
    _check_lora(ops, (x[:2], small, torch.full((1, 40, 8), 1000.0, dtype=torch.float16), adapters[:2], base[:2], scales), "small v")


def test_lora_bfloat16_largest_value(ops):
    """Between the two products, a number between the largest bfloat16 and the largest float, which rounds up to an infinity: (2 - 2^-9) 2^127."""
    x = torch.ones(1, 2, dtype=torch.bfloat16)
    a = torch.tensor([[[(2 - 2.0 ** -7) * 2.0 ** 127, 0.75 * 2.0 ** 120]]], dtype=torch.float64).bfloat16()
    b = torch.tensor([[[2.0 ** -100], [0.0]]], dtype=torch.bfloat16)
    got = ops.lora(x.cuda(), a.cuda(), b.cuda(), torch.zeros(1, dtype=torch.int32).cuda()).cpu().double()
    want = torch.tensor([[(2 - 2.0 ** -9) * 2.0 ** 27, 0.0]], dtype=torch.float64)
    _close(got, want, 2.0 ** -8 + 2.0 ** -15, 0.0, "largest")


@pytest.mark.parametrize("rank", [2, 16, 30, 64, 128])
def test_lora_float16_small_beside_large(ops, rank):
    """float16's v is handed on in two halves, its row scaled to 2^14 at least: off by 2^-21 of itself and twice 2^-25 of that, 2^-38 of the row's largest.
    Half of each row is 2^20 times smaller than the other, and meets b that is as much larger."""
    x, a, b, adapters, base, _ = _lora_case(70, 3, rank, 96, 130, torch.float16, seed=rank)
    a[:, ::2] = a[:, ::2] * 2.0 ** 10
    a[:, 1::2] = a[:, 1::2] * 2.0 ** -10
    b[:, :, ::2] = b[:, :, ::2] * 2.0 ** -10
    b[:, :, 1::2] = b[:, :, 1::2] * 2.0 ** 10
    base[:] = 0
    want, off = torch.zeros(70, 130, dtype=torch.float64), torch.zeros(70, 130, dtype=torch.float64)
    for t in range(70):
        n = int(adapters[t])
        if n < 0:
            continue
        an, bn = a[n].double(), b[n].double()
        v = an @ x[t].double()
        v_off = (an.abs() @ x[t].double().abs()) * (2 * 96 * 2.0 ** -24) + v.abs() * 2.0 ** -21 + v.abs().max() * 2.0 ** -38
        want[t] = bn @ v
        off[t] = bn.abs() @ v_off + (bn.abs() @ v.abs()) * ((4 * rank + 8) * 2.0 ** -24)
    _announce("lora small beside large", rank)
    got = ops.lora(x.cuda(), a.cuda(), b.cuda(), adapters.cuda(), base=base.cuda())
    _close(got, want, 2.0 ** -11, off * (1 + 2.0 ** -11) + 2.0 ** -25, "small beside large")


def test_lora_same_bits_on_streams_and_in_graphs(ops):
    cases = [[v.cuda() for v in _lora_case(t, 12, 16, 1024, 777, torch.bfloat16, seed=t)] for t in (1, 64, 300)]

    def run():
        return [ops.lora(x, a, b, adapters, base=base, scales=scales) for x, a, b, adapters, base, scales in cases]

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(4):
        for out in captured:
            out.zero_()
        graph.replay()
        eager = run()
        torch.cuda.synchronize()
        for one in (again, captured, eager):
            for got, w in zip(one, want):
                assert torch.equal(got, w)


def test_lora_refuses_forward_mode(ops):
    x, a, b, adapters, base, scales = (v.cuda() for v in _lora_case(6, 3, 8, 32, 48, torch.bfloat16, seed=1))
    args = dict(x=x, a=a, b=b, adapters=adapters, base=base, scales=scales)
    with torch.autograd.forward_ad.dual_level():
        for name in ("x", "a", "b", "base", "scales"):
            dual = dict(args)
            dual[name] = torch.autograd.forward_ad.make_dual(args[name], torch.ones_like(args[name]))
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                ops.lora(**dual)


def test_lora_into_a_given_tensor_is_a_write(ops):
    """What saved c for its gradient notices, as with torch's own writes; without a graph, and on tensors that keep no count of writes, it just writes."""
    x, a, b, adapters, base, scales = (v.cuda() for v in _lora_case(6, 3, 8, 32, 48, torch.bfloat16, seed=1))
    p = torch.ones_like(base).requires_grad_(True)
    y = (p * base).sum()
    ops.lora(x, a, b, adapters, base=base, scales=scales, c=base)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    fresh = base.clone()
    y = (p * base).sum()
    ops.lora(x, a, b, adapters, base=base, scales=scales, c=fresh)
    y.backward()
    assert torch.equal(p.grad, base)
    with torch.inference_mode():
        c = torch.empty_like(base)
        assert torch.equal(ops.lora(x, a, b, adapters, base=base, scales=scales, c=c), fresh)


def test_lora_refuses(ops):
    x, a, b, adapters, base, scales = (v.cuda() for v in _lora_case(6, 3, 8, 32, 48, torch.bfloat16, seed=1))

    def call(**kw):
        args = dict(x=x, a=a, b=b, adapters=adapters, base=base, scales=scales)
        args.update(kw)
        return ops.lora(**args)

    bad = [(dict(x=x.cpu()), "same GPU"), (dict(x=x[0]), "2-d"), (dict(x=x.float()), "bfloat16"), (dict(a=a[0]), "3-d"),
           (dict(a=a.half()), "element type"), (dict(a=a[:, :, :31].contiguous()), "hidden_in"), (dict(b=b[:2]), "hidden_out"),
           (dict(b=b[:, :, :7].contiguous()), "rank"), (dict(adapters=adapters.long()), "int32"), (dict(adapters=adapters[:5]), "int32"),
           (dict(scales=scales[:2]), "float32"), (dict(scales=scales.half()), "float32"), (dict(base=base[:, :47]), "hidden_out"),
           (dict(base=base.half()), "element type"), (dict(x=torch.zeros(32, 6, device="cuda", dtype=x.dtype).t()), "contiguous"),
           (dict(c=base[:5]), "hidden_out"), (dict(a=torch.zeros(1, 257, 32, device="cuda", dtype=x.dtype),
                                                   b=torch.zeros(1, 48, 257, device="cuda", dtype=x.dtype), scales=None), "at most 256"),
           (dict(a=a.clone().requires_grad_(True)), "no gradient"), (dict(base=base.clone().requires_grad_(True)), "no gradient")]
    for kw, message in bad:
        with pytest.raises(RuntimeError, match=message):
            call(**kw)
    both = torch.zeros(7 * 48, device="cuda", dtype=x.dtype)
    with pytest.raises(RuntimeError, match="overlap"):
        call(base=both[:288].view(6, 48), c=both[48:].view(6, 48))
    square = [v.cuda() for v in _lora_case(6, 3, 8, 48, 48, torch.bfloat16, seed=1)]
    with pytest.raises(RuntimeError, match="overlap"):
        ops.lora(square[0], square[1], square[2], square[3], c=square[0])


# ------------------------------------------------------------------ together

def test_example_runs_the_operators_together(ops):
    """Training lowers the loss; the decode form gives what the training form gives (which rounds the activation and each
    expert's row to bfloat16 in between, each by up to 2^-8 of itself); the adapted projection gives the sum of its parts."""
    import importlib.util
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "expert_layer.py")
    spec = importlib.util.spec_from_file_location("expert_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, one, other, y, projection, x, adapters = example.main(steps=12)
    assert losses[-1][0] < losses[0][0]
    scale = float(one.float().pow(2).mean().sqrt())
    assert float((one.float() - other.float()).abs().max()) <= 6 * 2.0 ** -8 * scale + 2.0 ** -7 * float(one.float().abs().max())
    want = x.double() @ projection.weight[0].detach().double().t()
    for i, n in enumerate(adapters.tolist()):
        if n >= 0:
            want[i] += 0.5 * (projection.b[n].double() @ (projection.a[n].double() @ x[i].double()))
    off = (y.double() - want).abs() - (2.0 ** -7 * want.abs() + 2.0 ** -8 * float(want.detach().abs().max()))   # (rounded twice: the shared part, the sum)
    assert float(off.max()) <= 0.0
