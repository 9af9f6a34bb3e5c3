"""The balance loss of a router, its z-loss, counts and gradients, against their definitions in 64 bits.

Everything is computed in fp32: exp(x - top) is off by 2^-24 |x - top| from the rounding of its argument and some units in the last
place, p by the same; the losses are sums of non-negative terms over at most some hundred roundings in a row (tokens of a lane,
units of a sequence, lanes, sequences), each 2^-24 of the sum: together below 2e-5 of balance for |x - top| <= 64.  A log of a sum of
exponentials is off by 1e-6 (1 + |it| + max |x|) at most, z by its square's share of that and the same sums.  A gradient is a difference of
such terms, off by 2e-5 of the largest term it is made of, and rounded to the logits' type (half a step)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
ROUNDING = {torch.float32: (2.0 ** -24, 0.0), torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25)}


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from grouped_gemm import ops as _ops
    return _ops


def _announce(*what):
    print("[case]", *what, flush=True)


def _reference(logits, experts, offsets, mask, score, grads=None):
    """By the formulas, in 64 bits, with the scale of each gradient's terms."""
    x = logits.double()
    t, e = x.shape
    k = experts.shape[1]
    offsets = [0, t] if offsets is None else offsets.tolist()
    counted = torch.ones(t, dtype=torch.bool) if mask is None else mask.clone()
    inside = torch.zeros(t, dtype=torch.bool)
    inside[offsets[0]:offsets[-1]] = True
    counted &= inside
    closed = (x == -INF).all(1, keepdim=True)
    safe = x.masked_fill(closed, 0.0)
    softmax = torch.softmax(safe, 1).masked_fill(closed, 0.0)
    lse = torch.logsumexp(safe, 1).masked_fill(closed.squeeze(1), 0.0)
    # (sigmoids divided by their sum: by their logarithms, which no size of theirs loses)
    p = softmax if score == "softmax" else torch.softmax(torch.nn.functional.logsigmoid(safe), 1).masked_fill(closed, 0.0)
    p = torch.where(x == -INF, torch.zeros_like(p), p)
    slope = torch.ones_like(x) if score == "softmax" else torch.sigmoid(-x)
    n = len(offsets) - 1
    all_tokens = int(counted.sum())
    counts = torch.zeros(n, e, dtype=torch.int64)
    balance, shares = 0.0, torch.zeros(t, e, dtype=torch.float64)
    for s in range(n):
        rows = torch.arange(offsets[s], offsets[s + 1])
        rows = rows[counted[rows]]
        chosen = experts[rows].long().reshape(-1)
        counts[s] = torch.bincount(chosen[(chosen >= 0) & (chosen < e)], minlength=e)
        if len(rows) == 0:
            continue
        share = counts[s].double() * e / (k * len(rows))
        shares[rows] = share
        balance = balance + (share * p[rows].sum(0)).sum()
    over = 1.0 / max(all_tokens, 1)
    out = dict(balance=torch.as_tensor(balance, dtype=torch.float64) * over, z=(lse ** 2)[counted].sum() * over, counts=counts,
               z_scale=((1.0 + lse.abs() + safe.masked_fill(x == -INF, 0.0).abs().amax(1)) * lse.abs())[counted].sum() * over)
    if grads is not None:
        g, h = grads
        c = counted.double().unsqueeze(1) * over
        out["grad"] = c * (g * p * slope * (shares - (shares * p).sum(1, keepdim=True)) + 2.0 * h * lse.unsqueeze(1) * softmax)
        most = safe.masked_fill(x == -INF, 0.0).abs().amax(1, keepdim=True)
        out["grad_scale"] = c * (abs(g) * p * shares.amax(1, keepdim=True) + 2.0 * abs(h) * (1.0 + lse.abs().unsqueeze(1) + most) * softmax)
    return out


def _check(ops, logits, experts, offsets=None, mask=None, score="softmax", what="", grads=(0.7, 1.3)):
    """All on the CPU."""
    gpu = lambda v: None if v is None else v.cuda()  # noqa: E731
    leaf = logits.cuda().requires_grad_(True)
    got = ops.balance_loss(leaf, experts.cuda(), offsets=gpu(offsets), mask=gpu(mask), score=score)
    want = _reference(logits, experts, offsets, mask, score, grads)
    assert got.counts.dtype == torch.int32 and got.balance.dtype == got.z.dtype == torch.float32 and got.balance.shape == got.z.shape == ()
    assert torch.equal(got.counts.cpu().long(), want["counts"]), what
    balance, z = float(got.balance), float(got.z)
    assert abs(balance - float(want["balance"])) <= 2e-5 * float(want["balance"]), (what, balance, float(want["balance"]))
    assert abs(z - float(want["z"])) <= 2e-5 * float(want["z"]) + 2e-6 * float(want["z_scale"]), (what, z, float(want["z"]))
    grad, = torch.autograd.grad((got.balance, got.z), leaf, tuple(torch.tensor(v, device="cuda") for v in grads))
    assert grad.dtype == logits.dtype
    half, least = ROUNDING[logits.dtype]
    off = (grad.double().cpu() - want["grad"]).abs() - (2e-5 * want["grad_scale"] + half * want["grad"].abs() + least + 1e-37)
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()))
    # without a gradient wanted: the same bits
    again = ops.balance_loss(logits.cuda(), experts.cuda(), offsets=gpu(offsets), mask=gpu(mask), score=score)
    assert torch.equal(again.balance, got.balance) and torch.equal(again.z, got.z) and torch.equal(again.counts, got.counts)
    assert not again.balance.requires_grad and got.balance.requires_grad and got.z.requires_grad and not got.counts.requires_grad
    return got, grad


def _inputs(tokens, experts, k, dtype, seed, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(tokens, experts, generator=g) * scale).to(dtype)
    return logits, torch.argsort(logits.float(), dim=1, descending=True)[:, :k].to(torch.int32).contiguous(), g


def _offsets(tokens, sequences, g):
    cuts = torch.sort(torch.randint(tokens + 1, (sequences - 1,), generator=g)).values
    return torch.cat([torch.tensor([0]), cuts, torch.tensor([tokens])]).to(torch.int32)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,experts,k,sequences", [(1, 1, 1, None), (1, 8, 2, 1), (1, 64, 6, 3), (17, 37, 3, None), (16, 5, 5, 4), (100, 64, 6, 7),
                                                        (257, 65, 4, 2), (333, 128, 8, 40), (1003, 200, 8, 17), (600, 256, 8, None), (130, 300, 2, 3),
                                                        (70, 512, 32, 5), (90, 1000, 8, 9), (40, 1024, 1, None), (4096, 64, 6, 5), (5000, 8, 2, 600)])
def test_losses_counts_and_gradient(ops, tokens, experts, k, sequences, dtype, score):
    _announce("losses", tokens, experts, k, sequences, dtype, score)
    logits, chosen, g = _inputs(tokens, experts, k, dtype, tokens + experts)
    offsets = None if sequences is None else _offsets(tokens, sequences, g)
    _check(ops, logits, chosen, offsets, None, score, "all tokens")
    _check(ops, logits, chosen, offsets, torch.rand(tokens, generator=g) < 0.7, score, "masked")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_sequences_of_every_kind(ops, score):
    _announce("sequences", score)
    logits, chosen, g = _inputs(500, 40, 4, torch.float32, 3)
    for offsets in ([0, 500], [0, 0, 500, 500], [0, 0, 0, 0], [500, 500], [100, 400], [3, 3, 17, 17, 17, 499], [0], [250], list(range(0, 501)),
                    [0] * 300 + [500] * 300, [7] + list(range(20, 480, 3))):
        _check(ops, logits, chosen, torch.tensor(offsets, dtype=torch.int32), None, score, offsets[:6])
    # a sequence none of whose tokens counts, and none that counts at all
    mask = torch.ones(500, dtype=torch.bool)
    mask[100:220] = False
    _check(ops, logits, chosen, torch.tensor([0, 100, 220, 500], dtype=torch.int32), mask, score, "a masked sequence")
    got, grad = _check(ops, logits, chosen, torch.tensor([0, 100, 500], dtype=torch.int32), torch.zeros(500, dtype=torch.bool), score, "nothing")
    assert float(got.balance) == 0 and float(got.z) == 0 and not grad.any()
    # no tokens
    for offsets in (None, torch.tensor([0], dtype=torch.int32), torch.tensor([0, 0, 0], dtype=torch.int32)):
        got, grad = _check(ops, logits[:0], chosen[:0], offsets, None, score, "no tokens")
        assert float(got.balance) == 0 and grad.shape == (0, 40)


def test_evenly_used_experts_give_one(ops):
    experts = (torch.arange(64).reshape(16, 4) % 16).to(torch.int32).cuda()
    got = ops.balance_loss(torch.zeros(16, 16, device="cuda"), experts)
    assert abs(float(got.balance) - 1.0) < 1e-6 and abs(float(got.z) - math.log(16.0) ** 2) < 1e-5
    assert (got.counts == 4).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_closed_experts_and_extreme_logits(ops, dtype, score):
    _announce("extremes", dtype, score)
    logits, chosen, g = _inputs(64, 30, 3, dtype, 5)
    logits = logits.masked_fill(torch.rand(64, 30, generator=g) < 0.4, -INF)
    logits[3] = -INF                      # a token that no expert is open to
    logits[4] = torch.finfo(dtype).min    # ... by the lowest value of the type: all alike
    logits[5, :29] = torch.finfo(dtype).min
    logits[6] = -60.0                     # sigmoids far below one
    logits[7] = 40.0
    logits[8, 1:] = -INF
    if dtype == torch.float32:            # (the log of a sum cannot show beside the lowest of fp32, whose square is no float)
        logits[4], logits[5, :29] = -1e4, -1e4
    if dtype == torch.bfloat16:
        logits[4], logits[5, :29] = -1e4, -1e4
    _check(ops, logits, chosen, torch.tensor([0, 20, 64], dtype=torch.int32), None, score, "extremes")
    # NaN and infinities where they are not counted do not show
    mask = torch.rand(64, generator=g) < 0.6
    wild = logits.clone()
    wild[~mask, 0] = NAN
    wild[~mask, 1] = INF
    got, grad = _check(ops, logits, chosen, None, mask, score, "masked")
    again = ops.balance_loss(wild.cuda().requires_grad_(True), chosen.cuda(), mask=mask.cuda(), score=score)
    assert torch.equal(again.balance, got.balance) and torch.equal(again.z, got.z)
    outside = ops.balance_loss(torch.cat([wild, wild]).cuda(), torch.cat([chosen, chosen]).cuda(), torch.tensor([0, 0], dtype=torch.int32, device="cuda"), score=score)
    assert float(outside.balance) == 0 and float(outside.z) == 0
    # ... and where they are, the losses are none
    logits[10, 2] = NAN
    got = ops.balance_loss(logits.cuda(), chosen.cuda(), score=score)
    assert math.isnan(got.balance) and math.isnan(got.z)


def test_numbers_that_name_no_expert_are_no_choice(ops):
    logits, chosen, g = _inputs(300, 20, 4, torch.float32, 8)
    chosen[torch.rand(300, 4, generator=g) < 0.3] = -1
    chosen[5] = torch.tensor([20, 2 ** 31 - 1, -2 ** 31, 19], dtype=torch.int32)
    chosen[6] = 3   # one expert four times
    _check(ops, logits, chosen, torch.tensor([0, 100, 300], dtype=torch.int32), None, "softmax", "no expert")


def test_one_gradient_alone_and_differences(ops):
    logits, chosen, g = _inputs(48, 10, 2, torch.float32, 9)
    offsets = torch.tensor([0, 20, 48], dtype=torch.int32)
    for score in ("softmax", "sigmoid"):
        for which in (0, 1):
            leaf = logits.cuda().requires_grad_(True)
            loss = ops.balance_loss(leaf, chosen.cuda(), offsets.cuda(), score=score)
            grad, = torch.autograd.grad(loss[which], leaf)
            want = _reference(logits, chosen, offsets, None, score, (1.0, 0.0) if which == 0 else (0.0, 1.0))
            assert ((grad.double().cpu() - want["grad"]).abs() <= 2e-5 * want["grad_scale"] + 1e-37).all()
            # central differences of the 64-bit loss: off by their second-order term, step^2 times a third derivative below 10
            step, name = 1e-4, ("balance", "z")[which]
            for at in ((0, 0), (19, 3), (20, 9), (47, 5)):
                up, down = logits.double(), logits.double()
                up[at] += step
                down[at] -= step
                slope = (_reference(up, chosen, offsets, None, score)[name] - _reference(down, chosen, offsets, None, score)[name]) / (2 * step)
                assert abs(float(slope) - float(grad[at])) <= 2e-5 * float(want["grad_scale"][at]) + 10 * step ** 2
    # an expanded gradient, and a sum of both losses
    leaf = logits.cuda().requires_grad_(True)
    loss = ops.balance_loss(leaf, chosen.cuda())
    (loss.balance * 0.01 + loss.z * 0.001).backward()
    want = _reference(logits, chosen, None, None, "softmax", (0.01, 0.001))
    assert ((leaf.grad.double().cpu() - want["grad"]).abs() <= 2e-5 * want["grad_scale"] + 2.0 ** -23 * want["grad"].abs()).all()
