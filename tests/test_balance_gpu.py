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
    balance, z = float(got.balance.detach()), float(got.z.detach())
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
@pytest.mark.parametrize("tokens,experts,sequences", [(50, 9, 50), (13, 111, 69), (280, 74, 109), (2, 300, 114), (700, 40, 3000), (3000, 6, 2500), (2500, 20, 900)])
def test_short_and_empty_sequences(ops, tokens, experts, sequences, score):
    """Sequences shorter than what a workgroup takes at once, with runs of empty ones before, between and behind them."""
    _announce("short", tokens, experts, sequences, score)
    logits, chosen, g = _inputs(tokens, experts, 2, torch.float32, tokens + sequences)
    at = torch.sort(torch.randint(tokens + 1, (sequences + 1,), generator=g)).values
    few = torch.sort(torch.randint(0, tokens // 3 + 1, (sequences + 1,), generator=g) * 3).values   # (runs of alike)
    one = torch.arange(sequences + 1).clamp(max=tokens)
    ends = torch.cat([torch.full((sequences - sequences // 2,), tokens // 2), torch.full((sequences // 2 + 1,), tokens)])
    for what, offsets in (("at random", at), ("runs", few), ("of one", one), ("two places", ends)):
        _check(ops, logits, chosen, offsets.clamp(max=tokens).to(torch.int32), torch.rand(tokens, generator=g) < 0.9, score, what)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,sequences", [(5003, 8, 1), (9001, 16, 2), (70001, 3, 1), (20011, 17, 3), (17000, 100, 1), (6000, 513, 2)])
def test_long_sequences(ops, tokens, experts, sequences, score):
    """More units to a sequence than one turn of the second kernel takes."""
    _announce("long", tokens, experts, sequences, score)
    logits, chosen, g = _inputs(tokens, experts, 2, torch.bfloat16, tokens)
    _check(ops, logits, chosen, _offsets(tokens, sequences, g), torch.rand(tokens, generator=g) < 0.8, score, "long")


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
    assert float(got.balance.detach()) == 0 and float(got.z.detach()) == 0 and not grad.any()
    # no tokens
    for offsets in (None, torch.tensor([0], dtype=torch.int32), torch.tensor([0, 0, 0], dtype=torch.int32)):
        got, grad = _check(ops, logits[:0], chosen[:0], offsets, None, score, "no tokens")
        assert float(got.balance.detach()) == 0 and grad.shape == (0, 40)


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


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masks_by_the_lowest_value_of_the_type(ops, dtype, score):
    """All of a row, or all but one: the balance and its gradient, and of fp16, whose lowest has a square in fp32, also z."""
    _announce("lowest", dtype, score)
    for experts in (8, 30, 256, 700):
        logits, chosen, g = _inputs(64, experts, 3, dtype, 7 + experts)
        low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
        logits[3] = low
        logits[4, 1:] = low
        logits[5, ::2] = low
        logits[6, :-1] = high     # (one expert closed, the others at the largest)
        logits[7] = low
        logits[7, 2] = -INF
        logits[8] = low / 2
        if score == "softmax":
            logits[9, :-1] = low  # (sigmoid(x) of the last is 1 whatever the others)
            logits[9, -1] = high
        for mask in (None, torch.rand(64, generator=g) < 0.7):
            if dtype == torch.float16:
                _check(ops, logits, chosen, torch.tensor([0, 20, 64], dtype=torch.int32), mask, score, (experts, "all"))
                continue
            offsets = torch.tensor([0, 20, 64], dtype=torch.int32)
            want = _reference(logits, chosen, offsets, mask, score, (0.7, 0.0))
            leaf = logits.cuda().requires_grad_(True)
            got = ops.balance_loss(leaf, chosen.cuda(), offsets=offsets.cuda(), mask=None if mask is None else mask.cuda(), score=score)
            assert torch.equal(got.counts.cpu().long(), want["counts"])
            assert abs(float(got.balance.detach()) - float(want["balance"])) <= 2e-5 * float(want["balance"]), (experts, float(got.balance.detach()))
            assert float(want["z"]) < 1e38 or float(got.z.detach()) == INF
            grad, = torch.autograd.grad(got.balance, leaf, torch.tensor(0.7, device="cuda"))
            half, least = ROUNDING[dtype]
            off = (grad.double().cpu() - want["grad"]).abs() - (2e-5 * want["grad_scale"] + half * want["grad"].abs() + least + 1e-37)
            assert float(off.max()) <= 0, (experts, float(off.max()))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_any_size(ops, dtype, score):
    """Rows whose largest logit is anywhere between ordinary numbers and the largest of the type: all alike, all but one, around a size, and among
    ordinary rows.  z and its gradient too where a float holds the sum of its squares: 17 of 3e18 do, one of 1e20 does not."""
    _announce("sizes", dtype, score)
    sizes = [1e3, 1e5, 2.0 ** 20 * 0.999, 2.0 ** 20 * 1.01, 1e7, 1e8, 1e9, 1.5e9, 3e9, 1e10, 1e12, 1e15, 1e18, 3e18, 1e20, 1e25, 1e30, 1e37, 2e38]
    offsets = torch.tensor([0, 20, 32], dtype=torch.int32)
    for experts in (8, 30, 256, 700):
        for size in sizes:
            for sign in (1.0, -1.0):
                logits, chosen, g = _inputs(32, experts, 3, dtype, 11 + experts)
                at = sign * size
                logits[3] = at
                logits[4, 1:] = at
                logits[5, ::2] = at
                logits[6] = (at + 3.0 * torch.randn(experts, generator=g).double()).to(dtype)
                logits[7, :-1] = at
                logits[7, -1] = -INF
                logits[8:12] = (at * (1.0 + torch.randint(3, (4, experts), generator=g) * 2.0 ** -7)).to(dtype)   # steps of bf16
                logits[25:28] = at
                if size < 1e19:
                    _check(ops, logits, chosen, offsets, None, score, (experts, at))
                    continue
                want = _reference(logits, chosen, offsets, None, score, (0.7, 0.0))
                leaf = logits.cuda().requires_grad_(True)
                got = ops.balance_loss(leaf, chosen.cuda(), offsets=offsets.cuda(), score=score)
                assert abs(float(got.balance.detach()) - float(want["balance"])) <= 2e-5 * float(want["balance"]), (experts, at, float(got.balance.detach()))
                assert float(got.z.detach()) == INF, (experts, at)
                grad, = torch.autograd.grad(got.balance, leaf, torch.tensor(0.7, device="cuda"))
                half, least = ROUNDING[dtype]
                off = (grad.double().cpu() - want["grad"]).abs() - (2e-5 * want["grad_scale"] + half * want["grad"].abs() + least + 1e-37)
                assert float(off.max()) <= 0, (experts, at, float(off.max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_infinite_logits_that_count(ops, dtype):
    """+inf in a counted token: z is none, and softmax's balance; sigmoid(+inf) is 1, so the balance of sigmoids and its gradient are what the
    definition gives (as at 1e4, where a sigmoid is 1 and its slope 0 in 64 bits), and other tokens' gradients are what they were."""
    _announce("infinite", dtype)
    for experts in (8, 30, 256, 700):
        logits, chosen, g = _inputs(64, experts, 3, dtype, 21 + experts)
        at = torch.zeros(64, experts, dtype=torch.bool)
        at[5, 2] = at[40, ::3] = at[41] = True
        logits[42, 1:] = -INF
        at[42, 0] = True
        offsets, near = torch.tensor([0, 20, 64], dtype=torch.int32), logits.double().masked_fill(at, 1e4)
        logits = logits.masked_fill(at, INF)
        rest = ~at.any(1)
        half, least = ROUNDING[dtype]
        for score in ("softmax", "sigmoid"):
            def grads(which, of):
                leaf = logits.cuda().requires_grad_(True)
                loss = ops.balance_loss(leaf, chosen.cuda(), offsets=offsets.cuda(), score=score)
                return loss, torch.autograd.grad(loss[which], leaf, torch.tensor(of, device="cuda"))[0].double().cpu()

            (balance, z, counts), grad = grads(0, 0.7)
            want = _reference(near, chosen, offsets, None, score, (0.7, 0.0))
            assert math.isnan(z.detach())
            off = (grad - want["grad"]).abs() - (2e-5 * want["grad_scale"] + half * want["grad"].abs() + least + 1e-37)
            if score == "sigmoid":
                assert abs(float(balance.detach()) - float(want["balance"])) <= 2e-5 * float(want["balance"]), (experts, float(balance.detach()))
                assert float(off.max()) <= 0, (experts, float(off.max()))
            else:
                assert math.isnan(balance.detach())
                assert float(off[rest].max()) <= 0, experts
            want = _reference(near, chosen, offsets, None, score, (0.0, 1.3))
            grad = grads(1, 1.3)[1]
            off = (grad - want["grad"]).abs() - (2e-5 * want["grad_scale"] + half * want["grad"].abs() + least + 1e-37)
            assert float(off[rest].max()) <= 0 and torch.isnan(grad[~rest]).any(1).all(), experts


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_small_sigmoids_beside_large_logits(ops, dtype):
    """A sigmoid has its size whatever the token's largest logit, and its element of the balance's gradient too: each to 2e-5 of itself (one
    exponential, off by 2^-24 of |x| <= 60, and some units in the last place), a rounding of the type, and 1e-37 where fp32 ends."""
    _announce("small sigmoids", dtype)
    for experts in (8, 30, 256, 700):
        logits, chosen, g = _inputs(64, experts, 3, dtype, 51 + experts)
        top = torch.linspace(0.0, 60.0, 64)
        logits = (torch.rand(64, experts, generator=g) * 110.0 - 60.0).minimum(top.unsqueeze(1))
        logits[:, 1] = top
        logits = logits.to(dtype)
        want = _reference(logits, chosen, None, None, "sigmoid", (64.0, 0.0))
        leaf = logits.cuda().requires_grad_(True)
        got = ops.balance_loss(leaf, chosen.cuda(), score="sigmoid")
        assert abs(float(got.balance.detach()) - float(want["balance"])) <= 2e-5 * float(want["balance"])
        grad, = torch.autograd.grad(got.balance, leaf, torch.tensor(64.0, device="cuda"))
        half, least = ROUNDING[dtype]
        # (the difference of share and its mean by p, each off by 2e-5 of itself, times the element's own p and slope)
        x = logits.double()
        p = torch.softmax(torch.nn.functional.logsigmoid(x), 1)
        share = want["counts"][0].double() * experts / (3 * 64)
        scale = p * torch.sigmoid(-x) * torch.maximum(share, (share * p).sum(1, keepdim=True))
        off = (grad.double().cpu() - want["grad"]).abs() - (2e-5 * scale + half * want["grad"].abs() + least + 1e-37)
        assert float(off.max()) <= 0, (experts, float(off.max()))


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


def test_second_derivatives_and_forward_mode_are_refused(ops):
    logits, chosen, g = _inputs(20, 8, 2, torch.float32, 10)
    leaf = logits.cuda().requires_grad_(True)
    loss = ops.balance_loss(leaf, chosen.cuda())
    grad, = torch.autograd.grad(loss.balance, leaf, create_graph=True)
    want = _reference(logits, chosen, None, None, "softmax", (1.0, 0.0))
    assert ((grad.detach().double().cpu() - want["grad"]).abs() <= 2e-5 * want["grad_scale"] + 1e-37).all()
    with pytest.raises(RuntimeError, match="second derivative"):
        grad.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ops.balance_loss(fwd.make_dual(logits.cuda(), torch.ones_like(logits).cuda()), chosen.cuda())
    q = torch.randn(3, 16, device="cuda", requires_grad=True)
    for call in (lambda: ops.quantize_rows(q), lambda: ops.swiglu_quantize(q)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    with torch.no_grad():
        v = ops.quantize_rows(q)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.gmm_int8(v.values, v.scales.clone().requires_grad_(True), v.values.view(1, 3, 16), v.scales.view(1, 3), torch.tensor([3]))


def test_wrong_arguments_on_the_device(ops):
    logits, chosen, g = _inputs(20, 8, 2, torch.float32, 10)
    x, e = logits.cuda(), chosen.cuda()
    offsets, mask = torch.tensor([0, 20], dtype=torch.int32, device="cuda"), torch.ones(20, dtype=torch.bool, device="cuda")
    for kw, text in ((dict(offsets=offsets.long()), "offsets"), (dict(offsets=offsets.cpu()), "offsets"), (dict(offsets=offsets[:0]), "offsets"),
                     (dict(offsets=offsets.view(1, 2)), "offsets"), (dict(mask=mask.int()), "mask"), (dict(mask=mask[:5]), "mask"), (dict(mask=mask.cpu()), "mask")):
        with pytest.raises(RuntimeError, match=text):
            ops.balance_loss(x, e, **kw)
    with pytest.raises(RuntimeError, match="same GPU"):
        ops.balance_loss(x, chosen)
    with pytest.raises(RuntimeError, match="row_index"):
        ops.quantize_rows(x, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="row_index"):
        ops.quantize_rows(x, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="2-d"):
        ops.quantize_rows(x.view(2, 10, 8), torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="even"):
        ops.swiglu_quantize(x[:, :7].contiguous())
    a, b = torch.zeros(2, 16, dtype=torch.int8, device="cuda"), torch.zeros(1, 8, 16, dtype=torch.int8, device="cuda")
    s, t = torch.ones(2, device="cuda"), torch.ones(1, 8, device="cuda")
    with pytest.raises(RuntimeError, match="same GPU"):
        ops.gmm_int8(a, s.cpu(), b, t, torch.tensor([2]))
    with pytest.raises(RuntimeError, match="negative"):
        ops.gmm_int8(a, s, b, t, torch.tensor([-1]))
    with pytest.raises(RuntimeError, match="sum past"):
        ops.gmm_int8(a, s, b, t, torch.tensor([3]))
    with pytest.raises(RuntimeError, match="overlap"):   # c within the rows of a
        ops.gmm_int8(a, s, b, t, torch.tensor([2]), c=a.view(-1).view(torch.bfloat16).view(2, 8))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_captured_with_its_gradient_and_replayed(ops, score):
    """Forward and backward in one graph, replayed with other logits, choices, sequences and masks, with eager work between."""
    logits, chosen, g = _inputs(700, 40, 4, torch.bfloat16, 12)
    x = logits.cuda().requires_grad_(True)
    experts, offsets, mask = chosen.cuda(), _offsets(700, 9, g).cuda(), torch.ones(700, dtype=torch.bool, device="cuda")
    grads = torch.tensor(0.3, device="cuda"), torch.tensor(0.2, device="cuda")

    def step():
        loss = ops.balance_loss(x, experts, offsets, mask, score)
        return loss, torch.autograd.grad((loss.balance, loss.z), x, grads)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = step()
    for n in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device="cuda") * (n + 1))
            experts.random_(0, 40)
            offsets.copy_(_offsets(700, 9, g))
            mask.copy_(torch.rand(700, device="cuda") < 0.8)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.detach().clone() for v in (loss.balance, loss.z, loss.counts, grad)]
        eager, eager_grad = step()
        torch.cuda.synchronize()
        for a, b in zip(got, (eager.balance, eager.z, eager.counts, eager_grad)):
            assert torch.equal(a, b.detach()), n


def test_a_captured_gradient_beside_a_living_graph_is_refused(ops):
    """While a graph of the same logits lives that was made outside the capture, on the default stream; then, without it, captured and replayed."""
    logits, chosen, g = _inputs(60, 20, 2, torch.float32, 31)
    x, experts = logits.cuda().requires_grad_(True), chosen.cuda()

    def step():
        loss = ops.balance_loss(x, experts)
        return torch.autograd.grad((loss.balance, loss.z), x, (torch.ones((), device="cuda"), torch.ones((), device="cuda")))[0]

    want = step()
    living = ops.balance_loss(x, experts)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="captured backward pass of balance_loss"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    torch.cuda.synchronize()
    grad, = torch.autograd.grad(living.balance, x)     # (the graph outside is as it was)
    assert torch.isfinite(grad).all()
    del living, grad
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_two_calls_at_once(ops):
    logits, chosen, g = _inputs(3000, 64, 6, torch.float32, 13)
    x, e, offsets = logits.cuda().requires_grad_(True), chosen.cuda(), _offsets(3000, 11, g).cuda()
    first = ops.balance_loss(x, e, offsets)
    want, = torch.autograd.grad((first.balance, first.z), x, (torch.ones((), device="cuda"), torch.ones((), device="cuda")))
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                loss = ops.balance_loss(x, e, offsets)
                outs.append((loss, torch.autograd.grad(loss.balance + loss.z, x)[0]))
    torch.cuda.synchronize()
    for loss, grad in outs:
        assert torch.equal(loss.balance, first.balance) and torch.equal(loss.z, first.z) and torch.equal(grad, want)


def test_a_router_learns_to_spread_its_tokens(ops):
    """route and balance_loss in a step, whose gradients are those of the same step by the formulas."""
    g = torch.Generator().manual_seed(14)
    tokens, hidden, experts, k = 256, 32, 16, 2
    x, w = torch.randn(tokens, hidden, generator=g), torch.randn(hidden, experts, generator=g)
    offsets = torch.tensor([0, 100, 256], dtype=torch.int32)
    weight = w.cuda().requires_grad_(True)
    logits = x.cuda() @ weight
    r = ops.route(logits, k)
    loss = ops.balance_loss(logits, r.experts, offsets.cuda())
    assert torch.equal(loss.counts.sum(0).long(), r.batch_sizes)
    (r.weights.square().sum() * 0.1 + loss.balance + 0.01 * loss.z).backward()
    # the same in 64 bits, from the logits and choices of the step
    l64 = logits.detach().double().cpu().requires_grad_(True)
    chosen = r.experts.cpu().long()
    picked = torch.softmax(l64, 1).gather(1, chosen)
    (0.1 * (picked / picked.sum(1, keepdim=True)).square().sum()).backward()
    want = l64.grad + _reference(logits.detach().cpu(), r.experts.cpu(), offsets, None, "softmax", (1.0, 0.01))["grad"]
    weight_grad = x.double().t() @ want
    # (a product of 256 terms in fp32, of gradients that are off by 2e-5 of terms below one)
    scale = (x.double().abs().t() @ (want.abs() + 0.2)).max()
    assert ((weight.grad.double().cpu() - weight_grad).abs() <= 1e-4 * scale).all()


def test_many_tokens_and_sequences(ops):
    """Offsets past 32 bits of bytes, and as many sequences as tokens."""
    _announce("large")
    tokens, experts = 1 << 22, 512   # 4.3e9 bytes of bf16
    x = torch.randn(1 << 16, experts, device="cuda", dtype=torch.bfloat16).repeat(tokens >> 16, 1).requires_grad_(True)
    e = torch.randint(experts, (1 << 16, 2), dtype=torch.int32, device="cuda").repeat(tokens >> 16, 1)
    loss = ops.balance_loss(x, e)
    grad, = torch.autograd.grad((loss.balance, loss.z), x, (torch.tensor(float(tokens), device="cuda"), torch.tensor(float(tokens), device="cuda")))
    part = x[:1 << 16].detach().requires_grad_(True)
    want = ops.balance_loss(part, e[:1 << 16])
    part_grad, = torch.autograd.grad((want.balance, want.z), part, (torch.tensor(65536.0, device="cuda"), torch.tensor(65536.0, device="cuda")))
    # the same tokens over and over: the same means, by other sums
    assert abs(float(loss.balance.detach() - want.balance.detach())) <= 4e-5 * float(want.balance.detach()) and abs(float(loss.z.detach() - want.z.detach())) <= 4e-5 * float(want.z.detach())
    assert torch.equal(loss.counts, want.counts * (tokens >> 16))
    last = grad[-(1 << 16):].float()
    assert ((last - part_grad.float()).abs() <= 2.0 ** -7 * part_grad.float().abs() + 1e-4).all()
    del x, e, grad, last
    tokens = 20000
    logits, chosen, g = _inputs(tokens, 24, 3, torch.float32, 15)
    _check(ops, logits, chosen, torch.arange(tokens + 1, dtype=torch.int32), None, "softmax", "a sequence to a token")


def test_more_sequences_than_30_bits_count(ops):
    """Sequences past 2^30, nearly all of them empty: the numbers of two that a search is between do not fit 31 bits together."""
    _announce("sequences past 2^30")
    tokens, experts, sequences = 8192, 2, (1 << 30) + 1000
    logits, chosen, g = _inputs(tokens, experts, 1, torch.float32, 61)
    # (token 8 n + 4 and those behind it are in another sequence than the four before: far apart for the first ones, among the last for the rest)
    places = torch.cat([torch.tensor([10, (1 << 30) + 100]), (1 << 30) + 101 + torch.sort(torch.randperm(890, generator=g)[:60]).values, torch.tensor([sequences - 2])])
    ends = torch.cat([torch.tensor([4, 8]), 12 + 8 * torch.sort(torch.randperm(1000, generator=g)[:60]).values, torch.tensor([tokens])])
    offsets = torch.zeros(sequences + 1, dtype=torch.int32, device="cuda")
    for place, end, behind in zip(places.tolist(), ends.tolist(), places.tolist()[1:] + [sequences]):
        offsets[place + 1:behind + 1] = end
    few = torch.cat([torch.tensor([0]), ends]).to(torch.int32)
    want = _reference(logits, chosen, few, None, "softmax", (0.7, 1.3))
    leaf = logits.cuda().requires_grad_(True)
    got = ops.balance_loss(leaf, chosen.cuda(), offsets)
    grad, = torch.autograd.grad((got.balance, got.z), leaf, (torch.tensor(0.7, device="cuda"), torch.tensor(1.3, device="cuda")))
    assert abs(float(got.balance.detach()) - float(want["balance"])) <= 2e-5 * float(want["balance"])
    assert abs(float(got.z.detach()) - float(want["z"])) <= 2e-5 * float(want["z"]) + 2e-6 * float(want["z_scale"])
    assert torch.equal(got.counts[places.cuda()].cpu().long(), want["counts"])
    assert ((grad.double().cpu() - want["grad"]).abs() <= 2e-5 * want["grad_scale"] + 2.0 ** -24 * want["grad"].abs() + 1e-37).all()


def test_the_example_runs(ops):
    """examples/int8_expert_layer.py: that it runs, that every parameter gets a gradient, and that the layer in 8 bits is the layer that
    was trained.  Quantising moves each element of a row by up to half a step, 1/254 of the row's largest: uniformly distributed, by 1/880 of it
    on average (root mean square), and a row's largest is 3 to 5 times its mean size.  Two operands in each of two products are
    quantised, so that results are off by about 2 * 5 / 880 = 1.1 % with all of them independent; 3 % leaves room for the router's ties."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "int8_expert_layer.py")
    spec = importlib.util.spec_from_file_location("int8_expert_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    layer, losses, one, other, served = example.main(steps=3)
    assert len(losses) == 3 and all(math.isfinite(v) for step in losses for v in step[:2])
    assert all(c.shape == (5, 16) and int(c.sum()) == 2 * (2048 - 40) for _, _, c in losses)
    assert float((one.float() - other.float()).norm()) <= 0.03 * float(one.float().norm())
    y, router = layer(torch.randn(64, 512, device="cuda").bfloat16())
    (y.float().sum() + router.balance + router.z).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any() for p in layer.parameters())
