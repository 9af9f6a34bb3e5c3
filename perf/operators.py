"""Performance cases of the operators around the grouped GEMM: the router, the gated expert layer for a few
tokens, and low-rank adapters beside a shared projection.

listed() is a fixed selection, draw() gives further cases of the same ranges, prepare() makes what a program has
in hand before the call, run() is one pass: where `own` is set, the calls a user makes of this package; otherwise
the same results by elementary torch operations in 32 bits, rounded once.  exact() gives them in 64 bits.  A case is
a dict of plain values:

  op       "route": router logits -> weights, experts, and the order that sorts rows by expert
               tokens, experts, top_k, dtype (of the logits), score ("softmax", "sigmoid"), normalize,
               masked (share of logits that are -inf), train (also the experts' mass, and the gradient of the logits)
           "moe": tokens through their experts' gated layers, summed by the router's weights
               tokens, experts, top_k, hidden, ffn, dtype, trans_b (weights stored (experts, out, in))
           "lora": base + scale * (x @ a^T) @ b^T, with the adapter of each row
               rows, requests (rows of one request are adjacent and share an adapter; some have none), adapters,
               rank, hidden_in, hidden_out, dtype
"""
import math

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def _route(tokens, experts, top_k, dtype="bfloat16", score="softmax", normalize=True, masked=0.0, train=False, name=None):
    case = dict(op="route", tokens=tokens, experts=experts, top_k=top_k, dtype=dtype, score=score, normalize=normalize,
                masked=masked, train=train)
    return case if name is None else dict(case, name=name)


def _moe(tokens, experts, top_k, hidden, ffn, dtype="bfloat16", trans_b=False, name=None):
    case = dict(op="moe", tokens=tokens, experts=experts, top_k=top_k, hidden=hidden, ffn=ffn, dtype=dtype, trans_b=trans_b)
    return case if name is None else dict(case, name=name)


def _lora(rows, requests, adapters, rank, hidden_in, hidden_out, dtype="bfloat16", name=None):
    case = dict(op="lora", rows=rows, requests=requests, adapters=adapters, rank=rank, hidden_in=hidden_in,
                hidden_out=hidden_out, dtype=dtype)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # Token generation for one request: nothing but latency.
        _route(1, 64, 6, name="route one token"),
        # A training micro-batch over fine-grained experts, logits in fp32 as many routers keep them, weights not
        # renormalized, the experts' mass for a balancing loss, and the gradient.
        _route(8192, 64, 6, dtype="float32", normalize=False, train=True, name="route training"),
        # A number of experts that no vector divides, some of them closed to some tokens, in fp16.
        _route(1003, 37, 3, dtype="float16", masked=0.1, train=True, name="route odd masked"),
        # The largest batch of tokens on one device over many experts, gates from a sigmoid.
        _route(65536, 256, 8, score="sigmoid", train=True, name="route large"),
        # Token generation for one request over few large experts: the weights of two of them.
        _moe(1, 8, 2, 4096, 14336, name="experts one token"),
        # A few requests over fine-grained experts, fp16, weights stored transposed.
        _moe(5, 64, 6, 2048, 1408, dtype="float16", trans_b=True, name="experts fine grained"),
        # Hidden sizes that are odd numbers (any size is allowed), a ragged batch.
        _moe(11, 8, 2, 1021, 2731, name="experts odd sizes"),
        # The largest: 64 tokens, top-8 of the 128 experts that one device holds, nearly all of their weights.
        _moe(64, 128, 8, 7168, 2048, trans_b=True, name="experts many"),
        # Token generation for one request with an adapter beside a square projection: latency.
        _lora(1, 1, 32, 16, 4096, 4096, name="adapters one token"),
        # A batch of requests in token generation, each with an adapter of its own choice.
        _lora(64, 64, 48, 16, 4096, 14336, dtype="float16", name="adapters decode"),
        # Sizes and a rank that are odd numbers, a handful of short prompts.
        _lora(333, 9, 5, 11, 2047, 1023, name="adapters odd sizes"),
        # Prompts of a dozen requests at once into a wide projection.
        _lora(8192, 12, 16, 64, 4096, 14336, name="adapters prefill"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _hidden(rng, lo, hi):
    """A hidden size: mostly a multiple of 64 or 8, one in four any number."""
    n, pick = _log_uniform(rng, lo, hi), rng.random()
    return max(64, n // 64 * 64) if pick < 0.5 else (max(8, n // 8 * 8) if pick < 0.75 else n)


def draw(rng):
    """One more case, no dearer than the dearest listed one of its operator."""
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), work(c)["bytes"])
    while True:
        op = rng.choice(["route", "moe", "lora"])
        two_byte = "float16" if rng.random() < 0.3 else "bfloat16"
        if op == "route":
            experts = _log_uniform(rng, 4, 512)
            case = _route(_log_uniform(rng, 1, 65536), experts, min(experts, rng.choice([1, 2, 3, 4, 6, 8])),
                          dtype=rng.choice(["float32", two_byte]), score=rng.choice(["softmax", "softmax", "sigmoid"]),
                          normalize=rng.random() < 0.6, masked=rng.choice([0.0, 0.0, 0.1]), train=rng.random() < 0.6)
        elif op == "moe":
            experts = _log_uniform(rng, 4, 128)
            case = _moe(_log_uniform(rng, 1, 64), experts, min(experts, rng.choice([1, 2, 4, 6, 8])), _hidden(rng, 256, 7168),
                        _hidden(rng, 128, 14336), dtype=two_byte, trans_b=rng.random() < 0.5)
            if experts * case["hidden"] * case["ffn"] > 128 * 7168 * 2048:   # (idle experts take memory too)
                continue
        else:
            rows = _log_uniform(rng, 1, 8192)
            case = _lora(rows, rows if rows <= 64 else _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 64),
                         rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)]), _hidden(rng, 256, 8192), _hidden(rng, 256, 14336),
                         dtype=two_byte)
        if work(case)["bytes"] <= most[op] and 3072 not in case.values():
            return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, gen, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype).mul_(scale)


def prepare(case, seed):
    gen, dtype = _generator(seed), _DTYPES[case["dtype"]]
    state = dict(case=case)
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        logits = _randn((t, e), gen, torch.float32, 1.5)
        if case["masked"] > 0:
            logits.masked_fill_(torch.rand((t, e), generator=gen, device="cuda") < case["masked"], -math.inf)
        state["logits"] = logits.to(dtype)
        if case["train"]:
            state["weights_grad"] = _randn((t, k), gen, torch.float32)
            state["mass_grad"] = _randn((e,), gen, torch.float32)
            state["logits"].requires_grad_(True)   # (a leaf; a model's own logits are a node of its graph)
    elif case["op"] == "moe":
        t, e, k, hidden, ffn = case["tokens"], case["experts"], case["top_k"], case["hidden"], case["ffn"]
        state["x"] = _randn((t, hidden), gen, dtype)
        first, second = (e, hidden, 2 * ffn), (e, ffn, hidden)
        if case["trans_b"]:
            first, second = (e, 2 * ffn, hidden), (e, hidden, ffn)
        state["w13"] = _randn(first, gen, dtype, hidden ** -0.5)
        state["w2"] = _randn(second, gen, dtype, ffn ** -0.5)
        logits = _randn((t, e), gen, torch.float32, 1.5)
        top, experts = torch.sort(logits, dim=1, descending=True)
        state["experts"] = experts[:, :k].to(torch.int32).contiguous()
        state["weights"] = torch.softmax(top[:, :k], dim=1).contiguous()
    else:
        rows, n, r = case["rows"], case["adapters"], case["rank"]
        state["x"] = _randn((rows, case["hidden_in"]), gen, dtype)
        state["a"] = _randn((n, r, case["hidden_in"]), gen, dtype, case["hidden_in"] ** -0.5)
        state["b"] = _randn((n, case["hidden_out"], r), gen, dtype, r ** -0.5)
        state["base"] = _randn((rows, case["hidden_out"]), gen, dtype)
        state["scales"] = torch.rand(n, generator=gen, device="cuda") + 0.5
        q = case["requests"]
        adapters = torch.randint(n, (q,), generator=gen, device="cuda")
        adapters = torch.where(torch.rand(q, generator=gen, device="cuda") < 0.1, -1, adapters)
        # (request i ends where the i-th of q - 1 sorted cuts lies)
        cuts = torch.sort(torch.randperm(rows - 1, generator=gen, device="cuda")[:q - 1] + 1).values if rows > 1 else None
        of_row = torch.zeros(rows, dtype=torch.int64, device="cuda")
        if cuts is not None:
            of_row[cuts] = 1
        state["adapters"] = adapters[torch.cumsum(of_row, 0)].to(torch.int32)
    return state


def _plain_route(s, case):
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    x = s["logits"].detach().float()
    chosen = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    picked = x.gather(1, chosen)
    top = picked[:, :1]
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    if case["score"] == "softmax":
        scores = torch.exp(x - top)
        scores = scores / scores.sum(1, keepdim=True).clamp_min(1e-30)
        kept = torch.exp(picked - top)
        own_slope = torch.ones_like(kept)           # d log(score) / d logit, without what all scores share
    else:
        scores = 1.0 / (1.0 + torch.exp(-x))
        kept = scores.gather(1, chosen)
        own_slope = 1.0 - kept
    share = kept / kept.sum(1, keepdim=True).clamp_min(1e-30)
    weights = share if case["normalize"] else scores.gather(1, chosen)
    flat = chosen.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    sizes = torch.zeros(e, dtype=torch.int64, device=x.device).scatter_add_(0, flat, torch.ones_like(flat))
    out = dict(weights=weights, experts=chosen.to(torch.int32), batch_sizes=sizes, row_index=(order // k).to(torch.int32),
               order=order.to(torch.int32))
    if case["train"]:
        out["mass"] = scores.sum(0)
        g, m = s["weights_grad"], s["mass_grad"].expand(t, e)
        if case["normalize"]:
            at_chosen = share * own_slope * (g - (g * share).sum(1, keepdim=True))
        else:
            at_chosen = torch.zeros_like(share)
            m = m.scatter_add(1, chosen, g)
        if case["score"] == "softmax":
            grad = scores * (m - (m * scores).sum(1, keepdim=True))
        else:
            grad = scores * (1.0 - scores) * m
        out["logits_grad"] = grad.scatter_add(1, chosen, at_chosen).to(s["logits"].dtype)
    return out


def _plain_moe(s, case):
    x, experts, slots = s["x"].float(), s["experts"].long(), case["tokens"] * case["top_k"]
    # (the experts of each slot where that is fewer than all experts, otherwise all experts on all tokens)
    gathered = slots < case["experts"]
    if gathered:
        w13, w2 = s["w13"][experts.reshape(-1)].float(), s["w2"][experts.reshape(-1)].float()
        x = x.repeat_interleave(case["top_k"], 0).unsqueeze(1)
    else:
        w13, w2 = s["w13"].float(), s["w2"].float()
        x = x.unsqueeze(0).expand(case["experts"], -1, -1)
    if case["trans_b"]:
        w13, w2 = w13.transpose(1, 2), w2.transpose(1, 2)
    gate, up = torch.matmul(x, w13).chunk(2, dim=2)
    y = torch.matmul(gate / (1.0 + torch.exp(-gate)) * up, w2)
    if gathered:
        y = y.view(case["tokens"], case["top_k"], -1)
    else:
        y = y[experts, torch.arange(case["tokens"], device=y.device).unsqueeze(1)]
    return (y * s["weights"].unsqueeze(2)).sum(1).to(s["x"].dtype)


def _plain_lora(s, case):
    x, base, adapters = s["x"].float(), s["base"].float(), s["adapters"].long()
    has = (adapters >= 0).unsqueeze(1)
    scale = s["scales"][adapters.clamp_min(0)].unsqueeze(1)
    n, r = case["adapters"], case["rank"]
    if case["rows"] < n:   # the adapter of each row
        a, b = s["a"][adapters.clamp_min(0)].float(), s["b"][adapters.clamp_min(0)].float()
        delta = torch.matmul(b, torch.matmul(a, x.unsqueeze(2))).squeeze(2)
    else:                  # all adapters side by side, each row keeping its own
        low = torch.matmul(x, s["a"].float().view(n * r, -1).t())
        mine = (torch.arange(n * r, device=x.device) // r) == adapters.unsqueeze(1)
        low = torch.where(mine, low, torch.zeros_like(low))
        delta = torch.matmul(low, s["b"].float().transpose(1, 2).reshape(n * r, -1))
    return torch.where(has, base + scale * delta, base).to(s["x"].dtype)


def run(s):
    case = s["case"]
    if not own:
        return {"route": _plain_route, "moe": _plain_moe, "lora": _plain_lora}[case["op"]](s, case)
    from grouped_gemm_amd import ops
    if case["op"] == "moe":
        return ops.moe_few_tokens(s["x"], s["w13"], s["w2"], s["experts"], s["weights"], trans_b=case["trans_b"])
    if case["op"] == "lora":
        return ops.lora(s["x"], s["a"], s["b"], s["adapters"], base=s["base"], scales=s["scales"])
    r = ops.route(s["logits"], case["top_k"], score=case["score"], normalize=case["normalize"], with_mass=case["train"])
    out = dict(weights=r.weights, experts=r.experts, batch_sizes=r.batch_sizes, row_index=r.row_index, order=r.order)
    if case["train"]:
        out["mass"] = r.mass
        out["logits_grad"], = torch.autograd.grad((r.weights, r.mass), s["logits"], (s["weights_grad"], s["mass_grad"]))
    return out


def _distinct(things, draws, of_each=1):
    """Expected number of different ones among `things` after `draws` draws of `of_each` different ones each."""
    return things * (1.0 - (1.0 - of_each / things) ** draws)


def work(case):
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        size = 4 if case["dtype"] == "float32" else 2
        once = t * e * size + t * k * (4 + 4 + 4 + 4) + 8 * e
        back = t * e * size * 2 + t * k * 8 + 8 * e   # (logits and chosen experts again, after the caller's loss)
        return {"bytes": once + (back if case["train"] else 0), "flops": t * e * (12 if case["train"] else 4)}
    if case["op"] == "moe":
        t, k, hidden, ffn = case["tokens"], case["top_k"], case["hidden"], case["ffn"]
        read = _distinct(case["experts"], t, k) * 3 * hidden * ffn
        return {"bytes": int(2 * (read + 2 * t * hidden) + 8 * t * k), "flops": 6 * t * k * hidden * ffn}
    t, r, hin, hout = case["rows"], case["rank"], case["hidden_in"], case["hidden_out"]
    read = _distinct(case["adapters"], 0.9 * case["requests"]) * r * (hin + hout)
    return {"bytes": int(2 * (read + t * (hin + 2 * hout)) + 4 * t), "flops": int(0.9 * 2 * t * r * (hin + hout))}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        x = s["logits"].detach().double().requires_grad_(True)
        k = case["top_k"]
        chosen = torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :k]
        closed = (x.detach() == -math.inf).all(1, keepdim=True)   # tokens that no expert is open to: weights of zero
        open_x = x.masked_fill(closed, 0.0)
        scores = (torch.softmax(open_x, 1) if case["score"] == "softmax" else torch.sigmoid(open_x)).masked_fill(closed, 0.0)
        weights = scores.gather(1, chosen)
        if case["normalize"]:
            weights = weights / weights.sum(1, keepdim=True).masked_fill(closed, 1.0)
        out = dict(weights=weights.detach(), experts=None, batch_sizes=None, row_index=None, order=None)
        if case["train"]:
            mass = scores.sum(0)
            out["mass"] = mass.detach()
            total = (weights * s["weights_grad"].double()).sum() + (mass * s["mass_grad"].double()).sum()
            out["logits_grad"], = torch.autograd.grad(total, x)
        return out
    if case["op"] == "moe":
        out = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        for e in torch.unique(s["experts"]).tolist():
            token, slot = torch.nonzero(s["experts"] == e, as_tuple=True)
            w13, w2 = s["w13"][e].double(), s["w2"][e].double()
            if case["trans_b"]:
                w13, w2 = w13.t(), w2.t()
            both = s["x"][token].double() @ w13
            gate, up = both[:, :case["ffn"]], both[:, case["ffn"]:]
            y = (torch.nn.functional.silu(gate) * up) @ w2
            out.index_add_(0, token, y * s["weights"][token, slot].double().unsqueeze(1))
        return out
    out = s["base"].double()
    for n in torch.unique(s["adapters"]).tolist():
        if n >= 0:
            rows = torch.nonzero(s["adapters"] == n).squeeze(1)
            delta = (s["x"][rows].double() @ s["a"][n].double().t()) @ s["b"][n].double().t()
            out.index_add_(0, rows, delta * s["scales"][n].double())
    return out
