"""Performance cases of an expert layer's operators in 8-bit integers, and of its balance loss: rows quantised with a
scale each, grouped products of 8-bit integers with scales per row and per column, a gated layer of them, and the
loss that keeps a router's experts evenly used.

listed() is a fixed selection, draw() gives further cases of the same ranges, prepare() makes what a program has
in hand before the call, run() is one pass: where `own` is set, the calls a user makes of this package; otherwise
the same results by elementary torch operations.  exact() gives them in 64 bits.  A case is a dict of plain values:

  op       "quantize": 8-bit integers and a scale per row
               rows, hidden, dtype, gathered_from (rows of the tensor that they are picked from; 0: all rows in place)
           "gmm": grouped product of 8-bit integers, times the scales of its row and of its column
               rows, experts, hidden_in, hidden_out, dtype (of the result), skew (of the groups' sizes, 0: by chance
               alone), on_device (where batch_sizes are)
           "layer": rows of tokens quantised, gate and up, their gated product quantised, down: four calls
               tokens, experts, top_k, hidden, ffn, dtype
           "balance": balance loss and z-loss of router logits, counts per sequence, and the logits' gradient
               tokens, experts, top_k, sequences (packed one after the other), dtype (of the logits), score ("softmax",
               "sigmoid"), masked (share of tokens that are left out)
"""
import math

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def _quantize(rows, hidden, dtype="bfloat16", gathered_from=0, name=None):
    case = dict(op="quantize", rows=rows, hidden=hidden, dtype=dtype, gathered_from=gathered_from)
    return case if name is None else dict(case, name=name)


def _gmm(rows, experts, hidden_in, hidden_out, dtype="bfloat16", skew=0.0, on_device=True, name=None):
    case = dict(op="gmm", rows=rows, experts=experts, hidden_in=hidden_in, hidden_out=hidden_out, dtype=dtype, skew=skew,
                on_device=on_device)
    return case if name is None else dict(case, name=name)


def _layer(tokens, experts, top_k, hidden, ffn, dtype="bfloat16", name=None):
    case = dict(op="layer", tokens=tokens, experts=experts, top_k=top_k, hidden=hidden, ffn=ffn, dtype=dtype)
    return case if name is None else dict(case, name=name)


def _balance(tokens, experts, top_k, sequences=1, dtype="bfloat16", score="softmax", masked=0.0, name=None):
    case = dict(op="balance", tokens=tokens, experts=experts, top_k=top_k, sequences=sequences, dtype=dtype, score=score,
                masked=masked)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # One token's activations on their way into a product: nothing but latency.
        _quantize(1, 4096, name="quantize one token"),
        # fp32 rows of a length that no vector divides.
        _quantize(1003, 2047, dtype="float32", name="quantize odd"),
        # A prompt's tokens, two rows of each, in the order of their experts.
        _quantize(16384, 4096, gathered_from=8192, name="quantize gathered prompt"),
        # Token generation for one request, gate and up of two large experts: a stream of weights.
        _gmm(2, 8, 4096, 28672, name="int8 product one token"),
        # A batch of requests in token generation over the many experts that one device holds.
        _gmm(512, 128, 7168, 4096, dtype="float16", name="int8 product decode"),
        # Sizes that are odd numbers (any size is allowed), a handful of groups, sizes on the host.
        _gmm(333, 5, 2047, 1023, on_device=False, name="int8 product odd sizes"),
        # The largest: prompts of a whole batch through 8 large experts, unevenly used.
        _gmm(32768, 8, 4096, 14336, skew=0.5, name="int8 product prompts"),
        # A gated layer for one token: four launches, and the weights of two experts.
        _layer(1, 8, 2, 4096, 14336, name="int8 layer one token"),
        # A prompt over fine-grained experts.
        _layer(4096, 64, 6, 2048, 1408, dtype="float16", name="int8 layer prompt"),
        # A micro-batch of short packed sequences, a number of experts that no vector divides, some padding, fp16.
        _balance(1003, 37, 3, sequences=17, dtype="float16", masked=0.1, name="balance odd masked"),
        # A training micro-batch over fine-grained experts, logits in fp32 as many routers keep them.
        _balance(8192, 64, 6, sequences=5, dtype="float32", name="balance training"),
        # The largest batch of tokens on one device over many experts, gates from a sigmoid.
        _balance(65536, 256, 8, sequences=64, score="sigmoid", name="balance large"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _hidden(rng, lo, hi):
    """A hidden size: mostly a multiple of 128 or 16, one in four any number."""
    n, pick = _log_uniform(rng, lo, hi), rng.random()
    return max(128, n // 128 * 128) if pick < 0.5 else (max(16, n // 16 * 16) if pick < 0.75 else n)


def draw(rng):
    """One more case, no dearer than the dearest listed one of its operator."""
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = tuple(max(a, b) for a, b in zip(most.get(c["op"], (0, 0)), (w["bytes"], w["flops"])))
    while True:
        op = rng.choice(["quantize", "gmm", "gmm", "layer", "balance"])
        two_byte = "float16" if rng.random() < 0.3 else "bfloat16"
        if op == "quantize":
            rows = _log_uniform(rng, 1, 32768)
            case = _quantize(rows, _hidden(rng, 64, 16384), dtype=rng.choice(["float32", two_byte, two_byte]),
                             gathered_from=rng.choice([0, max(1, rows // rng.choice([1, 2, 6]))]))
        elif op == "gmm":
            case = _gmm(_log_uniform(rng, 1, 32768), _log_uniform(rng, 1, 128), _hidden(rng, 128, 14336), _hidden(rng, 128, 28672),
                        dtype=two_byte, skew=rng.choice([0.0, 0.5, 1.0]), on_device=rng.random() < 0.7)
        elif op == "layer":
            experts = _log_uniform(rng, 4, 64)
            case = _layer(_log_uniform(rng, 1, 4096), experts, min(experts, rng.choice([1, 2, 4, 6])), _hidden(rng, 256, 4096),
                          _hidden(rng, 128, 14336), dtype=two_byte)
        else:
            experts, tokens = _log_uniform(rng, 4, 512), _log_uniform(rng, 1, 65536)
            case = _balance(tokens, experts, min(experts, rng.choice([1, 2, 4, 6, 8])), sequences=_log_uniform(rng, 1, 128),
                            dtype=rng.choice(["float32", two_byte]), score=rng.choice(["softmax", "softmax", "sigmoid"]),
                            masked=rng.choice([0.0, 0.0, 0.1]))
        w = work(case)
        held = case["experts"] * (case["hidden_in"] * case["hidden_out"] if op == "gmm" else 3 * case["hidden"] * case["ffn"]) \
            if op in ("gmm", "layer") else 0      # (idle experts take memory too)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and held <= 4 << 30:
            return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, gen, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype).mul_(scale)


def _activations(rows, hidden, gen, dtype):
    """Rows as a model has them: of different sizes, with a few channels much larger than the rest."""
    channels = torch.where(torch.rand(hidden, generator=gen, device="cuda") < 0.01, 10.0, 1.0)
    sizes = torch.exp(_randn((rows, 1), gen, torch.float32, 0.5))
    return (_randn((rows, hidden), gen, torch.float32) * channels * sizes).to(dtype)


def _int8(shape, gen):
    """What is left of normally distributed numbers after each row's largest is brought to 127 (about four deviations)."""
    return _randn(shape, gen, torch.bfloat16, 32.0).round_().clamp_(-127, 127).to(torch.int8)


def _weights(experts, hidden_out, hidden_in, gen):
    scales = (torch.rand((experts, hidden_out), generator=gen, device="cuda") + 0.5) * (hidden_in ** -0.5 / 32)
    return _int8((experts, hidden_out, hidden_in), gen), scales


def _groups(rows, experts, skew, gen):
    """Sizes of the groups that `rows` rows fall into, some experts more in demand than others."""
    demand = torch.exp(_randn((experts,), gen, torch.float32, skew)) if skew > 0 else torch.ones(experts, device="cuda")
    chosen = torch.multinomial(demand, rows, replacement=True, generator=gen)
    return torch.zeros(experts, dtype=torch.int64, device="cuda").scatter_add_(0, chosen, torch.ones_like(chosen))


def prepare(case, seed):
    gen, dtype = _generator(seed), _DTYPES[case["dtype"]]
    state = dict(case=case)
    if case["op"] == "quantize":
        rows, source = case["rows"], case["gathered_from"]
        state["x"] = _activations(source or rows, case["hidden"], gen, dtype)
        state["row_index"] = torch.randint(source, (rows,), generator=gen, device="cuda", dtype=torch.int32) if source else None
    elif case["op"] == "gmm":
        rows, experts = case["rows"], case["experts"]
        state["a"] = _int8((rows, case["hidden_in"]), gen)
        state["a_scales"] = torch.rand(rows, generator=gen, device="cuda") / 32 + 0.01
        state["b"], state["b_scales"] = _weights(experts, case["hidden_out"], case["hidden_in"], gen)
        sizes = _groups(rows, experts, case["skew"], gen)
        state["sizes"] = sizes.tolist()
        state["batch_sizes"] = sizes if case["on_device"] else sizes.cpu()
        state["expert_of_row"] = torch.repeat_interleave(torch.arange(experts, device="cuda"), sizes)
    elif case["op"] == "layer":
        tokens, experts, k, hidden, ffn = case["tokens"], case["experts"], case["top_k"], case["hidden"], case["ffn"]
        state["x"] = _activations(tokens, hidden, gen, dtype)
        state["w13"], state["w13_scales"] = _weights(experts, 2 * ffn, hidden, gen)
        state["w2"], state["w2_scales"] = _weights(experts, hidden, ffn, gen)
        chosen = torch.sort(torch.rand((tokens, experts), generator=gen, device="cuda"), dim=1).indices[:, :k].reshape(-1)
        expert_of_row, order = torch.sort(chosen, stable=True)
        sizes = torch.zeros(experts, dtype=torch.int64, device="cuda").scatter_add_(0, chosen, torch.ones_like(chosen))
        state["sizes"], state["batch_sizes"], state["expert_of_row"] = sizes.tolist(), sizes, expert_of_row
        state["row_index"] = (order // k).to(torch.int32)
    else:
        t, e, k, n = case["tokens"], case["experts"], case["top_k"], case["sequences"]
        logits = _randn((t, e), gen, torch.float32, 1.5).to(dtype)
        state["experts"] = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32).contiguous()
        state["logits"] = logits.requires_grad_(True)   # (a leaf; a model's own logits are a node of its graph)
        # (sequences end at sorted cuts, so that some are empty where there are many and the tokens are few)
        cuts = torch.sort(torch.randint(t + 1, (n - 1,), generator=gen, device="cuda")).values
        ends = torch.tensor([0], device="cuda"), cuts, torch.tensor([t], device="cuda")
        state["offsets"] = torch.cat(ends).to(torch.int32)
        state["mask"] = torch.rand(t, generator=gen, device="cuda") >= case["masked"] if case["masked"] > 0 else None
        state["grads"] = torch.rand((), generator=gen, device="cuda") + 0.5, torch.rand((), generator=gen, device="cuda") + 0.5
    return state


def _quantized(x):
    """Nearest integers of 127 x / max|x| of each row, ties to even, and max|x| / 127: in 64 bits, as a quotient next to a tie needs."""
    x = x.double()
    most = x.abs().amax(1, keepdim=True)
    return torch.round(x * 127.0 / torch.where(most > 0, most, torch.ones_like(most))).to(torch.int8), (most / 127.0).float().squeeze(1)


def _product(a, a_scales, b, b_scales, sizes, expert_of_row, dtype):
    if len(a) < len(b):   # the weights of each row
        out = torch.matmul(b[expert_of_row].float(), a.float().unsqueeze(2)).squeeze(2)
    else:
        out = torch.cat([x @ w.float().t() for x, w in zip(a.float().split(sizes), b) if len(x) > 0])
    return (out * a_scales.unsqueeze(1) * b_scales[expert_of_row]).to(dtype)


def _plain_layer(s, case):
    dtype, groups = s["x"].dtype, (s["sizes"], s["expert_of_row"])
    q, scales = _quantized(s["x"][s["row_index"].long()])
    gate, up = _product(q, scales, s["w13"], s["w13_scales"], *groups, dtype).float().chunk(2, dim=1)
    q, scales = _quantized(gate / (1.0 + torch.exp(-gate)) * up)
    return _product(q, scales, s["w2"], s["w2_scales"], *groups, dtype)


def _plain_balance(s, case):
    t, e, k, n = case["tokens"], case["experts"], case["top_k"], case["sequences"]
    x = s["logits"].detach().float()
    counted = torch.ones(t, device=x.device) if s["mask"] is None else s["mask"].float()
    sequence = torch.searchsorted(s["offsets"], torch.arange(t, device=x.device, dtype=torch.int32), right=True) - 1
    top = x.max(1, keepdim=True).values
    exps = torch.exp(x - top)
    total = exps.sum(1, keepdim=True)
    softmax, lse = exps / total, top + torch.log(total)
    if case["score"] == "softmax":
        scores, slope = softmax, torch.ones_like(x)
    else:
        sig = 1.0 / (1.0 + torch.exp(-x))
        scores, slope = sig / sig.sum(1, keepdim=True), 1.0 - sig
    all_tokens = counted.sum()
    tokens = torch.zeros(n, device=x.device).index_add_(0, sequence, counted)
    chosen = (sequence.unsqueeze(1) * e + s["experts"]).reshape(-1)
    counts = torch.zeros(n * e, device=x.device).index_add_(0, chosen, counted.repeat_interleave(k)).view(n, e)
    mass = torch.zeros((n, e), device=x.device).index_add_(0, sequence, scores * counted.unsqueeze(1))
    share = counts * (e / k) / (tokens.clamp_min(1.0) * all_tokens).unsqueeze(1)   # what a unit of mass adds to the loss
    g, h = s["grads"]
    f = share[sequence]
    grad = g * scores * slope * (f - (f * scores).sum(1, keepdim=True)) + h * (2.0 / all_tokens) * lse * softmax
    return dict(balance=(share * mass).sum(), z=(lse.squeeze(1) ** 2 * counted).sum() / all_tokens, counts=counts.to(torch.int32),
                logits_grad=(grad * counted.unsqueeze(1)).to(s["logits"].dtype))


def run(s):
    case = s["case"]
    if own:
        from grouped_gemm_amd import ops
        if case["op"] == "quantize":
            q = ops.quantize_rows(s["x"], row_index=s["row_index"])
            return dict(values=q.values, scales=q.scales)
        if case["op"] == "gmm":
            return ops.gmm_int8(s["a"], s["a_scales"], s["b"], s["b_scales"], s["batch_sizes"], dtype=_DTYPES[case["dtype"]])
        if case["op"] == "layer":
            dtype = _DTYPES[case["dtype"]]
            q = ops.quantize_rows(s["x"], row_index=s["row_index"])
            gate_up = ops.gmm_int8(q.values, q.scales, s["w13"], s["w13_scales"], s["batch_sizes"], dtype=dtype)
            h = ops.swiglu_quantize(gate_up)
            return ops.gmm_int8(h.values, h.scales, s["w2"], s["w2_scales"], s["batch_sizes"], dtype=dtype)
        loss = ops.balance_loss(s["logits"], s["experts"], offsets=s["offsets"], mask=s["mask"], score=case["score"])
        grad, = torch.autograd.grad((loss.balance, loss.z), s["logits"], s["grads"])
        return dict(balance=loss.balance.detach(), z=loss.z.detach(), counts=loss.counts, logits_grad=grad)
    if case["op"] == "quantize":
        values, scales = _quantized(s["x"] if s["row_index"] is None else s["x"][s["row_index"].long()])
        return dict(values=values, scales=scales)
    if case["op"] == "gmm":
        return _product(s["a"], s["a_scales"], s["b"], s["b_scales"], s["sizes"], s["expert_of_row"], _DTYPES[case["dtype"]])
    return (_plain_layer if case["op"] == "layer" else _plain_balance)(s, case)


def _distinct(things, draws, of_each=1):
    """Expected number of different ones among `things` after `draws` draws of `of_each` different ones each."""
    return things * (1.0 - (1.0 - of_each / things) ** draws)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "quantize":
        rows, hidden = case["rows"], case["hidden"]
        read = min(rows, case["gathered_from"]) or rows
        return {"bytes": read * hidden * size + rows * (hidden + 4) + (4 * rows if case["gathered_from"] else 0), "flops": 3 * rows * hidden}
    if case["op"] == "gmm":
        rows, hin, hout = case["rows"], case["hidden_in"], case["hidden_out"]
        read = _distinct(case["experts"], rows) * hout * (hin + 4)
        return {"bytes": int(read + rows * (hin + 4 + 2 * hout) + 8 * case["experts"]), "flops": 2 * rows * hin * hout}
    if case["op"] == "layer":
        t, k, hidden, ffn = case["tokens"], case["top_k"], case["hidden"], case["ffn"]
        read = _distinct(case["experts"], t, k) * (3 * hidden * ffn + 4 * (2 * ffn + hidden))
        return {"bytes": int(read + 2 * t * hidden + t * k * (2 * hidden + 4)), "flops": 6 * t * k * hidden * ffn}
    t, e, k, n = case["tokens"], case["experts"], case["top_k"], case["sequences"]
    # (the logits twice, before and after the caller's loss; the gradient and the counts written)
    return {"bytes": t * e * size * 3 + t * k * 4 + n * e * 4 + 4 * (n + 1), "flops": t * e * 16}


def _exact_rows(x):
    most = x.abs().amax(1, keepdim=True)
    return torch.round(127.0 * x / most.clamp_min(1e-300)), most / 127.0


def _exact_product(q, scales, b, b_scales, sizes):
    out = torch.empty((q.shape[0], b.shape[1]), dtype=torch.float64, device="cuda")
    start = 0
    for e, n in enumerate(sizes):
        if n > 0:
            out[start:start + n] = (q[start:start + n] @ b[e].double().t()) * scales[start:start + n] * b_scales[e].double()
        start += n
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["x"].double() if s["row_index"] is None else s["x"].double()[s["row_index"].long()]
        return dict(values=None, scales=_exact_rows(x)[1].squeeze(1))
    if case["op"] == "gmm":
        return _exact_product(s["a"].double(), s["a_scales"].double().unsqueeze(1), s["b"], s["b_scales"], s["sizes"])
    if case["op"] == "layer":
        dtype = _DTYPES[case["dtype"]]
        q, scales = _exact_rows(s["x"].double()[s["row_index"].long()])
        both = _exact_product(q, scales, s["w13"], s["w13_scales"], s["sizes"]).to(dtype).double()   # (a layer's rows in between are of its type)
        gate, up = both[:, :case["ffn"]], both[:, case["ffn"]:]
        q, scales = _exact_rows(torch.nn.functional.silu(gate) * up)
        return _exact_product(q, scales, s["w2"], s["w2_scales"], s["sizes"])
    x = s["logits"].detach().double().requires_grad_(True)
    k, e, offsets = case["top_k"], case["experts"], s["offsets"].tolist()
    counted = torch.ones(case["tokens"], dtype=torch.float64, device="cuda") if s["mask"] is None else s["mask"].double()
    lse = torch.logsumexp(x, 1)
    scores = torch.softmax(x, 1) if case["score"] == "softmax" else torch.sigmoid(x) / torch.sigmoid(x).sum(1, keepdim=True)
    hot = torch.zeros_like(scores).scatter_add_(1, s["experts"].long(), torch.ones(s["experts"].shape, dtype=torch.float64, device="cuda"))
    all_tokens, balance = counted.sum(), 0.0
    for begin, end in zip(offsets, offsets[1:]):
        weight = counted[begin:end].unsqueeze(1)
        tokens = weight.sum().clamp_min(1.0)
        evenly = (hot[begin:end] * weight).sum(0) * e / (k * tokens) * ((scores[begin:end] * weight).sum(0) / tokens)
        balance = balance + evenly.sum() * tokens / all_tokens
    z = (lse ** 2 * counted).sum() / all_tokens
    grad, = torch.autograd.grad((balance, z), x, (s["grads"][0].double(), s["grads"][1].double()))
    return dict(balance=balance.detach(), z=z.detach(), counts=None, logits_grad=grad)
