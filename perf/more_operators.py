"""Timed cases of the operators between attention and the next token, with their plain forms.

What a decoder step runs beside the operators of a paged cache, on device tensors:

  residual_norm  the norm behind a block, its gate and residual, and the norm before the next block, in one pass
  moe            a mixture-of-experts layer for a few tokens: router, gated experts, weighted sum
  sample         the next token by temperature, top-k, top-p and min-p from a given random number per row

``run`` computes the plain form in elementary torch operations, or, with ``own`` set, calls the
package. Sizes are generic ones, besides the 197 tokens of 768 that this repository's ViT-B has.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token's residual stream between two blocks of a decoder: all latency
        dict(name="norm_step", op="norm", rows=1, width=4096, kind="rms", post=False, gate="none", bias=False, stream="same", scale=1.0,
             dtype="bf16"),
        # a prompt's tokens, norms on both sides of the block, a gate per channel and a residual scale
        dict(name="norm_prompt", op="norm", rows=4099, width=4096, kind="rms", post=True, gate="channel", bias=False, stream="same",
             scale=0.7, dtype="bf16"),
        # 64 images' tokens of a ViT-B with a gate per token, layer norms, in 32 bits
        dict(name="norm_images", op="norm", rows=64 * 197, width=768, kind="layer", post=False, gate="token", bias=True, stream="same",
             scale=1.0, dtype="fp32"),
        # a width that no wide access divides, with the residual stream kept in 32 bits
        dict(name="norm_odd", op="norm", rows=777, width=11001, kind="layer", post=True, gate="none", bias=True, stream="fp32", scale=1.0,
             dtype="fp16"),
        # one token through many small experts: the smallest step
        dict(name="moe_token", op="moe", tokens=1, width=2048, inner=768, experts=128, top_k=8, scoring="softmax", biased=False, scale=1.0,
             dtype="bf16"),
        # sequences decoded together, scores by sigmoid, a bias that only chooses
        dict(name="moe_batch", op="moe", tokens=13, width=4096, inner=1400, experts=64, top_k=6, scoring="sigmoid", biased=True, scale=2.5,
             dtype="fp16"),
        # few wide experts, nearly all of them read
        dict(name="moe_wide", op="moe", tokens=5, width=4096, inner=12000, experts=8, top_k=2, scoring="softmax", biased=False, scale=1.0,
             dtype="bf16"),
        # a large batch: every expert has some tens of tokens
        dict(name="moe_many", op="moe", tokens=200, width=2048, inner=1024, experts=32, top_k=4, scoring="softmax", biased=False,
             scale=1.0, dtype="bf16"),
        # one stream's next token: latency
        dict(name="sample_one", op="sample", rows=1, vocab=32000, temperature=0.8, top_k=0, top_p=0.95, min_p=0.0, mixed=False, masked=0.0,
             dtype="bf16"),
        # a decode step's rows with filters of their own, some greedy, logits in 32 bits
        dict(name="sample_step", op="sample", rows=48, vocab=128000, temperature=0.7, top_k=50, top_p=0.9, min_p=0.02, mixed=True,
             masked=0.0, dtype="fp32"),
        # a large batch over a large odd vocabulary, mass alone decides
        dict(name="sample_batch", op="sample", rows=256, vocab=150001, temperature=1.0, top_k=0, top_p=0.9, min_p=0.0, mixed=False,
             masked=0.0, dtype="bf16"),
        # the distribution as it is, over a vocabulary of which a grammar leaves a tenth
        dict(name="sample_plain", op="sample", rows=7, vocab=50021, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, masked=0.9,
             dtype="fp16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "moe", "sample"])
    if op == "norm":
        width = rng.choice([8 * _log(rng, 8, 2000), _log(rng, 64, 16000)])
        return dict(op=op, rows=_log(rng, 1, min(20000, 16000000 // width)), width=width, kind=rng.choice(["rms", "layer"]),
                    post=rng.random() < 0.5, gate=rng.choice(["none", "channel", "token"]), bias=rng.random() < 0.5,
                    stream=rng.choice(["same", "same", "fp32"]), scale=rng.choice([1.0, 0.5]), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    if op == "moe":
        experts = rng.choice([4, 8, 16, 60, 64, 128])
        width = 8 * _log(rng, 32, 512)
        inner = 8 * _log(rng, 16, max(17, min(1500, 300000000 // (3 * 8 * experts * width))))
        return dict(op=op, tokens=_log(rng, 1, 200), width=width, inner=inner, experts=experts, top_k=rng.randint(1, min(8, experts)),
                    scoring=rng.choice(["softmax", "sigmoid"]), biased=rng.random() < 0.3, scale=rng.choice([1.0, 2.5]),
                    dtype=rng.choice(["bf16", "fp16"]))
    vocab = _log(rng, 1000, 200000)
    return dict(op=op, rows=_log(rng, 1, min(256, 38000000 // vocab)), vocab=vocab, temperature=rng.choice([0.3, 0.7, 1.0, 1.3]),
                top_k=rng.choice([0, 0, 1, _log(rng, 2, 1000)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.95]),
                min_p=rng.choice([0.0, 0.0, 0.05]), mixed=rng.random() < 0.3, masked=rng.choice([0.0, 0.0, 0.5]),
                dtype=rng.choice(["bf16", "fp16", "fp32"]))


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "norm":
        m, n = case["rows"], case["width"]
        loud = 1.0 + 20.0 * (torch.rand(n, device="cuda", generator=gen) < 0.01)   # a residual stream has a few loud channels
        stream = torch.float32 if case["stream"] == "fp32" else dtype
        s.update(x=_normal(gen, (m, n), dtype), residual=(torch.randn((m, n), device="cuda", generator=gen) * loud).to(stream),
                 weight=(1.0 + 0.2 * torch.randn(n, device="cuda", generator=gen)).to(dtype),
                 bias=_normal(gen, (n,), dtype, 0.1) if case["bias"] else None,
                 post_weight=(1.0 + 0.2 * torch.randn(n, device="cuda", generator=gen)).to(dtype) if case["post"] else None,
                 gate={"none": None, "channel": lambda: _normal(gen, (n,), dtype), "token": lambda: _normal(gen, (m, n), dtype)}[case["gate"]])
        if s["gate"] is not None:
            s["gate"] = s["gate"]()
        return s
    if case["op"] == "moe":
        t, h, f, e = case["tokens"], case["width"], case["inner"], case["experts"]
        s.update(x=_normal(gen, (t, h), dtype), router=_normal(gen, (e, h), dtype, 1.5 / math.sqrt(h)),
                 gate_up=torch.empty((e, 2 * f, h), dtype=dtype, device="cuda"), down=torch.empty((e, h, f), dtype=dtype, device="cuda"),
                 bias=torch.randn(e, device="cuda", generator=gen) * 0.05 if case["biased"] else None)
        for i in range(e):
            s["gate_up"][i] = _normal(gen, (2 * f, h), dtype, 1.0 / math.sqrt(h))
            s["down"][i] = _normal(gen, (h, f), dtype, 1.0 / math.sqrt(f))
        if own:
            from shorokoo_b200 import decoder
            s["weights"] = decoder.MoEWeights(s["router"], s["gate_up"], s["down"], top_k=case["top_k"], scoring=case["scoring"],
                                              selection_bias=s["bias"], scale=case["scale"])
        return s
    m, n = case["rows"], case["vocab"]
    spread = 1.0 + 2.0 * torch.rand((m, 1), device="cuda", generator=gen)   # rows from flat to peaked
    logits = torch.randn((m, n), device="cuda", generator=gen) * spread
    ahead = torch.randint(0, n, (m, 20), device="cuda", generator=gen)      # a few tokens that the context asks for
    logits.scatter_add_(1, ahead, 15.0 * torch.rand((m, 20), device="cuda", generator=gen))
    if case["masked"]:
        logits.masked_fill_(torch.rand((m, n), device="cuda", generator=gen) < case["masked"], float("-inf"))
    s.update(logits=logits.to(dtype), uniform=torch.rand(m, device="cuda", generator=gen))
    each = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    for name, kind in each.items():
        s[name] = case[name]
        if case["mixed"]:
            value = torch.full((m,), case[name], dtype=kind, device="cuda")
            other = torch.rand(m, device="cuda", generator=gen)
            s[name] = {"temperature": lambda: torch.where(other < 0.2, torch.zeros_like(value), value * (0.5 + other)),
                       "top_k": lambda: torch.where(other < 0.3, torch.zeros_like(value), (value * (0.5 + other)).int()),
                       "top_p": lambda: torch.where(other < 0.3, torch.ones_like(value), value * (1.0 - 0.3 * other)),
                       "min_p": lambda: value * other}[name]()
    return s


def _normed(z, case, weight, bias):
    if case["kind"] == "layer":
        z = z - z.mean(-1, keepdim=True)
    y = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + 1e-5) * weight.float()
    return y if bias is None else y + bias.float()


def _norm(s):
    case = s["case"]
    t = s["x"].float()
    if case["post"]:
        t = _normed(t, case, s["post_weight"], None)
    t = t * case["scale"]
    if s["gate"] is not None:
        t = t * s["gate"].float()
    h = s["residual"].float() + t
    return _normed(h, case, s["weight"], s["bias"]).to(s["x"].dtype), h.to(s["residual"].dtype)


def _moe(s):
    case = s["case"]
    x, k, f = s["x"].float(), case["top_k"], case["inner"]
    logits = s["x"].double() @ s["router"].double().t()   # a choice: values next to the border count
    scores = torch.softmax(logits, 1) if case["scoring"] == "softmax" else torch.sigmoid(logits)
    order = scores if s["bias"] is None else scores + s["bias"].double()
    chosen = torch.sort(order, dim=1, descending=True, stable=True)[1][:, :k]
    share = torch.gather(scores, 1, chosen)
    share = (share / share.sum(1, keepdim=True) * case["scale"]).float()
    if x.shape[0] * k <= case["experts"]:   # each token's own experts
        wide = torch.einsum("tkfh,th->tkf", s["gate_up"][chosen].float(), x)
        hidden = wide[..., :f] * torch.sigmoid(wide[..., :f]) * wide[..., f:]
        return torch.einsum("tkhf,tkf->th", s["down"][chosen].float(), hidden * share[..., None]).to(s["x"].dtype)
    y = torch.zeros_like(x)
    for e in range(case["experts"]):
        wide = x @ s["gate_up"][e].float().t()
        hidden = wide[:, :f] * torch.sigmoid(wide[:, :f]) * wide[:, f:]
        y += (hidden * (share * (chosen == e)).sum(1, keepdim=True)) @ s["down"][e].float().t()
    return y.to(s["x"].dtype)


def _per_row(value, rows, kind=torch.float32):
    """A setting of each row in 64 bits, as the 32-bit value that it is given in."""
    if not isinstance(value, torch.Tensor):
        value = torch.full((rows,), value, dtype=kind, device="cuda")
    return value.double()[:, None]


def _sample(s):
    logits = s["logits"].double()
    m, n = logits.shape
    temperature, top_p, min_p = (_per_row(s[name], m) for name in ("temperature", "top_p", "min_p"))
    top_k = _per_row(s["top_k"], m, torch.int32)
    top_k = torch.where(top_k > 0, top_k, torch.full_like(top_k, n))
    x = logits - logits.amax(1, keepdim=True)
    weight = torch.where(x == 0, 1.0, torch.exp(x / temperature))   # temperature 0: the largest alone
    weight = torch.where(weight >= min_p, weight, 0.0)
    order = torch.sort(logits, dim=1, descending=True, stable=True)[1]
    ranked = torch.gather(weight, 1, order)
    ranked = torch.where(torch.arange(n, device="cuda") < top_k, ranked, 0.0)
    mass = torch.cumsum(ranked, 1)
    ranked = torch.where((mass - ranked < top_p * mass[:, -1:]) | (top_p >= 1), ranked, 0.0)
    kept = torch.zeros_like(weight).scatter_(1, order, ranked)
    mass = torch.cumsum(kept, 1)
    target = torch.where(temperature > 0, s["uniform"].double()[:, None], 0.0) * mass[:, -1:]
    return (mass <= target).sum(1).clamp(max=n - 1)


def run(state):
    s, case = state, state["case"]
    if own:
        from shorokoo_b200 import decoder
        if case["op"] == "norm":
            return decoder.residual_norm(s["x"], s["weight"], bias=s["bias"], residual=s["residual"], post_weight=s["post_weight"],
                                         gate=s["gate"], scale=case["scale"], kind=case["kind"], eps=1e-5)
        if case["op"] == "moe":
            return decoder.moe(s["x"], s["weights"])
        return decoder.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"norm": _norm, "moe": _moe, "sample": _sample}[case["op"]](s)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        m, n = case["rows"], case["width"]
        stream = 4 if case["stream"] == "fp32" else size
        vectors = 1 + case["post"] + case["bias"] + (case["gate"] == "channel")
        return {"bytes": m * n * (2 * size + 2 * stream + (size if case["gate"] == "token" else 0)) + vectors * n * size,
                "flops": m * n * (6 + 4 * case["post"])}
    if case["op"] == "moe":
        t, h, f, e, k = (case[name] for name in ("tokens", "width", "inner", "experts", "top_k"))
        read = e * (1.0 - (1.0 - k / e) ** t)   # experts that t tokens' random choices are expected to reach
        return {"bytes": int(read * 3 * h * f + e * h + 2 * t * h) * size, "flops": 6 * t * k * h * f + 2 * t * e * h}
    values = case["rows"] * case["vocab"]
    return {"bytes": values * size + 12 * case["rows"], "flops": 4 * values}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        def scaled(z, weight, bias):
            if case["kind"] == "layer":
                z = z - z.sum(1, keepdim=True) / z.shape[1]
            deviation = torch.sqrt(z.pow(2).sum(1, keepdim=True) / z.shape[1] + 1e-5)
            y = z / deviation * weight.double()
            return y if bias is None else y + bias.double()
        t = s["x"].double()
        if case["post"]:
            t = scaled(t, s["post_weight"], None)
        if s["gate"] is not None:
            t = t * s["gate"].double()
        h = torch.add(s["residual"].double(), t, alpha=case["scale"])
        return scaled(h, s["weight"], s["bias"]), h
    if case["op"] == "moe":
        t, f = case["tokens"], case["inner"]
        x = s["x"].double()
        logits = torch.einsum("th,eh->te", x, s["router"].double())
        rate = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True)) if case["scoring"] == "softmax" else 1.0 / (1.0 + torch.exp(-logits))
        by = rate if s["bias"] is None else rate + s["bias"].double()
        picked = [sorted(range(case["experts"]), key=lambda e: (-row[e], e))[: case["top_k"]] for row in by.tolist()]
        y = torch.zeros_like(x)
        for e in sorted({e for row in picked for e in row}):
            who = [i for i in range(t) if e in picked[i]]
            total = torch.stack([rate[i, picked[i]].sum() for i in who])
            gate = torch.mm(x[who], s["gate_up"][e, :f].double().t())
            up = torch.mm(x[who], s["gate_up"][e, f:].double().t())
            out = torch.mm(gate / (1.0 + torch.exp(-gate)) * up, s["down"][e].double().t())
            y[who] += out * (case["scale"] * rate[who, e] / total)[:, None]
        return y
    m = case["rows"]
    setting = {name: s[name].tolist() if case["mixed"] else [case[name]] * m for name in ("temperature", "top_k", "top_p", "min_p")}
    one = lambda v: float(torch.tensor(v, dtype=torch.float32))
    tokens = torch.empty(m, dtype=torch.int64)
    for i in range(m):
        row = s["logits"][i].double()
        best = row.max()
        if setting["temperature"][i] == 0:
            tokens[i] = torch.nonzero(row == best)[0, 0].cpu()
            continue
        weight = torch.exp((row - best) / one(setting["temperature"][i]))
        value, place = torch.sort(row, descending=True, stable=True)
        w = weight[place]
        keep = int((w >= one(setting["min_p"][i])).sum())
        if setting["top_k"][i] > 0:
            keep = min(keep, setting["top_k"][i])
        p = one(setting["top_p"][i])
        if p < 1:
            run_of = torch.cumsum(w[:keep], 0)
            keep = min(keep, int((run_of < p * run_of[-1]).sum()) + 1)
        place = torch.sort(place[:keep])[0]
        run_of = torch.cumsum(weight[place], 0)
        at = int(torch.searchsorted(run_of, s["uniform"][i].double() * run_of[-1], right=True))
        tokens[i] = place[min(at, keep - 1)].cpu()
    return tokens.cuda()
