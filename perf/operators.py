"""Timed cases of the decoder-layer operators on device tensors, with their plain forms.

Four operators that one layer of a language model runs per step when it answers from a paged cache:

  linear_w4        y = x W^T (+ bias), W held in 4 bits with one scale (and zero point) per group of inputs
  rotary           rotary positions of a tensor of heads (and the adjoint, which a gradient needs)
  paged_append     rotary positions of a step's q and k, and k and v written into the cache's pages
  paged_attention  attention of each sequence's new tokens over its pages

``run`` computes the plain form in elementary torch operations, or, with ``own`` set, calls the
package. Sizes are generic ones, besides the 12 heads of 64 that this repository's ViT-B has.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token through a square projection: the smallest product of a single-stream decode, all latency
        dict(name="w4_square_row", op="w4", rows=1, out=4096, inp=4096, group=128, zeros=False, bias=False, dtype="bf16"),
        # one token through a wide feed-forward projection, larger than L2 together with the next layers': memory bandwidth
        dict(name="w4_wide_row", op="w4", rows=1, out=22016, inp=8192, group=32, zeros=True, bias=False, dtype="fp16"),
        # a small batch of sequences decoded together, an output width and batch that fill no tile
        dict(name="w4_batch", op="w4", rows=13, out=11000, inp=4096, group=64, zeros=True, bias=True, dtype="bf16"),
        # a prompt's queries at positions far out, scaled for a long context
        dict(name="rotary_prompt", op="rotary", tokens=4099, heads=32, dim=128, rotary=128, interleaved=False, scaling="by_parts",
             far=1000000, inverse=False, dtype="bf16"),
        # the gradient of interleaved rotary positions over half of ViT-B's head width, in 32 bits
        dict(name="rotary_gradient", op="rotary", tokens=2049, heads=12, dim=64, rotary=32, interleaved=True, scaling="none",
             far=4096, inverse=True, dtype="fp32"),
        # a decode step of 32 sequences: one token each into a long cache
        dict(name="append_step", op="append", batch=32, new=1, context=8000, ragged=3, heads=32, kv_heads=8, dim=128, page=16,
             rotary=128, interleaved=False, scaling="linear", dtype="bf16"),
        # chunks of several prompts at once, interleaved positions on half of each head
        dict(name="append_chunks", op="append", batch=5, new=1500, context=6000, ragged=4, heads=32, kv_heads=8, dim=128, page=64,
             rotary=64, interleaved=True, scaling="none", dtype="fp16"),
        # a single stream's token over a short context: latency
        dict(name="attend_one", op="attend", batch=1, new=1, context=1500, ragged=0, heads=32, kv_heads=8, dim=128, page=16, window=0,
             dtype="bf16"),
        # a decode step of 48 sequences of unlike lengths
        dict(name="attend_step", op="attend", batch=48, new=1, context=8000, ragged=7, heads=32, kv_heads=8, dim=128, page=16, window=0,
             dtype="bf16"),
        # two streams far into a long document, few key heads: the context has to be split over the card
        dict(name="attend_long", op="attend", batch=2, new=1, context=100003, ragged=0, heads=32, kv_heads=4, dim=128, page=64, window=0,
             dtype="fp16"),
        # a chunk of a long prompt over what the cache already holds
        dict(name="attend_chunk", op="attend", batch=1, new=2000, context=40009, ragged=0, heads=32, kv_heads=8, dim=128, page=64,
             window=0, dtype="bf16"),
        # whole prompts of unlike lengths, heads as ViT-B has them, a sliding window
        dict(name="attend_prompts", op="attend", batch=4, new=4000, context=4000, ragged=5, heads=12, kv_heads=12, dim=64, page=32,
             window=1024, dtype="fp16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["w4", "rotary", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "w4":
        group = rng.choice([32, 64, 128, 256])
        return dict(op=op, rows=_log(rng, 1, 40), out=_log(rng, 256, 20000), inp=8 * _log(rng, 32, 1024) + rng.choice([0, 0, 0, 2, 6]), group=group,
                    zeros=rng.random() < 0.5, bias=rng.random() < 0.5, dtype=dtype)
    interleaved, scaling = rng.random() < 0.5, rng.choice(["none", "linear", "ntk", "by_parts"])
    dim = rng.choice([64, 80, 96, 128])
    rotary = rng.choice([dim, dim // 2])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    if op == "rotary":
        return dict(op=op, tokens=_log(rng, 1, 6000), heads=min(heads, 32), dim=dim, rotary=rotary, interleaved=interleaved, scaling=scaling,
                    far=_log(rng, 1000, 1000000), inverse=rng.random() < 0.3, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if op == "append":
        new = rng.choice([1, 1, _log(rng, 2, 1500)])
        return dict(op=op, batch=_log(rng, 1, 64 if new < 16 else 6), new=new, context=new + _log(rng, 1, 8000), ragged=rng.randrange(1, 1000),
                    heads=heads, kv_heads=kv_heads, dim=dim, page=page, rotary=rotary, interleaved=interleaved, scaling=scaling, dtype=dtype)
    new = rng.choice([1, 1, rng.randrange(2, 9), _log(rng, 16, 2000)])
    if new == 1:
        batch = _log(rng, 1, 64)
        context = _log(rng, 64, min(100000, 400000 // batch))
    else:
        batch = _log(rng, 1, 32 if new < 9 else 4)
        context = new + _log(rng, 1, max(2, min(40000, int(1.2e9 / (batch * new * heads)), 200000 // batch)))
    return dict(op=op, batch=batch, new=new, context=context, ragged=rng.randrange(0, 1000), heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), dtype=dtype)


def _lengths(case):
    """New tokens and context (the new ones among it) of each sequence; ``ragged`` 0 gives all the largest."""
    new, context = [case["new"]] * case["batch"], [case["context"]] * case["batch"]
    if case["ragged"]:
        rng = random.Random(case["ragged"])
        new = [rng.randint(max(1, n // 4), n) for n in new]
        context = [max(n, rng.randint(c // 8, c)) for n, c in zip(new, context)]
        new[0], context[0] = case["new"], case["context"]
    return new, context


def _frequencies(case):
    """Radians per position of each pair, and the factor on the rotated values, of the case's scaling."""
    r, base = case["rotary"], 10000.0
    pairs = [2.0 * i / r for i in range(r // 2)]
    if case["scaling"] == "linear":
        return [base ** -p / 4.0 for p in pairs], 1.0
    if case["scaling"] == "ntk":
        base *= 4.0 ** (r / (r - 2.0))
    freqs = [base ** -p for p in pairs]
    if case["scaling"] != "by_parts":
        return freqs, 1.0
    mixed = []
    for f in freqs:
        share = min(1.0, max(0.0, (4096 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)))
        mixed.append(f * (share + (1.0 - share) / 8.0))
    return mixed, 0.1 * math.log(8.0) + 1.0


def _table(case):
    """The package's table of the case's rotary frequencies."""
    from shorokoo_b200 import decoder
    more = {"none": {}, "linear": dict(factor=4.0), "ntk": dict(factor=4.0), "by_parts": dict(factor=8.0, original_context=4096)}
    return decoder.RotaryTable(case["rotary"], 10000.0, interleaved=case["interleaved"], scaling=case["scaling"], device="cuda",
                               **more[case["scaling"]])


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "w4":
        n, k, g = case["out"], case["inp"], case["group"]
        groups = -(-k // g)
        s = dict(x=_normal(gen, (case["rows"], k), dtype),
                 packed=torch.randint(0, 256, (n, k // 2), device="cuda", generator=gen, dtype=torch.uint8),
                 scales=((torch.rand((n, groups), device="cuda", generator=gen) + 0.5) * (0.25 / math.sqrt(k))).to(dtype),
                 zeros=torch.randint(5, 11, (n, groups), device="cuda", generator=gen, dtype=torch.uint8) if case["zeros"] else None,
                 bias=_normal(gen, (n,), dtype, 0.1) if case["bias"] else None)
        if own:
            from shorokoo_b200 import decoder
            s["weights"] = decoder.W4Weights(s["packed"], s["scales"], s["zeros"], in_features=k, group_size=g)
        return dict(s, case=case)
    if case["op"] == "rotary":
        freqs, magnitude = _frequencies(case)
        s = dict(x=_normal(gen, (case["tokens"], case["heads"], case["dim"]), dtype), magnitude=magnitude,
                 positions=torch.randint(0, case["far"], (case["tokens"],), device="cuda", generator=gen),
                 freqs=torch.tensor(freqs, dtype=torch.float64, device="cuda"))
        if own:
            s["table"] = _table(case)
        return dict(s, case=case)
    new, context = _lengths(case)
    page, kv, d = case["page"], case["kv_heads"], case["dim"]
    width = -(-max(context) // page)
    pages = sum(-(-c // page) for c in context) + 3
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros((case["batch"], width), dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(context):
        table[b, : -(-c // page)] = order[at: at - (-c // page)]
        at += -(-c // page)
    tokens = sum(new)
    s = dict(q=_normal(gen, (tokens, case["heads"], d), dtype), k_pages=_normal(gen, (pages, page, kv, d), dtype),
             v_pages=_normal(gen, (pages, page, kv, d), dtype), page_table=table,
             context=torch.tensor(context, dtype=torch.int32, device="cuda"),
             starts=torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda"),
             most_new=max(new), most_context=max(context))
    if case["op"] == "append":
        freqs, s["magnitude"] = _frequencies(case)
        s.update(k=_normal(gen, (tokens, kv, d), dtype), v=_normal(gen, (tokens, kv, d), dtype),
                 freqs=torch.tensor(freqs, dtype=torch.float64, device="cuda"))
    if own:
        from shorokoo_b200 import decoder
        s["cache"] = decoder.PagedCache(s["k_pages"], s["v_pages"], s["page_table"], s["context"])
        if case["op"] == "append":
            s["table"] = _table(case)
    return dict(s, case=case)


def _rotate(x, positions, freqs, magnitude, interleaved, inverse=False):
    angle = positions.double()[:, None] * freqs
    cos, sin = (f(angle).float()[:, None] * magnitude for f in (torch.cos, torch.sin))
    if inverse:
        sin = -sin
    r = 2 * freqs.numel()
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., : r // 2], y[..., r // 2: r])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, y[..., r:]), -1).to(x.dtype)


def _of_rows(s):
    """The sequence and the position of each new token."""
    row = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(s["starts"], row, right=True, out_int32=True).long() - 1
    last = s["context"][b] - (s["starts"][b + 1] - s["starts"][b])
    return b, row - s["starts"][b] + last


def _linear(s):
    p, k, g = s["packed"], s["x"].shape[1], s["case"]["group"]
    w = torch.stack((p & 15, p >> 4), -1).flatten(1).float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(g, 1)[:, :k]
    w = (w - zero) * s["scales"].float().repeat_interleave(g, 1)[:, :k]
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _append(s):
    b, pos = _of_rows(s)
    q = _rotate(s["q"], pos, s["freqs"], s["magnitude"], s["case"]["interleaved"])
    k = _rotate(s["k"], pos, s["freqs"], s["magnitude"], s["case"]["interleaved"])
    size = s["k_pages"].shape[1]
    at = s["page_table"][b, pos // size].long(), pos % size
    s["k_pages"][at] = k
    s["v_pages"][at] = s["v"]
    return q, s["k_pages"], s["v_pages"]


def _attend(s):
    q, heads, dim = s["q"], s["q"].shape[1], s["q"].shape[2]
    size, kv = s["k_pages"].shape[1], s["k_pages"].shape[2]
    n, length, many = s["most_new"], s["most_context"], s["context"].numel()
    key = torch.arange(length, device="cuda")
    pages = s["page_table"].long()[:, key // size]
    k = s["k_pages"][pages, key % size].float().permute(0, 2, 3, 1)
    v = s["v_pages"][pages, key % size].float().permute(0, 2, 1, 3)
    count = (s["starts"][1:] - s["starts"][:-1])[:, None]
    i = torch.arange(n, device="cuda")
    rows = (s["starts"][:-1, None] + i).clamp(max=q.shape[0] - 1)
    qs = q[rows].float().view(many, n, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(many, kv, -1, dim)
    scores = (qs @ k).mul_(1.0 / math.sqrt(dim)).view(many, kv, heads // kv, n, length)
    pos = (s["context"][:, None] - count + i)[:, None, None, :, None]
    seen = key <= pos
    if s["case"]["window"]:
        seen = seen & (key > pos - s["case"]["window"])
    scores.masked_fill_(~seen, float("-inf"))
    scores -= scores.amax(-1, keepdim=True).clamp(min=-1e30)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    y = (scores.view(many, kv, -1, length) @ v).view(many, kv, -1, n, dim) / total
    b, p = _of_rows(s)
    at = p - (s["context"][b] - count[b, 0])
    return y.permute(0, 3, 1, 2, 4).reshape(many, n, heads, dim)[b, at].to(q.dtype)


def run(state):
    op = state["case"]["op"]
    if own:
        from shorokoo_b200 import decoder
        if op == "w4":
            return decoder.linear_w4(state["x"], state["weights"], state["bias"])
        if op == "rotary":
            return decoder.rotary(state["x"], state["positions"], state["table"], inverse=state["case"]["inverse"])
        if op == "append":
            q = decoder.paged_append(state["cache"], state["k"], state["v"], state["starts"], q=state["q"], table=state["table"])
            return q, state["k_pages"], state["v_pages"]
        return decoder.paged_attention(state["cache"], state["q"], state["starts"], window=state["case"]["window"])
    if op == "w4":
        return _linear(state)
    if op == "rotary":
        return _rotate(state["x"], state["positions"], state["freqs"], state["magnitude"], state["case"]["interleaved"],
                       state["case"]["inverse"])
    return _append(state) if op == "append" else _attend(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "w4":
        m, n, k = case["rows"], case["out"], case["inp"]
        groups = -(-k // case["group"])
        held = n * k // 2 + n * groups * size + (n * groups // 2 if case["zeros"] else 0) + (n * size if case["bias"] else 0)
        return {"bytes": held + (m * k + m * n) * size, "flops": 2 * m * n * k}
    if case["op"] == "rotary":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * values * size + 8 * case["tokens"], "flops": 3 * values * case["rotary"] // case["dim"]}
    new, context = _lengths(case)
    heads, kv, d, window = case["heads"], case["kv_heads"], case["dim"], case.get("window", 0)
    if case["op"] == "append":
        values = sum(new) * (heads + 2 * kv) * d
        return {"bytes": 2 * values * size + 4 * sum(new), "flops": 3 * sum(new) * (heads + kv) * case["rotary"]}
    keys = pairs = 0
    for n, c in zip(new, context):
        keys += min(c, window + n - 1) if window else c
        short = min(n, max(0, window - 1 - (c - n))) if window else n  # the rows that see less than a window
        pairs += short * (c - n + 1) + short * (short - 1) // 2 + (n - short) * window
    return {"bytes": (2 * sum(new) * heads * d + 2 * keys * kv * d) * size + 4 * keys // case["page"], "flops": 2 * d * heads * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "w4":
        n, k = case["out"], case["inp"]
        codes = torch.empty((n, k), dtype=torch.float64, device="cuda")
        codes[:, 0::2] = (s["packed"] % 16).double()
        codes[:, 1::2] = (s["packed"] // 16).double()
        for j in range(s["scales"].shape[1]):
            at = slice(j * case["group"], min(k, (j + 1) * case["group"]))
            codes[:, at] -= 8.0 if s["zeros"] is None else s["zeros"][:, j: j + 1].double()
            codes[:, at] *= s["scales"][:, j: j + 1].double()
        y = torch.einsum("mk,nk->mn", s["x"].double(), codes)
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "rotary":
        return _turned(case, s["x"], s["positions"], -1.0 if case["inverse"] else 1.0)
    new, context = _lengths(case)
    at = 0
    if case["op"] == "append":
        positions = torch.cat([torch.arange(c - n, c) for n, c in zip(new, context)]).cuda()
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        k, size = _turned(case, s["k"], positions, 1.0), case["page"]
        for b, (n, c) in enumerate(zip(new, context)):
            where = torch.arange(c - n, c, device="cuda")
            slot = s["page_table"][b].long()[torch.div(where, size, rounding_mode="floor")] * size + where % size
            k_pages.view(-1, *k.shape[1:])[slot] = k[at: at + n]
            v_pages.view(-1, *k.shape[1:])[slot] = s["v"][at: at + n].double()
            at += n
        return _turned(case, s["q"], positions, 1.0), k_pages, v_pages
    y = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for b, (n, c) in enumerate(zip(new, context)):
        held = s["page_table"][b, : -(-c // case["page"])].long()
        far = torch.arange(c, device="cuda")[None, :] - torch.arange(c - n, c, device="cuda")[:, None]
        hidden = far > 0
        if case["window"]:
            hidden |= far <= -case["window"]
        for h in range(case["heads"]):
            k = s["k_pages"][held, :, h // group].reshape(-1, case["dim"])[:c].double()
            v = s["v_pages"][held, :, h // group].reshape(-1, case["dim"])[:c].double()
            logits = torch.mm(s["q"][at: at + n, h].double(), k.t()) / case["dim"] ** 0.5
            y[at: at + n, h] = torch.mm(torch.softmax(logits.masked_fill(hidden, -math.inf), 1), v)
        at += n
    return y


def _turned(case, x, positions, sign):
    """Each pair of x as a complex number, times magnitude * e^(i sign angle), in 64 bits."""
    freqs, magnitude = _frequencies(case)
    r = case["rotary"]
    angle = sign * positions.double()[:, None, None] * torch.tensor(freqs, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, magnitude), angle)
    y = x.double().clone()
    if case["interleaved"]:
        z = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) * turn
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    else:
        z = torch.complex(y[..., : r // 2], y[..., r // 2: r]) * turn
        y[..., : r // 2], y[..., r // 2: r] = z.real, z.imag
    return y
