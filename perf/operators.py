"""The measured cases of two operators of the routed-MoE sublayer:

* ``route``: the choice of experts from router logits, with softmax or sigmoid
  scores, a bias that balances the load, groups of experts, top-k and
  renormalised weights (``Context.route_scores``);
* ``lora``: a Q4 projection shared by all tokens beside the low-rank adapters
  of many requests, one adapter or none per token (``Context.q4_gemv_lora``).

``run`` computes the plain form with elementary torch operations, or, where
``own`` is true, makes the calls of the framework.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---------------------------------------------------------------- cases

def listed():
    route = dict(op="route", groups=1, keep=1, pair=False, bias=False, renorm=True, scale=1.0,
                 masked=0, pad=0)
    lora = dict(op="lora", ragged=False, pad=0)
    return [
        # one decoded token on the router of the sublayer's own configuration (512 experts, top-10)
        dict(route, name="route 1x512 softmax", tokens=1, experts=512, k=10, score="softmax", dtype="fp32"),
        # a decode batch on a grouped sigmoid router with a balance bias
        dict(route, name="route 64x256 groups", tokens=64, experts=256, k=8, score="sigmoid", dtype="bf16",
             groups=8, keep=4, pair=True, bias=True, scale=2.5),
        # a chunk of a prompt where an eighth of the experts is masked out (not on this host), 128 experts, top-8
        dict(route, name="route 777x128 masked", tokens=777, experts=128, k=8, score="softmax", dtype="fp16",
             masked=16),
        # the 4096-token prefill of the sublayer's own configuration
        dict(route, name="route 4096x512 softmax", tokens=4096, experts=512, k=10, score="softmax", dtype="fp32"),
        # an odd number of prompt tokens, 160 experts in groups of 20 by their best score, rows with padding
        dict(route, name="route 8191x160 padded", tokens=8191, experts=160, k=6, score="softmax", dtype="bf16",
             groups=8, keep=3, renorm=False, scale=16.0, pad=8),
        # the largest: a long prompt on the grouped sigmoid router
        dict(route, name="route 16384x256 groups", tokens=16384, experts=256, k=8, score="sigmoid", dtype="fp32",
             groups=8, keep=4, pair=True, bias=True, scale=2.5),
        # one decoded token on an expert-sized gate projection
        dict(lora, name="lora 1 2048-512", tokens=1, cin=2048, cout=512, rank=16, adapters=8, requests=1, dtype="fp32"),
        # a decode batch: every token is another request, most with an adapter of their own
        dict(lora, name="lora 32 2048-2048", tokens=32, cin=2048, cout=2048, rank=16, adapters=32, requests=32,
             dtype="bf16"),
        # a large decode batch over adapters of different ranks on a down projection
        dict(lora, name="lora 256 512-2048", tokens=256, cin=512, cout=2048, rank=32, adapters=64, requests=256,
             dtype="fp16", ragged=True),
        # a few prompt chunks in fp32 with an odd total, rows with padding
        dict(lora, name="lora 777 2048-768", tokens=777, cin=2048, cout=768, rank=8, adapters=16, requests=5,
             dtype="fp32", pad=4),
        # a 4096-token prefill of eight requests
        dict(lora, name="lora 4096 2048-2048", tokens=4096, cin=2048, cout=2048, rank=16, adapters=8, requests=8,
             dtype="bf16"),
        # the largest: fp32 rows, rank 64, an odd number of tokens
        dict(lora, name="lora 6001 2048-2048", tokens=6001, cin=2048, cout=2048, rank=64, adapters=12, requests=12,
             dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        groups = rng.choice([1, 1, 4, 8, 16])
        size = _log_int(rng, 8 if groups == 1 else 2, 1024 // groups)
        experts = groups * size
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(16, keep * size))
        case = dict(op="route", experts=experts, groups=groups, keep=keep, k=k, pair=rng.random() < 0.5,
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                    renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]),
                    masked=rng.choice([0, 0, experts // 8]), pad=rng.choice([0, 0, 1, 8]),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]))
        case["tokens"] = _log_int(rng, 1, min(16384, 16384 * 256 // experts))
        return case
    cin, cout = 64 * _log_int(rng, 4, 64), _log_int(rng, 64, 4096)
    most = 6001 * 2048 * 2048 // (cin * cout)
    tokens = _log_int(rng, 1, min(6001, most))
    return dict(op="lora", tokens=tokens, cin=cin, cout=cout, rank=_log_int(rng, 4, 64),
                adapters=_log_int(rng, 1, 48), requests=min(tokens, _log_int(rng, 1, 256)),
                dtype=rng.choice(["fp32", "bf16", "fp16"]), ragged=rng.random() < 0.3,
                pad=rng.choice([0, 0, 1, 8]))


def work(case):
    T = case["tokens"]
    if case["op"] == "route":
        E, k = case["experts"], case["k"]
        return {"bytes": T * E * _BYTES[case["dtype"]] + (4 * E if case["bias"] else 0) + T * (8 * k + 4),
                "flops": 4 * T * E}
    cin, cout, r = case["cin"], case["cout"], case["rank"]
    used = min(case["adapters"], case["requests"])
    return {"bytes": cout * (cin // 2 + cin // 64 * 4) + T * (cin + cout) * _BYTES[case["dtype"]] + 4 * T
            + used * r * (cin + cout) * 2,
            "flops": 2 * T * cin * cout + 2 * T * r * (cin + cout)}


# ---------------------------------------------------------------- inputs

def _padded(values, pad):
    """`values` as the first columns of rows that are `pad` values longer."""
    if not pad:
        return values
    wide = torch.zeros(values.shape[0], values.shape[1] + pad, dtype=values.dtype, device=values.device)
    wide[:, :values.shape[1]] = values
    return wide[:, :values.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    f = dict(device="cuda", generator=g)
    T, dt = case["tokens"], _DTYPES[case["dtype"]]
    s = dict(case=dict(case))
    if case["op"] == "route":
        E, k = case["experts"], case["k"]
        logits = 1.5 * torch.randn(T, E, **f) + 0.7 * torch.randn(E, **f)
        logits = logits.to(dt)
        if case["masked"]:
            logits[:, torch.randperm(E, **f)[:case["masked"]]] = -math.inf
        s["logits"] = _padded(logits, case["pad"])
        s["bias"] = 0.1 * torch.randn(E, **f) if case["bias"] else None
        s["ids"] = torch.empty(T, k, dtype=torch.int32, device="cuda")
        s["weights"] = torch.empty(T, k, device="cuda")
        s["mass"] = torch.empty(T, device="cuda")
        return s
    cin, cout, r, n = case["cin"], case["cout"], case["rank"], case["adapters"]
    G = cin // 64
    # MLX-affine Q4 of a weight of about N(0, 0.02): eight nibbles per word, bf16 scale and bias per 64
    s["packed"] = torch.randint(-2**31, 2**31, (cout, cin // 8), dtype=torch.int32, **f)
    scale = 0.008 * (0.5 + torch.rand(cout, G, **f))
    s["scales"] = scale.to(torch.bfloat16)
    s["biases"] = (-7.5 * scale + 0.002 * torch.randn(cout, G, **f)).to(torch.bfloat16)
    x = torch.randn(T, cin, **f)
    x[:, :: 97] *= 8  # a few channels with large activations
    s["x"] = _padded(x.to(dt), case["pad"])
    half = torch.float16 if dt == torch.float16 else torch.bfloat16
    s["a"] = (torch.randn(n, r, cin, **f) / math.sqrt(cin)).to(half)
    s["b"] = (0.05 * torch.randn(n, cout, r, **f)).to(half)
    s["gain"] = 0.5 + 1.5 * torch.rand(n, **f)
    s["ranks"] = torch.randint(1, r + 1, (n,), dtype=torch.int32, **f) if case["ragged"] else None
    # each request is a run of tokens with one adapter; an eighth of the requests has none
    R = case["requests"]
    of_request = torch.randint(0, n, (R,), dtype=torch.int32, **f)
    of_request[torch.rand(R, **f) < 0.125] = -1
    s["adapter"] = of_request[torch.arange(T, device="cuda") * R // T].contiguous()
    s["y"] = _padded(torch.empty(T, cout, dtype=dt, device="cuda"), case["pad"])
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_route(s):
    c = s["case"]
    logits, k, G = s["logits"], c["k"], c["groups"]
    T, E = logits.shape
    masked = logits <= torch.finfo(logits.dtype).min
    l = logits.double().masked_fill(masked, -math.inf)
    if c["score"] == "softmax":
        e = torch.exp(l - l.max(1, keepdim=True).values)
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-l))
    choice = score if s["bias"] is None else score + s["bias"].double()
    choice = choice.masked_fill(masked, -math.inf)
    if G > 1:
        best = choice.view(T, G, E // G).sort(dim=2, descending=True).values
        value = best[:, :, 0]
        if c["pair"] and E // G > 1:
            second = best[:, :, 1]
            value = value + second.masked_fill(second == -math.inf, 0)
        order = value.sort(dim=1, descending=True, stable=True).indices
        kept = torch.zeros(T, G, dtype=torch.bool, device=logits.device)
        kept.scatter_(1, order[:, :c["keep"]], True)
        choice = choice.view(T, G, E // G).masked_fill(~kept[:, :, None], -math.inf).view(T, E)
    top = choice.sort(dim=1, descending=True, stable=True)
    ids = top.indices[:, :k]
    w = score.gather(1, ids).masked_fill(top.values[:, :k] == -math.inf, 0)
    mass = w.sum(1)
    if c["renorm"]:
        w = w / mass[:, None]
    return ids.int(), (w * c["scale"]).float(), mass.float()


def _plain_lora(s):
    c = s["case"]
    T, cin, cout, r, n = (c[v] for v in ("tokens", "cin", "cout", "rank", "adapters"))
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    q = ((s["packed"][:, :, None] >> shifts) & 15).view(cout, cin // 64, 64).float()
    w = (q * s["scales"].float()[:, :, None] + s["biases"].float()[:, :, None]).view(cout, cin)
    x = s["x"].float()
    y = x @ w.T
    a, b, ad = s["a"].float(), s["b"].float(), s["adapter"].long()
    gain = s["gain"]
    if s["ranks"] is not None:  # the first ranks[i] rows of an adapter are its own
        gain = gain[:, None] * (torch.arange(r, device="cuda") < s["ranks"][:, None])
    else:
        gain = gain[:, None].expand(n, r)
    has = (ad >= 0)[:, None]
    if T <= n:  # few tokens: each one's adapter
        at = ad.clamp(min=0)
        v = torch.bmm(a[at], x[:, :, None])[:, :, 0] * gain[at] * has
        y = y + torch.bmm(b[at], v[:, :, None])[:, :, 0]
    else:  # many: every adapter's products, each token's own kept
        v = (x @ a.view(n * r, cin).T).view(T, n, r) * gain
        v = v * (ad[:, None] == torch.arange(n, device="cuda"))[:, :, None]
        y = y + v.view(T, n * r) @ b.transpose(1, 2).reshape(n * r, cout)
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------- the framework's calls

_context = None


def _own(s):
    """The program's context, made once, and the descriptions that go with this state's tensors."""
    global _context
    at = os.path.join(os.getcwd(), "orbi-streammoe_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import osm_b200 as osm

    if _context is None:
        _context = osm.Context(torch.cuda.current_device(), max_tokens=64)
        _context.set_stream(torch.cuda.current_stream().cuda_stream)
    c = s["case"]
    if c["op"] == "route":
        s["routing"] = osm.Routing(c["experts"], c["k"], score=c["score"], bias=s["bias"], groups=c["groups"],
                                   top_groups=c["keep"], group_score="top2" if c["pair"] else "max",
                                   renormalize=c["renorm"], scale=c["scale"])
    else:
        s["lora"] = osm.Lora(s["a"], s["b"], scale=s["gain"], ranks=s["ranks"])
    s["ctx"] = _context
    return _context


def run(state):
    s = state
    c = s["case"]
    if not own:
        return _plain_route(s) if c["op"] == "route" else _plain_lora(s)
    ctx = s.get("ctx") or _own(s)
    if c["op"] == "route":
        ctx.route_scores(s["logits"], s["routing"], s["ids"], s["weights"], mass=s["mass"])
        return s["ids"], s["weights"], s["mass"]
    ctx.q4_gemv_lora(s["packed"], s["scales"], s["biases"], c["cout"], c["cin"], s["x"], c["tokens"], s["y"],
                     lora=s["lora"], adapter=s["adapter"])
    return s["y"]


# ---------------------------------------------------------------- from the definition, in 64 bits

def _exact_route(s):
    """Expert by expert, as the definition says: keep the best groups, then take the best expert k times."""
    c = s["case"]
    l = s["logits"].double()
    T, E = l.shape
    G, N = c["groups"], E // c["groups"]
    there = s["logits"] > torch.finfo(s["logits"].dtype).min
    if c["score"] == "softmax":
        score = torch.softmax(torch.where(there, l, -math.inf), 1)
    else:
        score = torch.sigmoid(l)
    choice = score + (s["bias"].double() if s["bias"] is not None else 0)
    index = torch.arange(E, device=l.device).expand(T, E)
    group = torch.arange(G, device=l.device).expand(T, G)
    if G > 1:
        value = torch.empty(T, G, dtype=torch.float64, device=l.device)
        for i in range(G):
            part = torch.where(there, choice, -math.inf)[:, i * N:(i + 1) * N]
            first = part.max(1)
            value[:, i] = first.values
            if c["pair"] and N > 1:
                rest = part.scatter(1, first.indices[:, None], -math.inf).max(1).values
                value[:, i] += torch.where(rest > -math.inf, rest, 0.0)
        kept = torch.zeros(T, G, dtype=torch.bool, device=l.device)
        for _ in range(c["keep"]):
            left = torch.where(kept, math.nan, value)
            m = torch.where(kept, -math.inf, value).max(1, keepdim=True).values
            kept.scatter_(1, torch.where(left == m, group, G - 1).min(1, keepdim=True).values, True)
        there = there & kept.repeat_interleave(N, 1)
    weights = torch.zeros(T, c["k"], dtype=torch.float64, device=l.device)
    taken = ~there
    for j in range(c["k"]):
        left = torch.where(taken, -math.inf, choice)
        m = left.max(1, keepdim=True).values
        at = torch.where((left == m) & ~taken, index, E).min(1, keepdim=True).values
        some = at < E
        at = at.clamp(max=E - 1)
        weights[:, j] = torch.where(some, score.gather(1, at), 0.0)[:, 0]
        taken = taken.scatter(1, at, True)
    mass = weights.sum(1)
    if c["renorm"]:
        weights = weights / mass[:, None]
    return None, weights * c["scale"], mass


def _exact_lora(s):
    """Nibble by nibble and adapter by adapter."""
    c = s["case"]
    cin, cout = c["cin"], c["cout"]
    w = torch.empty(cout, cin, dtype=torch.float64, device="cuda")
    word = s["packed"].long() & 0xFFFFFFFF
    for i in range(8):
        w[:, i::8] = ((word >> (4 * i)) & 15).double()
    w = w * s["scales"].double().repeat_interleave(64, 1) + s["biases"].double().repeat_interleave(64, 1)
    x = s["x"].double()
    y = torch.matmul(x, w.t())
    for i in range(c["adapters"]):
        rows = (s["adapter"] == i).nonzero()[:, 0]
        if rows.numel():
            r = c["rank"] if s["ranks"] is None else int(s["ranks"][i])
            low = torch.matmul(x[rows], s["a"][i, :r].double().t())
            y[rows] += s["gain"][i].double() * torch.matmul(low, s["b"][i, :, :r].double().t())
    return y


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_route(s) if case["op"] == "route" else _exact_lora(s)
