"""Experts with 4-bit weights: the operators of a decode step or a prefill chunk whose weights are held in 4 bits with group scales.

Three operators: the choice of experts by scores with a balance bias (`skein_b200.ops.experts.route_balanced`), dense products
(`skein_b200.ops.int4.linear`, `swiglu_linear`) and the experts' products (`skein_b200.ops.int4.grouped_linear`). A weight is
W[f, k] = scale[f, k / group] (code[f, k] - zero[f, k / group]) with codes 0 .. 15, two to a byte (the even k in the low half), and a zero of 8
where none is given. `exact` computes the same in 64 bits from the definitions.
"""
import math

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # one user's token, 128 experts, softmax scores: nothing but latency
        {"name": "route_1_of_128", "op": "route", "rows": 1, "experts": 128, "top": 8, "groups": 1, "keep": 1, "score": "softmax", "bias": False,
         "scale": 1.0, "type": "fp32"},
        # a decode batch through the router of configs/barorax_9b_config.json, with a balance bias
        {"name": "route_64_groups", "op": "route", "rows": 64, "experts": 64, "top": 6, "groups": 8, "keep": 4, "score": "sigmoid", "bias": True,
         "scale": 2.0, "type": "fp32"},
        # a prefill chunk of 4096 tokens over many experts in groups
        {"name": "route_4096_of_256", "op": "route", "rows": 4096, "experts": 256, "top": 8, "groups": 8, "keep": 4, "score": "sigmoid", "bias": True,
         "scale": 2.5, "type": "fp32"},
        # the output projection of attention (configs/mistral_7b_config.json), one user
        {"name": "linear_1_out_proj", "op": "linear", "rows": 1, "features": 4096, "k": 4096, "group": 128, "zeros": False, "scales": "bf16",
         "pair": False, "out": "bf16"},
        # gate and up of configs/llama3_70b_config.json, one user: the longest stream of weights of a single token
        {"name": "linear_1_gate_up", "op": "linear", "rows": 1, "features": 28672, "k": 8192, "group": 128, "zeros": True, "scales": "fp16",
         "pair": True, "out": "bf16"},
        # logits of a small batch over the vocabulary of configs/qwen2_5_7b_config.json, kept in 32 bits
        {"name": "linear_13_logits", "op": "linear", "rows": 13, "features": 152064, "k": 3584, "group": 64, "zeros": True, "scales": "bf16",
         "pair": False, "out": "fp32"},
        # down projection of the headline decode batch (configs/mistral_7b_config.json)
        {"name": "linear_64_down", "op": "linear", "rows": 64, "features": 4096, "k": 14336, "group": 128, "zeros": False, "scales": "fp16",
         "pair": False, "out": "bf16"},
        # gate and up of a prompt of no round length (configs/qwen2_5_7b_config.json)
        {"name": "linear_1000_gate_up", "op": "linear", "rows": 1000, "features": 18944, "k": 3584, "group": 128, "zeros": False, "scales": "bf16",
         "pair": True, "out": "bf16"},
        # gate and up of the two experts of one token (configs/mixtral_8x7b_config.json)
        {"name": "experts_1_gate_up", "op": "experts", "rows": 1, "experts": 8, "top": 2, "features": 14336, "k": 4096, "group": 128, "zeros": False,
         "scales": "bf16", "pair": True, "gather": True},
        # the same for the headline decode batch: every expert has some of the 64 tokens
        {"name": "experts_64_gate_up", "op": "experts", "rows": 64, "experts": 8, "top": 2, "features": 14336, "k": 4096, "group": 128, "zeros": False,
         "scales": "bf16", "pair": True, "gather": True},
        # many small experts with few rows each, down projection (configs/barorax_9b_config.json)
        {"name": "experts_48_down_of_64", "op": "experts", "rows": 48, "experts": 64, "top": 6, "features": 2048, "k": 1408, "group": 64, "zeros": True,
         "scales": "fp16", "pair": False, "gather": False},
        # down projection of a prefill chunk of 2048 tokens (configs/mixtral_8x7b_config.json)
        {"name": "experts_2048_down", "op": "experts", "rows": 2048, "experts": 8, "top": 2, "features": 4096, "k": 14336, "group": 128, "zeros": False,
         "scales": "bf16", "pair": False, "gather": False},
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))      # noqa: E731
    op = rng.choice(("route", "linear", "linear", "experts", "experts"))
    if op == "route":
        groups, per = rng.choice((1, 1, 2, 4, 8)), rng.choice((4, 8, 15, 16, 24, 32))
        if groups == 1:
            per = spread(8, 256)
        experts, keep = groups * per, rng.randint(1, groups)
        rows = spread(1, 4096)
        return {"op": op, "rows": rows, "experts": experts, "top": rng.randint(1, min(8, keep * per)), "groups": groups, "keep": keep,
                "score": rng.choice(("softmax", "sigmoid")), "bias": rng.random() < 0.7, "scale": rng.choice((1.0, 2.5)),
                "type": rng.choice(("fp32", "fp32", "bf16"))}
    group, pair = rng.choice((32, 64, 128, 128)), rng.random() < 0.5
    k = group * max(1, spread(256, 14336) // group)
    features = spread(100, 20000)
    if rng.random() < 0.7:
        features = max(16, features // 16 * 16)
    c = {"op": op, "features": features, "k": k, "group": group, "zeros": rng.random() < 0.5, "scales": rng.choice(("bf16", "fp16")), "pair": pair}
    wide = features * (2 if pair else 1) * k
    if op == "linear":
        return {**c, "rows": min(spread(1, 1000), max(1, (1 << 36) // wide)), "out": "bf16" if pair else rng.choice(("bf16", "fp32"))}
    experts = min(rng.choice((4, 8, 16, 40, 64, 96)), max(2, (1 << 29) // wide))
    top = rng.randint(1, min(6, experts))
    return {**c, "rows": min(spread(1, 2048), max(1, (1 << 36) // (wide * top))), "experts": experts, "top": top, "gather": rng.random() < 0.6}


TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _weight(gen, lead, rows, case):
    """Codes, scales and zeros of a matrix as a quantiser of trained weights leaves them: codes around the zero, scales that differ by row and group."""
    k, group = case["k"], case["group"]
    codes = torch.empty(*lead, rows, k // 2, dtype=torch.uint8, device=DEV)
    flat = codes.view(-1, k // 2)
    step = max(1, (1 << 27) // k)
    for r0 in range(0, flat.shape[0], step):     # in parts: the normal numbers take eight times the codes' memory
        n = torch.randn(min(step, flat.shape[0] - r0), k, generator=gen, device=DEV)
        n = n.mul_(2.7).round_().add_(8).clamp_(0, 15).to(torch.uint8)
        flat[r0:r0 + step] = n[:, 0::2] | (n[:, 1::2] << 4)
    scale = torch.randn(*lead, rows, k // group, generator=gen, device=DEV).mul_(0.3).exp_().mul_(0.35 / math.sqrt(k)).to(TYPES[case["scales"]])
    zero = None
    if case["zeros"]:
        zero = torch.randint(6, 11, (*lead, rows, k // group), generator=gen, device=DEV, dtype=torch.uint8)
    return codes, scale, zero


def _rows(gen, rows, k):
    """Normed activations: unit size, a few channels that stand out."""
    x = torch.randn(rows, k, generator=gen, device=DEV)
    loud = torch.randint(0, k, (max(1, k // 256),), generator=gen, device=DEV)
    x[:, loud] *= 8
    return x.to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = dict(case)
    if case["op"] == "route":
        lean = torch.randn(case["experts"], generator=gen, device=DEV) * 0.5
        z = torch.randn(case["rows"], case["experts"], generator=gen, device=DEV) * 1.5 + lean
        s["logits"] = z.to(TYPES[case["type"]])
        s["bias_of"] = -0.1 * lean if case["bias"] else None
        return s
    lead = (case["experts"],) if case["op"] == "experts" else ()
    s["codes"], s["scale"], s["zero"] = _weight(gen, lead, case["features"] * (2 if case["pair"] else 1), case)
    if case["op"] == "linear":
        s["x"] = _rows(gen, case["rows"], case["k"])
    else:
        # experts that are liked more and less, `top` different ones for a token; the layout that a router leaves
        like = torch.randn(case["rows"], case["experts"], generator=gen, device=DEV) + 0.7 * torch.randn(case["experts"], generator=gen, device=DEV)
        ids = like.argsort(1, descending=True)[:, :case["top"]].reshape(-1)
        order = ids.argsort(stable=True)
        count = torch.bincount(ids, minlength=case["experts"])
        s["counts"] = count.to(torch.int32)
        s["offsets"] = torch.cat((count.new_zeros(1), count.cumsum(0))).to(torch.int32)
        s["expert_of"] = ids[order]
        s["place"] = torch.arange(ids.numel(), device=DEV) - s["offsets"].long()[s["expert_of"]]
        s["most"] = int(count.max())
        s["src_row"] = (order // case["top"]).to(torch.int32) if case["gather"] else None
        s["x"] = _rows(gen, case["rows"] if case["gather"] else ids.numel(), case["k"])
    if own:
        from skein_b200.ops import int4
        s["weight"] = int4.pack_weight(s["codes"], s["scale"], s["zero"], pair=case["pair"])
    return s


def _dequant(s):
    codes, scale = s["codes"], s["scale"].float()
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    zero = s["zero"].float() if s["zero"] is not None else 8.0 * torch.ones_like(scale)
    shape = q.shape
    q = q.unflatten(-1, (scale.shape[-1], s["group"]))
    return ((q - zero[..., None]) * scale[..., None]).view(shape)


def _route(s):
    """The choice and the expert-sorted layout. Scores in 64 bits: two experts next to each other differ by less than a 32-bit exponential's error."""
    T, E, top = s["rows"], s["experts"], s["top"]
    z = s["logits"].double()
    z = torch.where(z == z, z, torch.full_like(z, -3e38)).clamp(-3e38, 3e38)
    if s["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-z))
    else:
        e = torch.exp(z - z.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    choice = score if s["bias_of"] is None else score + s["bias_of"].double()
    if s["keep"] < s["groups"]:
        per = E // s["groups"]
        best = choice.view(T, s["groups"], per).sort(dim=2, descending=True).values[:, :, :min(2, per)].sum(2)
        rank = best.sort(dim=1, descending=True, stable=True).indices[:, :s["keep"]]
        kept = torch.zeros(T, s["groups"], dtype=torch.bool, device=z.device).scatter_(1, rank, True)
        choice = torch.where(kept[:, :, None].expand(T, s["groups"], per).reshape(T, E), choice, torch.full_like(choice, -math.inf))
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :top]
    w = score.gather(1, ids)
    w = w * s["scale"] / (w.sum(1, keepdim=True) + 1e-20)
    flat = ids.reshape(-1)
    order = flat.sort(stable=True).indices
    count = (flat[:, None] == torch.arange(E, device=z.device)).sum(0)
    offsets = torch.cat((count.new_zeros(1), count.cumsum(0)))
    row_of = torch.empty_like(order).scatter_(0, order, torch.arange(T * top, device=z.device))
    whole = [v.to(torch.int32) for v in (ids, count, offsets, row_of, order // top)]
    return whole[0], w.float(), whole[1], whole[2], whole[3], whole[4]


def _pair(y):
    g, u = y.chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def run(s):
    if own:
        if s["op"] == "route":
            from skein_b200.ops import experts
            return experts.route_balanced(s["logits"], s["top"], bias=s["bias_of"], groups=s["groups"], keep=s["keep"], score=s["score"], group_best=2,
                                          renorm=True, scale=s["scale"])
        from skein_b200.ops import int4
        if s["op"] == "experts":
            return int4.grouped_linear(s["x"], s["weight"], s["counts"], s["offsets"], swiglu=s["pair"], src_row=s["src_row"])
        if s["pair"]:
            return int4.swiglu_linear(s["x"], s["weight"])
        return int4.linear(s["x"], s["weight"], out_f32=s["out"] == "fp32")
    if s["op"] == "route":
        return _route(s)
    w, x = _dequant(s), s["x"].float()
    if s["op"] == "linear":
        y = x @ w.t()
    else:
        if s["src_row"] is not None:
            x = x[s["src_row"].long()]
        padded = torch.zeros(s["experts"], s["most"], s["k"], device=x.device)
        padded[s["expert_of"], s["place"]] = x
        y = torch.bmm(padded, w.transpose(1, 2))[s["expert_of"], s["place"]]
    y = _pair(y) if s["pair"] else y
    return y if s.get("out") == "fp32" else y.to(torch.bfloat16)


def work(case):
    rows, top = case["rows"], case.get("top", 1)
    if case["op"] == "route":
        E = case["experts"]
        size = 2 if case["type"] == "bf16" else 4
        return {"bytes": rows * E * size + (4 * E if case["bias"] else 0) + rows * top * 16 + 4 * (2 * E + 1), "flops": rows * E * (8 + top)}
    f, k = case["features"] * (2 if case["pair"] else 1), case["k"]
    matrix = f * k / 2 + f * (k // case["group"]) * (3 if case["zeros"] else 2)
    if case["op"] == "linear":
        return {"bytes": matrix + 2 * rows * k + (4 if case["out"] == "fp32" else 2) * rows * case["features"], "flops": 2 * rows * f * k}
    touched = case["experts"] * (1 - (1 - top / case["experts"]) ** rows)        # experts that some token goes to, where all are liked alike
    read = rows if case["gather"] else rows * top
    return {"bytes": matrix * touched + 2 * read * k + 2 * rows * top * case["features"], "flops": 2 * rows * top * f * k}


def exact(case, seed):
    """From the definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    x = s["x"].double()
    out = torch.empty(s["src_row"].numel() if s.get("src_row") is not None else x.shape[0], case["features"], dtype=torch.float64, device=DEV)
    ends = [(None, 0, out.shape[0])]
    if case["op"] == "experts":
        off = s["offsets"].tolist()
        ends = [(e, off[e], off[e + 1]) for e in range(case["experts"])]
    for e, r0, r1 in ends:
        if r0 == r1:
            continue
        rows = x[r0:r1] if s.get("src_row") is None else x[s["src_row"][r0:r1].long()]
        codes, scale = (s["codes"], s["scale"]) if e is None else (s["codes"][e], s["scale"][e])
        zero = None if s["zero"] is None else s["zero"] if e is None else s["zero"][e]
        step = max(1, (1 << 27) // case["k"])
        parts = []
        for f0 in range(0, codes.shape[0], step):
            c = codes[f0:f0 + step]
            w = torch.empty(c.shape[0], case["k"], dtype=torch.float64, device=DEV)
            w[:, 0::2], w[:, 1::2] = (c % 16).double(), (c // 16).double()
            w -= 8.0 if zero is None else zero[f0:f0 + step].double().repeat_interleave(case["group"], 1)
            w *= scale[f0:f0 + step].double().repeat_interleave(case["group"], 1)
            parts.append(torch.matmul(rows, w.t()))
        y = torch.cat(parts, 1)
        if case["pair"]:
            g, u = y[:, :case["features"]], y[:, case["features"]:]
            y = g * torch.sigmoid(g) * u
        out[r0:r1] = y
    return out


def _exact_route(s):
    """Token by token on the host."""
    if s["rows"] * s["experts"] > 1 << 21:
        return None
    z = s["logits"].double().cpu()
    bias = s["bias_of"].double().cpu() if s["bias_of"] is not None else torch.zeros(s["experts"], dtype=torch.float64)
    score = torch.sigmoid(z) if s["score"] == "sigmoid" else torch.softmax(z, 1)
    rows, weights = [], []
    per = s["experts"] // s["groups"]
    for sc, ch in zip(score.tolist(), (score + bias).tolist()):
        worth = [sum(sorted(ch[g * per:(g + 1) * per], reverse=True)[:2]) for g in range(s["groups"])]
        kept = set(sorted(range(s["groups"]), key=lambda g: (-worth[g], g))[:s["keep"]])
        mine = sorted((e for e in range(s["experts"]) if e // per in kept), key=lambda e: (-ch[e], e))[:s["top"]]
        tot = sum(sc[e] for e in mine) + 1e-20
        rows.append(mine)
        weights.append([sc[e] * s["scale"] / tot for e in mine])
    of = [[] for _ in range(s["experts"])]
    for t, mine in enumerate(rows):
        for j, e in enumerate(mine):
            of[e].append((t, j))
    ends, row_of, src = [0], torch.zeros(s["rows"], s["top"], dtype=torch.int32), []
    for pairs in of:
        for t, j in pairs:
            row_of[t, j] = len(src)
            src.append(t)
        ends.append(len(src))
    whole = lambda v: torch.tensor(v, dtype=torch.int32)      # noqa: E731
    return (whole(rows), torch.tensor(weights, dtype=torch.float64), whole([len(p) for p in of]), whole(ends), row_of.reshape(-1), whole(src))
