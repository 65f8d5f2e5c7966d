"""The operators around the products of a feed-forward block: inputs, a pass, its minimum work and the result in 64 bits.

  layernorm           rows minus their mean, over their deviation, times a scale plus a shift; the statistics are kept for the gradient
  layernorm_backward  the gradients of the rows, the scale and the shift
  route               a router's scores and the experts that each token goes to, with their weights
  experts             a block of experts for the few tokens of a decoding step, gate, up and down products with the weighted sum

Everything lies on the GPU when a pass begins.  `own` chooses between the library's entry points and elementary torch operations in 32 bits
(64 where the order of scores is at stake).
"""
import math
import random

import torch

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
_BLOCK = 128
_E4M3_MOST = 448.0
_EPS = 1e-5


def _layernorm(rows, axis, dtype, params="same", backward=False):
    """params: type of scale and shift, "f32" or that of the rows."""
    return {"op": "layernorm_backward" if backward else "layernorm", "rows": rows, "axis": axis, "dtype": dtype,
            "params": dtype if params == "same" else params}


def _route(tokens, experts, hidden, top, dtype, router="f32", score="softmax", masked=0):
    """masked: experts that a bias of minus infinity takes out; sigmoid scores have a small bias for the choice anyway."""
    return {"op": "route", "tokens": tokens, "experts": experts, "hidden": hidden, "top": top, "dtype": dtype, "router": router, "score": score,
            "masked": masked}


def _experts(tokens, experts, busy, top, hidden, ffn, dtype, weights="same", idle=0):
    """busy: experts that have tokens; idle: tokens at the end without experts, as a padded batch has them."""
    return {"op": "experts", "tokens": tokens, "experts": experts, "busy": busy, "top": top, "hidden": hidden, "ffn": ffn, "dtype": dtype,
            "weights": dtype if weights == "same" else weights, "idle": idle}


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # the next tokens of eight sequences: one short launch
        named("layernorm_token", _layernorm(8, 4096, "bf16")),
        # a long batch of prompts
        named("layernorm_prompt", _layernorm(16384, 8192, "bf16")),
        # rows on odd boundaries
        named("layernorm_odd", _layernorm(9001, 4099, "f16", params="f32")),
        # a training step's batch of sequences
        named("layernorm_backward_batch", _layernorm(16384, 4096, "bf16", params="f32", backward=True)),
        # a few rows of fp32, a ragged length
        named("layernorm_backward_ragged", _layernorm(333, 2050, "f32", backward=True)),
        # one token to eight experts of sixty-four
        named("route_token", _route(1, 64, 4096, 8, "bf16")),
        # a batch of tokens, many experts, sigmoid scores with a bias for the choice, some experts taken out
        named("route_batch", _route(61, 128, 2048, 8, "bf16", score="sigmoid", masked=3)),
        # a prompt's tokens
        named("route_prompt", _route(4096, 64, 4096, 4, "f16", router="f16")),
        # one token, small experts: latency
        named("experts_small", _experts(1, 8, 2, 2, 1024, 704, "f16")),
        # one token to eight experts of sixty-four
        named("experts_token", _experts(1, 64, 8, 8, 4096, 2048, "bf16")),
        # a batch of tokens in 8 bits, every other expert busy, a padded end as a captured graph has it
        named("experts_batch8", _experts(16, 64, 50, 8, 4096, 2048, "bf16", weights="e4m3", idle=2)),
        # the largest batch, nearly all experts busy
        named("experts_batch", _experts(64, 128, 120, 8, 2048, 768, "bf16")),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step):
    """Spread over the logarithm of [lo, hi]: half are whole numbers of `step`, a quarter powers of two, the rest multiples of 8."""
    v, how = _log(rng, lo, hi), rng.random()
    if how < 0.5:
        return max(step, v // step * step)
    return 1 << (v.bit_length() - 1) if how < 0.75 else max(8, v // 8 * 8)


def draw(rng):
    kind = rng.choice(["layernorm", "layernorm_odd", "backward", "backward_odd", "route_token", "route_batch", "route_prompt", "experts_token",
                       "experts_batch", "experts_batch"])
    half = rng.choice(["bf16", "f16"])
    if kind in ("layernorm", "backward"):
        dtype = rng.choice(["bf16", "f16", "f32"])
        axis = _size(rng, 256, 16384, 640)
        rows = _log(rng, 1, max(1, min(65536, (1 << 26) // axis)))
        return _layernorm(rows, axis, dtype, params=rng.choice(["same", "f32"]), backward=kind == "backward")
    if kind in ("layernorm_odd", "backward_odd"):
        return _layernorm(_log(rng, 1, 4096), _log(rng, 33, 9001), rng.choice(["bf16", "f16", "f32"]), params=rng.choice(["same", "f32"]),
                          backward=kind == "backward_odd")
    experts = rng.choice([8, 16, 32, 60, 64, 128])
    top = rng.randint(1, min(8, experts))
    if kind.startswith("route"):
        tokens = {"route_token": rng.randint(1, 4), "route_batch": _log(rng, 5, 128), "route_prompt": _log(rng, 129, 4096)}[kind]
        score = rng.choice(["softmax", "sigmoid"])
        return _route(tokens, experts, _size(rng, 256, 4096 if tokens > 128 else 8192, 640), top, half, router=rng.choice(["f32", half]), score=score,
                      masked=rng.randint(0, experts - top) // 4)
    weights = rng.choice(["same", "same", "e4m3"])
    many = experts > 32
    hidden, ffn = _size(rng, 512, 4096 if many else 8192, 640), _size(rng, 256, 2048 if many else 4096, 640)
    tokens = rng.randint(1, 4) if kind == "experts_token" else _log(rng, 2, 64)
    idle = rng.choice([0, 0, 1]) if tokens > 1 else 0
    most = min(experts, (tokens - idle) * top)
    return _experts(tokens, experts, rng.randint(max(top, most // 2), most), top, hidden, ffn, half, weights=weights, idle=idle)


# ---- inputs


def _activations(gen, rows, k, dtype):
    """Normal values about a mean of their own, a few columns of them much larger than the others, as activations have them."""
    x = torch.empty((rows, k), dtype=dtype, device="cuda")
    loud = 1.0 + 20.0 * (torch.rand(k, generator=gen, device="cuda") < 0.002)
    step = max(1, (1 << 27) // k)
    for r in range(0, rows, step):
        part = x[r:r + step]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda").mul_(loud).add_(0.25))
    return x


def _pitch(k):
    """Rows of 8-bit values begin on 16-byte boundaries."""
    return -(-k // 16) * 16


def _blocks_up(scale, n, k):
    """A value for each 128 x 128 block at every element of it."""
    return scale.repeat_interleave(_BLOCK, dim=-2)[..., :n, :].repeat_interleave(_BLOCK, dim=-1)[..., :k]


def _weights(gen, groups, n, k, kind):
    """Weights [groups, n, k] and, for e4m3, their scales [groups, n / 128, k / 128]."""
    if kind != "e4m3":
        w = torch.empty((groups, n, k), dtype=_TORCH[kind], device="cuda")
        for g in range(groups):
            w[g].copy_(torch.randn((n, k), generator=gen, device="cuda").mul_(k ** -0.5))
        return w, None
    q = torch.zeros((groups, n, _pitch(k)), dtype=torch.float8_e4m3fn, device="cuda")
    nb, kb = -(-n // _BLOCK), -(-k // _BLOCK)
    scale = torch.empty((groups, nb, kb), dtype=torch.float32, device="cuda")
    for g in range(groups):
        w = torch.zeros((nb * _BLOCK, kb * _BLOCK), dtype=torch.float32, device="cuda")
        w[:n, :k] = torch.randn((n, k), generator=gen, device="cuda").mul_(k ** -0.5)
        scale[g] = w.view(nb, _BLOCK, kb, _BLOCK).abs().amax(dim=(1, 3)) / _E4M3_MOST
        q[g, :, :k] = (w[:n, :k] / _blocks_up(scale[g], n, k)).to(torch.float8_e4m3fn)
    return q[:, :, :k], scale


def _choices(case, seed):
    """Experts of each token: together exactly the busy ones, the first of them more often than the others; -1 for tokens without any."""
    chance = random.Random(seed)
    names = chance.sample(range(case["experts"]), case["busy"])
    top, tokens, rows = case["top"], case["tokens"] - case["idle"], []
    for t in range(tokens):
        if t * top < case["busy"]:
            rows.append([names[(t * top + j) % case["busy"]] for j in range(top)])
        else:
            left, row = list(range(case["busy"])), []
            for _ in range(top):
                row.append(left.pop(min(int(len(left) * chance.random() ** 1.3), len(left) - 1)))
            rows.append([names[i] for i in row])
    chance.shuffle(rows)
    return rows + [[-1] * top] * case["idle"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"].startswith("layernorm"):
        rows, axis, dtype, params = case["rows"], case["axis"], _TORCH[case["dtype"]], _TORCH[case["params"]]
        s["x"] = _activations(gen, rows, axis, dtype)
        s["scale"] = torch.randn(axis, generator=gen, device="cuda").mul_(0.1).add_(1.0).to(params)
        s["shift"] = torch.randn(axis, generator=gen, device="cuda").mul_(0.1).to(params)
        if case["op"] == "layernorm_backward":
            s["dy"] = torch.empty((rows, axis), dtype=dtype, device="cuda")
            step = max(1, (1 << 27) // axis)
            for r in range(0, rows, step):
                s["dy"][r:r + step].copy_(torch.randn((min(step, rows - r), axis), generator=gen, device="cuda"))
            s["mean"] = torch.empty(rows, device="cuda")
            s["variance"] = torch.empty(rows, device="cuda")
            for r in range(0, rows, step):
                v = s["x"][r:r + step].double()
                s["mean"][r:r + step] = v.mean(dim=1)
                s["variance"][r:r + step] = v.var(dim=1, unbiased=False)
        return s
    if case["op"] == "route":
        experts, hidden = case["experts"], case["hidden"]
        s["x"] = _activations(gen, case["tokens"], hidden, _TORCH[case["dtype"]])
        s["router"] = torch.randn((experts, hidden), generator=gen, device="cuda").mul_(hidden ** -0.5).to(_TORCH[case["router"]])
        s["bias"] = None
        if case["masked"] or case["score"] == "sigmoid":
            s["bias"] = torch.zeros(experts, device="cuda")
            if case["score"] == "sigmoid":
                s["bias"].copy_(torch.randn(experts, generator=gen, device="cuda").mul_(0.05))
            s["bias"][torch.randperm(experts, generator=gen, device="cuda")[:case["masked"]]] = -math.inf
        return s
    tokens, top, hidden, ffn = case["tokens"], case["top"], case["hidden"], case["ffn"]
    rows = _choices(case, seed)
    s["chosen"] = rows
    s["ids"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
    p = torch.rand((tokens, top), generator=gen, device="cuda").add_(0.1)
    s["p"] = p / p.sum(dim=1, keepdim=True)
    s["x"] = _activations(gen, tokens, hidden, _TORCH[case["dtype"]])
    s["gate_up"], s["gate_up_scale"] = _weights(gen, case["experts"], 2 * ffn, hidden, case["weights"])
    s["down"], s["down_scale"] = _weights(gen, case["experts"], hidden, ffn, case["weights"])
    return s


# ---- a pass in elementary operations


def _plain_layernorm(s):
    x = s["x"].float()
    mean = x.mean(dim=1)
    d = x - mean[:, None]
    variance = (d * d).mean(dim=1)
    y = d / torch.sqrt(variance + _EPS)[:, None] * s["scale"].float() + s["shift"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean, "variance": variance}


def _plain_layernorm_backward(s):
    r = 1.0 / torch.sqrt(s["variance"] + _EPS)
    xh = (s["x"].float() - s["mean"][:, None]) * r[:, None]
    dy = s["dy"].float()
    g = dy * s["scale"].float()
    dx = (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True)) * r[:, None]
    kind = s["scale"].dtype
    return {"dx": dx.to(s["x"].dtype), "dscale": (dy * xh).sum(dim=0).to(kind), "dshift": dy.sum(dim=0).to(kind)}


def _plain_route(s, case):
    """In 64 bits: the choice depends on the order of the scores."""
    logits = s["x"].double() @ s["router"].double().t()
    out = torch.zeros_like(logits, dtype=torch.bool) if s["bias"] is None else torch.isneginf(s["bias"])[None, :].expand_as(logits)
    if case["score"] == "softmax":
        logits = torch.where(out, torch.full_like(logits, -math.inf), logits)
        e = torch.exp(logits - logits.amax(dim=1, keepdim=True))
        score = e / e.sum(dim=1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-logits))
    key = score if s["bias"] is None else score + s["bias"].double()
    ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :case["top"]]
    p = torch.gather(score, 1, ids)
    p = p / p.sum(dim=1, keepdim=True)
    return {"weights": p.float(), "ids": ids.to(torch.int32)}


def _by_expert(s):
    """Expert -> its tokens and the places of the expert in their lists."""
    lists = {}
    for t, row in enumerate(s["chosen"]):
        for j, e in enumerate(row):
            if e >= 0:
                lists.setdefault(e, []).append((t, j))
    return sorted(lists.items())


def _wide(w, scale, e):
    v = w[e].float()
    return v if scale is None else v * _blocks_up(scale[e], *v.shape)


def _plain_experts(s, case):
    x = s["x"].float()
    y = torch.zeros((case["tokens"], case["hidden"]), device="cuda")
    for e, pairs in _by_expert(s):
        tokens, places = [t for t, _ in pairs], [j for _, j in pairs]
        h = x[tokens] @ _wide(s["gate_up"], s["gate_up_scale"], e).t()
        gate, up = h[:, :case["ffn"]], h[:, case["ffn"]:]
        h = gate / (1.0 + torch.exp(-gate)) * up
        y[tokens] += (h @ _wide(s["down"], s["down_scale"], e).t()) * s["p"][tokens, places][:, None]
    return y.to(s["x"].dtype)


# ---- the same pass through the library


def _own_plan(s, case):
    """What a program makes once per layer and batch size: the descriptor, the buffers for results and the workspace."""
    import kudnn_b200 as kb
    code = {"f32": kb.F32, "f16": kb.F16, "bf16": kb.BF16, "e4m3": kb.E4M3}
    if case["op"].startswith("layernorm"):
        rows, axis = case["rows"], case["axis"]
        desc = kb.make_layernorm_desc(rows, axis, code[case["dtype"]], param_dtype=code[case["params"]], has_scale=True, has_shift=True, eps=_EPS)
        if case["op"] == "layernorm":
            out = {"y": torch.empty_like(s["x"]), "mean": torch.empty(rows, device="cuda"), "variance": torch.empty(rows, device="cuda")}
            return lambda: kb.layernorm(desc, s["x"], out["y"], s["scale"], s["shift"], out["mean"], out["variance"]), out
        out = {"dx": torch.empty_like(s["x"]), "dscale": torch.empty_like(s["scale"]), "dshift": torch.empty_like(s["scale"])}
        size = kb.layernorm_backward_workspace(desc)
        space = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
        return lambda: kb.layernorm_backward(desc, s["x"], s["dy"], s["scale"], s["mean"], s["variance"], out["dx"], out["dscale"], out["dshift"],
                                             space, size), out
    if case["op"] == "route":
        tokens, top = case["tokens"], case["top"]
        desc = kb.make_route_desc(tokens, case["experts"], case["hidden"], top, code[case["dtype"]], router_dtype=code[case["router"]],
                                  score=kb.SCORE_SIGMOID if case["score"] == "sigmoid" else kb.SCORE_SOFTMAX)
        out = {"weights": torch.empty((tokens, top), device="cuda"), "ids": torch.empty((tokens, top), dtype=torch.int32, device="cuda")}
        return lambda: kb.route(desc, s["x"], s["router"], out["weights"], out["ids"], s["bias"]), out
    tokens, hidden, ffn = case["tokens"], case["hidden"], case["ffn"]
    desc = kb.make_experts_desc(tokens, hidden, ffn, case["experts"], case["top"], code[case["dtype"]], weight_dtype=code[case["weights"]],
                                gate_up_strides=s["gate_up"].stride(), down_strides=s["down"].stride())
    y = torch.empty_like(s["x"])
    size = kb.experts_workspace(desc)
    space = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    return lambda: kb.experts(desc, s["x"], s["p"], s["ids"], s["gate_up"], s["down"], y, space, size, s["gate_up_scale"], s["down_scale"]), y


def run(state):
    s, case = state, state["case"]
    if own:
        if "call" not in s:
            s["call"], s["out"] = _own_plan(s, case)
        s["call"]()
        return s["out"]
    if case["op"] == "layernorm":
        return _plain_layernorm(s)
    if case["op"] == "layernorm_backward":
        return _plain_layernorm_backward(s)
    if case["op"] == "route":
        return _plain_route(s, case)
    return _plain_experts(s, case)


# ---- what a pass cannot do without, and what it computes


def work(case):
    if case["op"].startswith("layernorm"):
        rows, axis, e = case["rows"], case["axis"], _SIZE[case["dtype"]]
        backward = case["op"] == "layernorm_backward"
        return {"bytes": rows * axis * e * (3 if backward else 2) + 8 * rows + axis * _SIZE[case["params"]] * (3 if backward else 2),
                "flops": rows * axis * (13 if backward else 7)}
    if case["op"] == "route":
        tokens, experts, hidden = case["tokens"], case["experts"], case["hidden"]
        return {"bytes": tokens * hidden * _SIZE[case["dtype"]] + experts * hidden * _SIZE[case["router"]] + 8 * tokens * case["top"],
                "flops": 2 * tokens * experts * hidden}
    tokens, top, hidden, ffn, kind = case["tokens"], case["top"], case["hidden"], case["ffn"], case["weights"]
    size = 3 * case["busy"] * hidden * ffn * _SIZE[kind] + 2 * tokens * hidden * _SIZE[case["dtype"]] + 8 * tokens * top
    if kind == "e4m3":
        kb, fb = -(-hidden // _BLOCK), -(-ffn // _BLOCK)
        size += 4 * case["busy"] * (-(-2 * ffn // _BLOCK) * kb + kb * fb)
    return {"bytes": size, "flops": 6 * (tokens - case["idle"]) * top * hidden * ffn}


# ---- the result in 64 bits


def _exact_layernorm(s, case):
    rows, axis = case["rows"], case["axis"]
    out = {"y": torch.empty((rows, axis), dtype=torch.float64, device="cuda"), "mean": torch.empty(rows, dtype=torch.float64, device="cuda"),
           "variance": torch.empty(rows, dtype=torch.float64, device="cuda")}
    step = max(1, (1 << 26) // axis)
    for r in range(0, rows, step):
        x = s["x"][r:r + step].double()
        out["variance"][r:r + step], out["mean"][r:r + step] = torch.var_mean(x, dim=1, correction=0)
        out["y"][r:r + step] = torch.nn.functional.layer_norm(x, (axis,), s["scale"].double(), s["shift"].double(), _EPS)
    return out


def _exact_layernorm_backward(s, case):
    rows, axis = case["rows"], case["axis"]
    out = {"dx": torch.empty((rows, axis), dtype=torch.float64, device="cuda"), "dscale": torch.zeros(axis, dtype=torch.float64, device="cuda"),
           "dshift": torch.zeros(axis, dtype=torch.float64, device="cuda")}
    step = max(1, (1 << 25) // axis)
    for r in range(0, rows, step):
        x, dy = s["x"][r:r + step].double(), s["dy"][r:r + step].double()
        deviation = (s["variance"][r:r + step].double() + _EPS).sqrt()[:, None]
        normal = (x - s["mean"][r:r + step].double()[:, None]) / deviation
        out["dscale"] += torch.einsum("ra,ra->a", dy, normal)
        out["dshift"] += dy.sum(dim=0)
        dn = dy * s["scale"].double()
        along = torch.einsum("ra,ra->r", dn, normal)[:, None] / axis
        out["dx"][r:r + step] = (dn - dn.sum(dim=1, keepdim=True) / axis - normal * along) / deviation
    return out


def _exact_route(s, case):
    logits = torch.einsum("th,eh->te", s["x"].double(), s["router"].double())
    bias = torch.zeros(case["experts"], dtype=torch.float64, device="cuda") if s["bias"] is None else s["bias"].double()
    if case["score"] == "softmax":
        score = torch.softmax(logits.masked_fill(torch.isinf(bias), -math.inf), dim=1)
    else:
        score = torch.sigmoid(logits)
    key, ids, weights = score + bias, [], []
    every = torch.arange(case["experts"], device="cuda")
    for _ in range(case["top"]):
        most = key.amax(dim=1, keepdim=True)
        at = torch.where(key == most, every, case["experts"]).amin(dim=1, keepdim=True)
        ids.append(at)
        weights.append(score.gather(1, at))
        key = key.scatter(1, at, -math.inf)
    weights = torch.cat(weights, dim=1)
    return {"weights": weights / weights.sum(dim=1, keepdim=True), "ids": torch.cat(ids, dim=1)}


def _exact_experts(s, case):
    ffn = case["ffn"]
    y = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device="cuda")

    def weight(name, e):
        w = s[name][e].double()
        return w if s[name + "_scale"] is None else w * _blocks_up(s[name + "_scale"][e].double(), *w.shape)

    for e in sorted({e for row in s["chosen"] for e in row if e >= 0}):
        mine = (s["ids"] == e)
        share = (s["p"].double() * mine).sum(dim=1)
        tokens = mine.any(dim=1).nonzero()[:, 0]
        both = torch.einsum("th,fh->tf", s["x"][tokens].double(), weight("gate_up", e))
        h = torch.nn.functional.silu(both[:, :ffn]) * both[:, ffn:]
        y.index_add_(0, tokens, torch.einsum("tf,hf->th", h, weight("down", e)) * share[tokens][:, None])
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layernorm":
        return _exact_layernorm(s, case)
    if case["op"] == "layernorm_backward":
        return _exact_layernorm_backward(s, case)
    if case["op"] == "route":
        return _exact_route(s, case)
    return _exact_experts(s, case)
