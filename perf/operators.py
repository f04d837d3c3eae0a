"""Measured calls of the operators around block-scaled 8-bit experts, each in two forms.

``own`` false: the operator in elementary torch operations, in 32 bits (the scores a selection ranks
by in 64), rounded once at the end.  ``own`` true: the calls a user makes of ``sparse_amd``.

route     scores of T tokens over E experts (softmax or sigmoid of the router's logits), a bias that
          takes part in the selection only, group limit, top-k, renormalised and scaled weights.
quantise  rows to float8_e4m3fn with one power-of-two scale for each run of 128 values: the smallest
          2^s with max|x| <= 448 * 2^s, s >= -120.
linear    y = x W^T with x quantised as above in the call and W held as float8_e4m3fn with one fp32
          scale for each 128 x 128 block.
experts   the SwiGLU expert FFN on such weights: routed rows in permuted order (expert, flat index),
          each times its route weight, and the shared expert's rows; the intermediate is quantised
          like the input.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128
LOWEST = -120      # smallest exponent of a scale
TOP = 448.0        # largest value of float8_e4m3fn


# ------------------------------------------------------------------------------------------ cases
def _route(name, T, E, K, score, bias, n_group, topk_group, group_score, renorm, scale, dtype, out):
    return {"name": name, "op": "route", "T": T, "E": E, "K": K, "score": score, "bias": bias, "n_group": n_group,
            "topk_group": topk_group, "group_score": group_score, "renorm": renorm, "scale": scale, "dtype": dtype,
            "out": out}


def _quantise(name, T, K, dtype):
    return {"name": name, "op": "quantise", "T": T, "K": K, "dtype": dtype}


def _linear(name, T, K, N, dtype, pow2):
    return {"name": name, "op": "linear", "T": T, "K": K, "N": N, "dtype": dtype, "pow2": pow2}


def _experts(name, T, H, E, I, K, Is, gate, dtype, pow2):
    return {"name": name, "op": "experts", "T": T, "H": H, "E": E, "I": I, "K": K, "Is": Is, "gate": gate,
            "dtype": dtype, "pow2": pow2}


def listed():
    return [
        # a decode step of one sequence through a gate balanced by a bias: latency is all there is
        _route("route one token", 1, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5, "fp32", "bf16"),
        # a prompt chunk through the same gate
        _route("route chunk", 4096, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5, "fp32", "bf16"),
        # a ragged batch through a softmax gate with a bias and no groups
        _route("route softmax ragged", 1537, 60, 4, "softmax", True, 1, 1, "max", False, 1.0, "bf16", "fp32"),
        # a few half-precision rows whose length ends inside a block
        _quantise("quantise ragged", 777, 1400, "fp16"),
        # a prompt chunk's rows as wide as a shared expert's intermediate
        _quantise("quantise chunk", 4096, 5632, "bf16"),
        # one token through a shared expert's projection: a stream of weights
        _linear("linear one token", 1, 2048, 5632, "bf16", False),
        # odd sizes throughout, weights from a checkpoint whose scales are any fp32 number
        _linear("linear odd", 333, 1000, 1418, "fp16", False),
        # a prompt chunk through the same projection as the first
        _linear("linear chunk", 4096, 2048, 5632, "bf16", True),
        # decode steps of one and of eight sequences
        _experts("experts one token", 1, 2048, 60, 1408, 4, 5632, True, "bf16", True),
        _experts("experts eight tokens", 8, 2048, 60, 1408, 4, 5632, True, "bf16", False),
        # a short prompt, an intermediate that ends inside a block, no shared expert
        _experts("experts short prompt", 301, 1024, 16, 704, 3, 0, False, "fp16", False),
        # a prompt chunk
        _experts("experts chunk", 4096, 2048, 64, 1408, 6, 2816, False, "bf16", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "quantise", "linear", "experts"])
    if op == "route":
        n_group = rng.choice([1, 1, 2, 4, 8])
        E = n_group * _log_int(rng, 8, 256 // n_group)
        topk_group = rng.randint(1, n_group)
        K = rng.randint(1, min(8, topk_group * (E // n_group)))
        c = _route("", _log_int(rng, 1, 8192), E, K, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.7, n_group,
                   topk_group, rng.choice(["max", "top2"]), rng.random() < 0.5, rng.choice([1.0, 2.5, 16.0]),
                   rng.choice(["bf16", "fp16", "fp32"]), rng.choice(["bf16", "fp16", "fp32"]))
    elif op == "quantise":
        c = _quantise("", _log_int(rng, 1, 8192), _log_int(rng, 17, 5632), rng.choice(["bf16", "fp16", "fp32"]))
    elif op == "linear":
        c = _linear("", _log_int(rng, 1, 4096), _log_int(rng, 33, 5632), _log_int(rng, 17, 5632),
                    rng.choice(["bf16", "fp16"]), rng.random() < 0.5)
    else:
        E = rng.choice([8, 16, 60, 64])
        Is = rng.choice([0, 64 * _log_int(rng, 4, 44)])
        c = _experts("", _log_int(rng, 1, 4096), 64 * _log_int(rng, 8, 32), E, 64 * _log_int(rng, 4, 22),
                     rng.randint(1, 6), Is, bool(Is) and rng.random() < 0.5, rng.choice(["bf16", "fp16"]),
                     rng.random() < 0.5)
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _hidden(g, T, H, dtype):
    """Rows as they leave a norm: unit normal, a few channels an order of magnitude louder."""
    loud = torch.exp(0.5 * _randn(g, H)) * torch.where(torch.rand(H, generator=g, device="cuda") < 0.01, 10.0, 1.0)
    return (_randn(g, T, H) * loud).to(DTYPES[dtype])


def _weight(g, N, K, pow2):
    """A weight as a checkpoint stores it: 8-bit values and a scale for each 128 x 128 block, a power
    of two or the block's largest value over 448."""
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    w = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
    w[:N, :K] = _randn(g, N, K) * 0.02
    w = w.view(nb, BLOCK, kb, BLOCK)
    scale = w.abs().amax(dim=(1, 3)).clamp_min(1e-12) / TOP
    if pow2:
        scale = torch.exp2(torch.ceil(torch.log2(scale)))
    q = (w / scale[:, None, :, None]).clamp(-TOP, TOP).reshape(nb * BLOCK, kb * BLOCK)[:N, :K]
    return q.to(torch.float8_e4m3fn).contiguous(), scale.contiguous()


def _stack(pairs):
    return torch.stack([q for q, _ in pairs]), torch.stack([s for _, s in pairs])


def prepare(case, seed):
    g = _generator(seed)
    c = dict(case)
    T = c["T"]
    s = {"case": c}
    if c["op"] == "route":
        E = c["E"]
        s["logits"] = (_randn(g, T, E) * 1.5 + 0.7 * _randn(g, E)).to(DTYPES[c["dtype"]])
        spread = 0.1 if c["score"] == "sigmoid" else 0.3 / E
        s["bias"] = _randn(g, E) * spread if c["bias"] else None
    elif c["op"] == "quantise":
        s["x"] = _hidden(g, T, c["K"], c["dtype"])
    elif c["op"] == "linear":
        s["x"] = _hidden(g, T, c["K"], c["dtype"])
        s["w"] = _weight(g, c["N"], c["K"], c["pow2"])
        if own:
            from sparse_amd import fp8
            s["own_w"] = fp8.Weight.from_quantized(*s["w"])
    else:
        H, E, I, K, Is = c["H"], c["E"], c["I"], c["K"], c["Is"]
        dtype = DTYPES[c["dtype"]]
        s["x"] = _hidden(g, T, H, c["dtype"])
        logits = _randn(g, T, E) * 1.5 + 0.7 * _randn(g, E)
        topv, topi = torch.softmax(logits, -1).topk(K, dim=-1)
        s["topv"], s["topi"] = topv.to(dtype).contiguous(), topi.contiguous()
        s["experts"] = [_stack([_weight(g, n, k, c["pow2"]) for _ in range(E)]) for n, k in ((I, H), (I, H), (H, I))]
        s["shared"] = [_weight(g, n, k, c["pow2"]) for n, k in ((Is, H), (Is, H), (H, Is))] if Is else None
        s["shared_gate"] = _randn(g, T).to(dtype) if c["gate"] else None
        # the plan of this routing: permuted order, and where a permuted row sits in its expert's run
        flat = s["topi"].reshape(-1)
        s["order"] = torch.argsort(flat, stable=True)
        count = torch.bincount(flat, minlength=E)
        first = torch.cumsum(count, 0) - count
        s["active"] = torch.nonzero(count).reshape(-1)
        s["height"] = int(count.max())
        run_of = torch.cumsum((count > 0).to(torch.int64), 0) - 1
        sorted_ids = flat[s["order"]]
        s["place"] = run_of[sorted_ids] * s["height"] + torch.arange(T * K, device="cuda") - first[sorted_ids]
        if own:
            from sparse_amd import fp8, ops
            (gq, gs), (uq, us), (dq, ds) = s["experts"]
            s["own_experts"] = fp8.ExpertSlab.from_quantized(
                [((gq[e], gs[e]), (uq[e], us[e]), (dq[e], ds[e])) for e in range(E)])
            s["own_shared"] = tuple(fp8.Weight.from_quantized(*p) for p in s["shared"]) if Is else None
            s["own_perm"] = ops.permute_build(s["topi"], E)
    return s


# ------------------------------------------------------------------------------------ plain forms
def _blocks(x):
    """fp32 rows [T, K] -> [T, blocks, 128], zeros behind the end."""
    T, K = x.shape
    nb = -(-K // BLOCK)
    padded = x.new_zeros(T, nb * BLOCK)
    padded[:, :K] = x
    return padded.view(T, nb, BLOCK)


def _plain_quantise(x):
    """(8-bit values [T, K], exponents [T, blocks]) of fp32 rows: s is the smallest integer >= -120
    with max|x| <= 448 * 2^s, read off the largest value's own exponent (448 = 0.875 * 2^9), so that no
    logarithm is rounded; dividing by a power of two is exact, and 8 bits are rounded to once."""
    b = _blocks(x)
    m, e = torch.frexp(b.abs().amax(-1))
    s = torch.where(m <= 0.875, e - 9, e - 8)
    s = torch.where(m == 0, LOWEST, s).clamp_min(LOWEST)
    q = torch.ldexp(b, -s[..., None]).to(torch.float8_e4m3fn)
    return q.reshape(x.shape[0], -1)[:, :x.shape[1]], s


def _plain_rows(x):
    """fp32 rows after the round trip through 8 bits."""
    q, s = _plain_quantise(x)
    return torch.ldexp(_blocks(q.float()), s[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _plain_weight(q, scale):
    """fp32 values of 8-bit weights [..., N, K] with a scale for each 128 x 128 block."""
    N, K = q.shape[-2:]
    full = scale.repeat_interleave(BLOCK, -2)[..., :N, :].repeat_interleave(BLOCK, -1)[..., :K]
    return q.float() * full


def _plain_route(s):
    c, K = s["case"], s["case"]["K"]
    # in 64 bits: two scores a rounding of 32 bits apart would be ranked by that rounding
    x = s["logits"].double()
    T, E = x.shape
    score = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.softmax(x, -1)
    rank = score + s["bias"].double() if s["bias"] is not None else score
    if c["topk_group"] < c["n_group"]:
        by_group = rank.view(T, c["n_group"], -1)
        if c["group_score"] == "top2":
            best = by_group.topk(min(2, by_group.shape[-1]), dim=-1).values.sum(-1)
        else:
            best = by_group.amax(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :c["topk_group"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        rank = torch.where(keep[..., None], by_group, -math.inf).reshape(T, E)
    topi = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :K]
    topv = score.gather(1, topi)
    if c["renorm"]:
        topv = topv / topv.sum(-1, keepdim=True).clamp_min(1e-20)
    return (topv * c["scale"]).to(DTYPES[c["out"]]), topi


def _plain_ffn(rows, gate, up, down):
    """SwiGLU of fp32 rows [n, m, H] on fp32 weights [n, ...]; the intermediate goes through 8 bits."""
    g = torch.bmm(rows, gate.transpose(1, 2))
    h = g * torch.sigmoid(g) * torch.bmm(rows, up.transpose(1, 2))
    n, m, I = h.shape
    return torch.bmm(_plain_rows(h.reshape(n * m, I)).view(n, m, I), down.transpose(1, 2))


def _plain_experts(s):
    c = s["case"]
    dtype, H = DTYPES[c["dtype"]], c["H"]
    x = _plain_rows(s["x"].float())
    n = s["active"].numel()
    rows = x.new_zeros(n * s["height"], H)
    rows[s["place"]] = x[s["order"] // c["K"]]
    y = _plain_ffn(rows.view(n, s["height"], H), *(_plain_weight(q[s["active"]], w[s["active"]]) for q, w in s["experts"]))
    parts = y.reshape(-1, H)[s["place"]] * s["topv"].reshape(-1)[s["order"]].float()[:, None]
    if s["shared"] is None:
        return parts.to(dtype), None
    shared = _plain_ffn(x[None], *(_plain_weight(q, w)[None] for q, w in s["shared"]))[0]
    if s["shared_gate"] is not None:
        shared = shared * torch.sigmoid(s["shared_gate"].float())[:, None]
    return parts.to(dtype), shared.to(dtype)


def _plain(s):
    c = s["case"]
    if c["op"] == "route":
        return _plain_route(s)
    if c["op"] == "quantise":
        q, e = _plain_quantise(s["x"].float())
        return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    if c["op"] == "linear":
        return (_plain_rows(s["x"].float()) @ _plain_weight(*s["w"]).t()).to(DTYPES[c["dtype"]])
    return _plain_experts(s)


# ------------------------------------------------------------------------------- framework's calls
def _own(s):
    from sparse_amd import fp8, ops
    c = s["case"]
    if c["op"] == "route":
        return ops.gate_select(s["logits"], c["K"], score=c["score"], bias=s["bias"], n_group=c["n_group"],
                               topk_group=c["topk_group"], group_score=c["group_score"], renorm=c["renorm"],
                               scale=c["scale"], out_dtype=DTYPES[c["out"]])
    if c["op"] == "quantise":
        rows = fp8.quantize(s["x"])
        return rows.values, rows.scales
    if c["op"] == "linear":
        return fp8.linear(s["x"], s["own_w"])
    return fp8.moe_ffn(s["own_experts"], s["x"], s["topv"], s["own_perm"], shared=s["own_shared"],
                       shared_gate=s["shared_gate"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    T = c["T"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    es = size[c["dtype"]]
    if c["op"] == "route":
        return {"bytes": T * c["E"] * es + 4 * c["E"] * c["bias"] + T * c["K"] * (8 + size[c["out"]]),
                "flops": 8 * T * c["E"]}
    if c["op"] == "quantise":
        return {"bytes": T * c["K"] * (es + 1) + T * -(-c["K"] // BLOCK), "flops": 2 * T * c["K"]}
    if c["op"] == "linear":
        N, K = c["N"], c["K"]
        return {"bytes": T * K * es + N * K + 4 * -(-N // BLOCK) * -(-K // BLOCK) + T * N * es, "flops": 2 * T * N * K}
    H, E, I, K, Is = c["H"], c["E"], c["I"], c["K"], c["Is"]
    busy = E * (1 - (1 - K / E) ** T)      # experts that an even routing of T tokens reaches
    return {"bytes": int(busy * 3 * H * I) + 3 * H * Is + T * H * es * (1 + K + (Is > 0)) + T * K * (es + 8),
            "flops": 6 * T * H * (K * I + Is)}


# ------------------------------------------------------------------------------- from the definition
def _exact_round(x, s):
    """fp64 values on the grid of float8_e4m3fn times 2^s: 3 fraction bits, smallest exponent -6."""
    t = x / torch.exp2(s)
    grid = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(t / grid) * grid * torch.exp2(s)


def _exact_rows(x):
    """(rows after the round trip, exponents) of fp64 rows, block by block."""
    values, exps = [], []
    for k in range(0, x.shape[1], BLOCK):
        b = x[:, k:k + BLOCK]
        top = b.abs().amax(1, keepdim=True)
        s = torch.ceil(torch.log2(top.clamp_min(2.0 ** -140) / TOP))
        s = torch.where(top > TOP * torch.exp2(s), s + 1, s)
        s = torch.where(top <= TOP * torch.exp2(s - 1), s - 1, s).clamp_min(LOWEST)
        values.append(_exact_round(b, s))
        exps.append(s)
    return torch.cat(values, 1), torch.cat(exps, 1)


def _exact_weight(q, scale):
    w = q.double()
    for i in range(scale.shape[0]):
        for k in range(scale.shape[1]):
            w[i * BLOCK:(i + 1) * BLOCK, k * BLOCK:(k + 1) * BLOCK] *= float(scale[i, k])
    return w


def _exact_swiglu(x, gate, up, down):
    g = x @ _exact_weight(*gate).t()
    h = g / (1 + torch.exp(-g)) * (x @ _exact_weight(*up).t())
    return _exact_rows(h)[0] @ _exact_weight(*down).t()


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    T = c["T"]
    if c["op"] == "route":
        x = s["logits"].double().cpu()
        bias = torch.zeros(c["E"], dtype=torch.float64) if s["bias"] is None else s["bias"].double().cpu()
        if c["score"] == "sigmoid":
            p = 1 / (1 + torch.exp(-x))
        else:
            p = torch.exp(x - x.max(1, keepdim=True).values)
            p = p / p.sum(1, keepdim=True)
        r = p + bias
        per, ids = c["E"] // c["n_group"], torch.arange(c["E"])
        take = 1 if c["group_score"] == "max" else min(2, per)
        groups = torch.stack([r[:, g * per:(g + 1) * per].sort(1, descending=True).values[:, :take].sum(1)
                              for g in range(c["n_group"])], 1)
        # a group stays if fewer than topk_group groups come before it (higher, or as high with a lower number)
        num = torch.arange(c["n_group"])
        before = (groups[:, None, :] > groups[:, :, None]) | ((groups[:, None, :] == groups[:, :, None]) & (num[None, :] < num[:, None]))
        r = torch.where((before.sum(2) < c["topk_group"])[:, ids // per], r, torch.full_like(r, -math.inf))
        chosen, v = [], []
        for _ in range(c["K"]):
            i = r.argmax(1)
            i = torch.where(r == r.gather(1, i[:, None]), ids, c["E"]).min(1).values
            chosen.append(i)
            v.append(p.gather(1, i[:, None])[:, 0])
            r = r.scatter(1, i[:, None], -math.inf)
        v = torch.stack(v, 1)
        if c["renorm"]:
            v = v / v.sum(1, keepdim=True)
        return v * c["scale"], torch.stack(chosen, 1)
    if c["op"] == "quantise":
        x = s["x"].double()
        rows, e = _exact_rows(x)
        return rows / torch.exp2(e).repeat_interleave(BLOCK, 1)[:, :x.shape[1]], torch.exp2(e)
    x = _exact_rows(s["x"].double())[0]
    if c["op"] == "linear":
        return x @ _exact_weight(*s["w"]).t()
    flat = s["topi"].reshape(-1).cpu()
    weight = s["topv"].double().reshape(-1)
    parts = []
    for e in range(c["E"]):
        items = torch.nonzero(flat == e).reshape(-1).cuda()
        if items.numel():
            y = _exact_swiglu(x[items // c["K"]], *((q[e], w[e]) for q, w in s["experts"]))
            parts.append(y * weight[items][:, None])
    shared = None
    if s["shared"] is not None:
        shared = _exact_swiglu(x, *s["shared"])
        if s["shared_gate"] is not None:
            shared = shared / (1 + torch.exp(-s["shared_gate"].double()))[:, None]
    return torch.cat(parts), shared
