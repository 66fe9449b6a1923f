"""The dense and expert products over unquantised weights (fp16, bf16): cases, plain forms and exact values.

Three operators, T tokens, K columns, N rows of a weight matrix W [N][K]:

  linear          y[t] = act(W x[t] + b) + r[t], act one of none, silu, gelu, gelu_tanh, swiglu (two matrices)
  expert_linear   y[p] = act(W_e x[rows[p]] + b_e) for the positions p of expert e's list
  expert_combine  out[t] = base[t] + sum over the token's slots, ascending, of w[t, s] * (W_e h[p])

`own` false computes them with elementary torch operations in 32 bits, rounded once at the end;
`own` true calls the framework's kernels.
"""
import importlib
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = 7.0  # the clamp of the repository's SwiGLU configurations


# ---- cases ----------------------------------------------------------------------------------


def _linear(name, tokens, k, n, dtype, act="none", bias=False, residual=False, pad=0):
    return {"name": name, "op": "linear", "tokens": tokens, "k": k, "n": n, "dtype": dtype, "act": act,
            "bias": bias, "residual": residual, "pad": pad}


def _experts(name, op, tokens, slots, experts, k, n, dtype, act="none", bias=False, skew=0.0, base=False):
    return {"name": name, "op": op, "tokens": tokens, "slots": slots, "experts": experts, "k": k, "n": n,
            "dtype": dtype, "act": act, "bias": bias, "skew": skew, "base": base}


def listed():
    return [
        # one token through a router gate: the smallest call, all latency
        _linear("linear 1 tok gate", 1, 4096, 256, "bf16", bias=True),
        # a decode batch through a square projection of the 7168-wide layer: one pass over the weights
        _linear("linear 64 tok residual", 64, 7168, 7168, "f16", residual=True),
        # nothing a multiple of anything, rows of a wider tensor: a classifier head, a pruned layer
        _linear("linear odd gelu", 333, 1001, 1999, "bf16", act="gelu", bias=True, residual=True, pad=3),
        # the shared expert's gate and up of a prefill chunk
        _linear("linear swiglu 512 tok", 512, 7168, 2048, "bf16", act="swiglu"),
        # the largest: a projection of a long prefill, with bias and residual
        _linear("linear 8192 tok", 8192, 7168, 7168, "bf16", bias=True, residual=True),
        # one token, top-8 of 256 experts: gate and up, latency and the stream of eight experts
        _experts("gate/up 1 tok top-8/256", "expert_linear", 1, 8, 256, 7168, 2048, "bf16", act="swiglu"),
        # a decode batch of 64: nearly every expert is drawn, two tokens each
        _experts("gate/up 64 tok top-8/256", "expert_linear", 64, 8, 256, 7168, 2048, "f16", act="swiglu"),
        # a prefill chunk, top-6 of 64 experts of unequal popularity
        _experts("gate/up 4096 tok top-6/64", "expert_linear", 4096, 6, 64, 4096, 2048, "bf16", act="swiglu", skew=0.6),
        # small odd experts without a gate matrix, one of them holding most positions, one perhaps none
        _experts("odd experts silu", "expert_linear", 777, 3, 13, 1000, 523, "f16", act="silu", bias=True, skew=1.1),
        # the down projection and the weighted sum of one token
        _experts("combine 1 tok top-8/256", "expert_combine", 1, 8, 256, 2048, 7168, "f16"),
        # the same of a decode batch over the shared expert's output
        _experts("combine 48 tok top-6/64", "expert_combine", 48, 6, 64, 2048, 4096, "bf16", base=True),
        # the same of a prefill chunk
        _experts("combine 4096 tok top-6/64", "expert_combine", 4096, 6, 64, 2048, 4096, "bf16", base=True, skew=0.6),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A matrix dimension: half the time a multiple of 64, else whatever comes."""
    v = _log_int(rng, low, high)
    return max(64, v // 64 * 64) if rng.random() < 0.5 else v


def draw(rng):
    while True:
        case = {"op": rng.choice(("linear", "linear", "expert_linear", "expert_combine")),
                "tokens": _log_int(rng, 1, 8192), "k": _width(rng, 64, 7168), "n": _width(rng, 16, 7168),
                "dtype": rng.choice(("f16", "bf16"))}
        acts = ("none", "silu", "gelu", "gelu_tanh", "swiglu")
        if case["op"] == "linear":
            case.update(act=rng.choice(acts), bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                        pad=rng.choice((0, 0, 0, 8, 5)))
        else:
            experts = _log_int(rng, 2, 256)
            case.update(slots=rng.randint(1, min(8, experts)), experts=experts, bias=rng.random() < 0.3,
                        skew=rng.choice((0.0, 0.6, 1.1)),
                        act=rng.choice(("none", "silu", "swiglu", "swiglu")) if case["op"] == "expert_linear" else "none",
                        base=case["op"] == "expert_combine" and rng.random() < 0.5)
            # what the plain form holds at once: every expert's rows padded to the longest list
            if experts * case["tokens"] * max(case["k"], case["n"]) > 1 << 32:
                continue
            if experts * case["k"] * case["n"] * (2 if case["act"] == "swiglu" else 1) > 1 << 32:
                continue
        if work(case)["flops"] <= 8.4e11:
            return case


# ---- inputs ---------------------------------------------------------------------------------


def _routing(case, gen, device):
    """ids [tokens][slots]: distinct experts per token, expert e drawn in proportion to
    (e + 1)^-skew, by adding Gumbel noise to the log popularity and taking the largest."""
    e = torch.arange(1, case["experts"] + 1, device=device, dtype=torch.float32)
    u = torch.rand(case["tokens"], case["experts"], generator=gen, device=device).clamp_(1e-9, 1 - 1e-6)
    keys = -case["skew"] * torch.log(e) - torch.log(-torch.log(u))
    return torch.topk(keys, case["slots"], dim=1).indices.to(torch.int32)


def _normal(shape, std, dtype, gen):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    tokens, k, n = case["tokens"], case["k"], case["n"]
    pair = case["act"] == "swiglu"
    state = {"case": case}
    # activations near unit size, weights such that pre-activations have a spread of 1.5
    std = 1.5 / math.sqrt(k)
    if case["op"] == "linear":
        pad = case["pad"]
        state["x"] = _normal((tokens, k + pad), 1.0, dtype, gen)[:, :k]
        state["w"] = _normal((n, k + pad), std, dtype, gen)[:, :k]
        state["w_up"] = _normal((n, k + pad), std, dtype, gen)[:, :k] if pair else None
        state["bias"] = _normal((n,), 0.5, dtype, gen) if case["bias"] else None
        state["bias_up"] = _normal((n,), 0.5, dtype, gen) if case["bias"] and pair else None
        state["residual"] = _normal((tokens, n + pad), 1.0, dtype, gen)[:, :n] if case["residual"] else None
        return state
    experts, slots = case["experts"], case["slots"]
    ids = _routing(case, gen, "cuda")
    # what the router and the permutation before these operators leave: the draws sorted by
    # expert (ascending inside one), the lists' bounds, the token of every position
    order = torch.argsort(ids.reshape(-1).long(), stable=True)
    counts = torch.bincount(ids.reshape(-1).long(), minlength=experts)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum(counts, 0).to(torch.int32)
    state["ids"], state["offsets"] = ids, offsets
    state["draws"] = order.to(torch.int32)
    state["rows"] = (order // slots).to(torch.int32)
    state["w"] = _normal((experts, n, k), std, dtype, gen)
    state["w_up"] = _normal((experts, n, k), std, dtype, gen) if pair else None
    state["bias"] = _normal((experts, n), 0.5, dtype, gen) if case["bias"] else None
    state["bias_up"] = _normal((experts, n), 0.5, dtype, gen) if case["bias"] and pair else None
    if case["op"] == "expert_linear":
        state["x"] = _normal((tokens, k), 1.0, dtype, gen)
    else:
        state["h"] = _normal((tokens * slots, k), 1.0, dtype, gen)
        w = torch.rand(tokens, slots, generator=gen, device="cuda") + 0.01
        state["weights"] = w / w.sum(dim=1, keepdim=True)
        state["base"] = _normal((tokens, n), 1.0, dtype, gen) if case["base"] else None
    return state


# ---- the plain forms ------------------------------------------------------------------------


def _activate(act, g, u):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    if act == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))
    if act == "swiglu":
        g = torch.clamp(g, max=LIMIT)
        return g / (1.0 + torch.exp(-g)) * torch.clamp(u, -LIMIT, LIMIT)
    return g


def _plain_linear(s):
    case = s["case"]
    x = s["x"].float()

    def product(w, b):
        y = torch.mm(x, w.float().t())
        return y if b is None else y + b.float()

    g = product(s["w"], s["bias"])
    u = product(s["w_up"], s["bias_up"]) if case["act"] == "swiglu" else None
    y = _activate(case["act"], g, u)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _expert_of(s):
    """The expert of every position."""
    p = torch.arange(s["draws"].numel(), device="cuda", dtype=torch.int32)
    return torch.searchsorted(s["offsets"][1:], p, right=True)


def _plain_products(s, x):
    """W_e x (+ b_e) of every position, 32 bits: a list of one or two [positions][n]."""
    e = _expert_of(s)
    pairs = [(s["w"], s["bias"])] + ([(s["w_up"], s["bias_up"])] if s["w_up"] is not None else [])
    found = []
    if x.shape[0] * 2 <= s["case"]["experts"]:  # few positions: only their experts' matrices
        for w, b in pairs:
            y = torch.bmm(w[e].float(), x.unsqueeze(2)).squeeze(2)
            found.append(y if b is None else y + b.float()[e])
        return found
    # every expert's rows padded to the longest list, one product an expert
    place = torch.arange(x.shape[0], device="cuda") - s["offsets"][e].long()
    longest = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    padded = torch.zeros(s["case"]["experts"], longest, x.shape[1], device="cuda")
    padded[e, place] = x
    padded = padded.transpose(1, 2).contiguous()
    for w, b in pairs:
        y = torch.bmm(w.float(), padded)[e, :, place]
        found.append(y if b is None else y + b.float()[e])
    return found


def _plain_expert_linear(s):
    found = _plain_products(s, s["x"][s["rows"].long()].float())
    return _activate(s["case"]["act"], found[0], found[-1]).to(s["x"].dtype)


def _plain_expert_combine(s):
    case = s["case"]
    y, = _plain_products(s, s["h"].float())
    by_draw = torch.empty_like(y)
    by_draw[s["draws"].long()] = y
    out = (by_draw.view(case["tokens"], case["slots"], -1) * s["weights"].unsqueeze(2)).sum(dim=1)
    if s["base"] is not None:
        out = out + s["base"].float()
    return out.to(s["h"].dtype)


# ---- one pass -------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if not own:
        return {"linear": _plain_linear, "expert_linear": _plain_expert_linear,
                "expert_combine": _plain_expert_combine}[case["op"]](state)
    dense = importlib.import_module("project-aeon_amd.dense")
    if case["op"] == "linear":
        return dense.linear(state["x"], state["w"], bias=state["bias"], activation=case["act"],
                            weight_up=state["w_up"], bias_up=state["bias_up"], swiglu_limit=LIMIT,
                            residual=state["residual"])
    if case["op"] == "expert_linear":
        return dense.expert_linear(state["x"], state["w"], state["offsets"], state["rows"], bias=state["bias"],
                                   activation=case["act"], weight_up=state["w_up"], bias_up=state["bias_up"],
                                   swiglu_limit=LIMIT)
    return dense.expert_combine(state["h"], state["w"], state["offsets"], state["draws"], state["ids"],
                                state["weights"], bias=state["bias"], base=state["base"])


def _distinct(case):
    """Experts that hold a position, for the work of a case: counted on a routing of its own."""
    gen = torch.Generator()
    gen.manual_seed(1)
    return int(torch.unique(_routing(case, gen, "cpu")).numel())


def work(case):
    tokens, k, n = case["tokens"], case["k"], case["n"]
    mats = 2 if case["act"] == "swiglu" else 1
    if case["op"] == "linear":
        values = tokens * k + mats * n * k + tokens * n * (2 if case["residual"] else 1) + (mats * n if case["bias"] else 0)
        return {"bytes": 2 * values, "flops": 2 * mats * tokens * n * k}
    positions, live = tokens * case["slots"], _distinct(case)
    values = live * mats * n * (k + (1 if case["bias"] else 0))
    lists = 4 * (case["experts"] + 1 + positions)
    if case["op"] == "expert_linear":
        values += tokens * k + positions * n
    else:
        values += positions * k + tokens * n * (2 if case["base"] else 1)
        lists += 8 * positions
    return {"bytes": 2 * values + lists, "flops": 2 * mats * positions * n * k}


# ---- 64 bits, from the definitions ----------------------------------------------------------


def _exact_act(act, g, u):
    if act == "silu":
        return g * torch.special.expit(g)
    if act == "gelu":
        return 0.5 * g * torch.special.erfc(-g / math.sqrt(2.0))
    if act == "gelu_tanh":
        return g * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))
    if act == "swiglu":
        g = torch.minimum(g, torch.full_like(g, LIMIT))
        return g * torch.special.expit(g) * torch.minimum(torch.maximum(u, torch.full_like(u, -LIMIT)),
                                                          torch.full_like(u, LIMIT))
    return g


def exact(case, seed):
    s = prepare(case, seed)

    def product(x, w, b):
        y = x @ w.double().t().contiguous()
        return y if b is None else y + b.double()

    if case["op"] == "linear":
        x = s["x"].double()
        u = product(x, s["w_up"], s["bias_up"]) if case["act"] == "swiglu" else None
        y = _exact_act(case["act"], product(x, s["w"], s["bias"]), u)
        return y if s["residual"] is None else y + s["residual"].double()
    bounds = s["offsets"].tolist()
    combine = case["op"] == "expert_combine"
    positions = case["tokens"] * case["slots"]
    if combine:
        out = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device="cuda")
        if s["base"] is not None:
            out += s["base"].double()
    else:
        out = torch.empty(positions, case["n"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        a, b = bounds[e], bounds[e + 1]
        if a == b:
            continue
        x = (s["h"][a:b] if combine else s["x"][s["rows"][a:b].long()]).double()
        g = product(x, s["w"][e], None if s["bias"] is None else s["bias"][e])
        if combine:
            d = s["draws"][a:b].long()
            out.index_add_(0, d // case["slots"], g * s["weights"].reshape(-1)[d].double().unsqueeze(1))
            continue
        u = None
        if case["act"] == "swiglu":
            u = product(x, s["w_up"][e], None if s["bias_up"] is None else s["bias_up"][e])
        out[a:b] = _exact_act(case["act"], g, u)
    return out
