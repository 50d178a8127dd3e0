"""The 8-bit integer linears and the operators of a sparse-expert layer as cases that can be timed: plain forms in elementary
torch operations, and the calls of the framework's operator-level entry points.

  linear   y = (q . W^T) a s (+ residual): x quantised per lane (a = amax / 127, q = x / a to the nearest, ties to even),
           int8 weights with one scale per output channel; bf16 or f32 outputs
  pair     y = silu(gate) * up of two such products of one input
  route    scores (softmax or sigmoid) -> experts of every token: a bias for the choice, groups, top-k, renormalised weights;
           -inf closes an expert
  experts  the routed experts' gate/up product, SiLU, down product and weighted sum, int8 throughout; a route of -1 is none

Sizes: the layers of the 8B (4096 / 14336, vocabulary 128256), 70B (8192 / 28672) and sparse-expert (2048, 128 experts of 768,
top 8) configurations, and generic ones.
"""

import ctypes
import math

import numpy as np
import torch

own = False


def listed():
    def linear(name, lanes, n, k, residual=False, to_f32=False):
        return {"name": name, "op": "linear", "lanes": lanes, "n": n, "k": k, "residual": residual, "to_f32": to_f32}

    def pair(name, lanes, n, k):
        return {"name": name, "op": "pair", "lanes": lanes, "n": n, "k": k}

    def route(name, tokens, experts, top_k, sigmoid=False, bias=False, groups=1, chosen_groups=1, group_scores=1, renormalise=True, scale=1.0,
              f32=True, closed=0.0):
        return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "sigmoid": sigmoid, "bias": bias, "groups": groups,
                "chosen_groups": chosen_groups, "group_scores": group_scores, "renormalise": renormalise, "scale": scale, "f32": f32, "closed": closed}

    def experts(name, tokens, count, top_k, hidden, inter, residual=False, closed=0.0):
        return {"name": name, "op": "experts", "tokens": tokens, "experts": count, "top_k": top_k, "hidden": hidden, "inter": inter, "residual": residual,
                "closed": closed}

    return [
        # the attention output's projection of one decoded token: all latency
        linear("linear_one_token", 1, 4096, 4096, residual=True),
        # the logits of a verify step of three drafts
        linear("linear_logits_verify", 4, 128256, 4096, to_f32=True),
        # a ragged batch through a matrix of odd sizes
        linear("linear_ragged", 37, 1031, 2032),
        # the down projection of a prompt's chunk
        linear("linear_down_prompt", 2048, 4096, 14336, residual=True),
        # gate and up of a verify step of three drafts
        pair("pair_verify", 4, 14336, 4096),
        # gate and up of the largest layer for thirty-two streams of five lanes
        pair("pair_many_streams", 160, 28672, 8192),
        # the router of one decoded token: the smallest call
        route("route_one_token", 1, 128, 8, f32=False),
        # a long prompt's router with a bias for balance and groups
        route("route_prompt_grouped", 16384, 256, 8, sigmoid=True, bias=True, groups=8, chosen_groups=4, group_scores=2, scale=2.5),
        # an odd number of experts, some closed to a token, some tokens (padding) closed to all
        route("route_ragged", 777, 60, 6, bias=True, renormalise=False, f32=False, closed=0.2),
        # one decoded token through the sparse experts
        experts("experts_one_token", 1, 128, 8, 2048, 768),
        # eight streams with two drafts each
        experts("experts_streams", 24, 128, 8, 2048, 768),
        # a prompt's chunk
        experts("experts_prompt", 2048, 128, 8, 2048, 768, residual=True),
    ]


def _log_uniform(rng, low, high, step=1):
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(1, round(value / step)) * step


def draw(rng):
    limit = max(_cost(case) for case in listed())
    while True:
        op = rng.choice(["linear", "pair", "route", "experts"])
        if op in ("linear", "pair"):
            case = {"op": op, "lanes": _log_uniform(rng, 1, 4096), "n": _log_uniform(rng, 64, 28672), "k": _log_uniform(rng, 64, 28672, 16)}
            if op == "linear":
                case |= {"residual": rng.random() < 0.5, "to_f32": rng.random() < 0.3}
                case["residual"] &= not case["to_f32"]
        elif op == "route":
            groups = rng.choice([1, 1, 4, 8])
            experts = groups * _log_uniform(rng, 4, 512 // groups)
            chosen = groups if groups == 1 else rng.randint(1, groups)
            case = {"op": op, "tokens": _log_uniform(rng, 1, 16384), "experts": experts, "top_k": rng.randint(1, min(16, chosen * (experts // groups))),
                    "sigmoid": rng.random() < 0.5, "bias": rng.random() < 0.5, "groups": groups, "chosen_groups": chosen, "group_scores": rng.choice([1, 2]),
                    "renormalise": rng.random() < 0.5, "scale": rng.choice([1.0, 1.5, 2.5]), "f32": rng.random() < 0.5,
                    "closed": rng.choice([0.0, 0.0, 0.1, 0.4])}
        else:
            experts = _log_uniform(rng, 4, 256)
            case = {"op": op, "tokens": _log_uniform(rng, 1, 4096), "experts": experts, "top_k": rng.randint(1, min(8, experts)),
                    "hidden": _log_uniform(rng, 64, 8192, 16), "inter": _log_uniform(rng, 64, 4096, 16), "residual": rng.random() < 0.5,
                    "closed": rng.choice([0.0, 0.0, 0.1])}
            if 3 * experts * case["hidden"] * case["inter"] > 1.3e9:
                continue
        if _cost(case) <= limit:
            return case


def work(case):
    if case["op"] == "route":
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        bytes_ = tokens * (experts * (4 if case["f32"] else 2) + 8 * top_k) + (4 * experts if case["bias"] else 0)
        return {"bytes": bytes_, "flops": tokens * experts * 4}
    if case["op"] == "experts":
        tokens, hidden, inter = case["tokens"], case["hidden"], case["inter"]
        pairs = tokens * case["top_k"] * (1.0 - case["closed"])
        touched = case["experts"] * (1.0 - (1.0 - 1.0 / case["experts"]) ** pairs)  # as many experts as that many even choices meet
        bytes_ = touched * (3 * hidden * inter + 4 * (2 * inter + hidden)) + tokens * (4 + 2 * case["residual"]) * hidden + 8 * tokens * case["top_k"]
        return {"bytes": bytes_, "flops": 6 * pairs * hidden * inter}
    lanes, n, k = case["lanes"], case["n"], case["k"]
    if case["op"] == "pair":
        return {"bytes": 2 * n * k + 8 * n + 2 * lanes * (k + n), "flops": 4 * lanes * n * k}
    return {"bytes": n * k + 4 * n + 2 * lanes * k + lanes * n * ((4 if case["to_f32"] else 2) + 2 * case["residual"]), "flops": 2 * lanes * n * k}


def _cost(case):
    needed = work(case)
    return needed["bytes"] / 6.0e12 + needed["flops"] / 2.0e15


# ---- inputs


def _activations(generator, rows, width):
    """Hidden states as layers see them: some columns larger than the rest, rows of different magnitudes."""
    x = torch.randn((rows, width), generator=generator, device="cuda")
    x *= torch.exp(0.5 * torch.randn((1, width), generator=generator, device="cuda"))
    x *= torch.exp(0.3 * torch.randn((rows, 1), generator=generator, device="cuda"))
    return x.to(torch.bfloat16)


def _weights(generator, *shape):
    """int8 weights of a normal distribution whose largest of a channel is at 127, and the channels' scales."""
    w = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = w.view(-1, shape[-1])
    rows = max(1, (1 << 26) // shape[-1])
    for first in range(0, flat.shape[0], rows):
        part = flat[first : first + rows]
        part.copy_(torch.randn(part.shape, generator=generator, device="cuda").mul_(33.0).round_().clamp_(-127, 127))
    scale = torch.exp(0.25 * torch.randn(shape[:-1], generator=generator, device="cuda")) * (0.6 / 33.0 / math.sqrt(shape[-1]))
    return w, scale


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    state = {"case": dict(case)}
    if case["op"] == "route":
        tokens, experts = case["tokens"], case["experts"]
        logits = torch.randn((tokens, experts), generator=generator, device="cuda") * 1.5
        if case["closed"]:
            logits.masked_fill_(torch.rand((tokens, experts), generator=generator, device="cuda") < case["closed"], -math.inf)
            logits[torch.rand(tokens, generator=generator, device="cuda") < case["closed"] / 4] = -math.inf
        state["logits"] = logits if case["f32"] else logits.to(torch.bfloat16)
        state["bias"] = torch.randn(experts, generator=generator, device="cuda") * 0.05 if case["bias"] else None
    elif case["op"] == "experts":
        tokens, experts, hidden, inter = case["tokens"], case["experts"], case["hidden"], case["inter"]
        state["x"] = _activations(generator, tokens, hidden)
        # some experts are chosen more often than others
        logits = torch.randn((tokens, experts), generator=generator, device="cuda") + 0.5 * torch.randn((1, experts), generator=generator, device="cuda")
        chosen = logits.topk(case["top_k"], dim=1)
        weights, ids = chosen.values.softmax(dim=1), chosen.indices.to(torch.int32)
        if case["closed"]:
            none = torch.rand((tokens, case["top_k"]), generator=generator, device="cuda") < case["closed"]
            weights, ids = weights.masked_fill(none, 0.0), ids.masked_fill(none, -1)
        state["weights"], state["ids"] = weights.contiguous(), ids.contiguous()
        state["gate_up"], state["gate_up_scale"] = _weights(generator, experts, 2 * inter, hidden)
        state["down"], state["down_scale"] = _weights(generator, experts, hidden, inter)
        state["residual"] = _activations(generator, tokens, hidden) if case["residual"] else None
    else:
        lanes, n, k = case["lanes"], case["n"], case["k"]
        state["x"] = _activations(generator, lanes, k)
        state["w"], state["scale"] = _weights(generator, n, k)
        if case["op"] == "pair":
            state["up"], state["up_scale"] = _weights(generator, n, k)
        else:
            state["residual"] = _activations(generator, lanes, n) if case["residual"] else None
    return state


# ---- plain forms


def _quantised(x):
    """(whole values in -127..127, scale) of every row.  127 x is exact in 32 bits for bf16 inputs, so that one rounded
    division meets the ties."""
    top = x.abs().amax(dim=-1, keepdim=True)
    return torch.where(top > 0, torch.round(x * 127.0 / top), 0.0), top / 127.0


def _plain_linear(state):
    q, a = _quantised(state["x"].float())
    y = q @ state["w"].float().T * a * state["scale"]
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y if state["case"]["to_f32"] else y.to(torch.bfloat16)


def _plain_pair(state):
    q, a = _quantised(state["x"].float())
    gate = q @ state["w"].float().T * a * state["scale"]
    up = q @ state["up"].float().T * a * state["up_scale"]
    return (gate / (1.0 + torch.exp(-gate)) * up).to(torch.bfloat16)


def _plain_route(state):
    case, logits = state["case"], state["logits"].double()  # choices next to one another: 64 bits
    tokens, experts = logits.shape
    open_ = logits > -math.inf
    if case["sigmoid"]:
        scores = torch.where(open_, 1.0 / (1.0 + torch.exp(-logits)), 0.0)
    else:
        top = logits.amax(dim=1, keepdim=True)
        terms = torch.where(open_, torch.exp(torch.where(logits == top, 0.0, logits - top)), 0.0)
        scores = torch.where(open_, terms / terms.sum(dim=1, keepdim=True), 0.0)
    choice = scores if state["bias"] is None else scores + state["bias"].double()
    choice = torch.where(open_, choice, -math.inf)
    if case["groups"] > 1:
        grouped = choice.view(tokens, case["groups"], -1)
        best = grouped.topk(case["group_scores"], dim=2).values
        rank = torch.where(best > -math.inf, best, 0.0).sum(dim=2).masked_fill(best[:, :, 0] == -math.inf, -math.inf)
        kept = rank.sort(dim=1, descending=True, stable=True).indices[:, : case["chosen_groups"]]
        closed = torch.ones_like(rank, dtype=torch.bool).scatter(1, kept, False)
        choice = grouped.masked_fill(closed[:, :, None], -math.inf).view(tokens, experts)
    picked, ids = choice.sort(dim=1, descending=True, stable=True)
    picked, ids = picked[:, : case["top_k"]], ids[:, : case["top_k"]]
    weights = torch.where(picked > -math.inf, scores.gather(1, ids), 0.0)
    if case["renormalise"]:
        total = weights.sum(dim=1, keepdim=True)
        weights = torch.where(total > 0, weights / total, 0.0)
    return {"ids": torch.where(picked > -math.inf, ids, -1).to(torch.int32), "weights": (weights * case["scale"]).float()}


def _plain_experts(state):
    case = state["case"]
    tokens, top_k, hidden, inter = case["tokens"], case["top_k"], case["hidden"], case["inter"]
    # the pairs in the order of their experts, each expert's in a block of its own of as many rows as the busiest has
    flat = state["ids"].reshape(-1)
    pairs = torch.nonzero(flat >= 0).reshape(-1)
    used, local, counts = torch.unique(flat[pairs], return_inverse=True, return_counts=True)
    order = local.argsort(stable=True)
    pairs, local = pairs[order], local[order]
    place = torch.arange(pairs.numel(), device="cuda") - (counts.cumsum(0) - counts)[local]
    rows = int(counts.max()) if counts.numel() else 0
    used = used.long()

    def product(values, w, scale):
        q, a = _quantised(values)
        block = torch.zeros((used.numel(), rows, q.shape[1]), device="cuda")
        block[local, place] = q
        out = torch.bmm(block, w[used].float().transpose(1, 2))
        return out[local, place] * a * scale[used][local]

    gate_up = product(state["x"].float()[pairs // top_k], state["gate_up"], state["gate_up_scale"])
    gate, up = gate_up[:, :inter], gate_up[:, inter:]
    out = product(gate / (1.0 + torch.exp(-gate)) * up, state["down"], state["down_scale"])
    routed = torch.zeros((tokens * top_k, hidden), device="cuda")
    routed[pairs] = out * state["weights"].reshape(-1)[pairs, None]
    y = routed.view(tokens, top_k, hidden).sum(dim=1)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(torch.bfloat16)


# ---- the framework's calls


def _pointer(tensor):
    return ctypes.c_void_p(None if tensor is None else tensor.data_ptr())


def _own_call(state):
    """The entry point, its arguments but for the stream, and its outputs: made once, with the scratch buffer that a program keeps."""
    import llmoop_b200 as nb
    from llmoop_b200.runtime import Routing

    case, library = state["case"], nb.library()
    new = lambda *shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if case["op"] == "route":
        ids, weights = (new(case["tokens"], case["top_k"], dtype=dtype) for dtype in (torch.int32, torch.float32))
        routing = Routing(experts=case["experts"], top_k=case["top_k"], sigmoid=case["sigmoid"], groups=case["groups"], chosen_groups=case["chosen_groups"],
                          group_scores=case["group_scores"], renormalise=case["renormalise"], scale=case["scale"])
        arguments = (_pointer(state["logits"]), _pointer(state["bias"]), _pointer(ids), _pointer(weights), case["tokens"], int(case["f32"]), ctypes.byref(routing))
        return library.nerve_b200_op_route_experts, arguments, {"ids": ids, "weights": weights}
    if case["op"] == "experts":
        sizes = (case["tokens"], case["top_k"], case["experts"], case["hidden"], case["inter"])
        state["scratch"] = new(library.nerve_b200_op_experts_int8_scratch_bytes(*sizes), dtype=torch.uint8)
        y = new(case["tokens"], case["hidden"], dtype=torch.bfloat16)
        tensors = [state[name] for name in ("x", "ids", "weights", "gate_up", "gate_up_scale", "down", "down_scale")] + [y, state["residual"], state["scratch"]]
        return library.nerve_b200_op_experts_int8, (*map(_pointer, tensors), *sizes), y
    lanes, n, k = case["lanes"], case["n"], case["k"]
    state["scratch"] = new(library.nerve_b200_op_linear_int8_scratch_bytes(lanes, k), dtype=torch.uint8)
    if case["op"] == "pair":
        y = new(lanes, n, dtype=torch.bfloat16)
        tensors = [state[name] for name in ("x", "w", "scale", "up", "up_scale")] + [y, state["scratch"]]
        return library.nerve_b200_op_linear_int8_silu_pair, (*map(_pointer, tensors), lanes, n, k), y
    y = new(lanes, n, dtype=torch.float32 if case["to_f32"] else torch.bfloat16)
    tensors = [state["x"], state["w"], state["scale"], y, state["residual"], state["scratch"]]
    return library.nerve_b200_op_linear_int8, (*map(_pointer, tensors), lanes, n, k, int(case["to_f32"])), y


def _own_run(state):
    if "call" not in state:
        state["call"] = _own_call(state)
    function, arguments, outputs = state["call"]
    if function(*arguments, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) != 0:
        import llmoop_b200 as nb

        raise RuntimeError(nb.library().nerve_b200_last_error().decode())
    return outputs


def run(state):
    if own:
        return _own_run(state)
    return {"linear": _plain_linear, "pair": _plain_pair, "route": _plain_route, "experts": _plain_experts}[state["case"]["op"]](state)


# ---- in 64 bits, from the definitions


def _exact_product(x, w, scale):
    """x [rows, k], w [n, k]: every row of x as whole multiples of its largest magnitude's 127th part, times w."""
    x = x.double()
    unit = x.abs().max(dim=1).values / 127
    steps = torch.zeros_like(x)
    some = unit > 0
    steps[some] = torch.round(127 * x[some] / x[some].abs().max(dim=1).values[:, None])
    return torch.einsum("mk,nk->mn", steps, w.double()) * unit[:, None] * scale.double()[None, :]


def _exact_route(state):
    case = state["case"]
    logits = state["logits"].double().cpu().numpy()
    scores = np.zeros_like(logits)
    for row, out in zip(logits, scores):
        able = np.isfinite(row)
        if case["sigmoid"]:
            out[able] = 1 / (1 + np.exp(-row[able]))
        elif able.any():
            terms = np.exp(row[able] - row[able].max())
            out[able] = terms / math.fsum(terms)
    bias = np.zeros(case["experts"]) if state["bias"] is None else state["bias"].double().cpu().numpy()
    ids = np.full((case["tokens"], case["top_k"]), -1, dtype=np.int32)
    weights = np.zeros((case["tokens"], case["top_k"]))
    size = case["experts"] // case["groups"]
    for token in range(case["tokens"]):
        able = np.flatnonzero(np.isfinite(logits[token]))
        value = scores[token] + bias
        if case["groups"] > 1:
            best = {}
            for group in set(able // size):
                members = np.sort(value[able[able // size == group]])[::-1]
                best[group] = members[: case["group_scores"]].sum()
            kept = sorted(best, key=lambda group: (-best[group], group))[: case["chosen_groups"]]
            able = able[np.isin(able // size, kept)]
        chosen = able[np.argsort(-value[able], kind="stable")][: case["top_k"]]
        ids[token, : len(chosen)] = chosen
        weights[token, : len(chosen)] = scores[token, chosen]
    if case["renormalise"]:
        total = weights.sum(axis=1, keepdims=True)
        weights = np.divide(weights, total, out=np.zeros_like(weights), where=total > 0)
    return {"ids": ids, "weights": weights * case["scale"]}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(state)
    if case["op"] == "linear":
        y = _exact_product(state["x"], state["w"], state["scale"])
        return y if state["residual"] is None else y + state["residual"].double()
    if case["op"] == "pair":
        gate = _exact_product(state["x"], state["w"], state["scale"])
        return gate * torch.sigmoid(gate) * _exact_product(state["x"], state["up"], state["up_scale"])
    y = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device="cuda") if state["residual"] is None else state["residual"].double()
    for expert in range(case["experts"]):
        token, slot = (state["ids"] == expert).nonzero(as_tuple=True)
        if len(token) == 0:
            continue
        both = _exact_product(state["x"][token], state["gate_up"][expert], state["gate_up_scale"][expert])
        gate, up = both.chunk(2, dim=1)
        out = _exact_product(gate * torch.sigmoid(gate) * up, state["down"][expert], state["down_scale"][expert])
        y.index_add_(0, token, out * state["weights"][token, slot].double()[:, None])
    return y
