"""Mixture-of-experts operators on packed weights: the workloads they are timed and compared on.

A layer of experts holds E matrices W[e], packed as 4-bit or 8-bit codes with a scale and a zero for every output
channel or for every group of input features and channel.  A router gives each token top_k expert numbers (a number
outside 0 .. E - 1 marks a token that goes nowhere, e.g. padding) and as many weights.  The operators:

  sort     the (token, choice) pairs in order of their expert, ties in order of the pair: the order, its inverse and
           where each expert's rows begin
  gather   rows of the tokens in that order, and the gradient (each token adds up its copies)
  combine  the rows back at their tokens, weighted and added up, and the gradients of rows and weights
  matmul   rows of expert e times W[e], and the gradient with respect to the tokens

Rows of pairs that go nowhere stand behind the last expert's rows and are zero.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _experts():
    """The package's operators (only where `own` is true)."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jax-gptq_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from jax_gptq_amd import experts
    return experts


# ---------------------------------------------------------------------------------------------- cases
def _route(op, name, tokens, top_k, experts, **more):
    case = {"name": name, "op": op, "tokens": tokens, "top_k": top_k, "experts": experts, "dropped": 0.0,
            "index": "int64"}
    case.update(more)
    return case


def listed():
    return [
        # a serving step's routing: a couple of dozen requests, two of eight experts each; launch latency decides
        _route("sort", "sort_24x2_of_8", 24, 2, 8),
        # routing of a large prompt batch over many small experts, some padding tokens
        _route("sort", "sort_32768x8_of_128_padded", 32768, 8, 128, dropped=0.02, index="int32"),
        # calibration or training rows of a small layer, fp32, an odd number of tokens
        _route("gather", "gather_333x2_768_fp32_train", 333, 2, 8, width=768, type="fp32", train=True),
        # rows of a prompt batch at the 4096 features of the layer benchmark, with the gradient
        _route("gather", "gather_8192x2_4096_bf16_train", 8192, 2, 8, width=4096, type="bf16", train=True),
        # a serving step's results back at their tokens
        _route("combine", "combine_6x2_4096_fp16", 6, 2, 8, width=4096, type="fp16", train=False),
        # the same in training, with both gradients, four of 32 experts, padded batch
        _route("combine", "combine_4096x4_4096_bf16_train", 4096, 4, 32, width=4096, type="bf16", train=True,
               dropped=0.05),
        # one token of one request: two matrix-vector products with 4-bit weights, up projection
        _route("matmul", "matmul_1x2_of_8_4096x11008_fp16", 1, 2, 8, k=4096, n=11008, bits=4, group=128,
               type="fp16", tables="fp16", train=False),
        # a dozen requests on many small experts: hardly any expert sees two rows
        _route("matmul", "matmul_12x4_of_64_2048x1424_bf16", 12, 4, 64, k=2048, n=1424, bits=4, group=64,
               type="bf16", tables="fp32", train=False),
        # 8-bit codes, one scale per channel, fp32 rows, an odd number of channels
        _route("matmul", "matmul_5x2_of_8_768x909_fp32_8bit", 5, 2, 8, k=768, n=909, bits=8, group=0,
               type="fp32", tables="fp32", train=False),
        # a short prompt or a batch of requests on the down projection: a few dozen rows per expert
        _route("matmul", "matmul_150x2_of_8_11008x4096_fp16", 150, 2, 8, k=11008, n=4096, bits=4, group=128,
               type="fp16", tables="fp32", train=False),
        # a prompt batch on the up projection: about a thousand rows per expert
        _route("matmul", "matmul_4096x2_of_8_4096x11008_bf16", 4096, 2, 8, k=4096, n=11008, bits=4, group=128,
               type="bf16", tables="fp32", train=False),
        # a training step through frozen experts: product and gradient of the tokens, padded batch
        _route("matmul", "matmul_2048x2_of_8_4096x4096_fp16_train", 2048, 2, 8, k=4096, n=4096, bits=4, group=128,
               type="fp16", tables="fp32", train=True, dropped=0.03),
    ]


def _spread(rng, low, high, multiple=1):
    """A size between low and high, spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(multiple, int(round(v / multiple)) * multiple)


def draw(rng):
    most = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(["sort", "gather", "combine", "matmul", "matmul", "matmul"])
        experts = rng.choice([2, 8, 8, 16, 32, 60, 64, 128])
        top_k = min(experts, rng.choice([1, 2, 2, 4, 6, 8]))
        case = _route(op, "", 0, top_k, experts, dropped=rng.choice([0.0, 0.0, 0.04]),
                      index=rng.choice(["int32", "int64"]))
        del case["name"]
        if op == "sort":
            case["tokens"] = _spread(rng, 1, 32768)
        elif op in ("gather", "combine"):
            case["tokens"] = _spread(rng, 1, 8192)
            case["width"] = _spread(rng, 256, 8192, rng.choice([1, 2, 8, 64]))
            case["type"] = rng.choice(["fp16", "bf16", "fp32"])
            case["train"] = rng.random() < 0.5
            if case["tokens"] * top_k * case["width"] > 80_000_000:
                continue
        else:
            case["tokens"] = _spread(rng, 1, 4096)
            case["group"] = rng.choice([0, 32, 64, 128, 128, 128, 256])
            case["k"] = _spread(rng, 512, 11008, case["group"] or rng.choice([2, 32, 32]))
            case["n"] = _spread(rng, 256, 11008, rng.choice([1, 16, 16, 64]))
            case["bits"] = rng.choice([4, 4, 4, 8])
            case["type"] = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"])
            case["tables"] = rng.choice(["fp16", "fp32", "fp32"])
            case["train"] = rng.random() < 0.3
            size = case["k"] * case["n"] * experts
            if size > 400_000_000 or work(case)["flops"] * (2 if case["type"] == "fp32" else 1) > most:
                continue
        return case


# ---------------------------------------------------------------------------------------------- inputs
def _popularity(experts):
    """How often a router picks each expert: some are picked about four times as often as others."""
    z = torch.linspace(-0.7, 0.7, experts, dtype=torch.float64)
    return torch.softmax(z, 0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, k, E = case["tokens"], case["top_k"], case["experts"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    # the k best experts of every token, by a score that favours some experts
    gumbel = -torch.log(-torch.log(uniform(T, E).clamp_(1e-9, 1 - 1e-7)))
    score = torch.log(_popularity(E)).float().cuda()[torch.randperm(E, generator=gen, device="cuda")] + gumbel
    best, ids = torch.topk(score, k, dim=1)
    if case["dropped"] > 0:
        nowhere = uniform(T) < case["dropped"]
        ids = torch.where(nowhere[:, None], torch.full_like(ids, -1), ids)
    ids = ids.to(torch.int32 if case["index"] == "int32" else torch.int64).contiguous()
    state = {"case": case, "ids": ids}
    if case["op"] == "sort":
        return state

    # a router's program keeps the sorted order and its counts for the operators that follow
    key = torch.where((ids < 0) | (ids >= E), torch.full_like(ids, E), ids).reshape(-1)
    order = torch.sort(key, stable=True).indices
    state["order"] = order
    state["counts"] = torch.bincount(key.long(), minlength=E + 1)[:E].tolist()
    state["weights"] = torch.softmax(best, dim=1)
    if own:
        state["plan"] = _experts().sort_tokens(ids, E)

    dtype = _TYPES[case["type"]]
    if case["op"] == "gather":
        state["x"] = normal(T, case["width"]).to(dtype)
        state["g"] = normal(T * k, case["width"]).to(dtype) if case["train"] else None
    elif case["op"] == "combine":
        state["y"] = normal(T * k, case["width"]).to(dtype)
        state["g"] = normal(T, case["width"]).to(dtype) if case["train"] else None
    else:
        K, N, group = case["k"], case["n"], case["group"]
        tables = (E, K // group, N) if group else (E, N)
        x = normal(T, K)
        x[:, :: max(1, K // 7)] *= 6.0                       # a few features are much larger than the rest
        state["x"] = x.to(dtype)
        state["g"] = normal(T * k, N).to(dtype) if case["train"] else None
        rows = K // 2 if case["bits"] == 4 else K
        state["packed"] = torch.randint(0, 256, (E, rows, N), generator=gen, device="cuda", dtype=torch.uint8)
        middle = 7.5 if case["bits"] == 4 else 127.5
        spread = 0.1 / (2.0 * middle)
        state["zero"] = torch.round(middle + middle * 0.3 * (2.0 * uniform(*tables) - 1.0)).to(_TYPES[case["tables"]])
        state["scale"] = (spread * (0.5 + uniform(*tables))).to(_TYPES[case["tables"]])
        if own:
            state["stack"] = _stack(state)
    return state


def _stack(state):
    case = state["case"]
    return _experts().QuantizedExperts(state["packed"], state["zero"], state["scale"], bits=case["bits"],
                                       group_size=case["group"])


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    ex = _experts()
    case, ids = state["case"], state["ids"]
    if case["op"] == "sort":
        plan = ex.sort_tokens(ids, case["experts"])
        return {"order": plan.order, "position": plan.position, "offsets": plan.offsets}
    plan = state["plan"]
    if case["op"] == "gather":
        if not case["train"]:
            return {"rows": ex.gather_tokens(state["x"], plan)}
        x = state["x"].detach().requires_grad_()
        rows = ex.gather_tokens(x, plan)
        (dx,) = torch.autograd.grad(rows, x, state["g"])
        return {"rows": rows.detach(), "dx": dx}
    if case["op"] == "combine":
        if not case["train"]:
            return {"out": ex.combine_tokens(state["y"], plan, state["weights"])}
        y, w = state["y"].detach().requires_grad_(), state["weights"].detach().requires_grad_()
        out = ex.combine_tokens(y, plan, w)
        dy, dw = torch.autograd.grad(out, (y, w), state["g"])
        return {"out": out.detach(), "dy": dy, "dw": dw}
    if not case["train"]:
        return {"y": ex.quantized_expert_matmul(state["x"], state["stack"], plan)}
    x = state["x"].detach().requires_grad_()
    y = ex.quantized_expert_matmul(x, state["stack"], plan)
    (dx,) = torch.autograd.grad(y, x, state["g"])
    return {"y": y.detach(), "dx": dx}


def _dense(state, e):
    """W[e] in 32 bits."""
    case = state["case"]
    codes = state["packed"][e]
    if case["bits"] == 4:
        codes = torch.stack((codes & 15, codes >> 4), dim=1).reshape(case["k"], case["n"])
    zero, scale = state["zero"][e].float(), state["scale"][e].float()
    if case["group"]:
        zero = zero.repeat_interleave(case["group"], dim=0)
        scale = scale.repeat_interleave(case["group"], dim=0)
    return (codes.float() - zero) * scale


def _run_plain(state):
    case, ids = state["case"], state["ids"]
    T, k, E = case["tokens"], case["top_k"], case["experts"]
    if case["op"] == "sort":
        key = torch.where((ids < 0) | (ids >= E), torch.full_like(ids, E), ids).reshape(-1)
        ordered, order = torch.sort(key, stable=True)
        position = torch.empty_like(order)
        position[order] = torch.arange(T * k, device=order.device)
        offsets = torch.searchsorted(ordered, torch.arange(E + 1, device=order.device, dtype=ordered.dtype))
        return {"order": order.int(), "position": position.int(), "offsets": offsets.int()}
    order, counts = state["order"], state["counts"]
    n = sum(counts)
    token = order[:n] // k
    if case["op"] == "gather":
        x = state["x"]
        rows = torch.zeros(T * k, x.shape[1], device=x.device, dtype=x.dtype)
        rows[:n] = x[token]
        if not case["train"]:
            return {"rows": rows}
        return {"rows": rows, "dx": _back(state["g"].float(), order, n, T, k, None).to(x.dtype)}
    if case["op"] == "combine":
        y, w = state["y"], state["weights"]
        out = _back(y.float(), order, n, T, k, w.float()).to(y.dtype)
        if not case["train"]:
            return {"out": out}
        g = state["g"].float()[token]
        dy = torch.zeros_like(y)
        dy[:n] = (g * w.reshape(-1)[order[:n], None].float()).to(y.dtype)
        dw = torch.zeros(T * k, device=y.device, dtype=torch.float32)
        dw[order[:n]] = (g * y[:n].float()).sum(dim=1)
        return {"out": out, "dy": dy, "dw": dw.reshape(T, k).to(w.dtype)}
    x = state["x"]
    rows = x[token].float()
    y = torch.zeros(T * k, case["n"], device=x.device, dtype=x.dtype)
    dr = torch.zeros(T * k, case["k"], device=x.device) if case["train"] else None
    at = 0
    for e, c in enumerate(counts):
        if c == 0:
            continue
        w = _dense(state, e)
        y[at:at + c] = (rows[at:at + c] @ w).to(x.dtype)
        if case["train"]:
            dr[at:at + c] = state["g"][at:at + c].float() @ w.t()
        at += c
    if not case["train"]:
        return {"y": y}
    return {"y": y, "dx": _back(dr, order, n, T, k, None).to(x.dtype)}


def _back(rows, order, n, T, k, weights):
    """Rows in sorted order added up at their tokens, in 32 bits."""
    pairs = torch.zeros(T * k, rows.shape[1], device=rows.device)
    pairs[order[:n]] = rows[:n]
    if weights is not None:
        pairs = pairs * weights.reshape(-1, 1)
    return pairs.reshape(T, k, -1).sum(dim=1)


# ---------------------------------------------------------------------------------------------- work
def work(case):
    T, k, E = case["tokens"], case["top_k"], case["experts"]
    P = T * k * (1.0 - case["dropped"])
    if case["op"] == "sort":
        return {"bytes": T * k * ((4 if case["index"] == "int32" else 8) + 8) + 4 * (E + 1), "flops": 2 * T * k}
    size = _BYTES[case["type"]]
    if case["op"] == "gather":
        moved = (T + T * k) * case["width"] * size
        # the gradient reads every copy and writes every token
        return {"bytes": (2 if case["train"] else 1) * moved + 8 * T * k,
                "flops": (P * case["width"] if case["train"] else 1)}
    if case["op"] == "combine":
        forward = (T + P) * case["width"] * size + 8 * T * k
        # rows and the tokens' gradients in, the rows' gradients out
        backward = (T + P + T * k) * case["width"] * size + 12 * T * k if case["train"] else 0
        return {"bytes": forward + backward, "flops": (2 + (3 if case["train"] else 0)) * P * case["width"]}
    K, N = case["k"], case["n"]
    # experts that at least one token picks, on average
    active = sum(1.0 - (1.0 - min(1.0, k * float(p))) ** T for p in _popularity(E))
    groups = K // case["group"] if case["group"] else 1
    weights = active * (K * N * case["bits"] / 8 + 2 * groups * N * _BYTES[case["tables"]])
    forward = T * K * size + T * k * N * size + 8 * T * k
    backward = T * k * N * size + T * K * size if case["train"] else 0
    return {"bytes": weights * (2 if case["train"] else 1) + forward + backward,
            "flops": 2 * P * K * N * (2 if case["train"] else 1)}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    T, k, E = case["tokens"], case["top_k"], case["experts"]
    flat = state["ids"].cpu().numpy().reshape(-1).astype(np.int64)
    members = [np.flatnonzero(flat == e) for e in range(E)]
    rest = np.flatnonzero((flat < 0) | (flat >= E))
    order = np.concatenate(members + [rest])
    starts = np.concatenate(([0], np.cumsum([len(m) for m in members])))
    if case["op"] == "sort":
        position = np.empty_like(order)
        for p, pair in enumerate(order.tolist()):
            position[pair] = p
        return {"order": order.astype(np.int32), "position": position.astype(np.int32),
                "offsets": starts.astype(np.int32)}
    live = int(starts[-1])
    pair = torch.from_numpy(order[:live]).cuda()
    token = pair // k
    if case["op"] == "gather":
        x = state["x"].double()
        rows = torch.cat((x.index_select(0, token), x.new_zeros(T * k - live, x.shape[1])))
        if not case["train"]:
            return {"rows": rows}
        dx = torch.zeros_like(x).index_add_(0, token, state["g"][:live].double())
        return {"rows": rows, "dx": dx}
    if case["op"] == "combine":
        y, w = state["y"][:live].double(), state["weights"].double().reshape(-1)
        out = torch.zeros(T, case["width"], dtype=torch.float64, device="cuda")
        out.index_add_(0, token, y * w[pair][:, None])
        if not case["train"]:
            return {"out": out}
        g = state["g"].double().index_select(0, token)
        tail = T * k - live
        dy = torch.cat((g * w[pair][:, None], g.new_zeros(tail, case["width"])))
        dw = torch.zeros(T * k, dtype=torch.float64, device="cuda")
        dw[pair] = torch.linalg.vecdot(g, y)
        return {"out": out, "dy": dy, "dw": dw.reshape(T, k)}
    K, N = case["k"], case["n"]
    y = torch.zeros(T * k, N, dtype=torch.float64, device="cuda")
    dx = torch.zeros(T, K, dtype=torch.float64, device="cuda")
    feature = torch.arange(K, device="cuda")
    for e in range(E):
        a, b = int(starts[e]), int(starts[e + 1])
        if a == b:
            continue
        if case["bits"] == 4:
            byte = state["packed"][e].index_select(0, feature // 2).long()
            codes = (byte >> (4 * (feature % 2))[:, None]) % 16
        else:
            codes = state["packed"][e].long()
        if case["group"]:
            zero = state["zero"][e].double().index_select(0, feature // case["group"])
            scale = state["scale"][e].double().index_select(0, feature // case["group"])
        else:
            zero, scale = state["zero"][e].double()[None], state["scale"][e].double()[None]
        w = scale * codes.double() - scale * zero
        y[a:b] = torch.mm(state["x"].double().index_select(0, token[a:b]), w)
        if case["train"]:
            dx.index_add_(0, token[a:b], torch.mm(state["g"][a:b].double(), w.t()))
    return {"y": y, "dx": dx} if case["train"] else {"y": y}
