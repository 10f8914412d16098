"""The performance cases of what a training step has around a model's linear
layers: the dense product with bias, activation and residual, forward and
backward; the router of a layer of experts with its balance loss; the norm of
all gradients and their clipping.

Fields of a case, by its "op":

    linear         y = act(x W^T + b) + r: rows M, N, K, dtype, act ("none",
                   "relu", "gelu", "gelu_tanh", "silu"), bias, residual; wt: W is
                   the transposed view of [K, N]
    linear_train   the same and the gradients of x, W and b for a given dy
    route          the router: tokens T, experts E, k of each token, dtype of the
                   logits, normalize (the k weights sum to 1), padded (share of
                   the tokens that are padding, masked out)
    route_train    the same and the logits' gradient from those of the weights and
                   of the balance loss
    norm           the norm of all gradients: tensors, elements in all, dtype
                   ("mixed": matrices in bfloat16, vectors in float32), odd: sizes
                   as they fall, not whole matrices
    clip           the same, and the gradients scaled to a norm of at most `limit`
                   times what these inputs have on average, into buffers of their own
"""
import math
import random

import torch

own = False

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _named(name, case):
    return dict(case, name=name) if name else case


def _linear(name, op, M, N, K, dtype, act, bias=True, residual=False, wt=False):
    return _named(name, dict(op=op, M=M, N=N, K=K, dtype=dtype, act=act, bias=bias,
                             residual=residual, wt=wt))


def _route(name, op, T, E, k, dtype, normalize=True, padded=0.0):
    return _named(name, dict(op=op, T=T, E=E, k=k, dtype=dtype, normalize=normalize, padded=padded))


def _grads(name, op, tensors, elements, dtype, limit=0.0, odd=False):
    return _named(name, dict(op=op, tensors=tensors, elements=elements, dtype=dtype, limit=limit,
                             odd=odd))


def listed():
    return [
        # one token through a square layer that adds to the residual stream: the latency of serving
        _linear("linear_token_bf16", "linear", 1, 4096, 4096, "bfloat16", "none", residual=True),
        # a batch of sequences, one token each, through a large layer with its activation
        _linear("linear_batch_f16", "linear", 32, 8192, 8192, "float16", "gelu"),
        # a prompt through the first layer of a feed-forward block
        _linear("linear_prompt_bf16", "linear", 4096, 4096, 1024, "bfloat16", "gelu_tanh"),
        # a training batch through it, with every gradient
        _linear("linear_train_bf16", "linear_train", 8192, 4096, 2048, "bfloat16", "gelu"),
        # a short batch whose sizes are no round numbers, with every gradient
        _linear("linear_train_ragged_f16", "linear_train", 1999, 520, 1000, "float16", "silu",
                residual=True),
        # a few sequences decoded at once: the router of one layer
        _route("route_decode_bf16", "route", 16, 16, 2, "bfloat16"),
        # a training batch with many small experts, with the logits' gradient
        _route("route_train_f32", "route_train", 32768, 64, 8, "float32"),
        # a padded batch, sizes no round numbers, weights straight from the softmax
        _route("route_train_padded_bf16", "route_train", 4099, 40, 3, "bfloat16", False, 0.25),
        # the gradients of one layer of experts: a few tensors, where latency counts
        _grads("norm_layer_f32", "norm", 5, 1 << 20, "float32"),
        # a model's gradients, clipped in every step of the warm-up
        _grads("clip_model_bf16", "clip", 60, 1 << 28, "bfloat16", 0.5),
        # matrices in 16 bits and vectors in 32, odd sizes, within the limit: nothing to scale
        _grads("clip_mixed_within", "clip", 43, 10000019, "mixed", 2.0, odd=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _extent(rng, lo, hi):
    """A size of lo .. hi, uniform in its logarithm: half of them multiples of
    64, a tenth of 4, the others odd or even as they fall."""
    n, kind = _log_uniform(rng, lo, hi), rng.random()
    step = 64 if kind < 0.5 else 4 if kind < 0.6 else 1
    return max(lo, min(hi, (n + step // 2) // step * step))


def draw(rng):
    while True:
        op = rng.choice(["linear"] * 3 + ["linear_train"] * 2 + ["route"] * 2 + ["route_train"] * 2 +
                        ["norm"] + ["clip"] * 2)
        if op.startswith("linear"):
            M = _log_uniform(rng, 1, 8192 if rng.random() < 0.6 else 64)
            case = _linear(None, op, M, _extent(rng, 64, 8192), _extent(rng, 64, 8192),
                           rng.choice(["bfloat16", "bfloat16", "float16"]),
                           # the step of relu's derivative: which side a sum next to 0 falls on
                           # is a matter of its order, so no gradients of it
                           rng.choice([a for a in ACTS if op == "linear" or a != "relu"]),
                           rng.random() < 0.7, rng.random() < 0.4, rng.random() < 0.25)
        elif op.startswith("route"):
            E = _log_uniform(rng, 2, 512)
            case = _route(None, op, _log_uniform(rng, 1, 32768), E, rng.randint(1, min(E, 8)),
                          rng.choice(["float32", "float32", "bfloat16", "float16"]),
                          rng.random() < 0.7, rng.choice([0.0, 0.0, round(rng.uniform(0, 0.9), 2)]))
        else:
            tensors = _log_uniform(rng, 1, 300 if op == "norm" else 60)
            case = _grads(None, op, tensors, _log_uniform(rng, max(1000, tensors), 1 << 28),
                          rng.choice(["bfloat16", "float32", "float16", "mixed"]),
                          0.0 if op == "norm" else rng.choice([0.1, 0.5, 2.0]), rng.random() < 0.5)
            if case["dtype"] in ("float32", "mixed"):
                case["elements"] = min(case["elements"], 1 << 27)
        # no dearer than the largest listed one
        if work(case)["flops"] <= 4.13e11:
            return case


def _dtype(case):
    return getattr(torch, case["dtype"])


def _sizes(case):
    """(elements, dtype) of each gradient: matrices and, after every three, a
    vector of the square root of a matrix's size."""
    n, left = case["tensors"], case["elements"]
    mixed = case["dtype"] == "mixed"
    rng = random.Random(n * 1000003 + left)
    vector = [i % 4 == 3 for i in range(n)]
    share = [rng.uniform(0.2, 1) if case["odd"] else 1.0 for _ in range(n)]
    whole = left / sum(s for s, v in zip(share, vector) if not v)
    sizes = []
    for s, v in zip(share, vector):
        size = max(1, int(math.sqrt(s * whole) if v else s * whole))
        if not case["odd"] and size >= 64:
            size -= size % 64
        dtype = (torch.float32 if v else torch.bfloat16) if mixed else _dtype(case)
        sizes.append((size, dtype))
    return sizes


def _normal(g, dtype, *size):
    return torch.randn(*size, generator=g, device="cuda").to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op.startswith("linear"):
        dt, M, N, K = _dtype(case), case["M"], case["N"], case["K"]
        x = _normal(g, dt, M, K)
        W = (_normal(g, torch.float32, N, K) / math.sqrt(K)).to(dt)
        if case["wt"]:
            W = W.mT.contiguous().mT
        b = (0.5 * _normal(g, torch.float32, N)).to(dt) if case["bias"] else None
        r = _normal(g, dt, M, N) if case["residual"] else None
        state = dict(case=case, x=x, W=W, b=b, r=r)
        if op == "linear_train":
            state["dy"] = _normal(g, dt, M, N)
            for t in (x, W, b):
                if t is not None:
                    t.requires_grad_()
        return state
    if op.startswith("route"):
        T, E = case["T"], case["E"]
        # experts are not equally liked
        logits = (_normal(g, torch.float32, T, E) + 0.5 * _normal(g, torch.float32, E)).to(_dtype(case))
        mask = None
        if case["padded"]:
            mask = torch.rand(T, generator=g, device="cuda") >= case["padded"]
        state = dict(case=case, logits=logits, mask=mask)
        if op == "route_train":
            state["dw"] = _normal(g, torch.float32, T, case["k"]) / T
            state["dloss"] = torch.full((), 0.01, device="cuda")
            logits.requires_grad_()
        return state
    grads, square = [], 0.0
    rng = random.Random(seed)
    for size, dtype in _sizes(case):
        scale = math.exp(rng.uniform(math.log(1e-4), math.log(1e-1)))
        grads.append((scale * _normal(g, torch.float32, size)).to(dtype))
        square += size * scale * scale
    state = dict(case=case, grads=grads)
    if op == "clip":
        state["limit"] = case["limit"] * math.sqrt(square)
        state["out"] = [torch.empty_like(t) for t in grads]
    return state


def _act(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * torch.sigmoid(-z))
    if act == "gelu":
        # the normal distribution's tail by erfc: 1 + erf loses it where z is well below 0
        tail = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * tail, tail + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    a, c = 2 * math.sqrt(2 / math.pi), 0.044715
    s = torch.sigmoid(a * (z + c * z * z * z))
    return z * s, s + z * s * torch.sigmoid(-a * (z + c * z * z * z)) * (a * (1 + 3 * c * z * z))


def _plain_linear(state, train):
    case, x, W = state["case"], state["x"].detach().float(), state["W"].detach().float()
    dt = state["x"].dtype
    z = torch.matmul(x, W.mT)
    if state["b"] is not None:
        z = z + state["b"].detach().float()
    y, d = _act(z, case["act"])
    if state["r"] is not None:
        y = y + state["r"].float()
    if not train:
        return y.to(dt)
    dz = state["dy"].float() * d
    out = [y.to(dt), torch.matmul(dz, W).to(dt), torch.matmul(dz.mT, x).to(dt)]
    if state["b"] is not None:
        out.append(dz.sum(0, dtype=torch.float64).to(dt))
    return out


def _plain_route(state, train):
    case, mask = state["case"], state["mask"]
    logits = state["logits"].detach().float()
    T, E, k = case["T"], case["E"], case["k"]
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    # the greatest first, of equal ones the lowest index
    experts = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    chosen = p.gather(1, experts)
    total = chosen.sum(1, keepdim=True)
    weights = chosen / total if case["normalize"] else chosen
    valid = torch.ones(T, dtype=torch.bool, device=p.device) if mask is None else mask
    weights = torch.where(valid[:, None], weights, 0.0)
    experts = torch.where(valid[:, None], experts, E)
    flat = experts.flatten()
    order = torch.sort(flat, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device=p.device)
    counts = (flat[:, None] == torch.arange(E, device=p.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    n = valid.sum().clamp(min=1)
    p = torch.where(valid[:, None], p, 0.0)
    f = counts.double() / (n * k)
    loss = (E * (f * (p.sum(0, dtype=torch.float64) / n)).sum()).float()
    out = [experts, order, place.view(T, k), offsets, counts]
    out = [v.to(torch.int32) for v in out] + [weights, loss]
    if train:
        dw = torch.where(valid[:, None], state["dw"], 0.0)
        grad = (state["dloss"] * E * f / n).float().expand(T, E)
        safe = torch.where(valid[:, None], experts, 0)
        if case["normalize"]:
            dl = torch.zeros_like(p).scatter_add(
                1, safe, weights * (dw - (weights * dw).sum(1, keepdim=True)))
        else:
            dl = torch.zeros_like(p)
            grad = grad.scatter_add(1, safe, dw)
        dl = dl + p * (grad - (p * grad).sum(1, keepdim=True))
        out.append(dl.to(state["logits"].dtype))
    return out


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        import ozaki_triton_amd as ozk
        if op.startswith("linear"):
            act = None if case["act"] == "none" else case["act"]
            y = ozk.fused_linear(state["x"], state["W"], state["b"], activation=act,
                                 residual=state["r"])
            if op == "linear":
                return y
            leaves = [t for t in (state["x"], state["W"], state["b"]) if t is not None]
            return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]
        if op.startswith("route"):
            r = ozk.route_tokens(state["logits"], case["k"], mask=state["mask"],
                                 normalize=case["normalize"])
            out = [r.experts, r.order, r.place, r.offsets, r.counts, r.weights.detach(),
                   r.balance_loss.detach()]
            if op == "route_train":
                out += torch.autograd.grad([r.weights, r.balance_loss], [state["logits"]],
                                           [state["dw"], state["dloss"]])
            return out
        if op == "norm":
            return ozk.gradient_norm(state["grads"])
        return [ozk.clip_gradients(state["grads"], state["limit"], out=state["out"]), *state["out"]]
    if op.startswith("linear"):
        return _plain_linear(state, op == "linear_train")
    if op.startswith("route"):
        return _plain_route(state, op == "route_train")
    square = sum(t.float().square().sum(dtype=torch.float64) for t in state["grads"])
    norm = square.sqrt()
    if op == "norm":
        return norm.float()
    factor = (state["limit"] / norm).clamp(max=1).float()
    return [norm.float(), *[(t.float() * factor).to(t.dtype) for t in state["grads"]]]


def exact(case, seed):
    state, op = prepare(case, seed), case["op"]
    if op.startswith("linear"):
        train = op == "linear_train"
        x, W, b, r = [None if state[n] is None else state[n].detach().double().contiguous()
                      for n in ("x", "W", "b", "r")]
        leaves = [t for t in (x, W, b) if t is not None]
        for t in leaves:
            t.requires_grad_(train)
        z = x @ W.T if b is None else x @ W.T + b
        act = case["act"]
        if act == "relu":
            y = torch.relu(z)
        elif act == "gelu":
            y = z * torch.special.ndtr(z)
        elif act == "gelu_tanh":
            y = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
        elif act == "silu":
            y = z / (1 + torch.exp(-z))
        else:
            y = z
        if r is not None:
            y = y + r
        if not train:
            return y
        return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"].double())]
    if op.startswith("route"):
        T, E, k, mask = case["T"], case["E"], case["k"], state["mask"]
        valid = torch.ones(T, dtype=torch.bool, device="cuda") if mask is None else mask
        x = state["logits"].detach().double()[valid].requires_grad_()
        n = x.shape[0]
        p = torch.softmax(x, 1)
        chosen = torch.sort(-x.detach(), dim=1, stable=True).indices[:, :k]
        w = torch.softmax(x.gather(1, chosen), 1) if case["normalize"] else p.gather(1, chosen)
        experts = torch.full((T, k), E, device="cuda")
        experts[valid] = chosen
        # each slot's place: those of lower experts, and of its own before it
        flat = experts.flatten()
        counts = torch.bincount(flat, minlength=E + 1)
        starts = counts.cumsum(0) - counts
        place = torch.empty_like(flat)
        for e in range(E + 1):
            at = (flat == e).nonzero()[:, 0]
            place[at] = starts[e] + torch.arange(at.shape[0], device="cuda")
        order = torch.empty_like(flat)
        order[place] = torch.arange(T * k, device="cuda")
        f = counts[:E].double() / max(n * k, 1)
        loss = E * (f * p.sum(0)).sum() / max(n, 1)
        weights = torch.zeros(T, k, dtype=torch.float64, device="cuda")
        weights[valid] = w.detach()
        out = [experts, order, place.view(T, k), starts, counts[:E]]
        out = [v.to(torch.int32) for v in out] + [weights, loss.detach()]
        if op == "route_train":
            dl = torch.zeros(T, E, dtype=torch.float64, device="cuda")
            if n:
                dl[valid] = torch.autograd.grad([w, loss], [x], [state["dw"].double()[valid],
                                                                 state["dloss"].double()])[0]
            out.append(dl)
        return out
    square = torch.zeros((), dtype=torch.float64, device="cuda")
    for t in state["grads"]:
        square += torch.dot(t.double(), t.double())
    norm = square.sqrt()
    if op == "norm":
        return norm
    factor = min(1.0, state["limit"] / float(norm))
    return [norm, *[t.double() * factor for t in state["grads"]]]


def work(case):
    op = case["op"]
    if op.startswith("linear"):
        M, N, K = case["M"], case["N"], case["K"]
        elements = M * K + N * K + M * N * (2 if case["residual"] else 1)
        elements += N if case["bias"] else 0
        if op == "linear":
            return {"bytes": 2.0 * elements, "flops": 2.0 * M * N * K}
        elements += M * N + M * K + N * K + (N if case["bias"] else 0)
        return {"bytes": 2.0 * elements, "flops": 6.0 * M * N * K}
    if op.startswith("route"):
        T, E, k = case["T"], case["E"], case["k"]
        size = torch.empty(0, dtype=_dtype(case)).element_size()
        moved = T * E * size + T * k * 16 + 8 * E + (T if case["padded"] else 0)
        if op == "route_train":
            moved += T * k * 4 + T * E * size
        return {"bytes": float(moved), "flops": (15.0 if op == "route_train" else 5.0) * T * E}
    moved = sum(size * torch.empty(0, dtype=dtype).element_size() for size, dtype in _sizes(case))
    return {"bytes": moved * (1.0 if op == "norm" else 2.0),
            "flops": case["elements"] * (2.0 if op == "norm" else 3.0)}
