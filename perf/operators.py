"""The performance cases of the operators for a model's linear layers: expert
(grouped) products with their gradients, products with 4-bit weights, and the
orthogonalised update of a weight matrix.

Fields of a case, by its "op":

    grouped        C[t] = A[t] B[g] for the rows t of group g: rows T, groups
                   G, K, N, dtype; skew: how uneven the groups are (0: every
                   group as likely, 1: log-normal shares); spare: rows at the
                   end of the buffer that belong to no group; bt: B is the
                   transposed view of [G, N, K]
    grouped_back   the gradients dA and dB of the same product
    w4             y = x W^T, W of 4 bits in groups of `group` along K: M, N, K;
                   dtype of x and y; zeros: with zero points
    quantize       a weight matrix to 4 bits and back: N, K, group, dtype, zeros
    orth           Newton-Schulz orthogonalisation of [batch, M, N], dtype, steps
"""
import math
import random

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


def _grouped(name, op, T, G, K, N, dtype, skew, spare=0, bt=False):
    c = dict(op=op, T=T, G=G, K=K, N=N, dtype=dtype, skew=skew, spare=spare, bt=bt)
    return dict(c, name=name) if name else c


def _w4(name, M, N, K, group, dtype, zeros):
    c = dict(op="w4", M=M, N=N, K=K, group=group, dtype=dtype, zeros=zeros)
    return dict(c, name=name) if name else c


def _quantize(name, N, K, group, dtype, zeros):
    c = dict(op="quantize", N=N, K=K, group=group, dtype=dtype, zeros=zeros)
    return dict(c, name=name) if name else c


def _orth(name, batch, M, N, dtype, steps=5):
    c = dict(op="orth", batch=batch, M=M, N=N, dtype=dtype, steps=steps)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a few tokens decoded at once: each expert that is hit reads its weights for a row or two
        _grouped("experts_decode_bf16", "grouped", 16, 16, 1024, 2048, "bfloat16", 1),
        # one sequence's prompt through a layer that stores its weights [N, K], experts unevenly hit
        _grouped("experts_prompt_f16", "grouped", 4096, 8, 1024, 4096, "float16", 1, bt=True),
        # a training batch's forward pass, the buffer a little longer than its rows
        _grouped("experts_train_bf16", "grouped", 32768, 16, 2048, 4096, "bfloat16", 0, spare=96),
        # the backward pass of a training batch with many experts
        _grouped("experts_back_bf16", "grouped_back", 16384, 32, 2048, 1024, "bfloat16", 1),
        # the backward pass of a short batch whose sizes are no round numbers
        _grouped("experts_back_ragged_f16", "grouped_back", 1999, 7, 1000, 520, "float16", 1),
        # one token through a square layer: the latency of serving
        _w4("w4_token_bf16", 1, 4096, 4096, 128, "bfloat16", False),
        # a batch of sequences, one token each, through a large layer with zero points
        _w4("w4_batch_f16", 32, 8192, 8192, 128, "float16", True),
        # odd sizes, short groups, full-precision activations
        _w4("w4_ragged_f32", 5, 1000, 2047, 32, "float32", True),
        # a layer's weights brought to 4 bits when a model is loaded
        _quantize("quantize_bf16", 8192, 8192, 128, "bfloat16", False),
        # the same of odd sizes, with zero points
        _quantize("quantize_ragged_f32", 1000, 2047, 32, "float32", True),
        # the optimiser's step on the small matrices of one layer's experts
        _orth("update_experts_f32", 8, 256, 512, "float32"),
        # the optimiser's step on one large matrix
        _orth("update_large_bf16", 1, 2048, 8192, "bfloat16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _extent(rng, lo, hi):
    """A size of lo .. hi, uniform in its logarithm: half of them multiples of
    64, a tenth of 4, the others odd or even as they fall."""
    n, kind = _log_uniform(rng, lo, hi), rng.random()
    step = 64 if kind < 0.5 else 4 if kind < 0.6 else 1
    n = max(lo, min(hi, (n + step // 2) // step * step))
    return n + step if n == 48 * 64 else n


def draw(rng):
    while True:
        op = rng.choice(["grouped"] * 3 + ["grouped_back"] * 3 + ["w4"] * 3 + ["quantize"] +
                        ["orth"] * 2)
        if op.startswith("grouped"):
            T, G = _log_uniform(rng, 1, 32768), _log_uniform(rng, 1, 64)
            K, N = _extent(rng, 64, 4096), _extent(rng, 64, 4096)
            case = _grouped(None, op, T, G, K, N, rng.choice(["bfloat16", "bfloat16", "float16"]),
                            rng.choice([0, 1]), rng.choice([0, 0, rng.randint(1, 200)]),
                            rng.random() < 0.5)
            ok = G * K * N <= 1 << 27 and G * T * max(K, N) <= 1 << 30
        elif op == "w4":
            case = _w4(None, _log_uniform(rng, 1, 64), _extent(rng, 64, 16384),
                       _extent(rng, 64, 16384), rng.choice([32, 64, 128]),
                       rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
                       rng.random() < 0.5)
            ok = case["N"] * case["K"] <= 1 << 27
        elif op == "quantize":
            case = _quantize(None, _extent(rng, 64, 8192), _extent(rng, 64, 8192),
                             rng.choice([32, 64, 128]), rng.choice(["bfloat16", "float16", "float32"]),
                             rng.random() < 0.5)
            ok = True
        else:
            case = _orth(None, 1 if rng.random() < 0.5 else _log_uniform(rng, 2, 32),
                         _extent(rng, 64, 8192), _extent(rng, 64, 8192),
                         rng.choice(["float32", "bfloat16", "bfloat16", "float16"]),
                         rng.choice([3, 5, 5, 6]))
            ok = case["batch"] * case["M"] * case["N"] <= 1 << 24
        # no dearer than the largest listed case
        if ok and work(case)["flops"] <= 5.8e11:
            return case


def _dtype(case):
    return getattr(torch, case["dtype"])


def _counts(case, seed):
    """Rows of each group: T rows, each of a group drawn by its share."""
    rng = random.Random(seed)
    share = [math.exp(rng.gauss(0, 1)) if case["skew"] else 1.0 for _ in range(case["G"])]
    counts = [0] * case["G"]
    for g in rng.choices(range(case["G"]), share, k=case["T"]):
        counts[g] += 1
    return counts


def _quantized(W, group, zeros):
    """The 4-bit form of W [N, K] in plain torch: whole numbers q of 0 .. 15
    [N, K], scales [N, groups] in W's type, zero points [N, groups]."""
    N, K = W.shape
    groups = -(-K // group)
    w = torch.nn.functional.pad(W.float(), (0, groups * group - K)).view(N, groups, group)
    if zeros:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scale = ((hi - lo) * (1 / 15)).to(W.dtype)
        s = scale.float()
        zero = torch.where(s > 0, torch.round(-lo / s), 0.0).clamp(0, 15)
    else:
        scale = (w.abs().amax(-1) * (1 / 7)).to(W.dtype)
        s = scale.float()
        zero = torch.full_like(s, 8.0)
    q = torch.where(s[..., None] > 0, torch.round(w / s[..., None]), 0.0) + zero[..., None]
    q = q.clamp(0, 15).to(torch.uint8).view(N, groups * group)[:, :K]
    return q, scale, zero.to(torch.uint8)


def _packed(q):
    """Two values a byte, the even one in the low half; rows of whole 16 bytes."""
    N, K = q.shape
    q = torch.nn.functional.pad(q, (0, -K % 32))
    return q[:, 0::2] | (q[:, 1::2] << 4)


def _normal(g, dtype, *size):
    return torch.randn(*size, generator=g, device="cuda").to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = _dtype(case), case["op"]
    if op.startswith("grouped"):
        rows, G, K, N = case["T"] + case["spare"], case["G"], case["K"], case["N"]
        counts = _counts(case, seed)
        offsets = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
        A = _normal(g, dt, rows, K)
        B = (_normal(g, dt, G, N, K) / math.sqrt(K)).to(dt)
        B = B.mT if case["bt"] else B.mT.contiguous()
        # the greatest count: what a program that pads its groups allots for each
        state = dict(case=case, A=A, B=B, offsets=offsets, most=max(counts))
        if op == "grouped_back":
            state["D"] = _normal(g, dt, rows, N)
        return state
    if op == "w4":
        W = torch.randn(case["N"], case["K"], generator=g, device="cuda") / math.sqrt(case["K"])
        scale_type = torch.float32 if dt == torch.float32 else dt
        q, scales, zeros = _quantized(W.to(scale_type), case["group"], case["zeros"])
        return dict(case=case, x=_normal(g, dt, case["M"], case["K"]), packed=_packed(q),
                    scales=scales, zeros=zeros if case["zeros"] else None)
    if op == "quantize":
        return dict(case=case, W=(_normal(g, torch.float32, case["N"], case["K"]) /
                                  math.sqrt(case["K"])).to(dt))
    # a gradient's momentum: a few strong directions over a weak rest
    b, M, N = case["batch"], case["M"], case["N"]
    r = min(M, N, 32)
    left = torch.randn(b, M, r, generator=g, device="cuda") * torch.logspace(0, -1, r, device="cuda")
    right = torch.randn(b, r, N, generator=g, device="cuda")
    G = 1e-3 * (torch.matmul(left, right) + 0.5 * torch.randn(b, M, N, generator=g, device="cuda"))
    return dict(case=case, G=G.to(dt))


def _places(state):
    """Each row's group and its place there, and whether it has a group."""
    offsets, rows = state["offsets"].long(), state["A"].shape[0]
    t = torch.arange(rows, device=offsets.device)
    group = torch.searchsorted(offsets[1:], t, right=True)
    inside = group < state["case"]["G"]
    group = group.clamp(max=state["case"]["G"] - 1)
    place = torch.where(inside, t - offsets[group], state["most"])
    return group, place, inside


def _padded(state, X, group, place):
    """X's rows as [G, most + 1, columns] in 32 bits: the last place of a group
    takes the rows that have none, and is not kept."""
    P = torch.zeros(state["case"]["G"], state["most"] + 1, X.shape[1], device=X.device)
    P[group, place] = X.float()
    P[:, state["most"]] = 0
    return P


def _plain_w4(state):
    case, packed = state["case"], state["packed"]
    q = torch.stack((packed & 15, packed >> 4), -1).flatten(1)[:, :case["K"]].float()
    s = state["scales"].float().repeat_interleave(case["group"], 1)[:, :case["K"]]
    z = 8.0 if state["zeros"] is None else \
        state["zeros"].float().repeat_interleave(case["group"], 1)[:, :case["K"]]
    W = (q - z) * s
    return torch.matmul(state["x"].float(), W.mT).to(state["x"].dtype)


def _plain_orth(G, steps):
    a, b, c = COEFFICIENTS
    X = G.float()
    if G.shape[-2] > G.shape[-1]:
        X = X.mT.contiguous()
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(steps):
        A = torch.matmul(X, X.mT)
        X = a * X + torch.matmul(b * A + c * torch.matmul(A, A), X)
    if G.shape[-2] > G.shape[-1]:
        X = X.mT.contiguous()
    return X.to(G.dtype)


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        import ozaki_triton_amd as ozk
        if op == "grouped":
            return ozk.grouped_matmul(state["A"], state["B"], state["offsets"])
        if op == "grouped_back":
            return ozk.grouped_matmul_backward(state["D"], state["A"], state["B"], state["offsets"])
        if op == "w4":
            return ozk.matmul_w4(state["x"], state["packed"], state["scales"], state["zeros"],
                                 group_size=case["group"])
        if op == "quantize":
            packed, scales, zeros = ozk.quantize_w4(state["W"], case["group"], zeros=case["zeros"])
            W = ozk.dequantize_w4(packed, scales, zeros, group_size=case["group"], K=case["K"])
            return (W, scales) if zeros is None else (W, scales, zeros)
        return ozk.orthogonalize(state["G"], case["steps"], COEFFICIENTS, EPS)
    if op.startswith("grouped"):
        group, place, inside = _places(state)
        keep = inside[:, None]
        A, dt = _padded(state, state["A"], group, place), state["A"].dtype
        if op == "grouped":
            C = torch.matmul(A, state["B"].float())[group, place]
            return torch.where(keep, C, 0.0).to(dt)
        D = _padded(state, state["D"], group, place)
        dA = torch.matmul(D, state["B"].float().mT)[group, place]
        return torch.where(keep, dA, 0.0).to(dt), torch.matmul(A.mT, D).to(dt)
    if op == "w4":
        return _plain_w4(state)
    if op == "quantize":
        q, scales, zeros = _quantized(state["W"], case["group"], case["zeros"])
        spread = [v.float().repeat_interleave(case["group"], 1)[:, :case["K"]]
                  for v in (zeros, scales)]
        W = ((q.float() - spread[0]) * spread[1]).to(state["W"].dtype)
        return (W, scales, zeros) if case["zeros"] else (W, scales)
    return _plain_orth(state["G"], case["steps"])


def exact(case, seed):
    state, op = prepare(case, seed), case["op"]
    if op.startswith("grouped"):
        # group by group, by the row counts that the inputs were made with
        A, B, ends = state["A"].double(), state["B"].double(), [0]
        for n in _counts(case, seed):
            ends.append(ends[-1] + n)
        spans = [slice(lo, hi) for lo, hi in zip(ends, ends[1:])]
        if op == "grouped":
            C = A.new_zeros(A.shape[0], case["N"])
            for n, at in enumerate(spans):
                C[at] = A[at] @ B[n]
            return C
        D = state["D"].double()
        dA, dB = torch.zeros_like(A), torch.zeros_like(B, memory_format=torch.contiguous_format)
        for n, at in enumerate(spans):
            dA[at] = D[at] @ B[n].T.contiguous()
            dB[n] = A[at].T.contiguous() @ D[at]
        return dA, dB
    if op == "w4":
        x, packed, K = state["x"].double(), state["packed"].long(), case["K"]
        y = x.new_zeros(case["M"], case["N"])
        for n, lo in enumerate(range(0, K, case["group"])):
            k = torch.arange(lo, min(K, lo + case["group"]), device=x.device)
            q = (packed[:, k // 2] >> (4 * (k % 2))) % 16
            z = 8 if state["zeros"] is None else state["zeros"][:, n:n + 1].long()
            y += (x[:, k] @ (q - z).double().T.contiguous()) * state["scales"][:, n].double()
        return y
    if op == "quantize":
        # rounding decides each value: in 64 bits other ones fall on the other
        # side, so only the scales before their own rounding have such a value
        W = state["W"].double()
        parts = W.split(case["group"], 1)
        if case["zeros"]:
            scales = [(p.amax(1).clamp(min=0) - p.amin(1).clamp(max=0)) / 15 for p in parts]
            return None, torch.stack(scales, 1), None
        return None, torch.stack([p.abs().amax(1) / 7 for p in parts], 1)
    G = state["G"].double()
    a, b, c = COEFFICIENTS
    X = G / (torch.linalg.vector_norm(G, dim=(-2, -1), keepdim=True) + EPS)
    for _ in range(case["steps"]):
        # X (a + b S + c S^2) with S the smaller of the two squares
        if case["M"] <= case["N"]:
            S = torch.matmul(X, X.mT.contiguous())
            X = a * X + b * torch.matmul(S, X) + c * torch.matmul(S, torch.matmul(S, X))
        else:
            S = torch.matmul(X.mT.contiguous(), X)
            X = a * X + b * torch.matmul(X, S) + c * torch.matmul(torch.matmul(X, S), S)
    return X


def work(case):
    op, size = case["op"], torch.empty(0, dtype=_dtype(case)).element_size()
    if op.startswith("grouped"):
        rows, K, N = case["T"] + case["spare"], case["K"], case["N"]
        hit = min(case["G"], case["T"])          # a group without rows reads no weights
        if op == "grouped":
            return {"bytes": size * (case["T"] * K + hit * K * N + rows * N) + 4 * case["G"],
                    "flops": 2.0 * case["T"] * K * N}
        return {"bytes": size * (case["T"] * (K + N) + hit * K * N + rows * K +
                                 case["G"] * K * N) + 4 * case["G"],
                "flops": 4.0 * case["T"] * K * N}
    N, K = case["N"], case.get("K", 0)
    if op in ("w4", "quantize"):
        each = size + (1 if case["zeros"] else 0)
        groups = -(-K // case["group"])
        if op == "w4":
            return {"bytes": N * K / 2 + N * groups * each + size * case["M"] * (N + K),
                    "flops": 2.0 * case["M"] * N * K}
        # the matrix in, its 4-bit form out and in again, the matrix out
        return {"bytes": 2 * size * N * K + 2 * (N * K / 2 + N * groups * each), "flops": 4.0 * N * K}
    m, n = sorted((case["M"], case["N"]))
    # two products of a matrix with its own transpose (half of each is the other half), one full
    return {"bytes": 2.0 * size * case["batch"] * m * n,
            "flops": case["steps"] * case["batch"] * (3.0 * m * m * n + 1.0 * m * m * m)}
