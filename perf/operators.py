"""Measured cases of the trainer's parameter operators: Muon's update of weight matrices (the orthogonalisation by
Newton-Schulz products, alone and inside the whole step) and learned row tables (the lookup of rows by index and the
gradient of the table).

``run`` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, with
``own`` set, by the framework's entry points on the same state; ``exact`` gives the definition's values in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False     # True: the framework's kernels

# the quintic's coefficients a, b, c (p(s) = a s + b s^3 + c s^5), the steps and the least norm of torch's Muon
COEFF = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# the weight matrices of the `grid` method with one rgb modality: SDF, radiance and head MLPs, the background's
RENDER_MLPS = ("256x71,256x256,257x256,256x317,256x256,256x256,64x256,64x64,3x64,256x39,256x256,256x256,256x256,"
               "256x283,256x256,256x256,128x256,1x256,3x128")


def listed():
    return [
        # the renderer's own matrices: latency, and every oddity of their shapes
        {"name": "ns_render_mlps_f32", "op": "ns", "shapes": RENDER_MLPS, "dtype": "f32"},
        # a stack of odd matrices, each its own problem
        {"name": "ns_stack_odd_f32", "op": "ns", "shapes": "6x701x1100", "dtype": "f32"},
        # the feed-forward matrices of eight blocks, wide
        {"name": "ns_blocks_bf16", "op": "ns", "shapes": "8x1024x4096", "dtype": "bf16"},
        # one large square projection
        {"name": "ns_large_bf16", "op": "ns", "shapes": "4096x4096", "dtype": "bf16"},
        # one training step's update of the renderer
        {"name": "muon_render_mlps_f32", "op": "muon", "shapes": RENDER_MLPS, "dtype": "f32"},
        # the update of one wide block with 32-bit master weights: four projections, a feed-forward pair
        {"name": "muon_block_f32", "op": "muon", "shapes": "4x2048x2048,5632x2048,2048x5632", "dtype": "f32"},
        # the same kind of block with 16-bit weights, tall and wide
        {"name": "muon_block_bf16", "op": "muon", "shapes": "4x1536x1536,6144x1536,1536x6144", "dtype": "bf16"},
        # one step of answering: a row for each of a few sequences
        {"name": "embed_step_bf16", "op": "embed", "n": 24, "rows": 50257, "dim": 2048, "dtype": "bf16",
         "scale": 45.25, "ids": "zipf", "pad": False},
        # a batch of prompts
        {"name": "embed_prompts_bf16", "op": "embed", "n": 16384, "rows": 32000, "dim": 4096, "dtype": "bf16",
         "scale": 64.0, "ids": "zipf", "pad": False},
        # per-view codes of a grid_raw batch: 5 modalities x 2048 rays over the 45 training views
        {"name": "embed_grad_views_f32", "op": "embed_grad", "n": 10240, "rows": 45, "dim": 32, "dtype": "f32",
         "scale": 1.0, "ids": "uniform", "pad": False},
        # odd everything, with a padded part
        {"name": "embed_grad_odd_f32", "op": "embed_grad", "n": 9001, "rows": 50257, "dim": 771, "dtype": "f32",
         "scale": 1.0, "ids": "zipf", "pad": True},
        # a large training batch
        {"name": "embed_grad_large_bf16", "op": "embed_grad", "n": 65536, "rows": 131072, "dim": 2048,
         "dtype": "bf16", "scale": 45.25, "ids": "zipf", "pad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ns", "muon", "embed", "embed_grad"])
    if op in ("ns", "muon"):
        # one to six kinds of matrices, each up to 8 times, up to about the largest listed product
        kinds, cost = [], 0.0
        for _ in range(rng.randint(1, 6)):
            b, m, n = rng.choice([1, 1, 1, 2, 5, 8]), _log(rng, 1, 4096), _log(rng, 8, 4096)
            r, c = min(m, n), max(m, n)
            cost += b * (3.0 * r * r * c + float(r) ** 3)
            if kinds and cost > 2.0e11:
                break
            kinds.append("%dx%dx%d" % (b, m, n) if b > 1 else "%dx%d" % (m, n))
            if cost > 2.0e11:
                # a first kind that is too much alone: one of it
                kinds = ["%dx%d" % (m, n)]
                break
        return {"op": op, "shapes": ",".join(kinds), "dtype": rng.choice(["f32", "bf16"])}
    n, rows, dim = _log(rng, 1, 65536), _log(rng, 2, 131072), _log(rng, 4, 4096)
    while n * dim > 65536 * 2048 or rows * dim > 131072 * 2048:
        dim //= 2
    return {"op": op, "n": n, "rows": rows, "dim": dim, "dtype": rng.choice(["f32", "bf16", "f16"]),
            "scale": rng.choice([1.0, round(math.sqrt(dim), 2)]), "ids": rng.choice(["zipf", "uniform"]),
            "pad": op == "embed_grad" and rng.random() < 0.5}


def _shapes(text):
    """"256x71,8x1024x4096" -> [(256, 71), (8, 1024, 4096)]"""
    return [tuple(int(d) for d in s.split("x")) for s in text.split(",")]


def _gradient(shape, gen):
    """A gradient as backward passes give it: a few strong directions whose strength falls like 1 / i over noise."""
    *lead, m, n = shape
    k = min(32, m, n)
    strength = 1.0 / torch.arange(1, k + 1, device="cuda", dtype=torch.float32)
    u = torch.randn(*lead, m, k, device="cuda", generator=gen)
    v = torch.randn(*lead, k, n, device="cuda", generator=gen)
    return 1e-3 * (torch.matmul(u * strength, v) + 0.3 * torch.randn(*lead, m, n, device="cuda", generator=gen))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] in ("ns", "muon"):
        shapes = _shapes(case["shapes"])
        s["grads"] = [_gradient(x, gen).to(dt) for x in shapes]
        if case["op"] == "muon":
            s["params"] = [(torch.randn(*x, device="cuda", generator=gen) / math.sqrt(x[-1])).to(dt) for x in shapes]
            s["momenta"] = [0.7 * _gradient(x, gen) for x in shapes]
        return s
    n, rows, dim = case["n"], case["rows"], case["dim"]
    if case["ids"] == "zipf":
        # how often words occur: the rank r with probability about 1 / r, the ranks scattered over the table
        rank = torch.exp(torch.rand(n, device="cuda", generator=gen, dtype=torch.float64) * math.log(rows)).long()
        ids = (rank.clamp(1, rows) * 40503 + 17) % rows
    else:
        ids = torch.randint(0, rows, (n,), device="cuda", generator=gen)
    s["padding_idx"] = None
    if case["pad"]:
        # the tail of each run of 64 positions is padding
        s["padding_idx"] = rows // 2
        ids = torch.where(torch.arange(n, device="cuda") % 64 >= 56, torch.full_like(ids, rows // 2), ids)
    s["index"] = ids
    if case["op"] == "embed":
        s["table"] = (0.02 * torch.randn(rows, dim, device="cuda", generator=gen)).to(dt)
    else:
        s["dout"] = torch.randn(n, dim, device="cuda", generator=gen).to(dt)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------
def _orthogonal(g):
    """Newton-Schulz in 32 bits: X = G / max(|G|, eps), then X <- a X + (b A + c A A) X with A = X X^T, on the side
    with fewer rows."""
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x * x).sum((-2, -1), keepdim=True).sqrt().clamp(min=EPS)
    a, b, c = COEFF
    for _ in range(STEPS):
        gram = torch.matmul(x, x.mT)
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.mT if tall else x


def _plain(s):
    op = s["op"]
    if op == "ns":
        return [_orthogonal(g).to(g.dtype) for g in s["grads"]]
    if op == "muon":
        for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
            m.copy_(MOMENTUM * m + (1.0 - MOMENTUM) * g.float())
            u = (1.0 - MOMENTUM) * g.float() + MOMENTUM * m
            lr = LR * math.sqrt(max(1.0, p.shape[-2] / p.shape[-1]))
            p.copy_((p.float() * (1.0 - LR * DECAY) - lr * _orthogonal(u)).to(p.dtype))
        return {"params": s["params"], "momenta": s["momenta"]}
    if op == "embed":
        return (s["table"][s["index"]].float() * s["scale"]).to(s["table"].dtype)
    d = s["dout"].float() * s["scale"]
    if s["padding_idx"] is not None:
        d = torch.where((s["index"] == s["padding_idx"])[:, None], torch.zeros_like(d), d)
    return torch.zeros(s["rows"], s["dim"], device=d.device).index_add_(0, s["index"], d).to(s["dout"].dtype)


def run(state):
    if not own:
        return _plain(state)
    from multimodalstudio_amd import hip_ops
    op = state["op"]
    if op == "ns":
        return hip_ops.newton_schulz(state["grads"], steps=STEPS, coefficients=COEFF, eps=EPS)
    if op == "muon":
        hip_ops.muon_step(state["params"], state["grads"], state["momenta"], lr=LR, momentum=MOMENTUM, nesterov=True,
                          weight_decay=DECAY, steps=STEPS, coefficients=COEFF, eps=EPS)
        return {"params": state["params"], "momenta": state["momenta"]}
    if op == "embed":
        return hip_ops.embedding(state["index"], state["table"], scale=state["scale"])
    return hip_ops.embedding_backward(state["index"], state["dout"], state["rows"], scale=state["scale"],
                                      padding_idx=state["padding_idx"])


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] in ("ns", "muon"):
        values = flops = 0
        for x in _shapes(case["shapes"]):
            count, r, c = math.prod(x[:-2]), min(x[-2:]), max(x[-2:])
            values += count * r * c
            # X X^T and A A are symmetric (half of a full product each), the product with X is full
            flops += count * STEPS * (r * r * c + r * r * r + 2 * r * r * c)
        # the gradient in, the result out; the step also reads its weights and reads and writes a 32-bit momentum
        return {"bytes": values * (2 * e if case["op"] == "ns" else 3 * e + 8), "flops": flops}
    n, rows, dim = case["n"], case["rows"], case["dim"]
    if case["op"] == "embed":
        # a row that occurs is read once: sum over the rows of 1 - (1 - p)^n of them are expected to
        r = torch.arange(1, rows + 1, dtype=torch.float64)
        p = torch.log1p(1.0 / r) / math.log(rows) if case["ids"] == "zipf" else torch.full_like(r, 1.0 / rows)
        seen = float(-torch.expm1(n * torch.log1p(-p.clamp(max=1.0 - 1e-12))).sum())
        return {"bytes": n * 8 + (min(seen, n, rows) + n) * dim * e, "flops": n * dim}
    return {"bytes": n * 8 + (n + rows) * dim * e, "flops": 2 * n * dim}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _polar64(g):
    """The iterated odd polynomial of G / |G|, from the right: Y <- Y (a I + M (b I + c M)), M = Y^T Y, tall Y."""
    wide = g.shape[-1] > g.shape[-2]
    y = (g.mT if wide else g).double().contiguous()
    y = y / torch.linalg.matrix_norm(y, keepdim=True).clamp_min(EPS)
    eye = torch.eye(y.shape[-1], dtype=torch.float64, device=y.device)
    a, b, c = COEFF
    for _ in range(STEPS):
        m = torch.matmul(y.mT.contiguous(), y)
        y = torch.matmul(y, a * eye + torch.matmul(m, b * eye + c * m))
    return y.mT.contiguous() if wide else y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ns":
        return [_polar64(g) for g in s["grads"]]
    if case["op"] == "muon":
        params, momenta = [], []
        for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
            m2 = m.double() + (1.0 - MOMENTUM) * (g.double() - m.double())
            u = g.double() + MOMENTUM * (m2 - g.double())
            rate = LR * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5
            params.append(p.double() - LR * DECAY * p.double() - rate * _polar64(u))
            momenta.append(m2)
        return {"params": params, "momenta": momenta}
    ids = s["index"]
    if case["op"] == "embed":
        return torch.index_select(s["table"], 0, ids).double() * s["scale"]
    # the rows of one index lie together once sorted: their sum is a difference of two running sums
    order = torch.argsort(ids, stable=True)
    run_sum = torch.zeros(ids.numel() + 1, case["dim"], dtype=torch.float64, device=ids.device)
    torch.cumsum(s["dout"].double()[order], 0, out=run_sum[1:])
    rows = torch.arange(case["rows"], device=ids.device)
    key = ids[order].contiguous()
    grad = run_sum[torch.searchsorted(key, rows, right=True)] - run_sum[torch.searchsorted(key, rows)]
    if s["padding_idx"] is not None:
        grad[s["padding_idx"]] = 0.0
    return grad * s["scale"]
