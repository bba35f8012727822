"""Operators around the experts of a mixture-of-experts layer, as they are timed and checked.

  permute    token rows into expert order (every token to its top-k experts), and the gradient
  unpermute  expert rows back to their tokens, weighted and summed, and the gradients
  rows8      activations to 8-bit floats (e4m3) with a scale for each 128 columns of a row,
             brought into expert order by the same call
  weight8    expert weights to e4m3 with a scale for each block of 128 x 128
  product    every expert's rows times its weights, both in e4m3 with those scales; plain, with
             the router weight of each row, or with SwiGLU between the halves of the weights

`own` chooses between this package's calls and the same mathematics in elementary torch
operations. Sizes are those of this package's decode sweep and prefill configurations (hidden 2048,
64 experts of width 1024, top-8, batches from 1 to 8192 tokens), of its tests (60 experts, top-4,
small odd widths) and odd ones between them."""

import math

import torch

own = False

BLOCK = 128          # columns (and weight rows) that share a scale
TOP = 448.0          # largest e4m3 value
TINY = 2.0 ** -96    # a block's largest magnitude counts as at least this
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------ the cases
def listed():
    layer = dict(H=2048, E=64, k=8)
    return [
        # a decode step of 64 requests: where launch latency is what a user waits for
        dict(name="permute decode", op="permute", T=64, dtype="bf16", grad=False, skew=False, **layer),
        # a training batch, forward and backward
        dict(name="permute train", op="permute", T=8192, dtype="bf16", grad=True, skew=True, **layer),
        # a decode step of 8 requests, the router weights in the rows' type
        dict(name="unpermute decode", op="unpermute", T=8, dtype="fp16", wdtype="fp16", grad=False, skew=False, **layer),
        # a training batch with an odd count of tokens, the router weights kept in 32 bits
        dict(name="unpermute train", op="unpermute", T=8191, dtype="bf16", wdtype="fp32", grad=True, skew=True, **layer),
        # one request being decoded: one token to its eight experts
        dict(name="rows8 one token", op="rows8", T=1, dtype="bf16", skew=False, **layer),
        # the prompts of a prefill batch
        dict(name="rows8 prefill", op="rows8", T=8192, dtype="bf16", skew=True, **layer),
        # a layer's gate and up projections when a checkpoint is loaded
        dict(name="weight8 load", op="weight8", E=64, N=2048, K=2048, halves=2, dtype="bf16"),
        # a small model whose widths are no multiple of a block
        dict(name="weight8 ragged", op="weight8", E=60, N=1000, K=1040, halves=1, dtype="fp16"),
        # decoding 8 requests: the weights of the experts that are hit, past a row or two each
        dict(name="product decode gate-up", op="product", T=8, K=2048, N=1024, E=64, k=8, swiglu=True, scaled=False,
             dtype="bf16", skew=False),
        # decoding 64 requests, down projection with the router weights: all experts are read
        dict(name="product decode down", op="product", T=64, K=1024, N=2048, E=64, k=8, swiglu=False, scaled=True,
             dtype="fp16", skew=False),
        # prefill of 8192 tokens with skewed routing: bound by arithmetic
        dict(name="product prefill gate-up", op="product", T=8192, K=2048, N=1024, E=64, k=8, swiglu=True, scaled=False,
             dtype="bf16", skew=True),
        # a middling batch on the small model: rows, columns and k that fill no tile
        dict(name="product ragged down", op="product", T=1237, K=1040, N=1000, E=60, k=4, swiglu=False, scaled=True,
             dtype="bf16", skew=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["permute", "unpermute", "rows8", "weight8", "product", "product"])
    E, k = rng.choice([(64, 8), (60, 4), (16, 4), (8, 2), (128, 8)])
    if op == "weight8":
        halves = rng.choice([1, 2])
        count = rng.choice([1, 5, min(E, 64)])
        return dict(op=op, E=count, N=8 * halves * _log(rng, 4, 1024 // 8), K=16 * _log(rng, 4, 2048 // 16), halves=halves,
                    dtype=rng.choice(["bf16", "fp16", "fp32"] if count < 16 else ["bf16", "fp16"]))
    T = _log(rng, 1, 8000)
    skew = T > 64
    if op == "product":
        swiglu = rng.random() < 0.5
        return dict(op=op, T=T, K=16 * _log(rng, 8, 2048 // 16), N=8 * _log(rng, 16, 1024 // 8), E=E, k=k, swiglu=swiglu,
                    scaled=not swiglu and rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]), skew=skew)
    dtype = rng.choice(["bf16", "fp16"] if op == "rows8" else ["bf16", "fp16", "fp32"])
    if dtype == "fp32":
        T = min(T, 4000)
    step = 16 if op == "rows8" else 8
    case = dict(op=op, T=T, H=step * _log(rng, 64 // step, 2048 // step), E=E, k=k, dtype=dtype, skew=skew)
    if op != "rows8":
        case["grad"] = rng.random() < 0.5
    if op == "unpermute":
        case["wdtype"] = rng.choice([dtype, "fp32"])
    return case


# ------------------------------------------------------------------------------ inputs
def _routing(case, g):
    """Distinct experts of every token, popular experts more often where `skew` is set, and the
    sorted order of the choices as this package's sort gives it."""
    T, E, k = case["T"], case["E"], case["k"]
    u = torch.rand(T, E, device="cuda", generator=g).clamp_(1e-9, 1 - 1e-7)
    score = -torch.log(-torch.log(u))
    if case["skew"]:
        rank = torch.randperm(E, device="cuda", generator=g).float() + 1
        score += -1.1 * 0.6 * torch.log(rank)
    idx = score.topk(k, dim=1).indices.int()
    flat = idx.flatten().long()
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=E)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    pos_of = torch.empty(T * k, dtype=torch.int32, device="cuda")
    pos_of[order] = torch.arange(T * k, dtype=torch.int32, device="cuda")
    return dict(counts=counts.int(), offsets=offsets, token=(order // k).int(), pos_of=pos_of.view(T, k))


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "weight8":
        s["w"] = (_randn(g, case["E"], case["N"], case["K"]) * 0.02).to(DTYPES[case["dtype"]])
        return s
    s.update(_routing(case, g))
    dtype, T, E, M = DTYPES[case["dtype"]], case["T"], case["E"], case["T"] * case["k"]
    if case["op"] == "product":
        K, N = case["K"], case["N"]
        rows = _randn(g, M, K) * torch.exp(0.5 * _randn(g, M, 1))
        s["q"], scale = _plain_blocks(rows, 1)
        s["s"] = scale.t().contiguous()
        halves = 2 if case["swiglu"] else 1
        s["wq"], s["ws"] = _plain_weight(_randn(g, E, halves * N, K) * K ** -0.5, halves)
        s["scale"] = torch.rand(M, device="cuda", generator=g).to(dtype) if case["scaled"] else None
        # the plain form's plan: every expert's rows padded to the longest
        s["longest"] = int(s["counts"].max())
        return s
    H = case["H"]
    s["h"] = _randn(g, T, H).to(dtype)
    if case["op"] == "permute":
        s["dx"] = _randn(g, M, H).to(dtype) if case["grad"] else None
    if case["op"] == "unpermute":
        s["y"] = _randn(g, M, H).to(dtype)
        s["w"] = torch.rand(T, case["k"], device="cuda", generator=g).to(DTYPES[case["wdtype"]])
        s["dout"] = s.pop("h") if case["grad"] else None
    return s


# ------------------------------------------------------------------------------ plain forms
def _plain_blocks(x, rows_per_block):
    """e4m3 values and scales of [..., R, K] in blocks of rows_per_block x 128: with m the block's
    largest magnitude, scale = m / 448 and value = round(448 x / m)."""
    lead, R, K = x.shape[:-2], x.shape[-2], x.shape[-1]
    nr, nk = -(-R // rows_per_block), -(-K // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, nk * BLOCK - K, 0, nr * rows_per_block - R))
    b = x.reshape(*lead, nr, rows_per_block, nk, BLOCK)
    top = b.abs().amax(dim=(-3, -1)).clamp(min=TINY)
    most = torch.full_like(top, TOP)
    q = (b * TOP / top[..., :, None, :, None]).reshape(*lead, nr * rows_per_block, nk * BLOCK)[..., :R, :K]
    return q.to(torch.float8_e4m3fn).contiguous(), top / most


def _plain_weight(w, halves):
    E, N, K = w.shape
    q, scale = _plain_blocks(w.reshape(E * halves, N // halves, K), BLOCK)
    return q.reshape(E, N, K), scale.reshape(E, -1, scale.shape[-1])


def _plain_product(s):
    c = s["case"]
    K, N, E = c["K"], c["N"], c["E"]
    x = s["q"].float() * s["s"].t().repeat_interleave(BLOCK, 1)[:, :K]
    halves = 2 if c["swiglu"] else 1
    ws = s["ws"].view(E * halves, -1, s["ws"].shape[-1]).repeat_interleave(BLOCK, 1)[:, :N].repeat_interleave(BLOCK, 2)
    w = s["wq"].float() * ws[:, :, :K].reshape(E, halves * N, K)
    at = s["offsets"][:-1, None].long() + torch.arange(s["longest"], device="cuda")
    padded = torch.bmm(x[at.clamp(max=x.shape[0] - 1)], w.transpose(1, 2))
    row = torch.arange(x.shape[0], device="cuda")
    e = torch.searchsorted(s["offsets"][1:].contiguous(), row.int(), right=True)
    acc = padded[e, row - s["offsets"][e]]
    if c["swiglu"]:
        gate, up = acc[:, :N], acc[:, N:]
        acc = gate / (1 + torch.exp(-gate)) * up
    if c["scaled"]:
        acc = acc * s["scale"].float()[:, None]
    return acc.to(DTYPES[c["dtype"]])


def run(s):
    c, op = s["case"], s["case"]["op"]
    if own:
        from switchyard_b200 import fp8, rows
        if op == "weight8":
            return fp8.quantize_weight(s["w"], halves=c["halves"])
        if op == "product":
            return fp8.grouped_gemm(fp8.Rows8(s["q"], s["s"]), fp8.Weight8(s["wq"], s["ws"]), s["offsets"],
                                    swiglu=c["swiglu"], scale=s["scale"], dtype=DTYPES[c["dtype"]])
        plan = rows.SortPlan(s["counts"], s["offsets"], s["token"], s["pos_of"])
        if op == "rows8":
            return fp8.quantize_rows(s["h"], plan)
        if op == "permute":
            if not c["grad"]:
                return rows.permute_rows(s["h"], plan)
            h = s["h"].detach().requires_grad_()
            x = rows.permute_rows(h, plan)
            return (x.detach(),) + torch.autograd.grad(x, h, s["dx"])
        if not c["grad"]:
            return rows.unpermute_rows(s["y"], s["w"], plan)
        y, w = s["y"].detach().requires_grad_(), s["w"].detach().requires_grad_()
        out = rows.unpermute_rows(y, w, plan)
        return (out.detach(),) + torch.autograd.grad(out, (y, w), s["dout"])
    if op == "weight8":
        return _plain_weight(s["w"], c["halves"])
    if op == "product":
        return _plain_product(s)
    token, pos_of = s["token"].long(), s["pos_of"].long()
    dtype = DTYPES[c["dtype"]]
    if op == "rows8":
        q, scale = _plain_blocks(s["h"], 1)
        return q.view(torch.uint8)[token].view(torch.float8_e4m3fn), scale[token].t().contiguous()
    if op == "permute":
        x = s["h"][token]
        return (x, s["dx"].float()[pos_of].sum(1).to(dtype)) if c["grad"] else x
    picked, w = s["y"].float()[pos_of], s["w"].float()[..., None]
    out = (picked * w).sum(1).to(dtype)
    if not c["grad"]:
        return out
    dout = s["dout"].float()[:, None]
    dy = torch.empty_like(s["y"])
    dy[pos_of.flatten()] = (dout * w).to(dtype).flatten(0, 1)
    return out, dy, (dout * picked).sum(-1).to(s["w"].dtype)


# ------------------------------------------------------------------------------ what a pass needs
def work(case):
    op = case["op"]
    if op == "weight8":
        n = case["E"] * case["N"] * case["K"]
        blocks = case["E"] * case["halves"] * -(-case["N"] // case["halves"] // BLOCK) * -(-case["K"] // BLOCK)
        return {"bytes": n * (BYTES[case["dtype"]] + 1) + 4 * blocks, "flops": 2 * n}
    T, k, E, M = case["T"], case["k"], case["E"], case["T"] * case["k"]
    if op == "product":
        K, N = case["K"], case["N"]
        wide = (2 if case["swiglu"] else 1) * N
        used = E * (1 - (1 - k / E) ** T)  # experts that a token goes to, as expected of even routing
        kb, nb = -(-K // BLOCK), -(-wide // BLOCK)
        n = used * (wide * K + 4 * nb * kb) + M * (K + 4 * kb) + M * N * 2 + (2 * M if case["scaled"] else 0)
        return {"bytes": int(n) + 4 * (E + 1), "flops": 2 * M * K * wide}
    H, b = case["H"], BYTES[case["dtype"]]
    if op == "rows8":
        return {"bytes": T * H * b + M * (H + 4 * -(-H // BLOCK)) + 4 * M, "flops": 2 * T * H}
    n = (T + M) * H * b + 4 * M
    if op == "permute":
        return {"bytes": 2 * n if case["grad"] else n, "flops": M * H if case["grad"] else 0}
    wb = BYTES[case["wdtype"]]
    n += M * wb
    if case["grad"]:
        n += (T + 2 * M) * H * b + 4 * M + 2 * M * wb
    return {"bytes": n, "flops": (5 if case["grad"] else 2) * M * H}


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "weight8":
        w, parts = s["w"].double(), case["halves"]
        each = case["N"] // parts
        q, scales = torch.empty_like(w), []
        for p in range(parts):
            for r in range(0, each, BLOCK):
                lo, hi = p * each + r, p * each + min(each, r + BLOCK)
                for c in range(0, case["K"], BLOCK):
                    b = w[:, lo:hi, c:c + BLOCK]
                    top = b.abs().amax((1, 2)).clamp(min=TINY)
                    scales.append(top / TOP)
                    q[:, lo:hi, c:c + BLOCK] = _nearest8(b * TOP / top[:, None, None])
        return q, torch.stack(scales, 1).view(case["E"], -1, -(-case["K"] // BLOCK))
    offsets, token, pos_of = s["offsets"].tolist(), s["token"].long(), s["pos_of"].long()
    if op == "product":
        K, N, out = case["K"], case["N"], []
        parts = 2 if case["swiglu"] else 1
        x = s["q"].double()
        for c in range(0, K, BLOCK):
            x[:, c:c + BLOCK] *= s["s"][c // BLOCK].double()[:, None]
        nb = -(-N // BLOCK)
        for e in range(case["E"]):
            w = s["wq"][e].double()
            for p in range(parts):
                for n in range(0, N, BLOCK):
                    for c in range(0, K, BLOCK):
                        w[p * N + n:p * N + min(N, n + BLOCK), c:c + BLOCK] *= s["ws"][e, p * nb + n // BLOCK, c // BLOCK].double()
            a = x[offsets[e]:offsets[e + 1]] @ w.t()
            if case["swiglu"]:
                a = a[:, :N] * torch.sigmoid(a[:, :N]) * a[:, N:]
            out.append(a)
        out = torch.cat(out)
        return out * s["scale"].double()[:, None] if case["scaled"] else out
    if op == "rows8":
        h, q, scales = s["h"].double(), [], []
        for c in range(0, case["H"], BLOCK):
            b = h[:, c:c + BLOCK]
            top = b.abs().amax(1).clamp(min=TINY)
            scales.append((top / TOP)[token])
            q.append(_nearest8(b * TOP / top[:, None]))
        return torch.cat(q, 1)[token], torch.stack(scales)
    T, k, H = case["T"], case["k"], case["H"]
    if op == "permute":
        x = s["h"].double()[token]
        if not case["grad"]:
            return x
        return x, torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, token, s["dx"].double())
    y, w = s["y"].double(), s["w"].double()
    out = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for j in range(k):
        out += y[pos_of[:, j]] * w[:, j:j + 1]
    if not case["grad"]:
        return out
    dout, dy, dw = s["dout"].double(), torch.empty_like(y), torch.empty_like(w)
    for j in range(k):
        dy[pos_of[:, j]] = dout * w[:, j:j + 1]
        dw[:, j] = (dout * y[pos_of[:, j]]).sum(1)
    return out, dy, dw


def _nearest8(v):
    """The nearest e4m3 value in 64 bits: steps of 2^(exponent - 3), 2^-9 below 2^-6; ties to even."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return torch.round(v / step) * step
