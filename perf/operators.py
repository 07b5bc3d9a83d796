"""Cases of the first-order operators of the adapter set: products grouped by adapter copy (forward, input gradient and
weight gradient), the scoring loss with its gradient, and the AdamW step over many tensors with 32-bit or 8-bit states.

``own`` false computes the plain forms with elementary torch operations, true calls the framework."""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
BLOCK = 256                      # elements of one scale of the 8-bit states
BETA1, BETA2, EPS, DECAY, LR = 0.9, 0.999, 1e-8, 0.01, 2e-4
FT = {"f32": torch.float32, "bf16": torch.bfloat16}


_package = None


def _framework():
    global _package
    if _package is None:
        root = os.path.join(os.getcwd(), "ds-mezo_b200")     # the package's folder under the working folder
        if root not in sys.path:
            sys.path.insert(0, root)
        import dsmezo_b200
        _package = dsmezo_b200
    return _package


# ----------------------------------------------------------------------------------------------------------- cases

def listed():
    """The cases; sizes are those of the 1.5B-, 7B- and 70B-shaped adapter sets of the benchmark."""
    return [
        # one rollout token for each of the 32 +/- copies of a 16-direction step through B of a 7B q/k/v input: latency
        dict(name="product_tokens_7b", op="product", rows=32, behind=0, groups=32, k=3584, n=64, major="k", out="bf16",
             split="even", mix=1),
        # the scored tokens of a 7B step through B of the + and - copies
        dict(name="product_down_7b", op="product", rows=4096, behind=0, groups=2, k=3584, n=64, major="k", out="bf16",
             split="even", mix=2),
        # the second product of the 7B MLP adapter (through A), 32 copies, ragged rollouts in a padded batch
        dict(name="product_up_7b_32", op="product", rows=4001, behind=95, groups=32, k=64, n=18944, major="k",
             out="bf16", split="ragged", mix=3),
        # gradient with respect to the rank rows of the 70B MLP adapter: A is read along its other dimension
        dict(name="product_grad_70b", op="product", rows=4133, behind=0, groups=4, k=28672, n=128, major="n",
             out="bf16", split="empty", mix=4),
        # full-width matrices, one for each group: the largest products
        dict(name="product_full_7b", op="product", rows=8192, behind=0, groups=8, k=3584, n=18944, major="k",
             out="bf16", split="ragged", mix=5),
        # gradient of A of the 7B MLP adapter, two micro-batches of copies
        dict(name="weight_grad_7b", op="weight_grad", rows=4096, behind=0, groups=2, k=64, n=18944, split="even", mix=6),
        # gradients of B of a 1.5B adapter for eight copies, few and odd numbers of rows, one copy without any
        dict(name="weight_grad_1p5b_ragged", op="weight_grad", rows=997, behind=27, groups=8, k=1536, n=16,
             split="empty", mix=7),
        # a 7B set's AdamW step, 392 factors: fp32 states, fp32 gradients, bf16 shadow for the rollout
        dict(name="adamw32_7b", op="adamw", tensors=392, total=161480704, bits=32, grad="f32", shadow=True, mix=8),
        # the same set with 8-bit states and bf16 gradients
        dict(name="adamw8_7b", op="adamw", tensors=392, total=161480704, bits=8, grad="bf16", shadow=True, mix=9),
        # a handful of small factors of odd sizes with 8-bit states: latency
        dict(name="adamw8_small", op="adamw", tensors=14, total=90001, bits=8, grad="f32", shadow=False, mix=10),
        # four completions of 512 scored tokens over the Qwen2.5 vocabulary
        dict(name="loss_grad_qwen_bf16", op="loss_grad", tokens=2048, sequences=4, vocab=152064, dtype="bf16", mix=11),
        # a few short completions over an odd vocabulary in fp32
        dict(name="loss_grad_small_f32", op="loss_grad", tokens=61, sequences=5, vocab=32003, dtype="f32", mix=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: ranks 8 to 128 against widths up to the 70B set's, 1 to 8192 rows in 1 to 64 groups; 1 to 400
    tensors; 1 to 2048 tokens over vocabularies up to Qwen2.5's."""
    op = rng.choice(["product", "product", "weight_grad", "adamw", "loss_grad"])
    mix = rng.randrange(1 << 30)
    if op in ("product", "weight_grad"):
        rank, wide = 8 * _log_int(rng, 1, 16), 8 * _log_int(rng, 32, 3584)
        rows, groups = _log_int(rng, 1, 8192), _log_int(rng, 1, 64)
        k, n = (rank, wide) if rng.random() < 0.5 else (wide, rank)
        case = dict(op=op, rows=rows, behind=rng.choice([0, 0, rng.randrange(1, 130)]), groups=groups, k=k, n=n,
                    split=rng.choice(["even", "ragged", "empty"]), mix=mix)
        if op == "product":
            case.update(major=rng.choice(["k", "n"]), out=rng.choice(["bf16", "bf16", "f32"]))
        return case
    if op == "adamw":
        tensors = _log_int(rng, 1, 400)
        return dict(op=op, tensors=tensors, total=_log_int(rng, 512 * tensors, 100000000), bits=rng.choice([32, 8]),
                    grad=rng.choice(["f32", "bf16"]), shadow=rng.choice([True, False]), mix=mix)
    tokens = _log_int(rng, 1, 2048)
    return dict(op=op, tokens=tokens, sequences=min(tokens, rng.randrange(1, 17)), vocab=_log_int(rng, 1000, 152064),
                dtype=rng.choice(["f32", "bf16"]), mix=mix)


def _parts(total, n, split, mix):
    """`total` things over `n` owners: evenly, unevenly, or unevenly with owners that have none."""
    rng = random.Random(mix)
    if split == "even":
        return [total * (i + 1) // n - total * i // n for i in range(n)]
    weight = [rng.expovariate(1.0) + 0.05 for _ in range(n)]
    if split == "empty" and n > 1:
        for i in rng.sample(range(n), max(1, n // 4)):
            weight[i] = 0.0
    edge, acc = [0], 0.0
    for w in weight:
        acc += w
        edge.append(int(round(total * acc / sum(weight))))
    return [b - a for a, b in zip(edge, edge[1:])]


def _tensor_sizes(case):
    """Sizes of the tensors of an AdamW case (each at least one element), summing to case["total"]."""
    n = case["tensors"]
    return [1 + p for p in _parts(case["total"] - n, n, "ragged", case["mix"])]


# --------------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + case["mix"])
    return {"product": _prepare_product, "weight_grad": _prepare_weight_grad, "adamw": _prepare_adamw,
            "loss_grad": _prepare_loss}[case["op"]](case, g)


def _rows_of(case):
    sizes = _parts(case["rows"], case["groups"], case["split"], case["mix"])
    edges = [0]
    for s in sizes:
        edges.append(edges[-1] + s)
    return sizes, edges


def _index(sizes, edges):
    """(group, position) of every row, and the longest group: what the plain form pads the groups with."""
    group = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.tensor(sizes, device=DEV))
    place = torch.arange(edges[-1], device=DEV) - torch.tensor(edges[:-1], device=DEV)[group]
    return group, place, max(1, max(sizes))


def _activations(rows, width, g):
    """Module inputs: normal, with the channel scales of a decoder (log-normal)."""
    scale = torch.exp(torch.randn(width, generator=g, device=DEV))
    return (torch.randn(rows, width, generator=g, device=DEV) * scale).to(torch.bfloat16)


def _prepare_product(case, g):
    sizes, edges = _rows_of(case)
    G, k, n = case["groups"], case["k"], case["n"]
    x = _activations(case["rows"] + case["behind"], k, g)
    w = torch.empty((G, n, k) if case["major"] == "k" else (G, k, n), dtype=torch.bfloat16, device=DEV)
    w.normal_(0.0, 1.0 / math.sqrt(k), generator=g)
    group, place, longest = _index(sizes, edges)
    return dict(op="product", x=x, w=w.transpose(1, 2) if case["major"] == "k" else w, out=FT[case["out"]],
                offsets=torch.tensor(edges, dtype=torch.int32, device=DEV), group=group, place=place, longest=longest)


def _prepare_weight_grad(case, g):
    sizes, edges = _rows_of(case)
    rows = case["rows"] + case["behind"]
    group, place, longest = _index(sizes, edges)
    # the wide side is an activation (or its gradient), the narrow one the rank rows
    x = _activations(rows, case["k"], g)
    dy = (torch.randn(rows, case["n"], generator=g, device=DEV) * 0.01).to(torch.bfloat16)
    return dict(op="weight_grad", x=x, dy=dy, groups=case["groups"],
                offsets=torch.tensor(edges, dtype=torch.int32, device=DEV), group=group, place=place, longest=longest)


def _pack8(m, root):
    """8-bit codes and scales of the mean m and of the root of the second moment (both in 64 bits: which of two codes a
    value next to a border takes is part of the result; a value on it takes the lower), blocks of 256 along the arena:
    m = sign q^2 s with |q| <= 127, root = q^2 s with q <= 255 (at least 1 where the root is positive)."""
    mb, rb = m.view(-1, BLOCK), root.view(-1, BLOCK)
    mt, rt = mb.abs().amax(1, keepdim=True), rb.amax(1, keepdim=True)
    mq = torch.ceil(127.0 * torch.sqrt(mb.abs() / mt) - 0.5).nan_to_num(0.0)
    rq = torch.ceil(255.0 * torch.sqrt(rb / rt) - 0.5).nan_to_num(0.0)
    rq = torch.where(rb > 0, rq.clamp(min=1.0), rq)
    return (torch.copysign(mq, mb).to(torch.int8).view(-1), (mt / 16129.0).float().view(-1),
            rq.to(torch.uint8).view(-1), (rt / 65025.0).float().view(-1))


def _unpack8(mq, ms, rq, rs):
    a, b = mq.view(-1, BLOCK).double(), rq.view(-1, BLOCK).double()
    root = b * b * rs.double()[:, None]
    return (a * a.abs() * ms.double()[:, None]).view(-1), (root * root).view(-1)


def _prepare_adamw(case, g):
    # tensors lie in arenas, each from a multiple of 256 elements on; the gaps between them stay zero
    sizes = _tensor_sizes(case)
    at, total = [], 0
    for s in sizes:
        at.append(total)
        total += (s + BLOCK - 1) // BLOCK * BLOCK
    live = torch.zeros(total, dtype=torch.bool, device=DEV)
    for a, s in zip(at, sizes):
        live[a:a + s] = True

    def normal(scale, dtype=torch.float32):
        t = torch.empty(total, device=DEV).normal_(0.0, scale, generator=g).mul_(live)
        return t.to(dtype)

    p, grad = normal(0.02), normal(1e-3, FT[case["grad"]])
    m, root = normal(3e-4), normal(1e-3).abs_()
    st = dict(op="adamw", bits=case["bits"], p=p, grad=grad, t=100,
              shadow=p.to(torch.bfloat16) if case["shadow"] else None)
    if case["bits"] == 32:
        st.update(m=m, v=root * root)
    else:
        st.update(zip(("mq", "ms", "rq", "rs"), _pack8(m.double(), root.double())))
    if own:
        optim = _framework().optim

        def views(t, step=1):
            return [t[a // step:a // step + -(-s // step)] for a, s in zip(at, sizes)]
        if case["bits"] == 32:
            states = [optim.AdamWState(*z) for z in zip(views(st["m"]), views(st["v"]))]
        else:
            states = [optim.AdamWState(*z) for z in zip(views(st["mq"]), views(st["rq"]), views(st["ms"], BLOCK),
                                                        views(st["rs"], BLOCK))]
            st["values"] = torch.zeros(total, device=DEV), torch.zeros(total, device=DEV)
            st["value_views"] = [views(t) for t in st["values"]]
        st["optimizer"] = optim.AdamW(views(p), lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                      grads=views(grad), states=states, step=st["t"],
                                      shadows=views(st["shadow"]) if case["shadow"] else None)
    return st


def _prepare_loss(case, g):
    lens = [1 + s for s in _parts(case["tokens"] - case["sequences"], case["sequences"], "ragged", case["mix"])]
    logits = torch.empty(case["tokens"], case["vocab"], dtype=FT[case["dtype"]], device=DEV).normal_(0.0, 4.0, generator=g)
    targets = torch.randint(0, case["vocab"], (case["tokens"],), generator=g, device=DEV, dtype=torch.int32)
    # scored completions are likely ones: their tokens stand out of the row
    rows = torch.arange(case["tokens"], device=DEV)
    logits[rows, targets.long()] += 12.0
    rng = random.Random(case["mix"])
    adv = [rng.uniform(0.1, 1.0) * (1 if i % 2 == 0 else -0.5) for i in range(case["sequences"])]
    weight = torch.tensor([a / s for a, s in zip(adv, lens) for _ in range(s)], dtype=torch.float64, device=DEV)
    return dict(op="loss_grad", logits=logits, targets=targets, lens=lens, adv=adv, weight=weight)


# -------------------------------------------------------------------------------------------------------- one pass

def run(state):
    if state["op"] == "product":
        if own:
            return _framework().grouped.grouped_matmul(state["x"], state["w"], state["offsets"], out_dtype=state["out"])
        return _plain_product(state)
    if state["op"] == "weight_grad":
        if own:
            return _framework().grouped.grouped_weight_grad(state["x"], state["dy"], state["offsets"])
        return _plain_weight_grad(state)
    if state["op"] == "adamw":
        if own:
            state["optimizer"].step()
            if state["bits"] == 32:
                return [state["p"], state["m"], state["v"], state["shadow"]]
            state["optimizer"].state_values(*state["value_views"])
            return [state["p"], *state["values"], state["shadow"]]
        return _plain_adamw(state)
    if own:
        return _framework().scoring.contrastive_loss_grad(state["logits"], state["lens"], state["adv"], state["targets"])
    return _plain_loss(state)


def _padded(state, t):
    """The rows of t by group, the short groups filled with zeros."""
    p = torch.zeros(state["offsets"].numel() - 1, state["longest"], t.shape[1], dtype=torch.float32, device=DEV)
    p[state["group"], state["place"]] = t[:state["group"].numel()].float()
    return p


def _plain_product(state):
    y = torch.bmm(_padded(state, state["x"]), state["w"].float())
    out = torch.zeros(state["x"].shape[0], y.shape[2], dtype=state["out"], device=DEV)
    out[:state["group"].numel()] = y[state["group"], state["place"]].to(state["out"])
    return out


def _plain_weight_grad(state):
    return torch.bmm(_padded(state, state["x"]).transpose(1, 2), _padded(state, state["dy"]))


def _plain_adamw(state):
    state["t"] += 1
    t, p = state["t"], state["p"]
    if state["bits"] == 32:
        g, m, v = state["grad"].float(), state["m"], state["v"]
    else:
        g = state["grad"].double()
        m, v = _unpack8(state["mq"], state["ms"], state["rq"], state["rs"])
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * (1.0 - BETA2)) * g
    root = torch.sqrt(v)
    step = (m / (root * (1.0 / math.sqrt(1.0 - BETA2 ** t)) + EPS)) * (LR / (1.0 - BETA1 ** t))
    p.copy_(p * (1.0 - LR * DECAY) - step)
    if state["shadow"] is not None:
        state["shadow"].copy_(p)
    if state["bits"] == 32:
        state["m"].copy_(m)
        state["v"].copy_(v)
        return [p, state["m"], state["v"], state["shadow"]]
    state.update(zip(("mq", "ms", "rq", "rs"), _pack8(m, root)))
    m, v = _unpack8(state["mq"], state["ms"], state["rq"], state["rs"])
    return [p, m.float(), v.float(), state["shadow"]]


def _plain_loss(state):
    x = state["logits"].float()
    rows, targets = torch.arange(x.shape[0], device=DEV), state["targets"].long()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    loss = ((top + torch.log(total)).flatten() - x[rows, targets]).double() * state["weight"]
    grad = e / total
    grad[rows, targets] -= 1.0
    grad *= state["weight"].float()[:, None]
    return loss.sum().float().reshape(1), grad.to(state["logits"].dtype)


# ------------------------------------------------------------------------------------------ what a pass cannot avoid

def work(case):
    if case["op"] in ("product", "weight_grad"):
        sizes, rows, k, n = _rows_of(case)[0], case["rows"], case["k"], case["n"]
        flops = 2.0 * rows * k * n
        if case["op"] == "product":
            live = sum(1 for s in sizes if s)
            size = 2 if case["out"] == "bf16" else 4
            return {"bytes": 2.0 * rows * k + 2.0 * live * k * n + size * float(rows + case["behind"]) * n, "flops": flops}
        return {"bytes": 2.0 * rows * (k + n) + 4.0 * case["groups"] * k * n, "flops": flops}
    if case["op"] == "adamw":
        each = 8 + (4 if case["grad"] == "f32" else 2) + (2 if case["shadow"] else 0)
        each += 16 if case["bits"] == 32 else 4 + 16.0 / BLOCK + 8     # 8 bits: the states' values are read out as well
        return {"bytes": float(each) * case["total"], "flops": 16.0 * case["total"]}
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": 2.0 * size * case["tokens"] * case["vocab"], "flops": 5.0 * case["tokens"] * case["vocab"]}


# ------------------------------------------------------------------------------------------------ the same in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("product", "weight_grad"):
        _, edges = _rows_of(case)
        pairs = list(zip(edges, edges[1:]))
        if case["op"] == "product":
            y = torch.zeros(st["x"].shape[0], case["n"], dtype=torch.float64, device=DEV)
            for g, (a, b) in enumerate(pairs):
                y[a:b] = st["x"][a:b].double() @ st["w"][g].double()
            return y
        return torch.stack([st["x"][a:b].double().T @ st["dy"][a:b].double() for a, b in pairs])
    if case["op"] == "adamw":
        return _exact_adamw(case, st)
    total, grad = 0.0, torch.empty(st["logits"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for a, s in zip(st["adv"], st["lens"]):
        for r0 in range(row, row + s, 256):
            r1 = min(row + s, r0 + 256)
            logp = torch.log_softmax(st["logits"][r0:r1].double(), 1)
            hit = torch.zeros_like(logp).scatter_(1, st["targets"][r0:r1, None].long(), 1.0)
            total = total - (logp * hit).sum() * a / s
            grad[r0:r1] = (logp.exp() - hit) * (a / s)
        row += s
    return total.reshape(1), grad


def _exact_adamw(case, st):
    t = st["t"] + 1
    g, p = st["grad"].double(), st["p"].double()
    if case["bits"] == 32:
        m, v = st["m"].double(), st["v"].double()
    else:
        m = st["mq"].double() * st["mq"].double().abs() * st["ms"].double().repeat_interleave(BLOCK)
        v = (st["rq"].double() ** 2 * st["rs"].double().repeat_interleave(BLOCK)) ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    p = (1 - LR * DECAY) * p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS)
    if case["bits"] == 8:
        top = m.abs().view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)
        q = (torch.where(top > 0, 127 * (m.abs() / top) ** 0.5, 0) - 0.5).ceil()
        m = m.sign() * (q / 127) ** 2 * top
        root = v ** 0.5
        top = root.view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)
        q = (torch.where(top > 0, 255 * (root / top) ** 0.5, 0) - 0.5).ceil()
        q = torch.where(v > 0, q.clamp(min=1), q)
        v = ((q / 255) ** 2 * top) ** 2
    return [p, m, v, p if case["shadow"] else None]
