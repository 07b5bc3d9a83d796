"""A first-order step of an adapter set: products through the adapters, the scoring loss with
its gradient, the factors' gradients and AdamW, run one after another as a user runs them and
checked against fp64."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U, UB = 2.0 ** -24, 2.0 ** -8
LENS, ADV = [9, 4, 12], [0.8, -0.5, 0.3]
LR, B1, B2, EPS, WD = 1e-3, 0.9, 0.999, 1e-8, 0.01


def make_set(seed=0, directions=1, rank=16, dt=torch.bfloat16):
    from dsmezo_b200 import AdapterSet, transformer_adapter_shapes
    mods, bases = transformer_adapter_shapes(1, 192, 520, 64, 64)
    aset = AdapterSet(mods, bases, rank, rank, copy_dtype=dt, directions=directions)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for i, m in enumerate(mods):
        aset.A(i).copy_(torch.randn(m.d_out, rank, generator=g, device=DEV) * rank ** -0.5)
        aset.B(i).copy_(torch.randn(rank, m.d_in, generator=g, device=DEV) * m.d_in ** -0.5)
    aset.sync_shadow()
    return aset, g


def batch(aset, g, i):
    rows = sum(LENS)
    x = torch.randn(rows, aset.modules[i].d_in, generator=g, device=DEV).bfloat16()
    base = (torch.randn(rows, aset.modules[i].d_out, generator=g, device=DEV) * 2).bfloat16()
    targets = torch.randint(0, aset.modules[i].d_out, (rows,), generator=g, device=DEV, dtype=torch.int32)
    return x, base, targets


def step(aset, opt, grad, data, i):
    """logits = base + delta(x); loss; gradients of A and B; AdamW."""
    from dsmezo_b200 import scoring
    x, base, targets = data
    logits = base.clone()
    _, t = aset.delta(i, x, out=logits, accumulate=True)
    loss, dlogits = scoring.contrastive_loss_grad(logits, LENS, ADV, targets, out=logits)
    dx = aset.delta_backward(i, dlogits, x, t, grad)
    opt.step()
    return loss, dx


@pytest.mark.parametrize("bits", [32, 8])
def test_one_step_against_fp64(bits):
    from dsmezo_b200 import AdamW
    aset, g = make_set()
    i = next(k for k, m in enumerate(aset.modules) if m.name == "gate_proj")
    data = batch(aset, g, i)
    x, base, targets = data
    A0, B0 = aset.A(i, aset.shadow).double().requires_grad_(), aset.B(i, aset.shadow).double().requires_grad_()
    xd = x.double().requires_grad_()
    logits = base.double() + (xd @ B0.T) @ A0.T
    w = torch.tensor([a / n for a, n in zip(ADV, LENS) for _ in range(n)], dtype=torch.float64, device=DEV)
    nll = torch.logsumexp(logits, 1) - logits.gather(1, targets.long()[:, None]).flatten()
    want = (w * nll).sum()
    want.backward()
    grad = aset.grad_arena()
    opt = AdamW.for_adapters(aset, grad, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits)
    before = aset.factors.clone()
    loss, dx = step(aset, opt, grad, data, i)
    # t, the logits, their gradient and the gradient in t are bf16: each rounding moves an entry by
    # at most 2^-8 of itself. A logit is off by 2^-8 of itself and of t's part, so the loss by that
    # times 2 |w|, and the gradients' entries by four such roundings, each of which is a random
    # fraction of its bound: a Frobenius distance of 4 * 2^-8 holds every one at its bound.
    size = float((logits.abs().max() + ((xd @ B0.T).abs() @ A0.abs().T).max()).detach())
    assert abs(float(loss) - float(want.detach())) <= 2 * UB * size * float(w.abs().sum())
    p = torch.softmax(logits.detach(), 1)
    for got, ref in ((aset.A(i, grad), A0.grad), (aset.B(i, grad), B0.grad), (dx, xd.grad)):
        # the softmax moves by at most the logits' error times itself
        assert float((got.double() - ref).norm() / ref.norm()) <= 4 * UB + 2 * UB * size * float(p.amax())
    # every factor moved as AdamW says from its own gradient: at step 1 from zeroed states the
    # update is lr g / (|g| + eps (1 - b2)^1/2 / ...): both moments are exact multiples of g
    gd = grad.double()
    m, v = (1 - B1) * gd, (1 - B2) * gd * gd
    upd = LR * (m / (1 - B1)) / ((v / (1 - B2)).sqrt() + EPS)
    p1 = before[:aset.numel].double() * (1 - LR * WD) - upd
    got = aset.factors[:aset.numel].double()
    assert bool(((got - p1).abs() <= 3 * U * before[:aset.numel].abs() + 20 * U * upd.abs() + 1e-12).all())
    assert torch.equal(aset.shadow[:aset.numel], aset.factors[:aset.numel].bfloat16())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays(bits):
    # the whole step in one graph, replayed, against the same steps run eagerly
    from dsmezo_b200 import AdamW

    def fresh(capturable):
        aset, g = make_set(3)
        i = 1
        data = batch(aset, g, i)
        grad = aset.grad_arena()
        return aset, AdamW.for_adapters(aset, grad, lr=LR, state_bits=bits, capturable=capturable), grad, data, i
    a = fresh(True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*a)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _ = step(*a)
    for _ in range(4):
        graph.replay()
    b = fresh(True)
    for _ in range(5):
        eager, _ = step(*b)
    torch.cuda.synchronize()
    assert torch.equal(a[0].factors, b[0].factors) and torch.equal(a[0].shadow, b[0].shadow)
    assert torch.equal(loss, eager) and torch.equal(a[2], b[2])
    assert int(a[1].step_counter) == 5


def test_accumulated_gradients_and_every_module():
    # two micro-batches into one arena equal the sum of their gradients
    aset, g = make_set(4)
    for i, m in enumerate(aset.modules):
        parts = []
        for _ in range(2):
            x = torch.randn(40, m.d_in, generator=g, device=DEV).bfloat16()
            dy = torch.randn(40, m.d_out, generator=g, device=DEV).bfloat16()
            parts.append((dy, x, aset.delta(i, x)[1]))
        both, one, two = aset.grad_arena(), aset.grad_arena(), aset.grad_arena()
        for k, (dy, x, t) in enumerate(parts):
            aset.delta_backward(i, dy, x, t, both, accumulate=k > 0, need_dx=False)
        aset.delta_backward(i, *parts[0], one)
        aset.delta_backward(i, *parts[1], two)
        assert bool(((both - (one + two)).abs() <= 2 * U * (one.abs() + two.abs())).all())
        n = aset.offA[i]
        assert both[:n].eq(0).all() and both[aset.offB[i] + aset.rank * m.d_in:].eq(0).all()


def test_products_of_the_perturbed_copies():
    # four directions: rows sorted by copy, ragged, one copy without rows
    aset, g = make_set(5, directions=4)
    aset.pos.copy_(torch.randn(aset.pos.shape, generator=g, device=DEV) * 0.2)
    aset.neg.copy_(torch.randn(aset.neg.shape, generator=g, device=DEV) * 0.2)
    edges = [0, 30, 30, 77, 100]
    off = torch.tensor(edges, dtype=torch.int32, device=DEV)
    for i, m in enumerate(aset.modules):
        x = torch.randn(100, m.d_in, generator=g, device=DEV).bfloat16()
        for which in ("pos", "neg"):
            y, t = aset.delta(i, x, which, off)
            for k in range(4):
                a, b = edges[k], edges[k + 1]
                arena = aset.pos_dir(k) if which == "pos" else aset.neg_dir(k)
                A, B = aset.A(i, arena).double(), aset.B(i, arena).double()
                tk = x[a:b].double() @ B.T
                lim = m.d_in * 2 * U * (x[a:b].double().abs() @ B.abs().T) + UB * tk.abs()
                assert bool(((t[a:b].double() - tk).abs() <= lim + 1e-30).all())
                yk = t[a:b].double() @ A.T
                lim = aset.rank * 2 * U * (t[a:b].double().abs() @ A.abs().T) + UB * yk.abs()
                assert bool(((y[a:b].double() - yk).abs() <= lim + 1e-30).all())


def test_refusals():
    aset, _ = make_set(6, directions=2)
    x = torch.zeros(8, aset.modules[0].d_in, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        aset.delta(0, x, "pos")                       # two copies, no offsets
    with pytest.raises(ValueError):
        aset.delta(0, x, "factors")
    with pytest.raises(ValueError):
        aset.delta(0, x[:, :8])
    y, t = aset.delta(0, x)
    with pytest.raises(ValueError):
        aset.delta_backward(0, y, x, t, torch.zeros(3, device=DEV))
    with pytest.raises(ValueError):
        make_set(7, dt=torch.float32)[0].delta(0, x)
    assert aset.delta(0, x[:0])[0].shape == (0, aset.modules[0].d_out)
