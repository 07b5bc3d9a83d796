"""The loss gradient of likely tokens, as scored completions mostly are: where the target has nearly
all of a row's probability, its gradient and its loss are the small rest, and must be right to
their own size.

u = 2^-24. An exponential carries the difference, the constant log2 e and the product (3 u d log2 e
for a logit d below the largest) and ex2 (4 u); the sum of the others 8 u for each of at most 48 merges and
of the V / 128 rounds of a thread; quotient, weight and product 8 u; then half a step of the output."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def make(V, dt, targets, rests, pitch=0, off=0, seed=0):
    """Rows whose targets have probability 1 - rest."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = len(targets)
    buf = torch.empty(n * (V + pitch) + off, device=DEV).normal_(0.0, 2.0, generator=g).to(dt)
    x = buf[off:].view(n, V + pitch)[:, :V]
    t = torch.tensor(targets, dtype=torch.int32, device=DEV)
    others = x.double().scatter(1, t.long()[:, None], float("-inf")).logsumexp(1)
    rest = torch.tensor(rests, dtype=torch.float64, device=DEV)
    x.scatter_(1, t.long()[:, None], (others + torch.log((1 - rest) / rest)).to(dt)[:, None])
    return x, t


def check(x, t, loss, grad, w):
    """w: the weight of every row."""
    xd, tl = x.double(), t.long()[:, None]
    V = x.shape[1]
    xt = xd.gather(1, tl)
    hidden = xd.scatter(1, tl, float("-inf"))
    ratio = torch.exp(hidden - xt)                                # e_c / e_target
    rest = ratio.sum(1, keepdim=True)
    nll = torch.log1p(rest).flatten()
    d = xd.amax(1, keepdim=True) - hidden.clamp(min=-1e30)
    # weighed by what each logit adds to the rest
    rel = 3 * U * 1.4427 * (torch.where(ratio > 0, d, 0.0) * ratio).sum(1, keepdim=True) / rest + (4 + 8 * (48 + V / 128) + 8) * U
    half = torch.finfo(grad.dtype).eps / 2
    want = -w * rest / (1 + rest)
    assert bool(((grad.double().gather(1, tl) - want).abs() <= (rel + half) * want.abs()).all())
    others = w * ratio / (1 + rest)
    tol = (3 * U * 1.4427 * torch.where(ratio > 0, d, 0.0) + rel + half) * others.abs() + 1e-37
    assert bool(((grad.double() - others).abs().scatter(1, tl, 0.0) <= tol).all())
    err = float((abs(w) * nll * rel.flatten()).sum())
    assert abs(float(loss) - w * float(nll.sum())) <= err + U * abs(w) * float(nll.sum())


RESTS = [0.5, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 1e-7, 1e-8, 1e-9, 1e-12]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [2, 9, 1000, 5001, 32003, 152064])
def test_likely_targets(V, dt):
    from dsmezo_b200 import scoring
    g = torch.Generator().manual_seed(V)
    for s in range(4):
        targets = torch.randint(0, V, (len(RESTS),), generator=g).tolist()
        x, t = make(V, dt, targets, RESTS, seed=s)
        w = 1.5 / len(RESTS)
        loss, grad = scoring.contrastive_loss_grad(x, [len(RESTS)], [1.5], t)
        check(x, t, loss, grad, w)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,pitch,off", [(5001, 3, 1), (20011, 5, 7), (203, 1, 3), (70007, 0, 0)])
def test_every_place_of_the_target(V, pitch, off, dt):
    """Head, tail, slice borders, every element of a vector: none is counted twice or left out."""
    from dsmezo_b200 import scoring
    per = [(V + c - 1) // c for c in (1, 2, 4, 8)]
    places = sorted({p for c in range(9) for q in per for p in range(c * q - 9, c * q + 10) if 0 <= p < V} | set(range(min(V, 24))) |
                    set(range(max(0, V - 24), V)) | set(range(V // 3, min(V, V // 3 + 40))))
    x, t = make(V, dt, places, [1e-6] * len(places), pitch, off)
    n = len(places)
    loss, grad = scoring.contrastive_loss_grad(x, [n], [-2.0], t)
    check(x, t, loss, grad, -2.0 / n)
    y = x.clone()
    loss2, grad2 = scoring.contrastive_loss_grad(y, [n], [-2.0], t, out=y)
    assert grad2 is y and torch.equal(loss, loss2)
    check(x, t, loss2, y, -2.0 / n)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_infinite_targets(dt):
    """+inf in the target's place: NaN, as the formula."""
    from dsmezo_b200 import scoring
    x = torch.randn(2, 1000, device=DEV).to(dt)
    t = torch.tensor([5, 700], dtype=torch.int32, device=DEV)
    x[0, 5] = float("inf")
    loss, grad = scoring.contrastive_loss_grad(x, [2], [1.0], t)
    assert torch.isnan(loss).all() and torch.isnan(grad[0]).all() and torch.isfinite(grad[1]).all()
    x[0, 5] = float("nan")
    loss, grad = scoring.contrastive_loss_grad(x, [2], [1.0], t)
    assert torch.isnan(loss).all() and torch.isnan(grad[0]).all() and torch.isfinite(grad[1]).all()
    x[0] = float("-inf")                                          # nothing but the target: a loss of 0
    x[0, 5] = -3.0
    loss, grad = scoring.contrastive_loss_grad(x[:1], [1], [1.0], t[:1])
    assert float(loss) == 0.0 and grad.eq(0).all()
