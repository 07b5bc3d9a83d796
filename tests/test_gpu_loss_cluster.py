"""The loss gradient where a row belongs to a cluster of CTAs whose slices are as short as the launch
makes them, so that a CTA reaches the exchange of the row's statistics right after its start:
results against fp64, equal on every run while other launches of both shapes come and go."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24                         # half a step of fp32


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
# row bytes just above 8, 16, 32 and 64 KB: 2, 4, 8 and 8 CTAs a row
@pytest.mark.parametrize("kb", [8, 16, 32, 64])
@pytest.mark.parametrize("ntok", [1, 7, 64])
def test_short_slices(kb, ntok, dt):
    from dsmezo_b200 import scoring
    V = kb * 1024 // dt.itemsize + 9
    g = torch.Generator(device=DEV).manual_seed(kb + ntok)
    x = torch.randn(ntok, V, generator=g, device=DEV).to(dt)
    t = torch.randint(0, V, (ntok,), generator=g, device=DEV, dtype=torch.int32)
    loss, grad = scoring.contrastive_loss_grad(x, [ntok], [1.5], t)
    xd, w = x.double(), 1.5 / ntok
    p = torch.softmax(xd, 1)
    hit = torch.zeros_like(p).scatter_(1, t.long()[:, None], 1.0)
    want = (p - hit) * w
    # an exponential: 3 u |x - m| log2 e <= 60 u and 4 u; a thread's run and the merges: 8 u each for at most
    # 48 of them and u for each of V / 128 elements; weight and quotient 6 u
    rel = (64 + 8 * 48 + V / 128) * U
    tol = w * (p * rel + 6 * U) + (torch.finfo(dt).eps / 2) * want.abs()
    assert bool(((grad.double() - want).abs() <= tol).all())
    nll = torch.logsumexp(xd, 1) - xd.gather(1, t.long()[:, None]).flatten()
    assert abs(float(loss) - w * float(nll.sum())) <= w * ntok * rel + U * w * float(nll.sum())
    other = torch.randn(3, 20000, generator=g, device=DEV).to(dt)
    ot = torch.zeros(3, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            scoring.contrastive_loss_grad(other, [3], [1.0], ot)
    for _ in range(20):
        again = scoring.contrastive_loss_grad(x, [ntok], [1.5], t)
        assert torch.equal(again[0], loss) and torch.equal(again[1], grad)
    torch.cuda.current_stream().wait_stream(side)
