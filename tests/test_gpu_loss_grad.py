"""The scoring loss with its gradient (scoring.contrastive_loss_grad) against fp64.

u = 2^-24. With x the logit and m the row's largest, an exponential carries the difference, the
constant log2 e and the product (3 u |x - m| log2 e) and ex2 (4 u); the sum adds up to
8 u for each of the merges of a thread's rounds and of the warp, CTA and cluster (at most 40
and the rounds), and u for each addition of a thread's run, bounded by its length. The
gradient then takes the quotient, the difference with 1, the weight and its product (6 u of
|w|), and half a step of its type (bf16 2^-8)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def S():
    from dsmezo_b200 import scoring
    return scoring


def weights(lens, adv):
    return torch.tensor([a / n for a, n in zip(adv, lens) for _ in range(n)], dtype=torch.float64, device=DEV)


def check(logits, lens, adv, targets, loss, grad, scale=1.0):
    """Against the formula in fp64; `logits` as they were."""
    x, w = logits.double(), weights(lens, adv)
    V = x.shape[1]
    # the maximum is subtracted first: next to the type's lowest value (3e38, where a step of fp64
    # is 4e22) x - logsumexp(x) would lose the logarithm
    top = x.amax(1, keepdim=True)
    total = torch.exp(x - top).sum(1, keepdim=True)
    nll = (top - x.gather(1, targets.long()[:, None]) + torch.log(total)).flatten()
    p = torch.exp(x - top) / total
    hit = torch.zeros_like(p).scatter_(1, targets.long()[:, None], 1.0)
    want = (p - hit) * w[:, None] * scale
    runs = 8.0 * (V / 128 + 48) * U                        # the sum's relative error
    d = torch.where(p > 0, (x.amax(1, keepdim=True) - x) * 1.4427, 0.0)
    tol = (w[:, None] * scale).abs() * (p * (3 * U * d + 4 * U + runs) + 6 * U) + HALF[grad.dtype] * want.abs() + 1e-37
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    assert bool(((grad.double() - want).abs() <= tol).all())
    err = float((w.abs() * (runs + U)).sum()) + U * abs(float((w * nll).sum()))
    assert loss.dtype == torch.float32 and loss.shape == (1,)
    assert abs(float(loss) - float((w * nll).sum())) <= err + 1e-37


def rows(ntok, V, dt, seed, scale=4.0, pitch=0, off=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    buf = torch.empty(ntok * (V + pitch) + off, dtype=dt, device=DEV).normal_(0, scale, generator=g)
    t = torch.randint(0, V, (ntok,), generator=g, device=DEV, dtype=torch.int32)
    return buf[off:].view(ntok, V + pitch)[:, :V], t


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 31, 100, 1000, 4099, 20480, 32003, 81929, 152064])
def test_vocabularies(S, V, dt):
    lens, adv = [3, 1, 2], [0.7, -1.3, 0.4]
    x, t = rows(6, V, dt, V)
    loss, grad = S.contrastive_loss_grad(x, lens, adv, t)
    check(x, lens, adv, t, loss, grad)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pitch,off,goff", [(1, 0, 0), (3, 1, 1), (0, 5, 5), (8, 8, 0), (5, 2, 7)])
def test_pitches_and_alignments(S, dt, pitch, off, goff):
    V, lens, adv = 5001, [4, 5], [1.0, -0.25]
    x, t = rows(9, V, dt, 3, pitch=pitch, off=off)
    wide = torch.full((9 * (V + 4) + 16,), 3.0, dtype=dt, device=DEV)
    out = wide[goff:goff + 9 * (V + 4)].view(9, V + 4)[:, :V]
    loss, grad = S.contrastive_loss_grad(x, lens, adv, t, out=out, grad_scale=0.5)
    assert grad is out
    check(x, lens, adv, t, loss, grad, 0.5)
    around = wide.clone()
    around[goff:goff + 9 * (V + 4)].view(9, V + 4)[:, :V] = 3.0
    assert around.eq(3.0).all()                                   # nothing beside the rows was written


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ntok", [1, 40, 700])
def test_in_place_and_repeatable(S, dt, ntok):
    V = 20011
    lens, adv = ([1], [2.0]) if ntok == 1 else ([1, ntok - 1], [2.0, -0.5])
    x, t = rows(ntok, V, dt, 17)
    a = S.contrastive_loss_grad(x, lens, adv, t)
    b = S.contrastive_loss_grad(x, lens, adv, t)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    y = x.clone()
    loss, grad = S.contrastive_loss_grad(y, lens, adv, t, out=y)
    assert grad is y and torch.equal(loss, a[0]) and torch.equal(y, a[1])
    check(x, lens, adv, t, loss, grad)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_masked_and_infinite_logits(S, dt):
    V, lens, adv = 3000, [7], [1.5]
    x, t = rows(7, V, dt, 29)
    t[:] = 1234
    x[0, :1000] = float("-inf")                                  # a masked stretch
    x[1, :1234], x[1, 1235:] = float("-inf"), float("-inf")      # only the target left
    x[2] = torch.finfo(dt).min                                   # every logit the type's lowest: uniform
    x[3, 1234] = torch.finfo(dt).max
    ok = torch.tensor([0, 1, 2, 3], device=DEV)
    loss, grad = S.contrastive_loss_grad(x[:4], [4], adv, t[:4])
    check(x[:4], [4], adv, t[:4], loss, grad)
    assert grad[1].eq(0).all() and len(ok) == 4
    x[4] = float("-inf")                                         # nothing left: NaN, as the formula
    x[5, 77] = float("inf")
    x[6, 5] = float("nan")
    loss, grad = S.contrastive_loss_grad(x, lens, adv, t)
    assert torch.isnan(loss).all() and torch.isnan(grad[4:]).all() and torch.isfinite(grad[:4]).all()
    x[4:] = 0.0
    x[4, 1234] = float("-inf")                                   # an impossible target: infinite loss, finite gradient
    loss, grad = S.contrastive_loss_grad(x, lens, adv, t)
    assert torch.isinf(loss).all() and torch.isfinite(grad).all()


def test_target_outside_the_vocabulary(S):
    x, t = rows(6, 400, torch.float32, 5)
    t[3] = 400
    loss, grad = S.contrastive_loss_grad(x, [3, 3], [1.0, -1.0], t)
    assert torch.isnan(loss).all() and torch.isnan(grad[3]).all()
    assert torch.isfinite(grad[[0, 1, 2, 4, 5]]).all()
    t[3] = -1
    assert torch.isnan(S.contrastive_loss_grad(x, [3, 3], [1.0, -1.0], t)[0]).all()


def test_agrees_with_the_loss_and_its_differences(S):
    V, lens, adv = 501, [2, 3], [0.9, -0.6]
    x, t = rows(5, V, torch.float32, 41, scale=1.0)
    loss, grad = S.contrastive_loss_grad(x, lens, adv, t)
    assert abs(float(loss) - float(S.contrastive_loss(x, lens, adv, t))) <= 1e-6 * max(1.0, abs(float(loss)))
    w = weights(lens, adv)

    def f(z):
        return float((w * (torch.logsumexp(z, 1) - z.gather(1, t.long()[:, None]).flatten())).sum())
    g = torch.Generator().manual_seed(0)
    for _ in range(8):
        i, j = int(torch.randint(5, (1,), generator=g)), int(torch.randint(V, (1,), generator=g))
        h = 1e-4
        up, dn = x.double().clone(), x.double().clone()
        up[i, j] += h
        dn[i, j] -= h
        # central difference: h^2 / 6 times a third derivative of at most 1, and fp64 noise over h
        assert abs((f(up) - f(dn)) / (2 * h) - float(grad[i, j])) < 1e-8 + 1e-11 / h + 8 * U


def test_many_sequences_and_zero_advantages(S):
    lens = [1 + i % 5 for i in range(128)]
    adv = [0.0 if i % 3 == 0 else (-1) ** i * 0.1 * i for i in range(128)]
    x, t = rows(sum(lens), 257, torch.bfloat16, 6)
    loss, grad = S.contrastive_loss_grad(x, lens, adv, t)
    check(x, lens, adv, t, loss, grad)
    assert grad[0].eq(0).all()


def test_captured_call_follows_its_inputs(S):
    V, lens, adv = 9000, [5, 3], [1.0, -1.0]
    x, t = rows(8, V, torch.bfloat16, 7)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        S.contrastive_loss_grad(x, lens, adv, t)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = S.contrastive_loss_grad(x, lens, adv, t)
    for seed in (8, 9):
        y, u = rows(8, V, torch.bfloat16, seed)
        x.copy_(y)
        t.copy_(u)
        graph.replay()
        torch.cuda.synchronize()
        check(x, lens, adv, t, loss, grad)


def test_offsets_past_32_bits(S):
    # 15000 rows of the Qwen2.5 vocabulary: 2.3e9 logits, in place; the rows are copies of 50
    V, n = 152064, 15000
    base, t50 = rows(50, V, torch.bfloat16, 12)
    x = base.repeat(n // 50, 1)
    t = t50.repeat(n // 50)
    lens, adv = [n], [float(n)]
    loss, _ = S.contrastive_loss_grad(x, lens, adv, t, out=x)
    for a in (0, 14100, n - 50):
        check(base, [50], [50.0], t50, loss / (n / 50), x[a:a + 50])
    assert torch.equal(x[:50], x[-50:])


@pytest.mark.parametrize("dt,V", [(torch.bfloat16, 40000), (torch.bfloat16, 32771), (torch.float32, 20001), (torch.float32, 65536)])
def test_many_long_rows(S, dt, V):
    # two waves of rows past 64 KB, ragged last slices, in place too
    n, pitch = 330, (-V) % 8 + 8
    x, t = rows(n, V, dt, 31, pitch=pitch)
    t[5], t[6], t[7] = V - 1, 0, V // 8 * 8 - 1
    lens, adv = [100, 1, 229], [1.0, -2.0, 0.5]
    loss, grad = S.contrastive_loss_grad(x, lens, adv, t)
    check(x, lens, adv, t, loss, grad)
    again = S.contrastive_loss_grad(x, lens, adv, t)
    assert torch.equal(again[0], loss) and torch.equal(again[1], grad)
    old = x.clone()
    x[300, 17:] = float("-inf")
    x[301] = float("-inf")
    x[302, 5] = float("nan")
    x[303] = torch.finfo(dt).min
    t[300], t[304] = 3, V
    bad = S.contrastive_loss_grad(x, lens, adv, t)
    assert torch.isnan(bad[0]).all() and torch.isnan(bad[1][[301, 302, 304]]).all()
    assert torch.isfinite(bad[1][:301]).all() and torch.isfinite(bad[1][303]).all()
    t[300], t[304] = 1, 1
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    keep[301:303] = False
    for i in (300, 303):
        one = S.contrastive_loss_grad(x[i:i + 1], [1], [0.5 / 229], t[i:i + 1])[1]
        check(x[i:i + 1], [1], [0.5 / 229], t[i:i + 1], S.contrastive_loss_grad(x[i:i + 1], [1], [0.5 / 229], t[i:i + 1])[0], one)
    x.copy_(old)
    buf = x.clone(memory_format=torch.preserve_format)
    loss2, out = S.contrastive_loss_grad(buf, lens, adv, t, out=buf)
    check(x, lens, adv, t, loss2, out)


def test_refusals(S):
    x, t = rows(4, 64, torch.float32, 1)
    ok = dict(seq_tokens=[4], advantages=[1.0], targets=t)
    bad = [dict(ok, seq_tokens=[3]), dict(ok, advantages=[]), dict(ok, targets=t.long()), dict(ok, targets=t[:3]),
           dict(ok, targets=t.cpu()), dict(ok, out=x[:3]), dict(ok, out=x.bfloat16()), dict(ok, out=x.t())]
    for kw in bad:
        with pytest.raises(ValueError):
            S.contrastive_loss_grad(x, **kw)
    with pytest.raises(TypeError):
        S.contrastive_loss_grad(x.half(), **ok)
    with pytest.raises(ValueError):
        S.contrastive_loss_grad(x.t(), [64], [1.0], t)
    from dsmezo_b200 import DsmzError
    buf = torch.zeros(8 * 64, device=DEV)
    for kw in (dict(ok, seq_tokens=[4, 0], advantages=[1.0, 1.0]), dict(ok, seq_tokens=[5, -1], advantages=[1.0, 1.0]),
               dict(ok, grad_scale=float("nan")), dict(ok, out=buf[32:32 + 256].view(4, 64))):
        with pytest.raises(DsmzError):
            S.contrastive_loss_grad(buf[:256].view(4, 64), **kw)
    many, tm = rows(129, 8, torch.float32, 2)
    with pytest.raises(DsmzError):
        S.contrastive_loss_grad(many, [1] * 129, [1.0] * 129, tm)
