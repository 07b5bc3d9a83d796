"""Products grouped by adapter copy (dsmezo_b200.grouped) against fp64.

Products of two bf16 numbers are exact in fp32. The tensor core adds with at most one step of
the running sum lost an addition (2^-23, rounding towards zero): n additions err by n 2^-23 of
sum |x w|. fp32 outputs take at most 512 products in an accumulator and add the accumulators
(and at most 8 partial sums of a split contraction): n = 512 + K / 512 + 8. bf16 outputs take
the whole contraction, n = K + 8, and half a bf16 step, 2^-8. alpha and an accumulated term
add a rounding each."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U23, U, UB = 2.0 ** -23, 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module")
def Gr():
    from dsmezo_b200 import grouped
    yield grouped
    assert grouped.device_error("cuda") == 0


def rnd(shape, seed, scale=1.0, dt=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dt)


def offs(edges):
    return torch.tensor(edges, dtype=torch.int32, device=DEV)


def split(M, G, kind, before=0, after=0):
    if kind == "even":
        cut = [before + (M - before - after) * i // G for i in range(G + 1)]
    else:
        g = torch.Generator().manual_seed(M * 31 + G)
        w = torch.rand(G, generator=g) ** 3
        if kind == "empty":
            w[::2] = 0
        c = torch.cat([torch.zeros(1), torch.cumsum(w, 0) / max(float(w.sum()), 1e-9)])
        cut = [before + int(round(float(v) * (M - before - after))) for v in c]
    return cut


def check_product(x, w, edges, y, old=None, alpha=1.0, accumulate=False):
    M, K = x.shape
    N = w.shape[2]
    got = y.double()
    covered = torch.zeros(M, dtype=torch.bool, device=DEV)
    for g, (a, b) in enumerate(zip(edges, edges[1:])):
        if b <= a:
            continue
        covered[a:b] = True
        p = x[a:b].double() @ w[g].double()
        s = x[a:b].double().abs() @ w[g].double().abs()
        want = alpha * p + (old[a:b].double() if accumulate else 0.0)
        n = 512 + K / 512 + 8 if y.dtype == torch.float32 else K + 8
        tol = abs(alpha) * (n * U23 * s + 2 * U * p.abs()) + 2 * U * want.abs() + 1e-30
        if y.dtype == torch.bfloat16:
            tol = tol + UB * want.abs()
        bad = (got[a:b] - want).abs() > tol
        assert not bool(bad.any()), (g, int(bad.sum()), bad.nonzero()[:3].tolist())
        assert bool(torch.isfinite(got[a:b]).all())
    rest = y[~covered]
    assert bool((rest == (0 if old is None else old[~covered])).all())      # zero, or as it was
    assert N == y.shape[1]


SHAPES = [(1, 1, 8, 8), (1, 1, 1, 1), (3, 2, 5, 3), (5, 3, 64, 64), (130, 2, 200, 72), (300, 4, 3584, 64),
          (257, 5, 64, 1000), (513, 7, 1536, 16), (1000, 32, 128, 520), (96, 64, 8, 2000), (700, 3, 1000, 128),
          (385, 2, 72, 264), (2048, 2, 3584, 16), (640, 6, 16, 8960)]


@pytest.mark.parametrize("M,G,K,N", SHAPES)
@pytest.mark.parametrize("major", ["k", "n"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_products(Gr, M, G, K, N, major, dt):
    for kind in ("even", "ragged", "empty"):
        edges = split(M, G, kind)
        x = rnd((M, K), 1)
        w = rnd((G, N, K), 2, K ** -0.5).transpose(1, 2) if major == "k" else rnd((G, K, N), 2, K ** -0.5)
        y = Gr.grouped_matmul(x, w, offs(edges), out_dtype=dt)
        check_product(x, w, edges, y)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,pitch", [(64, 72), (100, 101), (264, 300)])
def test_rows_outside_accumulation_and_pitches(Gr, dt, N, pitch):
    M, G, K = 400, 3, 320
    edges = split(M, G, "ragged", before=37, after=90)
    x = rnd((M, K + 24), 3)[:, 8:8 + K]                       # a column slice: its own pitch, aligned rows
    w = rnd((G, K, N + 8), 4, 0.05)[:, :, :N] if N % 8 == 0 else rnd((G, K, N), 4, 0.05)
    for off in (0, 1):
        buf = rnd(M * pitch + 8, 5, dt=dt)
        out = buf[off:off + M * pitch].view(M, pitch)[:, :N]
        keep = buf.clone()
        old = out.clone()
        assert Gr.grouped_matmul(x, w, offs(edges), out=out, alpha=-0.5, accumulate=True) is out
        check_product(x, w, edges, out, old, -0.5, True)
        Gr.grouped_matmul(x, w, offs(edges), out=out, alpha=2.0)
        check_product(x, w, edges, out, old, 2.0)
        out.copy_(old)
        assert torch.equal(buf, keep)                        # nothing beside the rows was written


def test_layouts_that_need_a_copy(Gr):
    M, G, K, N = 90, 2, 50, 30
    edges = [0, 40, 90]
    x = rnd((K, M), 6).t()                                   # column-major
    w = rnd((G, 2 * K, N), 7)[:, ::2]                        # every other row, odd pitch
    check_product(x, w, edges, Gr.grouped_matmul(x, w, offs(edges), out_dtype=torch.float32))
    one = rnd((1, K, N), 8).expand(G, K, N)                  # one matrix for all groups
    check_product(x, one, edges, Gr.grouped_matmul(x, one, offs(edges)))
    y = rnd((M, 3 * K), 9)[:, 1:1 + K]                       # rows that start off a 16-byte boundary
    check_product(y, w, edges, Gr.grouped_matmul(y, w, offs(edges)))


def test_neighbours_do_not_leak(Gr):
    M, G, K, N = 300, 4, 136, 40
    edges = [10, 75, 75, 200, 290]
    x, w, dy = rnd((M, K), 10), rnd((G, K, N), 11), rnd((M, N), 12)
    for bad in (float("nan"), float("inf")):
        xb, db = x.clone(), dy.clone()
        xb[:10], xb[75:200], xb[290:] = bad, bad, bad
        db[:10], db[75:200], db[290:] = bad, bad, bad
        y = Gr.grouped_matmul(xb, w, offs(edges))
        assert torch.equal(y[10:75], Gr.grouped_matmul(x, w, offs(edges))[10:75])
        assert torch.isfinite(y[200:290]).all() and y[290:].eq(0).all()
        a, b = Gr.grouped_weight_grad(xb, db, offs(edges)), Gr.grouped_weight_grad(x, dy, offs(edges))
        assert torch.equal(a[[0, 1, 3]], b[[0, 1, 3]]) and not torch.isfinite(a[2]).any()


def test_offsets_out_of_range_are_clamped(Gr):
    M, K, N = 200, 64, 32
    x, w, dy = rnd((M, K), 13), rnd((4, K, N), 14), rnd((M, N), 15)
    given, meant = [-5, 60, 20, 150, 900], [0, 60, 60, 150, 200]
    check_product(x, w, meant, Gr.grouped_matmul(x, w, offs(given)))
    assert torch.equal(Gr.grouped_weight_grad(x, dy, offs(given)), Gr.grouped_weight_grad(x, dy, offs(meant)))
    big = [2 ** 31 - 1] * 5
    assert Gr.grouped_matmul(x, w, offs(big)).eq(0).all() and Gr.grouped_weight_grad(x, dy, offs(big)).eq(0).all()


def test_many_groups(Gr):
    M, G, K, N = 1500, 1024, 24, 40
    edges = split(M, G, "ragged")
    x, w, dy = rnd((M, K), 16), rnd((G, K, N), 17), rnd((M, N), 18)
    check_product(x, w, edges, Gr.grouped_matmul(x, w, offs(edges), out_dtype=torch.float32))
    check_grad(x, dy, edges, Gr.grouped_weight_grad(x, dy, offs(edges)))


def check_grad(x, dy, edges, dw, old=None, alpha=1.0):
    for g, (a, b) in enumerate(zip(edges, edges[1:])):
        p = x[a:b].double().T @ dy[a:b].double()
        s = x[a:b].double().abs().T @ dy[a:b].double().abs()
        want = alpha * p + (0.0 if old is None else old[g].double())
        n = 512 + (b - a) / 512 + 8
        tol = abs(alpha) * (n * U23 * s + 2 * U * p.abs()) + 2 * U * want.abs() + 1e-30
        assert bool(((dw[g].double() - want).abs() <= tol).all()), (g, a, b)


@pytest.mark.parametrize("M,G,K,N", [(1, 1, 1, 1), (3, 2, 8, 5), (63, 1, 64, 64), (64, 1, 64, 128), (65, 2, 128, 64),
                                     (200, 3, 72, 600), (997, 8, 1536, 16), (1024, 2, 64, 3584), (4096, 2, 16, 1536),
                                     (500, 5, 300, 200), (2500, 1, 264, 520), (100, 40, 16, 264)])
def test_weight_gradients(Gr, M, G, K, N):
    for kind in ("even", "ragged", "empty"):
        edges = split(M, G, kind, before=min(2, M // 9), after=min(5, M // 9))
        x, dy = rnd((M, K), 19), rnd((M, N), 20, 0.1)
        dw = Gr.grouped_weight_grad(x, dy, offs(edges))
        check_grad(x, dy, edges, dw)
        old = rnd((G, K, N), 21, dt=torch.float32)
        acc = old.clone()
        Gr.grouped_weight_grad(x, dy, offs(edges), out=acc, alpha=0.25, accumulate=True)
        check_grad(x, dy, edges, acc, old, 0.25)


@pytest.mark.parametrize("tiles", [1, 12, 16, 20, 24, 30, 36, 50, 76, 150])
@pytest.mark.parametrize("N", [48, 128])
def test_every_way_to_split(Gr, tiles, N):
    # clusters of 8 down to 2 and none: as many row (or feature) tiles as each can hold, the last
    # one ragged, and contractions that do not divide
    M, K = 128 * tiles - 37, 64 * 17 + 8
    x, w = rnd((M, K), 41), rnd((1, K, N), 42, K ** -0.5)
    for dt in (torch.bfloat16, torch.float32):
        check_product(x, w, [0, M], Gr.grouped_matmul(x, w, offs([0, M]), out_dtype=dt))
    wide, rows = 128 * tiles - 24, 1100
    a, b = rnd((rows, wide), 43), rnd((rows, N), 44)
    for u, v in ((a, b), (b, a)):
        check_grad(u, v, [0, rows], Gr.grouped_weight_grad(u, v, offs([0, rows])))


@pytest.mark.parametrize("major", ["k", "n"])
@pytest.mark.parametrize("M,G,K,N", [(4096, 2, 512, 2560), (5000, 7, 776, 3000), (9000, 3, 1024, 1096), (2600, 4, 520, 8968),
                                     (9000, 3, 520, 1025)])
def test_wide_products(Gr, M, G, K, N, major):
    # long groups and wide outputs: pairs of CTAs on 256-row tiles, ragged in every dimension
    x = rnd((M, K), 45)
    w = rnd((G, N, K), 46, K ** -0.5).transpose(1, 2) if major == "k" else rnd((G, K, N), 46, K ** -0.5)
    for kind in ("even", "ragged", "empty"):
        edges = split(M, G, kind, before=3, after=130)
        for dt in (torch.bfloat16, torch.float32):
            check_product(x, w, edges, Gr.grouped_matmul(x, w, offs(edges), out_dtype=dt))
    out = rnd((M, N), 47, dt=torch.float32)
    old = out.clone()
    Gr.grouped_matmul(x, w, offs(edges), out=out, alpha=0.5, accumulate=True)
    check_product(x, w, edges, out, old, 0.5, True)
    assert torch.equal(Gr.grouped_matmul(x, w, offs(edges)), Gr.grouped_matmul(x, w, offs(edges)))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [48, 64, 100, 136, 257, 264])      # 257: most warps have no column of the last tile
@pytest.mark.parametrize("G", [37, 150])                         # long and short groups
def test_many_tiles_a_cta(Gr, dt, N, G):
    # a CTA walks several tiles, whole and partial pieces in turn through the same staging
    M, K = 20011, 72
    edges = split(M, G, "ragged", before=19, after=5)
    x, w = rnd((M, K), 21), rnd((G, N, K), 22, K ** -0.5).transpose(1, 2)
    buf = rnd((M, (N + 23) // 16 * 16), 23, dt=dt)
    out, old = buf[:, :N], buf[:, :N].clone()
    beside = buf[:, N:].clone()
    Gr.grouped_matmul(x, w, offs(edges), out=out)
    check_product(x, w, edges, out, old)
    first = out.clone()
    for _ in range(5):
        out.copy_(old)
        Gr.grouped_matmul(x, w, offs(edges), out=out)
        assert torch.equal(out, first)
    out.copy_(old)
    Gr.grouped_matmul(x, w, offs(edges), out=out, alpha=1.5, accumulate=True)
    check_product(x, w, edges, out, old, 1.5, True)
    assert torch.equal(buf[:, N:], beside)
    check_product(x, w, edges, Gr.grouped_matmul(x, w, offs(edges), out_dtype=dt))


def test_no_rows(Gr):
    w = rnd((3, 16, 24), 22)
    assert Gr.grouped_matmul(rnd((0, 16), 1), w, offs([0, 0, 0, 0])).shape == (0, 24)
    dw = Gr.grouped_weight_grad(rnd((0, 16), 1), rnd((0, 24), 1), offs([0, 0, 0, 0]))
    assert dw.shape == (3, 16, 24) and dw.eq(0).all()


def test_repeatable_and_on_two_streams(Gr):
    M, G, K, N = 900, 3, 2048, 48                             # a split contraction
    edges = offs(split(M, G, "ragged"))
    x, w, dy = rnd((M, K), 23), rnd((G, K, N), 24), rnd((M, N), 25)
    y, dw = Gr.grouped_matmul(x, w, edges), Gr.grouped_weight_grad(x, dy, edges)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [(Gr.grouped_matmul(x, w, edges), Gr.grouped_weight_grad(x, dy, edges)) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, y) and torch.equal(b, dw) for a, b in got)


def test_captured_calls_follow_their_offsets(Gr):
    M, G, K, N = 500, 4, 512, 96
    x, w, dy, o = rnd((M, K), 26), rnd((G, K, N), 27), rnd((M, N), 28), offs([0, 100, 200, 300, 500])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        Gr.grouped_matmul(x, w, o), Gr.grouped_weight_grad(x, dy, o)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dw = Gr.grouped_matmul(x, w, o), Gr.grouped_weight_grad(x, dy, o)
    for edges in ([0, 1, 1, 450, 451], [3, 250, 251, 499, 500], [0, 0, 0, 0, 0]):
        o.copy_(offs(edges))
        x.copy_(rnd((M, K), sum(edges)))
        graph.replay()
        torch.cuda.synchronize()
        check_product(x, w, edges, y)
        check_grad(x, dy, edges, dw)


def test_offsets_past_32_bits(Gr):
    # 150000 rows of 16384: 2.5e9 elements; the last group sits behind 2^31
    M, K, N = 150000, 16384, 16
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=DEV)
    x[-700:] = rnd((700, K), 29)
    w = rnd((2, K, N), 30, K ** -0.5)
    edges = [0, M - 300, M]
    y = Gr.grouped_matmul(x, w, offs(edges))
    assert y[:-700].eq(0).all()
    check_product(x[-700:], w, [0, 400, 700], y[-700:])
    dy = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV)
    dy[-700:] = rnd((700, N), 31)
    check_grad(x[-700:], dy[-700:], [0, 400, 700], Gr.grouped_weight_grad(x, dy, offs(edges)))


@pytest.mark.parametrize("M,G,d_in,d_out,r", [(37, 2, 64, 96, 8), (300, 3, 512, 1408, 16), (150, 4, 1536, 256, 64)])
def test_adapter_and_its_gradients(Gr, M, G, d_in, d_out, r):
    edges = split(M, G, "ragged", after=3)
    x, A, B = rnd((M, d_in), 32), rnd((G, d_out, r), 33, r ** -0.5), rnd((G, r, d_in), 34, d_in ** -0.5)
    dy = rnd((M, d_out), 35, 0.1)
    base = rnd((M, d_out), 36)
    y, t = Gr.adapter_forward(x, A, B, offs(edges), out=base.clone(), alpha=0.5, accumulate=True)
    check_product(x, B.transpose(1, 2), edges, t)
    check_product(t, A.transpose(1, 2), edges, y, base, 0.5, True)
    dx, dA, dB = Gr.adapter_backward(dy, x, t, A, B, offs(edges), alpha=0.5)
    dt = Gr.grouped_matmul(dy, A, offs(edges), alpha=0.5)
    check_product(dy, A, edges, dt, alpha=0.5)
    check_product(dt, B, edges, dx)
    check_grad(dy, t, edges, dA, alpha=0.5)
    check_grad(dt, x, edges, dB)
    # against differences of f = sum dy * y in fp64, where t is not rounded: what the gradients
    # differ by is the rounding of t and dt (2^-8 of their entries)

    def f(xx, AA, BB):
        return sum(float((dy[a:b].double() * (0.5 * (xx[a:b] @ BB[g].T) @ AA[g].T)).sum())
                   for g, (a, b) in enumerate(zip(edges, edges[1:])))
    X, AD, BD = x.double(), A.double(), B.double()
    for which, base_t, grad in (("x", X, dx), ("A", AD, dA), ("B", BD, dB)):
        d = torch.randn(base_t.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64).to(DEV)
        h = 1e-4
        args = {"x": X, "A": AD, "B": BD}
        up, dn = dict(args, **{which: base_t + h * d}), dict(args, **{which: base_t - h * d})
        slope = (f(up["x"], up["A"], up["B"]) - f(dn["x"], dn["A"], dn["B"])) / (2 * h)
        along = float((grad.double() * d).sum())
        # each entry of the gradient is off by at most 2^-8 of the sum of its terms' sizes from t
        # or dt, and 2^-8 of itself where it is bf16; along a random direction these add as a
        # random walk, of which six standard deviations are allowed
        size = float((grad.double() ** 2).sum().sqrt())
        assert abs(slope - along) <= 6 * 2 * UB * size + 1e-6 * abs(slope)


def test_refusals(Gr):
    x, w, o, dy = rnd((10, 16), 1), rnd((2, 16, 24), 2), offs([0, 5, 10]), rnd((10, 24), 3)
    for a in [(x.float(), w, o), (x, w.float(), o), (x, w[0], o), (x[:, :8], w, o), (x, w, o.long()), (x, w, o[:2]),
              (x, w, o.cpu()), (x[0], w, o), (x.cpu(), w, o)]:
        with pytest.raises(ValueError):
            Gr.grouped_matmul(*a)
    with pytest.raises(TypeError):
        Gr.grouped_matmul(x, w, o, out_dtype=torch.float16)
    for kw in (dict(accumulate=True), dict(out=dy[:9]), dict(out=dy.half()), dict(out=rnd((24, 10), 1).t())):
        with pytest.raises(ValueError):
            Gr.grouped_matmul(x, w, o, **kw)
    from dsmezo_b200 import DsmzError
    with pytest.raises(DsmzError):
        Gr.grouped_matmul(x, w, o, alpha=float("inf"))
    buf = rnd((10, 48), 4)
    with pytest.raises(DsmzError):                           # the output over the input
        Gr.grouped_matmul(buf[:, :16], w, o, out=buf[:, 8:32])
    for a in [(x, dy[:9], o), (x.float(), dy, o), (x, dy.float(), o), (x, dy, o.long()), (x, dy, o[:1])]:
        with pytest.raises(ValueError):
            Gr.grouped_weight_grad(*a)
    for kw in (dict(accumulate=True), dict(out=torch.zeros(2, 16, 23, device=DEV)),
               dict(out=torch.zeros(2, 16, 24, device=DEV, dtype=torch.bfloat16)),
               dict(out=torch.zeros(2, 24, 16, device=DEV).transpose(1, 2))):
        with pytest.raises(ValueError):
            Gr.grouped_weight_grad(x, dy, o, **kw)
    with pytest.raises(ValueError):
        Gr.grouped_matmul(rnd((4, 8), 1), rnd((1025, 8, 8), 2), offs([0] * 1026))
