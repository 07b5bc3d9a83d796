"""Grouped products whose barrier waits run out of time: with a limit of 0 nothing is loaded, the
waits give up after about a millisecond and the kernels end by themselves. What was not produced
must be NaN, the device's word must tell, and the next calls must be as good as ever."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def grouped():
    from dsmezo_b200 import grouped as G
    assert G.device_error(DEV) == 0
    yield G
    G.set_wait_limit(1.0)
    torch.cuda.synchronize()
    G.device_error(DEV)


def offsets(M, G, lead=0):
    edges = [lead + (M - lead) * i // G for i in range(G + 1)]
    return torch.tensor(edges, dtype=torch.int32, device=DEV)


def normal(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=g)


def check(G, call, start, made=None):
    """call(out) writes out; `start` is what it held before; made: the elements that call is for."""
    G.set_wait_limit(1.0)
    want = call(start.clone())
    torch.cuda.synchronize()
    assert not torch.isnan(want).any()
    G.set_wait_limit(0.0)
    got = call(start.clone())
    G.set_wait_limit(1.0)
    again = call(start.clone())                                   # before anything has read the word
    made = torch.ones_like(got, dtype=torch.bool) if made is None else made
    assert torch.isnan(got[made]).all() and torch.equal(got[~made], want[~made]) and torch.equal(again, want)
    assert G.device_error(DEV) == 1 and G.device_error(DEV) == 0


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,G,K,N,major", [
    (300, 2, 3584, 64, "k"),            # a cluster shares a tile's contraction
    (300, 2, 3584, 100, "n"),
    (4096, 2, 64, 18944, "k"),          # one CTA a tile, columns of 256
    (4001, 32, 64, 18944, "n"),         # sixteen epilogue warps
    (20000, 2, 200, 100, "k"),          # one CTA a tile, narrow
])
def test_products(grouped, M, G, K, N, major, dt):
    x, off = normal(M, K), offsets(M, G)
    w = normal(G, N, K, seed=1).transpose(1, 2) if major == "k" else normal(G, K, N, seed=1)
    check(grouped, lambda out: grouped.grouped_matmul(x, w, off, out=out), start=torch.zeros(M, N, dtype=dt, device=DEV))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_pairs_of_ctas(grouped, dt):
    M, G, K, N = 4096, 2, 1024, 4608
    x, off, w = normal(M, K), offsets(M, G), normal(G, N, K, seed=1).transpose(1, 2)
    check(grouped, lambda out: grouped.grouped_matmul(x, w, off, out=out), start=torch.zeros(M, N, dtype=dt, device=DEV))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K,N", [(64, 18944), (2000, 40)])
def test_accumulation_and_rows_outside(grouped, K, N, dt):
    M, G = 1000, 3
    x, off, w = normal(M, K), offsets(900, G, lead=17), normal(G, K, N, seed=1)
    wide = torch.randn(M, N + 3, device=DEV).to(dt)

    def call(buf):
        grouped.grouped_matmul(x, w, off, out=buf[:, :N], accumulate=True)
        return buf
    made = torch.zeros_like(wide, dtype=torch.bool)
    made[17:900, :N] = True                                       # rows of no group and the columns beside stay
    check(grouped, call, start=wide, made=made)


@pytest.mark.parametrize("K,N,M,G", [(64, 18944, 4096, 2), (18944, 64, 4096, 2), (300, 40, 997, 8), (40, 300, 997, 8), (1024, 2048, 600, 3)])
def test_weight_gradients(grouped, K, N, M, G):
    x, dy, off = normal(M, K), normal(M, N, seed=1), offsets(M, G)
    check(grouped, lambda out: grouped.grouped_weight_grad(x, dy, off, out=out),
          start=torch.zeros(G, K, N, device=DEV))


def test_an_adapter_set_reports_it(grouped):
    from dsmezo_b200 import AdapterSet, transformer_adapter_shapes
    mods, bases = transformer_adapter_shapes(1, 3584, 18944, 512, 512)
    aset = AdapterSet(mods, bases, 64, 64, copy_dtype=torch.bfloat16)
    aset.factors.normal_()
    aset.sync_shadow()
    i = next(k for k, m in enumerate(mods) if m.name == "gate_proj")
    x = normal(4096, mods[i].d_in)
    want, _ = aset.delta(i, x)
    assert aset.device_error() == 0
    grouped.set_wait_limit(0.0)
    y, _ = aset.delta(i, x)
    assert torch.isnan(y).all()
    assert aset.device_error() != 0 and aset.device_error() == 0
    grouped.set_wait_limit(1.0)
    assert torch.equal(aset.delta(i, x)[0], want) and aset.device_error() == 0
