"""bf16 products over contractions so long that an accumulator which rounds towards zero would
lose more than half a step of the output.

All products are positive, so every truncation has one sign. n additions to a growing sum, each
off by at most a of it, make n / 2 a of the result: 2^-23 for the 32 additions of 16 products
that one accumulator takes (2^-19), 2^-24 for the fp32 additions of at most 2^14 accumulators a
CTA (2^-11) and of 8 CTAs (2^-22). The result is rounded to bf16 once (half a step, 2^-8)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -19 + 2.0 ** -22


def positive(shape, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.empty(shape, dtype=torch.bfloat16, device=DEV).uniform_(1.0, 2.0, generator=g)


def dot(a, b):
    """Sum of the products in fp64."""
    return sum(float(p.double() @ q.double()) for p, q in zip(a.split(1 << 22), b.split(1 << 22)))


def test_contraction_split_over_a_cluster():
    from dsmezo_b200 import grouped
    K = 1 << 26
    x, w = positive((2, K), 1), positive((1, 2, K), 2)
    off = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    y = grouped.grouped_matmul(x, w.transpose(1, 2), off)
    for i in range(2):
        for j in range(2):
            want = dot(x[i], w[0, j])
            assert abs(float(y[i, j]) - want) <= TOL * want


@pytest.mark.parametrize("n", [1, 16])
def test_contraction_in_one_cta(n):
    from dsmezo_b200 import grouped
    G, K = 80, 1 << 23                  # more tiles than clusters: nothing is split
    x = positive((G, K), 3)
    buf = positive((K * n + 8 * G,), 4)
    w = buf.as_strided((G, K, n), (8, 1, K))           # group g's matrix starts 8 elements after that of g - 1
    off = torch.arange(G + 1, dtype=torch.int32, device=DEV)
    y = grouped.grouped_matmul(x, w, off)
    assert y.dtype == torch.bfloat16
    for i in (0, 1, 40, 79):
        for j in (0, n - 1):
            want = dot(x[i], w[i, :, j])
            assert abs(float(y[i, j]) - want) <= TOL * want


@pytest.mark.parametrize("M,G,K,N,pad", [
    (4096, 1, 33000, 4608, 0),          # pairs of CTAs
    (2600, 20, 32776, 1000, 0),         # 256 columns
    (90, 80, 33001, 70, 3),             # 128 columns, odd pitches
    (90, 80, 40000, 50, 0),             # 64 columns
])
def test_rounded_once_from_the_fp32_sums(M, G, K, N, pad):
    """Past the limit both output types sum in the same way: bf16 is the fp32 result rounded."""
    from dsmezo_b200 import grouped
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.empty(M, K, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    w = torch.empty(G, K, N, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    off = torch.tensor([M * i // G for i in range(G + 1)], dtype=torch.int32, device=DEV)
    wide = torch.zeros(M, N + pad, dtype=torch.bfloat16, device=DEV)
    y = grouped.grouped_matmul(x, w, off, out=wide[:, :N], alpha=0.7)
    z = grouped.grouped_matmul(x, w, off, out_dtype=torch.float32, alpha=0.7)
    assert torch.equal(y, z.bfloat16())
    row = M // 2
    k = row * G // M
    want = 0.7 * (x[row].double() @ w[k].double())
    size = x[row].double().abs() @ w[k].double().abs()
    # 32 additions an accumulator (2^-22 each at most of what it holds), then one of fp32 for each 512 products
    assert bool(((z[row].double() - want).abs() <= size * (32 * 2.0 ** -22 + (K / 512 + 2) * 2.0 ** -24)).all())
