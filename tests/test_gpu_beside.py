"""Outputs that lie beside their operands in one wider buffer, sharing no element with them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def wide(rows, cols, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(rows, cols, generator=g, device=DEV).bfloat16()


@pytest.mark.parametrize("rows", [1, 2, 150])
@pytest.mark.parametrize("at", [0, 72, 96])
def test_product_beside_its_input(rows, at):
    from dsmezo_b200 import grouped
    K, N, pitch = 64, 40, 136
    buf = wide(rows, pitch, 3)
    lo = 0 if at else 72                                 # x before or behind the output
    x, out = buf[:, lo:lo + K], buf[:, at:at + N]
    w = wide(K, N, 4).unsqueeze(0)
    off = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    want = grouped.grouped_matmul(x.clone(), w, off)
    before = buf.clone()
    grouped.grouped_matmul(x, w, off, out=out)
    assert torch.equal(out, want)
    before[:, at:at + N] = want
    assert torch.equal(buf, before)                      # nothing else was written


@pytest.mark.parametrize("at", [1, 24, 63, 104])
def test_shared_elements_are_refused(at):
    from dsmezo_b200 import DsmzError, grouped
    buf = wide(9, 136, 5)
    flat = buf.view(-1)
    x = buf[:, :64]
    # from column 104 on 40 columns reach 8 into the next row's x
    out = flat.as_strided((8, 40), (136, 1), at)
    off = torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    with pytest.raises(DsmzError):
        grouped.grouped_matmul(x[:8], wide(64, 40, 6).unsqueeze(0), off, out=out)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 3, 20])
def test_loss_gradient_beside_the_logits(rows, dt):
    from dsmezo_b200 import DsmzError, scoring
    V = 1000
    buf = torch.randn(rows, 2 * V + 3, device=DEV).to(dt)
    x, out = buf[:, :V], buf[:, V:2 * V]
    t = torch.arange(rows, device=DEV, dtype=torch.int32)
    before = buf.clone()
    loss, want = scoring.contrastive_loss_grad(x, [rows], [0.5], t)
    got, grad = scoring.contrastive_loss_grad(x, [rows], [0.5], t, out=out)
    # The sums of one x are the same wherever the gradient goes. An element is w (e r) or e (w r) as its row's
    # alignment has it: two roundings each (4 u), then one to the type each (bf16: eps in all).
    tol = 4 * 2.0 ** -24 + (torch.finfo(dt).eps if dt == torch.bfloat16 else 0.0)
    assert torch.equal(got, loss) and bool(((out.double() - want.double()).abs() <= tol * want.double().abs()).all())
    assert torch.equal(x, before[:, :V]) and torch.equal(buf[:, 2 * V:], before[:, 2 * V:])
    if rows > 1:
        with pytest.raises(DsmzError):
            scoring.contrastive_loss_grad(x, [rows], [0.5], t, out=buf[:, 1:V + 1])
