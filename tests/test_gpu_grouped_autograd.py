"""The grouped products record no graph: operands that ask for one are refused, not dropped."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def operands():
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(6, 64, generator=g, device=DEV).bfloat16()
    w = torch.randn(2, 64, 24, generator=g, device=DEV).bfloat16()
    return x, w, torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("which", ["x", "w", "out"])
def test_operands_that_require_grad(which):
    from dsmezo_b200 import grouped
    x, w, off = operands()
    want = grouped.grouped_matmul(x, w, off)
    out = torch.zeros(6, 24, dtype=torch.bfloat16, device=DEV)
    {"x": x, "w": w, "out": out}[which].requires_grad_()
    with pytest.raises(RuntimeError, match="no_grad"):
        grouped.grouped_matmul(x, w, off, out=out)
    with torch.no_grad():                               # asked for explicitly
        assert torch.equal(grouped.grouped_matmul(x, w, off, out=out), want)
    assert torch.equal(grouped.grouped_matmul(x.detach(), w.detach(), off, out=out.detach()), want)


def test_a_function_that_records_it():
    """The way into autograd: forward and backward of a torch.autograd.Function, whose gradients
    are those of the formula."""
    from dsmezo_b200 import grouped

    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, off):
            ctx.save_for_backward(x, w, off)
            return grouped.grouped_matmul(x, w, off)

        @staticmethod
        def backward(ctx, dy):
            x, w, off = ctx.saved_tensors
            return (grouped.grouped_matmul(dy, w.transpose(1, 2), off),
                    grouped.grouped_weight_grad(x, dy, off).to(w.dtype), None)

    x, w, off = operands()
    x.requires_grad_()
    w.requires_grad_()
    dy = torch.randn(6, 24, device=DEV).bfloat16()
    Product.apply(x, w, off).backward(dy)
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    torch.cat([xd[:2] @ wd[0], xd[2:] @ wd[1]]).backward(dy.double())
    # half a step of bf16, and fp32 sums of at most 24 products
    for got, ref in ((x.grad, xd.grad), (w.grad, wd.grad)):
        tol = 2.0 ** -8 * ref.abs() + 24 * 2.0 ** -23 * 64.0
        assert bool(((got.double() - ref).abs() <= tol).all())


def test_delta_refuses_too():
    from dsmezo_b200 import AdapterSet, transformer_adapter_shapes
    mods, bases = transformer_adapter_shapes(1, 192, 520, 64, 64)
    aset = AdapterSet(mods, bases, 16, 16, copy_dtype=torch.bfloat16)
    x = torch.randn(4, mods[0].d_in, device=DEV).bfloat16().requires_grad_()
    with pytest.raises(RuntimeError, match="no_grad"):
        aset.delta(0, x)
    with torch.no_grad():
        y, t = aset.delta(0, x)
    dy = torch.ones_like(y)
    assert aset.delta_backward(0, dy, x, t, aset.grad_arena()) is not None     # the gradients themselves need no graph
