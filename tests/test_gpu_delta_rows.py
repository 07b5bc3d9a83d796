"""Products through an adapter for a part of a batch: rows before and behind the copy's own take
no part in the forward pass, so none of their gradient may reach A, B or x."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U, UB = 2.0 ** -24, 2.0 ** -8          # half a step of fp32 and of bf16


def make_set(rank=16):
    from dsmezo_b200 import AdapterSet, transformer_adapter_shapes
    mods, bases = transformer_adapter_shapes(1, 192, 520, 64, 64)
    aset = AdapterSet(mods, bases, rank, rank, copy_dtype=torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(5)
    for i, m in enumerate(mods):
        aset.A(i).copy_(torch.randn(m.d_out, rank, generator=g, device=DEV) * rank ** -0.5)
        aset.B(i).copy_(torch.randn(rank, m.d_in, generator=g, device=DEV) * m.d_in ** -0.5)
    aset.sync_shadow()
    return aset, g


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("first,end", [(3, 20), (0, 20), (3, 26), (7, 7), (25, 26), (0, 26)])
def test_rows_outside_the_copy(first, end, accumulate):
    aset, g = make_set()
    i = next(k for k, m in enumerate(aset.modules) if m.name == "gate_proj")
    m, rows = aset.modules[i], 26
    x = torch.randn(rows, m.d_in, generator=g, device=DEV).bfloat16()
    dy = torch.randn(rows, m.d_out, generator=g, device=DEV).bfloat16()
    off = torch.tensor([first, end], dtype=torch.int32, device=DEV)
    y, t = aset.delta(i, x, row_offsets=off)
    assert y[:first].eq(0).all() and y[end:].eq(0).all() and t[:first].eq(0).all() and t[end:].eq(0).all()
    grad = aset.grad_arena()
    if accumulate:
        grad.fill_(0.5)
    dx = aset.delta_backward(i, dy, x, t, grad, accumulate=accumulate, row_offsets=off)
    A, B = aset.A(i, aset.shadow).double(), aset.B(i, aset.shadow).double()
    s = slice(first, end)
    xd, dyd, td = x[s].double(), dy[s].double(), t[s].double()
    dt = dyd @ A
    # dt: fp32 sums of d_out products (each addition at most 2 u of what is summed), then half a step of bf16
    edt = UB * dt.abs() + 2 * m.d_out * U * (dyd.abs() @ A.abs()) * (1 + UB)
    base = 0.5 if accumulate else 0.0
    for got, want, err, size in (
            (aset.A(i, grad), dyd.T @ td, 0.0, dyd.abs().T @ td.abs()),
            (aset.B(i, grad), dt.T @ xd, edt.T @ xd.abs(), dt.abs().T @ xd.abs())):
        tol = err + 2 * (rows + 2) * U * (size + base) + 1e-30
        assert bool(((got.double() - base - want).abs() <= tol).all())
    want = torch.zeros(rows, m.d_in, dtype=torch.float64, device=DEV)
    want[s] = dt @ B
    tol = torch.zeros_like(want)
    tol[s] = edt @ B.abs() + UB * (want[s].abs() + edt @ B.abs()) + 2 * aset.rank * U * (dt.abs() @ B.abs())
    assert bool(((dx.double() - want).abs() <= tol).all())           # zero outside the copy's rows
    assert aset.device_error() == 0


def test_without_offsets_every_row_counts():
    aset, g = make_set()
    x = torch.randn(9, aset.modules[0].d_in, generator=g, device=DEV).bfloat16()
    dy = torch.randn(9, aset.modules[0].d_out, generator=g, device=DEV).bfloat16()
    _, t = aset.delta(0, x)
    off = torch.tensor([0, 9], dtype=torch.int32, device=DEV)
    a, b = aset.grad_arena(), aset.grad_arena()
    dxa = aset.delta_backward(0, dy, x, t, a)
    dxb = aset.delta_backward(0, dy, x, t, b, row_offsets=off)
    assert torch.equal(a, b) and torch.equal(dxa, dxb)


def test_a_captured_step_takes_new_offsets():
    """Product, its gradients and AdamW in one graph, replayed with other offsets: as the same steps made
    one by one on a second set."""
    from dsmezo_b200 import AdamW
    sets, opts, grads = [], [], []
    for _ in range(2):
        aset, g = make_set()
        grad = aset.grad_arena()
        sets.append(aset)
        grads.append(grad)
        opts.append(AdamW.for_adapters(aset, grad, lr=1e-2, capturable=True))
    i = next(k for k, m in enumerate(sets[0].modules) if m.name == "gate_proj")
    m = sets[0].modules[i]
    x = torch.randn(26, m.d_in, generator=g, device=DEV).bfloat16()
    dy = torch.randn(26, m.d_out, generator=g, device=DEV).bfloat16()
    off = torch.tensor([0, 26], dtype=torch.int32, device=DEV)

    def step(k, offsets):
        _, t = sets[k].delta(i, x, row_offsets=offsets)
        dx = sets[k].delta_backward(i, dy, x, t, grads[k], row_offsets=offsets)
        opts[k].step()
        return dx

    step(0, off)                                          # outside the graph, as a program warms up
    step(1, off)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx0 = step(0, off)
    for first, end in ((2, 20), (0, 26), (25, 26), (7, 7), (0, 13)):
        off.copy_(torch.tensor([first, end], dtype=torch.int32))
        graph.replay()
        dx1 = step(1, off.clone())
        assert torch.equal(dx0, dx1) and torch.equal(grads[0], grads[1])
        assert torch.equal(sets[0].factors, sets[1].factors) and torch.equal(sets[0].shadow, sets[1].shadow)
    assert sets[0].device_error() == 0 and sets[1].device_error() == 0
