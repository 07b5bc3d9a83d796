"""A refused AdamW step changes nothing: neither the tensors nor the gradients that are bound."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(bits, seed=0, capturable=False):
    from dsmezo_b200 import AdamW
    g = torch.Generator(device=DEV).manual_seed(seed)
    params = [torch.randn(n, generator=g, device=DEV) for n in (700, 33)]
    grads = [torch.randn(n, generator=g, device=DEV) for n in (700, 33)]
    shadows = [p.bfloat16() for p in params]
    opt = AdamW(params, lr=1e-2, grads=grads, shadows=shadows, state_bits=bits, capturable=capturable)
    return opt, params, grads


def refusals(opt, other):
    """Calls of step(grads) that are refused, each for another reason."""
    from dsmezo_b200 import DsmzError
    with pytest.raises(ValueError):
        opt.step(other, lr=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError):
        opt.step(other, grad_scale=torch.zeros(1, device=DEV, dtype=torch.float64))
    opt.weight_decay = -1.0                              # refused by the library itself
    with pytest.raises(DsmzError):
        opt.step(other)
    opt.weight_decay = 1e-2
    keep = opt.params[0].data
    opt.params[0].data = keep.clone()
    with pytest.raises(RuntimeError):
        opt.step(other)
    opt.params[0].data = keep


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_step_keeps_the_bound_gradients(bits):
    a, pa, _ = make(bits)
    b, pb, _ = make(bits)
    other = [torch.full_like(p, 7.0, dtype=torch.bfloat16) for p in pa]
    refusals(a, other)
    assert a.step_count == 0 and all(torch.equal(x, y) for x, y in zip(pa, pb))
    for _ in range(2):
        a.step()
        b.step()
        refusals(a, other)
    assert a.step_count == 2
    for x, y in zip(pa, pb):
        assert torch.equal(x, y)
    for x, y in zip(a.states, b.states):
        assert torch.equal(x.m, y.m) and torch.equal(x.v, y.v)


def test_a_captured_step_with_a_host_count_is_refused_and_changes_nothing():
    a, pa, _ = make(32)
    b, pb, _ = make(32)
    other = [torch.full_like(p, 7.0) for p in pa]
    a.step()
    b.step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph, keep = torch.cuda.CUDAGraph(), torch.zeros(1, device=DEV)
    with torch.cuda.stream(s):
        graph.capture_begin()
        keep.add_(1.0)
        with pytest.raises(RuntimeError):
            a.step(other)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(s)
    a.step()
    b.step()
    assert all(torch.equal(x, y) for x, y in zip(pa, pb))
