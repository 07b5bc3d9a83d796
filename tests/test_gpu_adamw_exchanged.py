"""AdamW refuses a step once the memory under a tensor that it bound has been exchanged: the C table
holds addresses, and would read or write the old ones."""
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


@pytest.mark.parametrize("bits", [32, 8])
def test_exchanged_memory_is_refused(bits):
    opt, params, grads = make(bits)
    opt.step()
    s = opt.states[1]
    bound = [params[1], grads[0], grads[1], opt.shadows[0], s.m, s.v] + ([s.m_scale, s.v_scale] if bits == 8 else [])
    before = [p.clone() for p in params]
    for t in bound:
        keep = t.data
        t.data = keep.clone()
        with pytest.raises(RuntimeError, match="memory"):
            opt.step()
        t.data = keep
    assert opt.step_count == 1 and all(torch.equal(p, q) for p, q in zip(params, before))
    opt.step()
    assert opt.step_count == 2


def test_exchanged_gradients_matter_only_where_they_are_used():
    opt, params, grads = make(32)
    grads[0].data = grads[0].clone()
    opt.step([torch.ones_like(p) for p in params])       # brings its own
    assert opt.step_count == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_exchanged_states_of_many_parameters(bits):
    """Found when its turn comes, sixteen tensors a step; until then the old memory is stepped: it stays
    allocated."""
    from dsmezo_b200 import AdamW
    params = [torch.randn(300, device=DEV) for _ in range(10)]
    grads = [torch.randn(300, device=DEV) for _ in range(10)]
    for k in range(10):
        opt = AdamW(params, lr=1e-2, grads=grads, state_bits=bits)
        opt.step()
        m = opt.states[k].m
        at, m.data = m.data_ptr(), torch.zeros_like(m)
        fresh = [torch.full((300,), 3, dtype=m.dtype, device=DEV) for _ in range(200)]
        assert all(t.data_ptr() != at for t in fresh)        # nobody else gets it
        steps = 0
        with pytest.raises(RuntimeError, match="state or shadow"):
            for _ in range(3):
                opt.step()
                steps += 1
        assert steps <= 2 and opt.step_count == 1 + steps
        torch.cuda.synchronize()
        assert all(t.eq(3).all() for t in fresh) and m.eq(0).all()
