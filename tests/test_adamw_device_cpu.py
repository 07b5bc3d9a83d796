"""Which stream's capture AdamW asks about: that of its parameters' device, whichever device is
current. Devices and streams are stand-ins; no GPU is used."""
import pytest
import torch


class Cuda:
    """Two devices, one of whose current streams is being captured."""

    def __init__(self, current, capturing):
        self.current, self.which = current, capturing

    def device(self, index):
        outer = self

        class Switch:
            def __enter__(self):
                self.before, outer.current = outer.current, index

            def __exit__(self, *a):
                outer.current = self.before
        return Switch()


def stepped(monkeypatch, current, capturing, home, counter=None):
    """AdamW.step on device `home`; the launches it made."""
    from dsmezo_b200 import _lib, optim
    cuda = Cuda(current, capturing)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: cuda.current)
    monkeypatch.setattr(torch.cuda, "device", cuda.device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: cuda.current == cuda.which)
    made = []
    monkeypatch.setattr(_lib, "launch", lambda what, device, *a: made.append((what, device.index)))
    opt = optim.AdamW.__new__(optim.AdamW)
    opt.__dict__.update(_params=(), _states=(), _shadows=(), _grads=(), _pointers=[], _numels=[], _grad_pointers=[], _others=(), _other_pointers=[], _look=0, _table=None,
                        _desc=optim.AdamWDesc(), _counter=counter, device=torch.device("cuda", home), lr=1e-3,
                        betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, step_count=0, state_bits=32)
    opt.step()
    return made


@pytest.mark.parametrize("current", [0, 1])
def test_capture_on_the_parameters_device_is_refused(monkeypatch, current):
    with pytest.raises(RuntimeError, match="captured step"):
        stepped(monkeypatch, current, capturing=1, home=1)


@pytest.mark.parametrize("current", [0, 1])
def test_capture_on_another_device_does_not_matter(monkeypatch, current):
    assert stepped(monkeypatch, current, capturing=0, home=1) == [("adamw_step", 1)]


def test_an_interrupted_step_leaves_the_bound_gradients(monkeypatch):
    """Whatever ends a step(grads) early: the table holds the bound gradients again."""
    from dsmezo_b200 import _lib, optim
    cuda = Cuda(0, None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: cuda.current)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    def interrupted(*a):
        raise KeyboardInterrupt
    monkeypatch.setattr(_lib, "launch", interrupted)
    p, bound, other = torch.zeros(5), torch.ones(5), torch.full((5,), 2.0)
    table = (optim.AdamWTensor * 1)()
    opt = optim.AdamW.__new__(optim.AdamW)
    opt.__dict__.update(_params=(p,), _states=(), _shadows=(), _grads=(bound,), _pointers=[p.data_ptr()], _numels=[5],
                        _grad_pointers=[bound.data_ptr()], _others=(), _other_pointers=[], _look=0, _table=table,
                        _written=[], _starts=[], _desc=optim.AdamWDesc(), _counter=None, device=torch.device("cuda", 0),
                        lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, step_count=0, state_bits=32)
    with pytest.raises(KeyboardInterrupt):
        opt.step([other])
    assert table[0].grad == bound.data_ptr() and opt.grads == (bound,) and opt.step_count == 0
