"""The first-order operators without a GPU: what the C entry points and the Python layer
refuse before any CUDA call."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from dsmezo_b200 import build
    build.build()
    from dsmezo_b200 import _lib
    return _lib


def desc(lib, **kw):
    d = lib.AdamWDesc(param_dtype=0, grad_dtype=0, state_bits=32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
                      weight_decay=0.01, step=1)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def tensors(lib, **kw):
    t = (lib.AdamWTensor * 1)()
    e = t[0]
    e.param = e.grad = e.m = e.v = 4096          # never read: every call here is refused
    e.n = 8
    for k, v in kw.items():
        setattr(e, k, v)
    return t


@pytest.mark.parametrize("bad", [dict(param_dtype=2), dict(grad_dtype=-1), dict(state_bits=16), dict(beta1=1.0),
                                 dict(beta2=-0.1), dict(eps=float("nan")), dict(weight_decay=-1.0),
                                 dict(lr=float("inf")), dict(step=0)])
def test_adamw_refuses_descriptors(lib, bad):
    d = desc(lib, **bad)
    assert lib.lib().dsmz_adamw_step(ctypes.byref(d), tensors(lib), 1, None, 0, None) == 1
    assert b"dsmz_adamw_step" in lib.lib().dsmz_last_error()


@pytest.mark.parametrize("bad", [dict(param=None), dict(grad=None), dict(m=None), dict(v=None), dict(n=-1),
                                 dict(n=1 << 50), dict(param=4097), dict(m=4098), dict(shadow=4097)])
def test_adamw_refuses_tensors(lib, bad):
    d = desc(lib)
    assert lib.lib().dsmz_adamw_step(ctypes.byref(d), tensors(lib, **bad), 1, None, 0, None) == 1
    assert b"tensor 0" in lib.lib().dsmz_last_error()


def test_adamw_refuses_missing_pieces(lib):
    L = lib.lib()
    assert L.dsmz_adamw_step(None, tensors(lib), 1, None, 0, None) == 1
    d = desc(lib)
    assert L.dsmz_adamw_step(ctypes.byref(d), None, 1, None, 0, None) == 1
    assert L.dsmz_adamw_step(ctypes.byref(d), tensors(lib), -1, None, 0, None) == 1
    d8 = desc(lib, state_bits=8)
    assert L.dsmz_adamw_step(ctypes.byref(d8), tensors(lib), 1, None, 0, None) == 1         # no scales
    dc = desc(lib, step_counter=4096)
    assert L.dsmz_adamw_step(ctypes.byref(dc), tensors(lib), 1, None, 0, None) == 2         # no workspace
    db = desc(lib, param_dtype=1)
    assert L.dsmz_adamw_step(ctypes.byref(db), tensors(lib, shadow=4096), 1, None, 0, None) == 1
    assert L.dsmz_adamw_state_values(tensors(lib), 1, None) == 1
    # nothing to do is no error, and makes no CUDA call
    assert L.dsmz_adamw_step(ctypes.byref(d), tensors(lib, n=0), 1, None, 0, None) == 0
    assert L.dsmz_adamw_step(ctypes.byref(d), None, 0, None, 0, None) == 0


def test_adamw_takes_no_cpu_tensors(lib):
    from dsmezo_b200 import AdamW
    with pytest.raises(ValueError, match="CUDA"):
        AdamW([torch.zeros(4)])


def loss_grad(lib, **kw):
    a = dict(kind=0, logits=4096, V=8, ld=8, targets=4096, ntok=4, starts=(0, 4), adv=(1.0,), nseq=1, scale=1.0,
             loss=4096, grad=8192, ld_grad=8, ws=4096, ws_bytes=64)
    a.update(kw)
    starts = None if a["starts"] is None else (ctypes.c_int64 * len(a["starts"]))(*a["starts"])
    adv = None if a["adv"] is None else (ctypes.c_double * len(a["adv"]))(*a["adv"])
    return lib.lib().dsmz_contrastive_loss_grad(a["kind"], a["logits"], a["V"], a["ld"], a["targets"], a["ntok"], starts,
                                                adv, a["nseq"], a["scale"], a["loss"], a["grad"], a["ld_grad"], a["ws"],
                                                a["ws_bytes"], None)


@pytest.mark.parametrize("bad", [dict(kind=2), dict(logits=None), dict(targets=None), dict(loss=None), dict(grad=None),
                                 dict(starts=None), dict(adv=None), dict(V=0), dict(ld=7), dict(ld_grad=7),
                                 dict(ntok=0, starts=(0, 0)), dict(starts=(1, 4)), dict(starts=(0, 3)),
                                 dict(nseq=0), dict(nseq=129, starts=(0,) * 129 + (4,), adv=(1.0,) * 129),
                                 dict(nseq=2, starts=(0, 4, 4), adv=(1.0, 1.0)), dict(scale=float("inf")),
                                 dict(logits=4098), dict(grad=4100), dict(V=1 << 31, ld=1 << 31, ld_grad=1 << 31)])
def test_loss_grad_refuses(lib, bad):
    assert loss_grad(lib, **bad) == 1
    assert b"dsmz_contrastive_loss_grad" in lib.lib().dsmz_last_error()


def test_loss_grad_workspace(lib):
    assert lib.lib().dsmz_contrastive_loss_grad_workspace_bytes(4) == 32
    assert loss_grad(lib, ws_bytes=31) == 2 and loss_grad(lib, ws=4097) == 2 and loss_grad(lib, ws=None) == 1


def test_loss_grad_takes_no_cpu_tensors(lib):
    from dsmezo_b200 import scoring
    with pytest.raises(ValueError, match="CUDA"):
        scoring.contrastive_loss_grad(torch.zeros(2, 4), [2], [1.0], torch.zeros(2, dtype=torch.int32))


def product(lib, **kw):
    a = dict(x=1 << 20, M=10, K=16, ld_x=16, w=1 << 21, G=2, N=24, gs=384, w_ld=24, nc=1, offsets=4096, dt=1, out=1 << 22,
             ld=24, alpha=1.0, flags=0)
    a.update(kw)
    return lib.lib().dsmz_grouped_matmul(a["x"], a["M"], a["K"], a["ld_x"], a["w"], a["G"], a["N"], a["gs"], a["w_ld"], a["nc"],
                                         a["offsets"], a["dt"], a["out"], a["ld"], a["alpha"], a["flags"], None)


@pytest.mark.parametrize("bad,code", [(dict(M=-1), 1), (dict(K=0), 1), (dict(N=0), 1), (dict(G=0), 1), (dict(G=1025), 4),
                                      (dict(M=1 << 31), 4), (dict(dt=2), 1), (dict(flags=4), 1), (dict(x=None), 1),
                                      (dict(w=None), 1), (dict(out=None), 1), (dict(offsets=None), 1), (dict(ld_x=8), 1),
                                      (dict(w_ld=16), 1), (dict(ld=23), 1), (dict(gs=0), 1), (dict(gs=-8), 1),
                                      (dict(x=(1 << 20) + 8), 1), (dict(w=(1 << 21) + 2), 1), (dict(ld_x=20), 1),
                                      (dict(gs=388), 1), (dict(out=(1 << 22) + 1), 1), (dict(offsets=4098), 1),
                                      (dict(alpha=float("nan")), 1), (dict(out=(1 << 20) + 16), 1),
                                      (dict(out=(1 << 21) + 2), 1)])
def test_grouped_matmul_refuses(lib, bad, code):
    assert product(lib, **bad) == code
    assert b"dsmz_grouped_matmul" in lib.lib().dsmz_last_error()


def weight_grad(lib, **kw):
    a = dict(x=1 << 20, M=10, K=16, ld_x=16, dy=1 << 21, N=24, ld_dy=24, G=2, offsets=4096, out=1 << 22, alpha=1.0, flags=0)
    a.update(kw)
    return lib.lib().dsmz_grouped_weight_grad(a["x"], a["M"], a["K"], a["ld_x"], a["dy"], a["N"], a["ld_dy"], a["G"],
                                              a["offsets"], a["out"], a["alpha"], a["flags"], None)


@pytest.mark.parametrize("bad,code", [(dict(M=-1), 1), (dict(K=0), 1), (dict(N=0), 1), (dict(G=0), 1), (dict(G=1025), 4),
                                      (dict(flags=2), 1), (dict(x=None), 1), (dict(dy=None), 1), (dict(out=None), 1),
                                      (dict(offsets=None), 1), (dict(ld_x=8), 1), (dict(ld_dy=16), 1), (dict(ld_dy=28), 1),
                                      (dict(x=(1 << 20) + 8), 1), (dict(out=(1 << 22) + 2), 1), (dict(offsets=4097), 1),
                                      (dict(alpha=float("inf")), 1), (dict(out=(1 << 20) + 16), 1)])
def test_grouped_weight_grad_refuses(lib, bad, code):
    assert weight_grad(lib, **bad) == code
    assert b"dsmz_grouped_weight_grad" in lib.lib().dsmz_last_error()


def test_grouped_products_take_no_cpu_tensors(lib):
    from dsmezo_b200 import grouped
    x, w, o = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(1, 8, 8, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        grouped.grouped_matmul(x, w, o)
    with pytest.raises(ValueError, match="CUDA"):
        grouped.grouped_weight_grad(x, x, o)
