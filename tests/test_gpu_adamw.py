"""AdamW over many tensors (dsmezo_b200.optim) against the formula in fp64.

Tolerances count roundings, u = 2^-24 (fp32, half a step):
* m: each of its two terms carries a coefficient, a product and the sum (and the gradient's
  scale): 4 u of |b1 m| + |(1 - b1) g|;
* v: at most a coefficient, two products, the scale twice and the sum: 6 u of v;
* the update: half of v's, then root, coefficient, product, eps, sum, quotient, coefficient,
  product: 12 u of it, and m's error through the quotient; p itself: coefficient, product,
  difference: 3 u; a bf16 parameter or shadow adds half a bf16 step, 2^-8, at the end.
8-bit codes must equal those of fp64 arithmetic. With them the update takes the approximate
root and reciprocal (2 u each and a product in place of 1 and 1: 15 u in all; 16 are allowed);
the scales are those of fp64 arithmetic, rounded once, or to the next value where two fp64
evaluations straddle a rounding border (2 u)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U, UB = 2.0 ** -24, 2.0 ** -8
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.99, 1e-8, 0.1


@pytest.fixture(scope="module")
def O():
    from dsmezo_b200 import optim
    return optim


def blocks(x, fill=0.0):
    n = x.numel()
    return torch.nn.functional.pad(x.double().cpu(), (0, -n % 256), value=fill).view(-1, 256)


def decode(s, n):
    """fp64 (m, v) of a state."""
    if s.bits == 32:
        return s.m.double().cpu(), s.v.double().cpu()
    q, r = blocks(s.m), blocks(s.v)
    m = q.sign() * q * q * s.m_scale.double().cpu()[:, None]
    root = r * r * s.v_scale.double().cpu()[:, None]
    return m.flatten()[:n], (root * root).flatten()[:n]


def encode(m, v):
    """fp64 codes and scales: the highest code whose lower border (q - 1/2)^2 lies under the value."""
    out = []
    for x, top_code in ((m.abs(), 127), (v.sqrt(), 255)):
        b = blocks(x)
        top = b.amax(1, keepdim=True)
        q = torch.ceil(top_code * torch.sqrt(b / top) - 0.5).nan_to_num(0.0).clamp(0, top_code)
        out += [q, top / top_code ** 2]
    qm = torch.copysign(out[0], blocks(m))
    qv = torch.where(blocks(v) > 0, out[2].clamp(min=1), out[2])
    n = m.numel()
    return qm.flatten()[:n], out[1].flatten(), qv.flatten()[:n], out[3].flatten()


def reference(p, g, m, v, t, lr=LR, scale=1.0, roundings=12):
    g = g.double().cpu() * scale
    p = p.double().cpu()
    m1 = B1 * m + (1 - B1) * g
    v1 = B2 * v + (1 - B2) * g * g
    den = (v1 / (1 - B2 ** t)).sqrt() + EPS
    upd = lr / (1 - B1 ** t) * m1 / den
    em = 4 * U * (B1 * m.abs() + (1 - B1) * g.abs())
    p1 = p * (1 - lr * WD) - upd
    ep = 3 * U * p.abs() + roundings * U * upd.abs() + lr / (1 - B1 ** t) * em / den + 1e-44
    return p1, m1, v1, ep, em


def make(n, pdt, gdt, bits, seed, O, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rnd(dt, scale):
        return (torch.randn(n + offset, generator=g, device=DEV) * scale).to(dt)[offset:]
    p, grad = rnd(pdt, 1.0), rnd(gdt, 0.1)
    s = O.AdamWState.zeros(p, bits)
    if bits == 32:
        s.m.copy_(rnd(torch.float32, 0.05))
        s.v.copy_(rnd(torch.float32, 0.1) ** 2)
    else:
        s.m.copy_(torch.randint(-127, 128, (n,), generator=g, device=DEV))
        s.v.copy_(torch.randint(0, 256, (n,), generator=g, device=DEV))
        s.m_scale.copy_(torch.rand(s.m_scale.shape, generator=g, device=DEV) * 1e-5)
        s.v_scale.copy_(torch.rand(s.v_scale.shape, generator=g, device=DEV) * 1e-6)
    return p, grad, s


def check_step(p0, g, m, v, t, p, s, shadow=None, lr=LR, scale=1.0):
    p1, m1, v1, ep, em = reference(p0, g, m, v, t, lr, scale, 12 if s.bits == 32 else 16)
    got = p.double().cpu()
    extra = UB * p1.abs() if p.dtype == torch.bfloat16 else 0.0
    assert bool(((got - p1).abs() <= ep + extra).all())
    if shadow is not None:
        assert torch.equal(shadow, p.to(torch.bfloat16))
    if s.bits == 32:
        assert bool(((s.m.double().cpu() - m1).abs() <= em).all())
        assert bool(((s.v.double().cpu() - v1).abs() <= 6 * U * v1).all())
    else:
        qm, sm, qv, sv = encode(m1, v1)
        assert torch.equal(s.m.double().cpu(), qm) and torch.equal(s.v.double().cpu(), qv)
        assert bool(((s.m_scale.double().cpu() - sm).abs() <= 2 * U * sm).all())
        assert bool(((s.v_scale.double().cpu() - sv).abs() <= 2 * U * sv).all())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pdt,gdt", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                     (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_three_steps_of_odd_sizes(O, bits, pdt, gdt):
    sizes = [1, 3, 255, 256, 257, 0, 2047, 2048, 2049, 6007]
    made = [make(n, pdt, gdt, bits, 7 + n, O, offset=i % 2) for i, n in enumerate(sizes)]
    shadows = [torch.empty(n, dtype=torch.bfloat16, device=DEV) if pdt == torch.float32 else None for n in sizes]
    opt = O.AdamW([p for p, _, _ in made], LR, (B1, B2), EPS, WD, states=[s for _, _, s in made], shadows=shadows,
                  step=4)
    for t in (5, 6, 7):
        before = [(p.clone(), *decode(s, p.numel())) for p, _, s in made]
        opt.step([g for _, g, _ in made])
        for (p, g, s), (p0, m, v), sh in zip(made, before, shadows):
            check_step(p0, g, m, v, t, p, s, sh)
    assert opt.step_count == 7


@pytest.mark.parametrize("bits", [32, 8])
def test_from_nothing_and_many_tensors(O, bits):
    # zeroed states, more tensors than one launch takes, a gradient scale and a device lr
    sizes = [1 + (37 * i) % 700 for i in range(300)]
    made = [make(n, torch.float32, torch.float32, bits, i, O) for i, n in enumerate(sizes)]
    scale = torch.tensor([0.25], device=DEV)
    lr = torch.tensor([2.0 ** -9], device=DEV)
    opt = O.AdamW([p for p, _, _ in made], 1.0, (B1, B2), EPS, WD, grads=[g for _, g, _ in made], state_bits=bits)
    before = [p.clone() for p, _, _ in made]
    opt.step(lr=lr, grad_scale=scale)
    for (p, g, _), p0, s in zip(made, before, opt.states):
        z = torch.zeros(p.numel(), dtype=torch.float64)
        check_step(p0, g, z, z, 1, p, s, lr=2.0 ** -9, scale=0.25)


def test_codes_on_a_border_take_the_lower(O):
    # m_old of code Q/2 beside Q and gradients 4 : 1 put the new mean exactly a quarter of the
    # block's largest: the border between codes 63 and 64
    n = 256
    p = torch.zeros(n, device=DEV)
    s = O.AdamWState.zeros(p, 8)
    s.m[0], s.m[1] = 126, 63
    s.v[0], s.v[1] = 254, 127
    s.m_scale.fill_(1.2345e-7)
    s.v_scale.fill_(3.21e-8)
    g = torch.zeros(n, device=DEV)
    g[0], g[1] = 4 * 0.0123, 0.0123
    O.AdamW([p], states=[s], grads=[g], step=3).step()
    assert s.m[:3].tolist() == [127, 63, 0] and s.v[:3].tolist() == [255, 127, 0]


def test_small_second_moments_keep_a_code(O):
    p = torch.zeros(512, device=DEV)
    g = torch.full((512,), 1e-9, device=DEV)
    g[0] = 1.0
    opt = O.AdamW([p], grads=[g], state_bits=8)
    opt.step()
    assert opt.states[0].v[1:256].eq(1).all() and opt.states[0].v[256:].eq(255).all()
    assert opt.states[0].m[1:256].eq(0).all() and opt.states[0].m[256:].eq(127).all()


def test_nothing_but_nan_spreads_over_its_block_alone(O):
    n = 700
    p, g, s = make(n, torch.float32, torch.float32, 8, 3, O)
    g[300] = float("nan")
    g[650] = float("inf")
    opt = O.AdamW([p], states=[s], grads=[g])
    opt.step()
    m, v = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    opt.state_values([m], [v])
    assert torch.isfinite(m[:256]).all() and torch.isfinite(v[:256]).all()
    assert torch.isnan(m[256:]).all() and torch.isnan(v[256:]).all()
    finite = torch.isfinite(p)
    assert int((~finite).sum()) == 2 and not finite[300] and not finite[650]


def test_8_bit_states_over_the_whole_range(O):
    # blocks of tiny, huge, cancelling and mixed gradients: the codes stay those of fp64
    n = 256 * 12
    p, g, s = make(n, torch.float32, torch.float32, 8, 5, O)
    rows = g.view(12, 256)
    for i, f in enumerate((1e-30, 1e-25, 1e-20, 1e-12, 1.0, 1e8, 1e17)):
        rows[i] *= f
        s.m_scale[i] *= f
        s.v_scale[i] *= f
    rows[7].zero_()                                              # decay alone
    rows[8] = -B1 / (1 - B1) * decode(s, n)[0].view(12, 256)[8].float().to(DEV)      # the new mean cancels
    rows[9, ::2] *= 1e-20
    rows[10].zero_(), s.m.view(12, 256)[10].zero_(), s.v.view(12, 256)[10].zero_()   # all zero
    rows[11].zero_(), s.m_scale[11:].zero_(), s.v_scale[11:].zero_()
    m, v = decode(s, n)
    p0 = p.clone()
    O.AdamW([p], LR, (B1, B2), EPS, WD, states=[s], grads=[g], step=4).step()
    _, m1, v1, _, em = reference(p0, g, m, v, 5)
    qm, sm, qv, sv = encode(m1, v1)
    keep = torch.ones(12, 256, dtype=torch.bool)
    keep[8] = False      # cancelled means are rounding noise of fp64 itself: no code of theirs is defined
    keep = keep.flatten()
    assert torch.equal(s.m.double().cpu()[keep], qm[keep]) and torch.equal(s.v.double().cpu(), qv)
    off = torch.ones(12, dtype=torch.bool)
    off[8] = False
    assert bool(((s.m_scale.double().cpu() - sm).abs() <= 2 * U * sm + 1e-45)[off].all())
    assert bool(((s.v_scale.double().cpu() - sv).abs() <= 2 * U * sv + 1e-45).all())


@pytest.mark.parametrize("n", [256, 1000])
def test_blocks_of_equal_values(O, n):
    # every element can be the largest: constant and alternating gradients over several steps
    for g in (torch.full((n,), 0.37, device=DEV), 0.01 * (1.0 - 2.0 * (torch.arange(n, device=DEV) % 2))):
        p = torch.randn(n, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)
        opt = O.AdamW([p], LR, (B1, B2), EPS, WD, grads=[g], state_bits=8)
        for t in range(1, 5):
            p0, (m, v) = p.clone(), decode(opt.states[0], n)
            opt.step()
            check_step(p0, g, m, v, t, p, opt.states[0])


def test_replaced_parameter_is_refused(O):
    p, g = torch.zeros(8, device=DEV), torch.ones(8, device=DEV)
    opt = O.AdamW([p], grads=[g])
    opt.step()
    p.data = torch.zeros(8, device=DEV)
    with pytest.raises(RuntimeError, match="replaced"):
        opt.step()


def test_state_values(O):
    for n in (1, 256, 1000):
        p, g, s = make(n, torch.float32, torch.float32, 8, n, O)
        m, v = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
        O.AdamW([p], states=[s], grads=[g]).state_values([m], [v])
        mw, vw = decode(s, n)
        assert bool(((m.double().cpu() - mw).abs() <= U * mw.abs()).all())
        assert bool(((v.double().cpu() - vw).abs() <= U * vw).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_neighbours_stay(O, bits):
    # the tensors are slices of wider buffers, aligned and not: nothing around them changes
    for off in (0, 1, 4):
        n = 777
        wide = torch.full((n + 64,), 7.0, device=DEV)
        shw = torch.full((n + 64,), 5.0, device=DEV, dtype=torch.bfloat16)
        p, sh = wide[off:off + n], shw[off:off + n]
        opt = O.AdamW([p], state_bits=bits, grads=[torch.ones(n, device=DEV)], shadows=[sh])
        opt.step()
        assert wide[:off].eq(7).all() and wide[off + n:].eq(7).all()
        assert shw[:off].eq(5).all() and shw[off + n:].eq(5).all()
        assert p.ne(7).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(O, bits):
    def fresh(**kw):
        p, g, s = make(3000, torch.float32, torch.bfloat16, bits, 11, O)
        return p, g, O.AdamW([p], LR, (B1, B2), EPS, WD, states=[s], grads=[g], **kw)
    p, g, opt = fresh(capturable=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        opt.step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    q, _, plain = fresh()
    for _ in range(4):
        plain.step()
    torch.cuda.synchronize()
    assert int(opt.step_counter) == 4
    # the device computes the coefficients with its own pow: they may differ by a rounding
    assert torch.allclose(p, q, rtol=8 * U, atol=8 * U * 4 * LR)
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            plain.step()
    torch.cuda.synchronize()


def test_two_streams_at_once(O):
    runs = []
    for k in range(2):
        p, g, s = make(300000, torch.float32, torch.float32, 8, 20 + k, O)
        q, h, r = make(300000, torch.float32, torch.float32, 8, 20 + k, O)
        runs.append((p, O.AdamW([p], states=[s], grads=[g]), q, O.AdamW([q], states=[r], grads=[h]), s, r))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for st, (_, opt, *_rest) in zip(streams, runs):
        with torch.cuda.stream(st):
            for _ in range(5):
                opt.step()
    torch.cuda.synchronize()
    for p, _, q, alone, s, r in runs:
        for _ in range(5):
            alone.step()
        assert torch.equal(p, q) and torch.equal(s.m, r.m) and torch.equal(s.v, r.v)


def test_refusals(O):
    f = lambda n=8, dt=torch.float32: torch.zeros(n, dtype=dt, device=DEV)  # noqa: E731
    p, g = f(), f()
    bad = [dict(params=[]), dict(params=[f(8, torch.float16)]), dict(params=[p, f(8, torch.bfloat16)]),
           dict(params=[f(64).view(8, 8).t()]), dict(params=[p], grads=[f(9)]), dict(params=[p], grads=[]),
           dict(params=[p], grads=[f(8, torch.float16)]), dict(params=[p], shadows=[f()]),
           dict(params=[p], shadows=[]), dict(params=[p, p]), dict(params=[p], grads=[p]),
           dict(params=[p], betas=(1.0, 0.9)), dict(params=[p], eps=-1.0), dict(params=[p], weight_decay=-0.1),
           dict(params=[p], state_bits=4), dict(params=[p], state_bits=8, eps=1e-13), dict(params=[p], step=-1),
           dict(params=[p], states=[O.AdamWState(f(), f(9))]), dict(params=[p], states=[]),
           dict(params=[p, f()], states=[O.AdamWState.zeros(p, 8), O.AdamWState.zeros(p, 32)]),
           dict(params=[f(8, torch.bfloat16)], shadows=[f(8, torch.bfloat16)])]
    for kw in bad:
        with pytest.raises(ValueError):
            O.AdamW(**kw)
    opt = O.AdamW([p])
    with pytest.raises(ValueError):
        opt.step()
    with pytest.raises(ValueError):
        opt.step([g], grad_scale=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError):
        opt.step([g], lr=torch.zeros(1))
    with pytest.raises(ValueError):
        opt.state_values([f()], [f()])
    with pytest.raises(ValueError):
        O.AdamW([p], state_bits=8).state_values([f(9)], [f()])
    assert math.isfinite(float(p.sum()))


def test_refused_gradients_leave_the_bound_ones(O):
    runs = []
    for refuse in (True, False):
        made = [make(n, torch.float32, torch.float32, 32, 40 + n, O) for n in (300, 41)]
        opt = O.AdamW([p for p, _, _ in made], states=[s for _, _, s in made], grads=[g for _, g, _ in made])
        if refuse:
            with pytest.raises(ValueError, match="sizes"):
                opt.step([torch.ones(300, device=DEV), torch.ones(40, device=DEV)])
            assert opt.step_count == 0
        opt.step()
        runs.append([p.clone() for p, _, _ in made])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_bound_tensors_stay_and_settings_may_change(O):
    p, g, s = make(515, torch.float32, torch.float32, 8, 5, O)
    opt = O.AdamW([p], LR, (B1, B2), EPS, WD, states=[s], grads=[g])
    for name in ("params", "states", "shadows", "grads", "step_counter"):
        with pytest.raises(AttributeError):
            setattr(opt, name, [p])
    with pytest.raises(AttributeError):
        opt.states[0].m = torch.zeros_like(s.m)
    q, h, r = make(515, torch.float32, torch.float32, 8, 5, O)
    other = O.AdamW([q], states=[r], grads=[h])            # constructed with the defaults, then set
    other.lr, other.betas, other.eps, other.weight_decay = LR, (B1, B2), EPS, WD
    opt.step()
    other.step()
    assert torch.equal(p, q) and torch.equal(s.m, r.m) and torch.equal(s.v_scale, r.v_scale)
