"""The gated linear recurrence on the GPU (forward, backward, one-token
step) against the token-by-token recurrence in 64 bits.

Bounds are elementwise. The exponential's error (2 ulp) and the roundings of
one step, however the steps are grouped into segments, are within EPS = 2^-21
of the step's magnitude, so with |.| the recurrence of magnitudes
M_t = e^g M_{t-1} + |x_t| the error obeys E_t = e^g (E_{t-1} + EPS M_{t-1}) +
EPS M_t; one rounding to the output's type (u) comes on top."""

import math

import pytest
import torch

from nested_recurrent_memory_b200 import (check_status, gated_scan, gated_scan_bwd,
                                          gated_scan_fwd, step_gated_scan)

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
EPS = 2.0 ** -21


def _inputs(B, T, D, dtype, gdtype, seed=0, decay=5.0, resets=0.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, D, generator=gen)
    g = torch.nn.functional.logsigmoid(torch.randn(B, T, D, generator=gen)
                                       + decay * torch.rand(D, generator=gen))
    if resets:
        g[:, torch.rand(T, generator=gen) < resets] = -math.inf
    dh = torch.randn(B, T, D, generator=gen)
    init, dfin = torch.randn(B, D, generator=gen), torch.randn(B, D, generator=gen)
    return (x.to(dtype).cuda(), g.to(gdtype).cuda(), dh.to(dtype).cuda(), init.cuda(), dfin.cuda())


def _forward64(x, g, init):
    """States, their error bounds, decays."""
    x, a = x.double(), g.double().exp()
    h = torch.zeros_like(x[:, 0]) if init is None else init.double()
    M, E, hs, Es = h.abs(), torch.zeros_like(h), [], []
    for t in range(x.shape[1]):
        E = a[:, t] * (E + EPS * M)
        h, M = a[:, t] * h + x[:, t], a[:, t] * M + x[:, t].abs()
        E = E + EPS * M
        hs.append(h)
        Es.append(E)
    return torch.stack(hs, 1), torch.stack(Es, 1), a


def _within(got, ref, bound):
    u = UNIT[got.dtype]
    assert bool(torch.isfinite(got).all())
    err = (got.double() - ref).abs() - (bound * (1 + u) + u * ref.abs() + TINY[got.dtype])
    assert float(err.max()) <= 0, float((got.double() - ref).abs().max())


def _check(x, g, dh, init, dfin, out):
    h, final, dx, dg, dinit = out
    hs, Es, a = _forward64(x, g, init)
    _within(h, hs, Es)
    _within(final, hs[:, -1], Es[:, -1])
    T = x.shape[1]
    c = torch.zeros_like(hs[:, 0]) if dfin is None else dfin.double()
    M, E = c.abs(), torch.zeros_like(c)
    h0 = torch.zeros_like(c) if init is None else init.double()
    d, us, gs, Eu, Eg = dh.double(), [], [], [], []
    for t in range(T - 1, -1, -1):
        u, Mu = d[:, t] + c, d[:, t].abs() + M
        Eut = E + EPS * Mu
        c, M, E = a[:, t] * u, a[:, t] * Mu, a[:, t] * (Eut + EPS * Mu) + EPS * a[:, t] * Mu
        hp, Ep = (hs[:, t - 1], Es[:, t - 1]) if t else (h0, torch.zeros_like(h0))
        us.append(u)
        Eu.append(Eut)
        gs.append(c * hp)
        Eg.append(c.abs() * Ep + E * (hp.abs() + Ep) + EPS * (c * hp).abs())
    _within(dx, torch.stack(us[::-1], 1), torch.stack(Eu[::-1], 1))
    _within(dg, torch.stack(gs[::-1], 1), torch.stack(Eg[::-1], 1))
    if init is not None:
        _within(dinit, c, E)
    else:
        assert dinit is None


def _run(x, g, dh, init, dfin):
    h, final, aux = gated_scan_fwd(x, g, init, output_final_state=True, return_aux=True)
    return (h, final, *gated_scan_bwd(x, g, dh, dfin, init, aux))


SHAPES = [(1, 1, 1), (2, 1, 33), (1, 2, 64), (3, 7, 40), (2, 63, 32), (1, 64, 130), (2, 127, 5),
          (1, 128, 96), (2, 129, 36), (1, 257, 31), (1, 640, 128), (2, 1000, 77)]


@pytest.mark.parametrize(("B", "T", "D"), SHAPES)
@pytest.mark.parametrize(("dtype", "gdtype"), [
    (torch.float32, torch.float32), (torch.bfloat16, torch.float32),
    (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)])
def test_forward_and_backward(B, T, D, dtype, gdtype):
    ins = _inputs(B, T, D, dtype, gdtype, seed=T)
    _check(*ins, _run(*ins))


@pytest.mark.parametrize("gdtype", [torch.bfloat16, torch.float16])
def test_fp32_inputs_with_16_bit_decays(gdtype):
    ins = _inputs(2, 300, 48, torch.float32, gdtype, seed=1)
    _check(*ins, _run(*ins))


@pytest.mark.parametrize(("with_init", "with_dfin"), [(False, False), (True, False), (False, True)])
def test_without_state_or_final_gradient(with_init, with_dfin):
    x, g, dh, init, dfin = _inputs(2, 400, 64, torch.float32, torch.float32, seed=2)
    ins = (x, g, dh, init if with_init else None, dfin if with_dfin else None)
    _check(*ins, _run(*ins))


@pytest.mark.parametrize("resets", [0.02, 0.5, 1.0])
def test_packed_sequences(resets):
    """-inf decays, at every rate up to every token, the first and last
    among them."""
    x, g, dh, init, dfin = _inputs(2, 500, 72, torch.float32, torch.float32, seed=3, resets=resets)
    g[0, 0] = -math.inf
    g[1, -1] = -math.inf
    ins = (x, g, dh, init, dfin)
    _check(*ins, _run(*ins))


def test_packed_sequences_equal_separate_calls():
    x, g, _, _, _ = _inputs(1, 700, 64, torch.float32, torch.float32, seed=4)
    cuts = [0, 1, 130, 131, 400, 700]
    for c in cuts[:-1]:
        g[:, c] = -math.inf
    h, _ = gated_scan_fwd(x, g)
    for lo, hi in zip(cuts, cuts[1:]):
        hs, Es, _ = _forward64(x[:, lo:hi], g[:, lo:hi], None)
        _within(h[:, lo:hi], hs, Es)


def test_decays_to_nothing_and_none():
    """Decays that underflow, decays of exactly one, the lowest finite value."""
    x, g, dh, init, dfin = _inputs(1, 300, 96, torch.float32, torch.float32, seed=5)
    g[..., :32] = -200.0
    g[..., 32:64] = 0.0
    g[..., 64:] = torch.finfo(torch.float32).min
    ins = (x, g, dh, init, dfin)
    _check(*ins, _run(*ins))


def test_long_sequences_and_chunk_chain():
    """Many chunks in a chain for few channels, and many channels: against
    the recurrence, and the same bits every time."""
    for B, T, D in ((1, 9001, 40), (5, 1111, 515)):
        ins = _inputs(B, T, D, torch.bfloat16, torch.float32, seed=6, decay=8.0)
        first = _run(*ins)
        _check(*ins, first)
        for _ in range(4):
            again = _run(*ins)
            assert all(torch.equal(p, q) for p, q in zip(first, again))
    check_status()


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last sequence of a packed row, forward and
    backward, against the recurrence on its own."""
    T, D, last = 1100000, 2048, 300
    assert T * D > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(16)
    x = torch.randn(1, T, D, generator=gen, device="cuda", dtype=torch.bfloat16)
    g = torch.full((1, 1, 1), -0.05, device="cuda").expand(1, T, D).to(torch.bfloat16)
    g[:, T - last] = -math.inf
    h, final, aux = gated_scan_fwd(x, g, output_final_state=True, return_aux=True)
    hs, Es, _ = _forward64(x[:, -last:], g[:, -last:], None)
    _within(h[:, -last:], hs, Es)
    _within(final, hs[:, -1], Es[:, -1])
    dx, dg, _ = gated_scan_bwd(x, g, x, aux=aux)
    tail = [t[:, -last:].contiguous() for t in (x, g)]
    ref = gated_scan_bwd(*tail, tail[0])
    for a, b in zip((dx, dg), ref):
        a, b = a[:, -last:].float(), b.float()  # the same but for where tiles begin
        assert float((a - b).norm()) <= 2.0 ** -7 * float(b.norm())


def test_strides_broadcasts_and_offsets():
    B, T, D = 2, 270, 64
    x, g, dh, init, dfin = _inputs(B, T, D, torch.bfloat16, torch.float32, seed=7)
    ref = _run(x, g, dh, init, dfin)
    tm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731  time-major
    dm = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731  channel-major
    wide = lambda t: torch.cat([t[..., :3], t, t], -1)[..., 3:D + 3]  # noqa: E731  off the boundary
    for f in (tm, dm, wide):
        for p, q in zip(ref, _run(f(x), f(g), f(dh), init, dfin)):
            assert torch.equal(p, q)
    # One decay a head, and one a channel, as broadcast views.
    for gb in (g[..., :1].expand(B, T, D), g[:1, :1].expand(B, T, D), g[:, :1, :1].expand(B, T, D)):
        for p, q in zip(_run(x, gb.contiguous(), dh, init, dfin), _run(x, gb, dh, init, dfin)):
            assert torch.equal(p, q)
    one = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(B, T, D)
    for p, q in zip(_run(x, g, one.contiguous(), init, dfin), _run(x, g, one, init, dfin)):
        assert torch.equal(p, q)


def test_backward_without_the_forwards_states():
    x, g, dh, init, dfin = _inputs(2, 333, 48, torch.float32, torch.float32, seed=8)
    ref = _run(x, g, dh, init, dfin)[2:]
    assert all(torch.equal(p, q) for p, q in zip(ref, gated_scan_bwd(x, g, dh, dfin, init)))


def test_autograd_with_broadcast_decays():
    """A decay shared by the channels gets the sum of their gradients."""
    x, g, dh, init, dfin = _inputs(2, 200, 32, torch.float32, torch.float32, seed=9)
    leaves = [x.clone().requires_grad_(), g[..., :1].clone().requires_grad_(),
              init.clone().requires_grad_()]
    h, final = gated_scan(leaves[0], leaves[1].expand_as(x), leaves[2], output_final_state=True)
    ((h * dh).sum() + (final * dfin).sum()).backward()
    dx, dg, dinit = gated_scan_bwd(x, g[..., :1].expand_as(x), dh, dfin, init)
    assert torch.equal(leaves[0].grad, dx) and torch.equal(leaves[2].grad, dinit)
    assert torch.allclose(leaves[1].grad, dg.sum(-1, keepdim=True), rtol=1e-5, atol=1e-5)
    h, final = gated_scan(leaves[0].detach().requires_grad_(), g, None)
    assert final is None
    h.sum().backward()  # a broadcast gradient


def test_gradients_against_differences():
    """Central differences along random directions, in fp32 with a step of
    2^-7: the third derivatives leave about 2^-14 / 6 of the change's scale,
    the roundings 2^-22 * 2^7."""
    x, g, dh, init, dfin = _inputs(1, 90, 16, torch.float32, torch.float32, seed=10, decay=2.0)
    dx, dg, dinit = gated_scan_bwd(x, g, dh, dfin, init)

    def loss(x, g, init):
        h, f = gated_scan_fwd(x, g, init, output_final_state=True)
        return float((h.double() * dh.double()).sum() + (f.double() * dfin.double()).sum())

    gen = torch.Generator().manual_seed(11)
    s = 2.0 ** -7
    for which, grad in enumerate((dx, dg, dinit)):
        base = [x, g, init]
        v = torch.randn(base[which].shape, generator=gen).cuda()
        up, down = list(base), list(base)
        up[which], down[which] = base[which] + s * v, base[which] - s * v
        slope = (loss(*up) - loss(*down)) / (2 * s)
        scale = float(grad.double().norm() * v.double().norm())
        assert abs(slope - float((grad.double() * v.double()).sum())) <= 2e-3 * scale


def test_bad_values_stay_in_their_channel():
    """Infinities and NaN spread along their own channel only, and not past
    a packed sequence's start for infinities dropped by a decay of zero --
    there e^-inf times infinity is not a number, as in the formula."""
    x, g, dh, init, dfin = _inputs(1, 300, 64, torch.float32, torch.float32, seed=12)
    clean, _ = gated_scan_fwd(x, g, init)
    x2 = x.clone()
    x2[0, 150, 5] = math.nan
    x2[0, 40, 37] = math.inf
    h, _ = gated_scan_fwd(x2, g, init)
    keep = [c for c in range(64) if c not in (5, 37)]
    assert torch.equal(h[..., keep], clean[..., keep])
    assert torch.equal(h[:, :128, 5], clean[:, :128, 5])
    assert bool(torch.isnan(h[:, 150:, 5]).all()) and bool(torch.isinf(h[:, 40, 37]).all())


@pytest.mark.parametrize(("dtype", "gdtype"), [
    (torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize(("B", "D"), [(1, 1), (3, 33), (64, 1024), (7, 2050)])
def test_step(B, D, dtype, gdtype):
    x, g, _, init, _ = _inputs(B, 1, D, dtype, gdtype, seed=13)
    hs, Es, _ = _forward64(x, g, init)
    h, state = step_gated_scan(x[:, 0], g[:, 0], init)
    _within(h, hs[:, 0], Es[:, 0])
    _within(state, hs[:, 0], Es[:, 0])
    own = init.clone()
    h2, s2 = step_gated_scan(x[:, 0], g[:, 0], own, out_state=own)
    assert s2.data_ptr() == own.data_ptr() and torch.equal(h, h2) and torch.equal(state, own)
    h3, s3 = step_gated_scan(x[:, 0].t().contiguous().t(), g[:1, 0].expand(B, D)
                             if B == 1 else g[:, 0], init)
    assert torch.equal(h, h3) and torch.equal(state, s3)


def test_prefill_then_steps_match_one_pass():
    x, g, _, init, _ = _inputs(2, 140, 48, torch.float32, torch.float32, seed=14)
    hs, Es, _ = _forward64(x, g, init)
    h, state = gated_scan_fwd(x[:, :131], g[:, :131], init, output_final_state=True)
    _within(h, hs[:, :131], Es[:, :131])
    for t in range(131, 140):
        h, state = step_gated_scan(x[:, t], g[:, t], state)
        _within(h, hs[:, t], Es[:, t])


def test_empty_sequences():
    x = torch.zeros(2, 0, 8, device="cuda")
    init = torch.randn(2, 8, device="cuda")
    h, final = gated_scan_fwd(x, x, init, output_final_state=True)
    assert h.shape == x.shape and torch.equal(final, init)
    assert torch.equal(gated_scan_fwd(x, x, output_final_state=True)[1], torch.zeros_like(init))
    dx, dg, dinit = gated_scan_bwd(x, x, x, d_final=init, initial_state=init)
    assert dx.shape == dg.shape == x.shape and torch.equal(dinit, init)


def test_another_stream_and_graph_capture():
    ins = _inputs(2, 900, 96, torch.bfloat16, torch.float32, seed=15)
    ref = _run(*ins)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = _run(*ins)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ref, out))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(*ins)
    for _ in range(2):
        for t in out:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ref, out))
