"""Newton-Schulz orthogonalisation on the GPU against the polynomial of the
singular values in 64 bits (an eigendecomposition of the smaller Gram
matrix).

Bound. Operands hold 21 bits or more and sums are fp32, so a step's result
is off by at most DELTA = 2^-19 of its Frobenius norm; a later step stretches
what lies along small singular values by a = 3.4445, so with |X_k|_F <= a^k
the five steps' errors come to at most 6 a^5 DELTA in the Frobenius norm (of a
result of norm about sqrt(rank)), plus one rounding to the output's type."""

import pytest
import torch

from nested_recurrent_memory_b200 import check_status, orthogonalize

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
MUON = (3.4445, -4.7750, 2.0315)
DELTA = 2.0 ** -19


def _exact(G, steps=5, coefficients=MUON, eps=1e-7):
    G = G.double()
    tall = G.shape[-2] > G.shape[-1]
    G = G.transpose(-1, -2) if tall else G
    G = G / (torch.linalg.matrix_norm(G, keepdim=True) + eps)
    lam, U = torch.linalg.eigh(G @ G.transpose(-1, -2))
    a, b, c = coefficients
    f = torch.ones_like(lam)
    for _ in range(steps):
        q = a + b * lam + c * lam * lam
        f, lam = f * q, lam * q * q
    X = (U * f[..., None, :]) @ (U.transpose(-1, -2) @ G)
    return X.transpose(-1, -2) if tall else X


def _check(G, out, **kw):
    ref = _exact(G, **kw)
    assert out.shape == G.shape and bool(torch.isfinite(out).all())
    a, steps = kw.get("coefficients", MUON)[0], kw.get("steps", 5)
    err = torch.linalg.matrix_norm(out.double() - ref)
    bound = (steps + 1) * max(a, 1.0) ** steps * DELTA + UNIT[out.dtype] * torch.linalg.matrix_norm(ref)
    assert bool((err <= bound).all()), (err / bound).max().item()


def _update(shape, dtype, seed=0, remainder=0.1):
    gen = torch.Generator().manual_seed(seed)
    *lead, m, n = shape
    r = max(1, min(8, m, n))
    low = torch.randn(*lead, m, r, generator=gen) @ torch.randn(*lead, r, n, generator=gen)
    return (low / r ** 0.5 + remainder * torch.randn(*shape, generator=gen)).to(dtype).cuda()


SHAPES = [(1, 1), (1, 50), (7, 3), (16, 16), (24, 1024), (64, 64), (65, 63), (128, 128), (128, 130),
          (100, 256), (129, 129), (127, 257), (192, 640), (256, 256), (257, 300), (300, 700),
          (511, 513), (640, 384)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes(shape, dtype):
    G = _update(shape, dtype, seed=shape[0])
    _check(G, orthogonalize(G))


@pytest.mark.parametrize("shape", [(5, 48, 80), (2, 8, 128, 128), (3, 200, 136), (2, 1, 300, 260),
                                   (33, 96, 64), (4, 384, 1000)])
def test_batches(shape):
    """Each matrix of a batch on its own: the same bits as alone."""
    G = _update(shape, torch.float32, seed=1)
    out = orthogonalize(G)
    _check(G, out)
    flat, fo = G.reshape(-1, *shape[-2:]), out.reshape(-1, *shape[-2:])
    for i in (0, flat.shape[0] - 1):
        assert torch.equal(orthogonalize(flat[i]), fo[i])


@pytest.mark.parametrize("shape", [(128, 1500), (16, 2048), (5, 1999), (2049, 1), (1100, 112), (3, 100, 900),
                                   (128, 1600), (120, 4000), (2, 12, 64, 520)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_few_rows_and_many_columns(shape, dtype):
    """A small side of at most 128: on either side of what one launch holds, and
    slices that do not come out even."""
    G = _update(shape, dtype, seed=11)
    out = orthogonalize(G, dtype=torch.float32)
    _check(G, out)
    flat, fo = G.reshape(-1, *shape[-2:]), out.reshape(-1, *shape[-2:])
    assert torch.equal(orthogonalize(flat[-1], dtype=torch.float32), fo[-1])


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_types(dtype, out):
    for shape in ((2, 100, 72), (140, 270)):
        G = _update(shape, dtype, seed=2)
        got = orthogonalize(G, dtype=out)
        assert got.dtype == out
        _check(G, got)


@pytest.mark.parametrize("remainder", [1.0, 0.01, 0.001, 0.0])
def test_strong_directions_over_weak_ones(remainder):
    """Few large singular values over a small (or no) remainder, which the
    iteration stretches by up to a^5."""
    for shape in ((96, 120), (300, 410)):
        G = _update(shape, torch.float32, seed=3, remainder=remainder)
        _check(G, orthogonalize(G))


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_any_magnitude(scale):
    """The result does not depend on the update's scale (until eps matters)."""
    for shape in ((64, 80), (200, 260)):
        G = _update(shape, torch.float32, seed=4) * scale
        _check(G, orthogonalize(G, eps=0.0), eps=0.0)


def test_zero_one_and_bad_updates():
    zero = torch.zeros(3, 40, 50, device="cuda")
    assert bool((orthogonalize(zero) == 0).all())
    for shape in ((3, 40, 50), (2, 200, 300)):
        G = _update(shape, torch.float32, seed=5)
        clean = orthogonalize(G)
        for bad in (float("nan"), float("inf")):
            H = G.clone()
            H[1, 3, 4] = bad
            out = orthogonalize(H)
            assert torch.equal(out[0], clean[0])          # the others keep their bits
            assert not bool(torch.isfinite(out[1]).any())  # and it does not pass as a result
    H = G.clone()
    H[0].zero_()
    out = orthogonalize(H)
    assert bool((out[0] == 0).all()) and torch.equal(out[1], clean[1])


@pytest.mark.parametrize(("steps", "coefficients"), [
    (0, MUON), (1, MUON), (6, MUON), (12, (1.5, -0.5, 0.0)), (8, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(steps, coefficients):
    for shape in ((48, 64), (150, 270)):
        G = _update(shape, torch.float32, seed=6)
        _check(G, orthogonalize(G, steps=steps, coefficients=coefficients), steps=steps,
               coefficients=coefficients)


def test_result_is_nearly_orthogonal():
    """Muon's coefficients leave singular values within about 0.68 .. 1.14."""
    for shape in ((128, 128), (200, 900), (700, 256)):
        G = torch.randn(*shape, generator=torch.Generator().manual_seed(7)).cuda()
        s = torch.linalg.svdvals(orthogonalize(G).double())
        if shape[0] != shape[1]:  # a square Gaussian has singular values near zero
            assert 0.6 < float(s.min())
        assert float(s.max()) < 1.3


def test_strides():
    base = _update((3, 260, 300), torch.bfloat16, seed=8)
    ref = orthogonalize(base)
    wide = torch.cat([base[..., :5], base, base], -1)[..., 5:305]
    assert torch.equal(orthogonalize(wide), ref)
    T = base.transpose(-1, -2)
    assert torch.equal(orthogonalize(T.contiguous().transpose(-1, -2)), ref)
    assert torch.equal(orthogonalize(T), ref.transpose(-1, -2))
    assert torch.equal(orthogonalize(base[:1].expand(3, 260, 300))[2], ref[0])
    swapped = base.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(orthogonalize(swapped), ref)
    four = _update((2, 3, 40, 60), torch.float32, seed=9).transpose(0, 1)
    assert torch.equal(orthogonalize(four), orthogonalize(four.contiguous()))


def test_same_bits_every_time_streams_and_capture():
    for shape in ((6, 128, 96), (2, 384, 520)):
        G = _update(shape, torch.float32, seed=10)
        ref = orthogonalize(G, dtype=torch.bfloat16)
        for _ in range(3):
            assert torch.equal(orthogonalize(G, dtype=torch.bfloat16), ref)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out = orthogonalize(G, dtype=torch.bfloat16)
        s.synchronize()
        assert torch.equal(out, ref)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = orthogonalize(G, dtype=torch.bfloat16)
        for _ in range(2):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ref)
    check_status()


def test_empty():
    assert orthogonalize(torch.zeros(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert orthogonalize(torch.zeros(4, 0, device="cuda")).shape == (4, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(48, 80), (128, 130), (3, 16, 16), (100, 900), (200, 264), (300, 700),
                                   (1001, 345)])
def test_sixteen_bit_results_are_the_fp32_ones_rounded(shape, dtype):
    """Products and sums do not depend on the result's type: a 16-bit result is
    the fp32 result rounded once, bit for bit."""
    G = _update(shape, dtype, seed=12)
    full = orthogonalize(G, dtype=torch.float32)
    for out in (torch.bfloat16, torch.float16):
        assert torch.equal(orthogonalize(G, dtype=out), full.to(out))


def _stop_word(ws, batch, m, n, steps):
    """Where a call's kernels note in its workspace that a wait gave up: the
    second word after the planes of X (twice), A and B, the sums and scales."""
    up = lambda x, k: (x + k - 1) // k * k  # noqa: E731
    at = 2 * up(batch * 2 * m * up(n, 8) * 2, 256) + 2 * up(batch * 2 * m * up(m, 8) * 2, 256)
    at += up(batch * 128 * 8, 256) + up(batch * steps * 8, 256)
    assert ws.data_ptr() % 256 == 0
    return ws[at + 4:at + 8].view(torch.int32)


def _stopped_call(n=2048, steps=64):
    """A call of many launches during which another stream sets that word, as
    a wait that gives up does."""
    G = _update((n, n), torch.float32, seed=13)
    ws = torch.empty(32 * n * n, dtype=torch.uint8, device="cuda")
    stop = _stop_word(ws, 1, n, n, steps)
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    start = torch.cuda.Event()
    torch.cuda.synchronize()
    torch.cuda._sleep(10 ** 8)  # all of this is queued before any of it runs
    start.record(main)
    out = orthogonalize(G, steps=steps, coefficients=(1.5, -0.5, 0.0), workspace=ws)
    with torch.cuda.stream(side):
        side.wait_event(start)
        torch.cuda._sleep(10 ** 6)  # half a millisecond into the call
        stop.fill_(1)
    torch.cuda.synchronize()
    assert int(stop) == 1
    return G, out


def test_a_call_that_gave_up_ends_and_leaves_the_next_one_alone():
    G = _update((300, 700), torch.float32, seed=14)
    ref = orthogonalize(G)
    _stopped_call()
    assert torch.equal(orthogonalize(G), ref)
    check_status()


def test_a_call_that_gave_up_leaves_no_numbers():
    """Whatever later launches of the call compute from operands that were never
    finished does not pass as a result."""
    _, out = _stopped_call()
    assert bool(torch.isnan(out).all())
    check_status()


@pytest.mark.parametrize("norm", [1.0, 1e-3, 1e-7, 1e-11, 1e-14, 1e-20, 1e-30])
@pytest.mark.parametrize("shape", [(64, 80), (900, 100), (200, 260), (2, 384, 1000)])
def test_updates_below_eps_keep_their_digits(shape, norm):
    """X_0 = G / (|G| + eps) is small where |G| is far below eps, and every error
    is relative to it: the bound above times |X_0|."""
    G = _update(shape, torch.float32, seed=15)
    G = G / torch.linalg.matrix_norm(G, keepdim=True) * norm
    ref = _exact(G)
    size = torch.linalg.matrix_norm(G.double())
    X0 = size / (size + 1e-7)
    for dtype in (torch.float32, torch.bfloat16):
        err = torch.linalg.matrix_norm(orthogonalize(G, dtype=dtype).double() - ref)
        bound = 6 * MUON[0] ** 5 * DELTA * X0 + UNIT[dtype] * torch.linalg.matrix_norm(ref)
        assert bool((err <= bound).all()), (err / bound).max().item()


def test_iterations_that_shrink_keep_their_digits():
    """Coefficients below one: forty halvings."""
    for shape in ((48, 64), (150, 270)):
        G = _update(shape, torch.float32, seed=16)
        out = orthogonalize(G, steps=40, coefficients=(0.5, 0.0, 0.0), dtype=torch.float32)
        ref = _exact(G, steps=40, coefficients=(0.5, 0.0, 0.0))
        err = torch.linalg.matrix_norm(out.double() - ref)
        assert bool((err <= 41 * DELTA * 0.5 ** 40).all())
