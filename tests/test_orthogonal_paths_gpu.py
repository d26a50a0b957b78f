"""The ways in which large updates are orthogonalised: all products of a batch
in one launch, or a launch for each, in tiles of 256, 128 or 64 columns.
Each shape's way is worked out here by the same rules, so that a shape that
no longer takes the way it stands for fails. Bounds as for small updates:
2^-19 of a step's norm, stretched by a a step."""

import pytest
import torch

from nested_recurrent_memory_b200 import check_status, orthogonalize

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
MUON = (3.4445, -4.7750, 2.0315)
DELTA = 2.0 ** -19


def _way(batch, rows, cols):
    """("one", width), or ("each", width for A and B, width for B X)."""
    m, n = min(rows, cols), max(rows, cols)
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    up = lambda x, k: (x + k - 1) // k  # noqa: E731
    r = up(m, 256)
    sym = {w: r * up(m, w) - r * (r - 1) // 2 * (256 // w) for w in (256, 128, 64)}
    app = {w: r * up(n, w) for w in (256, 128, 64)}
    rounds = lambda tiles: up(batch * tiles, pairs)  # noqa: E731
    if batch > 1 and batch * sym[256] > pairs:
        total = {w: rounds(sym[w]) * (n + m) + rounds(app[w]) * m for w in (256, 128)}
        return "one", 128 if 0.6 * total[128] < total[256] else 256
    cost = {256: 1.0, 128: 0.6, 64: 0.5}
    best = []
    for tiles in (sym, app):
        t = {w: cost[w] * rounds(tiles[w]) for w in cost}
        best.append(64 if t[64] < min(t[128], t[256]) else 128 if t[128] < t[256] else 256)
    return "each", *best


def _update(shape, dtype=torch.float32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    *lead, m, n = shape
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return ((normal(*lead, m, 8) @ normal(*lead, 8, n)) / 8 ** 0.5 + 0.1 * normal(*shape)).to(dtype)


def _exact(G, steps=5, coefficients=MUON):
    G = G.double()
    tall = G.shape[-2] > G.shape[-1]
    G = G.mT if tall else G
    G = G / (torch.linalg.matrix_norm(G, keepdim=True) + 1e-7)
    a, b, c = coefficients
    X, one = G, torch.eye(G.shape[-2], dtype=G.dtype, device=G.device)
    for _ in range(steps):
        A = X @ X.mT
        X = (a * one + b * A + c * (A @ A)) @ X
    return X.mT if tall else X


def _check(G, out, steps=5):
    ref = _exact(G, steps)
    err = torch.linalg.matrix_norm(out.double() - ref)
    bound = (steps + 1) * MUON[0] ** steps * DELTA + UNIT[out.dtype] * torch.linalg.matrix_norm(ref)
    assert bool((err <= bound).all()), (err / bound).max().item()


ONE = [((26, 300, 400), 128), ((80, 200, 264), 128), ((30, 515, 777), 128), ((76, 129, 131), 128),
       ((12, 1024, 1024), 256), ((12, 1100, 1024), 256), ((9, 1025, 1290), 256)]
EACH = [((2048, 2048), 128, 256), ((4096, 4096), 256, 256), ((1024, 2816), 64, 256),
        ((2816, 1024), 64, 256), ((1536, 1536), 128, 128), ((1024, 1600), 64, 128), ((1001, 345), 64, 64),
        ((1700, 1801), 128, 256), ((2300, 2301), 256, 128), ((4, 384, 1000), 64, 128),
        ((7, 700, 900), 256, 128), ((40, 131, 1000), 256, 256)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize(("shape", "width"), ONE)
def test_batches_in_one_launch(shape, width, dtype):
    """Right, the same bits each time, and each matrix the bits that it has alone."""
    assert _way(*shape) == ("one", width)
    G = _update(shape, dtype, seed=1)
    for out in (torch.float32, torch.bfloat16):
        X = orthogonalize(G, dtype=out)
        _check(G, X)
        for _ in range(3):
            assert torch.equal(orthogonalize(G, dtype=out), X)
        for i in (0, shape[0] // 2, shape[0] - 1):
            assert torch.equal(orthogonalize(G[i], dtype=out), X[i])
    check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize(("shape", "sym", "app"), EACH)
def test_a_launch_for_each_product(shape, sym, app, dtype):
    assert _way(*((1,) * (3 - len(shape)) + shape)) == ("each", sym, app)
    G = _update(shape, dtype, seed=2)
    for out in (torch.float32, torch.bfloat16):
        X = orthogonalize(G, dtype=out)
        _check(G, X)
        assert torch.equal(orthogonalize(G, dtype=out), X)
    check_status()


@pytest.mark.parametrize("shape", [s for s, *_ in ONE + EACH])
@pytest.mark.parametrize("steps", [1, 2])
def test_few_steps_leave_little_room(shape, steps):
    """The bound after one or two steps is 1e-5 to 7e-5 of the update's norm: an
    operand's second plane left out anywhere would pass it."""
    for dtype in (torch.float32, torch.float16):
        G = _update(shape, dtype, seed=3)
        _check(G, orthogonalize(G, steps=steps, dtype=torch.float32), steps)


def test_one_launch_on_another_stream_and_in_a_graph():
    G = _update((12, 1024, 1024), seed=4)
    ref = orthogonalize(G)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = orthogonalize(G)
    s.synchronize()
    assert torch.equal(out, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(G)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
    check_status()


@pytest.mark.parametrize("shape", [(26, 300, 400), (12, 1024, 1024), (2, 1024, 1500)])
def test_a_bad_or_zero_matrix_leaves_the_others_alone(shape):
    G = _update(shape, seed=5)
    clean = orthogonalize(G)
    H = G.clone()
    H[0].zero_()
    H[1, 3, 4] = float("nan")
    out = orthogonalize(H)
    assert bool((out[0] == 0).all()) and not bool(torch.isfinite(out[1]).any())
    assert torch.equal(out[2:], clean[2:])


@pytest.mark.parametrize("shape", [(129, 20000), (200, 60000), (4096, 4100)])
def test_the_error_does_not_grow_with_the_reduction(shape):
    """The bound knows no sizes: sums of any length keep it."""
    G = _update(shape, seed=6)
    for steps in (1, 2, 5):
        _check(G, orthogonalize(G, steps=steps), steps)
