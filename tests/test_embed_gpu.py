"""The scaled embedding lookup and its gradient on the GPU against 64-bit
arithmetic. Bounds are elementwise: one rounding to the output's type (u),
and for the gradient n additions in fp32, in whatever order, of n terms:
n * 2^-24 of the sum of their magnitudes."""

import pytest
import torch

from nested_recurrent_memory_b200 import (KernelStatusError, check_status, embed_tokens,
                                          embed_tokens_bwd, embed_tokens_fwd)

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
F32 = 2.0 ** -24


def _inputs(N, V, D, dtype, seed=0, zipf=True):
    gen = torch.Generator().manual_seed(seed)
    u = torch.rand(N, generator=gen, dtype=torch.float64)
    ids = ((V + 1.0) ** u).long() - 1 if zipf else (u * V).long()
    w = torch.randn(V, D, generator=gen).to(dtype)
    d = torch.randn(N, D, generator=gen).to(dtype)
    return ids.clamp(0, V - 1).cuda(), w.cuda(), d.cuda()


def _grad64(ids, d, V, scale, pad=None):
    """The gradient and the sum of its terms' magnitudes, and each row's count."""
    d = d.double()
    keep = torch.ones_like(ids, dtype=torch.bool) if pad is None else ids != pad
    dw = torch.zeros(V, d.shape[1], dtype=torch.float64, device=d.device)
    mag = dw.clone()
    dw.index_put_((ids[keep],), d[keep] * scale, accumulate=True)
    mag.index_put_((ids[keep],), d[keep].abs() * abs(scale), accumulate=True)
    return dw, mag, torch.bincount(ids[keep], minlength=V)[:, None]


def _check_grad(dw, ids, d, scale, pad=None):
    ref, mag, n = _grad64(ids, d, dw.shape[0], scale, pad)
    bound = (UNIT[dw.dtype] + 2 * F32) * ref.abs() + (n + 2) * F32 * mag + TINY[dw.dtype]
    assert bool(((dw.double() - ref).abs() <= bound).all())
    assert bool((dw[(n == 0).flatten()] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("N", "V", "D"), [
    (1, 1, 1), (1, 100, 7), (3, 2, 33), (257, 1000, 64), (1000, 50, 321), (4099, 513, 128),
    (2049, 70001, 24), (33, 300, 2050)])
def test_lookup_and_gradient(N, V, D, dtype):
    ids, w, d = _inputs(N, V, D, dtype)
    scale = D ** 0.5
    y = embed_tokens_fwd(ids, w, scale=scale)
    f32_scale = float(torch.tensor(scale))
    ref = w.double()[ids] * f32_scale
    assert y.dtype == dtype
    assert bool(((y.double() - ref).abs() <= (UNIT[dtype] + F32) * ref.abs() + TINY[dtype]).all())
    dw = embed_tokens_bwd(ids, d, V, scale=scale)
    assert dw.dtype == dtype
    _check_grad(dw, ids, d, f32_scale)


@pytest.mark.parametrize("N", [2048, 2049, 70000, 140001])
def test_one_token_takes_every_position(N):
    """Every position holds the same token: one row sums them all, the
    others are zero."""
    V, D = 300, 40
    ids = torch.full((N,), 217, device="cuda")
    d = torch.randn(N, D, generator=torch.Generator().manual_seed(1)).cuda()
    dw = embed_tokens_bwd(ids, d, V)
    _check_grad(dw, ids, d, 1.0)


@pytest.mark.parametrize(("N", "V"), [(70001, 1 << 17), (50000, 1024), (300000, 33000)])
def test_gradient_of_long_batches_is_reproducible(N, V):
    D = 64
    ids, _, d = _inputs(N, V, D, torch.bfloat16, seed=3)
    first = embed_tokens_bwd(ids, d, V, scale=8.0, padding_idx=0)
    _check_grad(first, ids, d, 8.0, pad=0)
    for _ in range(3):
        assert torch.equal(embed_tokens_bwd(ids, d, V, scale=8.0, padding_idx=0), first)


@pytest.mark.parametrize("N", [5, 3000, 12000, 20000])
def test_tables_larger_than_what_is_zeroed_beside_the_sort(N):
    """164 MB of fp32 gradient, few of whose rows have a token."""
    V, D = 40000, 1024
    ids, _, d = _inputs(N, V, D, torch.float32, seed=8, zipf=False)
    dw = torch.full((V, D), float("nan"), device="cuda")  # (freed: the result may take its place)
    del dw
    dw = embed_tokens_bwd(ids, d, V, scale=2.0, padding_idx=7)
    _check_grad(dw, ids, d, 2.0, pad=7)


def test_offsets_past_32_bits():
    """Outputs and gradients of more than 2^31 elements: rows at the end."""
    N, V, D = 1100000, 50, 2048
    ids = torch.randint(0, V - 1, (N,), generator=torch.Generator().manual_seed(9)).cuda()
    ids[-3:] = V - 1
    w = torch.randn(V, D, generator=torch.Generator().manual_seed(10)).bfloat16().cuda()
    y = embed_tokens_fwd(ids, w)
    assert N * D > 2 ** 31 and torch.equal(y[-2000:], w[ids[-2000:]]) and torch.equal(y[:2000], w[ids[:2000]])
    dw = embed_tokens_bwd(ids, y, V)
    assert torch.equal(dw[V - 1], (3 * w[V - 1].float()).bfloat16())


@pytest.mark.parametrize("pad", [0, -1, 17])
def test_padding_row_gets_no_gradient(pad):
    V, D = 40, 48
    ids, w, d = _inputs(500, V, D, torch.float32, seed=4, zipf=False)
    assert torch.equal(embed_tokens(ids, w, 3.0, padding_idx=pad), embed_tokens_fwd(ids, w, 3.0))
    dw = embed_tokens_bwd(ids, d, V, scale=3.0, padding_idx=pad)
    _check_grad(dw, ids, d, 3.0, pad=pad % V)
    assert bool((dw[pad] == 0).all())


def test_all_tokens_padding_or_none():
    d = torch.randn(64, 16, device="cuda")
    dw = embed_tokens_bwd(torch.zeros(64, dtype=torch.long, device="cuda"), d, 10, padding_idx=0)
    assert bool((dw == 0).all())
    none = torch.zeros(0, dtype=torch.long, device="cuda")
    assert embed_tokens_fwd(none, torch.ones(5, 8, device="cuda")).shape == (0, 8)
    dw = embed_tokens_bwd(none, torch.zeros(0, 8, device="cuda"), 5)
    assert dw.shape == (5, 8) and bool((dw == 0).all())


def test_shapes_strides_and_index_types():
    ids, w, d = _inputs(6 * 20, 90, 36, torch.bfloat16, seed=5)
    ref = embed_tokens_fwd(ids, w, 2.0)
    ids2 = ids.view(6, 20)
    assert torch.equal(embed_tokens_fwd(ids2.int(), w, 2.0), ref.view(6, 20, 36))
    assert torch.equal(embed_tokens_fwd(ids2.t(), w, 2.0), ref.view(6, 20, 36).transpose(0, 1))
    wide = torch.randn(90, 77, device="cuda").bfloat16()
    part = wide[:, 5:41]  # rows off every vector boundary
    assert torch.equal(embed_tokens_fwd(ids, part, 2.0), embed_tokens_fwd(ids, part.contiguous(), 2.0))
    assert torch.equal(embed_tokens_fwd(ids, w.t().contiguous().t(), 2.0), ref)
    dw = embed_tokens_bwd(ids, d, 90)
    dwide = torch.randn(120, 77, device="cuda").bfloat16()
    dwide[:, 5:41] = d
    assert torch.equal(embed_tokens_bwd(ids2, dwide[:, 5:41].view(6, 20, 36), 90), dw)
    ones = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(120, 36)
    counts = torch.bincount(ids, minlength=90).bfloat16()[:, None].expand(90, 36)
    assert torch.equal(embed_tokens_bwd(ids, ones, 90), counts)
    f32 = embed_tokens_bwd(ids, d, 90, dtype=torch.float32)
    assert f32.dtype == torch.float32
    _check_grad(f32, ids, d, 1.0)


def test_autograd_and_differences():
    ids, w, d = _inputs(400, 60, 20, torch.float32, seed=6)
    w.requires_grad_(True)
    (embed_tokens(ids.view(20, 20), w, scale=4.0, padding_idx=3) * d.view(20, 20, 20)).sum().backward()
    assert torch.equal(w.grad, embed_tokens_bwd(ids, d, 60, 4.0, 3))
    # The lookup is linear: differences are exact up to the roundings of 400 * 20 products.
    v = torch.randn(60, 20, device="cuda")
    v[3] = 0  # the padding row takes no part
    loss = lambda s: (embed_tokens_fwd(ids, w.detach() + s * v, 4.0).double() * d.double()).sum()  # noqa: E731
    diff = float(loss(0.5) - loss(-0.5))
    terms = float((embed_tokens_fwd(ids, w.detach().abs() + v.abs(), 4.0).double() * d.abs().double()).sum())
    assert abs(diff - float((w.grad.double() * v.double()).sum())) <= 2 ** -21 * terms


def test_foreign_tokens_are_reported_and_not_read():
    check_status()
    w = torch.randn(30, 16, device="cuda")
    ids = torch.tensor([0, 30, 5, -1, 29], device="cuda")
    y = embed_tokens_fwd(ids, w)
    with pytest.raises(KernelStatusError, match="token id"):
        check_status()
    assert torch.equal(y[[0, 2, 4]], w[[0, 5, 29]]) and bool(torch.isnan(y[[1, 3]]).all())
    d = torch.randn(5, 16, device="cuda")
    dw = embed_tokens_bwd(ids, d, 30)
    with pytest.raises(KernelStatusError, match="token id"):
        check_status()
    assert torch.equal(dw[[0, 5, 29]], d[[0, 2, 4]])
    assert bool((dw[[i for i in range(30) if i not in (0, 5, 29)]] == 0).all())
    check_status()


def test_another_stream_and_graph_capture():
    ids, w, d = _inputs(3000, 700, 64, torch.bfloat16, seed=7)
    ref, dref = embed_tokens_fwd(ids, w, 8.0), embed_tokens_bwd(ids, d, 700, 8.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, dw = embed_tokens_fwd(ids, w, 8.0), embed_tokens_bwd(ids, d, 700, 8.0)
    s.synchronize()
    assert torch.equal(y, ref) and torch.equal(dw, dref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dw = embed_tokens_fwd(ids, w, 8.0), embed_tokens_bwd(ids, d, 700, 8.0)
    for _ in range(2):
        y.zero_()
        dw.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref) and torch.equal(dw, dref)


@pytest.mark.parametrize("N", [1, 700, 9000, 16385, 300001])
@pytest.mark.parametrize("V", [(1 << 18) - 1, 1 << 18, 1 << 20])
def test_tables_whose_tokens_take_three_passes(N, V):
    """Two sorting passes end at 2^18 - 1 rows; lists sorted by one cluster and in
    tiles of either size."""
    D = 8
    for zipf in (True, False):
        ids, _, d = _inputs(N, V, D, torch.float32, seed=11, zipf=zipf)
        ids[0] = V - 1
        dw = embed_tokens_bwd(ids, d, V, scale=3.0, padding_idx=5)
        _check_grad(dw, ids, d, 3.0, pad=5)
        assert torch.equal(embed_tokens_bwd(ids, d, V, scale=3.0, padding_idx=5), dw)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 72, 1000])
def test_gradients_of_another_type(dtype, out, D):
    """Rows read 16 bytes at a time, written in the gradient's own type."""
    ids, _, d = _inputs(3000, 200, D, dtype, seed=12)
    dw = embed_tokens_bwd(ids, d, 200, scale=2.0, dtype=out)
    assert dw.dtype == out
    _check_grad(dw, ids, d, 2.0)
    off = torch.empty(3000 * D + 1, dtype=dtype, device="cuda")[1:].view(3000, D)
    off.copy_(d)  # rows off every 16-byte boundary: element by element, the same sums
    assert torch.equal(embed_tokens_bwd(ids, off, 200, scale=2.0, dtype=out), dw)
