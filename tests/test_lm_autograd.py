"""The autograd functions of the embedding and the recurrence on the host,
their kernels replaced by plain operations that leave no graph (as kernels do
not): second derivatives and forward-mode tangents are right or refused,
never dropped."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F

from nested_recurrent_memory_b200 import (embedding, gated_scan, model, recurrence,
                                          step_gated_scan)
from nested_recurrent_memory_b200.embedding import embed_tokens

V, D, SCALE = 7, 3, 1.5


@pytest.fixture
def plain_embedding(monkeypatch):
    def fwd(ids, weight, scale=1.0):
        return (weight.detach()[ids] * scale).clone()

    def bwd(ids, d_out, num_embeddings, scale=1.0, padding_idx=None, dtype=None, workspace=None):
        d = d_out.detach().reshape(-1, d_out.shape[-1]) * scale
        keep = torch.ones(ids.numel(), dtype=torch.bool)
        if padding_idx is not None:
            keep = ids.flatten() != padding_idx % num_embeddings
        dw = torch.zeros(num_embeddings, d.shape[1], dtype=d.dtype)
        return dw.index_add_(0, ids.flatten()[keep], d[keep]).to(dtype or d.dtype)

    monkeypatch.setattr(embedding, "embed_tokens_fwd", fwd)
    monkeypatch.setattr(embedding, "embed_tokens_bwd", bwd)


def _case():
    gen = torch.Generator().manual_seed(0)
    ids = torch.randint(0, V, (4, 5), generator=gen)
    w, t = (torch.randn(V, D, generator=gen, dtype=torch.float64) for _ in range(2))
    return ids, w, t, torch.randn(4, 5, D, generator=gen, dtype=torch.float64)


def _torch(ids, w, pad):
    return F.embedding(ids, w, pad) * SCALE


@pytest.mark.parametrize("pad", [None, 2, -1])
def test_embedding_second_derivatives(plain_embedding, pad):
    """A penalty on the gradient of a loss that is not linear in the rows."""
    ids, w, t, c = _case()
    got = []
    for fn in (lambda x: embed_tokens(ids, x, SCALE, pad), lambda x: _torch(ids, x, pad)):
        x = w.clone().requires_grad_()
        (g,) = torch.autograd.grad((fn(x).sin() * c).sum(), x, create_graph=True)
        assert g.requires_grad
        (g2,) = torch.autograd.grad((g * g * t).sum(), x, create_graph=True)
        (g3,) = torch.autograd.grad(g2.pow(3).sum(), x)
        got.append((g, g2, g3))
    for p, q in zip(*got):
        assert torch.allclose(p, q, rtol=1e-12, atol=1e-12)


def test_embedding_gradients_against_differences(plain_embedding):
    ids, w, _, _ = _case()
    w.requires_grad_()
    torch.autograd.gradcheck(lambda x: embed_tokens(ids, x, SCALE, 2)[ids != 2], (w,),
                             check_forward_ad=True)
    torch.autograd.gradgradcheck(lambda x: embed_tokens(ids, x, SCALE, 2)[ids != 2].sin(), (w,))


@pytest.mark.parametrize("requires_grad", [False, True])
def test_embedding_forward_mode(plain_embedding, requires_grad):
    ids, w, t, _ = _case()
    w.requires_grad_(requires_grad)
    with fwAD.dual_level():
        x = fwAD.make_dual(w, t)
        y, ref = embed_tokens(ids, x, SCALE, 2), _torch(ids, x, 2)
        assert torch.equal(fwAD.unpack_dual(y).tangent, fwAD.unpack_dual(ref).tangent)


def test_embedding_reverse_over_forward(plain_embedding):
    """The tangent of a gradient (a Hessian-vector product) without second reverse."""
    ids, w, t, c = _case()
    got = []
    for fn in (lambda x: embed_tokens(ids, x, SCALE, 2), lambda x: _torch(ids, x, 2)):
        with fwAD.dual_level():
            x = fwAD.make_dual(w.clone().requires_grad_(), t)
            (g,) = torch.autograd.grad((fn(x).sin() * c).sum(), x)
            got.append(fwAD.unpack_dual(g).tangent)
    assert got[0] is not None and torch.allclose(*got, rtol=1e-12, atol=1e-12)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_embedding_derivatives_on_the_kernels(dtype):
    """All values are small whole numbers: no sum rounds, so both agree exactly."""
    gen = torch.Generator().manual_seed(1)
    small = lambda *s: torch.randint(-2, 3, s, generator=gen).to(dtype).cuda()  # noqa: E731
    ids = torch.randint(0, 50, (6, 9), generator=gen).cuda()
    w, t, c = small(50, 24), small(50, 24), small(6, 9, 24)
    got = []
    for fn in (lambda x: embed_tokens(ids, x, 2.0, 3), lambda x: F.embedding(ids, x, 3) * 2.0):
        x = w.clone().requires_grad_()
        (g,) = torch.autograd.grad((fn(x) ** 2 * c).sum(), x, create_graph=True)
        (g2,) = torch.autograd.grad((g * t).sum(), x)
        with fwAD.dual_level():
            tangent = fwAD.unpack_dual(fn(fwAD.make_dual(w, t))).tangent
        got.append((g.detach(), g2, tangent))
    for p, q in zip(*got):
        assert torch.equal(p, q)


@pytest.fixture
def plain_recurrence(monkeypatch):
    def fwd(x, g, initial_state=None, output_final_state=False, return_aux=False, workspace=None):
        h = x.detach() * 2
        final = h[:, -1].clone() if output_final_state else None
        return (h, final, dict(carries=h)) if return_aux else (h, final)

    def bwd(x, g, dh, d_final=None, initial_state=None, aux=None, workspace=None):
        init = None if initial_state is None else torch.zeros_like(initial_state)
        return dh.detach() * 2, torch.zeros_like(g), init

    monkeypatch.setattr(recurrence, "gated_scan_fwd", fwd)
    monkeypatch.setattr(recurrence, "gated_scan_bwd", bwd)


def test_recurrence_refuses_second_derivatives(plain_recurrence):
    x = torch.randn(2, 4, 3, requires_grad=True)
    gate = torch.zeros(2, 4, 3, requires_grad=True)
    (dx, dg) = torch.autograd.grad((gated_scan(x, gate)[0] ** 2).sum(), (x, gate), create_graph=True)
    for loss in ((dx ** 2).sum(), dg.sum(), dx.sum()):
        for leaf in (x, gate):
            with pytest.raises(RuntimeError, match="second derivatives"):
                torch.autograd.grad(loss + (x * gate).sum(), leaf, retain_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        (dx ** 2).sum().backward()
    (dx,) = torch.autograd.grad(gated_scan(x, gate)[0].sum(), x)  # first ones leave no graph
    assert not dx.requires_grad


@pytest.mark.parametrize("which", ["x", "g", "initial_state"])
def test_recurrence_refuses_forward_mode(plain_recurrence, which):
    ins = dict(x=torch.randn(2, 4, 3), g=torch.zeros(2, 4, 3), initial_state=torch.zeros(2, 3))
    with fwAD.dual_level():
        ins[which] = fwAD.make_dual(ins[which], torch.ones_like(ins[which]))
        with pytest.raises(NotImplementedError):
            gated_scan(**ins)


@pytest.mark.parametrize("which", ["x", "g", "state"])
def test_step_refuses_gradients_that_it_would_drop(which):
    """Refused before anything else is looked at."""
    ins = dict(x=torch.randn(2, 3), g=torch.zeros(2, 3), state=torch.zeros(2, 3))
    with fwAD.dual_level():
        dual = {**ins, which: fwAD.make_dual(ins[which], torch.ones(2, 3))}
        with pytest.raises(RuntimeError, match="not differentiable"):
            step_gated_scan(**dual)
    ins[which].requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        step_gated_scan(**ins)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
        step_gated_scan(**ins)


def test_decoding_takes_no_part_in_autograd(monkeypatch):
    """The model's step, with the states of a prefill that autograd follows."""
    def scan(x, g, initial_state=None, output_final_state=False):
        return x * 1.0, x[:, -1].float()

    def step(x, g, state, out_state=None):
        assert not torch.is_grad_enabled()
        out_state.copy_(state + x)
        return x * 1.0, out_state

    monkeypatch.setattr(model, "gated_scan", scan)
    monkeypatch.setattr(model, "step_gated_scan", step)
    lm = model.NestedGDN2ForCausalLM(model.ModelConfig(
        vocab_size=20, hidden_size=16, num_hidden_layers=2, num_heads=2, head_dim=8,
        recurrent_layers=(0, 1)))
    logits, states = lm.prefill(torch.zeros(1, 4, dtype=torch.long))
    assert logits.requires_grad and states[0].requires_grad
    assert not lm.step(torch.zeros(1, dtype=torch.long), states).requires_grad
    block = lm.layers[0]
    assert not block.step(torch.zeros(1, 16), states[0]).requires_grad
    assert not block.attn.step(torch.zeros(1, 16), states[0]).requires_grad


def test_recurrent_layer_gradients_where_nothing_decays():
    """A gate so far shut that softplus gives zero: no input, no gradient, no NaN."""
    layer = model.GatedRecurrence(model.ModelConfig(hidden_size=16, num_heads=2, head_dim=8))
    with torch.no_grad():
        layer.f_proj[1].weight.zero_()
        layer.dt_bias[:4] = -200.0
        layer.dt_bias[4:8] = -100.0
        layer.v_proj.weight.normal_()
    x = torch.randn(2, 3, 16, requires_grad=True)
    v, g = layer._inputs(x)
    assert bool((v[..., :4] == 0).all()) and bool((g[..., :4] == 0).all())
    want = layer.v_proj(x) * torch.sqrt(-torch.expm1(2.0 * g))
    assert torch.equal(v, want)
    (v.square().sum() + v.sum() + g.sum()).backward()
    for t in (x, layer.dt_bias, layer.A_log, layer.f_proj[0].weight, layer.v_proj.weight):
        assert bool(torch.isfinite(t.grad).all())
