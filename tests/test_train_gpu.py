"""The embedding, the recurrence and the orthogonalised updates together: a
model's loss and gradients against the same model on plain torch operations, a
few training steps, decoding token by token against one pass, and the
optimiser's step against its formula."""

import pathlib
import sys

import pytest
import torch
import torch.nn.functional as F

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "examples"))

import train_hybrid_lm  # noqa: E402
from nested_recurrent_memory_b200 import model as model_module  # noqa: E402
from nested_recurrent_memory_b200.model import ModelConfig, NestedGDN2ForCausalLM  # noqa: E402
from nested_recurrent_memory_b200.optim import Muon, split_parameters  # noqa: E402

pytestmark = pytest.mark.gpu


def plain_scan(x, g, initial_state=None, output_final_state=False):
    h = torch.zeros_like(x[:, 0], dtype=torch.float32) if initial_state is None else initial_state
    out = []
    for t in range(x.shape[1]):
        h = g[:, t].float().exp() * h + x[:, t].float()
        out.append(h.to(x.dtype))
    return torch.stack(out, 1), h


def plain_embed(ids, weight, scale=1.0, padding_idx=None):
    return F.embedding(ids, weight) * scale


def _recurrent_model(layers=2, **kw):
    cfg = ModelConfig(vocab_size=300, hidden_size=128, num_hidden_layers=layers, num_heads=2,
                      head_dim=64, embed_scale=11.0, recurrent_layers=tuple(range(layers)), **kw)
    return NestedGDN2ForCausalLM(cfg).cuda()


def test_gradients_match_plain_operations(monkeypatch):
    """fp32 throughout: the two differ by the order of fp32 sums, 1e-4 of each
    gradient's norm over this depth."""
    torch.manual_seed(0)
    model = _recurrent_model()
    ids = torch.randint(0, 300, (3, 71), device="cuda")

    def run():
        model.zero_grad(set_to_none=True)
        loss = F.cross_entropy(model(ids[:, :-1]).flatten(0, 1), ids[:, 1:].flatten())
        loss.backward()
        return loss.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}

    loss, grads = run()
    monkeypatch.setattr(model_module, "gated_scan", plain_scan)
    monkeypatch.setattr(model_module, "embed_tokens", plain_embed)
    ref_loss, ref = run()
    assert abs(float(loss - ref_loss)) < 1e-5 * abs(float(ref_loss))
    for n in ref:
        assert float((grads[n] - ref[n]).norm()) <= 1e-4 * float(ref[n].norm()) + 1e-12, n


@pytest.mark.parametrize("nested", [False, True])
def test_training_lowers_the_loss(nested):
    _, losses = train_hybrid_lm.train(steps=12, nested=nested, B=4, T=128, log=None)
    assert all(x == x for x in losses)
    assert losses[-1] < losses[0] - 0.5


def test_decoding_token_by_token_matches_one_pass():
    torch.manual_seed(1)
    model = _recurrent_model().eval()
    ids = torch.randint(0, 300, (2, 40), device="cuda")
    with torch.no_grad():
        full, _ = model.prefill(ids)
        assert torch.equal(full, model(ids))
        logits, states = model.prefill(ids[:, :31])
        assert torch.allclose(logits, full[:, :31], rtol=1e-4, atol=1e-5)
        for t in range(31, 40):
            assert torch.allclose(model.step(ids[:, t], states), full[:, t], rtol=1e-4, atol=1e-5)


def test_nested_layers_do_not_decode_here():
    cfg = ModelConfig(vocab_size=64, hidden_size=128, num_hidden_layers=2, num_heads=2, head_dim=64,
                      recurrent_layers=(1,))
    model = NestedGDN2ForCausalLM(cfg).cuda()
    with pytest.raises(ValueError, match="recurrent_layers"):
        model.prefill(torch.zeros(1, 4, dtype=torch.long, device="cuda"))


def test_muon_follows_its_formula():
    """Two steps of Muon on matrices of two shapes and a stack: the momentum
    exactly, the orthogonalised update to bf16's unit."""
    gen = torch.Generator().manual_seed(2)
    shapes = [(48, 32), (48, 32), (20, 60), (2, 3, 16, 24)]
    ps = [torch.nn.Parameter(torch.randn(*s, generator=gen).cuda()) for s in shapes]
    want = [p.detach().double().clone() for p in ps]
    bufs = [torch.zeros_like(w) for w in want]
    opt = Muon(ps, lr=0.1, momentum=0.9, weight_decay=0.01)
    for _ in range(2):
        for i, p in enumerate(ps):
            p.grad = torch.randn(*p.shape, generator=gen).cuda()
            bufs[i] = 0.9 * bufs[i] + p.grad.double()
            X = p.grad.double() + 0.9 * bufs[i]
            X = X / (torch.linalg.matrix_norm(X, keepdim=True) + 1e-7)
            for _ in range(5):
                A = X @ X.transpose(-1, -2)
                X = 3.4445 * X + (-4.7750 * A + 2.0315 * A @ A) @ X
            m, n = p.shape[-2:]
            want[i] = want[i] * (1 - 0.1 * 0.01) - 0.1 * max(1.0, m / n) ** 0.5 * X
        opt.step()
        for p, w, s in zip(ps, want, shapes):
            assert float((p.detach().double() - w).abs().max()) <= 2 * 0.1 * 1.3 * 1.25 * 2.0 ** -8


def test_split_parameters_keeps_vectors_embeddings_and_head_apart():
    model = NestedGDN2ForCausalLM(ModelConfig(vocab_size=64, hidden_size=128, num_hidden_layers=2,
                                              num_heads=2, head_dim=64, recurrent_layers=(0,)))
    matrices, rest = split_parameters(model)
    assert len(matrices) + len(rest) == len(list(model.parameters()))
    names = {id(p): n for n, p in model.named_parameters()}
    assert all(p.dim() >= 2 for p in matrices)
    kept = {names[id(p)] for p in rest}
    assert {"embeddings.weight", "lm_head.weight", "norm.weight"} <= kept
    assert all("conv1d" in n or "norm" in n or "bias" in n or "log" in n or "head" in n or "embed" in n
               for n in kept)
    assert any("key_projections" in names[id(p)] for p in matrices)


def test_the_models_embedding_takes_what_torchs_takes():
    """float64 tables (of a model with another op), and torch.func's transforms."""
    gen = torch.Generator().manual_seed(3)
    w, ids = torch.randn(12, 5, generator=gen).cuda(), torch.randint(0, 12, (4, 6), generator=gen).cuda()
    emb = model_module.ScaledEmbedding(12, 5, scale=4.0).cuda()
    with torch.no_grad():
        emb.weight.copy_(w)
    double = model_module.ScaledEmbedding(12, 5, scale=4.0).cuda().double()
    y = double(ids)
    assert y.dtype == torch.float64 and torch.equal(y, F.embedding(ids, double.weight) * 4.0)
    y.sin().sum().backward()
    assert double.weight.grad.dtype == torch.float64

    def loss(weight, one):
        return torch.func.functional_call(emb, {"weight": weight}, (one,)).sin().sum()

    each = torch.func.vmap(torch.func.grad(loss), in_dims=(None, 0))(emb.weight.detach(), ids)
    for i in range(4):
        x = emb.weight.detach().clone().requires_grad_()
        (ref,) = torch.autograd.grad((F.embedding(ids[i], x) * 4.0).sin().sum(), x)
        assert torch.allclose(each[i], ref, rtol=1e-5, atol=1e-5)
