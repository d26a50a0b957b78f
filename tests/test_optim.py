"""Muon on the host, with the orthogonalisation replaced by plain operations:
what a checkpoint keeps."""

import copy

import pytest
import torch

from nested_recurrent_memory_b200 import optim
from nested_recurrent_memory_b200.optim import Muon


@pytest.fixture(autouse=True)
def plain_orthogonalize(monkeypatch):
    def plain(update, steps=5, dtype=None):
        X = update.double()
        X = X / (torch.linalg.matrix_norm(X, keepdim=True) + 1e-7)
        for _ in range(steps):
            A = X @ X.mT
            X = 3.4445 * X + (-4.7750 * A + 2.0315 * A @ A) @ X
        return X.to(dtype or update.dtype)

    monkeypatch.setattr(optim, "orthogonalize", plain)


def _step(opt, params, seed):
    gen = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen).to(p.dtype)
    opt.step()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_checkpoint_keeps_fp32_momenta(dtype, tmp_path):
    """Training goes on from a checkpoint bit for bit as without it."""
    gen = torch.Generator().manual_seed(0)
    make = lambda: [torch.nn.Parameter(torch.zeros(*s, dtype=dtype)) for s in ((8, 6), (8, 6), (2, 5, 7))]  # noqa: E731
    params, resumed = make(), make()
    with torch.no_grad():
        for p in params:
            p.copy_(torch.randn(p.shape, generator=gen))
    opt = Muon([dict(params=params[:1], lr=0.1), dict(params=params[1:])], momentum=0.9)
    for i in range(3):
        _step(opt, params, i)
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    with torch.no_grad():
        for p, q in zip(resumed, params):
            p.copy_(q)
    again = Muon([dict(params=resumed[:1]), dict(params=resumed[1:])])
    saved = torch.load(tmp_path / "opt.pt")
    before = copy.deepcopy(saved)
    again.load_state_dict(saved)
    for p, q in zip(resumed, params):
        m = again.state[p]["momentum"]
        assert m.dtype == torch.float32 and torch.equal(m, opt.state[q]["momentum"])
    for i in range(3, 6):
        _step(opt, params, i)
        _step(again, resumed, i)
        assert all(torch.equal(p, q) for p, q in zip(resumed, params))
    for i, state in before["state"].items():  # the loaded dict is not written to
        assert torch.equal(state["momentum"], saved["state"][i]["momentum"])


def test_a_checkpoint_of_sixteen_bit_momenta_goes_on_in_fp32():
    p = torch.nn.Parameter(torch.ones(4, 4, dtype=torch.bfloat16))
    opt = Muon([p])
    _step(opt, [p], 0)
    state = opt.state_dict()
    state["state"][0]["momentum"] = state["state"][0]["momentum"].bfloat16()
    opt.load_state_dict(state)
    assert opt.state[p]["momentum"].dtype == torch.float32


def test_a_checkpoint_before_the_first_step():
    p = torch.nn.Parameter(torch.ones(4, 4))
    opt = Muon([p], lr=0.5)
    other = Muon([p])
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["lr"] == 0.5 and not other.state
