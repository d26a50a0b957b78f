"""The memory that a caller hands to the embedding, the recurrence and the
orthogonalisation beside their inputs: workspaces and the forward's states."""

import pytest
import torch

from nested_recurrent_memory_b200 import (embed_tokens_bwd, gated_scan_bwd, gated_scan_fwd,
                                          orthogonalize)

pytestmark = pytest.mark.gpu


def _calls():
    ids = torch.arange(40, device="cuda") % 7
    d = torch.randn(40, 12, device="cuda")
    x, g = torch.randn(2, 300, 36, device="cuda"), -torch.rand(2, 300, 36, device="cuda")
    G = torch.randn(2, 130, 140, device="cuda")
    return (lambda ws: embed_tokens_bwd(ids, d, 7, workspace=ws),
            lambda ws: gated_scan_fwd(x, g, workspace=ws)[0],
            lambda ws: gated_scan_bwd(x, g, x, workspace=ws)[1],
            lambda ws: orthogonalize(G, workspace=ws))


def test_workspaces_are_used_or_replaced():
    for call in _calls():
        ref = call(None)
        for ws in (torch.empty(1 << 22, dtype=torch.uint8, device="cuda"),
                   torch.empty(1 << 20, dtype=torch.float32, device="cuda"),
                   torch.empty(8, dtype=torch.uint8, device="cuda")):
            assert torch.equal(call(ws), ref)


def test_workspaces_elsewhere_or_with_gaps_are_refused():
    """Host memory, and views whose memory is smaller than their extent."""
    one = torch.empty(1, dtype=torch.uint8, device="cuda")
    for call in _calls():
        for ws in (torch.empty(1 << 22, dtype=torch.uint8), one.expand(1 << 22)):
            with pytest.raises(ValueError, match="workspace"):
                call(ws)


def test_forward_states_elsewhere_are_refused():
    x, g = torch.randn(2, 300, 36, device="cuda"), -torch.rand(2, 300, 36, device="cuda")
    carries = gated_scan_fwd(x, g, return_aux=True)[2]["carries"]
    ref = gated_scan_bwd(x, g, x, aux=dict(carries=carries))
    assert all(torch.equal(p, q) for p, q in zip(ref[:2], gated_scan_bwd(x, g, x)[:2]))
    for bad in (carries.cpu(), carries.double(), carries[:, :2], carries.mT.contiguous().mT):
        with pytest.raises(ValueError, match="aux"):
            gated_scan_bwd(x, g, x, aux=dict(carries=bad))
