"""What the embedding, gated recurrence and orthogonalisation refuse, on the
host: argument checks of the Python entry points and return codes of the
C ABI with dummy pointers. No kernel is launched."""

import ctypes

import pytest
import torch

from nested_recurrent_memory_b200 import (_lib, embed_tokens, embed_tokens_bwd, embed_tokens_fwd,
                                          gated_scan, gated_scan_bwd, gated_scan_fwd,
                                          orthogonalize, step_gated_scan)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _fill(a, pointers, **over):
    a.abi_version = _lib.ABI_VERSION
    for name in pointers:
        setattr(a, name, 0x1000)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _embed(**over):
    return _fill(_lib.EmbedArgs(), ("ids", "weight", "out", "status"),
                 **{**dict(N=4, V=10, D=8, weight_stride=8), **over})


def _embed_bwd(**over):
    return _fill(_lib.EmbedBwdArgs(), ("ids", "d_out", "dweight", "status"),
                 **{**dict(N=4, V=10, D=8, d_stride=8, padding_idx=-1), **over})


def _scan(**over):
    return _fill(_lib.ScanArgs(), ("x", "g", "h", "status"), **{**dict(B=2, T=300, D=8), **over})


def _orth(**over):
    a = _fill(_lib.OrthArgs(), ("update", "out", "status"),
              **{**dict(batch=2, rows=40, cols=50, steps=5, eps=1e-7), **over})
    if "coef" not in over:
        a.coef[0], a.coef[1], a.coef[2] = 3.4445, -4.7750, 2.0315
    return a


@pytest.mark.parametrize(("over", "code"), [
    (dict(abi_version=99), -13), (dict(dtype=5), -8), (dict(D=0), -7), (dict(V=0), -7),
    (dict(N=-1), -7), (dict(ids=None), -9), (dict(weight=None), -9), (dict(out=None), -9),
    (dict(status=None), -9)])
def test_embed_codes(lib, over, code):
    assert lib.ngdn2_embed(ctypes.byref(_embed(**over)), None) == code


@pytest.mark.parametrize(("over", "code"), [
    (dict(abi_version=99), -13), (dict(dtype=5), -8), (dict(out_dtype=-1), -8), (dict(D=0), -7),
    (dict(V=0), -7), (dict(d_out=None), -9), (dict(dweight=None), -9), (dict(status=None), -9)])
def test_embed_bwd_codes(lib, over, code):
    n = ctypes.c_size_t(0)
    a = _embed_bwd(**over)
    assert lib.ngdn2_embed_bwd_workspace_size(ctypes.byref(a), ctypes.byref(n)) == code
    assert lib.ngdn2_embed_bwd(ctypes.byref(a), None) == code


@pytest.mark.parametrize(("over", "code"), [
    (dict(abi_version=99), -13), (dict(x_dtype=5), -8), (dict(g_dtype=3), -8), (dict(B=0), -7),
    (dict(T=0), -7), (dict(D=0), -7), (dict(x=None), -9), (dict(g=None), -9), (dict(h=None), -9),
    (dict(status=None), -9)])
def test_scan_codes(lib, over, code):
    assert lib.ngdn2_scan(ctypes.byref(_scan(**over)), None) == code


def test_scan_bwd_codes(lib):
    def make(fwd=None, **over):
        a = _lib.ScanBwdArgs()
        a.fwd = _scan(carries=0x1000, **(fwd or {}))
        return _fill(a, ("d_h", "dx", "dg", "status"), **over)

    for fwd, over, code in ((None, dict(abi_version=1), -13), (dict(x_dtype=9), {}, -8),
                            (None, dict(d_h_dtype=1), -8), (dict(T=0), {}, -7),
                            (dict(carries=None), {}, -9), (None, dict(dx=None), -9),
                            (None, dict(status=None), -9)):
        if fwd and "carries" in fwd:
            a = make(**over)
            a.fwd.carries = None
        else:
            a = make(fwd, **over)
        assert lib.ngdn2_scan_bwd(ctypes.byref(a), None) == code


def test_scan_step_codes(lib):
    def make(**over):
        return _fill(_lib.ScanStepArgs(), ("x", "g", "state_in", "state_out", "h"),
                     **{**dict(B=2, D=8), **over})

    for over, code in ((dict(abi_version=1), -13), (dict(x_dtype=7), -8), (dict(B=0), -7),
                       (dict(state_in=None), -9), (dict(h=None), -9)):
        assert lib.ngdn2_scan_step(ctypes.byref(make(**over)), None) == code


@pytest.mark.parametrize(("over", "code"), [
    (dict(abi_version=99), -13), (dict(dtype=5), -8), (dict(out_dtype=4), -8), (dict(rows=0), -7),
    (dict(cols=0), -7), (dict(batch=0), -7), (dict(steps=-1), -7), (dict(eps=-1.0), -7),
    (dict(eps=float("nan")), -7), (dict(coef=(ctypes.c_float * 3)(9.0, 0.0, 0.0)), -15),
    (dict(coef=(ctypes.c_float * 3)(float("nan"), 0.0, 0.0)), -15), (dict(update=None), -9),
    (dict(out=None), -9), (dict(status=None), -9)])
def test_orth_codes(lib, over, code):
    n = ctypes.c_size_t(0)
    a = _orth(**over)
    assert lib.ngdn2_orth_workspace_size(ctypes.byref(a), ctypes.byref(n)) == code
    assert lib.ngdn2_orth(ctypes.byref(a), None) == code


def test_workspaces_are_required(lib):
    n = ctypes.c_size_t(0)
    assert lib.ngdn2_orth_workspace_size(ctypes.byref(_orth()), ctypes.byref(n)) == 0 and n.value > 0
    assert lib.ngdn2_orth(ctypes.byref(_orth()), None) == -10
    assert lib.ngdn2_orth(ctypes.byref(_orth(workspace=0x1000, workspace_bytes=n.value - 1)), None) == -10
    assert "coefficients" in _lib.error_string(_lib.ERR_COEFFICIENTS)


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros(2, 3, 8), torch.zeros(4, dtype=torch.long)
    for call in (lambda: embed_tokens_fwd(ids, torch.zeros(5, 8)),
                 lambda: embed_tokens(ids, torch.zeros(5, 8)),
                 lambda: embed_tokens_bwd(ids, torch.zeros(4, 8), 5),
                 lambda: gated_scan_fwd(x, x), lambda: gated_scan(x, x),
                 lambda: gated_scan_bwd(x, x, x), lambda: step_gated_scan(x[0], x[0], x[0]),
                 lambda: orthogonalize(x)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_shapes_are_refused():
    x, ids = torch.zeros(2, 3, 8), torch.zeros(4, dtype=torch.long)
    with pytest.raises(ValueError, match=r"\[V, D\]"):
        embed_tokens_fwd(ids, torch.zeros(5))
    with pytest.raises(ValueError, match=r"\[\*ids.shape, D\]"):
        embed_tokens_bwd(ids, torch.zeros(5, 8), 5)
    with pytest.raises(ValueError, match="padding_idx"):
        embed_tokens(ids, torch.zeros(5, 8), padding_idx=5)
    for fn in (gated_scan_fwd, gated_scan):
        with pytest.raises(ValueError, match=r"\[B, T, D\]"):
            fn(x, x[:, :2])
        with pytest.raises(ValueError, match=r"\[B, T, D\]"):
            fn(x[0], x[0])
    with pytest.raises(ValueError, match=r"\[B, D\]"):
        step_gated_scan(x, x, x)
    with pytest.raises(ValueError, match="rows, cols"):
        orthogonalize(torch.zeros(5))


def test_scratch_memory_is_checked():
    """Workspaces of another device or with gaps never reach a kernel."""
    from nested_recurrent_memory_b200.ops import _scratch

    cpu, need = torch.device("cpu"), 100
    own = torch.empty(200, dtype=torch.uint8)
    assert _scratch(need, own, cpu) is own
    assert _scratch(need, torch.empty(50), cpu).dtype == torch.float32  # 200 bytes
    assert _scratch(need, own[:99], cpu).numel() == need and _scratch(0, own, cpu) is None
    for bad in (own.to("meta"), own[::2], torch.empty(1, dtype=torch.uint8).expand(200)):
        with pytest.raises(ValueError, match="workspace"):
            _scratch(need, bad, cpu)


@pytest.mark.parametrize(("bits", "named", "not_named"), [
    (_lib.STATUS_WAIT_TIMEOUT, ("recurrence", "orthogonalisation", "nested GDN-2 forward", "wait"), ("embedding",)),
    (_lib.STATUS_GATE_TIMEOUT, ("nested GDN-2 forward", "start gate"), ("recurrence", "embedding")),
    (_lib.STATUS_BAD_INDEX, ("embedding", "token id"), ("nested", "wait"))])
def test_status_errors_name_the_calls_that_can_set_them(bits, named, not_named):
    """The word is shared: an error does not blame a forward that did not run."""
    from nested_recurrent_memory_b200 import KernelStatusError
    from nested_recurrent_memory_b200.ops import _DeviceStatus

    st = _DeviceStatus.__new__(_DeviceStatus)
    st.word = st.host = torch.full((1,), bits, dtype=torch.int32)
    with pytest.raises(KernelStatusError) as e:
        st._raise_if_set(bits)
    assert all(n in str(e.value) for n in named) and not any(n in str(e.value) for n in not_named)
    assert int(st.word) == 0
