"""Refusals of the feature operators (linear, causal_conv, selective_scan and their one-row forms), which need no GPU, and the C ABI's own
checks, which come before any launch."""
import ctypes

import pytest
import torch

import nerfacc_amd as nerfacc
from nerfacc_amd.cuda import _backend


@pytest.fixture(params=["extension", "python"])
def face(request, monkeypatch):
    """the operators as one call of the extension, and as the Python steps of the ctypes face"""
    from nerfacc_amd import dense

    if request.param == "python":
        monkeypatch.setattr(dense, "_EXT", False)
    elif _backend.BACKEND != "ext":
        pytest.skip("torch extension not the active backend")


def test_arguments_are_refused_before_the_device_is_asked_for(face):
    x, w = torch.rand(4, 8), torch.rand(8, 4)
    info = torch.tensor([[0, 4]])
    with pytest.raises(ValueError):
        nerfacc.linear(x, w.t()[:, :3])
    with pytest.raises(ValueError):
        nerfacc.linear(x, torch.rand(3, 8), activation="tanh")
    with pytest.raises(ValueError):
        nerfacc.linear(x, torch.rand(0, 8))
    with pytest.raises(TypeError):
        nerfacc.linear(x.numpy(), w)
    for bad in (dict(inputs=x), dict(inputs=x[None], packed_info=info), dict(inputs=x, packed_info=info[0]), dict(inputs=x, packed_info=info.t()[:1]),
                dict(inputs=x[:, :0], packed_info=info), dict(inputs=x, packed_info=info, activation="relu"),
                dict(inputs=x, packed_info=info, weight=torch.rand(8, 5)), dict(inputs=x, packed_info=info, weight=torch.rand(8, 1)),
                dict(inputs=x, packed_info=info, weight=torch.rand(7, 4))):
        with pytest.raises(ValueError):
            nerfacc.causal_conv(**{"weight": w, **bad})
    A, bc = torch.rand(8, 3), torch.rand(4, 3)
    for bad in (dict(A=A[0]), dict(A=torch.rand(8, 257)), dict(A=A[:, :0])):
        with pytest.raises(ValueError):
            nerfacc.selective_scan(**{"inputs": x, "delta": x, "A": A, "B": bc, "C": bc, "packed_info": info, **bad})
    with pytest.raises(TypeError):
        nerfacc.selective_scan(x, None, A, bc, bc, packed_info=info)
    with pytest.raises(ValueError):
        nerfacc.selective_scan_step(x[0], x, A, bc, bc, torch.rand(4, 8, 3))
    with pytest.raises(TypeError):
        nerfacc.causal_conv_step(x, None, w)


def test_host_tensors_are_refused(face):
    x, w, info = torch.rand(4, 8), torch.rand(8, 4), torch.tensor([[0, 4]])
    A, bc = torch.rand(8, 3), torch.rand(4, 3)
    for call in (lambda: nerfacc.linear(x, torch.rand(3, 8)), lambda: nerfacc.causal_conv(x, w, packed_info=info),
                 lambda: nerfacc.causal_conv_step(x, torch.rand(4, 3, 8), w), lambda: nerfacc.selective_scan(x, x, A, bc, bc, packed_info=info),
                 lambda: nerfacc.selective_scan_step(x, x, A, bc, bc, torch.rand(4, 8, 3))):
        with pytest.raises(RuntimeError, match="no CPU kernels"):
            call()


def _error(rc):
    assert rc == 1                                                       # NFA_ERR_INVALID_ARG
    return _backend.load_library().nfa_last_error().decode()


def test_the_c_abi_checks_before_it_launches():
    L, S = _backend.load_library(), _backend._STRUCTS
    p = 4096                                                             # (never followed: every call is refused first)
    good = dict(rows=4, in_features=8, out_features=8, dtype=1, activation=1, inputs=p, inputs_stride=8, weight=p, grad_outputs=p, grad_outputs_stride=8)
    for bad, text in ((dict(rows=-1), "bad size"), (dict(in_features=0), "bad size"), (dict(dtype=3), "dtype"), (dict(activation=9), "activation"),
                      (dict(inputs=None), "NULL"), (dict(inputs_stride=7), "inputs_stride"), (dict(in_features=1 << 21), "2^20"),
                      (dict(residual=p, residual_stride=3), "residual_stride")):
        assert text in _error(L.nfa_linear_fwd(ctypes.byref(S["nfa_linear_args"](**{**good, **bad})), p, None, None))
    a = S["nfa_linear_args"](**good)
    assert "NULL" in _error(L.nfa_linear_fwd(None, p, None, None)) and "NULL" in _error(L.nfa_linear_fwd(ctypes.byref(a), None, None, None))
    assert "saved" in _error(L.nfa_linear_bwd(ctypes.byref(a), None, p, p, p, p, None))
    assert "workspace" in _error(L.nfa_linear_bwd(ctypes.byref(a), p, p, p, p, None, None))
    assert L.nfa_linear_saved_bytes(10, 8, 1, 0, 1) == 0 and L.nfa_linear_saved_bytes(10, 8, 1, 6, 0) == 0 and L.nfa_linear_saved_bytes(10, 8, 1, 4, 0) == 160
    assert [L.nfa_linear_saved_bytes(10, n, t, 1, r) for n, t, r in ((16, 1, 1), (16, 0, 0), (9, 1, 0), (9, 1, 1))] == [20, 40, 0, 180]     # relu: bits
    good = dict(n_rays=2, rows=4, channels=8, width=4, dtype=0, activation=4, inputs=p, inputs_stride=8, weight=p, grad_outputs=p, grad_outputs_stride=8)
    for bad, text in ((dict(width=5), "width"), (dict(width=1), "width"), (dict(rows=5), "equal sequences"), (dict(packed_info=p), "row map"),
                      (dict(activation=1), "activation"), (dict(inputs_stride=2), "inputs_stride"), (dict(weight=None), "NULL"),
                      (dict(rows=1 << 31), "2^31"), (dict(n_rays=0), "without sequences")):
        assert text in _error(L.nfa_causal_conv_fwd(ctypes.byref(S["nfa_causal_conv_args"](**{**good, **bad})), p, None, None))
    a = S["nfa_causal_conv_args"](**good)
    assert "no initial state" in _error(L.nfa_causal_conv_bwd(ctypes.byref(a), p, p, p, p, p, None))
    assert "workspace" in _error(L.nfa_causal_conv_bwd(ctypes.byref(a), p, p, p, None, None, None))
    good = dict(n_rays=2, rows=4, channels=8, states=4, dtype=0, inputs=p, inputs_stride=8, delta=p, delta_stride=8, B=p, B_stride=4, C=p, C_stride=4, A=p,
                grad_outputs=p, grad_outputs_stride=8)
    for bad, text in ((dict(states=0), "states"), (dict(states=257), "states"), (dict(B_stride=3), "stride"), (dict(gate=p, gate_stride=1), "stride"),
                      (dict(A=None), "NULL"), (dict(rows=3), "equal sequences"), (dict(packed_info=p), "row map")):
        assert text in _error(L.nfa_selective_scan_fwd(ctypes.byref(S["nfa_selective_scan_args"](**{**good, **bad})), p, None, None, p, None))
    a = S["nfa_selective_scan_args"](**good)
    assert "NULL" in _error(L.nfa_selective_scan_bwd(ctypes.byref(a), p, None, p, None))
    assert "NULL" in _error(L.nfa_selective_scan_step(ctypes.byref(a), None, p, p, None))
    assert "negative" in _error(L.nfa_row_map(p, -1, 4, p, p, None)) and L.nfa_row_map(None, 0, 0, None, None, None) == 0


def test_workspaces_cover_both_layouts():
    """one size serves packed and equal sequences, and every vector width"""
    L = _backend.load_library()
    assert L.nfa_selective_scan_workspace_bytes(4096, 1 << 18, 64, 16, 0) == 0                      # whole rays: nothing to chain
    assert L.nfa_selective_scan_workspace_bytes(1, 1 << 15, 1024, 16, 0) >= 2 * 1024 * 17 * 4
    assert L.nfa_selective_scan_checkpoint_bytes(17, 3, 5) == 3 * 3 * 5 * 4
    assert L.nfa_causal_conv_bwd_workspace_bytes(0, 8, 4, 1) == 0 and L.nfa_linear_bwd_workspace_bytes(0, 8, 8, 1, 0) == 0
