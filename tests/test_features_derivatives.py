"""Derivatives that the feature operators do not have are refused before anything else: no GPU needed."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

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


def calls():
    x, bc, A = torch.rand(2, 8), torch.rand(2, 4), torch.rand(8, 4)
    conv, scan = dict(inputs=x[None], weight=torch.rand(8, 4), bias=torch.rand(8)), dict(inputs=x, delta=x, A=A, B=bc, C=bc, D=A[:, 0], gate=x, delta_bias=A[:, 1])
    batched = {k: v[None] if k in ("inputs", "delta", "B", "C", "gate") else v for k, v in scan.items()}
    return [(nerfacc.linear, dict(inputs=x, weight=torch.rand(3, 8), bias=torch.rand(3), residual=torch.rand(2, 3))),
            (nerfacc.causal_conv, dict(**conv, initial_state=torch.rand(1, 3, 8))),
            (nerfacc.causal_conv_step, dict(**{**conv, "inputs": x}, state=torch.rand(2, 3, 8))),
            (nerfacc.selective_scan, dict(**batched, initial_state=torch.rand(1, 8, 4))),
            (nerfacc.selective_scan_step, dict(**scan, state=torch.rand(2, 8, 4)))]


def test_forward_mode_is_refused(face):
    """every tensor of every operator: the output would have no tangent"""
    for call, kw in calls():
        for k in kw:
            with fwd.dual_level():
                dual = {**kw, k: fwd.make_dual(kw[k], torch.ones_like(kw[k]))}
                with pytest.raises(NotImplementedError, match="forward mode"):
                    call(**dual)
                with pytest.raises(RuntimeError, match="no CPU kernels"):
                    call(**kw)                                           # without a tangent the call goes on, to the device's refusal
                with fwd._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="no CPU kernels"):
                    call(**dual)                                         # and with tangents switched off


def test_a_captured_training_step_needs_the_extension(monkeypatch):
    """a capture beside an eager graph of the same leaves ends the process; the ctypes face cannot tell whether there is one"""
    from nerfacc_amd import dense

    x, w = torch.rand(2, 8), torch.rand(3, 8, requires_grad=True)
    monkeypatch.setattr(dense._C, "foreign_nodes", _backend._CtypesC.foreign_nodes)
    monkeypatch.setattr(dense, "_capturing", lambda tensors: True)
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        dense._records_grad("linear", x, w, None)
    assert not dense._records_grad("linear", x, w.detach(), None)
    with torch.no_grad():
        assert not dense._records_grad("linear", x, w, None)
    monkeypatch.setattr(dense, "_capturing", lambda tensors: False)
    assert dense._records_grad("linear", x, w, None)
