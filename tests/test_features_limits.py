"""Sizes that the feature operators refuse: no GPU and no memory needed."""
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


@pytest.mark.parametrize("n", [(1 << 23) + 1, (1 << 32) + 8])
def test_too_many_features_and_channels_are_refused(face, n):
    """never cut off to the low 32 bits of their number"""
    wide = lambda *shape: torch.empty(1).expand(shape)  # noqa: E731
    for call in (lambda: nerfacc.linear(wide(1, n), wide(1, n)), lambda: nerfacc.linear(wide(1, 1), wide(n, 1)),
                 lambda: nerfacc.causal_conv(wide(1, 1, n), wide(n, 4)), lambda: nerfacc.causal_conv_step(wide(1, n), wide(1, 3, n), wide(n, 4)),
                 lambda: nerfacc.selective_scan(wide(1, 1, n), wide(1, 1, n), wide(n, 1), wide(1, 1, 1), wide(1, 1, 1)),
                 lambda: nerfacc.selective_scan_step(wide(1, n), wide(1, n), wide(n, 1), wide(1, 1), wide(1, 1), wide(1, n, 1))):
        with pytest.raises(ValueError, match="more than 2"):
            call()


def test_a_weight_gradient_of_more_numbers_than_one_launch_joins_is_refused():
    """through the C ABI, before anything is launched"""
    import ctypes

    L, p = _backend.load_library(), 4096                             # (never followed)
    a = _backend._STRUCTS["nfa_linear_args"](rows=1, in_features=1 << 16, out_features=1 << 16, dtype=1, activation=0, inputs=p, inputs_stride=1 << 16, weight=p,
                                             grad_outputs=p, grad_outputs_stride=1 << 16)
    assert L.nfa_linear_bwd(ctypes.byref(a), None, None, p, None, p, None) == 1
    assert b"too many weights" in L.nfa_last_error()
