"""Memory that the feature operators ask for: no GPU needed."""
import pytest

from nerfacc_amd.cuda import _backend


@pytest.mark.parametrize("states", [1, 4, 16, 17, 32, 64, 100, 128, 256])
@pytest.mark.parametrize("rays,rows,channels", [(1, 1 << 15, 1024), (4096, 1 << 18, 64), (16, 1 << 16, 2048), (3, 3000, 70)])
def test_the_backward_scan_needs_no_more_than_the_forward_kept(states, rays, rows, channels):
    """partial sums of dB and dC grow with channels x states, as the kept states do, never with states squared; sums over rows and the
    chunks' states are a fraction of a row's states for each chunk or wave, of at least 32 rows"""
    L = _backend.load_library()
    kept, ws = L.nfa_selective_scan_checkpoint_bytes(rows, channels, states), L.nfa_selective_scan_workspace_bytes(rays, rows, channels, states, 1)
    padded, whole = max(4, 1 << (states - 1).bit_length()), -(-channels // 64) * 64          # places of the states; channels in whole waves
    chunks = rows / 32 + rays + 1
    joins = max(kept * padded / states * whole / channels, rows * 2 * padded * 4)
    assert ws <= joins + chunks * (states + 1) * channels * 4 + min(chunks, 32768) * (states + 2) * channels * 4 + 4096
