"""Calls of the feature operators at the edge of what their documentation allows: rays that overlap, values at the ends of their types'
ranges, derivatives that are refused."""
import pytest
import torch

from gpu_utils import DEV

pytestmark = pytest.mark.gpu


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=generator(seed), device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_conv_rays_that_overlap_leave_the_others_right(dtype):
    """rows claimed by a long and a short ray belong to either; the final state's gradient is added to rows of a ray only, so the rays that
    share no rows get what they get alone"""
    import nerfacc_amd as nerfacc

    info = torch.tensor([[0, 100], [0, 2], [40, 1], [100, 30]], device=DEV)
    x, w, gy, gf = normal(130, 24, dtype=dtype), normal(24, 4, seed=1, dtype=dtype), normal(130, 24, seed=2, dtype=dtype), normal(4, 3, 24, seed=3, dtype=dtype)

    def grad(x, gy, gf, info):
        x = x.clone().requires_grad_(True)
        out, last = nerfacc.causal_conv(x, w, activation="silu", packed_info=info, return_final_state=True)
        return torch.autograd.grad([out, last], x, [gy, gf])[0]

    got = grad(x, gy, gf, info)
    torch.cuda.synchronize()
    assert got.shape == x.shape
    assert torch.equal(got[100:], grad(x[100:], gy[100:], gf[3:], torch.tensor([[0, 30]], device=DEV)))
