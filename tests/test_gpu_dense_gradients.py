"""Gradients of `nerfacc_amd.linear` in 16-bit types where act' is small, where dz = dy act' leaves the type's range and where sums cancel.

What the backward pass may lose, with u = eps / 2 of the type:
  * every result is rounded once: u |result|, and half a smallest step of fp16;
  * act' is formed in 32 bits from z in 32 bits.  fp32 and fp16 keep 32 bits (fp32: z or the value, which lose as little); bf16 keeps act'
    rounded once, or differentiates from its own output: u |dz| a term;
  * None and relu multiply dy itself; the others take dz in two parts of bf16, the rest below 2^-17 |dz|, and inputs and weights of fp16 in
    two parts whose second product with the second part of dz, 2^-18 of the term, is left out: 2^-16 |term| with room for both;
  * sums of n terms in 32 bits: n 2^-24 sum |terms| (256 terms a lane and one more rounding per partial sum on the rows' axis).
The error of act' in 32 bits is at most 16 (1 + |z| + z^2) 2^-24 of the sizes of its parts (an exponential of z log2 e, or of z^2 / 2, behind it), plus
|act''| times the error of z, (k + 4) 2^-24 sum |terms| of z."""
import math

import pytest
import torch

from gpu_utils import DEV

pytestmark = pytest.mark.gpu

SMOOTH = ["sigmoid", "softplus", "silu", "gelu", "exp"]
HALF = [torch.bfloat16, torch.float16]


def parts(act, z):
    """act'(z) in 64 bits, the sum of its parts' sizes, |act''(z)|"""
    s, t = torch.sigmoid(z), torch.sigmoid(-z)
    if act is None or act == "relu":
        one = torch.ones_like(z) if act is None else (z > 0).to(z.dtype)
        return one, one, torch.zeros_like(z)
    if act == "exp":
        return z.exp(), z.exp(), z.exp()
    if act == "sigmoid":
        return s * t, s * t, (s * t * (t - s)).abs()
    if act == "softplus":
        return s, s, s * t
    if act == "silu":
        return s * (1 + z * t), s * (1 + z.abs() * t), (s * t * (2 + z * (t - s))).abs()
    phi, cdf = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi), 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return cdf + z * phi, cdf + z.abs() * phi, phi * (2 - z * z).abs()


def check(x, w, b, gy, act, slope=None, only=("inputs", "weight", "bias")):
    """gradients of linear against 64 bits; slope: act' to take in place of that of the 64-bit z (what the layer itself returned)"""
    import nerfacc_amd as nerfacc

    dt, (m, k), n = x.dtype, x.shape, w.shape[0]
    u, tiny = torch.finfo(dt).eps / 2, 2.0**-25 if dt == torch.float16 else 0.0
    own = [t.detach().requires_grad_(True) for t in (x, w, b)]
    out = nerfacc.linear(*own, activation=act)
    got = torch.autograd.grad(out, own, gy)
    X, W, G = x.double(), w.double(), gy.double()
    z = X @ W.t() + b.double()
    first, size, second = parts(act, z)
    soft = act not in (None, "relu")
    if slope is not None:
        first, size, off = slope(out), torch.zeros_like(z), torch.zeros_like(z)
    else:
        off = 16 * (1 + z.abs() + z * z) * 2.0**-24 * size + second * (k + 4) * 2.0**-24 * (X.abs() @ W.t().abs() + b.double().abs()) if soft else 0 * z
        if soft and dt == torch.bfloat16:
            off = off + u * first.abs()
    dz, off = G * first, G.abs() * off
    two = 2.0**-16 if soft and dt != torch.float32 else 0.0
    join = 256 + -(-m // 256)
    for what, g, ref, mag, err, sums, lost in (("inputs", got[0], dz @ W, dz.abs() @ W.abs(), off @ W.abs(), n, two),
                                               ("weight", got[1], dz.t() @ X, dz.abs().t() @ X.abs(), off.t() @ X.abs(), join, two),
                                               ("bias", got[2], dz.sum(0), dz.abs().sum(0), off.sum(0), join, 0.0)):
        if what not in only:
            continue
        tol = u * ref.abs() + tiny + err + (lost + (sums + 8) * 2.0**-24) * mag
        miss = (g.double() - ref).abs()
        over = (ref.abs() + tol > torch.finfo(dt).max) & (g.double() == ref.sign() * math.inf)      # what the type does not hold rounds to infinity
        assert ((miss <= tol) | over | (ref.isnan() & g.isnan())).all(), (what, (miss / tol).max().item(), miss.max().item())


def normal(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


@pytest.mark.parametrize("dtype", [*HALF, torch.float32])
@pytest.mark.parametrize("act", SMOOTH)
@pytest.mark.parametrize("m,k,n", [(70, 24, 64), (70, 23, 63)])
def test_slopes_far_from_the_middle(dtype, act, m, k, n):
    """z from -20 to 8 (gelu: -6), act' down to 2e-9 under a large loss scale; the bias gradient sums dz itself"""
    x, w = normal(m, k, seed=1).to(dtype), (normal(n, k, seed=2) * 0.1 / k**0.5).to(dtype)
    b = torch.linspace(-6.0 if act == "gelu" else -20.0, 8.0, n, device=DEV).to(dtype)
    gy = (normal(m, n, seed=3).abs().double() / b.double().clamp(max=0).exp().clamp(min=2.0**-14)).to(dtype)
    check(x, w, b, gy, act, only=("bias",))


SHAPES = [(70, 24, 40), (300, 96, 256), (200, 130, 300), (5000, 64, 64), (2000, 33, 65)]


@pytest.mark.parametrize("dtype", [*HALF, torch.float32])
@pytest.mark.parametrize("act", [None, "relu", *SMOOTH])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_far_from_the_middle(dtype, act, m, k, n):
    """z from -20 to 8 (gelu: -6): act' down to 2e-9, gradients that fp16 holds"""
    lo, hi = (-6.0, 5.0) if act == "gelu" else (-20.0, 8.0)
    x = normal(m, k, seed=1).to(dtype)
    w = (normal(n, k, seed=2) * 0.2 / k**0.5).to(dtype)
    b = torch.linspace(lo, hi, n, device=DEV).to(dtype)
    small = b.double().clamp(max=0).exp() if act not in (None, "relu") else torch.ones(n, device=DEV, dtype=torch.float64)
    gy = (normal(m, n, seed=3).double() / small.clamp(min=2.0**-14)).to(dtype)           # (a large loss scale: up to 2^14 times a normal number)
    check(x, w, b, gy, act)
    if act is not None:                                                                 # one column at a time: nothing larger hides it
        j = n // 16
        only = torch.zeros_like(gy)
        only[:, j] = gy[:, j]
        check(x, w, b, only, act)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,k,n", [(4096, 64, 48), (4096, 130, 256), (4096, 200, 300), (4099, 61, 63)])
def test_sums_that_cancel_see_both_parts_of_dz(dtype, m, k, n):
    """equal rows of both signs, so that dz's roundings would all go the same way and the sum is a small part of its terms"""
    g = torch.Generator(device=DEV).manual_seed(m + n)
    x = torch.ones(m, k, device=DEV, dtype=dtype)
    x[:, 1::2] = -1
    w = (normal(n, k, seed=5) * 0.4 / k**0.5).to(dtype)
    b = (torch.rand(n, generator=g, device=DEV) * 2 - 1).to(dtype)
    gy = (1 + torch.rand(1, n, generator=g, device=DEV)).to(dtype).expand(m, n).contiguous()
    gy[m // 2:] = (-(1 + 2.0**-6) * gy[m // 2:].float()).to(dtype)
    gy[m // 2] = 0
    # exp is differentiated from its own output in bf16: no rounding of act' is in the way
    check(x, w, b, gy, "exp", slope=(lambda out: out.detach().double()) if dtype == torch.bfloat16 else None)


@pytest.mark.parametrize("slope", [0.05, 0.005, 0.0005])
def test_small_gradients_of_many_rows_in_fp16(slope):
    """the gradient of a mean over 2^18 samples: each dz is below fp16's smallest step, their sum is not"""
    m, k, n = 1 << 18, 8, 16
    x, w = torch.ones(m, k, device=DEV).half(), (normal(n, k, seed=1) * 0.01).half()
    b = torch.full((n,), math.log(slope), device=DEV).half()
    gy = torch.full((m, n), 4e-6, device=DEV).half()
    check(x, w, b, gy, "softplus")
    check(torch.zeros_like(x[:3000]), (w.float() * 1e4).half(), torch.full((n,), -6.0, device=DEV).half(), gy[:3000], "sigmoid")


@pytest.mark.parametrize("m,k,n", [(300, 24, 40), (300, 130, 300), (257, 63, 65)])
def test_large_gradients_in_fp16(m, k, n):
    """dz up to 10^8, whose products with small weights and inputs fit"""
    x, w = (normal(m, k, seed=1) * 2.0**-11).half(), (normal(n, k, seed=2) * 2.0**-11).half()
    b = torch.linspace(2.0, 9.0, n, device=DEV).half()
    gy = (normal(m, n, seed=3) * 30).half()
    gy[:, -1] = gy[:, -1] * 100
    check(x, w, b, gy, "exp")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("act", SMOOTH)
@pytest.mark.parametrize("n", [40, 300])
def test_infinite_gradients_stay_infinite(dtype, act, n):
    import nerfacc_amd as nerfacc

    x, w, b = torch.full((5, 8), 0.25, device=DEV, dtype=dtype), torch.full((n, 8), 0.5, device=DEV, dtype=dtype), torch.zeros(n, device=DEV, dtype=dtype)
    own = [t.requires_grad_(True) for t in (x, w, b)]
    gy = torch.ones(5, n, device=DEV, dtype=dtype)
    gy[1, 3], gy[2, 3], gy[4] = float("inf"), float("inf"), float("nan")
    gx, gw, gb = torch.autograd.grad(nerfacc.linear(*own, activation=act), own, gy)
    assert gx[1:3].isposinf().all() and gx[0].isfinite().all() and gx[3].isfinite().all() and gx[4].isnan().all()
    gy[4] = 1.0
    gx, gw, gb = torch.autograd.grad(nerfacc.linear(*own, activation=act), own, gy)
    assert gw[3].isposinf().all() and gb[3].isposinf() and gw[:3].isfinite().all() and gw[4:].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("m,k,n", [(6, 8, 24), (6, 8, 25), (300, 12, 32), (400, 64, 320), (400, 30, 301)])
def test_relu_passes_gradients_where_its_output_is_nan(dtype, m, k, n):
    """as torch's: only z <= 0 stops them"""
    import nerfacc_amd as nerfacc

    x, w, b, gy = (normal(*s, seed=i).to(dtype) for i, s in enumerate([(m, k), (n, k), (n,), (m, n)]))
    x[3, 2] = float("nan")
    own = [t.requires_grad_(True) for t in (x, w, b)]
    out = nerfacc.linear(*own, activation="relu")
    assert out[3].isnan().all()
    gx, _, gb = torch.autograd.grad(out, own, gy)
    mask = (out.detach().double() > 0) | out.detach().isnan()
    dz = gy.double() * mask
    for got, ref, mag in ((gx, dz @ w.double(), dz.abs() @ w.double().abs()), (gb, dz.sum(0), dz.abs().sum(0))):
        assert ((got.double() - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs() + (m + n) * 2.0**-24 * mag + 2.0**-25).all()


@pytest.mark.parametrize("n", [24, 25, 5])
@pytest.mark.parametrize("residual", [False, True])
def test_relu_passes_gradients_where_its_fp16_output_rounds_to_zero(n, residual):
    """z = 2^-26 is above 0, whatever the output keeps of it"""
    import nerfacc_amd as nerfacc

    x, w = torch.full((6, 4), 2.0**-14, device=DEV).half(), torch.full((n, 4), 2.0**-14, device=DEV).half()
    own = [t.requires_grad_(True) for t in (x, w)]
    out = nerfacc.linear(*own, activation="relu", residual=torch.zeros(6, n, device=DEV).half() if residual else None)
    assert not out.any()
    gx, _ = torch.autograd.grad(out, own, torch.full((6, n), 1024.0, device=DEV).half())
    assert torch.equal(gx, torch.full_like(gx, n / 16))


@pytest.mark.parametrize("act,dtype", [(0, 0), (0, 2), (6, 0), (3, 1), (1, 1)])
def test_saved_is_left_alone_where_nothing_is_kept(act, dtype):
    """through the C ABI: an array of 0 bytes, as nfa_linear_saved_bytes asks for, is not written to"""
    import ctypes

    from nerfacc_amd.cuda import _backend

    L, m, k, n = _backend.load_library(), 4, 8, 9
    dt = [torch.float32, torch.bfloat16, torch.float16][dtype]
    x, w, out = normal(m, k).to(dt), normal(n, k, seed=1).to(dt), torch.empty(m, n, device=DEV, dtype=dt)
    saved = torch.full((m * n * 4,), 77, device=DEV, dtype=torch.uint8)                  # (room for whatever might be written)
    a = _backend._STRUCTS["nfa_linear_args"](rows=m, in_features=k, out_features=n, dtype=dtype, activation=act, inputs=x.data_ptr(), inputs_stride=k,
                                             weight=w.data_ptr())
    assert L.nfa_linear_saved_bytes(m, n, dtype, act, 0) == 0
    assert L.nfa_linear_fwd(ctypes.byref(a), out.data_ptr(), saved.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert saved.eq(77).all()


@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("python", [False, True])
def test_a_penalty_on_the_gradient_is_refused(act, python, monkeypatch):
    """it would need second derivatives, which the layer does not have: an error, never a term without effect"""
    import nerfacc_amd as nerfacc
    from nerfacc_amd import dense

    if python:
        monkeypatch.setattr(dense, "_EXT", False)
    x, w, b = (normal(*s, seed=i).requires_grad_(True) for i, s in enumerate([(4, 8), (6, 8), (6,)]))
    out = nerfacc.linear(x, w, b, activation=act)
    gx, gw = torch.autograd.grad(out, (x, w), torch.ones_like(out), create_graph=True)
    for g in (gx, gw):
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (out.detach().sum() + g.square().sum()).backward(retain_graph=True)
    # a gradient that depends on nothing that is learnt is a plain tensor, as torch's own is
    y = nerfacc.linear(x, w.detach(), b.detach(), activation="relu")
    assert not torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)[0].requires_grad


@pytest.mark.parametrize("python", [False, True])
def test_forward_mode_is_refused(python, monkeypatch):
    import torch.autograd.forward_ad as fwd

    import nerfacc_amd as nerfacc
    from nerfacc_amd import dense

    if python:
        monkeypatch.setattr(dense, "_EXT", False)
    x, w, b = normal(4, 8), normal(6, 8), normal(6)
    with fwd.dual_level():
        for i in range(3):
            args = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate((x, w, b))]
            with pytest.raises(NotImplementedError, match="forward mode"):
                nerfacc.linear(*args)
        with pytest.raises(NotImplementedError, match="forward mode"):
            nerfacc.linear(x, w, residual=fwd.make_dual(normal(4, 6), normal(4, 6)))
        nerfacc.linear(x, w, b)
