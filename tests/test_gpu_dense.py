"""`nerfacc_amd.linear` against the same layer in 64 bits, forward and backward.

Tolerances: u = eps / 2 of the type.  A sum of n products in 32 bits is off by at most about n 2^-24 sum |terms| (any order; in
practice sqrt(n)); the result is rounded once (u |y|).  The backward pass rounds dz = dy act'(z) to the type before the product
(u sum |terms|), and takes act' from a saved number that was rounded once: another u c sum |terms|, c = |s act''(s)| / |act'(s)|
<= 2 on the inputs used (|z| < 4).  The bound is 4 u sum |terms| + n 2^-24 sum |terms|, with sum |terms| formed in 64 bits too."""
import gc

import pytest
import torch

from gpu_utils import DEV

pytestmark = pytest.mark.gpu

ACTS = {None: lambda z: z, "relu": torch.relu, "sigmoid": torch.sigmoid, "softplus": lambda z: torch.logaddexp(z, torch.zeros_like(z)),
        "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "exp": torch.exp}


def make(m, k, n, dtype, seed=0, bias=True, residual=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    x, w = r(m, k).to(dtype), (r(n, k) * 0.7 / max(k, 1) ** 0.5).to(dtype)
    return x, w, (0.2 * r(n)).to(dtype) if bias else None, r(m, n).to(dtype) if residual else None, r(m, n).to(dtype)


def check(x, w, b, r, gy, act):
    """outputs and gradients of linear against 64 bits, element by element"""
    import nerfacc_amd as nerfacc

    dt, (m, k), n = x.dtype, x.shape, w.shape[0]
    u = torch.finfo(dt).eps / 2
    leaves = [t for t in (x, w, b, r) if t is not None]
    own = [t.detach().requires_grad_(True) for t in leaves]
    it = iter(own)
    args = [next(it) if t is not None else None for t in (x, w, b, r)]
    out = nerfacc.linear(*args[:3], activation=act, residual=args[3])
    assert out.dtype == dt and out.shape == (m, n)
    quiet = nerfacc.linear(x, w, b, activation=act, residual=r)
    assert torch.equal(out, quiet)
    grads = torch.autograd.grad(out, own, gy)
    X, W, G = x.double(), w.double(), gy.double()
    z = X @ W.t() + (0 if b is None else b.double())
    zl = z.detach().requires_grad_(True)
    y = ACTS[act](zl)
    slope = torch.autograd.grad(y.sum(), zl)[0]
    want = y.detach() + (0 if r is None else r.double())
    size = X.abs() @ W.t().abs() + (0 if b is None else b.double().abs())
    steep = slope.abs().clamp(min=1.0) * (2.0 if act == "exp" else 1.0)     # e^z over an error of z: its own slope, with room for the curvature
    tol = u * want.abs() + steep * (k + 4) * 2.0**-24 * size + 8 * 2.0**-24 * y.detach().abs() + (6e-8 if dt == torch.float16 else 0)
    assert ((out.double() - want).abs() <= tol).all(), ((out.double() - want).abs() / tol).max()
    # what an error of z (in 32 bits) does to the slope: |act''| <= 1.2 except for exp, where it is the slope
    bend = (slope.abs() if act == "exp" else torch.ones_like(slope)) * (k + 4) * 2.0**-24 * size
    dz, dza = G * slope, (G * slope).abs()
    soft = 0.0 if act in (None, "relu") else 1.0
    edge = (z.abs() <= (k + 4) * 2.0**-24 * size) if act == "relu" else torch.zeros_like(z, dtype=torch.bool)
    dz_err = 4 * u * dza + soft * G.abs() * (bend + 4 * u * 0.5 * (act in ("sigmoid", "silu", "gelu")) + 8 * 2.0**-24) + G.abs() * edge
    refs = [(dz @ W, dza @ W.abs(), dz_err @ W.abs(), n), (dz.t() @ X, dza.t() @ X.abs(), dz_err.t() @ X.abs(), m)]
    if b is not None:
        refs.append((dz.sum(0), dza.sum(0), dz_err.sum(0), m))
    if r is not None:
        refs.append((G, G.abs(), torch.zeros_like(G), 1))
    tiny = 6e-8 if dt == torch.float16 else 0                                # fp16's smallest steps
    for got, (ref, mag, err, terms) in zip(grads, refs):
        tol = u * ref.abs() + err + (terms + 4) * 2.0**-24 * mag + tiny * (1 + mag / mag.mean().clamp(min=1e-30))
        assert got.dtype == dt and got.shape == ref.shape
        assert ((got.double() - ref).abs() <= tol).all(), ((got.double() - ref).abs() / tol).max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 256, 256), (3, 7, 5), (64, 64, 64), (127, 63, 65), (129, 8, 32), (130, 33, 4), (257, 72, 136), (700, 256, 128),
                                   (2000, 130, 200)])
def test_sizes(dtype, m, k, n):
    check(*make(m, k, n, dtype), "relu")
    check(*make(m, k, n, dtype, seed=1, bias=False, residual=True), None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(1, 300, 3), (17, 1000, 33), (40, 257, 300), (300, 512, 64), (9000, 272, 130), (5, 64, 700)])
def test_long_contractions_and_wide_outputs(dtype, m, k, n):
    """contractions beyond what stays in LDS: few rows, tiles; and a weight in several blocks of columns"""
    check(*make(m, k, n, dtype, seed=9, residual=True), "relu")
    check(*make(m, k, n, dtype, seed=10), "silu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_tiles(dtype):
    """enough rows and columns for the largest tiles, with rows and columns that end inside them"""
    check(*make(16500, 520, 1000, dtype, seed=11), "relu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("residual", [False, True])
def test_activations(dtype, act, residual):
    check(*make(333, 48, 72, dtype, seed=2, residual=residual), act)


def test_strides_and_shapes():
    import nerfacc_amd as nerfacc

    wide, w, b, r, g = make(200, 96, 40, torch.bfloat16, seed=3)
    for x in (wide[:, 16:80], wide[:, 1:65], wide[::2, 8:72], wide[:64].t()[:64, :64], wide[:1, :64].expand(50, 64)):
        check(x, w[:, :64].contiguous(), b, None, g[:x.shape[0]], "silu")
        wt = w[:, 16:80]                                                    # a strided weight
        assert torch.equal(nerfacc.linear(x, wt, b), nerfacc.linear(x.contiguous(), wt.contiguous(), b))
    x3 = wide.view(4, 50, 96)
    out = nerfacc.linear(x3, w, b, activation="gelu", residual=g.view(4, 50, 40))
    assert out.shape == (4, 50, 40) and torch.equal(out.view(200, 40), nerfacc.linear(wide, w, b, activation="gelu", residual=g))
    one = nerfacc.linear(wide[0], w, b)
    assert one.shape == (40,) and torch.equal(one, nerfacc.linear(wide[:1], w, b)[0])
    gx = torch.autograd.grad(nerfacc.linear(wide.requires_grad_(True), w).sum(), wide)[0]           # an expanded gradient
    assert torch.allclose(gx.float(), w.float().sum(0).expand(200, 96), atol=2.0**-7 * w.float().abs().sum(0).max().item())


def test_empty_batch_and_partial_gradients():
    import nerfacc_amd as nerfacc

    x, w, b, r, g = make(9, 16, 24, torch.float32, seed=4, residual=True)
    e = torch.zeros(0, 16, device=DEV, requires_grad=True)
    wl, bl = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    out = nerfacc.linear(e, wl, bl, activation="relu")
    assert out.shape == (0, 24)
    gx, gw, gb = torch.autograd.grad(out.sum(), (e, wl, bl))
    assert gx.shape == (0, 16) and not gw.any() and not gb.any()
    full = torch.autograd.grad(nerfacc.linear(x.requires_grad_(True), wl, bl, activation="silu"), (x, wl, bl), g)
    x = x.detach()
    only_b = torch.autograd.grad(nerfacc.linear(x, w, bl, activation="silu"), bl, g)[0]
    only_w = torch.autograd.grad(nerfacc.linear(x, wl, b, activation="silu"), wl, g)[0]
    assert torch.equal(only_b, full[2]) and torch.equal(only_w, full[1])
    rl = r.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(nerfacc.linear(x, w, b, residual=rl), rl, g)[0], g)


def test_same_bits_every_time_and_nan_stays_in_its_row():
    import nerfacc_amd as nerfacc

    x, w, b, r, g = make(5000, 96, 96, torch.bfloat16, seed=5, residual=True)
    first = None
    for _ in range(3):
        own = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]
        got = torch.autograd.grad(nerfacc.linear(own[0], own[1], own[2], activation="gelu", residual=own[3]), own, g)
        first = first or got
        assert all(torch.equal(a, c) for a, c in zip(first, got))
    clean = nerfacc.linear(x, w, b, activation="relu")
    x2 = x.clone()
    x2[77, 5] = float("nan")
    out = nerfacc.linear(x2, w, b, activation="relu")
    assert out[77].isnan().all()
    keep = torch.arange(5000, device=DEV) != 77
    assert torch.equal(out[keep], clean[keep])


def test_gradient_against_differences():
    import nerfacc_amd as nerfacc

    x, w, b, r, g = make(40, 12, 20, torch.float32, seed=6)
    v = torch.randn(40, 12, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    xl = x.clone().requires_grad_(True)
    gx = torch.autograd.grad(nerfacc.linear(xl, w, b, activation="silu"), xl, g)[0]
    h = 2.0**-6
    up, down = (nerfacc.linear(x + s * h * v, w, b, activation="silu").double() for s in (1, -1))
    slope = ((up - down) * g.double()).sum() / (2 * h)
    # central difference: h^2 / 6 |f'''| |v W|^3 (|silu'''| < 1) plus 2 * 32 * 2^-24 |y| / (2 h), summed with |g|
    vw = (v.double() @ w.double().t()).abs()
    tol = (g.double().abs() * (h * h / 6 * vw**3 + 32 * 2.0**-24 * (1 + up.abs()) / h)).sum()
    assert abs(slope - (gx.double() * v.double()).sum()) <= tol


def test_other_stream_and_graph_replays():
    import nerfacc_amd as nerfacc

    x, w, b, r, g = make(3000, 64, 64, torch.bfloat16, seed=7, residual=True)
    own = [t.detach().requires_grad_(True) for t in (x, w, b, r)]

    def step():
        out = nerfacc.linear(own[0], own[1], own[2], activation="silu", residual=own[3])
        return [out, *torch.autograd.grad(out, own, g)]

    want = [t.detach().clone() for t in step()]              # (an eager graph of the same leaves must not outlive this line)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    del got
    gc.collect()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator(device=DEV).manual_seed(k), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, c) for a, c in zip(held, eager)), k


def test_nodes_of_another_stream_are_counted():
    """what a captured call is refused by: an autograd node that another stream recorded"""
    from nerfacc_amd import cuda as C
    from nerfacc_amd.cuda import _backend

    if _backend.BACKEND != "ext":
        pytest.skip("torch extension not the active backend")
    x = torch.ones(4, device=DEV, requires_grad=True)
    assert C.foreign_nodes([x, None]) == 0                   # a leaf that nothing has recorded yet
    y = (x * 2).exp()
    assert C.foreign_nodes([y]) == 0 and C.foreign_nodes([x.detach()]) == 0
    with torch.cuda.stream(torch.cuda.Stream()):
        assert C.foreign_nodes([y]) == 3 and C.foreign_nodes([x]) == 1
        z = torch.ones(4, device=DEV, requires_grad=True) * 2
        assert C.foreign_nodes([z, x * 1]) == 1
    del y, z
    with torch.cuda.stream(torch.cuda.Stream()):
        assert C.foreign_nodes([x]) == 0                     # the eager graph is gone, and its accumulator with it


def test_both_host_faces_agree():
    from nerfacc_amd.cuda import _backend

    if _backend.BACKEND != "ext":
        pytest.skip("torch extension not the active backend")
    ext, ct = _backend._C, _backend._CtypesC
    x, w, b, r, g = make(500, 72, 40, torch.float16, seed=8, residual=True)
    wide = torch.cat([x, x], 1)
    for act in (0, 1, 4):
        for res in (None, r):
            a, c = (f.linear_fwd(wide[:, 8:80], w, b, res, act, True) for f in (ext, ct))
            assert torch.equal(a[0], c[0]) and (a[1] is None) == (c[1] is None) and (a[1] is None or torch.equal(a[1], c[1]))
            saved = a[1] if a[1] is not None else (a[0] if act else None)
            p, q = (f.linear_bwd(g, wide[:, 8:80], w, saved, act, True, True, True) for f in (ext, ct))
            assert all(torch.equal(u, v) for u, v in zip(p, q))


def test_refusals():
    import nerfacc_amd as nerfacc

    x, w, b, r, g = make(8, 16, 24, torch.float32)
    for bad, err in ((lambda: nerfacc.linear(x, w.half()), TypeError), (lambda: nerfacc.linear(x.double(), w.double()), TypeError),
                     (lambda: nerfacc.linear(x, w, activation="tanh"), ValueError), (lambda: nerfacc.linear(x, w[:, :8]), ValueError),
                     (lambda: nerfacc.linear(x, w, b[:5]), ValueError), (lambda: nerfacc.linear(x, w, residual=r), ValueError) if r is not None else
                     (lambda: nerfacc.linear(x, w, residual=g[:4]), ValueError), (lambda: nerfacc.linear(x.cpu(), w.cpu()), RuntimeError),
                     (lambda: nerfacc.linear(x, w.cpu()), RuntimeError), (lambda: nerfacc.linear(x, w[:0]), ValueError)):
        with pytest.raises(err):
            bad()
    xl = x.clone().requires_grad_(True)
    gx = torch.autograd.grad(nerfacc.linear(xl, w).sum(), xl, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_the_grid_and_mlp_field_through_it():
    """a training step of the bench's grid + MLP field (sampling, field, rendering, gradients) with its decoder's layers fused"""
    import nerfacc_amd as nerfacc
    from benchlib.scene import AABB, GridMlpField, make_ray_pool, render_rays

    torch.manual_seed(0)
    plain, fused = GridMlpField(AABB, res=32).to(DEV), GridMlpField(AABB, res=32, fused=True).to(DEV)
    fused.load_state_dict(plain.state_dict())
    est = nerfacc.OccGridEstimator(roi_aabb=AABB, resolution=32, levels=1).to(DEV).eval()
    est.binaries.fill_(True)
    o, d = make_ray_pool(512, seed=3, device=DEV)
    x = torch.rand(1000, 3, device=DEV) * 3 - 1.5
    for a, b in zip(plain(x), fused(x)):                    # three layers of at most 32 terms: some hundred last places of 32 bits
        assert torch.allclose(a, b, rtol=2e-5, atol=2e-6)
    grads = []
    for field in (plain, fused):
        rgb, acc, depth, n = render_rays(field, est, o, d, torch.ones(3, device=DEV), False)
        assert n > 1000
        grads.append([rgb.detach(), *torch.autograd.grad((rgb - 0.3).square().sum(), list(field.parameters()))])
    for a, b in zip(*grads):                                # atomic sums in torch's scatter and products: relative to the tensor's own size
        assert (a - b).abs().max() <= 1e-4 * a.abs().max() + 1e-7


def test_fp16_dz_beyond_its_range():
    """dz = dy act'(z) over 65504 with gradients that fit: the two parts of dz hold it, and an infinite gradient stays infinite"""
    import nerfacc_amd as nerfacc

    x = torch.full((3, 8), 1.0, device=DEV, dtype=torch.float16, requires_grad=True)
    w = torch.full((16, 8), 0.5, device=DEV, dtype=torch.float16)
    gy = torch.full((3, 16), 2000.0, device=DEV, dtype=torch.float16)                # e^4 = 54.6: dz = 109200
    gy[2] = float("inf")
    out = nerfacc.linear(x, w, activation="exp")
    gx = torch.autograd.grad(out, x, gy)[0]
    assert gx[2].isposinf().all() and gx[:2].isposinf().all()                        # 16 x 54600 does not fit fp16: inf, not NaN
    gx = torch.autograd.grad(nerfacc.linear(x, w * torch.tensor([[1.0]] + [[0.0]] * 15, device=DEV).half(), activation="exp"), x, gy[:1].expand(3, 16))[0]
    assert (gx.float() - 54.598 * 2000 * 0.5).abs().max() <= 2.0**-10 * 54600


def test_offsets_beyond_32_bits():
    """outputs of more than 2^31 numbers: their end is what the last rows give alone"""
    import nerfacc_amd as nerfacc

    x = torch.randn((1 << 23) + 77, 8, generator=torch.Generator(device=DEV).manual_seed(0), device=DEV).bfloat16()
    w = torch.randn(264, 8, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).bfloat16()
    out = nerfacc.linear(x, w, activation="relu")
    assert out.numel() > 1 << 31 and torch.equal(out[-3000:], nerfacc.linear(x[-3000:], w, activation="relu"))
    assert torch.equal(out[:500], nerfacc.linear(x[:500], w, activation="relu"))


def test_a_large_weight_in_a_captured_step():
    """the form whose workgroups take more than 64 KiB of LDS, captured and replayed"""
    import nerfacc_amd as nerfacc

    x, w, b, r, g = make(900, 256, 256, torch.bfloat16, seed=12, residual=True)
    own = [t.detach().requires_grad_(True) for t in (x, w, b, r)]

    def step():
        out = nerfacc.linear(own[0], own[1], own[2], activation="relu", residual=own[3])
        return [out.detach(), *torch.autograd.grad(out, own, g)]

    step()
    gc.collect()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator(device=DEV).manual_seed(k), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, step())), k


def test_capture_beside_an_eager_graph_is_refused():
    """a backward pass that could not be captured: the forward call says so instead"""
    import nerfacc_amd as nerfacc
    from nerfacc_amd.cuda import _backend

    if _backend.BACKEND != "ext":
        pytest.skip("torch extension not the active backend")
    x, w, b, r, g = make(64, 32, 32, torch.float32, seed=13)
    own = [t.detach().requires_grad_(True) for t in (x, w, b)]
    alive = nerfacc.linear(*own)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(graph):
            nerfacc.linear(*own)
    with torch.cuda.graph(torch.cuda.CUDAGraph()), torch.no_grad():
        nerfacc.linear(*own)                                                         # without gradients there is nothing to capture
    assert alive.shape == (64, 32)
    torch.cuda.synchronize()


def test_docstring_example():
    import nerfacc_amd as nerfacc

    x = torch.tensor([[1., 2.]], device=DEV)
    assert nerfacc.linear(x, torch.tensor([[1., 1.], [1., -1.]], device=DEV), activation="relu").tolist() == [[3.0, 0.0]]


@pytest.mark.parametrize("m,k,n", [(1, 4, 4), (13, 8, 32), (999, 16, 4), (700, 64, 64), (5000, 32, 12), (2100, 20, 48)])
@pytest.mark.parametrize("act", list(ACTS))
def test_narrow_layers(m, k, n, act):
    """up to 64 features in and out: rows and columns that end inside a step"""
    check(*make(m, k, n, torch.float32, seed=12), act)


@pytest.mark.parametrize("m,k,n", [(20011, 301, 4), (9000, 256, 256), (2049, 200, 132)])
def test_choices_of_32_bits(m, k, n):
    """many rows with few outputs and a long contraction; a backward product that goes by tiles"""
    check(*make(m, k, n, torch.float32, seed=14), "softplus")
