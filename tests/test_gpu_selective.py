"""`causal_conv`, `selective_scan` and their one-row forms against the same operators in 64 bits, forward and backward.

Tolerances: u = eps / 2 of the type, for the one rounding of an output.  In 32 bits a term of a scan that has lived for m rows has been
through m products with a decay: each brings the exponential's last place, the product's rounding and, once over the whole decay
exp(-x), x times the relative error of its exponent (x e^-x <= 0.4; step is good to about 12 last places, the product with A and
log2 e to 2).  That is at most (16 + 3 m) 2^-24 of the term; its path back through the gradient doubles it, and sums over rows add
one rounding per term.  Bounds are these factors times the sums of absolute values (feature_cases.scan_sizes)."""
import gc

import pytest
import torch

import feature_cases as ref
from gpu_utils import DEV

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LENS = [3, 0, 1, 17, 8, 9, 0, 40, 2]


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def packed(lens):
    lens = torch.tensor(lens)
    return torch.stack([lens.cumsum(0) - lens, lens], -1).to(DEV)


def near(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    assert (off <= tol).all(), (what, (off / tol.clamp(min=1e-300)).max().item(), off.max().item())


# ------------------------------------------------------------------------------------------------------------- convolution
def conv_inputs(rows, rays, d, width, dtype, seed=0, bias=True, state=False):
    g = generator(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    return dict(x=r(rows, d), w=r(d, width) * 0.5, b=r(d) if bias else None, init=r(rays, width - 1, d) if state else None,
                gy=r(rows, d), gf=r(rays, width - 1, d))


def check_conv(c, act, info=None, shape=None, final=True):
    import nerfacc_amd as nerfacc

    x, dt = c["x"], c["x"].dtype
    u, width = torch.finfo(dt).eps / 2, c["w"].shape[1]
    seqs = ref.rows_of(info, None if shape is None else shape[:2])
    own = {k: c[k].detach().requires_grad_(True) for k in ("x", "w", "b", "init") if c[k] is not None}
    out, last = nerfacc.causal_conv(own["x"] if shape is None else own["x"].view(shape), own["w"], own.get("b"), activation=act, packed_info=info,
                                    initial_state=own.get("init"), return_final_state=True)
    alone = nerfacc.causal_conv(x if shape is None else x.view(shape), c["w"], c["b"], activation=act, packed_info=info, initial_state=c["init"])
    assert torch.equal(alone, out) and out.dtype == dt
    flat = out.reshape(x.shape)
    gf = c["gf"] if final else None
    grads = torch.autograd.grad([flat, last] if final else [flat], list(own.values()), [c["gy"], gf] if final else [c["gy"]])
    wide = {k: v.detach().double().requires_grad_(True) for k, v in own.items()}
    ro, rl = ref.conv(wide["x"], wide["w"], wide.get("b"), act, seqs, wide.get("init"))
    rg = torch.autograd.grad([ro, rl] if final else [ro], list(wide.values()), [c["gy"].double(), c["gf"].double()] if final else [c["gy"].double()],
                             allow_unused=True)
    mags = {k: v.detach().double().abs().requires_grad_(True) for k, v in own.items()}
    mo, ml = ref.conv(mags["x"], mags["w"], mags.get("b"), None, seqs, mags.get("init"))
    mg = torch.autograd.grad([mo, ml] if final else [mo], list(mags.values()), [c["gy"].double().abs(), c["gf"].double().abs()] if final
                             else [c["gy"].double().abs()], allow_unused=True)
    tiny = 6e-8 if dt == torch.float16 else 0
    # |silu'| <= 1.1, |silu''| <= 0.5: an error of z in the last places moves the slope by half of it
    mo = mo.detach()
    near(flat, ro.detach(), u * ro.detach().abs() + (width + 12) * 2.0**-24 * (mo + 1e-30) * 1.2 + tiny, "out")
    near(last, rl.detach(), u * 0 * rl.detach().abs(), "final state")
    bend = 1.0 + 0.5 * mo.max().item() if act else 1.0
    for (k, got), want, mag in zip(zip(own, grads), rg, mg):
        want = torch.zeros_like(wide[k]) if want is None else want
        mag = torch.zeros_like(wide[k]) if mag is None else mag
        terms = 2 * width + 16 + (x.shape[0] if k in ("w", "b") else 0)
        near(got, want, u * want.abs() + terms * 2.0**-24 * mag * 1.2 * bend + tiny, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,width", [(1, 2), (5, 3), (8, 4), (64, 4), (72, 2), (130, 3), (600, 4)])
def test_conv_packed(dtype, d, width):
    info = packed(LENS)
    check_conv(conv_inputs(80, 9, d, width, dtype, seed=d, state=True), "silu", info)
    check_conv(conv_inputs(80, 9, d, width, dtype, seed=d + 1, bias=False), None, info, final=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rays,n,d", [(1, 1, 16), (1, 2, 3), (3, 5, 64), (2, 133, 40), (40, 32, 8)])
def test_conv_batched(dtype, rays, n, d):
    check_conv(conv_inputs(rays * n, rays, d, 4, dtype, seed=n, state=True), "silu", shape=(rays, n, d))


def test_conv_order_gaps_and_nan_outside():
    import nerfacc_amd as nerfacc

    info = torch.tensor([[50, 10], [5, 20], [30, 0], [33, 3]], device=DEV)          # out of order, rows 0-4, 25-32, 36-49, 60-69 of no ray
    c = conv_inputs(70, 4, 24, 4, torch.float32, seed=2, state=True)
    check_conv(c, "silu", info)
    gap = torch.ones(70, dtype=torch.bool, device=DEV)
    for s, n in info.tolist():
        gap[s:s + n] = False
    x2 = c["x"].clone()
    x2[gap] = float("nan")
    out = nerfacc.causal_conv(x2, c["w"], c["b"], activation="silu", packed_info=info, initial_state=c["init"])
    assert torch.equal(out, nerfacc.causal_conv(c["x"], c["w"], c["b"], activation="silu", packed_info=info, initial_state=c["init"]))
    assert not out[gap].any()
    gy = c["gy"].clone()
    gy[gap] = float("nan")
    xl, wl = x2.requires_grad_(True), c["w"].detach().requires_grad_(True)
    gx, gw = torch.autograd.grad(nerfacc.causal_conv(xl, wl, c["b"], activation="silu", packed_info=info, initial_state=c["init"]), (xl, wl), gy)
    assert not gx[gap].any() and gx.isfinite().all() and gw.isfinite().all()
    # rows outside the array are cut off
    cut = nerfacc.causal_conv(c["x"], c["w"], packed_info=torch.tensor([[-3, 10], [60, 1000], [1000, 5], [20, -4]], device=DEV))
    want = nerfacc.causal_conv(c["x"], c["w"], packed_info=torch.tensor([[0, 7], [60, 10], [0, 0], [0, 0]], device=DEV))
    assert torch.equal(cut, want)


def test_conv_pieces_of_a_ray_are_the_whole():
    """a ray taken a few samples at a time, and one at a time, with its state"""
    import nerfacc_amd as nerfacc

    c = conv_inputs(3 * 21, 3, 40, 4, torch.bfloat16, seed=4, state=True)
    x = c["x"].view(3, 21, 40)
    whole, end = nerfacc.causal_conv(x, c["w"], c["b"], activation="silu", initial_state=c["init"], return_final_state=True)
    state, parts = c["init"], []
    for a, b in ((0, 2), (2, 3), (3, 14), (14, 21)):
        out, state = nerfacc.causal_conv(x[:, a:b], c["w"], c["b"], activation="silu", initial_state=state, return_final_state=True)
        parts.append(out)
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(state, end)
    state, place = c["init"].clone(), c["init"].clone()
    for t in range(21):
        out, state = nerfacc.causal_conv_step(x[:, t], state, c["w"], c["b"], activation="silu")
        again, same = nerfacc.causal_conv_step(x[:, t], place, c["w"], c["b"], activation="silu", out_state=place)
        assert same is place and torch.equal(out, whole[:, t]) and torch.equal(again, out)
    assert torch.equal(state, end) and torch.equal(place, end)


# ------------------------------------------------------------------------------------------------------------------- scan
def scan_inputs(rows, rays, d, s, dtype, seed=0, softplus=True, gate=True, skip=True, state=True):
    g = generator(seed)
    r = lambda *sh: torch.randn(sh, generator=g, device=DEV)  # noqa: E731
    v = lambda *sh: r(*sh).to(dtype)  # noqa: E731
    return dict(u=v(rows, d), delta=(r(rows, d) * 0.5).to(dtype) if softplus else (0.2 * r(rows, d).abs()).to(dtype),
                A=-torch.rand((d, s), generator=g, device=DEV) * 3, B=v(rows, s), C=v(rows, s), D=r(d) if skip else None,
                z=v(rows, d) if gate else None, bias=r(d) - 2 if softplus else None, init=r(rays, d, s) if state else None,
                gy=v(rows, d), gf=r(rays, d, s), softplus=softplus)


NAMES = ("u", "delta", "A", "B", "C", "D", "z", "bias", "init")


def call_scan(c, t, info=None, shape=None, final=True):
    import nerfacc_amd as nerfacc

    v = (lambda a: a if a is None or shape is None else a.view(*shape[:2], a.shape[-1]))
    return nerfacc.selective_scan(v(t["u"]), v(t["delta"]), t["A"], v(t["B"]), v(t["C"]), D=t.get("D"), gate=v(t.get("z")),
                                  delta_bias=t.get("bias"), delta_softplus=c["softplus"], packed_info=info, initial_state=t.get("init"),
                                  return_final_state=final)


def check_scan(c, info=None, shape=None, final=True):
    dt = c["u"].dtype
    u = torch.finfo(dt).eps / 2
    seqs = ref.rows_of(info, None if shape is None else shape[:2])
    own = {k: c[k].detach().requires_grad_(True) for k in NAMES if c[k] is not None}
    out, last = call_scan(c, own, info, shape)
    with torch.no_grad():
        assert torch.equal(call_scan(c, own, info, shape, final=False), out)
    flat = out.reshape(c["u"].shape)
    outs, gs = ([flat, last], [c["gy"], c["gf"]]) if final else ([flat], [c["gy"]])
    grads = dict(zip(own, torch.autograd.grad(outs, list(own.values()), gs)))
    wide = {k: v.detach().double().requires_grad_(True) for k, v in own.items()}
    raw = wide["delta"] + wide["bias"] if "bias" in wide else wide["delta"]
    args = (wide["u"], raw, wide["A"], wide["B"], wide["C"], wide.get("D"), wide.get("z"), c["softplus"], seqs, wide.get("init"))
    ro, rl = ref.scan(*args)
    rg = torch.autograd.grad([ro, rl] if final else [ro], list(wide.values()), [g.double() for g in gs], allow_unused=True)
    with torch.no_grad():
        size = ref.scan_sizes(*args, c["gy"].double(), c["gf"].double() if final else None)
    longest = max([n for _, n in seqs] + [1])
    tiny = 6e-8 if dt == torch.float16 else 1e-37
    f = (16 + 3 * longest) * 2.0**-24
    near(flat, ro.detach(), u * ro.detach().abs() + f * size["out"] + tiny, "out")
    near(last, rl.detach(), f * size["final"] + tiny, "final state")
    for (k, got), want in zip(grads.items(), rg):
        want = torch.zeros_like(wide[k]) if want is None else want
        once = u if got.dtype == dt else 2.0**-24
        terms = c["u"].shape[0] if k in ("A", "D", "bias") else c["u"].shape[1] if k in ("B", "C") else 0
        near(got, want, once * want.abs() + (2 * f + terms * 2.0**-24) * size[k] + tiny, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,s", [(1, 1), (3, 16), (64, 16), (70, 4), (5, 3), (33, 8), (20, 17), (40, 40)])
def test_scan_packed(dtype, d, s):
    check_scan(scan_inputs(80, 9, d, s, dtype, seed=d + s), packed(LENS))


@pytest.mark.parametrize("s", [100, 130, 256])
def test_scan_many_states(s):
    check_scan(scan_inputs(20, 3, 3, s, torch.float32, seed=s), packed([9, 0, 11]))


@pytest.mark.parametrize("flags", [dict(softplus=False), dict(gate=False), dict(skip=False), dict(state=False),
                                   dict(softplus=False, gate=False, skip=False, state=False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_optional_parts(flags, dtype):
    check_scan(scan_inputs(80, 9, 24, 16, dtype, seed=3, **flags), packed(LENS), final=flags.get("state", True))


@pytest.mark.parametrize("rays,n,d,s", [(1, 1, 16, 16), (4, 8, 70, 16), (2, 33, 8, 4)])
def test_scan_batched(rays, n, d, s):
    check_scan(scan_inputs(rays * n, rays, d, s, torch.float16, seed=n), shape=(rays, n, d))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_cut_into_chunks(dtype):
    """few long sequences: the chunked passes, with lengths around the chunk (32 rows or more) and none"""
    check_scan(scan_inputs(2 * 300, 2, 6, 16, dtype, seed=1), shape=(2, 300, 6))
    check_scan(scan_inputs(700, 5, 6, 16, dtype, seed=2), packed([513, 0, 32, 1, 154]))
    check_scan(scan_inputs(420, 3, 70, 20, dtype, seed=5, state=False), packed([129, 31, 260]))


def test_scan_order_gaps_and_nan_outside():
    info = torch.tensor([[150, 100], [5, 120], [130, 0], [133, 9]], device=DEV)     # out of order, with rows of no ray; chunked
    c = scan_inputs(270, 4, 24, 16, torch.float32, seed=2)
    check_scan(c, info)
    gap = torch.ones(270, dtype=torch.bool, device=DEV)
    for s, n in info.tolist():
        gap[s:s + n] = False
    dirty = dict(c)
    for k in ("u", "delta", "B", "C", "z", "gy"):
        dirty[k] = c[k].clone()
        dirty[k][gap] = float("nan")
    res = []
    for v in (c, dirty):
        own = {k: v[k].detach().requires_grad_(True) for k in NAMES}
        out, last = call_scan(v, own, info)
        res.append([out.detach(), last.detach(), *torch.autograd.grad([out, last], list(own.values()), [v["gy"], v["gf"]])])
    assert all(torch.equal(a, b) for a, b in zip(*res))
    for k in (0, 2, 3, 5, 6, 8):
        assert not res[0][k][gap].any()
    cut = call_scan(c, {**c, "init": None}, torch.tensor([[-3, 10], [260, 1000], [1000, 5], [20, -4]], device=DEV), final=False)
    want = call_scan(c, {**c, "init": None}, torch.tensor([[0, 7], [260, 10], [0, 0], [0, 0]], device=DEV), final=False)
    assert torch.equal(cut, want)


def test_scan_steps_are_the_whole():
    import nerfacc_amd as nerfacc

    rays, n, d, s = 3, 21, 40, 16
    c = scan_inputs(rays * n, rays, d, s, torch.bfloat16, seed=4)
    whole, end = call_scan(c, c, shape=(rays, n, d))
    row = lambda k, t: c[k].view(rays, n, -1)[:, t]  # noqa: E731
    state, place = c["init"], c["init"].clone()
    f = (16 + 3 * n) * 2.0**-24
    for t in range(n):
        args = (row("u", t), row("delta", t), c["A"], row("B", t), row("C", t))
        kw = dict(D=c["D"], gate=row("z", t), delta_bias=c["bias"], delta_softplus=True)
        out, state = nerfacc.selective_scan_step(*args, state, **kw)
        again, same = nerfacc.selective_scan_step(*args, place, **kw, out_state=place)
        assert same is place and torch.equal(out, again) and torch.equal(place, state)
        # two roundings of nearly the same number: one step of bf16 apart at most, plus what the order of 32-bit sums moves
        assert ((out.float() - whole[:, t].float()).abs() <= 2.0**-7 * whole[:, t].float().abs() + 1e-4).all()
    assert ((state - end).abs() <= 2 * f * (end.abs() + state.abs().max())).all()


def test_scan_running_sums_are_the_framework_s_own():
    """no decay, unit steps, one state: the packed sums of scan.py"""
    import nerfacc_amd as nerfacc

    x = torch.randn(80, generator=generator(1), device=DEV)
    one, info = torch.ones(80, 1, device=DEV), packed(LENS)
    got = nerfacc.selective_scan(x[:, None], one, torch.zeros(1, 1, device=DEV), one, one, packed_info=info)[:, 0]
    assert torch.allclose(got, nerfacc.inclusive_sum(x, packed_info=info), rtol=0, atol=80 * 2.0**-24 * 3 * 40)


def test_scan_extreme_values():
    """steps that underflow and overflow the decay, a NaN in one ray, infinite inputs stay in their ray"""
    c = scan_inputs(60, 3, 8, 16, torch.float32, seed=9)
    info = packed([20, 20, 20])
    clean = call_scan(c, c, info)[0]
    for bad in (float("nan"), float("inf")):
        t = {**c, "u": c["u"].clone()}
        t["u"][25, 3] = bad
        out = call_scan(c, t, info)[0]
        keep = torch.ones(60, 8, dtype=torch.bool, device=DEV)
        keep[25:40, 3] = False
        assert torch.equal(out[keep], clean[keep]) and not out[25, 3].isfinite()
    t = {**c, "delta": c["delta"].clone()}
    t["delta"][10] = 1e4                                              # everything before it is forgotten
    t["delta"][30] = -1e4                                             # and here nothing happens: no decay, no input
    out, last = call_scan(c, t, info)
    assert out.isfinite().all() and last.isfinite().all()


def test_scan_gradient_against_differences():
    c = scan_inputs(60, 3, 6, 4, torch.float32, seed=11)
    info = packed([33, 0, 27])
    own = {k: c[k].detach().requires_grad_(True) for k in NAMES}
    out, last = call_scan(c, own, info)
    grads = dict(zip(own, torch.autograd.grad([out, last], list(own.values()), [c["gy"], c["gf"]])))
    g = generator(5)
    for k in NAMES:
        v = torch.randn(c[k].shape, generator=g, device=DEV) * 0.2
        h = 2.0**-6
        ends = []
        for s in (1, -1):
            with torch.no_grad():
                o, e = call_scan(c, {**c, k: c[k] + s * h * v}, info)
            ends.append((o.double() * c["gy"].double()).sum() + (e.double() * c["gf"].double()).sum())
        slope = (ends[0] - ends[1]) / (2 * h)
        want = (grads[k].double() * v.double()).sum()
        # curvature: h^2 / 6 of a third derivative that is of the order of the gradient's own sum of terms here; rounding: 1e-5 / h
        size = (grads[k].double() * v.double()).abs().sum()
        assert abs(slope - want) <= 4e-3 * size + 2e-3, k


# ---------------------------------------------------------------------------------------------------- strides, streams, faces
def test_strided_rows_and_slices():
    import nerfacc_amd as nerfacc

    g = generator(0)
    both, bc = torch.randn(4, 20, 96, generator=g, device=DEV), torch.randn(4, 20, 32, generator=g, device=DEV)
    u, z, dt = both[..., :40], both[..., 56:], torch.randn(4, 40, 20, generator=g, device=DEV).transpose(1, 2)
    A = -torch.rand(16, 40, generator=g, device=DEV).t()
    args = (u, dt, A, bc[..., :16], bc[..., 16:])
    tight = [t.contiguous() for t in args]
    out = nerfacc.selective_scan(*args, gate=z, delta_softplus=True)
    assert torch.equal(out, nerfacc.selective_scan(*tight, gate=z.contiguous(), delta_softplus=True))
    w = torch.randn(3, 40, generator=g, device=DEV).t()
    assert torch.equal(nerfacc.causal_conv(u, w), nerfacc.causal_conv(u.contiguous(), w.contiguous()))
    assert torch.equal(nerfacc.causal_conv(both[..., 1:42], w[:1].expand(41, 3)), nerfacc.causal_conv(both[..., 1:42].contiguous(), w[:1].expand(41, 3).contiguous()))
    # a step shared by the channels and an input shared by the rays: broadcast views, whose gradients are summed by autograd
    one = torch.rand(4, 20, 1, generator=g, device=DEV, requires_grad=True)
    full = one.detach().expand(4, 20, 40).contiguous().requires_grad_(True)
    got = torch.autograd.grad(nerfacc.selective_scan(u, one.expand(4, 20, 40), *tight[2:]).sum(), one)[0]
    want = torch.autograd.grad(nerfacc.selective_scan(u, full, *tight[2:]).sum(), full)[0].sum(-1, keepdim=True)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5 * want.abs().max().item())


def test_empty_calls():
    import nerfacc_amd as nerfacc

    w, A = torch.rand(8, 4, device=DEV, requires_grad=True), torch.rand(8, 4, device=DEV, requires_grad=True)
    info = torch.zeros((0, 2), dtype=torch.int64, device=DEV)
    for shape, kw, rays in (((0, 8), dict(packed_info=info), 0), ((5, 8), dict(packed_info=info), 0), ((0, 3, 8), {}, 0), ((3, 0, 8), {}, 3),
                            ((0, 8), dict(packed_info=torch.zeros((3, 2), dtype=torch.int64, device=DEV)), 3)):
        x = torch.rand(shape, device=DEV, requires_grad=True)
        init = torch.rand(rays, 3, 8, device=DEV, requires_grad=True)
        out, end = nerfacc.causal_conv(x, w, initial_state=init, return_final_state=True, **kw)
        assert out.shape == shape and not out.any() and torch.equal(end, init)
        gx, gw, gi = torch.autograd.grad([out, end], (x, w, init), [torch.ones_like(out), torch.ones_like(end)])
        assert gx.shape == shape and not gx.any() and not gw.any() and torch.equal(gi, torch.ones_like(init))
        bc = torch.rand((*shape[:-1], 4), device=DEV)
        init = torch.rand(rays, 8, 4, device=DEV, requires_grad=True)
        out, end = nerfacc.selective_scan(x, x, A, bc, bc, initial_state=init, return_final_state=True, **kw)
        assert out.shape == shape and not out.any() and torch.equal(end, init)
        gx, gA, gi = torch.autograd.grad([out, end], (x, A, init), [torch.ones_like(out), torch.ones_like(end)])
        assert gx.shape == shape and not gx.any() and not gA.any() and torch.equal(gi, torch.ones_like(init))
    out, st = nerfacc.causal_conv_step(torch.rand(0, 8, device=DEV), torch.rand(0, 3, 8, device=DEV), w.detach())
    assert out.shape == (0, 8) and st.shape == (0, 3, 8)


def layer(c, info):
    """a layer that mixes features along rays: in, convolution, steps and B and C, scan with its gate, out with the residual"""
    import nerfacc_amd as nerfacc

    d, s = c["A"].shape
    xz = nerfacc.linear(c["x"], c["w_in"])
    u = nerfacc.causal_conv(xz[:, :d], c["w_conv"], c["b_conv"], activation="silu", packed_info=info)
    p = nerfacc.linear(u, c["w_p"])
    dt = nerfacc.linear(p[:, :4], c["w_dt"])
    y = nerfacc.selective_scan(u, dt, c["A"], p[:, 4:4 + s], p[:, 4 + s:], D=c["D"], gate=xz[:, d:], delta_bias=c["bias"], delta_softplus=True,
                               packed_info=info)
    return nerfacc.linear(y, c["w_out"], c["b_out"], residual=c["x"])


def layer_inputs(rows, dtype, seed=0, d=32, s=16, width=24):
    g = generator(seed)
    r = lambda *sh, scale=1.0: (torch.randn(sh, generator=g, device=DEV) * scale).to(dtype)  # noqa: E731
    f = lambda *sh: torch.randn(sh, generator=g, device=DEV)  # noqa: E731
    return dict(x=r(rows, width), w_in=r(2 * d, width, scale=width**-0.5), w_conv=r(d, 4, scale=0.5), b_conv=r(d, scale=0.1),
                w_p=r(4 + 2 * s, d, scale=d**-0.5), w_dt=r(d, 4, scale=0.5), A=-torch.rand((d, s), generator=g, device=DEV) * 2, D=f(d),
                bias=f(d) - 2, w_out=r(width, d, scale=d**-0.5), b_out=r(width, scale=0.1))


def test_a_layer_of_them_together():
    """outputs and gradients of the whole run, in 32 bits, against 64"""
    c, info = layer_inputs(80, torch.float32), packed(LENS)
    own = {k: v.detach().requires_grad_(True) for k, v in c.items()}
    out = layer(own, info)
    gy = torch.randn(out.shape, generator=generator(7), device=DEV)
    grads = torch.autograd.grad(out, list(own.values()), gy)
    w = {k: v.detach().double().requires_grad_(True) for k, v in c.items()}
    seqs, d, s = ref.rows_of(info), 32, 16
    xz = w["x"] @ w["w_in"].t()
    u = ref.conv(xz[:, :d], w["w_conv"], w["b_conv"], "silu", seqs, None)[0]
    p = u @ w["w_p"].t()
    y = ref.scan(u, p[:, :4] @ w["w_dt"].t() + w["bias"], w["A"], p[:, 4:4 + s], p[:, 4 + s:], w["D"], xz[:, d:], True, seqs, None)[0]
    want = y @ w["w_out"].t() + w["b_out"] + w["x"]
    # seven operators behind one another, each good to some hundred last places of its own sums: 2^-24 * 1000 = 6e-5 of each result's size
    near(out, want.detach(), 6e-5 * want.detach().abs().max(), "out")
    for (k, got), g in zip(zip(own, grads), torch.autograd.grad(want, list(w.values()), gy.double())):
        near(got, g, 2e-4 * g.abs().max(), k)


def test_streams_graphs_and_same_bits():
    c, info = layer_inputs(640, torch.bfloat16, seed=1), packed(LENS * 8)
    own = {k: v.detach().requires_grad_(True) for k, v in c.items()}
    gy = torch.randn(640, 24, generator=generator(7), device=DEV).bfloat16()

    def step():
        out = layer(own, info)
        return [out.detach(), *torch.autograd.grad(out, list(own.values()), gy)]

    want = step()
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(want, step()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    gc.collect()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                                # two graphs of the same work, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    for k in range(4):
        with torch.no_grad():
            c["x"].copy_(torch.randn(c["x"].shape, generator=generator(20 + k), device=DEV))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        eager = step()
        for _, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, eager)), k


def test_both_host_faces_agree():
    from nerfacc_amd.cuda import _backend

    if _backend.BACKEND != "ext":
        pytest.skip("torch extension not the active backend")
    ext, ct = _backend._C, _backend._CtypesC

    def same(a, b):
        assert len(a) == len(b)
        for p, q in zip(a, b):
            assert (p is None) == (q is None) and (p is None or torch.equal(p, q))

    info = packed(LENS)
    maps = ext.row_map(info, 85)
    same(maps, ct.row_map(info, 85))
    assert maps[0][80:].eq(-1).all() and maps[1][:6].tolist() == [0, 1, 2, 0, 0, 1]
    c = conv_inputs(85, 9, 24, 4, torch.bfloat16, state=True)
    for rows, rays in (((info, *maps), 9), ((None, None, None), 17)):
        init = c["init"] if rays == 9 else None
        same(*(f.causal_conv_fwd(c["x"], c["w"], c["b"], init, *rows, rays, 4, True) for f in (ext, ct)))
        same(*(f.causal_conv_bwd(c["gy"], c["gf"] if init is not None else None, c["x"], c["w"], c["b"], init, *rows, rays, 4, True, True, True,
                                 init is not None) for f in (ext, ct)))
    same(*((f.causal_conv_step(c["x"][:9], c["init"], c["w"], c["b"], 4, to), to) for f, to in ((ext, c["init"].clone()), (ct, c["init"].clone()))))
    c = scan_inputs(85, 9, 24, 16, torch.float16)
    flat = [c[k] for k in ("u", "delta", "z", "B", "C", "A", "D", "bias")]
    order, other = ext.ray_order(info, 85), ct.ray_order(info, 85)
    assert torch.equal(order.sort()[0], other.sort()[0])
    a, b = (f.selective_scan_fwd(*flat, c["init"], info, *maps, None, 9, True, True, True) for f in (ext, ct))
    same(a[:2], b[:2])
    grads = [f.selective_scan_bwd(c["gy"], c["gf"], *flat, c["init"], kept, info, *maps, o, 9, True)
             for f, kept, o in ((ext, a[2], None), (ct, b[2], None), (ext, a[2], order), (ct, b[2], other))]
    for g in grads[1:]:                                               # the dealing order leaves no trace in the results
        same(grads[0], g)
    same(a[:2], ext.selective_scan_fwd(*flat, c["init"], info, *maps, order, 9, True, True, True)[:2])
    first = [t[:9] if t.shape[0] == 85 else t for t in flat]
    same(*((f.selective_scan_step(*first, c["init"], True, to), to) for f, to in ((ext, c["init"].clone()), (ct, c["init"].clone()))))


@pytest.mark.parametrize("n_rays", [1, 7, 1024, 3001])
def test_ray_order(n_rays):
    """every ray once, longer classes first"""
    from nerfacc_amd import cuda as C

    lens = torch.randint(0, 200, (n_rays,), generator=torch.Generator().manual_seed(n_rays))
    lens[torch.rand(n_rays, generator=torch.Generator().manual_seed(1)) < 0.3] = 0
    order = C.ray_order(packed(lens.tolist()), int(lens.sum())).long().cpu()
    assert order.sort()[0].tolist() == list(range(n_rays))
    cls = (lens.float() * (torch.tensor(32.0) / (lens.max() + 1).float())).int().clamp(max=31)[order]
    assert (cls[1:] <= cls[:-1]).all()


def test_scan_of_many_rays():
    """enough rays for the dealing order (and more than one ray per wave place)"""
    lens = torch.randint(0, 9, (1500,), generator=torch.Generator().manual_seed(4)).tolist()
    check_scan(scan_inputs(sum(lens) + 5, 1500, 3, 4, torch.bfloat16, seed=6), packed(lens))


def test_python_and_extension_steps_agree(monkeypatch):
    """the operators as one call of the extension and as the Python steps of the ctypes face: the same bits, gradients included"""
    import nerfacc_amd as nerfacc
    from nerfacc_amd import dense

    c, info = layer_inputs(80, torch.bfloat16, seed=3), packed(LENS)
    gy = torch.randn(80, 24, generator=generator(7), device=DEV).bfloat16()
    s = scan_inputs(80, 9, 24, 16, torch.float32, seed=2)
    k = conv_inputs(80, 9, 24, 4, torch.float32, seed=2, state=True)

    def everything():
        own = {n: v.detach().requires_grad_(True) for n, v in c.items()}
        out = layer(own, info)
        res = [out.detach(), *torch.autograd.grad(out, list(own.values()), gy)]
        own = {n: s[n].detach().requires_grad_(True) for n in NAMES}
        for outs in (call_scan(s, own, info), call_scan(s, own, info)[:1], call_scan(s, own, info)[1:]):      # both results used, or one
            gs = [s["gy"] if o.dim() == 2 else s["gf"] for o in outs]
            res += [g for g in torch.autograd.grad(outs, list(own.values()), gs, allow_unused=True) if g is not None]
        x, w, init = (k[n].detach().requires_grad_(True) for n in ("x", "w", "init"))
        for w_, b_ in ((w, k["b"]), (k["w"], None)):
            outs = nerfacc.causal_conv(x, w_, b_, packed_info=info, initial_state=init, return_final_state=True)
            res += torch.autograd.grad(outs, [t for t in (x, w_, init) if t.requires_grad], [k["gy"], k["gf"]])
        with torch.no_grad():
            res += [*nerfacc.causal_conv_step(k["x"][:9], k["init"], k["w"], k["b"]),
                    *nerfacc.selective_scan_step(s["u"][:9], s["delta"][:9], s["A"], s["B"][:9], s["C"][:9], s["init"], D=s["D"], delta_bias=s["bias"],
                                                 delta_softplus=True)]
        return res

    a = everything()
    monkeypatch.setattr(dense, "_EXT", False)
    b = everything()
    assert len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


def test_steps_refuse_gradients_and_overlapping_states(monkeypatch):
    import nerfacc_amd as nerfacc
    from nerfacc_amd import dense

    for ext in (None, False):
        monkeypatch.setattr(dense, "_EXT", ext)
        w, A = torch.rand(8, 4, device=DEV), torch.rand(8, 4, device=DEV)
        x, bc = torch.rand(2, 8, device=DEV), torch.rand(2, 4, device=DEV)
        pool, wide = torch.rand(3, 3, 8, device=DEV), torch.rand(3, 8, 4, device=DEV)
        with pytest.raises(RuntimeError, match="not differentiable"):
            nerfacc.causal_conv_step(x, pool[:2], w.clone().requires_grad_(True))
        with pytest.raises(RuntimeError, match="not differentiable"):
            nerfacc.selective_scan_step(x, x, A, bc, bc, wide[:2].clone().requires_grad_(True))
        with pytest.raises(ValueError, match="overlaps"):
            nerfacc.causal_conv_step(x, pool[:2], w, out_state=pool[1:])
        with pytest.raises(ValueError, match="overlaps"):
            nerfacc.selective_scan_step(x, x, A, bc, bc, wide[:2], out_state=wide[1:])
        with pytest.raises(ValueError, match="contiguous"):
            nerfacc.causal_conv_step(x, pool[:2], w, out_state=torch.rand(2, 8, 3, device=DEV).transpose(1, 2))
        before = pool._version
        nerfacc.causal_conv_step(x, pool[:2], w, out_state=pool[:2])
        assert pool._version > before                                 # autograd and views see the write


def test_differentiating_twice_is_refused(monkeypatch):
    import nerfacc_amd as nerfacc
    from nerfacc_amd import dense

    for ext in (None, False):
        monkeypatch.setattr(dense, "_EXT", ext)
        x = torch.rand(4, 8, device=DEV, requires_grad=True)
        w = torch.rand(8, 8, device=DEV)
        gy = torch.rand(4, 8, device=DEV, requires_grad=True)
        gx = torch.autograd.grad(nerfacc.linear(x, w, activation="silu"), x, gy, create_graph=True)[0]
        with pytest.raises(RuntimeError, match="once_differentiable"):
            gx.sum().backward()


def test_offsets_beyond_32_bits():
    """tensors of more than 2^31 numbers: the last rays are what they give alone"""
    import nerfacc_amd as nerfacc

    rays, n, d = 2100, 1000, 1040
    x = torch.randn(64, n, d, generator=generator(0), device=DEV).bfloat16().repeat(33, 1, 1)[:rays]
    assert x.numel() > 1 << 31
    w = torch.randn(d, 4, generator=generator(1), device=DEV).bfloat16()
    assert torch.equal(nerfacc.causal_conv(x, w, activation="silu")[-2:], nerfacc.causal_conv(x[-2:], w, activation="silu"))
    A, bc = -torch.rand(d, 1, generator=generator(2), device=DEV), torch.randn(rays, n, 1, generator=generator(3), device=DEV).bfloat16()
    out = nerfacc.selective_scan(x, x, A, bc, bc, delta_softplus=True)
    tail = nerfacc.selective_scan(x[-70:], x[-70:], A, bc[-70:], bc[-70:], delta_softplus=True)
    assert torch.equal(out[-70:], tail)                               # (70 rays: whole ones there too)


def test_docstring_examples():
    import nerfacc_amd as nerfacc

    info = torch.tensor([[0, 2], [2, 1]], device=DEV)
    x = torch.tensor([[1.], [2.], [3.]], device=DEV)
    assert nerfacc.causal_conv(x, torch.tensor([[1., 10.]], device=DEV), packed_info=info).flatten().tolist() == [10.0, 21.0, 30.0]
    y, state = nerfacc.causal_conv_step(torch.tensor([[3.]], device=DEV), torch.tensor([[[2.]]], device=DEV), torch.tensor([[1., 10.]], device=DEV))
    assert y.tolist() == [[32.0]] and state.tolist() == [[[3.0]]]
    one = torch.ones(3, 1, device=DEV)
    assert nerfacc.selective_scan(one, one, torch.zeros(1, 1, device=DEV), one, one, packed_info=info).flatten().tolist() == [1.0, 2.0, 1.0]


def test_scan_cut_into_longer_chunks():
    """enough channels that the forward pass takes chunks of its own length, with a last one that is not whole; packed rays of which one is
    much longer than the mean"""
    check_scan(scan_inputs(3 * 1400, 3, 4096, 4, torch.bfloat16, seed=7), shape=(3, 1400, 4096))
    lens = [3] * 20 + [1500] + [0, 5]
    check_scan(scan_inputs(sum(lens), len(lens), 6, 16, torch.float32, seed=8), packed(lens))
