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


# ------------------------------------------------------------------------------------------------------------------ values
@pytest.mark.parametrize("rays,n", [(1, 300), (2, 700)])
def test_scan_of_growing_states(rays, n):
    """positive A: a chunk's decay overflows 32 bits while there is no state yet, or a tiny one, and the sum itself is small"""
    import nerfacc_amd as nerfacc

    d, s = 6, 4
    step, A = torch.ones(rays, n, d, device=DEV), torch.full((d, s), 3.0, device=DEV)
    u = torch.zeros(rays, n, d, device=DEV)
    u[:, -3:] = 1.0
    B = C = torch.ones(rays, n, s, device=DEV)
    own = [t.clone().requires_grad_(True) for t in (u, step)]
    out, end = nerfacc.selective_scan(own[0], own[1], A, B, C, return_final_state=True)
    e = torch.exp(torch.tensor(3.0)).item()
    want = torch.tensor([1.0, 1 + e, 1 + e + e * e], device=DEV) * s
    assert not out[:, :-3].any()
    assert torch.allclose(out[:, -3:], want[None, :, None].expand(rays, 3, d), rtol=1e-5) and torch.allclose(end, want[-1].expand_as(end) / s, rtol=1e-5)
    # backwards the same: a gradient that only the first rows' states could see
    gy = torch.zeros_like(out)
    gy[:, :2] = 1.0
    gu, _ = torch.autograd.grad(out, own, gy)
    assert not gu[:, 2:].any() and torch.allclose(gu[:, 1], torch.full_like(gu[:, 1], s), rtol=1e-5)
    assert torch.allclose(gu[:, 0], torch.full_like(gu[:, 0], s * (1 + e)), rtol=1e-5)
    # a tiny initial state that grows into an ordinary number: e^(0.15 n) 1e-25 over more rows than a chunk has
    init = torch.full((rays, d, s), 1e-25, device=DEV)
    A = torch.full((d, s), 70.0 / n, device=DEV)
    out = nerfacc.selective_scan(torch.zeros_like(u), step, A, B, C, initial_state=init)
    ref = s * 1e-25 * torch.exp(70.0 / n * torch.arange(1, n + 1, device=DEV, dtype=torch.float64))
    assert torch.allclose(out.double(), ref[None, :, None].expand(rays, n, d), rtol=(16 + 3 * n + 70 * 4) * 2.0**-24, atol=0)


def infinite_inputs(states, n, skip):
    import nerfacc_amd as nerfacc

    d = 5
    A, one = -torch.rand(d, states, generator=generator(0), device=DEV), torch.ones(2, n, states, device=DEV)
    u, dt = normal(2, n, d, seed=1), torch.rand(2, n, d, generator=generator(2), device=DEV) + 0.1
    D = torch.ones(d, device=DEV) if skip else None
    clean = nerfacc.selective_scan(u, dt, A, one, one, D=D)
    step, _ = nerfacc.selective_scan_step(u[:, 4], dt[:, 4], A, one[:, 4], one[:, 4], torch.zeros(2, d, states, device=DEV), D=D)
    u[1, 4, 2] = float("inf")
    out, end = nerfacc.selective_scan(u, dt, A, one, one, D=D, return_final_state=True)
    assert out[1, 4:, 2].isposinf().all() and end[1, 2].isposinf().all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[1, 4:, 2] = False
    assert torch.equal(out[keep], clean[keep])
    got, _ = nerfacc.selective_scan_step(u[:, 4], dt[:, 4], A, one[:, 4], one[:, 4], torch.zeros(2, d, states, device=DEV), D=D)
    assert got[1, 2].isposinf() and torch.equal(got[0], step[0])
    u[1, 4, 2] = 1.0
    own = [t.clone().requires_grad_(True) for t in (u, dt)]
    gy = torch.ones_like(out)
    gy[1, 10, 3] = float("inf")
    gu, _ = torch.autograd.grad(nerfacc.selective_scan(*own, A, one, one, D=D), own, gy)
    assert gu[1, :11, 3].isposinf().all() and gu[1, 11:].isfinite().all() and gu[0].isfinite().all()


@pytest.mark.parametrize("states", [4, 16, 32])
@pytest.mark.parametrize("n", [20, 400])
@pytest.mark.parametrize("skip", [False, True])
def test_scan_of_infinite_inputs(states, n, skip):
    """inf is inf, and a D that is not there adds nothing"""
    infinite_inputs(states, n, skip)


@pytest.mark.parametrize("states", [1, 2, 3, 5, 9, 20])
@pytest.mark.parametrize("n", [20, 400])
@pytest.mark.parametrize("skip", [False, True])
def test_scan_of_infinite_inputs_with_states_that_fill_no_power_of_two(states, n, skip):
    """places of no state add nothing either"""
    infinite_inputs(states, n, skip)


# -------------------------------------------------------------------------------------------------------------- derivatives
def scan_arguments(n=6, d=8, s=4):
    return dict(inputs=normal(1, n, d), delta=normal(1, n, d, seed=1).abs(), A=-normal(d, s, seed=2).abs(), B=normal(1, n, s, seed=3), C=normal(1, n, s, seed=4),
                D=normal(d, seed=5), gate=normal(1, n, d, seed=6), delta_bias=normal(d, seed=7), initial_state=normal(1, d, s, seed=8))


def conv_arguments(n=6, d=8):
    return dict(inputs=normal(1, n, d), weight=normal(d, 4, seed=1), bias=normal(d, seed=2), initial_state=normal(1, 3, d, seed=3))


@pytest.mark.parametrize("python", [False, True])
def test_forward_mode_is_refused(python, monkeypatch):
    import torch.autograd.forward_ad as fwd

    import nerfacc_amd as nerfacc
    from nerfacc_amd import dense

    if python:
        monkeypatch.setattr(dense, "_EXT", False)
    steps = [(nerfacc.causal_conv_step, {**{k: v[:, 0] if k == "inputs" else v for k, v in conv_arguments().items()}}),
             (nerfacc.selective_scan_step, {k: v[:, 0] if k in ("inputs", "delta", "B", "C", "gate") else v for k, v in scan_arguments().items()})]
    for _, kw in steps:
        kw["state"] = kw.pop("initial_state")
    for call, kw in [(nerfacc.causal_conv, conv_arguments()), (nerfacc.selective_scan, scan_arguments()), *steps]:
        call(**kw)
        for k in kw:
            with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
                call(**{**kw, k: fwd.make_dual(kw[k], torch.ones_like(kw[k]))})


@pytest.mark.parametrize("python", [False, True])
def test_a_penalty_on_the_gradient_is_refused(python, monkeypatch):
    import nerfacc_amd as nerfacc
    from nerfacc_amd import dense

    if python:
        monkeypatch.setattr(dense, "_EXT", False)
    for call, kw in ((nerfacc.causal_conv, conv_arguments()), (nerfacc.selective_scan, scan_arguments())):
        own = {k: v.requires_grad_(True) for k, v in kw.items()}
        out = call(**own)
        for k, g in zip(own, torch.autograd.grad(out, list(own.values()), torch.ones_like(out), create_graph=True)):
            if k == "bias":
                continue                                              # (a sum of dy: it depends on nothing that is learnt)
            assert g.requires_grad, k
            with pytest.raises(RuntimeError, match="once_differentiable"):
                g.square().sum().backward(retain_graph=True)


@pytest.mark.parametrize("python", [False, True])
def test_packed_info_changed_between_the_passes_is_noticed(python, monkeypatch):
    import nerfacc_amd as nerfacc
    from nerfacc_amd import dense

    if python:
        monkeypatch.setattr(dense, "_EXT", False)
    for call, kw in ((nerfacc.causal_conv, conv_arguments()), (nerfacc.selective_scan, scan_arguments())):
        kw = {k: v[0] if v.dim() == 3 and k != "initial_state" else v for k, v in kw.items()}
        x, info = kw.pop("inputs").requires_grad_(True), torch.tensor([[0, 6]], device=DEV)
        out = call(x, packed_info=info, **kw)
        info[0, 1] = 3
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


# ------------------------------------------------------------------------------------------------------------------- steps
@pytest.mark.parametrize("python", [False, True])
def test_steps_refuse_a_state_that_would_overwrite_their_inputs(python, monkeypatch):
    import nerfacc_amd as nerfacc
    from nerfacc_amd import dense

    if python:
        monkeypatch.setattr(dense, "_EXT", False)
    pool = normal(4, 3, 8)
    with pytest.raises(ValueError, match="overlaps"):
        nerfacc.causal_conv_step(pool[2:, 0], pool[:2].clone(), normal(8, 4), out_state=pool[2:])
    with pytest.raises(ValueError, match="overlaps"):
        nerfacc.causal_conv_step(normal(2, 8), pool[:2], pool.view(-1)[4:36].view(8, 4), out_state=pool[:2])
    pool, A, bc, x = normal(6, 8, 4), normal(8, 4), normal(2, 4), normal(2, 8)
    flat = pool.view(-1)
    for kw in (dict(inputs=flat[8:24].view(2, 8)), dict(delta=flat[:16].view(2, 8)), dict(B=flat[60:68].view(2, 4)), dict(C=flat[:8].view(2, 4)),
               dict(A=flat[32:64].view(8, 4)), dict(D=flat[:8]), dict(gate=flat[40:56].view(2, 8)), dict(delta_bias=flat[56:64])):
        with pytest.raises(ValueError, match="overlaps"):
            nerfacc.selective_scan_step(**{**dict(inputs=x, delta=x, A=A, B=bc, C=bc, state=pool[:2]), **kw}, out_state=pool[:2])
    # neighbours that share no memory are fine
    nerfacc.selective_scan_step(flat[64:80].view(2, 8), x, A, bc, bc, pool[:2], out_state=pool[:2])


# ---------------------------------------------------------------------------------------------------------------- C entries
def test_gradients_of_calls_without_rows_are_written():
    """zeros, and the final state's gradient for the initial one"""
    import ctypes

    from nerfacc_amd.cuda import _backend

    L, S, stream = _backend.load_library(), _backend._STRUCTS, torch.cuda.current_stream().cuda_stream
    dirty = lambda *shape, dtype=torch.float32: torch.full(shape, 7.0, device=DEV, dtype=dtype)  # noqa: E731
    for code, dt in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        w, gw, gb = normal(5, 3).to(dt), dirty(5, 3, dtype=dt), dirty(5, dtype=dt)
        a = S["nfa_linear_args"](rows=0, in_features=3, out_features=5, dtype=code, activation=1, weight=w.data_ptr())
        a.grad_outputs = a.inputs = w.data_ptr()
        assert L.nfa_linear_bwd(ctypes.byref(a), w.data_ptr(), None, gw.data_ptr(), gb.data_ptr(), w.data_ptr(), stream) == 0
        assert not gw.any() and not gb.any()
        w, gw, gb, gi, gf, init = normal(5, 4).to(dt), dirty(5, 4, dtype=dt), dirty(5, dtype=dt), dirty(2, 3, 5, dtype=dt), normal(2, 3, 5).to(dt), normal(2, 3, 5).to(dt)
        a = S["nfa_causal_conv_args"](n_rays=2, rows=0, channels=5, width=4, dtype=code, weight=w.data_ptr(), initial_state=init.data_ptr(),
                                      grad_final_state=gf.data_ptr())
        assert L.nfa_causal_conv_bwd(ctypes.byref(a), None, gw.data_ptr(), gb.data_ptr(), gi.data_ptr(), None, stream) == 0
        assert not gw.any() and not gb.any() and torch.equal(gi, gf)
        for rays, rows, final in ((2, 0, True), (2, 0, False), (0, 6, False)):
            A, init, gf, info = normal(5, 4), normal(2, 5, 4), normal(2, 5, 4), torch.zeros(1, 2, dtype=torch.int64, device=DEV)
            x, bc, pos = normal(6, 5).to(dt), normal(6, 4).to(dt), torch.full((6,), -1, dtype=torch.int32, device=DEV)
            g = dict(inputs=dirty(6, 5, dtype=dt), delta=dirty(6, 5, dtype=dt), gate=dirty(6, 5, dtype=dt), B=dirty(6, 4, dtype=dt), C=dirty(6, 4, dtype=dt),
                     A=dirty(5, 4), D=dirty(5), delta_bias=dirty(5), initial_state=dirty(2, 5, 4))
            a = S["nfa_selective_scan_args"](n_rays=rays, rows=rows, channels=5, states=4, dtype=code, A=A.data_ptr(), D=A.data_ptr(), delta_bias=A.data_ptr(),
                                             inputs=x.data_ptr(), delta=x.data_ptr(), gate=x.data_ptr(), B=bc.data_ptr(), C=bc.data_ptr(), inputs_stride=5,
                                             delta_stride=5, gate_stride=5, B_stride=4, C_stride=4, initial_state=init.data_ptr(), packed_info=info.data_ptr(),
                                             row_ray=pos.data_ptr(), row_pos=pos.data_ptr(), grad_final_state=gf.data_ptr() if final else None)
            gr = S["nfa_selective_scan_grads"](**{k: v.data_ptr() for k, v in g.items()})
            assert L.nfa_selective_scan_bwd(ctypes.byref(a), None, ctypes.byref(gr), None, stream) == 0
            torch.cuda.synchronize()
            for k, v in g.items():
                if k == "initial_state":
                    assert torch.equal(v, gf) if final else (not v.any() if rays else v.eq(7).all())
                elif k in ("A", "D", "delta_bias"):
                    assert not v.any(), k
                else:
                    assert not v[:rows].any() and v[rows:].eq(7).all(), k


# --------------------------------------------------------------------------------------------------------------- workspaces
@pytest.mark.parametrize("states,channels", [(100, 70), (256, 70), (256, 33), (129, 129)])
@pytest.mark.parametrize("lens", [[9, 0, 11], [130, 1, 200]])
def test_scan_of_many_states_and_many_channels(states, channels, lens):
    """sums over channels that one wave takes a block of channels at a time"""
    from test_gpu_selective import check_scan, packed, scan_inputs

    check_scan(scan_inputs(sum(lens), len(lens), channels, states, torch.float32, seed=states), packed(lens))
