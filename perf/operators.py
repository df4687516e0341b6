"""The feature operators between sampling and rendering, as a user's program calls them: a dense layer with its epilogue
(`nerfacc_amd.linear`), the short causal convolution along each ray (`causal_conv`, `causal_conv_step`) and the selective
state space scan along each ray (`selective_scan`, `selective_scan_step`).

`own` chooses between the framework's calls and the same operators in elementary torch operations (32 bits, rounded once).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ACTIVATIONS = ("none", "relu", "sigmoid", "softplus", "silu", "gelu", "exp")


# ---------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    def linear(name, rows, k, n, dtype, act, residual, train, bias=True):
        return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "activation": act, "bias": bias,
                "residual": residual, "train": train}

    def conv(name, rays, rows, d, width, dtype, packed, state, train, act="silu", bias=True):
        return {"name": name, "op": "conv", "rays": rays, "rows": rows, "d": d, "width": width, "dtype": dtype, "packed": packed,
                "state": state, "train": train, "activation": act, "bias": bias}

    def scan(name, rays, rows, d, s, dtype, packed, state, train, gate=True, softplus=True, skip=True, sliced=False):
        return {"name": name, "op": "scan", "rays": rays, "rows": rows, "d": d, "s": s, "dtype": dtype, "packed": packed,
                "state": state, "train": train, "gate": gate, "softplus": softplus, "skip": skip, "sliced": sliced}

    return [
        # one query of a field's hidden layer: the smallest call, all latency
        linear("linear_one_row", 1, 256, 256, "bfloat16", "relu", False, False),
        # the first layer of the grid + MLP field (8 features to 32) on a training batch of 2^18 samples, in 32 bits
        linear("linear_grid_features_train", 1 << 18, 8, 32, "float32", "relu", False, True),
        # a hidden layer of a 256-wide residual field on the same batch
        linear("linear_hidden_train", 1 << 18, 256, 256, "bfloat16", "relu", True, True),
        # an encoded position of 63 numbers into an odd width, an odd number of samples: nothing is aligned
        linear("linear_odd_train", 100003, 63, 65, "float16", "softplus", False, True),
        # a wide layer over a frame's samples, inference: the one case that the matrix units bound
        linear("linear_wide", 1 << 16, 1024, 1024, "bfloat16", "silu", False, False),
        # features of a training batch of rays, mixed along each ray before the scan
        conv("conv_rays_train", 4096, 1 << 18, 128, 4, "bfloat16", True, False, True),
        # one long sequence, with the state that its continuation needs
        conv("conv_prompt", 1, 1 << 15, 2048, 4, "float16", False, True, False),
        # one more sample of each of 256 rays
        {"name": "conv_step", "op": "conv_step", "rays": 256, "d": 2048, "width": 4, "dtype": "bfloat16", "activation": "silu", "bias": True},
        # the scan of the same training batch of rays: ragged, some rays empty
        scan("scan_rays_train", 4096, 1 << 18, 64, 16, "bfloat16", True, False, True),
        # two long sequences trained in 32 bits, with a state in and out: few rows, a long axis
        scan("scan_long_train", 2, 1 << 14, 512, 16, "float32", False, True, True, gate=False),
        # one long sequence, the features and the gate as two halves of one projection
        scan("scan_prompt", 1, 1 << 15, 1024, 16, "bfloat16", False, True, False, sliced=True),
        # one more sample of each of 256 rays
        {"name": "scan_step", "op": "scan_step", "rays": 256, "d": 1024, "s": 16, "dtype": "bfloat16", "gate": True, "softplus": True, "skip": True},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    def flag(p=0.5):
        return rng.random() < p

    case = {"op": rng.choice(["linear", "linear", "linear", "conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step"]),
            "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    if case["op"] == "linear":
        k, n = log(1, 1024), log(1, 1024)
        if flag():
            k, n = 8 * -(-k // 8), 8 * -(-n // 8)
        rows = log(1, min(1 << 18, (1 << 36) // (3 * k * n), (1 << 27) // (k + n)))
        return {**case, "rows": rows, "k": k, "n": n, "activation": rng.choice(ACTIVATIONS), "bias": flag(0.8), "residual": flag(0.3), "train": flag()}
    if case["op"] == "conv":
        d = log(1, 2048)
        if flag():
            d = 8 * -(-d // 8)
        rows = log(1, min(1 << 18, (1 << 26) // d))
        packed = flag()
        rays = log(1, min(4096, rows))
        rows = rows if packed else rays * (rows // rays)
        return {**case, "rays": rays, "rows": rows, "d": d, "width": rng.choice([2, 3, 4]), "packed": packed, "state": flag(), "train": flag(),
                "activation": rng.choice(["none", "silu"]), "bias": flag()}
    if case["op"] == "conv_step":
        return {**case, "rays": log(1, 1024), "d": log(1, 2048), "width": rng.choice([2, 3, 4]), "activation": rng.choice(["none", "silu"]),
                "bias": flag()}
    flags = {"gate": flag(), "softplus": flag(0.7), "skip": flag()}
    s = rng.choice([1, 4, 8, 16, 16, 16, log(1, 64)])
    if case["op"] == "scan_step":
        d = log(1, 2048)
        return {**case, "rays": log(1, min(1024, (1 << 22) // (d * s))), "d": d, "s": s, **flags}
    d = log(4, 1024)
    if flag():
        d = 16 * -(-d // 16)
    train = flag()
    rows = log(1, min(1 << 18, (1 << 27) // (d * s)))
    packed = flag()
    rays = log(1, min(4096, rows))
    rows = rows if packed else rays * (rows // rays)
    return {**case, "rays": rays, "rows": rows, "d": d, "s": s, "packed": packed, "state": flag(), "train": train, **flags, "sliced": flag(0.3)}


# ---------------------------------------------------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(case, seed):
    """rows of each sequence: equal ones, or a batch of rays of which a fifth hit nothing"""
    if not case["packed"]:
        return np.full(case["rays"], case["rows"] // case["rays"], np.int64)
    g = np.random.default_rng(seed)
    w = (0.05 + g.random(case["rays"])) * (g.random(case["rays"]) > 0.2)
    w[g.integers(case["rays"])] += 0.5
    ends = np.floor(np.cumsum(w) / w.sum() * case["rows"] + 0.5).astype(np.int64)
    ends[-1] = case["rows"]
    return np.diff(ends, prepend=0)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    train = case.get("train", False)

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0, dtype=torch.float32):
        return (torch.rand(shape, generator=g, device=DEV) * (hi - lo) + lo).to(dtype)

    s = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        s["x"], s["w"] = normal(m, k), uniform(n, k, lo=-1.7 / math.sqrt(k), hi=1.7 / math.sqrt(k), dtype=dt)
        s["b"] = normal(n, scale=0.1) if case["bias"] else None
        s["r"] = normal(m, n) if case["residual"] else None
        s["leaves"] = [t for t in (s["x"], s["w"], s["b"], s["r"]) if t is not None]
        if train:
            s["g"] = normal(m, n)
    elif case["op"] in ("conv", "conv_step"):
        d, w = case["d"], case["width"]
        s["w"] = uniform(d, w, lo=-1 / math.sqrt(w), hi=1 / math.sqrt(w), dtype=dt)
        s["b"] = normal(d, scale=0.1) if case["bias"] else None
        if case["op"] == "conv_step":
            s["x"], s["h0"] = normal(case["rays"], d), normal(case["rays"], w - 1, d)
            s["next"] = torch.empty_like(s["h0"])
            return s
        _sequences(s, case, seed)
        s["x"] = normal(*s["shape"], d)
        s["h0"] = normal(case["rays"], w - 1, d) if case["state"] else None
        s["leaves"] = [t for t in (s["x"], s["w"], s["b"], s["h0"]) if t is not None]
        if train:
            s["g"] = normal(*s["shape"], d)
            s["gh"] = normal(case["rays"], w - 1, d) if case["state"] else None
    else:
        d, n = case["d"], case["s"]
        if case["op"] == "scan":
            _sequences(s, case, seed)
        else:
            s["shape"] = (case["rays"],)
        # decays of 1 .. n per state with a spread over channels, steps of 0.001 .. 0.1: what such a layer starts from
        s["A"] = -(torch.arange(1, n + 1, device=DEV, dtype=torch.float32) * uniform(d, 1, lo=0.5, hi=1.5)).contiguous()
        step = torch.exp(uniform(d, lo=math.log(1e-3), hi=math.log(1e-1)))
        s["bias"] = step + torch.log(-torch.expm1(-step)) if case["softplus"] else None
        s["dt"] = normal(*s["shape"], d, scale=0.5) if case["softplus"] else (step * torch.exp(normal(*s["shape"], d, scale=0.3, dtype=torch.float32))).to(dt)
        if case.get("sliced"):
            both = normal(*s["shape"], 2 * d)
            s["u"], s["z"] = both[..., :d], (both[..., d:] if case["gate"] else None)
            bc = normal(*s["shape"], 2 * n)
            s["B"], s["C"] = bc[..., :n], bc[..., n:]
        else:
            s["u"], s["z"] = normal(*s["shape"], d), (normal(*s["shape"], d) if case["gate"] else None)
            s["B"], s["C"] = normal(*s["shape"], n), normal(*s["shape"], n)
        s["D"] = normal(d, dtype=torch.float32) if case["skip"] else None
        s["h0"] = normal(case["rays"], d, n, dtype=torch.float32) if case.get("state") or case["op"] == "scan_step" else None
        if case["op"] == "scan_step":
            s["next"] = torch.empty_like(s["h0"])
            return s
        s["leaves"] = [t for t in (s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["bias"], s["h0"]) if t is not None]
        if train:
            s["g"] = normal(*s["shape"], d)
            s["gh"] = normal(case["rays"], d, n, dtype=torch.float32) if case["state"] else None
    if train:
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


def _sequences(s, case, seed):
    lens = _lengths(case, seed)
    s["longest"] = int(lens.max())
    s["shape"] = (case["rows"],) if case["packed"] else (case["rays"], case["rows"] // case["rays"])
    starts = np.cumsum(lens) - lens
    s["info"] = torch.from_numpy(np.stack([starts, lens], -1)).to(DEV)


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _call(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


def _call(s):
    import nerfacc_amd as nerfacc

    c = s["case"]
    act = None if c.get("activation", "none") == "none" else c["activation"]
    info = s.get("info") if c.get("packed") else None
    if c["op"] == "linear":
        out = nerfacc.linear(s["x"], s["w"], s["b"], activation=act, residual=s["r"])
        return [out, *torch.autograd.grad(out, s["leaves"], s["g"])] if c["train"] else [out]
    if c["op"] == "conv_step":
        return list(nerfacc.causal_conv_step(s["x"], s["h0"], s["w"], s["b"], activation=act, out_state=s["next"]))
    if c["op"] == "conv":
        out = nerfacc.causal_conv(s["x"], s["w"], s["b"], activation=act, packed_info=info, initial_state=s["h0"],
                                  return_final_state=c["state"])
    elif c["op"] == "scan_step":
        return list(nerfacc.selective_scan_step(s["u"], s["dt"], s["A"], s["B"], s["C"], s["h0"], D=s["D"], gate=s["z"],
                                                delta_bias=s["bias"], delta_softplus=c["softplus"], out_state=s["next"]))
    else:
        out = nerfacc.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], gate=s["z"], delta_bias=s["bias"],
                                     delta_softplus=c["softplus"], packed_info=info, initial_state=s["h0"],
                                     return_final_state=c["state"])
    outs = list(out) if c["state"] else [out]
    if c["train"]:
        outs += torch.autograd.grad(outs, s["leaves"], [s["g"], s["gh"]] if c["state"] else [s["g"]])
    return outs


# -- the plain forms ----------------------------------------------------------------------------------------------------
def _act(name, z):
    """act(z) and its derivative"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "exp":
        e = torch.exp(z)
        return e, e
    sig = 1 / (1 + torch.exp(-z))
    if name == "sigmoid":
        return sig, sig * (1 - sig)
    if name == "softplus":
        return z.clamp(min=0) + torch.log1p(torch.exp(-z.abs())), sig
    if name == "silu":
        return z * sig, sig * (1 + z * (1 - sig))
    cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _plain_linear(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y, slope = _act(c["activation"], z)
    out = y if s["r"] is None else y + s["r"].float()
    if not c["train"]:
        return [out.to(dt)]
    dz = s["g"].float() * slope
    grads = [dz @ w, dz.t() @ x] + ([dz.sum(0)] if s["b"] is not None else []) + ([s["g"]] if s["r"] is not None else [])
    return [out.to(dt)] + [t.to(dt) for t in grads]


def _rows(s):
    """of every row: its sequence, its position in it, and how many rows follow it there"""
    lens = s["info"][:, 1]
    seq = torch.repeat_interleave(torch.arange(lens.numel(), device=DEV), lens, output_size=s["case"]["rows"])
    pos = torch.arange(s["case"]["rows"], device=DEV) - s["info"][seq, 0]
    return seq, pos, lens[seq] - 1 - pos


def _plain_conv(s):
    # every sequence behind its state's rows in one array: a convolution there is a sum over shifted views
    c, dt, d, w = s["case"], s["x"].dtype, s["case"]["d"], s["case"]["width"]
    rays, rows = c["rays"], c["rows"]
    seq, _, _ = _rows(s)
    at = torch.arange(rows, device=DEV) + (seq + 1) * (w - 1)
    heads = (s["info"][:, :1] + torch.arange(rays, device=DEV)[:, None] * (w - 1)) + torch.arange(w - 1, device=DEV)
    tails = heads + s["info"][:, 1:]
    ext = torch.zeros(rows + rays * (w - 1), d, device=DEV)
    ext[at] = s["x"].reshape(rows, d).float()
    if s["h0"] is not None:
        ext[heads] = s["h0"].float()
    taps = s["w"].float()
    z = (ext.unfold(0, w, 1)[at - (w - 1)] * taps).sum(-1)
    if s["b"] is not None:
        z = z + s["b"].float()
    y, slope = _act(c["activation"], z)
    outs = [y.view(s["x"].shape).to(dt)] + ([ext[tails].to(dt)] if c["state"] else [])
    if not c["train"]:
        return outs
    dz = s["g"].reshape(rows, d).float() * slope
    back = torch.zeros(ext.shape[0] + w - 1, d, device=DEV)
    back[at] = dz
    dext = (back.unfold(0, w, 1) * taps.flip(-1)).sum(-1)
    if c["state"]:
        dext[tails] = dext[tails] + s["gh"].float()
    dw = (ext.unfold(0, w, 1)[at - (w - 1)] * dz[..., None]).sum(0)
    grads = [dext[at].view(s["x"].shape), dw] + ([dz.sum(0)] if s["b"] is not None else []) + ([dext[heads]] if c["state"] else [])
    return outs + [t.to(dt) for t in grads]


def _plain_conv_step(s):
    dt = s["x"].dtype
    window = torch.cat([s["h0"], s["x"][:, None]], 1)
    z = (window.float() * s["w"].float().t()).sum(1)
    if s["b"] is not None:
        z = z + s["b"].float()
    return [_act(s["case"]["activation"], z)[0].to(dt), window[:, 1:]]


def _recurrence(a, b, pos, longest):
    """h[t] = a[t] h[t - 1] + b[t] within each sequence, by doubling"""
    k = 1
    while k < longest:
        m = (pos[k:] >= k)[:, None, None]
        b = torch.cat([b[:k], b[k:] + torch.where(m, a[k:] * b[:-k], 0.0)])
        a = torch.cat([a[:k], a[k:] * torch.where(m, a[:-k], 1.0)])
        k *= 2
    return b


def _scan_inputs(s):
    c = s["case"]
    d, n = c["d"], c["s"]
    flat = lambda t: t.reshape(-1, t.shape[-1]).float()  # noqa: E731
    u, raw, B, C = flat(s["u"]), flat(s["dt"]), flat(s["B"]), flat(s["C"])
    if s["bias"] is not None:
        raw = raw + s["bias"]
    step, slope = _act("softplus" if c["softplus"] else "none", raw)
    return d, n, u, step, slope, B, C, (None if s["z"] is None else flat(s["z"]))


def _plain_scan(s):
    c, dt = s["case"], s["u"].dtype
    d, n, u, step, slope, B, C, z = _scan_inputs(s)
    seq, pos, rest = _rows(s)
    first, last, full = (pos == 0).nonzero()[:, 0], (rest == 0).nonzero()[:, 0], (s["info"][:, 1] > 0).nonzero()[:, 0]
    a = torch.exp(step[:, :, None] * s["A"])
    b = (step * u)[:, :, None] * B[:, None, :]
    if s["h0"] is not None:
        b[first] += a[first] * s["h0"][full]
    h = _recurrence(a, b, pos, s["longest"])
    y = (h * C[:, None, :]).sum(-1)
    if s["D"] is not None:
        y = y + s["D"] * u
    gate, gate_slope = _act("silu", z) if z is not None else (None, None)
    out = y if z is None else y * gate
    outs = [out.view(s["u"].shape).to(dt)]
    if c["state"]:
        end = s["h0"].clone()
        end[full] = h[last]
        outs.append(end)
    if not c["train"]:
        return outs
    dout = s["g"].reshape(-1, d).float()
    dy = dout if z is None else dout * gate
    dh = dy[:, :, None] * C[:, None, :]
    if c["state"]:
        dh[last] += s["gh"][full]
    after = torch.cat([a[1:], torch.zeros_like(a[:1])])
    dh = _recurrence(after.flip(0), dh.flip(0), rest.flip(0), s["longest"]).flip(0)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[first] = s["h0"][full] if s["h0"] is not None else 0.0
    kept = dh * a * before                                   # dh/d(log a) times dh
    through = (dh * B[:, None, :]).sum(-1)
    du = step * through
    if s["D"] is not None:
        du = du + s["D"] * dy
    draw_ = ((kept * s["A"]).sum(-1) + u * through) * slope
    grads = [du.view(s["u"].shape).to(dt), draw_.view(s["u"].shape).to(dt), (kept * step[:, :, None]).sum(0),
             (dh * (step * u)[:, :, None]).sum(1).view(s["B"].shape).to(dt), (h * dy[:, :, None]).sum(1).view(s["B"].shape).to(dt)]
    if s["D"] is not None:
        grads.append((dy * u).sum(0))
    if z is not None:
        grads.append((dout * y * gate_slope).view(s["u"].shape).to(dt))
    if s["bias"] is not None:
        grads.append(draw_.sum(0))
    if c["state"]:
        dstate = s["gh"].clone()
        dstate[full] = dh[first] * a[first]
        grads.append(dstate)
    return outs + grads


def _plain_scan_step(s):
    _, _, u, step, _, B, C, z = _scan_inputs(s)
    h = torch.exp(step[:, :, None] * s["A"]) * s["h0"] + (step * u)[:, :, None] * B[:, None, :]
    y = (h * C[:, None, :]).sum(-1)
    if s["D"] is not None:
        y = y + s["D"] * u
    if z is not None:
        y = y * _act("silu", z)[0]
    return [y.to(s["u"].dtype), h]


_PLAIN = {"linear": _plain_linear, "conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_step": _plain_scan_step}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "linear":
        m, k, n, r = case["rows"], case["k"], case["n"], case["residual"]
        once = m * k + n * k + n * case["bias"] + m * n * r
        values = once + m * n
        if case["train"]:
            values += m * n + once - m * n * r             # the residual's gradient is the output's own
        return {"bytes": e * values, "flops": 2 * m * n * k * (3 if case["train"] else 1)}
    if case["op"] == "conv_step":
        r, d, w = case["rays"], case["d"], case["width"]
        return {"bytes": e * (2 * r * d + 2 * r * (w - 1) * d + d * w + d * case["bias"]), "flops": 2 * r * d * w}
    if case["op"] == "conv":
        rows, d, w = case["rows"], case["d"], case["width"]
        weights, state = d * w + d * case["bias"], 2 * case["rays"] * (w - 1) * d * case["state"]
        if not case["train"]:
            return {"bytes": e * (2 * rows * d + weights + state), "flops": 2 * rows * d * w}
        return {"bytes": e * (4 * rows * d + 2 * weights + 2 * state), "flops": 6 * rows * d * w}
    rows, d, n = case["rows" if case["op"] == "scan" else "rays"], case["d"], case["s"]
    each = 3 + case["gate"]                                 # features, steps, (gate), output
    weights = 4 * (d * n + d * case["skip"] + d * case["softplus"])
    if case["op"] == "scan_step":
        return {"bytes": e * rows * (each * d + 2 * n) + weights + 8 * rows * d * n, "flops": 7 * rows * d * n}
    state = 8 * case["rays"] * d * n * case["state"]
    if not case["train"]:
        return {"bytes": e * rows * (each * d + 2 * n) + weights + state, "flops": 7 * rows * d * n}
    return {"bytes": e * rows * ((2 * each) * d + 4 * n) + 2 * weights + 2 * state, "flops": 7 * rows * d * n + 14 * rows * d * n}


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda t: None if t is None else t.detach().double()  # noqa: E731
    acts = {"none": lambda v: v, "relu": torch.relu, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu, "exp": torch.exp,
            "gelu": torch.nn.functional.gelu, "softplus": lambda v: torch.logaddexp(v, torch.zeros_like(v))}
    act = acts[case.get("activation", "none")]
    train = case.get("train", False)

    if case["op"] == "linear":
        x, w, b, r = (wide(s[key]) for key in ("x", "w", "b", "r"))
        if case["rows"] * (case["k"] + case["n"]) > 1 << 28:
            return None
        leaves = [t.requires_grad_(train) for t in (x, w, b, r) if t is not None]
        out = act(torch.nn.functional.linear(x, w, b))
        out = out if r is None else out + r
        grads = torch.autograd.grad(out, leaves, wide(s["g"])) if train else ()
        return [out.detach(), *grads]

    if case["op"] == "conv_step":
        x, w, b, h = (wide(s[key]) for key in ("x", "w", "b", "h0"))
        window = torch.cat([h, x[:, None]], 1)
        z = torch.einsum("rwd,dw->rd", window, w) + (0 if b is None else b)
        return [act(z), window[:, 1:]]

    # sequences side by side, the longest first, one time step at a time over those that still run
    if case["op"] == "scan_step":
        rays, lens, starts, rows = case["rays"], np.ones(case["rays"], np.int64), np.arange(case["rays"]), case["rays"]
    else:
        info = s["info"].cpu().numpy()
        rays, starts, lens, rows = case["rays"], info[:, 0], info[:, 1], case["rows"]
    order = np.argsort(-lens, kind="stable")
    running = [int((lens > t).sum()) for t in range(int(lens.max()))]
    at = [torch.from_numpy(starts[order[:n]] + t).to(DEV) for t, n in enumerate(running)]
    back = torch.from_numpy(np.argsort(order, kind="stable")).to(DEV)
    place = torch.empty(rows, dtype=torch.long, device=DEV)
    place[torch.cat(at)] = torch.arange(rows, device=DEV)
    order = torch.from_numpy(order).to(DEV)
    flat = lambda t: t.reshape(rows, t.shape[-1])  # noqa: E731

    def ended(states):
        """the state of each sequence after its own last step, from the states after every step (shrinking prefixes)"""
        parts = [st[n:] for st, n in zip(states, running[1:] + [0])]
        return torch.cat([states[-1][:0]] + parts[::-1]) if len(parts) else states[0]

    if case["op"] == "conv":
        x, w, b, h0 = (wide(s[key]) for key in ("x", "w", "b", "h0"))
        leaves = [t.requires_grad_(train) for t in (x, w, b, h0) if t is not None]
        start = torch.zeros(rays, case["width"] - 1, case["d"], dtype=torch.float64, device=DEV) if h0 is None else h0
        width, d = case["width"], case["d"]
        # sequences laid out one behind the other, each after its state; the convolution is torch's own
        index = torch.cat([torch.cat([torch.arange(r * (width - 1), (r + 1) * (width - 1)), rays * (width - 1) + torch.arange(a, a + n)])
                           for r, (a, n) in enumerate(zip(starts.tolist(), lens.tolist()))]).to(DEV)
        line = torch.cat([start.reshape(-1, d), flat(x)])[index]
        where = torch.empty(rows + rays * (width - 1), dtype=torch.long, device=DEV)
        where[index] = torch.arange(index.numel(), device=DEV)
        z = sum(line[j:line.shape[0] - (width - 1) + j] * w[:, j] for j in range(width))
        z = z[where[rays * (width - 1):] - (width - 1)]
        out = act(z if b is None else z + b).view(s["x"].shape)
        outs = [out]
        if case["state"]:
            ends = torch.from_numpy(np.cumsum(lens + width - 1)).to(DEV)[:, None] + torch.arange(1 - width, 0, device=DEV)
            outs.append(line[ends])
        grads = torch.autograd.grad(outs, leaves, [wide(s["g"])] + ([wide(s["gh"])] if case["state"] else [])) if train else ()
        return [t.detach() for t in outs] + list(grads)

    if rows * case["d"] * case["s"] > 1 << 30 or len(running) > 40000:
        return None
    names = ("u", "dt", "A", "B", "C", "D", "z", "bias", "h0")
    v = {key: wide(s[key]) for key in names}
    leaves = [v[key].requires_grad_(train) for key in names if v[key] is not None]
    raw = v["dt"] if v["bias"] is None else v["dt"] + v["bias"]
    step = flat(acts["softplus"](raw) if case["softplus"] else raw)
    u, B, C = flat(v["u"]), flat(v["B"]), flat(v["C"])
    start = v["h0"] if v["h0"] is not None else torch.zeros(rays, case["d"], case["s"], dtype=torch.float64, device=DEV)
    first = start[order]
    h, states, ys = first, [], []
    for n, rows_t in zip(running, at):
        d_t = step[rows_t]
        h = torch.exp(d_t[:, :, None] * v["A"]) * h[:n] + (d_t * u[rows_t])[:, :, None] * B[rows_t][:, None, :]
        ys.append(torch.matmul(h, C[rows_t][:, :, None])[:, :, 0])
        states.append(h if case["op"] == "scan_step" or case.get("state") else None)
    y = torch.cat(ys)[place]
    y = y if v["D"] is None else y + v["D"] * u
    out = (y if v["z"] is None else y * torch.nn.functional.silu(flat(v["z"]))).view(s["u"].shape)
    outs = [out]
    if case["op"] == "scan_step" or case["state"]:
        done = ended(states)
        outs.append(torch.cat([done, first[done.shape[0]:]])[back])
    grads = torch.autograd.grad(outs, leaves, [wide(s["g"])] + ([wide(s["gh"])] if case["state"] else [])) if train else ()
    return [t.detach() for t in outs] + list(grads)
