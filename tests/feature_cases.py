"""Plain 64-bit forms of the operators along rays, one row at a time, and the size of their sums (for tolerances)."""
import torch


def rows_of(info, batched=None):
    """list of (start, count) of a packed_info tensor, or of `batched` = (n_rays, n)"""
    if batched is not None:
        return [(r * batched[1], batched[1]) for r in range(batched[0])]
    return [tuple(p) for p in info.tolist()]


def conv(x, w, b, act, seqs, init):
    """outputs (rows of no sequence: 0) and final states, in the types given"""
    width, out, finals = w.shape[1], {}, []
    for r, (start, n) in enumerate(seqs):
        head = init[r] if init is not None else x.new_zeros((width - 1, x.shape[1]))
        line = torch.cat([head, x[start:start + n]])
        z = sum(line[j:j + n] * w[:, j] for j in range(width))
        z = z if b is None else z + b
        out[r] = torch.nn.functional.silu(z) if act == "silu" else z
        finals.append(line[n:])
    return place(out, seqs, x), torch.stack(finals) if finals else x.new_zeros((0, width - 1, x.shape[1]))


def place(parts, seqs, like):
    """the sequences' rows at their places in an array like `like`, zeros elsewhere"""
    out = torch.zeros_like(like)
    index = torch.cat([torch.arange(s, s + n, device=like.device) for s, n in seqs] or [torch.empty(0, dtype=torch.long, device=like.device)])
    return out.index_copy(0, index, torch.cat([parts[r] for r in range(len(seqs))]).to(like.dtype)) if index.numel() else out


def scan(u, raw, A, B, C, D, z, softplus, seqs, init):
    """outputs and final states by the recurrence; raw = delta + bias"""
    step = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    out, finals = {}, []
    for r, (start, n) in enumerate(seqs):
        h = init[r] if init is not None else u.new_zeros(A.shape)
        ys = []
        for t in range(start, start + n):
            h = torch.exp(step[t][:, None] * A) * h + (step[t] * u[t])[:, None] * B[t]
            ys.append(h @ C[t])
        finals.append(h)
        out[r] = torch.stack(ys) if ys else u.new_zeros((0, u.shape[1]))
    y = place(out, seqs, u)
    y = y if D is None else y + place({r: D * u[s:s + n] for r, (s, n) in enumerate(seqs)}, seqs, u)
    y = y if z is None else y * torch.nn.functional.silu(z)
    covered = place({r: torch.ones_like(u[s:s + n]) for r, (s, n) in enumerate(seqs)}, seqs, u)
    return torch.where(covered > 0, y, torch.zeros_like(y)), torch.stack(finals) if finals else u.new_zeros((0, *A.shape))


def scan_sizes(u, raw, A, B, C, D, z, softplus, seqs, init, gy, gfinal):
    """the sums behind outputs and gradients with every term's absolute value: what rounding errors are relative to.  Keys: out, final,
    u, delta, A, B, C, D, z, bias, init."""
    step = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw.abs()
    decay = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    u, B, C, gy = u.abs(), B.abs(), C.abs(), gy.abs()
    Aa = A.abs()
    D = torch.zeros_like(A[:, 0]) if D is None else D.abs()
    gate = torch.ones_like(u) if z is None else torch.nn.functional.silu(z).abs()
    zz = torch.zeros_like(u) if z is None else z
    gate_slope = (torch.sigmoid(zz) * (1 + zz.abs() * torch.sigmoid(-zz)))
    size = {k: torch.zeros_like(v) for k, v in (("out", u), ("u", u), ("delta", u), ("z", u), ("B", B), ("C", C), ("A", A))}
    size["D"], size["bias"] = torch.zeros_like(D), torch.zeros_like(D)
    size["final"], size["init"] = (u.new_zeros((len(seqs), *A.shape)) for _ in range(2))
    for r, (start, n) in enumerate(seqs):
        h = init[r].abs() if init is not None else u.new_zeros(A.shape)
        states = [h]
        for t in range(start, start + n):
            h = torch.exp(decay[t][:, None] * A) * h + (step[t] * u[t])[:, None] * B[t]
            states.append(h)
        size["final"][r] = h
        G = gfinal[r].abs() if gfinal is not None else torch.zeros_like(h)
        for k in range(n - 1, -1, -1):
            t = start + k
            h, before = states[k + 1], states[k]
            a = torch.exp(decay[t][:, None] * A)
            y = h @ C[t] + D * u[t]
            dy = gy[t] * gate[t]
            G = G + dy[:, None] * C[t]
            size["out"][t] = y * gate[t]
            size["z"][t] = gy[t] * y * gate_slope[t]
            size["C"][t] = (dy[:, None] * h).sum(0)
            size["B"][t] = (G * (step[t] * u[t])[:, None]).sum(0)
            size["u"][t] = step[t] * (G * B[t]).sum(-1) + D * dy
            through = G * a * before
            size["delta"][t] = slope[t] * ((through * Aa).sum(-1) + u[t] * (G * B[t]).sum(-1))
            size["A"] += through * step[t][:, None]
            size["D"] += dy * u[t]
            size["bias"] += size["delta"][t]
            G = G * a
        size["init"][r] = G
    return size
