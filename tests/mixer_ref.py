"""Plain 64-bit forms of linear attention and of the norms around a block, and the error bounds of their kernels."""
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}   # a rounding is off by at most this, relatively


def _pairs(t, H):
    return t.double().repeat_interleave(H // t.shape[1], 1)


def _fold(t, Hkv):
    B, H, L, D = t.shape
    return t.reshape(B, Hkv, H // Hkv, L, D).sum(2)


def attention(q, k, v, log_decay, scale, s0=None, lengths=None, dy=None, ds=None):
    """Definition over all pairs of positions.  Returns {name: (value, magnitude)}; a magnitude is the same expression
    with every factor replaced by its absolute value, what rounding errors are relative to."""
    B, H, L, D = q.shape
    Hkv, Dv = k.shape[1], v.shape[3]
    dev = q.device
    n = torch.full((B,), L, device=dev) if lengths is None else lengths.long().clamp(0, L)
    pos = torch.arange(L, device=dev)
    there = (pos[None] < n[:, None])[:, None, :, None]
    def clean(t):
        return torch.where(there, _pairs(t, H), 0.0)
    q, k, v = clean(q), clean(k), clean(v)
    a = log_decay.double().clamp(min=-1e30)[None, :, None, None]
    lag = (pos[:, None] - pos[None, :]).double()
    w = torch.where(lag >= 0, torch.exp(a * lag.clamp(min=0)), 0.0)
    grow = torch.exp(a * (pos + 1).double()[None, None, :, None])
    rest = torch.exp(a * (n[:, None] - 1 - pos[None]).clamp(min=0).double()[:, None, :, None])
    whole = torch.exp(a * n.double()[:, None, None, None])
    s0 = torch.zeros((B, H, D, Dv), dtype=torch.float64, device=dev) if s0 is None else s0.double()
    T = lambda t: t.transpose(2, 3)  # noqa: E731

    def forms(q, k, v, s0, dy, ds, sc):
        out = {}
        P = (q @ T(k)) * w
        out["y"] = sc * (P @ v + grow * (q @ s0)) * there
        out["state"] = T(k * rest) @ v + whole * s0
        if dy is not None:
            G = (dy @ T(v)) * w
            out["dq"] = sc * (G @ k + grow * (dy @ T(s0))) * there
            out["dk"] = _fold((sc * T(G) @ q + rest * (v @ T(ds))) * there, Hkv)
            out["dv"] = _fold((sc * T(P) @ dy + rest * (k @ ds)) * there, Hkv)
            out["ds0"] = sc * T(q * grow) @ dy + whole * ds
        return out

    if dy is not None:
        dy = torch.where(there, dy.double(), 0.0)
        ds = torch.zeros_like(s0) if ds is None else ds.double()
    val = forms(q, k, v, s0, dy, ds, scale)
    mag = forms(*(None if t is None else t.abs() for t in (q, k, v, s0, dy, ds)), abs(scale))
    return {name: (val[name], mag[name]) for name in val}


def attention_bound(name, value, mag, dtype, L, D, Dv, share=1):
    """Outputs are rounded once to their type.  With bf16 operands the tensor cores take one factor of each product pair
    (the products q.k, or the state) rounded to bf16: half a step of the magnitude, and half a step of that again in
    its second order.  Sums in 32 bits: no output's chain has more additions than max(D, Dv) for a product of two
    rows, 2 * 128 in a chunk, one or two for each of the chunks, and 64 for scales, segments and shared heads; each
    is off by at most 2^-23 (truncation) of the magnitude."""
    state = name in ("state", "ds0")
    out = HALF_STEP[torch.float32 if state else dtype]
    n = max(D, Dv) + 256 + 2 * (L // 32) + 64 + share
    tol = out * value.abs() + n * 2.0 ** -23 * mag
    if dtype == torch.bfloat16 and not state:
        tol = tol + 2.0 ** -8 * (1 + 2.0 ** -7) * mag
    return tol + 1e-30


def norm(x, y, gate, pw, w, scale, eps, groups, act, dim, dh=None, dn=None):
    """block_norm and its gradients by their formulas in 64 bits."""
    def last(t):
        if t is None:
            return None
        t = t.double()
        return t.transpose(1, 2) if dim == 1 and t.dim() == 3 else t

    def put(t):
        return t.transpose(1, 2) if dim == 1 and t.dim() == 3 else t

    x, y, gate, dh, dn = last(x), last(y), last(gate), last(dh), last(dn)
    pw, w = (None if t is None else t.double() for t in (pw, w))
    C = (y if y is not None else x).shape[-1]
    g = lambda t: t.reshape(t.shape[:-1] + (groups, C // groups))  # noqa: E731
    out = {}
    if y is not None:
        a = y
        if pw is not None:
            r1 = (g(y).square().mean(-1, keepdim=True) + eps) ** -0.5
            u = (g(y) * r1).reshape(y.shape)
            a = u * pw
        f, df = torch.ones_like(a), torch.zeros_like(a)
        if gate is not None:
            sg = torch.sigmoid(gate)
            f, df = {"silu": (gate * sg, sg * (1 + gate * (1 - sg))), "sigmoid": (sg, sg * (1 - sg)),
                     "none": (gate, torch.ones_like(gate))}[act]
        h = scale * f * a
        if x is not None:
            h = h + x
        out["h"] = put(h)
    else:
        h = x
    if w is not None:
        r2 = (h.square().mean(-1, keepdim=True) + eps) ** -0.5
        out["n"] = put(h * r2 * w)
    if dh is None and dn is None:
        return out
    d = torch.zeros_like(h) if dh is None else dh
    if w is not None:
        z = h * r2
        d = d + r2 * (dn * w - z * (dn * w * z).mean(-1, keepdim=True))
        out["dw"] = (dn * z).reshape(-1, C).sum(0)
    if x is not None:
        out["dx"] = put(d)
    if y is not None:
        da = scale * f * d
        if pw is not None:
            s = g(da * pw)
            out["dy"] = put((r1 * (s - g(u) * (s * g(u)).mean(-1, keepdim=True))).reshape(y.shape))
            out["dpw"] = (da * u).reshape(-1, C).sum(0)
        else:
            out["dy"] = put(da)
        if gate is not None:
            dg = scale * d * a * df
            out["dgate"] = dg.reshape(-1, C).sum(0) if gate.dim() == 1 and y.dim() > 1 else put(dg)
    return out


def norm_magnitudes(x, y, gate, pw, w, scale, eps, groups, act, dim, dh=None, dn=None):
    """The expressions of norm() with the absolute value of every term."""
    def last(t):
        if t is None:
            return None
        t = t.double()
        return t.transpose(1, 2) if dim == 1 and t.dim() == 3 else t

    def put(t):
        return t.transpose(1, 2) if dim == 1 and t.dim() == 3 else t

    full = {k: last(v) if k not in ("dw", "dpw", "dgate") or v.dim() > 1 else v
            for k, v in norm(x, y, gate, pw, w, scale, eps, groups, act, dim, dh, dn).items()}
    x, y, gate, dh, dn = last(x), last(y), last(gate), last(dh), last(dn)
    pw, w = (None if t is None else t.double().abs() for t in (pw, w))
    C = (y if y is not None else x).shape[-1]
    g = lambda t: t.reshape(t.shape[:-1] + (groups, C // groups))  # noqa: E731
    out = {}
    hm = 0.0 if x is None else x.abs()
    if y is not None:
        a = y.abs()
        if pw is not None:
            r1 = (g(y).square().mean(-1, keepdim=True) + eps) ** -0.5
            u = (g(y.abs()) * r1).reshape(y.shape)
            a = u * pw
        f, df = torch.ones_like(a), torch.zeros_like(a)
        if gate is not None:
            sg = torch.sigmoid(gate)
            f, df = {"silu": ((gate * sg).abs(), sg * (1 + gate.abs())), "sigmoid": (sg, sg),
                     "none": (gate.abs(), torch.ones_like(gate))}[act]
        hm = hm + abs(scale) * f * a
        out["h"] = put(hm)
    h = full["h"] if y is not None else x
    if w is not None:
        r2 = (h.square().mean(-1, keepdim=True) + eps) ** -0.5
        out["n"] = put(hm * r2 * w)
    if dh is None and dn is None:
        return out
    d = torch.zeros_like(h) if dh is None else dh.abs()
    if w is not None:
        z = hm * r2
        d = d + r2 * (dn.abs() * w + z * (dn.abs() * w * z).mean(-1, keepdim=True))
        out["dw"] = (dn.abs() * z).reshape(-1, C).sum(0)
    if x is not None:
        out["dx"] = put(d)
    if y is not None:
        da = abs(scale) * f * d
        if pw is not None:
            s = g(da * pw)
            out["dy"] = put((r1 * (s + g(u) * (s * g(u)).mean(-1, keepdim=True))).reshape(y.shape))
            out["dpw"] = (da * u).reshape(-1, C).sum(0)
        else:
            out["dy"] = put(da)
        if gate is not None:
            dg = abs(scale) * d * a * df
            out["dgate"] = dg.reshape(-1, C).sum(0) if gate.dim() == 1 and y.dim() > 1 else put(dg)
    return out


def norm_bound(name, value, mag, dtype, C, rows):
    """One rounding to the output's type.  In 32 bits: the longest chain of additions over a row's channels has 64 + C / 8
    (a thread's own, then a tree), it enters a gradient three times (two rstd, one mean); 64 for exp, division, rsqrt and
    products; sums over rows add at most one for each row.  Each is half a step of the magnitude."""
    n = 3 * (64 + C // 8) + 64 + (rows if value.dim() == 1 else 0)
    return HALF_STEP[dtype] * value.abs() + n * 2.0 ** -24 * mag + 1e-30
