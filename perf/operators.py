"""Cases of the token-mixing operators beside the convolution: linear attention with a decay for each head (prompts,
training, single tokens) and the norms that join a mixing block to the residual stream.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, where
`own` is true, through sffft_b200.torch_ops.  `exact` evaluates the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
PLAIN_CHUNK = 128   # tokens that the plain form of linear attention takes together


# ---------------------------------------------------------------------------------------------------------------
# cases

def _prompt(name, B, H, Hkv, L, D, Dv, dtype, **kw):
    c = dict(name=name, op="attention", B=B, H=H, Hkv=Hkv, L=L, D=D, Dv=Dv, dtype=dtype, ragged=False, state=True,
             train=False, token_major=True, decay="slow")
    c.update(kw)
    return c


def _step(name, B, H, Hkv, D, Dv, dtype, pool, **kw):
    c = dict(name=name, op="step", B=B, H=H, Hkv=Hkv, D=D, Dv=Dv, dtype=dtype, pool=pool, decay="slow")
    c.update(kw)
    return c


def _norm(name, B, L, C, dtype, **kw):
    c = dict(name=name, op="norm", B=B, L=L, C=C, dtype=dtype, res=dtype, groups=1, gate="full", act="silu", post=True,
             residual=True, pre=True, train=False, first=False)
    c.update(kw)
    return c


def listed():
    return [
        # a short chat turn that continues from a kept state: one row, the convolution's 768 channels as 12 heads
        _prompt("prompt_short", 1, 12, 12, 128, 64, 64, "bf16"),
        # few heads over a long document: too few sequences to fill the GPU without cutting the length
        _prompt("prompt_long", 2, 8, 8, 16384, 128, 128, "bf16", state=False),
        # a served batch of prompts of different lengths, padded to an odd longest one, keys and values shared
        _prompt("prompt_ragged", 8, 12, 4, 1999, 64, 128, "bf16", ragged=True, decay="fast"),
        # full precision, as in evaluation and in checks against a 32-bit model
        _prompt("prompt_fp32", 2, 12, 12, 2047, 64, 64, "fp32", token_major=False),
        # a training step's mixer at the convolution benchmark's batch, channels and length
        _prompt("train_4096", 8, 12, 12, 4096, 64, 64, "bf16", train=True, state=False),
        # training on pieces of long sequences: the state enters and its gradient leaves; shared heads, odd length
        _prompt("train_pieces", 3, 8, 4, 1023, 128, 128, "bf16", train=True),
        # one user's next token
        _step("step_one", 1, 12, 12, 64, 64, "bf16", 1),
        # next tokens of a full serving batch whose states lie in a larger pool
        _step("step_batch", 200, 8, 8, 128, 128, "bf16", 256),
        # between two blocks while decoding: a few rows
        _norm("norm_token", 4, 1, 768, "bf16"),
        # between two blocks on prompts: norms by heads, 32-bit residual stream
        _norm("norm_prompt", 8, 4096, 768, "bf16", res="fp32", groups=12),
        # between two blocks in training, learned gate for each channel, odd row count
        _norm("norm_train", 7, 2047, 1024, "bf16", train=True, gate="channel", act="none"),
        # behind the convolution, in its own [B][C][L] layout, trained
        _norm("norm_conv", 8, 1024, 768, "fp32", train=True, act="sigmoid", first=True),
    ]


def _log_range(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "step", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    decay = rng.choice(["slow", "fast"])
    if op == "attention":
        Hkv = rng.choice([1, 2, 3, 4, 6, 8])
        H = Hkv * rng.choice([1, 1, 2, 3])
        D = rng.choice([16, 32, 40, 64, 64, 64, 80, 96, 128, 128])
        Dv = rng.choice([D, D, 32, 64, 72, 128])
        L = _log_range(rng, 1, 16384)
        train = rng.random() < 0.4
        most = (1 << 21) if train else (1 << 22)          # heads x tokens
        if dtype == "fp32":
            most >>= 3
        B = max(1, min(_log_range(rng, 1, 16), most // (H * L)))
        return dict(op=op, B=B, H=H, Hkv=Hkv, L=L, D=D, Dv=Dv, dtype=dtype, ragged=rng.random() < 0.4,
                    state=rng.random() < 0.5, train=train, token_major=rng.random() < 0.5, decay=decay)
    if op == "step":
        Hkv = rng.choice([1, 2, 4, 6, 8, 12])
        H = Hkv * rng.choice([1, 1, 2])
        B = _log_range(rng, 1, 160)
        return dict(op=op, B=B, H=H, Hkv=Hkv, D=rng.choice([16, 40, 64, 64, 96, 128, 128]),
                    Dv=rng.choice([32, 64, 64, 100, 128, 128]), dtype=dtype, pool=B + rng.randrange(0, 40), decay=decay)
    first = rng.random() < 0.4
    C = rng.choice([64, 96, 256, 512, 768, 768, 1000, 1024, 2048, 4096])
    rows = _log_range(rng, 1, 20000)
    rows = max(1, min(rows, 20000 * 768 // C))
    B = max(1, min(rows, rng.choice([1, 2, 3, 8, 16])))
    residual = rng.random() < 0.8
    pre = rng.random() < 0.8
    res = rng.choice([dtype, "fp32"]) if residual else dtype
    return dict(op=op, B=B, L=max(1, rows // B), C=C, dtype=dtype, res=res, groups=rng.choice([1, 1, 4, 8]),
                gate=rng.choice(["full", "full", "channel", "none"]), act=rng.choice(["silu", "sigmoid", "none"]),
                post=rng.random() < 0.7, residual=residual, pre=pre, train=rng.random() < 0.5, first=first)


# ---------------------------------------------------------------------------------------------------------------
# inputs

def _log_decay(kind, H, device):
    h = torch.arange(H, dtype=torch.float64)
    if kind == "slow":      # 1 - 2^-5 ... 1 - 2^-12: memories of 32 to 4096 tokens
        ld = torch.log1p(-torch.exp2(-(5 + 7 * h / max(1, H - 1))))
    else:                   # slopes from 1/2 down to 1/256
        ld = -torch.exp2(-(1 + 7 * h / max(1, H - 1)))
    return ld.float().to(device)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt, scale=1.0):
        return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)

    st = {"case": case}
    if case["op"] == "norm":
        B, L, C = case["B"], case["L"], case["C"]
        shape = (B, C, L) if case["first"] else (B, L, C)
        rt = DTYPES[case["res"]]
        st["y"] = randn(*shape)
        st["x"] = randn(*shape, dtype=rt, scale=2.0) if case["residual"] else None
        st["gate"] = {"full": lambda: randn(*shape), "channel": lambda: randn(C), "none": lambda: None}[case["gate"]]()
        st["post_weight"] = 1 + randn(C, dtype=torch.float32, scale=0.1) if case["post"] else None
        st["weight"] = 1 + randn(C, dtype=torch.float32, scale=0.1) if case["pre"] else None
        if case["train"]:
            st["dh"] = randn(*shape, dtype=rt)
            st["dn"] = randn(*shape) if case["pre"] else None
        return st
    B, H, Hkv, D, Dv = (case[n] for n in ("B", "H", "Hkv", "D", "Dv"))
    st["log_decay"] = _log_decay(case["decay"], H, dev)
    if case["op"] == "step":
        st["q"], st["k"], st["v"] = randn(B, H, D), randn(B, Hkv, D), randn(B, Hkv, Dv)
        st["state"] = randn(case["pool"], H, D, Dv, dtype=torch.float32, scale=4.0)
        order = torch.randperm(case["pool"], generator=g, device=dev)
        st["slots"] = order[:B].to(torch.int32)
        return st
    L = case["L"]

    def heads(n, d):
        if case["token_major"]:     # as a projection leaves them: [B][L][heads][d]
            return randn(B, L, n, d).transpose(1, 2)
        return randn(B, n, L, d)

    st["q"], st["k"], st["v"] = heads(H, D), heads(Hkv, D), heads(Hkv, Dv)
    st["state"] = randn(B, H, D, Dv, dtype=torch.float32, scale=2.0) if case["state"] else None
    st["lengths"] = None
    if case["ragged"]:
        n = torch.randint(0, L + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        n[0] = L
        st["lengths"] = n
    if case["train"]:
        st["dy"] = heads(H, Dv)
        st["dstate"] = randn(B, H, D, Dv, dtype=torch.float32) if case["state"] else None
    return st


# ---------------------------------------------------------------------------------------------------------------
# plain forms

def _plain_attention(q, k, v, log_decay, scale, state, lengths):
    B, H, L, D = q.shape
    Hkv, Dv = k.shape[1], v.shape[3]
    share = torch.arange(H, device=q.device) // (H // Hkv)
    ld = log_decay.double()
    n = torch.full((B,), L, device=q.device) if lengths is None else lengths.long()
    S = torch.zeros((B, H, D, Dv), device=q.device) if state is None else state
    ys = []
    i = torch.arange(PLAIN_CHUNK, device=q.device)
    lag = i[:, None] - i[None, :]
    inside = torch.where(lag >= 0, torch.exp(ld[:, None, None] * lag.clamp(min=0)), 0.0).float()
    before = torch.exp(ld[:, None] * (i + 1)).float()
    for t in range(0, L, PLAIN_CHUNK):
        m = min(PLAIN_CHUNK, L - t)
        there = t + i[:m] < n[:, None]                                   # [B][m]
        qc = q[:, :, t:t + m].float()
        kc = torch.where(there[:, None, :, None], k[:, :, t:t + m].float(), 0.0)[:, share]
        vc = torch.where(there[:, None, :, None], v[:, :, t:t + m].float(), 0.0)[:, share]
        p = (qc @ kc.transpose(2, 3)) * inside[:, :m, :m]
        yc = scale * (p @ vc + before[:, :m, None] * (qc @ S))
        ys.append(torch.where(there[:, None, :, None], yc, 0.0).to(q.dtype))
        left = (n - t).clamp(0, m)                                       # tokens of each row in this chunk
        back = (left[:, None] - 1 - i[:m]).clamp(min=0)                  # [B][m]
        w = torch.exp(ld[None, :, None] * back[:, None, :]).float()
        S = torch.exp(ld[None, :] * left[:, None]).float()[:, :, None, None] * S + (kc * w[..., None]).transpose(2, 3) @ vc
    return torch.cat(ys, 2), S


def _plain_step(q, k, v, log_decay, state, slots, scale):
    share = torch.arange(q.shape[1], device=q.device) // (q.shape[1] // k.shape[1])
    rows = slots.long()
    kf, vf = k.float()[:, share], v.float()[:, share]
    S = torch.exp(log_decay.double()).float()[:, None, None] * state[rows] + kf[..., :, None] * vf[..., None, :]
    state[rows] = S
    return (scale * (q.float()[..., None] * S).sum(2)).to(q.dtype)


def _rms(a, groups, eps):
    """a [..., C] divided by the root of the mean of squares over each of the groups of channels."""
    s = a.unflatten(-1, (groups, a.shape[-1] // groups))
    return (s * torch.rsqrt((s * s).mean(-1, keepdim=True) + eps)).flatten(-2)


def _plain_norm(x, y, gate, post_weight, weight, scale, eps, groups, act, first):
    def last(t):
        return t.transpose(1, 2) if first and t.dim() == 3 else t

    out_type, res_type = y.dtype, (y if x is None else x).dtype
    a = last(y).float()
    if post_weight is not None:
        a = _rms(a, groups, eps) * post_weight
    if gate is not None:
        gt = last(gate).float()
        a = a * {"silu": lambda t: t / (1 + torch.exp(-t)), "sigmoid": lambda t: 1 / (1 + torch.exp(-t)),
                 "none": lambda t: t}[act](gt)
    h = scale * a
    if x is not None:
        h = last(x).float() + h
    n = None if weight is None else last(_rms(h, 1, eps) * weight).to(out_type)
    return last(h).to(res_type), n


EPS = 1e-6
RES_SCALE = 0.5


def _leaf(t):
    return None if t is None else t.detach().requires_grad_()


def run(st):
    case = st["case"]
    if own:
        import sffft_b200.torch_ops as ops
    if case["op"] == "step":
        args = (st["q"], st["k"], st["v"], st["log_decay"], st["state"])
        scale = case["D"] ** -0.5
        if own:
            y = ops.linear_attention_step(*args, slots=st["slots"], scale=scale)
        else:
            y = _plain_step(*args, st["slots"], scale)
        return {"y": y, "state": st["state"]}
    if case["op"] == "attention":
        q, k, v, s0 = st["q"], st["k"], st["v"], st["state"]
        if case["train"]:
            q, k, v, s0 = _leaf(q), _leaf(k), _leaf(v), _leaf(s0)
        scale = case["D"] ** -0.5
        if own:
            y, s1 = ops.linear_attention(q, k, v, st["log_decay"], scale=scale, initial_state=s0, lengths=st["lengths"])
        else:
            y, s1 = _plain_attention(q, k, v, st["log_decay"], scale, s0, st["lengths"])
        out = {"y": y.detach(), "state": s1.detach()}
        if case["train"]:
            if s0 is None:
                grads = torch.autograd.grad([y], [q, k, v], [st["dy"]])
            else:
                grads = torch.autograd.grad([y, s1], [q, k, v, s0], [st["dy"], st["dstate"]])
            out.update(zip(("dq", "dk", "dv", "dstate"), grads))
        return out
    x, y, gate, pw, w = (st[n] for n in ("x", "y", "gate", "post_weight", "weight"))
    if case["train"]:
        x, y, gate, pw, w = (_leaf(t) for t in (x, y, gate, pw, w))
    if own:
        h, n = ops.block_norm(x, y, gate, pw, w, scale=RES_SCALE, eps=EPS, groups=case["groups"], act=case["act"],
                              dim=1 if case["first"] else -1)
    else:
        h, n = _plain_norm(x, y, gate, pw, w, RES_SCALE, EPS, case["groups"], case["act"], case["first"])
    out = {"h": h.detach()}
    if n is not None:
        out["n"] = n.detach()
    if case["train"]:
        ins = {"dx": x, "dy": y, "dgate": gate, "dpost_weight": pw, "dweight": w}
        ins = {name: t for name, t in ins.items() if t is not None}
        outs = [h] if n is None else [h, n]
        grads = torch.autograd.grad(outs, list(ins.values()), [st["dh"]] if n is None else [st["dh"], st["dn"]])
        out.update(zip(ins, grads))
    return out


# ---------------------------------------------------------------------------------------------------------------
# definitions in 64 bits

def _exact_attention(case, st):
    """One head of one row at a time, as a masked product over all pairs of positions."""
    H, Hkv, D, Dv = (case[n] for n in ("H", "Hkv", "D", "Dv"))
    scale, dev = D ** -0.5, st["q"].device
    B, L = case["B"], case["L"]
    out = {"y": torch.zeros((B, H, L, Dv), dtype=torch.float64, device=dev),
           "state": torch.zeros((B, H, D, Dv), dtype=torch.float64, device=dev)}
    if case["train"]:
        out["dq"] = torch.zeros((B, H, L, D), dtype=torch.float64, device=dev)
        out["dk"] = torch.zeros((B, Hkv, L, D), dtype=torch.float64, device=dev)
        out["dv"] = torch.zeros((B, Hkv, L, Dv), dtype=torch.float64, device=dev)
        if case["state"]:
            out["dstate"] = torch.zeros((B, H, D, Dv), dtype=torch.float64, device=dev)
    ends = [L] * B if st["lengths"] is None else st["lengths"].tolist()
    for b in range(B):
        n = ends[b]
        pos = torch.arange(n, dtype=torch.float64, device=dev)
        for h in range(H):
            hk = h * Hkv // H
            a = st["log_decay"][h].double()
            q, k, v = st["q"][b, h, :n].double(), st["k"][b, hk, :n].double(), st["v"][b, hk, :n].double()
            s0 = st["state"][b, h].double() if case["state"] else torch.zeros((D, Dv), dtype=torch.float64, device=dev)
            grow = torch.exp(a * (pos + 1))[:, None]
            rest = torch.exp(a * (n - 1 - pos))[:, None]
            out["state"][b, h] = (k * rest).T @ v + torch.exp(a * n) * s0
            if case["train"]:
                dy = st["dy"][b, h, :n].double()
                ds = st["dstate"][b, h].double() if case["state"] else torch.zeros_like(s0)
                out["dk"][b, hk, :n] += rest * (v @ ds.T)
                out["dv"][b, hk, :n] += rest * (k @ ds)
                if case["state"]:
                    out["dstate"][b, h] = scale * (q * grow).T @ dy + torch.exp(a * n) * ds
            for t in range(0, n, 4096):
                e = min(n, t + 4096)
                lag = pos[t:e, None] - pos[None, :e]
                w = torch.where(lag >= 0, torch.exp(a * lag.clamp(min=0)), 0.0)
                m = (q[t:e] @ k[:e].T) * w
                out["y"][b, h, t:e] = scale * (m @ v[:e] + grow[t:e] * (q[t:e] @ s0))
                if case["train"]:
                    out["dv"][b, hk, :e] += scale * m.T @ dy[t:e]
                    m = (dy[t:e] @ v[:e].T) * w
                    out["dq"][b, h, t:e] = scale * (m @ k[:e] + grow[t:e] * (dy[t:e] @ s0.T))
                    out["dk"][b, hk, :e] += scale * m.T @ q[t:e]
    return out


def _exact_step(case, st):
    scale = case["D"] ** -0.5
    state = st["state"].double()
    y = torch.zeros((case["B"], case["H"], case["Dv"]), dtype=torch.float64, device=state.device)
    for h in range(case["H"]):
        hk = h * case["Hkv"] // case["H"]
        rows = st["slots"].long()
        s = torch.exp(st["log_decay"][h].double()) * state[rows, h]
        s = s + torch.einsum("bd,be->bde", st["k"][:, hk].double(), st["v"][:, hk].double())
        state[rows, h] = s
        y[:, h] = scale * torch.einsum("bd,bde->be", st["q"][:, h].double(), s)
    return {"y": y, "state": state}


def _exact_norm(case, st):
    """Values and, for a training case, the gradients from their formulas; the channels are brought to the end."""
    C, G = case["C"], case["groups"]

    def get(name):
        t = st.get(name)
        if t is None:
            return None
        t = t.double()
        return t.transpose(1, 2) if case["first"] and t.dim() == 3 else t

    def put(t):
        return t.transpose(1, 2) if case["first"] else t

    def by_group(t):
        return t.reshape(t.shape[:-1] + (G, C // G))

    x, y, gate, pw, w = get("x"), get("y"), get("gate"), get("post_weight"), get("weight")
    if pw is not None:
        r1 = (by_group(y).square().mean(-1, keepdim=True) + EPS) ** -0.5
        u = (by_group(y) * r1).reshape(y.shape)
        a = u * pw
    else:
        a = y
    if gate is None:
        f = torch.ones((), dtype=torch.float64, device=y.device)
    else:
        sg = torch.sigmoid(gate)
        f, df = {"silu": (gate * sg, sg * (1 + gate * (1 - sg))), "sigmoid": (sg, sg * (1 - sg)),
                 "none": (gate, torch.ones_like(gate))}[case["act"]]
    h = RES_SCALE * f * a
    if x is not None:
        h = h + x
    out = {"h": put(h)}
    if w is not None:
        r2 = (h.square().mean(-1, keepdim=True) + EPS) ** -0.5
        out["n"] = put(h * r2 * w)
    if not case["train"]:
        return out
    gh = get("dh")
    if w is not None:
        dn = get("dn")
        gh = gh + r2 * (dn * w - h * r2 * (dn * w * h * r2).mean(-1, keepdim=True))
    if x is not None:
        out["dx"] = put(gh)
    da = RES_SCALE * f * gh
    if pw is not None:
        dg, ug = by_group(da * pw), by_group(u)
        out["dy"] = put((r1 * (dg - ug * (dg * ug).mean(-1, keepdim=True))).reshape(y.shape))
    else:
        out["dy"] = put(da)
    if gate is not None:
        dgate = RES_SCALE * gh * a * df
        out["dgate"] = dgate.sum((0, 1)) if gate.dim() == 1 else put(dgate)
    if pw is not None:
        out["dpost_weight"] = (da * u).sum((0, 1))
    if w is not None:
        out["dweight"] = (dn * h * r2).sum((0, 1))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "step": _exact_step, "norm": _exact_norm}[case["op"]](case, st)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    size = {"bf16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "norm":
        n, C = case["B"] * case["L"] * case["C"], case["C"]
        rs = {"bf16": 2, "fp32": 4}[case["res"]]
        gate_full = case["gate"] == "full"
        streams = size * (1 + gate_full + case["pre"]) + rs * (case["residual"] + 1)       # y, gate, n; x, h
        small = 4 * C * (case["post"] + case["pre"]) + size * C * (case["gate"] == "channel")
        flops = 12 * n
        if case["train"]:
            streams += size * (1 + gate_full + case["pre"]) + rs * (case["residual"] + 1)  # dy, dgate, dn; dx, dh
            small *= 2
            flops += 30 * n
        return {"bytes": n * streams + small, "flops": flops}
    B, H, Hkv, D, Dv = (case[n] for n in ("B", "H", "Hkv", "D", "Dv"))
    if case["op"] == "step":
        heads = B * (H * (D + Dv) + Hkv * (D + Dv)) * size
        return {"bytes": heads + 8 * B * H * D * Dv + 4 * (B + H), "flops": 6 * B * H * D * Dv}
    L = case["L"]
    qkv = B * L * (H * D + Hkv * (D + Dv))
    y = B * H * L * Dv
    states = 4 * B * H * D * Dv * (1 + case["state"])
    total = (qkv + y) * size + states + 4 * H
    flops = 4 * B * H * L * D * Dv
    if case["train"]:
        total += (qkv + y) * size + (states if case["state"] else 0)
        flops += 10 * B * H * L * D * Dv
    return {"bytes": total, "flops": flops}
