"""Cases, inputs and plain forms of the linear-attention operators and the block norm.

Three operators are run here, as a user of the package calls them:

``attention``  ``linear_attention(Q, K, V, log_gamma, H0) -> (y, H_T)``: per head
               ``S_t = exp(log_gamma_t) S_{t-1} + k_t v_t^T``, ``y_t = S_t^T q_t``, over whole
               sequences, forward alone (a prompt) or with its backward (training).
``step``       ``step_ops.linear_attention_step``: the same recurrence for one token of every
               sequence of a batch, the new state written to a buffer of the caller's.
``norm``       ``block_norm``: ``h = residual + scale * x`` and a LayerNorm or RMS norm of ``h`` per
               group of channels, times ``silu(gate)`` where there is a gate.

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_CHUNK = 128  # tokens of a chunk of the plain form


# ------------------------------------------------------------------ cases --


def _attention(B, H, T, dk, dv, dtype, train, layout="bthd", decay="token", h0=False, resets=False):
    return dict(op="attention", B=B, H=H, T=T, dk=dk, dv=dv, dtype=dtype, train=train, layout=layout,
                decay=decay, h0=h0, resets=resets)


def _step(B, H, dk, dv, dtype):
    return dict(op="step", B=B, H=H, dk=dk, dv=dv, dtype=dtype)


def _norm(rows, D, dtype, train, rms=False, groups=1, gate=False, residual=False, scale=False,
          bias=False):
    return dict(op="norm", rows=rows, D=D, dtype=dtype, train=train, rms=rms, groups=groups, gate=gate,
                residual=residual, scale=scale, bias=bias)


def listed():
    named = {
        # a short prompt of one request: four heads of a 256-wide model, where latency counts
        "prompt-short": _attention(1, 4, 97, 64, 64, "bf16", False),
        # a chunk of a long document in serving, going on from the state of the part before it
        "prompt-long": _attention(1, 8, 65536, 64, 64, "bf16", False, h0=True),
        # a training step's mixer at the batch, heads and length of the delta rule's benchmark
        "train-bf16": _attention(8, 8, 8192, 64, 64, "bf16", True),
        # training in 32 bits at the width of the stack benchmark, head-major tensors
        "train-fp32": _attention(8, 8, 1024, 64, 64, "fp32", True, layout="bhtd", h0=True),
        # odd lengths and head sizes, a fixed decay for each head, packed documents (decay to nothing
        # at their starts)
        "train-ragged": _attention(3, 5, 1537, 40, 72, "fp16", True, decay="head", resets=True),
        # wide heads
        "train-wide": _attention(4, 4, 4096, 128, 128, "bf16", True, h0=True),
        # one token of one request
        "step-one": _step(1, 4, 64, 64, "bf16"),
        # one token of each request of a large serving batch
        "step-batch": _step(512, 8, 64, 64, "bf16"),
        # one token's residual and norm in a block's step
        "norm-token": _norm(1, 512, "bf16", False, residual=True, bias=True),
        # a block's residual and LayerNorm in training in 32 bits, the stack benchmark's width
        "norm-residual": _norm(8192, 512, "fp32", True, residual=True, bias=True),
        # the gated norm of each head after a mixer, the tokens of the large training step
        "norm-gate": _norm(65536, 512, "bf16", True, rms=True, groups=8, gate=True),
        # a wide residual stream of an odd size with a learnt scale for the branch
        "norm-wide": _norm(4097, 5001, "fp16", True, residual=True, scale=True, rms=True),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "step", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "attention":
        d = [rng.choice([64, 64, 128, 32, 8 * rng.randint(2, 16), rng.randint(9, 128)]) for _ in range(2)]
        B, H, train = _log_int(rng, 1, 16), rng.randint(1, 12), rng.random() < 0.6
        # tokens over all heads: no more than the largest listed case has at this width and type
        room = (8 * 8 * 8192 if train else 8 * 65536) * 64 * 64 // (max(64, d[0]) * max(64, d[1]))
        T = _log_int(rng, 1, min(65536 if not train else 16384, max(2, room * 2 // (_SIZE[dtype] * B * H))))
        return _attention(B, H, T, d[0], d[1], dtype, train, rng.choice(["bthd", "bhtd"]),
                          rng.choice(["token", "head"]), rng.random() < 0.5, rng.random() < 0.4)
    if op == "step":
        d = [rng.choice([64, 128, 8 * rng.randint(2, 16), rng.randint(9, 128)]) for _ in range(2)]
        return _step(_log_int(rng, 1, 512 * 4096 // (max(64, d[0]) * max(64, d[1]))), rng.randint(1, 8),
                     d[0], d[1], dtype)
    gate = rng.random() < 0.4
    groups = rng.choice([1, 4, 8, rng.randint(2, 16)]) if gate else 1
    n = rng.choice([64, 128, rng.randint(9, 256)]) if groups > 1 else _log_int(rng, 17, 8192)
    residual = not gate and rng.random() < 0.7
    return _norm(_log_int(rng, 1, max(1, 65536 * 512 // (groups * n))), groups * n, dtype, rng.random() < 0.6,
                 rng.random() < 0.5, groups, gate, residual, residual and rng.random() < 0.4,
                 rng.random() < 0.5)


def work(case):
    c, e = case, _SIZE[case["dtype"]]
    if c["op"] == "attention":
        heads = c["B"] * c["H"]
        tokens = heads * c["T"]
        lg = 4 * (tokens if c["decay"] == "token" or c["resets"] else c["H"])
        state = 4 * heads * c["dk"] * c["dv"]
        qkvy = e * tokens * 2 * (c["dk"] + c["dv"])
        # forward: q, k, v and the decay in, y out, the state in and out
        nbytes = qkvy + lg + state * (2 if c["h0"] else 1)
        # a token decays the state, adds k v^T and reads it with q
        flops = 5 * tokens * c["dk"] * c["dv"]
        if c["train"]:
            # backward: dy in, the gradients of q, k, v, the decay and the state out
            nbytes += qkvy + lg + state * (2 if c["h0"] else 1)
            # the state's gradient decays and adds q dy^T; it meets v, k and the state, the state dy
            flops += 11 * tokens * c["dk"] * c["dv"]
        return {"bytes": nbytes, "flops": flops}
    if c["op"] == "step":
        heads = c["B"] * c["H"]
        return {"bytes": heads * (8 * c["dk"] * c["dv"] + e * 2 * (c["dk"] + c["dv"]) + 4),
                "flops": 5 * heads * c["dk"] * c["dv"]}
    n = c["rows"] * c["D"]
    tensors = 2 + c["gate"] + 2 * c["residual"]  # x, y; gate; residual, h
    weights = 1 + c["bias"] + c["scale"]
    flops = 8 * n
    if c["train"]:
        # dy (and dh) in; dx, dgate out, and the residual's gradient where a scale makes it another
        tensors += 2 + c["gate"] + c["residual"] + c["scale"]
        weights += 1 + c["bias"] + c["scale"]
        flops += 16 * n
    return {"bytes": e * (tensors * n + weights * c["D"]), "flops": flops}


# ----------------------------------------------------------------- inputs --


def _inputs(case, seed):
    """The tensors of a case, by name, as leaves (head-major shapes whatever their layout)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    c = case
    if c["op"] == "norm":
        rows, D = c["rows"], c["D"]
        x = {"x": r(rows, D).to(dt), "weight": (1 + 0.2 * r(D)).to(dt)}
        if c["bias"]:
            x["bias"] = (0.2 * r(D)).to(dt)
        if c["residual"]:  # the stream has grown over the blocks before; the branch is smaller
            x["residual"] = (2 * r(rows, D) + 0.3).to(dt)
        if c["scale"]:
            x["scale"] = (0.5 + 0.2 * r(D)).to(dt)
        if c["gate"]:
            x["gate"] = r(rows, D).to(dt)
        if c["train"]:
            x["dy"] = r(rows, D).to(dt)
            if c["residual"]:
                x["dh"] = r(rows, D).to(dt)
        return x
    B, H, dk, dv = c["B"], c["H"], c["dk"], c["dv"]
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)  # noqa: E731
    # heads forget at rates from a few tokens to thousands; a token's gate varies about its head's
    rate = -4.0 * torch.arange(H, device="cuda", dtype=torch.float32) / max(1, H - 1) - 1.5
    if c["op"] == "step":
        return {"q": (r(B, H, dk) * dk**-0.5).to(dt), "k": unit(r(B, H, dk)).to(dt), "v": r(B, H, dv).to(dt),
                "log_gamma": -torch.nn.functional.softplus(rate + r(B, H)), "H": r(B, H, dk, dv)}
    T = c["T"]
    shape = (lambda d: (B, T, H, d)) if c["layout"] == "bthd" else (lambda d: (B, H, T, d))
    x = {"Q": (r(*shape(dk)) * dk**-0.5).to(dt), "K": unit(r(*shape(dk))).to(dt), "V": r(*shape(dv)).to(dt)}
    if c["decay"] == "head":
        lg = -torch.nn.functional.softplus(rate).view(1, H, 1)
    else:
        lg = -torch.nn.functional.softplus(rate.view(1, H, 1) + r(B, H, T))
    if c["resets"]:  # packed documents: about one start in 300 tokens, the same for all heads
        starts = torch.rand(B, 1, T, device="cuda", generator=g) < 1 / 300
        lg = torch.where(starts, torch.full_like(lg, -math.inf), lg)
    x["log_gamma"] = lg.contiguous()
    if c["h0"]:
        x["H0"] = r(B, H, dk, dv)
    if c["train"]:
        x["dy"] = r(*shape(dv)).to(dt)
        x["dH"] = r(B, H, dk, dv)
    return x


_LEAVES = {"attention": ("Q", "K", "V", "log_gamma", "H0"),
           "norm": ("x", "weight", "bias", "residual", "scale", "gate")}


def prepare(case, seed):
    x = _inputs(case, seed)
    if case.get("train"):
        for n in _LEAVES[case["op"]]:
            if n in x:
                x[n].requires_grad_(True)
    if case["op"] == "step":  # the buffer that the new state is written to
        x["out"] = torch.empty_like(x["H"])
    return {"case": dict(case), "x": x}


# ------------------------------------------------------------ plain forms --


def _spans(lg):
    """``sum_{s=j+1..i} lg_s`` for j <= i over the last axis, ``-inf`` for j > i."""
    n = lg.shape[-1]
    below = torch.ones(n, n, dtype=torch.bool, device=lg.device).tril(-1)
    s = torch.where(below, lg.unsqueeze(-1), torch.zeros((), dtype=lg.dtype, device=lg.device)).cumsum(-2)
    upper = torch.ones(n, n, dtype=torch.bool, device=lg.device).triu(1)
    return s.masked_fill(upper, -math.inf)


def _plain_attention(Q, K, V, lg, H0):
    """Chunks of the sequence: inside one as a masked product, between them through their states."""
    dt = Q.dtype
    B, H, T, dk = Q.shape
    dv = V.shape[-1]
    n = -(-T // _CHUNK)
    pad = n * _CHUNK - T
    cut = lambda t: torch.nn.functional.pad(t.float(), (0, 0, 0, pad)).reshape(B, H, n, _CHUNK, -1)  # noqa: E731
    q, k, v = cut(Q), cut(K), cut(V)
    lg = torch.nn.functional.pad(lg.expand(B, H, T), (0, pad)).reshape(B, H, n, _CHUNK)
    span = _spans(lg)
    inside = ((q @ k.mT) * span.exp()) @ v
    states = (k * span[..., -1, :].exp().unsqueeze(-1)).mT @ v
    S0 = torch.zeros(B, H, 1, dk, dv, device=Q.device) if H0 is None else H0.float().unsqueeze(2)
    total = lg.sum(-1)
    # state before chunk m, and after the last: decayed sums of H0 and the earlier chunks' states
    between = _spans(torch.nn.functional.pad(total, (1, 0))).exp()
    S = (between @ torch.cat([S0, states], 2).flatten(3)).unflatten(3, (dk, dv))
    y = inside + (q * lg.cumsum(-1).exp().unsqueeze(-1)) @ S[:, :, :-1]
    return y.reshape(B, H, n * _CHUNK, dv)[:, :, :T].to(dt), S[:, :, -1]


def _plain_norm(x, weight, bias, residual, scale, gate, groups, eps, rms):
    h = x.float()
    if scale is not None:
        h = h * scale.float()
    if residual is not None:
        h = residual.float() + h
    z = h.unflatten(-1, (groups, -1))
    if not rms:
        z = z - z.mean(-1, keepdim=True)
    z = (z * (z.square().mean(-1, keepdim=True) + eps).rsqrt()).flatten(-2) * weight.float()
    if bias is not None:
        z = z + bias.float()
    if gate is not None:
        z = z * (gate.float() * torch.sigmoid(gate.float()))
    z = z.to(x.dtype)
    return z if residual is None else (z, h.to(x.dtype))


# -------------------------------------------------------------------- run --


def _run_attention(c, x):
    heads = (lambda t: t.transpose(1, 2)) if c["layout"] == "bthd" else (lambda t: t)
    args = (heads(x["Q"]), heads(x["K"]), heads(x["V"]), x["log_gamma"], x.get("H0"))
    if own:
        import mingru_b200 as mb

        y, HT = mb.linear_attention(*args)
    else:
        y, HT = _plain_attention(*args)
    out = {"y": y, "H_T": HT}
    if c["train"]:
        leaves = [n for n in _LEAVES["attention"] if n in x]
        grads = torch.autograd.grad((y, HT), [x[n] for n in leaves], (heads(x["dy"]), x["dH"]))
        out = {"y": y.detach(), "H_T": HT.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}
    return out


def _run_step(x):
    if own:
        from mingru_b200 import step_ops

        y, H = step_ops.linear_attention_step(x["q"], x["k"], x["v"], x["log_gamma"], x["H"], out=x["out"])
    else:
        k, v = x["k"].float(), x["v"].float()
        H = x["log_gamma"].exp()[..., None, None] * x["H"] + k.unsqueeze(-1) * v.unsqueeze(-2)
        y = (x["q"].float().unsqueeze(-2) @ H).squeeze(-2).to(x["q"].dtype)
    return {"y": y, "H": H}


def _run_norm(c, x):
    residual = x.get("residual")
    if own:
        import mingru_b200 as mb

        got = mb.block_norm(x["x"], x["weight"], x.get("bias"), residual=residual, scale=x.get("scale"),
                            gate=x.get("gate"), groups=c["groups"], eps=1e-5, rms=c["rms"])
    else:
        got = _plain_norm(x["x"], x["weight"], x.get("bias"), residual, x.get("scale"), x.get("gate"),
                          c["groups"], 1e-5, c["rms"])
    got = (got,) if residual is None else got
    out = dict(zip(("y", "h"), got))
    if c["train"]:
        leaves = [n for n in _LEAVES["norm"] if n in x]
        grads = torch.autograd.grad(got, [x[n] for n in leaves], (x["dy"], x["dh"]) if len(got) > 1 else x["dy"])
        out = {n: t.detach() for n, t in out.items()} | {"d" + n: g for n, g in zip(leaves, grads)}
    return out


def run(state):
    c, x = state["case"], state["x"]
    if c["op"] == "attention":
        return _run_attention(c, x)
    return _run_step(x) if c["op"] == "step" else _run_norm(c, x)


# ------------------------------------------------------------------ exact --


def _exact_attention(c, x):
    """The recurrence itself, token by token; its gradients by the recurrence of the state's gradient
    ``G_t = q_t dy_t^T + gamma_{t+1} G_{t+1}``."""
    major = (lambda t: t.detach().double().permute(1, 0, 2, 3).contiguous()) if c["layout"] == "bthd" else (
        lambda t: t.detach().double().permute(2, 0, 1, 3).contiguous())  # time first: (T, B, H, d)
    q, k, v = (major(x[n]) for n in ("Q", "K", "V"))
    T, B, H, dk = q.shape
    dv = v.shape[-1]
    gam = x["log_gamma"].detach().double().exp().expand(B, H, T).permute(2, 0, 1).contiguous()[..., None, None]
    S = x["H0"].detach().double().clone() if c["h0"] else torch.zeros(B, H, dk, dv, dtype=torch.float64, device=q.device)
    y = torch.empty_like(v)
    back = (lambda t: t.permute(1, 0, 2, 3)) if c["layout"] == "bthd" else (lambda t: t.permute(1, 2, 0, 3))
    if c["train"]:
        dy, dq = major(x["dy"]), torch.empty_like(q)
    for t in range(T):
        S = torch.baddbmm((S * gam[t]).view(B * H, dk, dv), k[t].reshape(B * H, dk, 1), v[t].reshape(B * H, 1, dv)).view(S.shape)
        y[t] = (q[t].unsqueeze(-2) @ S).squeeze(-2)
        if c["train"]:
            dq[t] = (S @ dy[t].unsqueeze(-1)).squeeze(-1)
    out = {"y": back(y).transpose(1, 2) if c["layout"] == "bthd" else back(y), "H_T": S}
    if not c["train"]:
        return out
    G = x["dH"].double()
    f = (S * G).sum((-1, -2))  # <S_t, the gradient of S_t>
    dk_, dv_, dl = torch.empty_like(k), torch.empty_like(v), torch.empty(T, B, H, dtype=torch.float64, device=q.device)
    for t in range(T - 1, -1, -1):
        G = torch.baddbmm(G.reshape(B * H, dk, dv), q[t].reshape(B * H, dk, 1), dy[t].reshape(B * H, 1, dv)).view(G.shape)
        dk_[t] = (G @ v[t].unsqueeze(-1)).squeeze(-1)
        dv_[t] = (k[t].unsqueeze(-2) @ G).squeeze(-2)
        G = G * gam[t]
    # <S_t, G_t> steps by q.dq on entering a token from the right, and loses k.dk on leaving it
    a, b = (q * dq).sum(-1), (k * dk_).sum(-1)
    dl = f + (a - b).flip(0).cumsum(0).flip(0)
    dl = torch.where(gam[..., 0, 0] == 0, torch.zeros_like(dl), dl).permute(1, 2, 0)
    if x["log_gamma"].shape != dl.shape:
        dl = dl.sum((0, 2)).view(1, H, 1)
    out |= {"dQ": back(dq), "dK": back(dk_), "dV": back(dv_), "dlog_gamma": dl}
    if c["h0"]:
        out["dH0"] = G
    return out


def _exact_norm(c, x):
    """Group by group from the definition; gradients by their formulas."""
    d = {n: t.detach().double() for n, t in x.items()}
    rows, D, G = c["rows"], c["D"], c["groups"]
    h = d["x"] * d["scale"] if c["scale"] else d["x"]
    h = h + d["residual"] if c["residual"] else h
    hg = h.view(rows, G, D // G)
    mu = torch.zeros_like(hg[..., :1]) if c["rms"] else hg.sum(-1, keepdim=True) / (D // G)
    s = 1 / torch.sqrt(((hg - mu) ** 2).sum(-1, keepdim=True) / (D // G) + 1e-5)
    z = ((hg - mu) * s).view(rows, D)
    a = z * d["weight"] + (d["bias"] if c["bias"] else 0)
    sig = 1 / (1 + torch.exp(-d["gate"])) if c["gate"] else None
    out = {"y": a * d["gate"] * sig if c["gate"] else a}
    if c["residual"]:
        out["h"] = h
    if c["train"]:
        da = d["dy"] * d["gate"] * sig if c["gate"] else d["dy"]
        dz = (da * d["weight"]).view(rows, G, -1)
        zg = z.view(rows, G, -1)
        dh = dz - zg * (dz * zg).sum(-1, keepdim=True) / (D // G)
        if not c["rms"]:
            dh = dh - dz.sum(-1, keepdim=True) / (D // G)
        dh = (dh * s).view(rows, D) + (d["dh"] if c["residual"] else 0)
        out |= {"dx": dh * d["scale"] if c["scale"] else dh, "dweight": (da * z).sum(0)}
        if c["bias"]:
            out["dbias"] = da.sum(0)
        if c["residual"]:
            out["dresidual"] = dh
        if c["scale"]:
            out["dscale"] = (dh * d["x"]).sum(0)
        if c["gate"]:
            out["dgate"] = d["dy"] * a * (sig + d["gate"] * sig * (1 - sig))
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, x)
    if case["op"] == "norm":
        return _exact_norm(case, x)
    q, k, v, H = (x[n].double() for n in ("q", "k", "v", "H"))
    H = x["log_gamma"].double().exp()[..., None, None] * H + torch.einsum("bhk,bhv->bhkv", k, v)
    return {"y": torch.einsum("bhk,bhkv->bhv", q, H), "H": H}
