"""The transformer-block operators -- attention of any length, rotary positions, the fused block boundary -- as cases to
measure: their inputs, their plain forms in elementary torch operations and their values in 64 bits.

``own = False``: ``run`` computes the plain forms in fp32.  ``own = True``: it calls the framework's operators.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BASE, _EPS = 10000.0, 1e-6
_FACTOR, _ORIGINAL, _FAST, _SLOW = 8.0, 4096, 32.0, 1.0      # long-context scaling: 8 x the trained length of 4096


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attention(name, batch, q_len, kv_len, heads, kv_heads, head_dim, causal, ragged, train):
    c = dict(op="attention", batch=batch, q_len=q_len, kv_len=kv_len, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             causal=causal, ragged=ragged, train=train)
    return dict(c, name=name) if name else c


def _rotary(name, batch, length, heads, kv_heads, head_dim, rot_dim, interleaved, scaling, far, dtype, train):
    c = dict(op="rotary", batch=batch, length=length, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rot_dim=rot_dim,
             interleaved=interleaved, scaling=scaling, far=far, dtype=dtype, train=train)
    return dict(c, name=name) if name else c


def _norm(name, batch, length, hidden, kind, post, gate, scale, dtype, train):
    c = dict(op="norm", batch=batch, length=length, hidden=hidden, kind=kind, post=post, gate=gate, scale=scale, dtype=dtype,
             train=train)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a handful of short padded sentences through BERT-base's heads: the call's latency counts
        _attention("attention-short", 2, 37, 37, 12, 12, 64, False, True, True),
        # an encoder's training step at a length that is no multiple of anything, padded sequences
        _attention("attention-encoder", 8, 1000, 1000, 12, 12, 64, False, True, True),
        # a decoder's training step over one long document, grouped heads
        _attention("attention-decoder", 1, 8192, 8192, 16, 4, 128, True, False, True),
        # the next piece of a long prompt against what is already there (no gradient)
        _attention("attention-piece", 2, 257, 7000, 32, 8, 128, True, False, False),
        # one new token for each of four sequences of different lengths (no gradient)
        _attention("attention-token", 4, 1, 4100, 32, 8, 128, False, True, False),
        # rotary positions of one new token for each of eight sequences, far out in a stretched context
        _rotary("rotary-token", 8, 1, 32, 8, 128, 128, False, "by_parts", 30000, "bf16", False),
        # a long training batch, queries and keys still inside their packed projection
        _rotary("rotary-train", 2, 8192, 32, 8, 128, 128, False, "none", 0, "bf16", True),
        # interleaved pairs in two thirds of the head, full precision, odd length, base-stretched
        _rotary("rotary-interleaved", 3, 501, 16, 4, 96, 64, True, "ntk", 100, "f32", True),
        # block boundary of one new token for each of eight sequences
        _norm("norm-token", 8, 1, 4096, "rms", True, "none", 0.5, "bf16", False),
        # LayerNorm block boundary at BERT-base's width with a learned scale per channel, training
        _norm("norm-encoder", 8, 1000, 768, "layer", False, "channel", 1.0, "bf16", True),
        # norms on both sides of the block, a gate per sequence, training: the largest
        _norm("norm-sandwich", 4, 4096, 4096, "rms", True, "sequence", 0.25, "bf16", True),
        # full precision, odd width and length, a gate per element
        _norm("norm-odd", 3, 333, 1001, "rms", False, "full", 0.7071, "f32", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "norm"])
    if op == "attention":
        largest = 16 * 8192 * 8192 * 128
        while True:
            train = rng.random() < 0.6
            kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
            heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 8])
            head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
            batch = rng.randint(1, 8)
            causal = rng.random() < 0.6
            kv_len = _log(rng, 1, 8192)
            q_len = kv_len if train and rng.random() < 0.8 else _log(rng, 1, 600)
            if heads <= 40 and batch * heads * q_len * kv_len * head_dim * (14 if train else 4) <= largest * 7:
                return _attention(None, batch, q_len, kv_len, heads, kv_heads, head_dim, causal, rng.random() < 0.5, train)
    if op == "rotary":
        while True:
            kv_heads = rng.choice([1, 2, 4, 8, 12])
            heads = kv_heads * rng.choice([1, 2, 4])
            head_dim = rng.choice([64, 96, 128, 128, 256])
            rot_dim = rng.choice([head_dim, head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2)])
            batch, length = rng.randint(1, 8), _log(rng, 1, 8192)
            if batch * length * (heads + kv_heads) * head_dim <= 2 * 8192 * 40 * 128:
                return _rotary(None, batch, length, heads, kv_heads, head_dim, rot_dim, rng.random() < 0.5,
                               rng.choice(["none", "linear", "ntk", "by_parts"]), rng.choice([0, 1000, 30000, 1000000]),
                               rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.7)
    while True:
        hidden = rng.choice([_log(rng, 16, 8192), 64 * _log(rng, 1, 128)])
        batch, length = rng.randint(1, 8), _log(rng, 1, 8192)
        if batch * length * hidden <= 4 * 4096 * 4096:
            return _norm(None, batch, length, hidden, rng.choice(["rms", "rms", "layer"]), rng.random() < 0.5,
                         rng.choice(["none", "channel", "sequence", "full"]), rng.choice([1.0, 0.5, 0.1]),
                         rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.7)


def _lens(case):
    """Keys of each sequence: ragged ones grow evenly to the full length (and reach 0 where there are fewer keys than sequences)."""
    B, n = case["batch"], case["kv_len"]
    return [n * (b + 1) // B for b in range(B)] if case["ragged"] else [n] * B


def work(case):
    B = case["batch"]
    if case["op"] == "attention":
        nq, nk, Hq, Hk, D = case["q_len"], case["kv_len"], case["heads"], case["kv_heads"], case["head_dim"]
        pairs, keys = 0, 0
        for n in _lens(case):
            keys += n
            if not case["causal"]:
                pairs += nq * n
            else:                                       # query i sees min(n, max(0, i + 1 + nk - nq)) keys
                first = max(0, nq - nk)                 # rows before it see none
                full = max(first, min(nq, n - 1 + nq - nk))
                a, b = first + 1 + nk - nq, full + nk - nq      # keys of the rows first .. full - 1
                pairs += (a + b) * (full - first) // 2 + (nq - full) * n
        io = 2 * (B * nq * Hq * D * 2 + 2 * keys * Hk * D)                    # q, out, k, v
        if case["train"]:
            io += 2 * (B * nq * Hq * D * 2 + 2 * B * nk * Hk * D)             # dout, dq, dk, dv
        return {"bytes": io, "flops": pairs * Hq * D * (14 if case["train"] else 4)}
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rotary":
        n = B * case["length"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        times = 2 if case["train"] else 1
        return {"bytes": times * 2 * n * e + 8 * B * case["length"], "flops": times * 3 * n}
    n = B * case["length"] * case["hidden"]
    groups = {"none": 0, "channel": case["hidden"], "sequence": B * case["hidden"], "full": n}[case["gate"]]
    io = 4 * n + groups + (4 * n + groups if case["train"] else 0)
    return {"bytes": io * e, "flops": n * (40 if case["train"] else 12)}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _frequencies(dim, scaling):
    """(frequency of each pair in 64 bits, amplitude)."""
    j = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    base = _BASE
    if scaling == "ntk" and dim > 2:
        base = _BASE * _FACTOR ** (dim / (dim - 2))
    f = base ** -j
    if scaling == "linear":
        return f / _FACTOR, 1.0
    if scaling == "by_parts":
        turns = _ORIGINAL * f / (2 * math.pi)                      # full turns within the trained length
        keep = ((turns - _SLOW) / (_FAST - _SLOW)).clamp(0, 1)     # 1: fast pairs stay, 0: slow pairs are stretched
        return f * keep + f / _FACTOR * (1 - keep), 0.1 * math.log(_FACTOR) + 1.0
    return f, 1.0


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = dict(case=case)
    B = case["batch"]
    if case["op"] == "attention":
        nq, nk, Hq, Hk, D = case["q_len"], case["kv_len"], case["heads"], case["kv_heads"], case["head_dim"]
        if nq == nk:                                     # one packed projection
            qkv = randn(B, nq, Hq + 2 * Hk, D).to(torch.bfloat16)
            q, k, v = qkv.split([Hq, Hk, Hk], dim=2)
        else:                                            # queries of their own, keys and values from one buffer
            q = randn(B, nq, Hq, D).to(torch.bfloat16)
            k, v = randn(B, nk, 2 * Hk, D).to(torch.bfloat16).split([Hk, Hk], dim=2)
        s["q"], s["k"], s["v"] = (t.detach().requires_grad_(case["train"]) for t in (q, k, v))
        s["dout"] = randn(B, nq, Hq, D).to(torch.bfloat16) if case["train"] else None
        n = _lens(case)
        n = n[seed % B:] + n[:seed % B]
        s["lens"] = torch.tensor(n, dtype=torch.int32, device=dev) if case["ragged"] else None
        return s
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        S, Hq, Hk, D = case["length"], case["heads"], case["kv_heads"], case["head_dim"]
        qkv = randn(B, S, Hq + 2 * Hk, D).to(dt)
        q, k, _ = qkv.split([Hq, Hk, Hk], dim=2)
        s["q"], s["k"] = (t.detach().requires_grad_(case["train"]) for t in (q, k))
        start = torch.randint(0, case["far"] + 1, (B, 1), generator=g, device=dev)
        s["positions"] = start + torch.arange(S, device=dev)
        f, s["amplitude"] = _frequencies(case["rot_dim"], case["scaling"])
        s["inv_freq"] = f.to(dev)
        if case["train"]:
            s["dq"], s["dk"] = randn(B, S, Hq, D).to(dt), randn(B, S, Hk, D).to(dt)
        return s
    S, H = case["length"], case["hidden"]
    channels = torch.exp(randn(H))                       # a residual stream has channels far larger than others
    s["x"] = (randn(B, S, H) * channels).to(dt)
    s["h"] = (randn(B, S, H) * 1.5 + 0.1).to(dt)
    s["weight"] = (1 + 0.2 * randn(H)).to(dt)
    s["bias"] = (0.1 * randn(H)).to(dt) if case["kind"] == "layer" else None
    s["post_weight"] = (1 + 0.2 * randn(H)).to(dt) if case["post"] else None
    s["post_bias"] = (0.1 * randn(H)).to(dt) if case["post"] and case["kind"] == "layer" else None
    shape = {"none": None, "channel": (H,), "sequence": (B, 1, H), "full": (B, S, H)}[case["gate"]]
    s["gate"] = None if shape is None else (0.3 + 0.5 * randn(*shape)).to(dt)
    if case["train"]:
        s["dy"], s["dr"] = randn(B, S, H).to(dt), (0.5 * randn(B, S, H)).to(dt)
    for n in ("x", "h", "weight", "bias", "post_weight", "post_bias", "gate"):
        if s[n] is not None:
            s[n].requires_grad_(case["train"])
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _plain_attention(q, k, v, causal, lens):
    B, nq, Hq, D = q.shape
    nk, Hk = k.shape[1], k.shape[2]
    qg = q.view(B, nq, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)      # a kv head's queries in one product
    kt, vt = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    score = (torch.matmul(qg, kt) * (1.0 / math.sqrt(D))).view(B, Hk, Hq // Hk, nq, nk)
    at = torch.arange(nk, device=q.device)
    hidden = torch.zeros(B, 1, 1, 1, nk, dtype=torch.bool, device=q.device)
    if lens is not None:
        hidden = (at >= lens[:, None]).view(B, 1, 1, 1, nk)
    if causal:
        hidden = hidden | (at > torch.arange(nq, device=q.device)[:, None] + (nk - nq))
    score = score.masked_fill(hidden, -math.inf)
    top = score.detach().amax(-1, keepdim=True).clamp_min(-1e30)
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))                         # a row that sees no key: zeros
    o = torch.matmul(p.view(B, Hk, -1, nk), vt)
    return o.view(B, Hk, Hq // Hk, nq, D).permute(0, 3, 1, 2, 4).reshape(B, nq, Hq, D)


def _plain_rotate(x, cos, sin, interleaved, amplitude):
    d = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:d:2], x[..., 1:d:2]
    else:
        a, b = x[..., :d // 2], x[..., d // 2:d]
    ra, rb = amplitude * (a * cos - b * sin), amplitude * (a * sin + b * cos)
    turned = torch.stack([ra, rb], dim=-1).flatten(-2) if interleaved else torch.cat([ra, rb], dim=-1)
    return torch.cat([turned, x[..., d:]], dim=-1)


def _plain_normed(x, weight, bias, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight
    return x if bias is None else x + bias


def _in_32(*tensors):
    return [None if t is None else t.detach().float().requires_grad_(t.requires_grad) for t in tensors]


def _with_gradients(outs, leaves, grads, dtype):
    """Outputs and gradients, rounded once."""
    leaves = [t for t in leaves if t is not None]
    if not leaves[0].requires_grad:
        return [t.to(dtype) for t in outs]
    return [t.detach().to(dtype) for t in outs] + [t.to(dtype) for t in torch.autograd.grad(outs, leaves, grads)]


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    s, case = state, state["case"]
    if case["op"] == "attention":
        leaves, grads = [s["q"], s["k"], s["v"]], [s["dout"]]
        if own:
            from distributed_tensorflow_amd.ops.attention import attention
            outs = [attention(*leaves, causal=case["causal"], kv_len=s["lens"])]
        else:
            leaves, grads = _in_32(*leaves), _in_32(*grads)
            outs = [_plain_attention(*leaves, case["causal"], s["lens"])]
        return _with_gradients(outs, leaves, grads, torch.bfloat16)
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        leaves, grads = [s["q"], s["k"]], [s.get("dq"), s.get("dk")]
        if own:
            from distributed_tensorflow_amd.ops.rotary import rotary
            outs = rotary(*leaves, s["inv_freq"], s["positions"], interleaved=case["interleaved"], amplitude=s["amplitude"])
        else:
            leaves, grads = _in_32(*leaves), _in_32(*grads)
            angle = (s["positions"].double().unsqueeze(-1) * s["inv_freq"]).unsqueeze(2)
            cos, sin = angle.cos().float(), angle.sin().float()
            outs = [_plain_rotate(x, cos, sin, case["interleaved"], s["amplitude"]) for x in leaves]
        return _with_gradients(outs, leaves, grads, dt)
    names = ("x", "h", "weight", "bias", "post_weight", "post_bias", "gate")
    leaves, grads = [s[n] for n in names], [s.get("dy"), s.get("dr")]
    if own:
        from distributed_tensorflow_amd.ops.residual_norm import residual_norm
        outs = residual_norm(s["x"], s["h"], s["weight"], s["bias"], gate=s["gate"], scale=case["scale"],
                             post_weight=s["post_weight"], post_bias=s["post_bias"], kind=case["kind"], eps=_EPS)
    else:
        leaves, grads = _in_32(*leaves), _in_32(*grads)
        x, h, weight, bias, post_weight, post_bias, gate = leaves
        n = h if post_weight is None else _plain_normed(h, post_weight, post_bias, case["kind"])
        n = n if gate is None else n * gate
        r = x + case["scale"] * n
        outs = [_plain_normed(r, weight, bias, case["kind"]), r]
    return _with_gradients(outs, leaves, grads, dt)


# ---------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits, gradients by formula
# ---------------------------------------------------------------------------------------------------------------------
def _exact_attention(s):
    case = s["case"]
    q, k, v = (s[n].detach() for n in "qkv")
    B, nq, Hq, D = q.shape
    nk, Hk = k.shape[1], k.shape[2]
    group, c = Hq // Hk, D ** -0.5
    out = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in ((q, q, k, v) if case["train"] else (q,))]
    row, col = torch.arange(nq, device=q.device)[:, None], torch.arange(nk, device=q.device)[None, :]
    for b in range(B):
        n = nk if s["lens"] is None else int(s["lens"][b])
        seen = (col < n) & (row >= 0)
        if case["causal"]:
            seen = seen & (col - row <= nk - nq)
        for h in range(Hq):
            Q, K, V = q[b, :, h].double(), k[b, :, h // group].double(), v[b, :, h // group].double()
            w = torch.where(seen, torch.exp(torch.clamp(c * (Q @ K.T.contiguous()), max=600.0)), 0.0)   # scores of unit variance: no shift is needed
            z = w.sum(1, keepdim=True)
            P = w / torch.where(z == 0, 1.0, z)
            O = P @ V
            out[0][b, :, h] = O
            if case["train"]:
                G = s["dout"][b, :, h].double()
                dP = G @ V.T.contiguous()
                dS = c * P * (dP - (P * dP).sum(1, keepdim=True))      # exactly 0 in a row that sees one key
                out[1][b, :, h] = dS @ K
                out[2][b, :, h // group] += dS.T.contiguous() @ Q
                out[3][b, :, h // group] += P.T.contiguous() @ G
    return out


def _exact_rotary(s):
    case = s["case"]
    m = case["rot_dim"] // 2
    turn = torch.polar(torch.full((), float(s["amplitude"]), dtype=torch.float64, device="cuda").expand(*s["positions"].shape, m),
                       torch.remainder(s["positions"].double()[..., None] * s["inv_freq"], 2 * math.pi)).unsqueeze(2)

    def apply(x, w):
        x = x.detach().double()
        y = x.clone()
        first, second = (slice(0, 2 * m, 2), slice(1, 2 * m, 2)) if case["interleaved"] else (slice(0, m), slice(m, 2 * m))
        z = torch.complex(x[..., first], x[..., second]) * w
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = [apply(s["q"], turn), apply(s["k"], turn)]
    return out + [apply(s["dq"], turn.conj()), apply(s["dk"], turn.conj())] if case["train"] else out


def _exact_norm(s):
    case = s["case"]
    H = case["hidden"]
    x, h, w, b, pw, pb, gate = (None if s[n] is None else s[n].detach().double() for n in
                                ("x", "h", "weight", "bias", "post_weight", "post_bias", "gate"))
    layer = case["kind"] == "layer"

    def forward(v):
        mean = v.sum(-1, keepdim=True) / H if layer else torch.zeros_like(v[..., :1])
        rstd = (((v - mean) ** 2).sum(-1, keepdim=True) / H + _EPS) ** -0.5
        return (v - mean) * rstd, rstd

    def backward(g, unit, rstd):
        g = g - unit * ((g * unit).sum(-1, keepdim=True) / H)
        if layer:
            g = g - g.sum(-1, keepdim=True) / H
        return g * rstd

    unit_h, rstd_h = forward(h) if pw is not None else (None, None)
    n = h if pw is None else unit_h * pw + (0 if pb is None else pb)
    gated = n if gate is None else n * gate
    r = x + case["scale"] * gated
    unit, rstd = forward(r)
    out = [unit * w + (0 if b is None else b), r]
    if not case["train"]:
        return out
    dy, dr = s["dy"].double(), s["dr"].double()
    dx = dr + backward(dy * w, unit, rstd)
    dgated = case["scale"] * dx
    dn = dgated if gate is None else dgated * gate
    dh = dn if pw is None else backward(dn * pw, unit_h, rstd_h)
    out += [dx, dh, (dy * unit).sum((0, 1))]
    if b is not None:
        out.append(dy.sum((0, 1)))
    if pw is not None:
        out.append((dn * unit_h).sum((0, 1)))
    if pb is not None:
        out.append(dn.sum((0, 1)))
    if gate is not None:
        over = {"channel": (0, 1), "sequence": (1,), "full": ()}[case["gate"]]
        dg = dgated * n
        out.append(dg.sum(over, keepdim=case["gate"] == "sequence") if over else dg)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "rotary": _exact_rotary, "norm": _exact_norm}[case["op"]](s)
