"""64-bit definitions of the transformer-block operators, their gradients by formula, and how far an implementation with
bf16 (fp32) results may be from them.  Rounding constants: bf16 half a step is ``U16 = 2^-8`` relative, fp32 ``U32 = 2^-24``."""
import math

import torch

U16, U32 = 2.0 ** -8, 2.0 ** -24


def step(dtype):
    return U16 if dtype == torch.bfloat16 else U32


def close(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), what + ": not finite"
    worst = ((got - want).abs() - tol).max().item()
    at = ((got - want).abs() / tol.clamp_min(1e-300)).max().item()
    assert worst <= 0, "%s: %.3g times the tolerance" % (what, at)


def attention(q, k, v, do=None, causal=False, lens=None, scale=None):
    """-> dict of out (dq, dk, dv) in 64 bits and their tolerances for bf16 kernels.

    out: P is rounded once (its relative error U16 falls on P |V|), the result once (U16 |out|); scores, exponentials and sums are
    fp32: their relative errors, (D + |s|) U32 and a few U32 each, stay under E = 4e-5 for the sizes tested.
    dS = c P (dP - D): D comes from the rounded out (|dO| . tol(out)), dS is rounded once; dq, dk then like out."""
    E = 4e-5
    q, k, v = q.double(), k.double(), v.double()
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G, c = Hq // Hk, D ** -0.5 if scale is None else scale
    want = {n: torch.zeros(s, dtype=torch.float64, device=q.device) for n, s in (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    tol = {n: torch.zeros_like(t) for n, t in want.items()}
    i, j = torch.arange(Sq, device=q.device)[:, None], torch.arange(Sk, device=q.device)[None, :]
    for b in range(B):
        n = Sk if lens is None else max(0, min(Sk, int(lens[b])))
        seen = (j < n) & (i >= 0)
        if causal:
            seen = seen & (j <= i + Sk - Sq)
        for h in range(Hq):
            Q, K, V = q[b, :, h], k[b, :, h // G].clone(), v[b, :, h // G].clone()
            K[n:], V[n:] = 0, 0
            s = (c * (Q @ K.T.contiguous())).masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True).clamp_min(-1e300)
            e = torch.exp(s - top)
            z = e.sum(1, keepdim=True)
            P = e / torch.where(z == 0, torch.ones_like(z), z)
            O = P @ V
            tO = U16 * O.abs() + (U16 + E) * (P @ V.abs())
            want["out"][b, :, h], tol["out"][b, :, h] = O, tO
            if do is None:
                continue
            g = do[b, :, h].double()
            dP = g @ V.T.contiguous()
            dS = P * (dP - (P * dP).sum(1, keepdim=True))
            aP = g.abs() @ V.T.abs().contiguous()
            eS = (U16 + E) * dS.abs() + P * ((g.abs() * tO).sum(1, keepdim=True) + E * aP + E * (P * aP).sum(1, keepdim=True))
            eP = (U16 + E) * P
            want["dq"][b, :, h] = c * dS @ K
            tol["dq"][b, :, h] = U16 * want["dq"][b, :, h].abs() + c * eS @ K.abs()
            want["dk"][b, :, h // G] += c * dS.T.contiguous() @ Q
            tol["dk"][b, :, h // G] += c * eS.T.contiguous() @ Q.abs()
            want["dv"][b, :, h // G] += P.T.contiguous() @ g
            tol["dv"][b, :, h // G] += eP.T.contiguous() @ g.abs()
    for n in ("dk", "dv"):
        tol[n] = tol[n] + U16 * want[n].abs()
    return want, {n: t * 1.01 + 1e-30 for n, t in tol.items()}


def rotary(x, inv_freq, positions, interleaved, amplitude, inverse=False):
    """-> (y, tolerance).  The angle's part of a turn is rounded to fp32 (off by at most U32 half-turns: pi U32 in the angle), sine and
    cosine are good to 2 ulp (4 U32), the amplitude and the two products and their sum round (4 U32): 12 U32 (|a| + |b|) in all."""
    dt = x.dtype
    x = x.double()
    m = inv_freq.numel()
    angle = (positions.double().reshape(-1, x.shape[1], 1, 1) * inv_freq) * (-1 if inverse else 1)
    a_at, b_at = (slice(0, 2 * m, 2), slice(1, 2 * m, 2)) if interleaved else (slice(0, m), slice(m, 2 * m))
    a, b = x[..., a_at], x[..., b_at]
    y, t = x.clone(), torch.zeros_like(x)
    y[..., a_at] = amplitude * (a * angle.cos() - b * angle.sin())
    y[..., b_at] = amplitude * (a * angle.sin() + b * angle.cos())
    t[..., a_at] = t[..., b_at] = 12 * U32 * abs(amplitude) * (a.abs() + b.abs())
    if dt == torch.bfloat16:
        t[..., :2 * m] += U16 * y[..., :2 * m].abs() * 1.01
    return y, t


def _norm(v, vmag, w, b, layer, eps):
    """unit, its magnitude (what fp32 rounds), rstd, normed, magnitude."""
    mean = v.mean(-1, keepdim=True) if layer else torch.zeros_like(v[..., :1])
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    unit, umag = (v - mean) * rstd, (vmag + mean.abs()) * rstd
    return unit, umag, rstd, unit * w + (0 if b is None else b), umag * w.abs() + (0 if b is None else b.abs())


def residual_norm(x, h, w, b=None, gate=None, scale=1.0, pw=None, pb=None, kind="rms", eps=1e-6, dy=None, dr=None, rows_sum=64):
    """-> (values, tolerances) of y, r, dx, dh, dw, db, dgate, dpw, dpb in 64 bits.  Every fp32 value is off by at most N U32 times its
    magnitude (the same expression with absolute values): sums of a row go over up to 32 terms a thread and 10 levels, a norm, a gate
    and a residual round about 10 times: N = 64 forward, 256 through both backward norms (their sums multiply two such values), and
    ``rows_sum`` more for the sums over rows.  Then the result's own rounding."""
    u = step(x.dtype)
    up = step(w.dtype)
    x, h, w, b, gate, pw, pb, dy, dr = (None if t is None else t.double() for t in (x, h, w, b, gate, pw, pb, dy, dr))
    layer = kind == "layer"
    H = x.shape[-1]
    n, nmag = h, h.abs()
    if pw is not None:
        hu, humag, hr, n, nmag = _norm(h, h.abs(), pw, pb, layer, eps)
    gn, gmag = (n, nmag) if gate is None else (n * gate, nmag * gate.abs())
    r, rmag = x + scale * gn, x.abs() + abs(scale) * gmag
    unit, umag, rstd, y, ymag = _norm(r, rmag, w, b, layer, eps)
    want, mag = {"y": y, "r": r}, {"y": 64 * ymag, "r": 64 * rmag}
    if dy is not None or dr is not None:
        zero = torch.zeros_like(x)
        dy, dr = (zero if t is None else t for t in (dy, dr))

        def back(g, gm, un, um, rs):
            d = g - un * (g * un).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if layer else 0)
            m = gm + um * (gm * um).mean(-1, keepdim=True) + (gm.mean(-1, keepdim=True) if layer else 0)
            return d * rs, m * rs

        def rows(t):
            return t.reshape(-1, H).sum(0)

        d, m = back(dy * w, dy.abs() * w.abs(), unit, umag, rstd)
        d, m = d + dr, m + dr.abs()
        want["dx"], mag["dx"] = d, 256 * m
        want["dw"], mag["dw"] = rows(dy * unit), (64 + rows_sum) * rows(dy.abs() * umag)
        if b is not None:
            want["db"], mag["db"] = rows(dy), (64 + rows_sum) * rows(dy.abs())
        dg, dgm = scale * d * n, abs(scale) * m * nmag
        if gate is not None:
            full = gate.expand_as(x)
            over = [i for i in range(x.dim()) if full.shape[i] != ((1,) * (x.dim() - gate.dim()) + tuple(gate.shape))[i]]
            red = (lambda t: t.sum(over, keepdim=True).reshape(gate.shape)) if over else (lambda t: t)
            want["dgate"], mag["dgate"] = red(dg), (256 + rows_sum) * red(dgm)
        dn, dnm = scale * d, abs(scale) * m
        if gate is not None:
            dn, dnm = dn * gate, dnm * gate.abs()
        if pw is not None:
            want["dpw"], mag["dpw"] = rows(dn * hu), (256 + rows_sum) * rows(dnm * humag)
            if pb is not None:
                want["dpb"], mag["dpb"] = rows(dn), (256 + rows_sum) * rows(dnm)
            dn, dnm = back(dn * pw, dnm * pw.abs(), hu, humag, hr)
        want["dh"], mag["dh"] = dn, 512 * dnm
    tol = {}
    for k, t in want.items():
        own = up if k in ("dw", "db", "dpw", "dpb") else u
        tol[k] = (own * t.abs() if own > U32 else 0) * 1.01 + U32 * mag[k] + 1e-35
    return want, tol


def attention_noise(q, k, v, do, causal=False, lens=None, few=256, tile=128):
    """-> the norm that the error of out, dq, dk, dv may have where exactly the documented roundings are made: P, dS and the results
    to bf16, D from the rounded out except in tiles of ``tile`` queries that see up to ``few`` keys (fp32 there).

    A rounding is off by up to half a step, evenly spread: in the mean square U16^2 / 3 times the value's square just above a power of
    two, and 3 / (8 ln 2) = 0.541 of that over mantissas as they occur (density 1 / (m ln 2) on 1 <= m < 2).  Roundings are
    independent of each other, so the squares add up over the sums that they go through; fp32's part is a thousandth of them.
    A tenth more than that norm is allowed: it is a sum over thousands of elements, and scatters by one or two parts in a hundred."""
    W = U16 ** 2 / 3 * 3 / (8 * math.log(2))
    q, k, v, do = q.double(), k.double(), v.double(), do.double()
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G, c = Hq // Hk, D ** -0.5
    val = {n: torch.zeros(s, dtype=torch.float64, device=q.device) for n, s in (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    var = {n: torch.zeros_like(t) for n, t in val.items()}
    i, j = torch.arange(Sq, device=q.device)[:, None], torch.arange(Sk, device=q.device)[None, :]
    last = ((i // tile + 1) * tile).clamp_max(Sq) - 1
    for b in range(B):
        n = Sk if lens is None else max(0, min(Sk, int(lens[b])))
        seen = (j < n) & (i >= 0)
        sees = torch.full_like(last, n)
        if causal:
            seen = seen & (j <= i + Sk - Sq)
            sees = torch.minimum(sees, last + 1 + Sk - Sq)
        for h in range(Hq):
            Q, K, V, g = q[b, :, h], k[b, :, h // G].clone(), v[b, :, h // G].clone(), do[b, :, h]
            K[n:], V[n:] = 0, 0
            s = (c * (Q @ K.T.contiguous())).masked_fill(~seen, -math.inf)
            e = torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e300))
            z = e.sum(1, keepdim=True)
            P = e / torch.where(z == 0, torch.ones_like(z), z)
            P2 = P ** 2
            val["out"][b, :, h] = P @ V
            var["out"][b, :, h] = W * (P2 @ V ** 2)
            dP = g @ V.T.contiguous()
            dS = P * (dP - (P * dP).sum(1, keepdim=True))
            D2 = (g ** 2 * (var["out"][b, :, h] + W * val["out"][b, :, h] ** 2)).sum(1, keepdim=True)
            D2 = torch.where(sees <= few, torch.zeros_like(D2), D2)
            val["dq"][b, :, h] = c * dS @ K
            var["dq"][b, :, h] = c * c * (W * dS ** 2 @ K ** 2 + D2 * (P @ K) ** 2)
            val["dk"][b, :, h // G] += c * dS.T.contiguous() @ Q
            var["dk"][b, :, h // G] += c * c * (W * dS ** 2 + P2 * D2).T.contiguous() @ Q ** 2
            val["dv"][b, :, h // G] += P.T.contiguous() @ g
            var["dv"][b, :, h // G] += W * P2.T.contiguous() @ g ** 2
    return val, {n: 1.1 * math.sqrt((t + W * val[n] ** 2).sum().item()) for n, t in var.items()}


def attention_rounded(q, k, v, do, causal=False, lens=None, few=256, tile=128, rounded_d=False, rounded_s=False, lost_key=None):
    """The backward's and forward's arithmetic with exactly the documented roundings; ``rounded_d``, ``rounded_s``, ``lost_key`` plant a
    mistake (D or the scores in bf16, one key left out of the sums)."""
    def r(t):
        return t.to(torch.bfloat16).double()

    q, k, v, do = q.double(), k.double(), v.double(), do.double()
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G, c = Hq // Hk, D ** -0.5
    got = {n: torch.zeros(s, dtype=torch.float64) for n, s in (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    i, j = torch.arange(Sq)[:, None], torch.arange(Sk)[None, :]
    last = ((i // tile + 1) * tile).clamp_max(Sq) - 1
    for b in range(B):
        n = Sk if lens is None else max(0, min(Sk, int(lens[b])))
        seen = (j < n) & (i >= 0) & (j != (-1 if lost_key is None else lost_key))
        sees = torch.full_like(last, n)
        if causal:
            seen = seen & (j <= i + Sk - Sq)
            sees = torch.minimum(sees, last + 1 + Sk - Sq)
        for h in range(Hq):
            Q, K, V, g = q[b, :, h], k[b, :, h // G], v[b, :, h // G], do[b, :, h]
            s = c * (Q @ K.T)
            s = (r(s) if rounded_s else s).masked_fill(~seen, -math.inf)
            m = s.amax(1, keepdim=True).clamp_min(-1e300)
            e = torch.exp(s - m)
            z = e.sum(1, keepdim=True)
            z = torch.where(z == 0, torch.ones_like(z), z)
            O = r((r(e) @ V) / z)
            P, dP = e / z, g @ V.T
            d = torch.where(sees <= few, (P * dP).sum(1, keepdim=True), (g * O).sum(1, keepdim=True))
            dS = r(P * (dP - (r(d) if rounded_d else d)))
            got["out"][b, :, h] = O
            got["dq"][b, :, h] = c * dS @ K
            got["dk"][b, :, h // G] += c * dS.T @ Q
            got["dv"][b, :, h // G] += r(P).T @ g
    return {n: r(t) for n, t in got.items()}
