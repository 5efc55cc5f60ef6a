"""The transformer-block kernels (K22 attention of any length, K23 rotary positions, K24 block boundary) against their
definitions in 64 bits, with tolerances derived in ``block_oracles``."""
import pytest
import torch

import block_oracles as oracle

pytestmark = pytest.mark.gpu

from distributed_tensorflow_amd.ops import hip  # noqa: E402
from distributed_tensorflow_amd.ops.attention import attention  # noqa: E402
from distributed_tensorflow_amd.ops.residual_norm import FusedRMSNorm, residual_norm, rms_norm  # noqa: E402
from distributed_tensorflow_amd.ops.rotary import rotary, rotary_frequencies  # noqa: E402

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    hip.lib()
    return torch.device("cuda", 0)


def _randn(dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device=dev)


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
ATT = [
    # B, Sq, Sk, Hq, Hk, D, causal, lens
    (1, 1, 1, 1, 1, 64, False, None), (2, 1, 1, 2, 1, 128, True, None), (1, 2, 2, 3, 3, 64, True, None),
    (2, 37, 37, 12, 12, 64, False, (18, 37)), (3, 33, 33, 4, 2, 64, True, (0, 1, 33)),
    (1, 64, 64, 2, 2, 128, True, None), (1, 65, 65, 2, 1, 128, True, None), (2, 129, 129, 4, 1, 64, True, (129, 70)),
    (1, 300, 300, 2, 2, 80, True, None), (1, 257, 257, 6, 2, 96, False, (200,)), (1, 200, 200, 1, 1, 8, True, None),
    (1, 130, 130, 2, 2, 32, False, None), (1, 1000, 1000, 2, 1, 64, True, None), (1, 640, 640, 5, 1, 128, True, (513,)),
    # queries and keys of different lengths; causal ones end together; the third leaves 60 rows empty
    (2, 1, 300, 8, 2, 128, False, (300, 5)), (2, 7, 515, 8, 1, 128, True, None), (1, 100, 40, 2, 2, 64, True, None),
    (2, 140, 1, 3, 1, 64, True, None), (1, 257, 1100, 4, 4, 64, True, (900,)), (4, 1, 129, 4, 4, 64, False, (0, 1, 64, 129)),
    (1, 31, 2000, 40, 8, 128, True, None), (1, 513, 65, 2, 1, 128, False, None),
    # every width of the products, with and without columns behind the head's
    (2, 150, 150, 4, 2, 24, True, (150, 31)), (2, 1, 400, 4, 1, 32, False, (400, 9)), (1, 90, 333, 8, 1, 40, False, None),
    (1, 200, 200, 3, 3, 72, True, None), (2, 3, 700, 8, 2, 96, True, None), (1, 130, 190, 2, 1, 104, False, (150,)),
]


def _att_inputs(dev, B, Sq, Sk, Hq, Hk, D, packed):
    r = _randn(dev, Sq * 1000 + Sk + D)
    if packed and Sq == Sk:
        q, k, v = r(B, Sq, Hq + 2 * Hk, D).to(BF).split([Hq, Hk, Hk], 2)
    else:
        q, k, v = r(B, Sq, Hq, D).to(BF), r(B, Sk, Hk, D).to(BF), r(B, Sk, Hk, D).to(BF)
    return q, k, v, r(B, Sq, Hq, D).to(BF)


@pytest.mark.parametrize("B,Sq,Sk,Hq,Hk,D,causal,lens", ATT)
def test_attention_matches_the_definition(dev, B, Sq, Sk, Hq, Hk, D, causal, lens):
    q, k, v, do = _att_inputs(dev, B, Sq, Sk, Hq, Hk, D, True)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*leaves, causal=causal, kv_len=n)
    grads = torch.autograd.grad(out, leaves, do)
    want, tol = oracle.attention(q, k, v, do, causal, lens)
    for name, got in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        oracle.close(got.detach(), want[name], tol[name], name)
    again = attention(q, k, v, causal=causal, kv_len=n)
    assert torch.equal(again, out)                                     # without gradients, and again: the same bits
    if Sk == 1:
        assert not grads[0].any() and not grads[1].any()               # one key: the probabilities are constant


NOISE = [
    (8, 16, 16, 4, 2, 64, True, None), (2, 37, 37, 12, 12, 64, False, (18, 37)), (2, 64, 64, 4, 4, 128, True, None), (2, 129, 129, 4, 1, 64, True, (129, 70)),
    (1, 300, 300, 4, 2, 80, True, None), (1, 640, 640, 5, 1, 128, True, (513,)), (3, 1000, 1000, 12, 12, 64, False, (333, 666, 1000)),
    (1, 2048, 2048, 8, 2, 128, True, None), (2, 257, 1500, 8, 2, 128, True, None), (4, 1, 1100, 32, 8, 128, False, (275, 550, 825, 1100)), (2, 200, 200, 6, 2, 32, True, None),
]


@pytest.mark.parametrize("B,Sq,Sk,Hq,Hk,D,causal,lens", NOISE)
def test_attention_rounds_only_where_it_says(dev, B, Sq, Sk, Hq, Hk, D, causal, lens):
    """The norms of the errors: far sharper than the bounds of single elements, they would show D or scores held in bf16."""
    q, k, v, do = _att_inputs(dev, B, Sq, Sk, Hq, Hk, D, True)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*leaves, causal=causal, kv_len=n)
    got = (out.detach(),) + torch.autograd.grad(out, leaves, do)
    want, most = oracle.attention_noise(q, k, v, do, causal, lens)
    over = {m: ((g.double() - want[m]).norm().item() / most[m]) for m, g in zip(("out", "dq", "dk", "dv"), got)}
    assert max(over.values()) < 1, over


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_attention_scale_and_large_scores(dev, scale):
    q, k, v, do = _att_inputs(dev, 1, 150, 150, 2, 2, 64, False)
    q = (q.float() * 8).to(BF)                                         # scores of standard deviation 64 at scale 1
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*leaves, causal=True, scale=scale)
    grads = torch.autograd.grad(out, leaves, do)
    want, tol = oracle.attention(q, k, v, do, True, scale=scale)
    for name, got in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        oracle.close(got.detach(), want[name], tol[name], name)


def test_attention_padding_is_never_read(dev):
    B, S, H, D = 3, 200, 2, 64
    q, k, v, do = _att_inputs(dev, B, S, S, H, H, D, False)
    lens = (200, 77, 0)
    n = torch.tensor(lens, dtype=torch.int64, device=dev)
    got = []
    for poison in (0.0, float("nan"), float("inf")):
        kk, vv = k.clone(), v.clone()
        for b, m in enumerate(lens):
            kk[b, m:], vv[b, m:] = poison, poison
        leaves = [t.detach().requires_grad_() for t in (q, kk, vv)]
        out = attention(*leaves, kv_len=n)
        got.append((out.detach(),) + torch.autograd.grad(out, leaves, do))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)
    assert not got[0][0][2].any() and not got[0][1][2].any()            # no key: zeros, and no gradient
    for g in got[0][2:]:
        for b, m in enumerate(lens):
            assert not g[b, m:].any()


def test_attention_key_lengths_outside_the_range(dev):
    q, k, v, _ = _att_inputs(dev, 3, 70, 70, 2, 2, 64, False)
    a = attention(q, k, v, kv_len=torch.tensor([-5, 70, 2 ** 40], device=dev))
    b = attention(q, k, v, kv_len=torch.tensor([0, 70, 70], dtype=torch.int32))
    c = attention(q, k, v, kv_len=torch.tensor([-1, 1000, 70], dtype=torch.int32, device=dev))
    assert torch.equal(a, b) and torch.equal(a, c)
    assert torch.equal(attention(q, k, v, kv_len=torch.tensor([0, 255, 70], dtype=torch.uint8, device=dev)), a)


def test_attention_other_strides_and_orders(dev):
    B, S, H, D = 2, 90, 4, 64
    q, k, v, do = _att_inputs(dev, B, S, S, H, H, D, False)
    plain = attention(q, k, v, causal=True)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]              # [B, H, S, D] memory
    assert torch.equal(attention(*heads_first, causal=True), plain)
    last = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]                     # D not dense: copied
    assert torch.equal(attention(*last, causal=True), plain)
    odd = [torch.cat([t.new_zeros(3), t.reshape(-1)])[3:].view(t.shape) for t in (q, k, v)]        # not 16-B aligned: copied
    assert torch.equal(attention(*odd, causal=True), plain)
    one = k[:, :, :1].expand(B, S, H, D)                                                           # a broadcast key head
    leaf = k[:, :, :1].detach().clone().requires_grad_()
    out = attention(q, leaf.expand(B, S, H, D), v, causal=True)
    assert torch.equal(out, attention(q, one.contiguous(), v, causal=True))
    dk, = torch.autograd.grad(out, leaf, do)
    full = one.contiguous().requires_grad_()
    want, = torch.autograd.grad(attention(q, full, v, causal=True), full, do)
    assert torch.equal(dk, want.sum(2, keepdim=True))
    wide = q.detach().requires_grad_()
    g1, = torch.autograd.grad(attention(wide, k, v).sum(), wide)                                   # an expanded gradient
    g2, = torch.autograd.grad(attention(wide, k, v), wide, torch.ones_like(q))
    assert torch.equal(g1, g2)


@pytest.mark.parametrize("Hk", [4, 1])
def test_attention_of_a_query_does_not_depend_on_the_others(dev, Hk):
    q, k, v, do = _att_inputs(dev, 2, 300, 300, 4, Hk, 64, False)
    out = attention(q, k, v)
    g, = torch.autograd.grad(attention(leaf := q.detach().requires_grad_(), k, v), leaf, do)
    other = q.clone()
    other[:, 5], other[:, 200] = other[:, 5] * 50, 0
    got = attention(other, k, v)
    h, = torch.autograd.grad(attention(leaf := other.detach().requires_grad_(), k, v), leaf, do)
    keep = [i for i in range(300) if i not in (5, 200)]
    assert torch.equal(got[:, keep], out[:, keep]) and torch.equal(h[:, keep], g[:, keep])
    assert torch.equal(attention(q[1:], k[1:], v[1:]), out[1:])


@pytest.mark.parametrize("B,Sq,Sk,Hq,Hk,D,causal", [(2, 1000, 1000, 12, 12, 64, False), (2, 257, 1500, 8, 2, 128, True), (3, 700, 700, 4, 1, 96, True)])
def test_attention_of_a_sequence_does_not_depend_on_what_the_others_hold(dev, B, Sq, Sk, Hq, Hk, D, causal):
    """Sums split over workgroups: one sequence's results have the same bits whatever the others hold and however long they are, in a
    call of the same shapes.  (In a batch of another size the parts may be others, and the bits with them.)"""
    from distributed_tensorflow_amd.ops import attention as A

    q, k, v, do = _att_inputs(dev, B, Sq, Sk, Hq, Hk, D, False)

    def parts(rows):
        how = A._general_operands(*(t.expand(rows, -1, -1, -1) for t in (q[:1], k[:1], v[:1])), None, int(causal), 1.0)[3]
        return A._general_kernels()[2](how)

    assert parts(B) > 0 and parts(64) == 0
    got = []
    for other, n in ((1.0, Sk), (1.0, Sk), (-3.0, Sk // 3), (100.0, 0)):
        t = [x.clone() for x in (q, k, v, do)]
        for x in t:
            x[1:] *= other
        lens = torch.tensor([Sk - 9] + [n] * (B - 1), dtype=torch.int32, device=dev)
        leaves = [x.requires_grad_() for x in t[:3]]
        out = attention(*leaves, causal=causal, kv_len=lens)
        got.append([x[0] for x in (out.detach(),) + torch.autograd.grad(out, leaves, t[3])])
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)


def test_attention_nan_reaches_its_query(dev):
    q, k, v, _ = _att_inputs(dev, 1, 70, 70, 1, 1, 64, False)
    clean = attention(q, k, v, causal=True)
    q[0, 40, 0, 3] = float("nan")
    out = attention(q, k, v, causal=True)
    assert bool(out[0, 40].isnan().all())
    keep = [i for i in range(70) if i != 40]
    assert torch.equal(out[:, keep], clean[:, keep])


# ---------------------------------------------------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------------------------------------------------
ROT = [
    # B, S, Hq, Hk, D, pairs, dtype
    (1, 1, 1, 1, 2, 1, F32), (8, 1, 32, 8, 128, 64, BF), (2, 37, 12, 12, 64, 32, BF), (3, 50, 4, 2, 96, 32, F32),
    (2, 33, 3, 1, 128, 7, BF), (1, 129, 2, 2, 80, 40, BF), (1, 65, 2, 1, 64, 8, BF), (2, 17, 5, 5, 10, 3, F32), (1, 300, 40, 8, 128, 64, BF),
    (1, 70, 2, 1, 256, 128, F32), (2, 19, 2, 2, 2048, 1024, BF), (1, 21, 4, 4, 128, 38, BF),
    # pairs and rests that are no whole vectors: the last one over the one before, a rest of less than a vector
    (2, 23, 4, 2, 128, 37, BF), (1, 40, 3, 1, 128, 63, BF), (2, 9, 2, 2, 96, 45, BF), (1, 31, 2, 1, 64, 29, F32), (2, 13, 2, 1, 26, 9, BF),
    (1, 17, 3, 2, 20, 9, F32), (1, 25, 2, 1, 6, 2, BF), (1, 26, 2, 1, 4, 1, BF), (1, 27, 1, 1, 8, 3, F32), (3, 7, 2, 1, 22, 8, BF),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,Hq,Hk,D,m,dt", ROT)
def test_rotary_matches_the_definition(dev, B, S, Hq, Hk, D, m, dt, interleaved):
    r = _randn(dev, S * 100 + D)
    q, k, _ = r(B, S, Hq + 2 * Hk, D).to(dt).split([Hq, Hk, Hk], 2)
    gq, gk = r(B, S, Hq, D).to(dt), r(B, S, Hk, D).to(dt)
    f, amp = rotary_frequencies(2 * m, scaling="by_parts", factor=4.0, original_length=2048, device=dev)
    pos = torch.randint(0, 1 << 20, (B, 1), device=dev, generator=torch.Generator(dev).manual_seed(S)) + torch.arange(S, device=dev)
    leaves = [t.detach().requires_grad_() for t in (q, k)]
    outs = rotary(*leaves, f, pos, interleaved=interleaved, amplitude=amp)
    grads = torch.autograd.grad(outs, leaves, (gq, gk))
    for name, x, got, inv in (("q", q, outs[0], False), ("k", k, outs[1], False), ("dq", gq, grads[0], True), ("dk", gk, grads[1], True)):
        want, tol = oracle.rotary(x, f, pos, interleaved, amp, inv)
        oracle.close(got.detach(), want, tol, name)
    assert torch.equal(outs[0][..., 2 * m:], q[..., 2 * m:]) and torch.equal(grads[1][..., 2 * m:], gk[..., 2 * m:])


def test_rotary_positions(dev):
    r = _randn(dev, 5)
    q, k = r(2, 40, 4, 64).to(BF), r(2, 40, 2, 64).to(BF)
    f, _ = rotary_frequencies(64, device=dev)
    at = torch.arange(40, device=dev)
    base = rotary(q, k, f, offset=7)
    for pos in (at + 7, (at + 7).int(), (at + 7).expand(2, 40), (at + 7)[None], torch.stack([at + 7, at + 7], 1).t()):
        for a, b in zip(base, rotary(q, k, f, pos)):
            assert torch.equal(a, b)
    alone = rotary(q, None, f, offset=7)
    assert alone[1] is None and torch.equal(alone[0], base[0])
    zero = rotary(q, k, f, torch.zeros(40, dtype=torch.int64, device=dev))
    assert torch.equal(zero[0], q) and torch.equal(zero[1], k)
    far = torch.tensor([[-3, 0, 1 << 40, 2 ** 31 + 11]], device=dev)                  # negative, and past 32 bits
    y, _ = rotary(q[:1, :4].float(), None, f, far)
    want, tol = oracle.rotary(q[:1, :4].float(), f, far, False, 1.0)
    # (position 2^40: position * frequency carries 2^40 * 2^-53 = 1.3e-4 in the angle, on both sides)
    oracle.close(y, want, tol + 2 * 2 ** -13 * torch.tensor([0, 0, 1.0, 0], device=dev).view(1, 4, 1, 1) * q[:1, :4].abs().amax() * 2, "far")
    leaf = q.detach().requires_grad_()
    g, = torch.autograd.grad(rotary(leaf, None, f, offset=7)[0].sum(), leaf)          # an expanded gradient
    assert torch.equal(g, rotary(torch.ones_like(q), None, f, -(at + 7))[0])


# ---------------------------------------------------------------------------------------------------------------------
# block boundary
# ---------------------------------------------------------------------------------------------------------------------
NORM = [
    # shape, kind, post, gate, scale, dtype, parameter dtype
    ((1, 1, 1), "rms", False, "none", 1.0, F32, F32), ((8, 1, 4096), "rms", True, "none", 0.5, BF, BF),
    ((2, 100, 768), "layer", False, "channel", 1.0, BF, BF), ((3, 37, 768), "layer", True, "sequence", 0.3, BF, F32),
    ((2, 65, 1024), "rms", True, "full", 0.25, BF, BF), ((3, 33, 1001), "rms", False, "full", 0.7, F32, F32),
    ((2, 20, 1001), "layer", True, "channel", 0.7, BF, BF), ((1, 50, 2000), "rms", True, "sequence", 1.0, BF, BF),
    ((2, 9, 4100), "layer", True, "sequence", 2.0, F32, F32), ((1, 6, 8192), "rms", True, "channel", 0.1, BF, BF),
    ((2, 3, 16384), "layer", True, "full", 0.1, BF, BF), ((2, 3, 16381), "layer", True, "sequence", 0.1, F32, F32),
    ((5, 40, 16), "rms", False, "none", 1.0, BF, BF), ((3, 11, 520), "layer", True, "none", 1.0, F32, F32),
    ((700, 128), "rms", True, "channel", 0.5, BF, BF), ((6, 3, 5, 256), "rms", True, "sequence", 0.5, BF, BF),
    ((1500, 2, 64), "layer", False, "sequence", 1.0, BF, BF), ((2, 17, 5000), "rms", False, "channel", 1.0, BF, F32),
    ((600, 3, 4096), "rms", True, "sequence", 0.5, BF, BF),              # more gate rows than workgroups (as 1500 x 64 above)
    # rows that end inside a vector, and rows shorter than one
    ((3, 41, 2047), "rms", True, "sequence", 0.5, BF, BF), ((2, 30, 4094), "layer", True, "full", 1.0, BF, BF),
    ((1, 9, 513), "layer", False, "channel", 1.0, BF, F32), ((2, 8, 1022), "rms", True, "full", 0.5, BF, F32),
    ((2, 20, 2051), "layer", True, "sequence", 1.0, F32, F32), ((2, 33, 9), "layer", True, "none", 1.0, BF, BF),
    ((4, 7, 7), "layer", True, "channel", 1.0, BF, BF), ((2, 70, 5), "rms", True, "sequence", 1.0, BF, F32),
    ((3, 5, 3), "layer", True, "full", 1.0, F32, F32), ((2, 40, 2), "rms", False, "full", 1.0, BF, BF), ((2, 9, 6001), "rms", True, "full", 1.0, BF, BF),
]


def _norm_inputs(dev, shape, kind, post, gate, dt, pdt):
    r = _randn(dev, shape[-1] + len(shape))
    H = shape[-1]
    x, h = (r(*shape) * torch.exp(r(H))).to(dt), (r(*shape) * 1.5 + 0.3).to(dt)
    w, b = (1 + 0.2 * r(H)).to(pdt), (0.1 * r(H)).to(pdt) if kind == "layer" else None
    pw = (1 + 0.2 * r(H)).to(pdt) if post else None
    pb = (0.1 * r(H)).to(pdt) if post and kind == "layer" else None
    gs = {"none": None, "channel": (H,), "sequence": shape[:1] + (1,) * (len(shape) - 2) + (H,), "full": shape}[gate]
    return dict(x=x, h=h, w=w, b=b, gate=None if gs is None else (0.3 + 0.5 * r(*gs)).to(dt), pw=pw, pb=pb), r(*shape).to(dt), (0.5 * r(*shape)).to(dt)


@pytest.mark.parametrize("grads", ["both", "y", "r"])
@pytest.mark.parametrize("shape,kind,post,gate,scale,dt,pdt", NORM)
def test_residual_norm_matches_the_definition(dev, shape, kind, post, gate, scale, dt, pdt, grads):
    t, dy, dr = _norm_inputs(dev, shape, kind, post, gate, dt, pdt)
    leaf = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    y, r = residual_norm(leaf["x"], leaf["h"], leaf["w"], leaf["b"], gate=leaf["gate"], scale=scale, post_weight=leaf["pw"],
                         post_bias=leaf["pb"], kind=kind)
    dy, dr = dy if grads != "r" else None, dr if grads != "y" else None
    names = [n for n, v in leaf.items() if v is not None]
    outs = [(o, g) for o, g in ((y, dy), (r, dr)) if g is not None]
    got = torch.autograd.grad([o for o, _ in outs], [leaf[n] for n in names], [g for _, g in outs], allow_unused=True)
    want, tol = oracle.residual_norm(**t, scale=scale, kind=kind, dy=dy, dr=dr)
    oracle.close(y.detach(), want["y"], tol["y"], "y")
    oracle.close(r.detach(), want["r"], tol["r"], "r")
    for n, g in zip(names, got):
        if g is None:
            assert grads == "r" and n in ("w", "b"), n
            continue
        assert g.dtype == leaf[n].dtype and g.shape == leaf[n].shape
        oracle.close(g, want["d" + n], tol["d" + n], "d" + n)


def test_rms_norm_and_module(dev):
    r = _randn(dev, 3)
    x, w, dy = r(3, 50, 768).to(BF), (1 + 0.2 * r(768)).to(BF), r(3, 50, 768).to(BF)
    lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = rms_norm(lx, lw, 1e-5)
    dx, dw = torch.autograd.grad(y, (lx, lw), dy)
    zero = torch.zeros_like(x)
    want, tol = oracle.residual_norm(x, zero, w, dy=dy, eps=1e-5)
    for n, got in (("y", y), ("dx", dx), ("dw", dw)):
        oracle.close(got.detach(), want[n], tol[n], n)
    m = FusedRMSNorm(768, eps=1e-5).to(dev, BF)
    assert torch.equal(m(x), rms_norm(x, m.weight, 1e-5))
    a, b = m(x, dy, scale=0.5), residual_norm(x, dy, m.weight, scale=0.5, eps=1e-5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_residual_norm_unaligned_rows_equal_aligned_ones(dev):
    t, dy, dr = _norm_inputs(dev, (2, 21, 768), "rms", True, "full", BF, BF)
    res = []
    for off in (0, 1):
        v = {n: None if u is None else torch.cat([u.new_zeros(off), u.reshape(-1)])[off:].view(u.shape).requires_grad_() for n, u in t.items()}
        y, r = residual_norm(v["x"], v["h"], v["w"], gate=v["gate"], scale=0.5, post_weight=v["pw"])
        g = torch.autograd.grad((y, r), [u for u in v.values() if u is not None], (dy, dr))
        res.append((y.detach(), r.detach()) + g)
    want, tol = oracle.residual_norm(**t, scale=0.5, dy=dy, dr=dr)
    for got in res:
        for n, g in zip(("y", "r", "dx", "dh", "dw", "dgate", "dpw"), got):
            oracle.close(g, want[n], tol[n], n)


# ---------------------------------------------------------------------------------------------------------------------
# how they are called: offsets past 32 bits, the same tensor twice, streams, graphs, refusals
# ---------------------------------------------------------------------------------------------------------------------
def test_saved_tensors_that_come_back_in_another_layout(dev):
    """Hooks on saved tensors (moved to the host and back, or laid out anew) change addresses and strides under the backward."""
    r = _randn(dev, 21)
    q, k, v = r(2, 70, 8, 64).to(BF).split([4, 2, 2], 2)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    lens = torch.tensor([70, 31], dtype=torch.int32, device=dev)
    f, _ = rotary_frequencies(64, device=dev)
    x, h, w, pw = (t.to(BF).requires_grad_() for t in (r(2, 70, 256), r(2, 70, 256), 1 + 0.1 * r(256), 1 + 0.1 * r(256)))
    gate = r(2, 1, 256).to(BF).requires_grad_()
    every = leaves + [x, h, w, pw, gate]
    pos = (3 + torch.arange(70, device=dev)).expand(2, 70)

    def run():
        a, b = rotary(leaves[0], leaves[1], f, pos)
        o = attention(a, b, leaves[2], causal=True, kv_len=lens) + attention(*leaves, kv_len=lens)
        y, s = residual_norm(x, h + o.flatten(2), w, gate=gate, post_weight=pw)
        return y, s

    dy, ds = r(2, 70, 256).to(BF), r(2, 70, 256).to(BF)
    want = torch.autograd.grad(run(), every, (dy, ds))

    def apart(t):                                         # every second element of a buffer, last dimension first
        buf = t.new_zeros(tuple(reversed(t.shape)) + (2,))[..., 0].permute(*reversed(range(t.dim())))
        return buf.copy_(t)

    hooks = (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: apart(t.detach()), lambda t: t))
    for hook in hooks:
        with hook:
            outs = run()
        junk = [torch.full_like(t, 7) for t in every for _ in range(3)]                 # memory given back is in other hands
        for a, b in zip(torch.autograd.grad(outs, every, (dy, ds)), want):
            assert torch.equal(a, b)
        del junk


def test_attention_offsets_past_32_bits(dev):
    r = _randn(dev, 11)
    B, S, H, D = 2, 130, 2, 64
    q, k, v, do = (r(B, S, H, D).to(BF) for _ in range(4))
    want = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*want, causal=True)
    ref = (out.detach(),) + torch.autograd.grad(out, want, do)
    far, rows = (1 << 31) + 64, (1 << 24) + 8
    for bs, ss, n in ((far, H * D, S), (H * D, rows, S), (H * D, 1 << 25, 5)):      # sequences, tokens far apart; tokens too far: copied
        buf = torch.empty(bs + n * ss + H * D, dtype=BF, device=dev)
        kk = buf.as_strided((B, n, H, D), (bs, ss, D, 1))
        kk.copy_(k[:, :n])
        leaf = [t.detach().requires_grad_() for t in (q[:, :n], kk, v[:, :n])]
        out = attention(*leaf, causal=True)
        got = (out.detach(),) + torch.autograd.grad(out, leaf, do[:, :n])
        for a, b in zip(ref[:4 if n == S else 2], got):                 # (the first tokens' outputs and dq do not depend on later ones)
            assert torch.equal(a[:, :n], b)
        del buf, kk, leaf, out


def test_attention_results_past_32_bits(dev):
    r = _randn(dev, 12)
    B, S, H, D = (1 << 18) + 3, 16, 8, 64                               # 2^31 elements a tensor
    q, k, v, do = (r(5, S, H, D).to(BF).repeat((B + 4) // 5, 1, 1, 1)[:B] for _ in range(4))
    leaf = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*leaf, causal=True)
    got = (out.detach(),) + torch.autograd.grad(out, leaf, do)
    few = [t[-5:].clone().requires_grad_() for t in (q, k, v)]
    out = attention(*few, causal=True)
    for a, b in zip(got, (out.detach(),) + torch.autograd.grad(out, few, do[-5:])):
        assert torch.equal(a[-5:], b)


def test_rotary_and_norm_past_32_bits(dev):
    r = _randn(dev, 13)
    B, S, H, D = 1030, 512, 32, 128                                     # 2.16e9 elements a tensor
    q = r(2, S, H, D).to(BF).repeat(B // 2, 1, 1, 1)
    f, _ = rotary_frequencies(D, device=dev)
    y, _ = rotary(q, None, f)
    few, _ = rotary(q[-3:].clone(), None, f)
    assert torch.equal(y[-3:], few)
    x, h = q.view(-1, H * D), y.view(-1, H * D)
    w, pw, gate = (1 + 0.1 * r(H * D).to(BF) for _ in range(3))
    leaf = [t.detach().requires_grad_() for t in (x, h)]
    out = residual_norm(*leaf, w, gate=gate, post_weight=pw, scale=0.5)
    got = tuple(t.detach()[-40:].clone() for t in out) + tuple(t[-40:].clone() for t in torch.autograd.grad(out, leaf, (h, x)))
    leaf = [t.detach()[-40:].clone().requires_grad_() for t in (x, h)]
    out = residual_norm(*leaf, w, gate=gate, post_weight=pw, scale=0.5)
    for a, b in zip(got, tuple(t.detach() for t in out) + torch.autograd.grad(out, leaf, (h[-40:], x[-40:]))):
        assert torch.equal(a, b)


def test_the_same_tensor_in_several_places(dev):
    r = _randn(dev, 14)
    x, do = r(2, 70, 4, 64).to(BF), r(2, 70, 4, 64).to(BF)
    leaf = x.detach().requires_grad_()
    g, = torch.autograd.grad(attention(leaf, leaf, leaf, causal=True), leaf, do)
    three = [x.detach().clone().requires_grad_() for _ in range(3)]
    dq, dk, dv = torch.autograd.grad(attention(*three, causal=True), three, do)
    # autograd adds the three in bf16: two roundings of the sums
    tol = 2 * oracle.U16 * (dq.double().abs() + dk.double().abs() + dv.double().abs())
    oracle.close(g, dq.double() + dk.double() + dv.double(), tol, "sum of the three")
    f, _ = rotary_frequencies(64, device=dev)
    a, b = rotary(x, x, f)
    assert torch.equal(a, b)
    h = x.view(2, 70, 256)
    w = torch.ones(256, device=dev, dtype=BF)
    one, two = (h.detach().clone().requires_grad_() for _ in range(2))
    y, s = residual_norm(one, two, w)
    (y.sum() + (s * s.detach()).sum()).backward()
    assert torch.equal(one.grad, two.grad) and one.grad.data_ptr() != two.grad.data_ptr()
    both = h.detach().clone().requires_grad_()
    y, s = residual_norm(both, both, w)
    (y.sum() + (s * s.detach()).sum()).backward()
    y2, s2 = residual_norm(h, h, w)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    assert torch.equal(both.grad, one.grad + two.grad)


def _block(dev, seed):
    """What one block of a decoder does with the operators: a step that returns its outputs and every gradient."""
    r = _randn(dev, seed)
    B, S, A, KV, D, H = 2, 150, 4, 2, 64, 256
    p = dict(x=r(B, S, H), qkv=r(H, (A + 2 * KV) * D) / 16, out=r(A * D, H) / 16, n1=1 + 0.1 * r(H), n2=1 + 0.1 * r(H), post=1 + 0.1 * r(H),
             gate=r(B, 1, H))
    p = {n: t.to(BF).requires_grad_() for n, t in p.items()}
    f, amp = rotary_frequencies(D, scaling="ntk", factor=2.0, device=dev)
    lens = torch.tensor([S, 97], dtype=torch.int32, device=dev)
    dy, dr = r(B, S, H).to(BF), r(B, S, H).to(BF)

    def step():
        y = rms_norm(p["x"], p["n1"])
        q, k, v = (y.view(-1, H) @ p["qkv"]).view(B, S, A + 2 * KV, D).split([A, KV, KV], 2)
        q, k = rotary(q, k, f, amplitude=amp)
        o = attention(q, k, v, causal=True, kv_len=lens)
        outs = residual_norm(p["x"], (o.view(-1, A * D) @ p["out"]).view(B, S, H), p["n2"], gate=p["gate"], post_weight=p["post"], scale=0.5)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, list(p.values()), (dy, dr)))

    return step, p, (f, amp, lens, dy, dr)


def test_a_block_of_them_together(dev):
    """One block's outputs and gradients against the same block in 64 bits on the CPU, where each operator is its definition.
    Every tensor between two operators is rounded to bf16 (relative error of one rounding: 2^-9 in the mean square at most, and
    with it the error its gradient carries): 16 of them on the longest way forward and back, and two roundings inside each
    of five products; independent, so 2^-9 sqrt(26) = 1.0e-2 of a result's norm; twice that is allowed."""
    step, p, (f, amp, lens, dy, dr) = _block(dev, 21)
    got = step()
    B, S, A, KV, D, H = 2, 150, 4, 2, 64, 256
    w = {n: t.detach().cpu().double().requires_grad_() for n, t in p.items()}
    f, dy, dr = f.cpu(), dy.cpu().double(), dr.cpu().double()

    def normed(t, weight):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * weight

    y = normed(w["x"], w["n1"])
    q, k, v = (y @ w["qkv"]).view(B, S, A + 2 * KV, D).split([A, KV, KV], 2)
    angle = (torch.arange(S).double()[:, None] * f)[None, :, None, :]

    def turn(t):
        a, b = t.chunk(2, -1)
        return amp * torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)

    q, k = turn(q), turn(k).repeat_interleave(A // KV, 2)
    v = v.repeat_interleave(A // KV, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
    j = torch.arange(S)
    seen = (j[None, None, :] <= j[None, :, None]) & (j[None, None, :] < lens.cpu()[:, None, None])
    o = torch.einsum("bhij,bjhd->bihd", s.masked_fill(~seen[:, None], -float("inf")).softmax(-1), v).reshape(B, S, A * D)
    n = normed(o @ w["out"], w["post"]) * w["gate"]
    r = w["x"] + 0.5 * n
    outs = (normed(r, w["n2"]), r)
    want = [t.detach() for t in outs] + list(torch.autograd.grad(outs, list(w.values()), (dy, dr)))
    for name, a, b in zip(["y", "r"] + list(p), got, want):
        off = ((a.cpu().double() - b).norm() / b.norm()).item()
        assert off < 2 * 2 ** -9 * 26 ** 0.5, (name, off)


def test_captured_and_replayed(dev):
    """Two blocks captured into two graphs, replayed in turn with eager work between: every replay gives the eager bits."""
    blocks = [_block(dev, s) for s in (31, 32)]
    want = [b[0]() for b in blocks]
    graphs, outs = [], []
    for step, _, _ in blocks:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for rep in range(4):
        for i in (0, 1, 0) if rep % 2 else (1, 0):
            for t in outs[i]:
                t.fill_(7)
            graphs[i].replay()
            again = blocks[1 - i][0]()                                  # eager work right behind the replay
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want[i]):
                assert torch.equal(a, b)
            for a, b in zip(again, want[1 - i]):
                assert torch.equal(a, b)
    x = blocks[0][1]["x"]
    with torch.no_grad():
        x.mul_(0.5)                                                     # new values in the captured inputs
    new = blocks[0][0]()
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(outs[0], new):
        assert torch.equal(a, b)
    assert not torch.equal(new[0], want[0][0])


def test_two_streams_at_once(dev):
    blocks = [_block(dev, s) for s in (41, 42)]
    want = [b[0]() for b in blocks]
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for (step, _, _), st in zip(blocks, streams):
            with torch.cuda.stream(st):
                got.append(step())
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for a, b in zip(g, w):
                assert torch.equal(a, b)


def test_gpu_refusals(dev):
    q = torch.zeros(1, 4, 2, 64, device=dev)
    with pytest.raises(TypeError):
        attention(q, q, q)
    with pytest.raises(TypeError):
        attention(q.half(), q.half(), q.half())
    with pytest.raises(ValueError):
        attention(q.to(BF), q.to(BF).cpu(), q.to(BF))
    f, _ = rotary_frequencies(64)
    with pytest.raises(ValueError):
        rotary(q, q, f)                                                 # frequencies on another device
    with pytest.raises(ValueError):
        rotary(q, q, f.to(dev), torch.arange(4))
    with pytest.raises(TypeError):
        rotary(q.half(), None, f.to(dev))
    with pytest.raises(ValueError):
        rotary(q[:, :0], None, f.to(dev))
    x = torch.zeros(2, 8, device=dev)
    with pytest.raises(ValueError):
        residual_norm(x, x, torch.ones(8))
    with pytest.raises(TypeError):
        rms_norm(x.half(), torch.ones(8, device=dev))
    for make in (lambda t: attention(t, t, t), lambda t: rotary(t, None, f.to(dev))[0], lambda t: rms_norm(t, torch.ones(64, device=dev, dtype=BF))):
        leaf = torch.randn(1, 4, 2, 64, device=dev).to(BF).requires_grad_()
        g, = torch.autograd.grad(make(leaf).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), leaf)                          # not differentiable twice


@pytest.mark.parametrize("kw", [dict(positions="rotary"), dict(kv_heads=2), dict(positions="rotary", kv_heads=1, norm="pre_rms")])
def test_bert_options_match_the_plain_fp32_model(dev, kw):
    """The model's options on the GPU in bf16 against the same module on the CPU in fp32, a padded batch at a length that is no
    tile's multiple.  Bounds as for the published form of the model: 6e-2 of a gradient's norm at worst, 2.5e-2 in the mean."""
    import copy

    from distributed_tensorflow_amd.models import bert

    torch.manual_seed(0)
    ref = bert.build(layers=2, hidden=256, heads=4, intermediate=512, vocab=3000, seq_len=150, **kw).train()
    batch = list(bert.synthetic_batch(8, device="cpu", seed=2, seq_len=150, vocab=3000))
    batch[2][3, 100:] = 0
    fused = bert.prepare(copy.deepcopy(ref), dev).train()
    l_ref = bert.loss_fn(ref, tuple(batch))
    l_ref.backward()
    l_fused = bert.loss_fn(fused, tuple(t.to(dev) for t in batch))
    l_fused.backward()
    assert abs(l_fused.item() - l_ref.item()) / l_ref.item() < 1e-2
    worst = []
    for (n, p), (_, q) in zip(fused.named_parameters(), ref.named_parameters()):
        if q.grad.norm() > 1e-6:
            worst.append((((p.grad.float().cpu() - q.grad).norm() / q.grad.norm()).item(), n))
    worst.sort(reverse=True)
    assert worst[0][0] < 6e-2, worst[:5]
    assert sum(w for w, _ in worst) / len(worst) < 2.5e-2, worst[:5]


def test_bert_options_in_a_captured_step_equal_the_eager_loop(dev):
    """The training loop behind a job with these options, eager and with its step captured and replayed: the same parameters."""
    import copy

    from distributed_tensorflow_amd.models import get_model_module
    from distributed_tensorflow_amd.parallel.ps_runtime import ShardedPS
    from distributed_tensorflow_amd.train.trainer import train_loop

    mod = get_model_module("bert_base")
    torch.manual_seed(0)
    opts = dict(layers=2, hidden=256, heads=4, intermediate=512, vocab=2000, seq_len=150, positions="rotary", kv_heads=2, norm="pre_rms")
    m1 = mod.prepare(mod.build(**opts), dev).train()
    m2 = copy.deepcopy(m1)
    batch = mod.synthetic_batch(4, device=dev, seed=3, seq_len=150, vocab=2000)
    out = []
    for m, graph in ((m1, False), (m2, True)):
        ps = ShardedPS(list(m.named_parameters()), None, mod.default_optimizer())
        ps.set_lr(1e-3)
        last, _, n = train_loop(m, mod, ps, batch, 9, log_every=0, graph=graph)
        assert n == 9 and last == last
        out.append((ps.master.clone(), last))
        ps.remove_hooks()
    assert out[0][1] == out[1][1] and torch.equal(out[0][0], out[1][0])


def test_constants_made_under_inference_mode_train(dev):
    """Frequencies, positions and lengths that inference_mode made: a recorded call keeps copies of its own."""
    r = _randn(dev, 51)
    q, k, v, do = (r(2, 40, 2, 64).to(BF) for _ in range(4))
    with torch.inference_mode():
        f, _ = rotary_frequencies(64, device=dev)
        pos, lens = torch.arange(5, 45, device=dev), torch.tensor([40, 13], dtype=torch.int32, device=dev)
    res = []
    for how in ((f, pos, lens), (f.clone(), pos.clone(), lens.clone())):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        a, b = rotary(leaves[0], leaves[1], how[0], how[1])
        out = attention(a, b, leaves[2], kv_len=how[2])
        res.append((out.detach(),) + torch.autograd.grad(out, leaves, do))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_bert_with_rotary_positions_evaluated_first_then_trained(dev):
    import copy

    from distributed_tensorflow_amd.models import bert

    torch.manual_seed(0)
    m = bert.prepare(bert.build(layers=2, hidden=128, heads=2, intermediate=256, vocab=2000, seq_len=40, positions="rotary"), dev)
    fresh = copy.deepcopy(m)
    batch = bert.synthetic_batch(2, device=dev, seed=1, seq_len=40, vocab=2000)
    with torch.inference_mode():
        m.eval()(*batch[:4])
    for model in (m, fresh):
        bert.loss_fn(model.train(), batch).backward()
    for (n, p), (_, q) in zip(m.named_parameters(), fresh.named_parameters()):
        assert torch.equal(p.grad, q.grad), n
    # the model's first call of all inside a capture: nothing is copied from the host there
    first = bert.build(layers=1, hidden=128, heads=2, intermediate=256, vocab=2000, positions="rotary").to(dev).layers[0].positions
    r = _randn(dev, 52)
    q, k = r(2, 40, 2, 64).to(BF), r(2, 40, 2, 64).to(BF)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = first(q, k)
    want = rotary(q, k, rotary_frequencies(64, device=dev)[0])
    for _ in range(3):
        for t in out:
            t.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
