"""CPU side of the transformer-block operators: the plain forms against the 64-bit definitions, the definitions' gradients
against differences, and every refusal."""
import math

import pytest
import torch

import block_oracles as oracle
from distributed_tensorflow_amd.ops import attention as A
from distributed_tensorflow_amd.ops.residual_norm import FusedRMSNorm, residual_norm, rms_norm
from distributed_tensorflow_amd.ops.rotary import rotary, rotary_frequencies

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _g(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g)


def _differences(f, leaves, grads, weights, eps=1e-6, count=5):
    """Central differences of sum(weights * f()) in a few places of every leaf against ``grads``."""
    def total():
        return sum((w * o).sum().item() for w, o in zip(weights, f()))

    for name, leaf in leaves.items():
        flat, grad = leaf.view(-1), grads[name].reshape(-1)
        for at in range(0, flat.numel(), max(1, flat.numel() // count)):
            old = flat[at].item()
            flat[at] = old + eps
            up = total()
            flat[at] = old - eps
            down = total()
            flat[at] = old
            assert (up - down) / (2 * eps) == pytest.approx(grad[at].item(), rel=2e-5, abs=2e-6), (name, at)


@pytest.mark.parametrize("causal,lens,Sq,Sk", [(False, None, 5, 5), (True, None, 6, 6), (True, (0, 3), 5, 7), (True, None, 7, 3),
                                               (False, (2, 9), 1, 9)])
def test_attention_gradients(causal, lens, Sq, Sk):
    r = _g(1)
    t = {"q": r(2, Sq, 4, 8).double(), "k": r(2, Sk, 2, 8).double(), "v": r(2, Sk, 2, 8).double()}
    do = r(2, Sq, 4, 8).double()
    want, _ = oracle.attention(**t, do=do, causal=causal, lens=lens)
    _differences(lambda: [oracle.attention(**t, causal=causal, lens=lens)[0]["out"]], t, {n: want["d" + n] for n in t}, [do])
    leaves = [v.clone().requires_grad_() for v in t.values()]
    n = None if lens is None else torch.tensor(lens)
    out = A.attention(*leaves, causal=causal, kv_len=n)
    torch.testing.assert_close(out, want["out"], rtol=1e-12, atol=1e-12)
    for g, m in zip(torch.autograd.grad(out, leaves, do), t):
        torch.testing.assert_close(g, want["d" + m], rtol=1e-11, atol=1e-12)


def test_attention_on_the_cpu_rounds_once():
    r = _g(2)
    q, k, v = r(2, 9, 4, 64).to(BF), r(2, 9, 2, 64).to(BF), r(2, 9, 2, 64).to(BF)
    want, tol = oracle.attention(q, k, v, causal=True)
    oracle.close(A.attention(q, k, v, causal=True), want["out"], tol["out"], "out")
    few = torch.tensor([5, 200], dtype=torch.uint8)
    assert torch.equal(A.attention(q, k, v, kv_len=few), A.attention(q, k, v, kv_len=torch.tensor([5, 9])))
    poisoned = v.clone()
    poisoned[:, 5:] = float("nan")
    n = torch.tensor([5, 0])
    out = A.attention(q, k, poisoned, kv_len=n)
    assert torch.equal(out, A.attention(q, k, v, kv_len=n)) and not out[1].any()


def test_attention_refusals():
    q, k = torch.zeros(2, 4, 4, 64), torch.zeros(2, 6, 2, 64)
    bad = [
        (ValueError, dict(q=q[0])), (ValueError, dict(k=k.double())), (ValueError, dict(v=k[:, :5])), (ValueError, dict(k=k[:1], v=k[:1])),
        (ValueError, dict(q=torch.zeros(2, 4, 3, 64))), (ValueError, dict(q=q[..., :60], k=k[..., :60], v=k[..., :60])),
        (ValueError, dict(q=torch.zeros(2, 4, 4, 136), k=torch.zeros(2, 6, 2, 136), v=torch.zeros(2, 6, 2, 136))),
        (ValueError, dict(q=q[:, :0])), (ValueError, dict(k=k[:, :0], v=k[:, :0])), (ValueError, dict(kv_len=torch.tensor([1]))),
        (ValueError, dict(kv_len=torch.tensor([1.0, 2.0]))), (ValueError, dict(kv_len=torch.tensor([True, False]))),
        (TypeError, dict(scale=torch.tensor(1.0))), (ValueError, dict(scale=0.0)), (ValueError, dict(scale=-1.0)), (ValueError, dict(scale=math.inf)), (ValueError, dict(scale=math.nan)),
        (TypeError, dict(q=q.int(), k=k.int(), v=k.int())),
    ]
    for err, kw in bad:
        with pytest.raises(err):
            A.attention(**{**dict(q=q, k=k, v=k), **kw})


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", [BF, F32])
def test_rotary_on_the_cpu(interleaved, dt):
    r = _g(3)
    q, k = r(2, 11, 4, 20).to(dt), r(2, 11, 2, 20).to(dt)
    f, amp = rotary_frequencies(12, scaling="by_parts", factor=8.0, original_length=512)
    pos = torch.tensor([[100000], [3]]) + torch.arange(11)
    leaves = [q.clone().requires_grad_(), k.clone().requires_grad_()]
    outs = rotary(*leaves, f, pos, interleaved=interleaved, amplitude=amp)
    grads = torch.autograd.grad(outs, leaves, (q, k))
    for x, y, g in ((q, outs[0], grads[0]), (k, outs[1], grads[1])):
        for got, inv in ((y, False), (g, True)):
            want, tol = oracle.rotary(x, f, pos, interleaved, amp, inv)
            oracle.close(got.detach(), want, tol, "rotary")
    x = {"x": q.double()}
    w = r(2, 11, 4, 20).double()
    back, _ = oracle.rotary(w, f, pos, interleaved, amp, True)
    _differences(lambda: [oracle.rotary(x["x"], f, pos, interleaved, amp)[0]], x, {"x": back}, [w])


def test_rotary_frequencies():
    f, a = rotary_frequencies(8, base=100.0)
    torch.testing.assert_close(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=F64))
    assert a == 1.0 and torch.equal(rotary_frequencies(8, 100.0, "linear", 4.0)[0], f / 4)
    n, _ = rotary_frequencies(8, 100.0, "ntk", 4.0)
    assert n[0] == 1.0 and n[3].item() == pytest.approx(f[3].item() / 4)             # ends: kept, and stretched by the factor
    assert rotary_frequencies(2, 100.0, "ntk", 4.0)[0].tolist() == [1.0]
    b, a = rotary_frequencies(64, 10000.0, "by_parts", 8.0, original_length=4096)
    g, _ = rotary_frequencies(64)
    turns = 4096 * g / (2 * math.pi)
    assert torch.equal(b[turns >= 32], g[turns >= 32]) and torch.equal(b[turns <= 1], g[turns <= 1] / 8)
    assert a == pytest.approx(0.1 * math.log(8) + 1) and bool((b[:-1] >= b[1:]).all())
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, scaling="other"), dict(dim=8, factor=0.0), dict(dim=8, base=-1.0),
                dict(dim=8, scaling="by_parts"), dict(dim=8, scaling="by_parts", original_length=10, beta_fast=1.0, beta_slow=1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_rotary_refusals():
    q, k = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16)
    f, _ = rotary_frequencies(16)
    bad = [
        (ValueError, dict(q=q[0])), (ValueError, dict(k=k[:, :4])), (ValueError, dict(k=k.to(BF))), (ValueError, dict(q=q[..., :15], k=None)),
        (TypeError, dict(q=q.double(), k=k.double())), (ValueError, dict(inv_freq=f.float())), (ValueError, dict(inv_freq=f[:0])),
        (ValueError, dict(inv_freq=torch.ones(9, dtype=F64))), (ValueError, dict(inv_freq=f.view(2, 4))), (ValueError, dict(inv_freq=f.repeat(2)[::2])),
        (ValueError, dict(positions=torch.zeros(5))), (ValueError, dict(positions=torch.zeros(4, dtype=torch.int64))),
        (ValueError, dict(positions=torch.zeros(3, 5, dtype=torch.int64))), (TypeError, dict(amplitude=torch.ones(()))),
        (ValueError, dict(positions=torch.zeros(5, dtype=torch.int64), offset=3)), (ValueError, dict(offset=1 << 60)),
        (TypeError, dict(offset=0.5)), (ValueError, dict(inv_freq=f.clone().requires_grad_())),
    ]
    for err, kw in bad:
        with pytest.raises(err):
            rotary(**{**dict(q=q, k=k, inv_freq=f), **kw})


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, (10,), (2, 1, 10), (2, 3, 10)])
def test_residual_norm_gradients(kind, post, gate):
    r = _g(4)
    layer = kind == "layer"
    t = {"x": r(2, 3, 10) * 3, "h": r(2, 3, 10), "w": 1 + 0.2 * r(10)}
    if layer:
        t["b"] = r(10)
    if post:
        t["pw"] = 1 + 0.2 * r(10)
        if layer:
            t["pb"] = r(10)
    if gate:
        t["gate"] = r(*gate)
    dy, dr = r(2, 3, 10), r(2, 3, 10)
    want, tol = oracle.residual_norm(**t, scale=0.3, kind=kind, dy=dy, dr=dr)
    wide = {n: v.double() for n, v in t.items()}

    def forward():
        v, _ = oracle.residual_norm(**wide, scale=0.3, kind=kind)
        return [v["y"], v["r"]]

    _differences(forward, wide, {n: want["d" + n] for n in t}, [dy.double(), dr.double()])
    leaf = {n: v.clone().requires_grad_() for n, v in t.items()}
    outs = residual_norm(leaf["x"], leaf["h"], leaf["w"], leaf.get("b"), gate=leaf.get("gate"), scale=0.3, post_weight=leaf.get("pw"),
                         post_bias=leaf.get("pb"), kind=kind)
    oracle.close(outs[0].detach(), want["y"], tol["y"], "y")
    oracle.close(outs[1].detach(), want["r"], tol["r"], "r")
    for n, g in zip(leaf, torch.autograd.grad(outs, list(leaf.values()), (dy, dr))):
        oracle.close(g, want["d" + n], tol["d" + n], "d" + n)


def test_rms_norm_on_the_cpu():
    r = _g(5)
    x, w = r(3, 4, 24).to(BF), 1 + 0.1 * r(24)
    want, tol = oracle.residual_norm(x, torch.zeros_like(x), w, eps=1e-5)
    oracle.close(rms_norm(x, w, 1e-5), want["y"], tol["y"], "y")
    m = FusedRMSNorm(24)
    y, s = m(x, x, scale=2.0)
    assert torch.equal(s, (x.float() + 2 * x.float()).to(BF)) and y.dtype == BF and m(x).shape == x.shape


def test_residual_norm_refusals():
    x, w = torch.zeros(2, 3, 10), torch.ones(10)
    bad = [
        (ValueError, dict(kind="batch")), (ValueError, dict(h=None)), (ValueError, dict(h=x[:1])), (ValueError, dict(h=x.to(BF))),
        (TypeError, dict(x=x.double(), h=x.double())), (ValueError, dict(x=x[:0], h=x[:0])), (ValueError, dict(weight=w[:9])),
        (ValueError, dict(weight=w.to(BF))), (ValueError, dict(bias=w)), (ValueError, dict(kind="layer", bias=w.to(BF))),
        (ValueError, dict(kind="layer", post_bias=w)), (ValueError, dict(gate=w[:9])), (ValueError, dict(gate=w.to(BF))),
        (ValueError, dict(gate=torch.ones(1, 3, 10))), (ValueError, dict(gate=torch.ones(2, 3, 1))), (ValueError, dict(gate=torch.ones(1, 2, 3, 10))),
        (TypeError, dict(scale=torch.ones(()))), (ValueError, dict(x=torch.zeros(1, 16385), h=torch.zeros(1, 16385), weight=torch.ones(16385))),
        (TypeError, dict(eps=torch.ones(()))), (ValueError, dict(eps=-1e-6)), (ValueError, dict(eps=math.nan)), (ValueError, dict(eps=math.inf)),
    ]
    for err, kw in bad:
        with pytest.raises(err):
            residual_norm(**{**dict(x=x, h=x, weight=w), **kw})


# ---------------------------------------------------------------------------------------------------------------------
# the model that calls them
# ---------------------------------------------------------------------------------------------------------------------
BERT = dict(layers=2, hidden=64, heads=4, intermediate=64, vocab=2000, seq_len=21)


def _bert(**kw):
    from distributed_tensorflow_amd.models import bert

    torch.manual_seed(0)
    m = bert.build(**BERT, **kw)
    batch = list(bert.synthetic_batch(3, seed=1, seq_len=21, vocab=2000))
    batch[2][1, 13:] = 0                                               # the second sequence is padded
    return bert, m, tuple(batch)


@pytest.mark.parametrize("kw", [dict(positions="rotary"), dict(kv_heads=2), dict(norm="pre_rms"),
                                dict(positions="rotary", kv_heads=1, norm="pre_rms", rotary_scaling="by_parts", rotary_factor=4)])
def test_bert_options_train(kw):
    bert, m, batch = _bert(**kw)
    loss = bert.loss_fn(m, batch)
    loss.backward()
    assert bool(torch.isfinite(loss))
    for n, p in m.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n
    assert ("position_embeddings.weight" in dict(m.named_parameters())) == (kw.get("positions") != "rotary")
    names = bert.tf_variable_names(m)
    flat = [v if isinstance(v, str) else [x[0] for x in v] for v in names.values()]
    flat = [x for v in flat for x in ([v] if isinstance(v, str) else v)]
    assert len(set(flat)) == len(flat) and set(names) == {n for n, _ in m.named_parameters()}
    rows = names["layers.0.qkv.weight"]
    assert [b - a for _, a, b in rows] == [64, 16 * (kw.get("kv_heads") or 4), 16 * (kw.get("kv_heads") or 4)]
    assert rows[-1][2] == m.layers[0].qkv.weight.shape[0]
    # padding takes no part: other tokens there, the same loss
    other = list(batch)
    other[0] = batch[0].clone()
    masked = {int(p) for p in batch[3][1]}
    for at in range(13, 21):
        if at not in masked:
            other[0][1, at] = 1500
    keep = torch.tensor([p < 13 for p in batch[3][1].tolist()])
    a, _ = m(*batch[:4])
    b, _ = m(*other[:4])
    n = batch[3].shape[1]
    torch.testing.assert_close(a[n:2 * n][keep], b[n:2 * n][keep], rtol=1e-5, atol=1e-6)


def test_bert_fewer_key_heads_equal_repeated_ones():
    """kv_heads=2 of 4 is the full-head model whose key and value heads come in equal pairs; the gradient of a shared head is
    the sum of its copies'."""
    import copy

    bert, m, batch = _bert(kv_heads=2)
    _, full, _ = _bert()
    wide = copy.deepcopy(m)
    for layer, src in zip(full.layers, m.layers):
        for n in ("weight", "bias"):
            q, k, v = getattr(src.qkv, n).detach().split([64, 32, 32])
            k, v = (t.view(2, 16, -1).repeat_interleave(2, 0).reshape(64, -1) if n == "weight" else
                    t.view(2, 16).repeat_interleave(2, 0).reshape(64) for t in (k, v))
            getattr(layer.qkv, n).data.copy_(torch.cat([q, k, v]))
    rest = {n: p for n, p in wide.named_parameters() if ".qkv." not in n}
    with torch.no_grad():
        for n, p in full.named_parameters():
            if n in rest:
                p.copy_(rest[n])
    a, b = bert.loss_fn(m, batch), bert.loss_fn(full, batch)
    torch.testing.assert_close(a, b, rtol=2e-6, atol=2e-6)
    a.backward()
    b.backward()
    for s, f in zip(m.layers, full.layers):
        gs, gf = s.qkv.weight.grad, f.qkv.weight.grad
        torch.testing.assert_close(gs[:64], gf[:64], rtol=1e-4, atol=1e-6)
        torch.testing.assert_close(gs[64:96].view(2, 16, 64), gf[64:128].view(2, 2, 16, 64).sum(1), rtol=1e-4, atol=1e-6)
        torch.testing.assert_close(gs[96:].view(2, 16, 64), gf[128:].view(2, 2, 16, 64).sum(1), rtol=1e-4, atol=1e-6)


def test_bert_option_refusals():
    from distributed_tensorflow_amd.models import bert

    for kw in (dict(kv_heads=3), dict(positions="sine"), dict(norm="none"), dict(positions="rotary", rotary_scaling="x"), dict(hidden=50),
               dict(hidden=48, kv_heads=2), dict(hidden=1024, norm="pre_rms")):
        with pytest.raises(ValueError):
            bert.build(**{**BERT, **kw})


@pytest.mark.parametrize("kv_heads", [-1, -2, -4])
def test_bert_refuses_negative_key_heads(kv_heads):
    from distributed_tensorflow_amd.models import bert

    with pytest.raises(ValueError, match="kv_heads"):
        bert.build(**{**BERT, "kv_heads": kv_heads})


def test_rotary_positions_belong_to_the_model_not_to_its_first_call(monkeypatch):
    """A model evaluated under inference_mode first trains afterwards: its frequencies are made where it is built or moved, never
    inside a call.  (Only the GPU's backward saves them, so what the operator is handed is looked at.)"""
    bert, m, batch = _bert(positions="rotary")
    seen = []
    plain = bert.rotary

    def spy(q, k, inv_freq, **kw):
        seen.append(inv_freq)
        return plain(q, k, inv_freq, **kw)

    monkeypatch.setattr(bert, "rotary", spy)
    with torch.inference_mode():
        m(*batch[:4])
    bert.loss_fn(m, batch).backward()
    assert len(seen) == 4 and not any(f.is_inference() for f in seen) and all(f is seen[0] for f in seen)
    assert seen[0].dtype == F64 and torch.equal(seen[0], rotary_frequencies(16)[0])
    turn = m.layers[0].positions
    before = set(m.state_dict())
    m.to(torch.bfloat16)
    assert turn._table(torch.device("cpu")) is seen[0] and seen[0].dtype == F64           # the model's dtype leaves them alone
    assert set(m.state_dict()) == before and not any("positions" in n for n in before)
    m.to("meta").to_empty(device="cpu")
    assert torch.equal(turn._table(torch.device("cpu")), rotary_frequencies(16)[0])


def test_rotary_positions_refuse_a_capture_on_a_device_they_were_not_moved_to(monkeypatch):
    _, m, _ = _bert(positions="rotary")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="move the model"):
        m.layers[0].positions._table(torch.device("cuda", 0))


def test_constants_of_a_recorded_call_can_be_saved():
    from distributed_tensorflow_amd.ops import hip

    with torch.inference_mode():
        a = torch.arange(3)
    b = torch.arange(3)
    assert hip.savable(b) is b and hip.savable(None) is None
    assert not hip.savable(a).is_inference() and torch.equal(hip.savable(a), b)


NOISE = [(2, 16, 16, 4, 2, 64, True, None), (1, 64, 64, 2, 2, 128, True, None), (2, 129, 129, 2, 1, 64, True, (129, 70)),
         (1, 31, 700, 4, 2, 128, True, None), (2, 60, 320, 2, 1, 64, False, (320, 111))]


@pytest.mark.parametrize("B,Sq,Sk,Hq,Hk,D,causal,lens", NOISE)
def test_attention_noise_tells_the_documented_roundings_from_others(B, Sq, Sk, Hq, Hk, D, causal, lens):
    """The norms that the kernels' errors are held to: the documented roundings stay under them; a D or scores in bf16, where such
    roundings are not lost among the others, and a key left out do not."""
    r = _g(Sq + Sk)
    q, k, v, do = (t.to(BF) for t in (r(B, Sq, Hq, D), r(B, Sk, Hk, D), r(B, Sk, Hk, D), r(B, Sq, Hq, D)))
    want, most = oracle.attention_noise(q, k, v, do, causal, lens)
    plain, _ = oracle.attention(q, k, v, do, causal, lens)
    for n in want:
        torch.testing.assert_close(want[n], plain[n], rtol=1e-12, atol=1e-12)

    def over(**kw):
        got = oracle.attention_rounded(q, k, v, do, causal, lens, **kw)
        return {n: (got[n] - want[n]).norm().item() / most[n] for n in want}

    right = over()
    assert max(right.values()) < 1, right
    lost = over(lost_key=Sk // 3)
    assert min(lost.values()) > 3, lost
    if Sk <= 64:                                       # few keys: dS is a difference of like terms
        d = over(rounded_d=True)
        assert min(d["dq"], d["dk"]) > 1, d
    if Sk > 128:
        scores = over(rounded_s=True)
        assert min(scores.values()) > 1, scores
