"""BERT-base pre-training (config #4: PS-sharded Adam, bf16, sequence length 512).

L=12, H=768, A=12, intermediate 3072, vocab 30522, masked-LM + next-sentence heads; ~110 M
parameters whose Adam state (fp32 master + m + v) is sharded over the PS ranks and updated
by the K2 fused Adam shard-apply kernel.  Linear layers are :class:`FusedLinear` (K6 MFMA
GEMM with the bias / GELU / residual epilogue fused, K6T weight gradients), LayerNorm is K10 and
attention is K11 (``ops/attention.py``; PyTorch SDPA when a mask or dropout is requested).

Variables are named like google-research/bert checkpoints: ``bert/embeddings/word_embeddings``,
``bert/encoder/layer_0/attention/self/query/kernel``, ``cls/predictions/transform/dense/kernel``
(TF stores kernels ``[in, out]``; the flat shard bytes here are torch's ``[out, in]``, recorded
as such in the checkpoint index).

Job options beside the published model: ``positions=rotary`` (K23 on queries and keys instead of the learned table, so the
sequence length has no bound; ``rotary_scaling``, ``rotary_factor``, ``rotary_original`` stretch it), ``kv_heads=N`` (fewer key and value heads)
and ``norm=pre_rms`` (RMS norms in front of attention and MLP, every block boundary one K24 pass).  With any of them attention
is K22, which has no limit on length and takes bf16 on the GPU (as :func:`prepare` makes the model there; fp32 on the CPU).
"""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import attention
from ..ops.layernorm import FusedLayerNorm
from ..ops.cross_entropy import cross_entropy
from ..ops.embedding import dense_embedding
from ..ops.linear import FusedLinear, linear_residual_layernorm
from ..ops.residual_norm import FusedRMSNorm
from ..ops.rotary import rotary, rotary_frequencies


class _SplitQKV(torch.autograd.Function):
    """Packed projection output ``[B, S, 3, A, D]`` -> q, k, v views ``[B, A, S, D]`` for the attention
    kernel.  Backward gathers dq, dk, dv straight into the packed layout with one copy kernel; plain
    autograd stacks them as ``[3, B, A, S, D]`` and the next op then re-copies that into token-major
    order (two passes over the 3H-wide tensor per layer: 276 us at batch 64)."""

    @staticmethod
    def forward(ctx, qkv):
        q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)
        return q, k, v

    @staticmethod
    def backward(ctx, dq, dk, dv):
        return torch.stack([dq.transpose(1, 2), dk.transpose(1, 2), dv.transpose(1, 2)], dim=2)


class RotaryPositions(nn.Module):
    """The frequencies of ``positions=rotary``, on every device that the model has been moved to.  They are in 64 bits and the
    model's buffers follow its dtype, so they are no buffer: a table is made, once per device, where the model is built or moved
    -- not by the call that first needs it, which may run under ``inference_mode`` (no training step could save the table) or
    inside a graph capture (a copy from the host must not)."""

    def __init__(self, dim, base, scaling, factor, original_length):
        super().__init__()
        self.spec = dict(dim=dim, base=base, scaling=scaling, factor=factor, original_length=original_length)
        _, self.amplitude = rotary_frequencies(**self.spec)               # checks the options where the model is built
        self._on, self._at = {}, torch.device("cpu")
        self._table(self._at)

    def _table(self, device):
        if device not in self._on:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("rotary positions: no frequencies on %s yet; move the model there before capturing its step" % device)
            with torch.inference_mode(False):
                self._on[device] = rotary_frequencies(**self.spec, device=device)[0]
        return self._on[device]

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self._at = fn(torch.empty(0, device=self._at)).device             # (what is moved has no tensor of its own to tell where)
        if self._at.type != "meta":
            self._table(self._at)
        return self

    def forward(self, q, k):
        return rotary(q, k, self._table(q.device), amplitude=self.amplitude)


def _general_attention(qkv, A, KV, kv_len, positions):
    """Context ``[B, S, H]`` of a packed projection ``[B, S, (A + 2 KV) D]`` through K22 (and K23)."""
    B, S, W = qkv.shape
    q, k, v = qkv.view(B, S, A + 2 * KV, W // (A + 2 * KV)).split([A, KV, KV], dim=2)
    if positions is not None:
        q, k = positions(q, k)
    return attention.attention(q, k, v, kv_len=kv_len).flatten(2)


class PreNormLayer(nn.Module):
    """``norm=pre_rms``: takes the residual stream and the output of the block before, returns the stream and its own output
    -- the addition, and the norm behind it, are the next block's first pass."""

    def __init__(self, H, A, I, act, KV, positions):
        super().__init__()
        self.A, self.KV, self.positions = A, KV, positions
        self.attn_in_ln = FusedRMSNorm(H, eps=1e-6)
        self.qkv = FusedLinear(H, (A + 2 * KV) * (H // A))
        self.attn_out = FusedLinear(H, H)
        self.mlp_in_ln = FusedRMSNorm(H, eps=1e-6)
        self.inter = FusedLinear(H, I, act=act)
        self.out = FusedLinear(I, H)

    def forward(self, x, h, kv_len):
        if h is None:
            y = self.attn_in_ln(x)
        else:
            y, x = self.attn_in_ln(x, h)
        y, x = self.mlp_in_ln(x, self.attn_out(_general_attention(self.qkv(y), self.A, self.KV, kv_len, self.positions)))
        return x, self.out(self.inter(y))


class Layer(nn.Module):
    def __init__(self, H, A, I, p, act="gelu_tanh", KV=None, positions=None):
        super().__init__()
        self.A = A
        self.KV, self.positions = KV or A, positions
        self.qkv = FusedLinear(H, (A + 2 * self.KV) * (H // A))
        self.attn_out = FusedLinear(H, H)
        self.attn_ln = FusedLayerNorm(H, eps=1e-12)
        self.inter = FusedLinear(H, I, act=act)
        self.out = FusedLinear(I, H)
        self.out_ln = FusedLayerNorm(H, eps=1e-12)
        self.p = p

    def forward(self, x, mask, kv_len=None):
        B, S, H = x.shape
        # x feeds the projection and the residual: the fork sums both gradients inside the dX GEMM
        qkv, x = self.qkv.forward_fork(x, own_skip_grad=True)
        drop = self.p if self.training else 0.0
        general = self.positions is not None or self.KV != self.A
        qkv5 = None if general else qkv.view(B, S, 3, self.A, H // self.A)
        if general:
            if drop:
                raise ValueError("rotary positions and kv_heads are without attention dropout")
            ctx = _general_attention(qkv, self.A, self.KV, kv_len, self.positions)
        elif drop == 0.0 and attention.kernel_eligible(qkv5):
            # K11: consumes the packed projection in place, writes the context token-major, and its backward
            # writes dQ / dK / dV straight into the packed gradient -- no transposes or copies either way.
            # The padding mask is a prefix mask: handed over as one length per sequence.
            ctx = attention.attention_packed(qkv5, kv_len)
        else:
            q, k, v = _SplitQKV.apply(qkv5)
            ctx = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, dropout_p=drop)
            ctx = ctx.transpose(1, 2).reshape(B, S, H)
        x = linear_residual_layernorm(ctx, self.attn_out, x, self.attn_ln)      # residual in the GEMM (beta = 1), bias in K10
        h, x = self.inter.forward_fork(x, own_skip_grad=True)
        return linear_residual_layernorm(h, self.out, x, self.out_ln)


class Bert(nn.Module):
    def __init__(self, vocab=30522, hidden=768, layers=12, heads=12, intermediate=3072, max_pos=512,
                 type_vocab=2, dropout=0.0, act="gelu_tanh", kv_heads=0, positions="learned", norm="post_ln", rotary_base=10000.0,
                 rotary_scaling="none", rotary_factor=1.0, rotary_original=512):
        super().__init__()
        kv_heads = kv_heads or heads
        if kv_heads < 0 or hidden % heads or heads % kv_heads:
            raise ValueError("hidden %d must divide over %d heads, and these over %d kv_heads" % (hidden, heads, kv_heads))
        if positions not in ("learned", "rotary") or norm not in ("post_ln", "pre_rms"):
            raise ValueError("positions is learned or rotary, norm post_ln or pre_rms; got %r, %r" % (positions, norm))
        if norm == "pre_rms" and dropout:
            raise ValueError("norm=pre_rms is without dropout")
        if (positions == "rotary" or norm == "pre_rms" or kv_heads != heads) and (hidden // heads % 8 or hidden // heads > 128):
            raise ValueError("these options need head sizes that are multiples of 8 to 128, got %d" % (hidden // heads))
        turn = None
        if positions == "rotary":
            turn = RotaryPositions(hidden // heads, rotary_base, rotary_scaling, rotary_factor, rotary_original)
        self.hidden, self.vocab, self.kv_width = hidden, vocab, kv_heads * (hidden // heads)
        self.word_embeddings = nn.Embedding(vocab, hidden)
        if turn is None:
            self.position_embeddings = nn.Embedding(max_pos, hidden)
        self.token_type_embeddings = nn.Embedding(type_vocab, hidden)
        self.emb_ln = FusedLayerNorm(hidden, eps=1e-12)
        # act: "gelu_tanh" is the google-research/bert definition (tanh form); "gelu" the erf form
        self.pre_norm = norm == "pre_rms"
        if self.pre_norm:
            self.layers = nn.ModuleList(PreNormLayer(hidden, heads, intermediate, act, kv_heads, turn) for _ in range(layers))
            self.final_ln = FusedRMSNorm(hidden, eps=1e-6)
        else:
            self.layers = nn.ModuleList(Layer(hidden, heads, intermediate, dropout, act, kv_heads, turn) for _ in range(layers))
        self.learned_positions = turn is None
        self.pooler = FusedLinear(hidden, hidden)
        self.mlm_transform = FusedLinear(hidden, hidden, act=act)
        self.mlm_ln = FusedLayerNorm(hidden, eps=1e-12)
        self.mlm_bias = nn.Parameter(torch.zeros(vocab))
        self.nsp = nn.Linear(hidden, 2)
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.trunc_normal_(m.weight, std=0.02, a=-0.04, b=0.04)
            if isinstance(m, nn.Linear) and m.bias is not None:
                nn.init.zeros_(m.bias)

    def forward(self, input_ids, token_type_ids, attention_mask, masked_positions):
        B, S = input_ids.shape
        x = dense_embedding(input_ids, self.word_embeddings.weight)
        if self.learned_positions:
            x = x + self.position_embeddings(torch.arange(S, device=input_ids.device)).unsqueeze(0)
        x = x + dense_embedding(token_type_ids, self.token_type_embeddings.weight)
        x = self.emb_ln(x)
        mask = kv_len = None
        if attention_mask is not None:
            # BERT's input mask marks real tokens with 1 and trailing padding with 0 (a prefix mask)
            mask = attention_mask[:, None, None, :].to(torch.bool)
            kv_len = attention_mask.sum(-1, dtype=torch.int32)
        if self.pre_norm:
            h = None
            for layer in self.layers:
                x, h = layer(x, h, kv_len)
            x, _ = self.final_ln(x, h)
        else:
            for layer in self.layers:
                x = layer(x, mask, kv_len)
        pooled = torch.tanh(self.pooler(x[:, 0]))
        # masked-LM head on the masked positions only (max_predictions_per_seq)
        idx = masked_positions.unsqueeze(-1).expand(-1, -1, self.hidden)
        h = torch.gather(x, 1, idx).reshape(-1, self.hidden)
        h = self.mlm_ln(self.mlm_transform(h))
        mlm_logits = F.linear(h, self.word_embeddings.weight, self.mlm_bias)      # tied decoder
        return mlm_logits, self.nsp(pooled)


def build(layers=12, hidden=768, heads=12, intermediate=3072, vocab=30522, seq_len=512, act="gelu_tanh", kv_heads=0,
          positions="learned", norm="post_ln", rotary_base=10000.0, rotary_scaling="none", rotary_factor=1.0,
          rotary_original=512, **_):
    return Bert(int(vocab), int(hidden), int(layers), int(heads), int(intermediate), max(512, int(seq_len)), act=act,
                kv_heads=int(kv_heads), positions=positions, norm=norm, rotary_base=float(rotary_base), rotary_scaling=rotary_scaling,
                rotary_factor=float(rotary_factor), rotary_original=int(rotary_original))


def prepare(model, device):
    device = torch.device(device)
    if device.type == "cuda":
        return model.to(device=device, dtype=torch.bfloat16)
    return model.to(device)


def tf_variable_names(model):
    """torch name -> TF name, or -> ``[(TF name, row0, row1), ...]`` for the packed QKV projection, which the
    checkpoint index lists as google-research/bert's three variables ``attention/self/{query,key,value}/{kernel,bias}``
    (row ranges of the same shard bytes: output rows are ordered q, k, v)."""
    out = {}
    ln = {"weight": "gamma", "bias": "beta"}
    kb = {"weight": "kernel", "bias": "bias"}
    H, KV = model.hidden, model.kv_width
    rms = {"attn_in_ln": "attention/input/RMSNorm/gamma", "mlp_in_ln": "intermediate/input/RMSNorm/gamma"}
    for n, _ in model.named_parameters():
        p = n.split(".")
        if p[0] == "layers" and p[2] == "qkv":
            base = "bert/encoder/layer_%s/attention/self/" % p[1]
            out[n] = [(base + "%s/%s" % (part, kb[p[3]]), a, b)
                      for part, a, b in (("query", 0, H), ("key", H, H + KV), ("value", H + KV, H + 2 * KV))]
            continue
        if p[0] == "final_ln":
            tf = "bert/encoder/output/RMSNorm/gamma"
        elif p[0] == "layers" and p[2] in rms:
            tf = "bert/encoder/layer_%s/" % p[1] + rms[p[2]]
        elif p[0] in ("word_embeddings", "position_embeddings", "token_type_embeddings"):
            tf = "bert/embeddings/" + p[0]
        elif p[0] == "emb_ln":
            tf = "bert/embeddings/LayerNorm/" + ln[p[1]]
        elif p[0] == "layers":
            base = "bert/encoder/layer_%s/" % p[1]
            sub = {"attn_out": "attention/output/dense/",
                   "attn_ln": "attention/output/LayerNorm/", "inter": "intermediate/dense/",
                   "out": "output/dense/", "out_ln": "output/LayerNorm/"}[p[2]]
            tf = base + sub + (ln[p[3]] if p[2].endswith("ln") else kb[p[3]])
        elif p[0] == "pooler":
            tf = "bert/pooler/dense/" + kb[p[1]]
        elif p[0] == "mlm_transform":
            tf = "cls/predictions/transform/dense/" + kb[p[1]]
        elif p[0] == "mlm_ln":
            tf = "cls/predictions/transform/LayerNorm/" + ln[p[1]]
        elif p[0] == "mlm_bias":
            tf = "cls/predictions/output_bias"
        elif p[0] == "nsp":
            tf = "cls/seq_relationship/" + ("output_weights" if p[1] == "weight" else "output_bias")
        else:
            tf = n
        out[n] = tf
    return out


def synthetic_batch(batch, device="cpu", seed=None, seq_len=512, vocab=30522, max_predictions=76, **_):
    g = torch.Generator().manual_seed(seed) if seed is not None else None
    seq_len = int(seq_len)
    ids = torch.randint(1000, vocab, (batch, seq_len), generator=g)
    types = (torch.arange(seq_len).unsqueeze(0) >= seq_len // 2).long().expand(batch, -1).contiguous()
    mask = torch.ones(batch, seq_len, dtype=torch.long)
    npred = min(max_predictions, max(1, int(seq_len * 0.15)))
    pos = torch.stack([torch.randperm(seq_len, generator=g)[:npred] for _ in range(batch)])
    labels = torch.gather(ids, 1, pos)
    ids = ids.scatter(1, pos, 103)          # [MASK]
    nsp = torch.randint(0, 2, (batch,), generator=g)
    return tuple(t.to(device) for t in (ids, types, mask, pos, labels, nsp))


def loss_fn(model, batch):
    ids, types, mask, pos, labels, nsp = batch
    # "no padding" is decided once per mask tensor: the check reads a device value (a host sync), which per
    # step would drain the launch queue
    full = getattr(mask, "_dtf_all_ones", None)
    if full is None:
        full = bool((mask == 1).all())
        mask._dtf_all_ones = full
    mlm_logits, nsp_logits = model(ids, types, None if full else mask, pos)
    # K12: the [B*76, 30522] MLM logits stay bf16 in memory, softmax arithmetic in fp32 registers
    return cross_entropy(mlm_logits, labels.reshape(-1)) + F.cross_entropy(nsp_logits.float(), nsp)


def default_optimizer():
    from ..parallel.ps_runtime import OptimizerSpec

    # BERT's AdamWeightDecayOptimizer: decoupled decay 0.01, no bias correction, and its exclusion list
    # ("LayerNorm", "layer_norm", "bias"): those variables form their own bucket group applied with decay 0
    return OptimizerSpec(kind="adam", lr=1e-4, beta1=0.9, beta2=0.999, eps=1e-6, weight_decay=0.01, adamw=True,
                         bias_correction=False, max_grad_norm=1.0, no_decay=("_ln.", ".bias", "mlm_bias"))
