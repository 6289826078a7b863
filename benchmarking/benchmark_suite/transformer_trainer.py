"""Language-model clients: `bert_loop` (BERT-base question answering, reference
benchmarking/benchmark_suite/bert_trainer_mock.py:49-234) and `transformer_loop` (language-model
training, reference benchmarking/benchmark_suite/transformer_trainer.py:43-200), with the
reference's argument lists.  The request loop is `run_client` of train_imagenet.py.

Models are defined here (the reference imports NVIDIA's example repositories, which are not part
of it): BERT-base = 12 layers, hidden 768, 12 heads, FFN 3072, vocabulary 30522 padded to 30528,
sequence 384; the training "transformer" client is the benchmark configuration's decoder-only LM
(16 layers, d_model 1024, 16 heads, FFN 4096, vocabulary 32000, sequence 512) — the reference's
Transformer-XL is not reproduced.  Everything is bfloat16 with synthetic token ids.

Inference runs on the orion kernels (tcgen05 GEMM and fused attention, LayerNorm, softmax, GELU), and so does
training (ORION_PREPARE=1, the default): linear layers and attention with all their gradient products on the
bfloat16 GEMM, LayerNorm / GELU / softmax / embedding / cross-entropy forward and backward, one-launch AdamW.
ORION_FUSED_LINEAR=1 runs every linear layer with what follows it (bias, GELU, dropout, residual) as one launch, ORION_FUSED_LOSS=1
computes the decoder's loss from the hidden states, without logits, and ORION_DROPOUT=p trains with dropout of the embeddings and
of both residual branches, as the reference's clients do (reference benchmarking/model_kernels/bert_8_fb1, dropout rows); the
masks are drawn from counters and never stored; ORION_DROPOUT_SEED names their seed.  All three are off by default: recorded profiles
have a row per launch.
With ORION_PREPARE=0 training uses stock PyTorch modules, whose cuBLASLt / flash-attention / elementwise
launches are captured and scheduled like any other op.
"""
import math
import os

import torch
import torch.nn as nn
import torch.nn.functional as F

from .train_imagenet import run_client

# Training clients use the orion LayerNorm / GELU / cross-entropy / AdamW kernels unless ORION_PREPARE=0 or the overrides are off.
ORION_TRAIN_KERNELS = os.environ.get("ORION_PREPARE", "1") == "1" and os.environ.get("ORION_DISABLE_OVERRIDES", "0") != "1"

FUSED_ATTENTION = os.environ.get("ORION_FUSED_ATTENTION", "1") == "1"
# ORION_OWN_GEMM_TRAINING=0 leaves the GEMMs, the attention and the embeddings of the training clients on the stock kernels
OWN_GEMM_TRAINING = os.environ.get("ORION_OWN_GEMM_TRAINING", "1") == "1"

# linear layers of the text clients with their bias, GELU, dropout and residual in one launch; loss of the decoder without its logits
FUSED_LINEAR = os.environ.get("ORION_FUSED_LINEAR", "0") == "1"
FUSED_LOSS = os.environ.get("ORION_FUSED_LOSS", "0") == "1"
# dropout probability of the training clients (embeddings and both residual branches), and the seed of a run's masks (default: torch's)
DROPOUT = float(os.environ.get("ORION_DROPOUT", "0"))
DROPOUT_SEED = os.environ.get("ORION_DROPOUT_SEED")

BERT = dict(layers=12, hidden=768, heads=12, ffn=3072, vocab=30528, max_pos=512, seq=384)
LM = dict(layers=16, hidden=1024, heads=16, ffn=4096, vocab=32000, seq=512)


def _f32(module, p):
    """float32 copy of a parameter for the kernels that take their bias / scale in float32, made once per parameter version
    (an inference model never changes it) instead of one cast kernel per use."""
    cache = module.__dict__.setdefault("_f32_cache", {})
    hit = cache.get(id(p))
    if hit is None or hit[0] != p._version or hit[2] != p.data_ptr():
        hit = (p._version, p.detach().float(), p.data_ptr())
        cache[id(p)] = hit
    return hit[1]


def _fit_checkpoint(model, state, prefix, *_):
    """A checkpoint of a model built without dropout has no `rng`, and such a model takes none."""
    if "rng" in model._non_persistent_buffers_set:
        state.pop(prefix + "rng", None)
    else:
        state.setdefault(prefix + "rng", model.rng)


def _dropout_state(module, cfg):
    """`rng`, the seed and the step of the model's dropout masks.  The seed is cfg["dropout_seed"], or drawn from torch's generator, so that
    masks follow torch.manual_seed and no two models share theirs."""
    p, seed = cfg.get("dropout", 0.0), cfg.get("dropout_seed")
    if seed is None:
        seed = int(torch.randint(2 ** 62, ())) if p > 0.0 else 0   # without dropout nothing is drawn
    module.register_buffer("rng", torch.tensor([seed, 0]), persistent=p > 0.0)   # a checkpoint goes on with the step that it stopped at
    module.register_load_state_dict_pre_hook(_fit_checkpoint)


def _client_seed(tid, local_rank):
    """A client's own masks: the run's seed with the process's rank and the client's number in it."""
    base = int(DROPOUT_SEED) if DROPOUT_SEED else torch.initial_seed()
    return (base + (int(os.environ.get("RANK", local_rank)) << 40) + (tid << 52)) % 2 ** 62


def _count_step(rng):
    """(seed, step) of this forward pass, a copy that its backward pass can go by while the model counts on."""
    rng[1:] += 1
    return rng.clone()


class BertLayer(nn.Module):
    def __init__(self, h, heads, ffn, dropout=0.0, site=0):
        super().__init__()
        self.heads = heads
        self.dropout, self.site = dropout, site   # probability; number of the layer's first dropout in the model
        self.qkv = nn.Linear(h, 3 * h)
        self.out = nn.Linear(h, h)
        self.ln1 = nn.LayerNorm(h, eps=1e-12)
        self.fc1 = nn.Linear(h, ffn)
        self.fc2 = nn.Linear(ffn, h)
        self.ln2 = nn.LayerNorm(h, eps=1e-12)

    def forward(self, x, causal=False, rng=None):
        b, s, h = x.shape
        p = self.dropout if self.training else 0.0
        if ORION_TRAIN_KERNELS and OWN_GEMM_TRAINING and x.is_cuda and self.training and x.dtype == torch.bfloat16 and (FUSED_LINEAR or p > 0.0):
            # the same with bias, GELU, dropout and residual behind the products, not beside them
            ops = torch.ops.orion
            ctx = ops.attention_train(ops.linear_act(x, self.qkv.weight, self.qkv.bias), self.heads, 1.0 / math.sqrt(h // self.heads), causal)
            x = ops.layernorm_train(ops.linear_act(ctx, self.out.weight, self.out.bias, x, "none", p, rng, self.site), self.ln1.weight,
                                    self.ln1.bias, self.ln1.eps)
            hid = ops.linear_act(x, self.fc1.weight, self.fc1.bias, None, "gelu")
            return ops.layernorm_train(ops.linear_act(hid, self.fc2.weight, self.fc2.bias, x, "none", p, rng, self.site + 1), self.ln2.weight,
                                       self.ln2.bias, self.ln2.eps)
        if ORION_TRAIN_KERNELS and OWN_GEMM_TRAINING and x.is_cuda and self.training and x.dtype == torch.bfloat16:
            # every op of the layer, forward and backward, on the orion kernels; residual adds ride in the GEMM epilogues
            ops = torch.ops.orion
            qkv = ops.linear_train(x, self.qkv.weight, self.qkv.bias)
            ctx = ops.attention_train(qkv, self.heads, 1.0 / math.sqrt(h // self.heads), causal)
            x = ops.layernorm_train(ops.linear_train(ctx, self.out.weight, self.out.bias, x), self.ln1.weight, self.ln1.bias, self.ln1.eps)
            hid = ops.bias_gelu_train(ops.linear_train(x, self.fc1.weight, None), self.fc1.bias)
            return ops.layernorm_train(ops.linear_train(hid, self.fc2.weight, self.fc2.bias, x), self.ln2.weight, self.ln2.bias,
                                       self.ln2.eps)
        q, k, v = self.qkv(x).view(b, s, 3, self.heads, h // self.heads).permute(2, 0, 3, 1, 4)
        ctx = F.scaled_dot_product_attention(q, k, v, is_causal=causal).transpose(1, 2).reshape(b, s, h)
        if ORION_TRAIN_KERNELS and x.is_cuda and self.training:
            # LayerNorm and bias + GELU, forward and backward, on the orion kernels (the GEMMs and the attention stay stock)
            ops = torch.ops.orion
            x = ops.layernorm_train((x + F.dropout(self.out(ctx), p)).contiguous(), self.ln1.weight, self.ln1.bias, self.ln1.eps)
            hid = ops.bias_gelu_train(F.linear(x, self.fc1.weight), self.fc1.bias)
            return ops.layernorm_train((x + F.dropout(self.fc2(hid), p)).contiguous(), self.ln2.weight, self.ln2.bias, self.ln2.eps)
        x = self.ln1(x + F.dropout(self.out(ctx), p))
        return self.ln2(x + F.dropout(self.fc2(F.gelu(self.fc1(x))), p))

    def forward_orion(self, x, causal=False):
        """Same math on the orion kernels (inference): x [B, S, H] bfloat16."""
        ops = torch.ops.orion
        b, s, h = x.shape
        d = h // self.heads
        flat = x.reshape(b * s, h)
        if FUSED_LINEAR and d == 64 and (s <= 384 or s % 8 == 0) and x.dtype == torch.bfloat16 and FUSED_ATTENTION:
            attend = ops.attention if s <= 384 else ops.attention_long
            ctx = attend(ops.linear_act(flat, self.qkv.weight, self.qkv.bias).view(b, s, 3 * h), self.heads, 1.0 / math.sqrt(d), causal)
            attn = ops.linear_act(ctx, self.out.weight, self.out.bias, flat)
            y = ops.layernorm(attn, _f32(self, self.ln1.weight), _f32(self, self.ln1.bias), self.ln1.eps)
            out = ops.linear_act(ops.linear_act(y, self.fc1.weight, self.fc1.bias, None, "gelu"), self.fc2.weight, self.fc2.bias, y)
            return ops.layernorm(out, _f32(self, self.ln2.weight), _f32(self, self.ln2.bias), self.ln2.eps).view(b, s, h)
        qkv = ops.linear(flat, self.qkv.weight, _f32(self, self.qkv.bias), False)
        if d == 64 and s <= 384 and x.dtype == torch.bfloat16 and FUSED_ATTENTION:
            # scores, softmax and the context product in one kernel, read straight from the projection's output
            ctx = ops.attention(qkv.view(b, s, 3 * h), self.heads, 1.0 / math.sqrt(d), causal)
        elif d == 64 and s % 8 == 0 and x.dtype == torch.bfloat16 and FUSED_ATTENTION:
            ctx = ops.attention_long(qkv.view(b, s, 3 * h), self.heads, 1.0 / math.sqrt(d), causal)
        else:
            qkv = qkv.view(b, s, 3, self.heads, d)
            q = qkv[:, :, 0].permute(0, 2, 1, 3).reshape(b * self.heads, s, d).contiguous()
            k = qkv[:, :, 1].permute(0, 2, 1, 3).reshape(b * self.heads, s, d).contiguous()
            vt = qkv[:, :, 2].permute(0, 2, 3, 1).reshape(b * self.heads, d, s).contiguous()
            probs = ops.softmax(ops.linear_batched(q, k), 1.0 / math.sqrt(d), s if causal else 0)
            ctx = ops.linear_batched(probs, vt).view(b, self.heads, s, d).permute(0, 2, 1, 3).reshape(b * s, h).contiguous()
        # the residual stream is added in the GEMM epilogue, in float32, before the sum is rounded to bfloat16
        attn = ops.linear(ctx, self.out.weight, _f32(self, self.out.bias), False, flat)
        y = ops.layernorm(attn, _f32(self, self.ln1.weight), _f32(self, self.ln1.bias), self.ln1.eps)
        hid = ops.bias_gelu(ops.linear(y, self.fc1.weight, None, False), _f32(self, self.fc1.bias))
        out = ops.linear(hid, self.fc2.weight, _f32(self, self.fc2.bias), False, y)
        return ops.layernorm(out, _f32(self, self.ln2.weight), _f32(self, self.ln2.bias), self.ln2.eps).view(b, s, h)


class BertQA(nn.Module):
    def __init__(self, cfg=BERT):
        super().__init__()
        h = cfg["hidden"]
        self.word = nn.Embedding(cfg["vocab"], h)
        self.pos = nn.Embedding(cfg["max_pos"], h)
        self.typ = nn.Embedding(2, h)
        self.ln = nn.LayerNorm(h, eps=1e-12)
        self.dropout = cfg.get("dropout", 0.0)
        self.layers = nn.ModuleList([BertLayer(h, cfg["heads"], cfg["ffn"], self.dropout, 2 * i + 1) for i in range(cfg["layers"])])
        self.qa = nn.Linear(h, 2)
        _dropout_state(self, cfg)

    def _own_training(self, ids):
        return ORION_TRAIN_KERNELS and OWN_GEMM_TRAINING and ids.is_cuda and self.training and self.word.weight.dtype == torch.bfloat16

    def embed(self, ids, rng=None, orion=False):
        p = self.dropout if self.training and not orion else 0.0   # a request (orion) drops nothing
        if self._own_training(ids):
            ops = torch.ops.orion
            x = ops.layernorm_train(ops.embedding_train(ids, self.word.weight, self.pos.weight, self.typ.weight), self.ln.weight,
                                    self.ln.bias, self.ln.eps)
            return ops.dropout(x, p, rng, 0) if p > 0.0 else x
        pos = torch.arange(ids.shape[1], device=ids.device)
        return F.dropout(self.ln(self.word(ids) + self.pos(pos)[None] + self.typ.weight[0]), p)

    def forward(self, ids, orion=False):
        if orion and ids.is_cuda and self.word.weight.dtype == torch.bfloat16:
            ops = torch.ops.orion   # the three lookups and their sum in one kernel, then the orion LayerNorm
            b, s = ids.shape
            emb = ops.embedding_train(ids.contiguous(), self.word.weight, self.pos.weight, self.typ.weight)
            x = ops.layernorm(emb.view(b * s, -1), _f32(self, self.ln.weight), _f32(self, self.ln.bias), self.ln.eps).view(b, s, -1)
        else:
            rng = None if orion else self._step(ids)
            x = self.embed(ids, rng, orion)
        for layer in self.layers:
            x = layer.forward_orion(x) if orion else layer(x, False, rng)
        return self.qa(x)   # [B, S, 2]: start / end logits

    def _step(self, ids):
        return _count_step(self.rng) if self.dropout > 0.0 and self._own_training(ids) else None

    def span_logits(self, ids):
        """Training on the orion kernels: the start / end logits as [2, B, S] (positions contiguous, the layout the
        loss reads), computed as qa.weight . x^T.  The head's bias is left out: it shifts all positions of a row alike,
        so the position softmax, the loss and every gradient are the same without it (its own gradient is zero)."""
        b, s = ids.shape
        rng = self._step(ids)
        x = self.embed(ids, rng)
        for layer in self.layers:
            x = layer(x, False, rng)
        return torch.ops.orion.linear_train(self.qa.weight, x.view(b * s, -1), None).view(2, b, s)


class DecoderLM(nn.Module):
    def __init__(self, cfg=LM):
        super().__init__()
        h = cfg["hidden"]
        self.word = nn.Embedding(cfg["vocab"], h)
        self.pos = nn.Embedding(cfg["seq"], h)
        self.dropout = cfg.get("dropout", 0.0)
        self.layers = nn.ModuleList([BertLayer(h, cfg["heads"], cfg["ffn"], self.dropout, 2 * i + 1) for i in range(cfg["layers"])])
        self.ln = nn.LayerNorm(h)
        self.head = nn.Linear(h, cfg["vocab"], bias=False)
        _dropout_state(self, cfg)

    def hidden(self, ids, orion=False):
        """What the vocabulary projection takes: [B, S, H], behind the last LayerNorm.  A request (orion) drops nothing."""
        p = self.dropout if self.training and not orion else 0.0
        if (not orion and ORION_TRAIN_KERNELS and OWN_GEMM_TRAINING and ids.is_cuda and self.training
                and self.word.weight.dtype == torch.bfloat16):
            ops = torch.ops.orion
            rng = _count_step(self.rng) if p > 0.0 else None
            x = ops.embedding_train(ids.contiguous(), self.word.weight, self.pos.weight)
            if p > 0.0:
                x = ops.dropout(x, p, rng, 0)
            for layer in self.layers:
                x = layer(x, True, rng)
            return ops.layernorm_train(x, self.ln.weight, self.ln.bias, self.ln.eps)
        if orion and ids.is_cuda and self.word.weight.dtype == torch.bfloat16:
            x = torch.ops.orion.embedding_train(ids.contiguous(), self.word.weight, self.pos.weight)
        else:
            pos = torch.arange(ids.shape[1], device=ids.device)
            x = F.dropout(self.word(ids) + self.pos(pos)[None], p)
        if not orion:
            for layer in self.layers:
                x = layer(x, causal=True)
            return self.ln(x)
        # inference on the orion kernels: causal softmax, final LayerNorm and the vocabulary projection included
        for layer in self.layers:
            x = layer.forward_orion(x, causal=True)
        b, s, h = x.shape
        return torch.ops.orion.layernorm(x.reshape(b * s, h), _f32(self, self.ln.weight), _f32(self, self.ln.bias), self.ln.eps).view(b, s, h)

    def forward(self, ids, orion=False):
        x = self.hidden(ids, orion)
        if orion:
            return torch.ops.orion.linear(x.view(-1, x.shape[-1]), self.head.weight, None, False).view(*ids.shape, -1)
        if ORION_TRAIN_KERNELS and OWN_GEMM_TRAINING and ids.is_cuda and self.training and x.dtype == torch.bfloat16:
            return torch.ops.orion.linear_train(x, self.head.weight, None)
        return self.head(x)

    def loss(self, ids, target):
        """Mean cross-entropy of the next tokens `target` [B, S] (-100: not asked for; 0 where none is), from the hidden states: on the
        orion kernels neither the logits nor their gradient, 2 x B x S x vocabulary, are ever in memory."""
        x = self.hidden(ids)
        if x.is_cuda and x.dtype == torch.bfloat16 and ORION_TRAIN_KERNELS:
            return torch.ops.orion.linear_cross_entropy(x, self.head.weight, target.contiguous())
        total = F.cross_entropy(self.head(x).float().flatten(0, 1), target.flatten(), reduction="sum")
        return total / (target != -100).sum().clamp(min=1)

    def score(self, ids):
        """Log-likelihood of every token given those before it, [B, S - 1] (a scoring request), without the logits."""
        with torch.no_grad():
            if ids.is_cuda and self.word.weight.dtype == torch.bfloat16:
                target = F.pad(ids[:, 1:], (0, 1), value=-100)   # nothing follows the last token
                return -torch.ops.orion.linear_cross_entropy(self.hidden(ids, orion=True), self.head.weight, target, reduction="none")[:, :-1]
            modes = [(m, m.training) for m in self.modules()]   # the stock path's request: without dropout, whatever mode the model is in
            try:
                logits = self.eval().head(self.hidden(ids))[:, :-1].float()
            finally:
                for m, mode in modes:
                    m.training = mode
            return -F.cross_entropy(logits.flatten(0, 1), ids[:, 1:].flatten(), reduction="none").view(ids.shape[0], -1)


def _adamw(params, lr):
    if ORION_TRAIN_KERNELS and torch.cuda.is_available():
        from orion_b200.optim import AdamW
        return AdamW(params, lr=lr)
    return torch.optim.AdamW(params, lr=lr)


def _pinned(t):
    return t.pin_memory() if torch.cuda.is_available() else t


def bert_loop(batchsize, train, num_iters, rps, uniform, dummy_data, local_rank, barriers, client_barrier, tid, input_file=""):
    seq, vocab = BERT["seq"], 30522
    resident = os.environ.get("ORION_RESIDENT_INPUTS", "0") == "1"

    def build(device):
        model = BertQA(dict(BERT, dropout=DROPOUT, dropout_seed=_client_seed(tid, local_rank))).to(device).to(torch.bfloat16)
        ids = _pinned(torch.randint(0, vocab, (batchsize, seq)))
        labels = _pinned(torch.randint(0, seq, (2, batchsize)))
        state = {"ids": ids.to(device, non_blocking=True), "lab": labels.to(device, non_blocking=True)}
        if train:
            model.train()
            opt = _adamw(model.parameters(), lr=3e-5)

            def step(batch_idx):
                if not resident:
                    state["ids"] = ids.to(device, non_blocking=True)
                    state["lab"] = labels.to(device, non_blocking=True)
                opt.zero_grad()
                if ORION_TRAIN_KERNELS and OWN_GEMM_TRAINING:
                    # both span losses in one pass over the [2 * B, S] logits: mean over 2B rows = half the sum of the two means
                    lt = model.span_logits(state["ids"])
                    loss = 2.0 * torch.ops.orion.cross_entropy(lt.view(-1, seq), state["lab"].view(-1))
                else:
                    logits = model(state["ids"]).float()
                    loss = F.cross_entropy(logits[:, :, 0], state["lab"][0]) + F.cross_entropy(logits[:, :, 1], state["lab"][1])
                loss.backward()
                opt.step()
                return loss
            return step
        model.eval()
        use_orion = os.environ.get("ORION_PREPARE", "1") == "1"

        def step(batch_idx):
            if not resident:
                state["ids"] = ids.to(device, non_blocking=True)
            return model(state["ids"], orion=use_orion)
        return step

    run_client(tid, train, num_iters, rps, uniform, barriers, input_file, batchsize, build)


def transformer_loop(batchsize, train, num_iters, rps, uniform, dummy_data, local_rank, barriers, client_barrier, tid, input_file=""):
    seq, vocab = LM["seq"], LM["vocab"]
    resident = os.environ.get("ORION_RESIDENT_INPUTS", "0") == "1"

    def build(device):
        model = DecoderLM(dict(LM, dropout=DROPOUT, dropout_seed=_client_seed(tid, local_rank))).to(device).to(torch.bfloat16)
        tokens = _pinned(torch.randint(0, vocab, (batchsize, seq + 1)))
        state = {"tok": tokens.to(device, non_blocking=True)}
        if train:
            model.train()
            opt = _adamw(model.parameters(), lr=3e-4)

            def step(batch_idx):
                if not resident:
                    state["tok"] = tokens.to(device, non_blocking=True)
                opt.zero_grad()
                if FUSED_LOSS:
                    loss = model.loss(state["tok"][:, :-1], state["tok"][:, 1:])
                    loss.backward()
                    opt.step()
                    return loss
                logits = model(state["tok"][:, :-1])
                if ORION_TRAIN_KERNELS:   # loss and its gradient straight from the bfloat16 logits, one pass each
                    loss = torch.ops.orion.cross_entropy(logits.reshape(-1, vocab), state["tok"][:, 1:].reshape(-1))
                else:
                    loss = F.cross_entropy(logits.float().view(-1, vocab), state["tok"][:, 1:].reshape(-1))
                loss.backward()
                opt.step()
                return loss
            return step
        model.eval()
        use_orion = os.environ.get("ORION_PREPARE", "1") == "1"

        def step(batch_idx):
            if not resident:
                state["tok"] = tokens.to(device, non_blocking=True)
            return model(state["tok"][:, :-1], orion=use_orion)[:, -1]
        return step

    run_client(tid, train, num_iters, rps, uniform, barriers, input_file, batchsize, build)
