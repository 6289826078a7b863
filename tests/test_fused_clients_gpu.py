"""The language-model clients on the fused layer, counter-based dropout and the loss without logits, against float64 models with the same
masks and against the clients' other paths.  Bounds are the ones of the framework's other whole-model tests: 2e-2 of a tensor's largest
entry for activations and 3e-2 for gradients (a handful of bfloat16 roundings of activations a layer, 2^-8 each)."""
import math

import pytest
import torch
import torch.nn.functional as F

from tests.test_fused_training_gpu import keep_mask

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tt(built):
    from orion_b200 import torch_ops
    torch_ops.load()
    from benchmarking.benchmark_suite import transformer_trainer
    assert transformer_trainer.ORION_TRAIN_KERNELS and transformer_trainer.OWN_GEMM_TRAINING
    return transformer_trainer


@pytest.fixture(autouse=True)
def status(built):
    yield
    from orion_b200 import kernels
    assert kernels.read_status() == 0


def close(got, want, bound, what):
    assert (got.double() - want.double()).abs().max() <= bound * want.double().abs().max(), what


def decoder(tt, p, layers=2, vocab=1001):
    torch.manual_seed(3)
    cfg = dict(tt.LM, layers=layers, hidden=256, heads=4, ffn=512, vocab=vocab, seq=96, dropout=p)
    return tt.DecoderLM(cfg).to(torch.bfloat16).cuda().train(), cfg


def decoder64(model, cfg, ids, masks):
    """Hidden states of a float64 copy, with masks[site] in place of the dropouts (None: none)."""
    p = {k: v.detach().double().requires_grad_(True) for k, v in model.named_parameters()}
    h, heads = cfg["hidden"], cfg["heads"]
    b, s = ids.shape
    drop = lambda v, site: v if masks is None else v * masks[site].view(b, s, h)  # noqa: E731
    lin = lambda v, n: v @ p[n + ".weight"].T + p[n + ".bias"]  # noqa: E731
    norm = lambda v, n, eps: F.layer_norm(v, (h,), p[n + ".weight"], p[n + ".bias"], eps)  # noqa: E731
    x = drop(p["word.weight"][ids] + p["pos.weight"][:s], 0)
    future = torch.ones(s, s, dtype=torch.bool, device=ids.device).triu(1)
    for i in range(cfg["layers"]):
        n = "layers.%d." % i
        q, k, v = lin(x, n + "qkv").view(b, s, 3, heads, h // heads).permute(2, 0, 3, 1, 4)
        ctx = (q @ k.transpose(-1, -2) / math.sqrt(h // heads)).masked_fill(future, -math.inf).softmax(-1) @ v
        x = norm(x + drop(lin(ctx.transpose(1, 2).reshape(b, s, h), n + "out"), 2 * i + 1), n + "ln1", 1e-12)
        x = norm(x + drop(lin(F.gelu(lin(x, n + "fc1")), n + "fc2"), 2 * i + 2), n + "ln2", 1e-12)
    return norm(x, "ln", 1e-5), p


@pytest.mark.parametrize("p", [0.0, 0.1])
def test_decoder_step_with_dropout_and_loss_without_logits(tt, monkeypatch, p):
    monkeypatch.setattr(tt, "FUSED_LINEAR", True)
    model, cfg = decoder(tt, p)
    model.rng[0] = 12345
    ids, target = torch.randint(0, 1001, (3, 88), device="cuda"), torch.randint(0, 1001, (3, 88), device="cuda")
    target[0, 50:] = -100
    before = torch.ops.orion.fallbacks()
    loss = model.loss(ids, target)
    loss.backward()
    assert torch.ops.orion.fallbacks() == before
    assert model.rng.tolist() == [12345, 1 if p else 0]
    masks = None
    if p:
        masks = []
        for site in range(2 * cfg["layers"] + 1):
            keep, f = keep_mask(3 * 88 * 256, p, model.rng, site)
            masks.append(keep.double() * f)
    x, params = decoder64(model, cfg, ids, masks)
    want = F.cross_entropy((x @ params["head.weight"].T).flatten(0, 1), target.flatten())
    want.backward()
    assert abs(loss.item() - want.item()) < 2e-2 * want.item()
    for name, q in model.named_parameters():
        close(q.grad, params[name].grad, 3e-2, name)


def test_a_step_counts_on_and_its_mask_outlives_the_next_forward_pass(tt):
    """Two forward passes before either backward pass, as accumulating gradients does: each backward pass goes by its own step."""
    model, _ = decoder(tt, 0.3, layers=1)
    ids, target = torch.randint(0, 1001, (2, 64), device="cuda"), torch.randint(0, 1001, (2, 64), device="cuda")
    a, b = model.loss(ids, target), model.loss(ids, target)
    assert a.item() != b.item() and model.rng[1].item() == 2
    w = model.layers[0].fc2.weight
    ga, gb = torch.autograd.grad(a, w, retain_graph=True)[0], torch.autograd.grad(b, w)[0]
    assert not torch.equal(ga, gb)
    model.rng[1] = 0
    assert torch.equal(torch.autograd.grad(model.loss(ids, target), w)[0], ga)
    model.eval()
    with torch.no_grad():
        assert torch.equal(model(ids, orion=True), model(ids, orion=True)) and model.rng[1].item() == 1


def test_fused_and_separate_launches_agree(tt, monkeypatch):
    """The same step and the same request with and without ORION_FUSED_LINEAR; the loss from hidden states and from logits."""
    model, _ = decoder(tt, 0.0, vocab=1000)   # the separate projection takes vocabularies of a multiple of 8
    ids, target = torch.randint(0, 1000, (2, 96), device="cuda"), torch.randint(0, 1000, (2, 96), device="cuda")
    results = []
    for fused in (False, True):
        monkeypatch.setattr(tt, "FUSED_LINEAR", fused)
        model.zero_grad(set_to_none=True)
        logits = model(ids)
        loss = torch.ops.orion.cross_entropy(logits.view(-1, 1000), target.view(-1))
        loss.backward()
        with torch.no_grad():
            request = model.eval()(ids, orion=True)
        model.train()
        results.append((logits.detach(), request, {n: q.grad.clone() for n, q in model.named_parameters()}))
    close(results[1][0], results[0][0], 2e-2, "training logits")
    close(results[1][1], results[0][1], 2e-2, "request")
    for name, g in results[0][2].items():
        close(results[1][2][name], g, 3e-2, name)


def test_scoring_request(tt):
    model, cfg = decoder(tt, 0.0)
    model.eval()
    ids = torch.randint(0, 1001, (3, 96), device="cuda")
    got = model.score(ids)
    x, p = decoder64(model, cfg, ids, None)
    want = torch.log_softmax(x @ p["head.weight"].T, -1)[:, :-1].gather(2, ids[:, 1:, None])[..., 0]
    assert got.shape == (3, 95)
    close(got, want.detach(), 2e-2, "scores")
    host = tt.DecoderLM(cfg).double().eval()
    host.load_state_dict({k: v.double().cpu() for k, v in model.state_dict().items()})
    close(host.score(ids.cpu()).cuda(), want.detach(), 1e-5, "scores on the host")


def test_bert_trains_with_dropout(tt):
    """The question-answering client's step with dropout: the loss falls into line with the one without, gradients reach every parameter
    but the head's bias, and the mask moves with the step."""
    torch.manual_seed(5)
    cfg = dict(tt.BERT, layers=2, hidden=256, heads=4, ffn=512, vocab=512, max_pos=64, seq=64, dropout=0.1)
    model = tt.BertQA(cfg).to(torch.bfloat16).cuda().train()
    ids, lab = torch.randint(0, 512, (4, 64), device="cuda"), torch.randint(0, 64, (8,), device="cuda")
    before = torch.ops.orion.fallbacks()
    first = model.span_logits(ids)
    loss = 2.0 * torch.ops.orion.cross_entropy(first.view(-1, 64), lab)
    loss.backward()
    assert torch.ops.orion.fallbacks() == before
    for name, p in model.named_parameters():
        assert name == "qa.bias" or (p.grad is not None and p.grad.isfinite().all() and p.grad.any()), name
    assert not torch.equal(model.span_logits(ids), first)
    model.rng[1] = 0
    assert torch.equal(model.span_logits(ids), first)
