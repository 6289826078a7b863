"""The language clients' dropout state, loss and scores as far as the CPU goes."""
import pickle

import pytest
import torch

from benchmarking.benchmark_suite import transformer_trainer as tt

SMALL = dict(layers=1, hidden=64, heads=2, ffn=128, vocab=96, seq=16, max_pos=16)


def build(kind, **more):
    return getattr(tt, kind)(dict(tt.BERT if kind == "BertQA" else tt.LM, **SMALL, **more))


@pytest.mark.parametrize("kind", ["BertQA", "DecoderLM"])
def test_masks_have_seeds_of_their_own(kind):
    """The seed follows torch.manual_seed, no two models of a process have the same one, and a configuration may name it."""
    def seed(**more):
        rng = build(kind, dropout=0.1, **more).rng
        assert rng.dtype == torch.int64 and rng.shape == (2,) and rng[1] == 0
        return int(rng[0])
    torch.manual_seed(1)
    a, b = seed(), seed()
    torch.manual_seed(1)
    assert seed() == a != b
    torch.manual_seed(2)
    assert seed() not in (a, b)
    assert seed(dropout_seed=77) == 77


@pytest.mark.parametrize("kind", ["BertQA", "DecoderLM"])
def test_a_model_without_dropout_draws_no_seed(kind):
    """What is drawn behind it, a client's token ids say, stays what it was."""
    torch.manual_seed(3)
    plain = build(kind)
    after = torch.get_rng_state()
    torch.manual_seed(3)
    named = build(kind, dropout=0.1, dropout_seed=5)
    assert torch.equal(torch.get_rng_state(), after)
    assert all(torch.equal(p, q) for p, q in zip(plain.parameters(), named.parameters()))


def test_clients_and_ranks_have_different_masks(monkeypatch):
    monkeypatch.delenv("RANK", raising=False)
    torch.manual_seed(42)   # what every client starts with
    seeds = [tt._client_seed(tid, rank) for tid in range(8) for rank in range(8)]
    assert len(set(seeds)) == 64 and all(0 <= s < 2 ** 62 for s in seeds)
    monkeypatch.setenv("RANK", "11")
    assert tt._client_seed(0, 0) not in seeds
    monkeypatch.setattr(tt, "DROPOUT_SEED", "123456789")
    assert tt._client_seed(0, 0) != tt._client_seed(1, 0) and tt._client_seed(0, 0) not in seeds


@pytest.mark.parametrize("kind", ["BertQA", "DecoderLM"])
def test_a_checkpoint_goes_on_with_its_masks(kind):
    """Seed and step are in the checkpoint of a model with dropout; checkpoints of models with and without fit each other."""
    model, other, plain = build(kind, dropout=0.1), build(kind, dropout=0.1), build(kind)
    model.rng[1] = 1234567
    state = model.state_dict()
    assert not torch.equal(other.rng, model.rng)
    other.load_state_dict(state)
    assert torch.equal(other.rng, model.rng) and other.rng.data_ptr() != model.rng.data_ptr()
    assert "rng" not in plain.state_dict()
    plain.load_state_dict(state)
    assert not plain.rng.any() and "rng" in state                   # the caller's dictionary is as it was
    before = other.rng.clone()
    other.load_state_dict(plain.state_dict())
    assert torch.equal(other.rng, before)
    # dropout switched off or on afterwards changes nothing of that
    plain.dropout, other.dropout = 0.1, 0.0
    plain.load_state_dict(state)
    plain.load_state_dict(plain.state_dict())
    other.load_state_dict(plain.state_dict())
    other.load_state_dict(state)
    assert torch.equal(other.rng, model.rng)
    # a whole model, and one inside a larger module
    assert torch.equal(pickle.loads(pickle.dumps(model)).rng, model.rng)
    outer, again = (torch.nn.Sequential(build(kind, dropout=0.1)) for _ in range(2))
    again.load_state_dict(outer.state_dict())
    assert torch.equal(again[0].rng, outer[0].rng)


def test_loss_of_no_tokens_is_zero_on_the_stock_path_too():
    """As on the orion kernels: a step whose targets are all masked has no loss and no gradient.  With targets the mean is torch's."""
    import torch.nn.functional as F
    torch.manual_seed(4)
    model = build("DecoderLM")
    ids, target = torch.randint(0, 96, (2, 16)), torch.randint(0, 96, (2, 16))
    target[0, 5:] = -100
    want = F.cross_entropy(model(ids).flatten(0, 1), target.flatten())
    assert abs(model.loss(ids, target) - want) <= 16 * 2.0 ** -23 * want   # 21 terms in another order, each rounding half of 2^-23
    loss = model.loss(ids, torch.full_like(target, -100))
    loss.backward()
    assert loss.item() == 0 and not any(p.grad.any() for p in model.parameters() if p.grad is not None)


def test_requests_drop_nothing():
    """Scores, and embeddings of a request, are the same in training mode as in evaluation; the modes stay what they were."""
    torch.manual_seed(5)
    ids = torch.randint(0, 96, (2, 16))
    model = build("DecoderLM", dropout=0.5)
    want = model.eval().score(ids)
    model.train()
    model.ln.eval()
    assert torch.equal(model.score(ids), want) and model.training and model.layers[0].training and not model.ln.training
    assert not torch.equal(model(ids), model(ids))
    bert = build("BertQA", dropout=0.5).train()
    assert torch.equal(bert.embed(ids, orion=True), bert.embed(ids, orion=True)) and not torch.equal(bert.embed(ids), bert.embed(ids))
