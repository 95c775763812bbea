"""Backbones with ``dropout_generator: counter``: configuration, reproducibility, checkpointing, kernels against fp32."""

from __future__ import annotations

import copy

import pytest
import torch
from transformers import DebertaV2Config

from deberta_b200.config import ModelConfig, validate_model_config
from deberta_b200.models.builder import _apply_dropout
from deberta_b200.models.deberta_v2 import DebertaV2Model
from deberta_b200.models.drop import counter_based
from deberta_b200.models.rope_encoder import DebertaRoPEConfig, DebertaRoPEModel


def _model(kind, generator="counter", p=0.1, heads=2, conv=0):
    if kind == "deberta":
        cfg = DebertaV2Config(vocab_size=100, hidden_size=64 * heads, num_hidden_layers=2, num_attention_heads=heads,
                              intermediate_size=192, hidden_act="gelu", max_position_embeddings=128, position_buckets=32,
                              relative_attention=True, position_biased_input=False, share_att_key=True,
                              norm_rel_ebd="layer_norm", pos_att_type=["p2c", "c2p"], type_vocab_size=0, layer_norm_eps=1e-7,
                              hidden_dropout_prob=p, attention_probs_dropout_prob=p)
        cfg.conv_kernel_size = conv
        cls = DebertaV2Model
    else:
        cfg = DebertaRoPEConfig(vocab_size=100, hidden_size=64 * heads, num_hidden_layers=2, num_attention_heads=heads,
                                intermediate_size=192, type_vocab_size=0, norm_arch=kind, hidden_dropout_prob=p,
                                attention_probs_dropout_prob=p)
        cls = DebertaRoPEModel
    cfg.dropout_generator = generator
    torch.manual_seed(0)
    return cls(cfg).train()


def _ids(device="cpu", B=3, S=50):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(1, 100, (B, S), generator=g)
    keep = torch.ones(B, S, dtype=torch.bool)
    keep[0, S - 7:] = False
    ids[0, S - 7:] = 0
    return ids.to(device), keep.to(device)


def _grads(model, ids, keep, seed):
    model.zero_grad()
    torch.manual_seed(seed)
    out = model(ids, attention_mask=keep).last_hidden_state
    # the gradient that arrives at a bf16 output is rounded to bf16; the fp32 model has to be given the same one: the ramp is
    # nearly constant within a row, which the last norm cancels, so a row keeps about 2 * 128 / numel of it against a
    # rounding of 2^-9
    w = torch.linspace(-1, 1, out.numel(), device=out.device).view(out.shape).bfloat16().float()
    (out.float() * w).sum().backward()
    return out.detach(), {n: p.grad.detach().clone() for n, p in model.named_parameters() if p.grad is not None}


KINDS = ["deberta", "post", "keel"]


@pytest.mark.parametrize("kind", KINDS)
def test_masks_follow_the_seed_and_vanish_in_evaluation(kind):
    model, (ids, keep) = _model(kind, conv=3 if kind == "deberta" else 0), _ids()
    a, ga = _grads(model, ids, keep, 5)
    b, gb = _grads(model, ids, keep, 5)
    c, _ = _grads(model, ids, keep, 6)
    assert torch.equal(a, b) and not torch.equal(a, c)
    assert all(torch.equal(ga[n], gb[n]) for n in ga)
    model.eval()
    plain = _model(kind, "torch", conv=3 if kind == "deberta" else 0).eval()
    plain.load_state_dict(model.state_dict())
    assert torch.equal(model(ids, attention_mask=keep).last_hidden_state, plain(ids, attention_mask=keep).last_hidden_state)


@pytest.mark.parametrize("kind", KINDS)
def test_recomputed_layers_draw_the_same_masks(kind):
    model, (ids, keep) = _model(kind), _ids()
    a, ga = _grads(model, ids, keep, 5)
    model.gradient_checkpointing_enable()
    b, gb = _grads(model, ids, keep, 5)
    assert torch.equal(a, b)
    for n in ga:
        assert torch.allclose(ga[n], gb[n], rtol=1e-5, atol=1e-6), n


@pytest.mark.parametrize("kind", KINDS)
def test_the_mean_over_masks_is_near_the_undropped_layer_input(kind):
    """The embeddings' dropout alone: averaged over n seeds it returns to the undropped value within six standard errors."""
    model, (ids, keep) = _model(kind, p=0.3), _ids()
    emb = model.embeddings
    with torch.no_grad():
        model.eval()
        want = emb(input_ids=ids)
        model.train()
        got = torch.stack([emb(input_ids=ids) for _ in range(400)]).mean(0)
    assert ((got - want).abs() <= 6 * want.abs() * (0.3 / 0.7 / 400) ** 0.5 + 1e-6).all()


def test_the_default_is_torchs_generator_and_unknown_names_are_refused():
    cfg = ModelConfig()
    assert cfg.dropout.generator == "torch"
    hf = DebertaV2Config()
    _apply_dropout(hf, cfg)
    assert not counter_based(hf) and getattr(hf, "dropout_generator", None) is None
    cfg = ModelConfig(dropout_generator="counter", hidden_dropout_prob=0.1)
    validate_model_config(cfg)
    _apply_dropout(hf, cfg)
    assert counter_based(hf) and hf.hidden_dropout_prob == 0.1
    again = copy.deepcopy(hf)
    _apply_dropout(again, ModelConfig())
    assert not counter_based(again)
    assert counter_based(DebertaRoPEConfig(dropout_generator="counter"))
    with pytest.raises(ValueError):
        validate_model_config(ModelConfig(dropout_generator="philox"))
    hf.dropout_generator = "other"
    with pytest.raises(ValueError):
        counter_based(hf)


def test_torchs_generator_gives_what_it_gave():
    """The same draws in the same order as the written-out layers."""
    import torch.nn.functional as F

    model, (ids, keep) = _model("post", "torch", p=0.2), _ids()
    torch.manual_seed(9)
    got = model(ids, attention_mask=keep).last_hidden_state
    torch.manual_seed(9)
    x = F.dropout(model.embeddings.norm(model.embeddings.word_embeddings(ids)), 0.2, True)
    for layer in model.encoder.layers:
        x = layer.norm1(x + F.dropout(layer.attn(x, keep), 0.2, True))
        x = layer.norm2(x + F.dropout(layer.mlp(x), 0.2, True))
    assert torch.equal(got, x)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_kernels_match_the_fp32_statements_with_the_same_masks(kind):
    from deberta_b200.ops import _lib

    wide = _model(kind, p=0.15).cuda()
    model = copy.deepcopy(wide).bfloat16()
    wide.load_state_dict({n: t.float() for n, t in model.state_dict().items()})
    ids, keep = _ids("cuda", S=150 if kind != "deberta" else 128)
    a, ga = _grads(wide, ids, keep, 5)
    before = _lib.LAUNCH_COUNT
    b, gb = _grads(model, ids, keep, 5)
    _lib.check_status()
    assert _lib.LAUNCH_COUNT - before > 20
    # two layers of about ten bf16 roundings each; another mask would differ by the order of one
    assert (b.float() - a).norm() < 0.03 * a.norm()
    for n in ga:
        if ga[n].norm() > 0:
            assert (gb[n].float() - ga[n]).norm() < 0.08 * ga[n].norm(), n
    c, _ = _grads(model, ids, keep, 6)
    assert (c.float() - a).norm() > 0.1 * a.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_training_steps_run_on_the_kernels_with_checkpointing(kind):
    model = _model(kind).cuda().bfloat16()
    ids, keep = _ids("cuda", S=128)
    a, ga = _grads(model, ids, keep, 5)
    model.gradient_checkpointing_enable()
    b, gb = _grads(model, ids, keep, 5)
    assert torch.equal(a, b)
    for n in ga:  # (fp32 atomics in the norms' and the query gradients)
        assert (ga[n].float() - gb[n].float()).norm() <= 0.01 * ga[n].float().norm() + 1e-6, n
