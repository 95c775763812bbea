"""Counter-based dropout, residual norms, attention dropout and the scaled embedding: PyTorch statements and refusals."""

from __future__ import annotations

import math

import pytest
import torch

from deberta_b200.ops.attention import (disentangled_attention, disentangled_attention_reference, relative_positions,
                                        rope_attention, rope_attention_reference)
from deberta_b200.ops.dropout import draw_seed, dropout, dropout_add, dropout_keep_mask, dropout_threshold
from deberta_b200.ops.embedding import scaled_embedding
from deberta_b200.ops.norm import add_layer_norm, add_rms_norm


def _philox(counter, key):
    """Philox4x32 with seven rounds in Python integers."""
    c, k = list(counter), list(key)
    for _ in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


@pytest.mark.parametrize("seed", [0, 1, 0x0123456789ABCDEF, (1 << 62) - 5, -1])
def test_mask_is_the_published_generator(seed):
    rows, cols, p = 5, 21, 0.37
    mask = dropout_keep_mask((rows, cols), p, seed)
    again = dropout_keep_mask((rows, cols), p, torch.tensor([seed]))
    assert torch.equal(mask, again)
    key = (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)
    for r in range(rows):
        for c in range(cols):
            word = _philox((c // 8, r, 0, 0), key)[(c % 8) // 2]
            assert bool(mask[r, c]) == ((word >> (16 * (c % 2))) & 0xFFFF >= dropout_threshold(p))


def test_mask_of_leading_dimensions_is_that_of_their_rows():
    flat = dropout_keep_mask((24, 19), 0.2, 7)
    assert torch.equal(dropout_keep_mask((2, 3, 4, 19), 0.2, 7), flat.view(2, 3, 4, 19))


@pytest.mark.parametrize("p", [0.05, 0.1, 0.5, 0.9])
def test_share_of_dropped_places(p):
    n = 512 * 1024
    dropped = int((~dropout_keep_mask((512, 1024), p, 11)).sum())
    q = dropout_threshold(p) / 65536
    assert abs(dropped - n * q) < 6 * math.sqrt(n * q * (1 - q))  # six standard deviations


def test_seeds_and_places_are_independent():
    a, b = dropout_keep_mask((256, 512), 0.5, 1), dropout_keep_mask((256, 512), 0.5, 2)
    n = a.numel()
    for x, y in ((a, b), (a[1:], a[:-1]), (a[:, 1:], a[:, :-1]), (a[:, 8:], a[:, :-8])):
        same = int((x == y).sum())
        assert abs(same - x.numel() / 2) < 6 * math.sqrt(n / 4)


@pytest.mark.parametrize("p", [-0.1, 1.0, 0.999999, float("nan"), 2])
def test_probabilities_that_are_refused(p):
    x = torch.zeros(2, 4)
    with pytest.raises(ValueError):
        dropout(x, p, 0)
    with pytest.raises(ValueError):
        add_rms_norm(x, x, torch.ones(4), 1e-6, dropout_p=p, seed=0)
    if p > 0:
        with pytest.raises(ValueError):
            rope_attention(x.view(1, 2, 4), x.view(1, 2, 4), x.view(1, 2, 4), None, None, heads=1, rotary_dim=0, dropout_p=p,
                           training=True, dropout_seed=0)


@pytest.mark.parametrize("seed,error", [(1.5, TypeError), (True, TypeError), (None, TypeError),
                                        (torch.zeros(2, dtype=torch.int64), ValueError),
                                        (torch.zeros(1, dtype=torch.int32), ValueError)])
def test_seeds_that_are_refused(seed, error):
    with pytest.raises(error):
        dropout(torch.zeros(2, 4), 0.1, seed)
    with pytest.raises(error):
        dropout_add(torch.zeros(2, 4), torch.zeros(2, 4), 0.1, seed)


def test_arguments_that_are_refused():
    x = torch.zeros(2, 4)
    with pytest.raises(TypeError):
        dropout(x.long(), 0.1, 0)
    for other in (torch.zeros(4), torch.zeros(2, 4, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            dropout_add(x, other, 0.1, 0)
        with pytest.raises(ValueError):
            add_layer_norm(x, other, torch.ones(4), None, 1e-6)
    for w in (torch.ones(3), torch.ones(1, 4)):
        with pytest.raises(ValueError):
            add_rms_norm(x, x, w, 1e-6)
    with pytest.raises(ValueError):
        add_layer_norm(x, x, torch.ones(4), torch.ones(2), 1e-6)
    with pytest.raises(ValueError):
        add_rms_norm(x, x, torch.ones(4), 1e-6, dropout_p=0.1)  # no seed
    table = torch.zeros(5, 4)
    for ids, tab, pad in ((torch.zeros(2), table, None), (torch.zeros(2, dtype=torch.int16), table, None),
                          (torch.zeros(2, dtype=torch.long), table[0], None), (torch.zeros(2, dtype=torch.long), table, 5),
                          (torch.zeros(2, dtype=torch.long), table.long(), None)):
        with pytest.raises(ValueError):
            scaled_embedding(ids, tab, 1.0, pad)


def test_nothing_is_dropped_out_of_training_or_below_the_resolution():
    x, r = torch.randn(3, 9), torch.randn(3, 9)
    assert dropout(x, 0.5, 0, training=False) is x and dropout(x, 1e-6, 0) is x
    assert torch.equal(dropout_add(x, r, 0.5, 0, training=False), x + r)
    y, total = add_rms_norm(x, r, torch.ones(9), 1e-6, dropout_p=0.5, training=False)
    assert torch.equal(total, x + r)


@pytest.mark.parametrize("shape", [(), (1,), (0, 7), (3, 0), (2, 3, 5)])
def test_dropout_statement_on_any_shape(shape):
    x = torch.randn(shape, dtype=torch.float64, requires_grad=True)
    r = torch.randn(shape, dtype=torch.float64, requires_grad=True)
    f = dropout_keep_mask(shape, 0.25, 3).double() / 0.75
    out = dropout_add(x, r, 0.25, 3)
    assert torch.equal(out, torch.where(f > 0, x * (1 / 0.75), torch.zeros_like(x)) + r)
    g = torch.randn_like(out)
    dx, dr = torch.autograd.grad(out, (x, r), g)
    assert torch.allclose(dx, g * f, rtol=1e-15) and torch.equal(dr, g)


def test_dropped_infinities_leave_no_nan():
    x = torch.full((4, 64), float("inf"))
    out = dropout(x, 0.5, 9)
    keep = dropout_keep_mask((4, 64), 0.5, 9)
    assert torch.equal(out, torch.where(keep, x, torch.zeros_like(x)))


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_residual_norm_statement_and_differences(rms, p):
    torch.manual_seed(0)
    x, r, w, b = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((3, 10), (3, 10), (10,), (10,)))
    f = (dropout_keep_mask((3, 10), p, 5).double() / (1 - dropout_threshold(p) / 65536)) if p else 1.0

    def op(x, r, w, b):
        return (add_rms_norm(x, r, w, 1e-3, dropout_p=p, seed=5) if rms
                else add_layer_norm(x, r, w, b, 1e-3, dropout_p=p, seed=5))

    y, total = op(x, r, w, b)
    t = r + x * f
    c = t if rms else t - t.mean(-1, keepdim=True)
    want = c / torch.sqrt(c.pow(2).mean(-1, keepdim=True) + 1e-3) * w + (0 if rms else b)
    assert torch.allclose(total, t, rtol=1e-14) and torch.allclose(y, want, rtol=1e-12, atol=1e-14)
    assert torch.autograd.gradcheck(lambda *a: op(*a), (x, r, w, b))


def test_attention_statements_drop_the_map_of_the_generator():
    torch.manual_seed(1)
    B, S, heads, d, span = 2, 9, 2, 4, 8
    q, k, v = (torch.randn(B, S, heads * d) for _ in range(3))
    pk, pq = torch.randn(2 * span, heads * d), torch.randn(2 * span, heads * d)
    keep = torch.ones(B, S, dtype=torch.bool)
    keep[1, 6:] = False
    keep[0] = False  # a row that sees nothing
    rel = relative_positions(S, S, 0, 0)
    seed, p = torch.tensor([77]), 0.4
    factor = dropout_keep_mask((B, heads, S, S), p, seed).float() / (1 - dropout_threshold(p) / 65536)
    split = lambda t: t.view(B, S, heads, d).permute(0, 2, 1, 3)  # noqa: E731

    def by_hand(run, **kw):
        # the undropped map of every query, read off with unit vectors as values
        maps = []
        for h in range(heads):
            for j in range(S):
                unit = torch.zeros(B, S, heads * d)
                unit[:, j, h * d] = 1.0
                maps.append(run(q, k, unit, **kw)[:, :, h * d])
        prob = torch.stack(maps, -1).view(B, S, heads, S).permute(0, 2, 1, 3)
        return ((prob * factor) @ split(v)).permute(0, 2, 1, 3).reshape(B, S, heads * d)

    dis = lambda a, b, c, **kw: disentangled_attention(  # noqa: E731
        a, b, c, pk, pq, heads=heads, scale_factor=3, bucket_size=0, max_position=0, att_span=span, key_keep=keep, **kw)
    rope = lambda a, b, c, **kw: rope_attention(a, b, c, None, None, heads=heads, rotary_dim=0, key_keep=keep, **kw)  # noqa: E731
    for run in (dis, rope):
        got = run(q, k, v, dropout_p=p, training=True, dropout_seed=seed)
        assert torch.allclose(got, by_hand(run), atol=1e-5)
        assert not got[0].any()
        assert torch.equal(run(q, k, v, dropout_p=p, training=False, dropout_seed=seed), run(q, k, v))
    a = disentangled_attention_reference(q, k, v, pk, pq, heads=heads, scale_factor=3, rel_pos=rel, att_span=span,
                                         dropout_p=p, training=True, dropout_seed=3)
    b = disentangled_attention_reference(q, k, v, pk, pq, heads=heads, scale_factor=3, rel_pos=rel, att_span=span,
                                         dropout_p=p, training=True, dropout_seed=torch.tensor([3]))
    assert torch.equal(a, b)
    with pytest.raises(TypeError):
        rope_attention_reference(q, k, v, None, None, heads=heads, rotary_dim=0, dropout_p=p, training=True,
                                 dropout_seed=0.5)


def test_attention_without_a_seed_keeps_torchs_generator():
    q = torch.randn(1, 5, 8)
    kw = dict(heads=2, rotary_dim=0, dropout_p=0.5, training=True)
    torch.manual_seed(3)
    a = rope_attention(q, q, q, None, None, **kw)
    torch.manual_seed(3)
    scores = (q.view(1, 5, 2, 4).transpose(1, 2) @ q.view(1, 5, 2, 4).permute(0, 2, 3, 1)) / 2.0
    probs = torch.nn.functional.dropout(torch.softmax(scores, -1), 0.5, True)
    assert torch.allclose(a, (probs @ q.view(1, 5, 2, 4).transpose(1, 2)).transpose(1, 2).reshape(1, 5, 8), atol=1e-6)


def test_scaled_embedding_statement():
    torch.manual_seed(2)
    table = torch.randn(7, 5, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[0, 3, 3], [6, 1, 3]])
    out = scaled_embedding(ids, table, 2.5, padding_idx=-6)
    assert torch.equal(out, table[ids] * 2.5)
    g = torch.randn_like(out)
    (d,) = torch.autograd.grad(out, (table,), g)
    want = torch.zeros_like(table).index_add_(0, ids.view(-1), g.view(-1, 5) * 2.5)
    want[1] = 0
    assert torch.allclose(d, want, rtol=1e-14)
    assert scaled_embedding(ids.int(), table).shape == (2, 3, 5)
    assert scaled_embedding(ids[:0], table).shape == (0, 3, 5)


def test_draw_seed_follows_the_generator():
    torch.manual_seed(5)
    a, b = draw_seed(), draw_seed()
    torch.manual_seed(5)
    assert torch.equal(a, draw_seed()) and not torch.equal(a, b) and a.dtype == torch.int64


def test_operators_under_a_compiler_draw_the_same_masks():
    x, r, w = torch.randn(6, 40), torch.randn(6, 40), torch.randn(40)
    seed = torch.tensor([99])

    def f(x, r, w, seed):
        y, total = add_rms_norm(dropout(x, 0.3, seed), r, w, 1e-6, dropout_p=0.2, seed=seed + 1)
        a = rope_attention(y.view(1, 6, 40), r.view(1, 6, 40), x.view(1, 6, 40), None, None, heads=2, rotary_dim=0,
                           dropout_p=0.2, training=True, dropout_seed=seed + 2)
        return y, total, a

    for got, want in zip(torch.compile(f, backend="aot_eager", fullgraph=True)(x, r, w, seed), f(x, r, w, seed)):
        assert torch.allclose(got, want, atol=1e-6)


def _op_cases():
    from deberta_b200.ops import library as L

    g = torch.Generator().manual_seed(0)
    t = lambda *s, grad=False: torch.randn(*s, generator=g).requires_grad_(grad)  # noqa: E731
    seed = torch.tensor([5])
    x, r, w, b = t(6, 24, grad=True), t(6, 24, grad=True), t(24, grad=True), t(24, grad=True)
    yield "dropout_keep", L.dropout_keep, (seed, 6, 21, 9000)
    yield "dropout", L.dropout, (x, None, seed, 9000)
    yield "dropout-residual", L.dropout, (x, r, seed, 9000)
    yield "add_layer_norm", L.add_norm, (x, r, w, b, seed, 9000, 1e-6, False)
    yield "add_rms_norm", L.add_norm, (x, r, w, None, None, 0, 1e-6, True)
    y, total, stats = L.add_norm(x.detach(), r.detach(), w.detach(), b.detach(), seed, 9000, 1e-6, False)
    yield "add_norm_bwd", L.add_norm_bwd, (t(6, 24), t(6, 24), total, w.detach(), stats, seed, 9000, False, True)
    yield "add_norm_bwd-plain", L.add_norm_bwd, (t(6, 24), t(6, 24), total, w.detach(), stats[:6], None, 0, True, False)
    q, k, v = (t(2, 12, 128, grad=True) for _ in range(3))
    pk, pq = t(16, 128, grad=True), t(16, 128, grad=True)
    keep = torch.ones(2, 12, dtype=torch.bool)
    keep[1, 9:] = False
    yield "flash_attn_drop", L.flash_attn_drop, (q, k, v, pk, pq, keep, None, seed, 13000, 2, 13.86, 8, 16, 8)
    yield "flash_attn_drop-content", L.flash_attn_drop, (q, k, v, None, None, None, None, seed, 13000, 2, 8.0, 0, 0, 0)


OP_CASES = list(_op_cases())


@pytest.mark.parametrize("name,op,args", OP_CASES, ids=[c[0] for c in OP_CASES])
def test_custom_ops_of_a_compiler(name, op, args):
    torch.library.opcheck(op, args)


@pytest.mark.parametrize("rms,p", [(False, 0.0), (False, 0.3), (True, 0.3)])
def test_residual_norm_op_has_the_gradients_of_the_statement(rms, p):
    from deberta_b200.ops import library as L

    torch.manual_seed(3)
    leaves = [torch.randn(*s, requires_grad=True) for s in ((5, 16), (5, 16), (16,), (16,))][: 3 if rms else 4]
    x, r, w, b = leaves + [None] * (4 - len(leaves))
    g = [torch.randn(5, 16), torch.randn(5, 16)]
    threshold = dropout_threshold(p)
    a = L.add_norm(x, r, w, b, torch.tensor([8]) if threshold else None, threshold, 1e-5, rms)[:2]
    c = (add_rms_norm(x, r, w, 1e-5, dropout_p=p, seed=8) if rms else add_layer_norm(x, r, w, b, 1e-5, dropout_p=p, seed=8))
    for u, v in zip(a, c):
        assert torch.allclose(u, v, atol=1e-6)
    for u, v in zip(torch.autograd.grad(a, leaves, g), torch.autograd.grad(c, leaves, g)):
        assert torch.allclose(u, v, atol=1e-5)


@pytest.mark.parametrize("positions", [True, False])
def test_attention_op_has_the_gradients_of_the_statement(positions):
    from deberta_b200.ops import library as L

    torch.manual_seed(4)
    q, k, v = (torch.randn(2, 9, 32, requires_grad=True) for _ in range(3))
    pk, pq = (torch.randn(16, 32, requires_grad=True) for _ in range(2)) if positions else (None, None)
    keep = torch.ones(2, 9, dtype=torch.bool)
    keep[0, 6:] = False
    leaves = [t for t in (q, k, v, pk, pq) if t is not None]
    out = L.flash_attn_drop(q, k, v, pk, pq, keep, None, torch.tensor([6]), dropout_threshold(0.3), 2,
                            math.sqrt(16.0 * 3), 0, 0, 8)[0]
    ref = disentangled_attention_reference(q, k, v, pk, pq, heads=2, scale_factor=3,
                                           rel_pos=relative_positions(9, 9, 0, 0) if positions else None, att_span=8,
                                           key_keep=keep, dropout_p=0.3, training=True, dropout_seed=6)
    g = torch.randn_like(out)
    assert torch.allclose(out, ref, atol=1e-5)
    for u, v in zip(torch.autograd.grad(out, leaves, g), torch.autograd.grad(ref, leaves, g)):
        assert torch.allclose(u, v, atol=1e-4)
