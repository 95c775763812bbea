"""Kernels of counter-based dropout, residual norms, attention with dropout and the sorted embedding gradient against 64 bits.

Tolerances are bounds by arithmetic, evaluated place by place in 64 bits: every rounding to a type counts ``eps / 2`` of the
value (``half`` below), every fp32 sum of n terms n * 2^-24 of the sum of their magnitudes (``U``).
"""

from __future__ import annotations

import math

import pytest
import torch

from deberta_b200.ops import _lib
from deberta_b200.ops.attention import disentangled_attention, relative_positions, rope_attention
from deberta_b200.ops.dropout import dropout, dropout_add, dropout_keep_mask, dropout_threshold
from deberta_b200.ops.embedding import embedding_lookup, scaled_embedding
from deberta_b200.ops.norm import add_layer_norm, add_rms_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)


def within(got, want, bound, dtype):
    """|got - want| <= bound + half a step of ``dtype`` at want, everywhere (its smallest subnormal for fp16 underflow)."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got.double() - want).abs() - bound - half(dtype) * (want.abs() + bound) - tiny
    assert torch.isfinite(got.double()).all()
    assert off.max().item() <= 0, f"over by {off.max().item()}"


def factor(shape, p, seed):
    """64-bit map of 0 and 1 / (1 - p), drawn on the CPU."""
    keep = dropout_keep_mask(shape, p, int(seed)).cuda()
    return keep.double() * 65536 / (65536 - dropout_threshold(p))


# ---- dropout ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (5, 768), (129, 770), (1000, 384), (2, 8200), (4099, 24)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_forward_backward(dtype, rows, cols, residual):
    x, r, g = (rand(rows, cols, dtype=dtype, seed=s).requires_grad_(s < 2) for s in range(3))
    p, seed = 0.3, torch.tensor([0x1234567811223344], device="cuda")
    f = factor((rows, cols), p, seed)
    out = dropout_add(x, r, p, seed) if residual else dropout(x, p, seed)
    want = x.detach().double() * f + (r.detach().double() if residual else 0)
    within(out, want, 3 * U * (x.detach().double().abs() * f + r.detach().double().abs()), dtype)
    (dx,) = torch.autograd.grad(out, (x,), g, retain_graph=True)
    within(dx, g.double() * f, 2 * U * g.double().abs() * f, dtype)
    if residual:
        assert torch.equal(torch.autograd.grad(out, (r,), g)[0], g)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_dropout_of_strided_views(dtype):
    base = rand(40, 3, 200, dtype=dtype)
    views = [base[:, 1], base[:, :, :64], base[::3, 2, 8:72], base[:, 0, 1:66], base.transpose(0, 2), base[:, 0, ::2],
             base[:1].expand(9, 3, 200), base[5, 1, 3:40], base[0, 0, 0]]
    for v in views:
        assert torch.equal(dropout(v, 0.4, 5), dropout(v.contiguous(), 0.4, 5))
        assert torch.equal(dropout_add(v, v, 0.4, 5), dropout_add(v.contiguous(), v.contiguous(), 0.4, 5))


def test_dropout_reads_an_int_and_a_tensor_alike_and_rows_past_32_bits_of_places():
    x = rand(64, 96)
    for seed in (0, -1, (1 << 63) - 1, 1 << 40):
        t = torch.tensor([seed], device="cuda")
        assert torch.equal(dropout(x, 0.5, seed), dropout(x, 0.5, t))
    big = torch.ones(70001, 65536, dtype=torch.bfloat16, device="cuda")  # 4.6e9 values, 5.7e8 vectors
    out = dropout(big, 0.5, 3)
    assert torch.equal(out[:4] != 0, dropout_keep_mask((4, 65536), 0.5, 3, "cuda"))
    tail = dropout_keep_mask((70001, 8), 0.5, 3, "cuda")
    assert torch.equal(out[:, :8] != 0, tail)


def test_dropout_of_more_vectors_than_31_bits_count():
    rows, p, seed = (1 << 31) + 77, 0.5, 0x123456789
    out = dropout(torch.ones(rows, 1, dtype=torch.bfloat16, device="cuda"), p, seed)
    at = [0, 1, (1 << 31) - 1, 1 << 31, (1 << 31) + 1, rows - 1, *range((1 << 31) - 20, (1 << 31) + 20)]
    got = out.view(-1)[torch.tensor(at, device="cuda")].cpu()
    for r, y in zip(at, got.tolist()):
        c, k = [0, r, 0, 0], [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(7):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        assert y == (2.0 if (c[0] & 0xFFFF) >= 32768 else 0.0)


def test_a_captured_draw_is_fresh_at_every_replay():
    from deberta_b200.ops.dropout import draw_seed

    x = torch.ones(64, 256, device="cuda")
    dropout(x, 0.5, draw_seed(x.device))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = dropout(x, 0.5, draw_seed(x.device))
    graph.replay()
    first = out.clone()
    graph.replay()
    assert 0.4 < (first != out).float().mean() < 0.6


def test_dropout_differentiates_twice():
    x = rand(6, 16).requires_grad_(True)
    (d,) = torch.autograd.grad((dropout(x, 0.5, 1) ** 3).sum(), (x,), create_graph=True)
    (dd,) = torch.autograd.grad(d.sum(), (x,))
    f = factor((6, 16), 0.5, 1)
    want = 6 * x.detach().double() * f ** 3
    within(dd, want, 16 * U * want.abs(), torch.float32)


def test_an_overwritten_seed_is_an_error():
    x, seed = rand(4, 8).requires_grad_(True), torch.tensor([4], device="cuda")
    out = dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_seeds_on_another_device_are_refused():
    with pytest.raises(ValueError):
        dropout(rand(2, 8), 0.5, torch.tensor([1]))


# ---- norms of a residual sum ----------------------------------------------------------------------------------------------
def _norm_case(dtype, rows, cols, rms, p, has_bias=True, seed=9):
    x, r, dy, dt = (rand(rows, cols, dtype=dtype, seed=s, scale=1.5, shift=0.25) for s in range(4))
    w, b = rand(cols, dtype=dtype, seed=4, scale=0.2, shift=1.0), rand(cols, dtype=dtype, seed=5)
    leaves = [t.requires_grad_(True) for t in (x, r, w)] + ([] if rms or not has_bias else [b.requires_grad_(True)])
    kw = {"dropout_p": p, "seed": seed}
    out = add_rms_norm(x, r, w, 1e-6, **kw) if rms else add_layer_norm(x, r, w, b if has_bias else None, 1e-6, **kw)
    return out, leaves, (x, r, w, b if has_bias else None, dy, dt)


def _norm_check(dtype, rows, cols, rms, p, has_bias=True, use=(True, True)):
    (y, total), leaves, (x, r, w, b, dy, dt) = _norm_case(dtype, rows, cols, rms, p, has_bias)
    grads = torch.autograd.grad([o for o, u in zip((y, total), use) if u], leaves, [g for g, u in zip((dy, dt), use) if u],
                                allow_unused=True)
    wide = [t.detach().double() for t in (x, r, w)]
    f = factor((rows, cols), p, 9) if p else torch.ones((), dtype=torch.float64, device="cuda")
    t = wide[1] + wide[0] * f
    terms = 64 + cols // 32  # adds on the longest path of a row's sum, with room to spare
    err_t = 3 * U * (wide[1].abs() + wide[0].abs() * f)
    within(total, t, err_t, dtype)
    mean = 0 if rms else t.mean(-1, keepdim=True)
    c = t - mean
    rstd = (c.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()
    xh = c * rstd
    size = t.abs() + t.abs().mean(-1, keepdim=True)
    err_xh = 4 * terms * U * (size * rstd + xh.abs())
    wv, bv = wide[2], (b.detach().double() if b is not None and not rms else torch.zeros_like(wide[2]))
    within(y, xh * wv + bv, err_xh * wv.abs() + 4 * U * (xh * wv).abs() + 2 * U * bv.abs(), dtype)
    # backward: xhat comes from the rounded sum
    err_xh = err_xh + rstd * half(dtype) * t.abs()
    gy = dy.double() if use[0] else torch.zeros_like(t)
    gt = dt.double() if use[1] else torch.zeros_like(t)
    g = gy * wv
    s1 = 0 if rms else g.mean(-1, keepdim=True)
    s2 = (g * xh).mean(-1, keepdim=True)
    err_s = terms * U * g.abs().mean(-1, keepdim=True)
    err_s2 = (g.abs() * err_xh).mean(-1, keepdim=True) + terms * U * (g * xh).abs().mean(-1, keepdim=True)
    d = rstd * (g - s1 - xh * s2)
    err_d = rstd * (err_xh * (s2.abs() + err_s2) + xh.abs() * err_s2 + err_s) + 8 * terms * U * rstd * (
        g.abs() + g.abs().mean(-1, keepdim=True) + (xh * s2).abs()) + 2 * U * gt.abs()
    within(grads[1], d + gt, err_d, dtype)
    within(grads[0], (d + gt) * f, err_d * f + 2 * U * (d + gt).abs() * f, dtype)
    n = rows + 64
    within(grads[2], (gy * xh).sum(0), (gy.abs() * err_xh).sum(0) + n * U * (gy * xh).abs().sum(0), dtype)
    if not rms and has_bias:
        within(grads[3], gy.sum(0), n * U * gy.abs().sum(0), dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rms", [False, True], ids=["layer", "rms"])
@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 1), (7, 384), (61, 770), (33, 768), (300, 1024), (9, 1025), (5, 2048),
                                       (6, 2056), (3, 4100), (2, 8192), (4000, 40), (5000, 5)])
def test_residual_norm_forward_backward(dtype, rms, rows, cols):
    _norm_check(dtype, rows, cols, rms, 0.25)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rms", [False, True], ids=["layer", "rms"])
@pytest.mark.parametrize("use", [(True, True), (True, False), (False, True)], ids=["both", "y", "total"])
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_residual_norm_gradients_that_do_not_arrive(dtype, rms, use, p):
    _norm_check(dtype, 50, 256, rms, p, use=use)


def test_layer_norm_without_bias_and_wider_than_the_kernel():
    _norm_check(torch.bfloat16, 20, 128, False, 0.1, has_bias=False)
    _norm_check(torch.float32, 3, 8200, True, 0.1)  # PyTorch statement
    _norm_check(torch.float32, 3, 8200, False, 0.0)


def test_residual_norm_on_views_buffers_and_repeats():
    base = rand(30, 4, 512, dtype=torch.bfloat16)
    w = rand(256, dtype=torch.bfloat16, shift=1.0)
    for x, r in ((base[:, 1, :256], base[:, 2, 256:]), (base[:, 0, 1:257], base[:, 3, :256]), (base[:1, 0, :256].expand(30, 256),) * 2):
        a = add_rms_norm(x, r, w, 1e-6, dropout_p=0.2, seed=1)
        b = add_rms_norm(x.contiguous(), r.contiguous(), w, 1e-6, dropout_p=0.2, seed=1)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    out, leaves, (x, r, w, b, dy, dt) = _norm_case(torch.bfloat16, 5000, 768, False, 0.1)
    first = torch.autograd.grad(out, leaves, (dy, dt), retain_graph=True)
    for p, q in zip(first, torch.autograd.grad(out, leaves, (dy, dt), retain_graph=True)):
        assert torch.equal(p, q)
    for t in (w, b):
        t.main_grad = torch.ones(768, device="cuda")
    torch.autograd.backward(out, (dy, dt))
    assert w.grad is None and b.grad is None
    for t, g in zip((w, b), first[2:]):
        got = t.main_grad.double() - 1
        assert ((got - g.double()).abs() <= half(torch.bfloat16) * got.abs() + 2 * U * (1 + got.abs())).all()


def test_first_derivatives_with_a_graph_and_second_ones_refused():
    x, r, w = rand(9, 64), rand(9, 64, seed=1), rand(64, seed=2)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, total = add_rms_norm(x, r, w, 1e-6, dropout_p=0.2, seed=3)
    g = torch.ones_like(y, requires_grad=True)
    a = torch.autograd.grad((y, total), (x, r, w), (g, g), retain_graph=True)
    b = torch.autograd.grad((y, total), (x, r, w), (g, g), create_graph=True)
    assert all(torch.equal(p, q.detach()) for p, q in zip(a, b))
    with pytest.raises(RuntimeError):
        b[0].sum().backward()
    table = rand(20, 64).requires_grad_(True)
    out = scaled_embedding(torch.arange(9, device="cuda"), table)
    (d,) = torch.autograd.grad(out, (table,), g, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_dropout_and_residual_norm_draw_the_same_mask():
    x, r = rand(37, 640, dtype=torch.bfloat16), rand(37, 640, dtype=torch.bfloat16, seed=1)
    w = torch.ones(640, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(add_rms_norm(x, r, w, 1e-6, dropout_p=0.3, seed=8)[1], dropout_add(x, r, 0.3, 8))


# ---- attention with dropout ------------------------------------------------------------------------------------------------
@pytest.fixture(params=[64, 65, 128], ids=["kt64ws", "kt64", "kt128"])
def key_tile(request):
    from deberta_b200.ops.attention_cuda import set_backward_persistent, set_forward_key_tile

    old = set_forward_key_tile(request.param)
    old_bwd = set_backward_persistent({64: 1, 65: 0, 128: 3}[request.param])
    yield request.param
    set_forward_key_tile(old)
    set_backward_persistent(old_bwd)


def _mask(kind, B, S):
    if kind == "pad":
        keep = torch.ones(B, S, dtype=torch.bool, device="cuda")
        keep[0, S - S // 3:] = False
        if B > 1:
            keep[1] = False  # a row of the batch that sees nothing
        return {"key_keep": keep}
    if kind == "docs":
        doc = 1 + torch.arange(S, device="cuda").expand(B, S) // 150
        doc = torch.where(torch.arange(S, device="cuda") >= S - S // 10, 0, doc)
        return {"doc_ids": doc}
    return {}


def _attention_check(rotary, B, S, heads, mask, p, seed, dtype=torch.bfloat16, buckets=256, max_position=512):
    """Runs the operator and holds every output to a bound that follows its roundings: rotated q and k (or the position
    bias), the probabilities and their gradients in bf16, the output that the row term of the gradient is taken from."""
    d, span, h2 = 64, 256, half(torch.bfloat16)
    H = heads * d
    mk = lambda i, *s: rand(*s, dtype=dtype, seed=i, scale=0.7)  # noqa: E731
    q, k, v, do = (mk(i, B, S, H) for i in range(4))
    pos = [] if rotary else [mk(4, 2 * span, H), mk(5, 2 * span, H)]
    leaves = [t.requires_grad_(True) for t in (q, k, v, *pos)]
    kw = dict(_mask(mask, B, S), heads=heads, dropout_p=p, training=True, dropout_seed=seed)
    split = lambda t: t.detach().double().view(B, S, heads, d).permute(0, 2, 1, 3)  # noqa: E731
    merge = lambda t: t.permute(0, 2, 1, 3).reshape(B, S, H)  # noqa: E731
    Q, K, V, DO = split(q), split(k), split(v), split(do)
    if rotary:
        ang = torch.arange(S, device="cuda")[:, None] * (10000.0 ** (-torch.arange(0, d, 2, device="cuda") / d)).repeat_interleave(2)
        cos, sin = ang.cos().float(), ang.sin().float()
        out = rope_attention(q, k, v, cos, sin, rotary_dim=d, **kw)

        def turn(x, sign):
            c, s = cos.double(), sign * sin.double()
            other = torch.stack((-x[..., 1::2], x[..., 0::2]), -1).flatten(-2)
            return x * c + other * s, x.abs() * c.abs() + other.abs() * s.abs()

        Q, K = turn(Q, 1)[0], turn(K, 1)[0]
        scale = 1 / math.sqrt(d)
        raw = Q @ K.transpose(-1, -2)
        err_s = (2 * h2 + h2 * h2 + 80 * U) * (Q.abs() @ K.abs().transpose(-1, -2)) * scale
        bias = torch.zeros_like(raw)
    else:
        out = disentangled_attention(q, k, v, *pos, scale_factor=3, bucket_size=buckets, max_position=max_position,
                                     att_span=span, **kw)
        rel = relative_positions(S, S, buckets, max_position, device="cuda").clamp(-span, span)
        ic = (rel + span).clamp(0, 2 * span - 1).expand(B, heads, S, S)
        ip = (span - rel).clamp(0, 2 * span - 1).expand(B, heads, S, S)  # [q, k]
        PK, PQ = (t.detach().double().view(2 * span, heads, d).permute(1, 0, 2) for t in pos)
        scale = 1 / math.sqrt(3 * d)
        bias = (Q @ PK.transpose(-1, -2)).gather(-1, ic)
        part = (K @ PQ.transpose(-1, -2)).gather(-1, ip.transpose(-1, -2)).transpose(-1, -2)
        raw = Q @ K.transpose(-1, -2)
        # the two terms meet in bf16 (each may be rounded before their sum is)
        err_s = (h2 * (2 * bias.abs() + 2 * part.abs()) + 80 * U * (Q.abs() @ K.abs().transpose(-1, -2))) * scale
        bias = bias + part
    torch.cuda.synchronize()
    _lib.check_status()
    s = (raw + bias) * scale
    seen = torch.ones(B, 1, S, S, dtype=torch.bool, device="cuda")
    if "key_keep" in kw:
        seen = (kw["key_keep"][:, :, None] & kw["key_keep"][:, None, :])[:, None]
    if "doc_ids" in kw:
        seen = ((kw["doc_ids"][:, :, None] == kw["doc_ids"][:, None, :]) & (kw["doc_ids"] != 0)[:, :, None])[:, None]
    live = seen.any(-1, keepdim=True)
    P = torch.softmax(s.masked_fill(~seen, -1e300), -1) * live
    F = factor((B, heads, S, S), p, seed)
    M = (F > 0).double()
    top = (err_s * seen).amax(-1, keepdim=True)  # a row's scores are off by at most this, up to the row's sum as well
    err_p = torch.expm1(2 * top) + (S + 200) * U  # relative; (exponentials and the row sum in fp32)
    PD = P * F
    O = PD @ V
    err_o = (err_p + h2 + err_p * h2) * (PD @ V.abs()) + S * U * (PD @ V.abs())
    within(out, merge(O), merge(err_o), dtype)
    grads = torch.autograd.grad(out, leaves, do)
    _lib.check_status()
    e = err_p + h2 + err_p * h2
    DV = PD.transpose(-1, -2) @ DO
    within(grads[2], merge(DV), merge((e * PD).transpose(-1, -2) @ DO.abs()) + S * U * merge(PD.transpose(-1, -2) @ DO.abs()), dtype)
    dp = (DO @ V.transpose(-1, -2)) * F
    delta = (DO * O).sum(-1, keepdim=True)
    err_o = err_o + h2 * (O.abs() + err_o)
    err_delta = (DO.abs() * err_o).sum(-1, keepdim=True) + 80 * U * (DO * O).abs().sum(-1, keepdim=True)
    err_dp = 80 * U * (DO.abs() @ V.abs().transpose(-1, -2)) * F
    DS = P * (dp - delta) * scale
    err_ds = (P * (1 + err_p) * (err_delta + err_dp) + P * (dp - delta).abs() * err_p) * scale
    err_ds = err_ds + h2 * (DS.abs() + err_ds)
    size = DS.abs() + err_ds
    KT, QT = K.abs() * (1 + (h2 if rotary else 0)), Q.abs() * (1 + (h2 if rotary else 0))
    slip = (h2 if rotary else 0) + S * U
    DQ, DK = DS @ K, DS.transpose(-1, -2) @ Q
    eq = err_ds @ KT + slip * (size @ KT)
    ek = err_ds.transpose(-1, -2) @ QT + slip * (size.transpose(-1, -2) @ QT)
    if rotary:  # the gradients are rounded before they are turned back
        for got, want, err in ((grads[0], DQ, eq), (grads[1], DK, ek)):
            err = err + h2 * (want.abs() + err)
            back = turn(want, -1)[0]
            within(got, merge(back), merge(turn(err, -1)[1].abs() * 1.0), dtype)
        return
    fold = lambda t, i: torch.zeros(B, heads, S, 2 * span, dtype=torch.float64, device="cuda").scatter_add_(-1, i, t)  # noqa: E731
    ipt = ip.transpose(-1, -2)
    # the folded gradients are differences of fp32 prefix sums, rounded to bf16
    FK, FQ = fold(DS, ic), fold(DS.transpose(-1, -2), ipt)
    reach = 2 * S * U * size.sum(-1, keepdim=True)
    eFK = fold(err_ds, ic) + reach
    eFQ = fold(err_ds.transpose(-1, -2), ipt) + 2 * S * U * size.sum(-2)[..., None]
    eFK, eFQ = eFK + h2 * (FK.abs() + eFK), eFQ + h2 * (FQ.abs() + eFQ)
    T = 1024 * U + S * B * U
    within(grads[0], merge(DQ + FK @ PK), merge(eq + eFK @ PK.abs() + T * (FK.abs() @ PK.abs()) + h2 * (DQ.abs() + eq)), dtype)
    within(grads[1], merge(DK + FQ @ PQ), merge(ek + eFQ @ PQ.abs() + T * (FQ.abs() @ PQ.abs()) + h2 * (DK.abs() + ek)), dtype)
    for got, f, ef, x in ((grads[3], FK, eFK, Q), (grads[4], FQ, eFQ, K)):
        want = (f.transpose(-1, -2) @ x).sum(0).permute(1, 0, 2).reshape(2 * span, H)
        err = (ef.transpose(-1, -2) @ x.abs() + T * (f.abs().transpose(-1, -2) @ x.abs())).sum(0).permute(1, 0, 2).reshape(2 * span, H)
        within(got, want, err, dtype)


@pytest.mark.parametrize("B,S,heads,mask", [(2, 1, 1, "none"), (1, 2, 2, "none"), (2, 64, 1, "pad"), (3, 93, 3, "pad"), (1, 128, 2, "none"),
                                            (1, 200, 1, "docs"), (2, 513, 1, "docs"), (1, 640, 2, "none")])
@pytest.mark.parametrize("rotary", [True, False], ids=["rotary", "disentangled"])
def test_attention_with_dropout(rotary, B, S, heads, mask, key_tile):
    _attention_check(rotary, B, S, heads, mask, 0.2, 0x55AA55AA12345678)


def test_attention_with_dropout_over_a_row_of_the_batch_without_documents():
    q, k, v, g = (rand(2, 200, 128, dtype=torch.bfloat16, seed=i).requires_grad_(i < 3) for i in range(4))
    docs = torch.zeros(2, 200, dtype=torch.long, device="cuda")
    docs[1, :150] = 1 + torch.arange(150, device="cuda") // 40
    kw = dict(heads=2, rotary_dim=0, doc_ids=docs, dropout_p=0.2, training=True, dropout_seed=3)
    out = rope_attention(q, k, v, None, None, **kw)
    for t in (out, *torch.autograd.grad(out, (q, k, v), g)):
        assert not t[0].any() and not t[1, 150:].any() and t[1, :150].any()


@pytest.mark.parametrize("p", [0.01, 0.5, 0.9])
def test_attention_with_other_probabilities(p):
    _attention_check(True, 1, 300, 2, "none", p, 3)
    _attention_check(False, 1, 300, 2, "pad", p, 3)


def test_disentangled_attention_with_dropout_beyond_the_bias_mode():
    """Above 1024 tokens the position terms are gathered inside the kernels."""
    from deberta_b200.ops import attention_cuda

    old, attention_cuda.BIAS_MODE_MAX_SEQ = attention_cuda.BIAS_MODE_MAX_SEQ, 0
    try:
        _attention_check(False, 1, 256, 1, "pad", 0.2, 6)
        _attention_check(False, 1, 200, 2, "docs", 0.2, 6)
        _attention_check(False, 2, 77, 1, "none", 0.2, 6)
    finally:
        attention_cuda.BIAS_MODE_MAX_SEQ = old


def test_attention_with_dropout_at_lengths_of_the_gather_mode():
    _attention_check(False, 1, 1100, 1, "none", 0.1, 17)


def test_attention_with_dropout_over_a_map_that_the_bias_kernel_refuses():
    """Offsets 100 .. 127 on 100 buckets: the diagonal tile of 128 x 128 reaches from bucket -199 to 199, further than the tile
    kernel's 256 rows. Offsets without buckets do fit."""
    from deberta_b200.ops import attention_cuda

    _attention_check(False, 2, 300, 1, "pad", 0.2, 8, buckets=0, max_position=0)
    for S in (300, 300, 140):
        _attention_check(False, 2, S, 1, "pad", 0.2, 8, buckets=200, max_position=128)
    assert None in attention_cuda._TRAIN_TABLES.values()


def _near(got, want, share):
    assert (got.float() - want.float()).norm() <= share * want.float().norm()


@pytest.mark.parametrize("which", ["pos_k", "pos_q"])
@pytest.mark.parametrize("S", [90, 256])
def test_attention_with_dropout_and_one_position_table(which, S):
    """Against the fp32 statement with the same mask: a few bf16 roundings (2^-9 of a value on average) next to another mask's
    difference of the order of one."""
    from deberta_b200.ops.attention import disentangled_attention_reference

    q, k, v, g = (rand(2, S, 128, dtype=torch.bfloat16, seed=i).requires_grad_(i < 3) for i in range(4))
    tab = rand(512, 128, dtype=torch.bfloat16, seed=5).requires_grad_(True)
    pos = (tab, None) if which == "pos_k" else (None, tab)
    out = disentangled_attention(q, k, v, *pos, heads=2, scale_factor=2, bucket_size=256, max_position=512, att_span=256,
                                 dropout_p=0.2, training=True, dropout_seed=4)
    wide = [t.detach().float().requires_grad_(True) for t in (q, k, v, tab)]
    ref = disentangled_attention_reference(*wide[:3], *((wide[3], None) if which == "pos_k" else (None, wide[3])), heads=2,
                                           scale_factor=2, rel_pos=relative_positions(S, S, 256, 512, device="cuda"),
                                           att_span=256, dropout_p=0.2, training=True, dropout_seed=4)
    _near(out, ref, 0.02)
    for a, b in zip(torch.autograd.grad(out, (q, k, v, tab), g), torch.autograd.grad(ref, wide, g.float())):
        _near(a, b, 0.02)
    _lib.check_status()


@pytest.mark.parametrize("rotary_dim", [2, 18, 32, 64])
def test_rotary_attention_with_dropout_and_part_of_the_columns_turned(rotary_dim):
    from deberta_b200.ops.attention import rope_attention_reference

    B, S, heads = 2, 150, 2
    q, k, v, g = (rand(B, S, heads * 64, dtype=torch.bfloat16, seed=i).requires_grad_(i < 3) for i in range(4))
    ang = torch.arange(S, device="cuda")[:, None] * (100.0 ** (-torch.arange(0, rotary_dim, 2, device="cuda") / rotary_dim)).repeat_interleave(2)
    kw = dict(heads=heads, rotary_dim=rotary_dim, dropout_p=0.2, training=True, dropout_seed=torch.tensor([31], device="cuda"))
    out = rope_attention(q, k, v, ang.cos(), ang.sin(), **kw)
    wide = [t.detach().float().requires_grad_(True) for t in (q, k, v)]
    ref = rope_attention_reference(*wide, ang.cos(), ang.sin(), **kw)
    _near(out, ref, 0.02)
    for a, b in zip(torch.autograd.grad(out, (q, k, v), g), torch.autograd.grad(ref, wide, g.float())):
        _near(a, b, 0.02)


def test_attention_with_dropout_of_an_empty_batch():
    q = torch.zeros(0, 40, 128, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    tab = rand(512, 128, dtype=torch.bfloat16).requires_grad_(True)
    kw = dict(heads=2, dropout_p=0.2, training=True, dropout_seed=4)
    out = disentangled_attention(q, q, q, tab, tab, scale_factor=3, bucket_size=256, max_position=512, att_span=256, **kw)
    dq, dt = torch.autograd.grad(out, (q, tab), torch.zeros_like(out))
    assert out.shape == q.shape == dq.shape and not dt.any()
    assert rope_attention(q, q, q, None, None, rotary_dim=0, **kw).shape == q.shape


def test_an_overwritten_padding_mask_is_an_error():
    q = rand(1, 40, 64, dtype=torch.bfloat16).requires_grad_(True)
    keep = torch.ones(1, 40, dtype=torch.bool, device="cuda")
    out = rope_attention(q, q, q, None, None, heads=1, rotary_dim=0, key_keep=keep, dropout_p=0.2, training=True, dropout_seed=1)
    keep[0, 5] = False
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()


def test_attention_takes_ints_tensors_and_strided_projections():
    qkv = rand(2, 100, 3 * 128, dtype=torch.bfloat16)
    q, k, v = qkv.split(128, dim=-1)
    kw = dict(heads=2, rotary_dim=0, dropout_p=0.3, training=True)
    a = rope_attention(q, k, v, None, None, dropout_seed=12, **kw)
    b = rope_attention(q.contiguous(), k.contiguous(), v.contiguous(), None, None,
                       dropout_seed=torch.tensor([12], device="cuda"), **kw)
    assert torch.equal(a, b)
    assert torch.equal(rope_attention(q, k, v, None, None, heads=2, rotary_dim=0, dropout_p=1e-7, training=True, dropout_seed=1),
                       rope_attention(q, k, v, None, None, heads=2, rotary_dim=0))
    with pytest.raises(ValueError):
        rope_attention(q, k, v, None, None, dropout_seed=torch.tensor([12]), **kw)


def test_attention_falls_back_to_the_same_mask_where_the_kernels_do_not_reach():
    """Head dimension 32 and fp32 take the PyTorch statement; the same fp32 inputs in bf16 take the kernel."""
    q, k, v = (rand(1, 70, 128, dtype=torch.bfloat16, seed=i) for i in range(3))
    kw = dict(rotary_dim=0, dropout_p=0.4, training=True, dropout_seed=21)
    a = rope_attention(q, k, v, None, None, heads=2, **kw).float()
    b = rope_attention(q.float(), k.float(), v.float(), None, None, heads=2, **kw)
    assert (a - b).norm() < 0.02 * b.norm()
    assert rope_attention(q, k, v, None, None, heads=4, **kw).shape == q.shape


# ---- embedding -----------------------------------------------------------------------------------------------------------
def _ids(kind, n, vocab):
    g = torch.Generator(device="cuda").manual_seed(n + vocab)
    ids = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    if kind == "one":
        ids.fill_(vocab - 1)
    elif kind == "hot":
        ids[torch.rand(n, device="cuda", generator=g) < 0.6] = vocab // 2
    elif kind == "runs":
        ids = torch.arange(n, device="cuda") // 45 % vocab
    return ids


def _embedding_check(ids, table, scale, pad, g):
    cols = table.shape[1]
    out = scaled_embedding(ids, table, scale, padding_idx=pad)
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    within(out, table.detach().double()[ids.long()] * s32, 0.0, table.dtype)
    (d,) = torch.autograd.grad(out, (table,), g, retain_graph=True)
    flat, rows = ids.reshape(-1).long(), g.reshape(-1, cols).double()
    if pad is not None:
        rows = rows * (flat != pad)[:, None]
    zero = torch.zeros(table.shape, dtype=torch.float64, device="cuda")
    want, size = zero.index_add(0, flat, rows) * s32, zero.index_add(0, flat, rows.abs()) * abs(s32)
    count = torch.bincount(flat, minlength=table.shape[0])[:, None].double()
    within(d, want, (count + 2) * U * size, table.dtype)
    assert torch.equal(d[count[:, 0] == 0], torch.zeros_like(d[count[:, 0] == 0]))
    assert torch.equal(d, torch.autograd.grad(out, (table,), g, retain_graph=True)[0])
    table.main_grad = torch.full(table.shape, 0.5, dtype=torch.float32, device="cuda")
    out.backward(g)
    assert table.grad is None
    within(table.main_grad, want + 0.5, (count + 3) * U * (size + 0.5), torch.float32)
    del table.main_grad


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 1000, 9001])
@pytest.mark.parametrize("kind", ["uniform", "one", "hot", "runs"])
def test_embedding_forward_backward(dtype, n, kind):
    vocab, cols = 1000, 264
    table = rand(vocab, cols, dtype=dtype).requires_grad_(True)
    _embedding_check(_ids(kind, n, vocab), table, 1.7, 3, rand(n, cols, dtype=dtype, seed=1))


@pytest.mark.parametrize("vocab,cols", [(1, 8), (2, 1), (7, 770), (511, 8), (512, 96), (4096, 1024), (128100, 24), (262143, 8), (262144, 8),
                                        (1 << 20, 3)])
def test_embedding_of_other_tables(vocab, cols):
    table = rand(vocab, cols, dtype=torch.bfloat16).requires_grad_(True)
    _embedding_check(_ids("uniform", 3000, vocab), table, 32.0, None, rand(3000, cols, dtype=torch.bfloat16, seed=1))


@pytest.mark.parametrize("n", [1, 255, 256, 257, 511, 512, 513])
@pytest.mark.parametrize("kind", ["uniform", "one", "hot"])
@pytest.mark.parametrize("vocab,cols", [(1, 520), (592, 8), (593, 257), (128100, 136), (592 * 8192 + 1, 1)])
def test_embedding_on_either_side_of_the_one_launch_path(n, kind, vocab, cols):
    table = rand(vocab, cols, dtype=torch.float16).requires_grad_(True)
    _embedding_check(_ids(kind, n, vocab), table, 3.0, None, rand(n, cols, dtype=torch.float16, seed=1))
    if vocab == 593:
        _embedding_check(_ids(kind, n, vocab), table, 3.0, 7, rand(n, 300, dtype=torch.float16, seed=1)[:, 9:9 + cols])


def test_embedding_of_many_tokens():
    table = rand(5000, 16).requires_grad_(True)
    _embedding_check(_ids("hot", 400_000, 5000), table, 1.0, 0, rand(400_000, 16, seed=1))


def test_embedding_ids_and_gradients_in_other_layouts():
    table = rand(100, 64, dtype=torch.bfloat16).requires_grad_(True)
    ids = _ids("uniform", 60, 100).view(3, 20)
    g = rand(3, 20, 128, dtype=torch.bfloat16, seed=2)[:, :, 32:96]
    _embedding_check(ids.int(), table, 2.0, None, g)
    _embedding_check(ids.t(), table, 2.0, 5, g.transpose(0, 1))
    _embedding_check(ids, table, 2.0, 5, g[:, :, :1].expand(3, 20, 64))


def test_embedding_ids_out_of_range_are_clamped_and_left_out():
    table = rand(10, 16).requires_grad_(True)
    ids = torch.tensor([-1, 3, 10, 1 << 40, -(1 << 40), 3], device="cuda")
    out = scaled_embedding(ids, table)
    assert torch.equal(out, table.detach()[torch.tensor([0, 3, 9, 9, 0, 3], device="cuda")])
    (d,) = torch.autograd.grad(out, (table,), torch.ones_like(out))
    want = torch.zeros_like(d)
    want[3] = 2
    assert torch.equal(d, want)


def test_lookup_is_reproducible_under_deterministic_algorithms():
    table, delta = (rand(50, 128, dtype=torch.bfloat16, seed=s).requires_grad_(True) for s in range(2))
    ids, g = _ids("hot", 5000, 50), rand(5000, 128, dtype=torch.bfloat16, seed=3)
    rows = g.double() * (ids != 0)[:, None]
    zero = torch.zeros(50, 128, dtype=torch.float64, device="cuda")
    want, size = zero.index_add(0, ids, rows), zero.index_add(0, ids, rows.abs())
    seen = []
    torch.use_deterministic_algorithms(True)
    try:
        for _ in range(3):
            for t in (table, delta):
                t.main_grad = torch.zeros(50, 128, device="cuda")
            embedding_lookup(ids, table, delta, padding_idx=0).backward(g)
            assert torch.equal(table.main_grad, delta.main_grad)
            seen.append(table.main_grad)
    finally:
        torch.use_deterministic_algorithms(False)
    assert torch.equal(seen[0], seen[1]) and torch.equal(seen[0], seen[2])
    within(seen[0], want, 5000 * U * size, torch.float32)


def test_deterministic_lookup_takes_gradients_of_any_layout():
    table = rand(50, 128, dtype=torch.bfloat16).requires_grad_(True)
    ids = _ids("uniform", 40, 50)
    torch.use_deterministic_algorithms(True)
    try:
        for g in (rand(1, 128, dtype=torch.bfloat16).expand(40, 128), rand(40, 200, dtype=torch.bfloat16)[:, 3:131],
                  rand(128, 40, dtype=torch.bfloat16).t()):
            table.main_grad = torch.zeros(50, 128, device="cuda")
            embedding_lookup(ids, table).backward(g)
            want = torch.zeros(50, 128, dtype=torch.float64, device="cuda").index_add(0, ids, g.double())
            within(table.main_grad, want, 40 * U * torch.zeros_like(want).index_add(0, ids, g.double().abs()), torch.float32)
        table.main_grad = torch.zeros(50, 128, device="cuda")
        embedding_lookup(ids[:1], table).backward(rand(1, 1, dtype=torch.bfloat16).expand(1, 128))
        assert int((table.main_grad != 0).any(1).sum()) == 1
    finally:
        torch.use_deterministic_algorithms(False)


# ---- writes stay inside the outputs -----------------------------------------------------------------------------------------
MARK = -61440.0  # exact in every type, and further out than any output here


class _Canary:
    """Outputs inside larger buffers of a value that must survive around them, and be gone inside."""

    def __init__(self):
        self.all = []

    def __call__(self, n, dtype, lead=64):
        buf = torch.full((n + lead + 256,), MARK, dtype=dtype, device="cuda")
        self.all.append((buf, lead, n))
        return buf[lead:lead + n]

    def check(self):
        torch.cuda.synchronize()
        for buf, lead, n in self.all:
            assert (buf[:lead] == MARK).all() and (buf[lead + n:] == MARK).all()
            assert (buf[lead:lead + n] != MARK).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols,lead", [(3, 8, 64), (5, 770, 64), (37, 768, 64), (37, 768, 65), (2, 1025, 64), (600, 24, 72), (1, 1, 1)])
def test_row_kernels_write_inside_their_outputs(dtype, rows, cols, lead):
    from deberta_b200.ops.dropout import DTYPE_CODES, _dropout_kernel, inverse_keep
    from deberta_b200.ops.norm import _add_norm_bwd, _add_norm_fwd, _parts

    code, t, st = DTYPE_CODES[dtype], 20000, _lib.raw_stream()
    x, r, dy, dt = (rand(rows, cols, dtype=dtype, seed=i, shift=3.0) for i in range(4))
    w, b = rand(cols, dtype=dtype, shift=2.0), rand(cols, dtype=dtype, shift=2.0)
    c, n = _Canary(), rows * cols
    seed = (None, 5, t, inverse_keep(t))
    out = c(n, dtype, lead)
    _dropout_kernel(x.data_ptr(), cols, r.data_ptr(), cols, out.data_ptr(), rows, cols, code, *seed, st)
    total, y, stats = c(n, dtype, lead), c(n, dtype, lead), c(2 * rows, torch.float32)
    _add_norm_fwd(x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), b.data_ptr(), total.data_ptr(), y.data_ptr(),
                  stats.data_ptr() + 4 * rows, stats.data_ptr(), rows, cols, 1e-6, code, *seed, st)
    dx, dr, dw, db = c(n, dtype, lead), c(n, dtype, lead), c(cols, dtype), c(cols, dtype)
    parts = c(2 * _parts(rows, cols) * cols, torch.float32)
    _add_norm_bwd(dy.data_ptr(), total.data_ptr(), dt.data_ptr(), w.data_ptr(), stats.data_ptr() + 4 * rows, stats.data_ptr(),
                  dx.data_ptr(), dr.data_ptr(), parts.data_ptr(), dw.data_ptr(), None, db.data_ptr(), None, 1, rows, cols, code,
                  *seed, st)
    c.check()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens,vocab,cols", [(3, 5, 7), (200, 700, 24), (257, 1000, 9), (3000, 777, 264), (5000, 3, 40)])
def test_embedding_kernels_write_inside_their_outputs(dtype, tokens, vocab, cols):
    from deberta_b200.ops.dropout import DTYPE_CODES
    from deberta_b200.ops.embedding import _gather, _sorted_sums, _workspace_bytes

    code, st = DTYPE_CODES[dtype], _lib.raw_stream()
    table, dout = rand(vocab, cols, dtype=dtype, shift=9.0), rand(tokens, cols, dtype=dtype, shift=9.0)
    ids = _ids("hot", tokens, vocab)
    c = _Canary()
    out = c(tokens * cols, dtype)
    _gather(ids.data_ptr(), table.data_ptr(), out.data_ptr(), tokens, cols, vocab, 1.0, code, st)
    size = _workspace_bytes(tokens, cols, vocab)
    work = c(size // 4, torch.float32) if size else None
    grad = c(vocab * cols, dtype)
    _sorted_sums(ids.data_ptr(), dout.data_ptr(), cols, tokens, cols, vocab, -1, 1.0, code, grad.data_ptr(), None, None,
                 None if work is None else work.data_ptr(), st)
    if work is not None:
        torch.cuda.synchronize()
        buf, lead, n = c.all.pop(1)  # (parts of the scratch stay as they were)
        assert (buf[:lead] == MARK).all() and (buf[lead + n:] == MARK).all()
    c.check()


# ---- together, as a training step uses them --------------------------------------------------------------------------------
def _step(ids, table, wqkv, w, b, seeds, g):
    x = scaled_embedding(ids, table, 8.0, padding_idx=0)
    x = dropout(x, 0.1, seeds[0:1])
    q, k, v = (x @ wqkv).split(128, dim=-1)
    a = disentangled_attention(q, k, v, None, None, heads=2, scale_factor=1, bucket_size=0, max_position=0, att_span=0,
                               key_keep=ids != 0, dropout_p=0.1, training=True, dropout_seed=seeds[1:2])
    y, total = add_layer_norm(a, x, w, b, 1e-6, dropout_p=0.1, seed=seeds[2:3])
    # (detached: an eager autograd graph of the same leaves must not be alive while a backward pass is captured)
    return [y.detach(), *torch.autograd.grad((y, total), (table, wqkv, w, b), (g, g))]


def test_operators_together_captured_and_replayed_with_new_seeds():
    ids = _ids("uniform", 2 * 70, 300).view(2, 70)
    ids[0, 50:] = 0
    table = rand(300, 128, dtype=torch.bfloat16, scale=0.1).requires_grad_(True)
    wqkv = rand(128, 384, dtype=torch.bfloat16, scale=0.1, seed=1).requires_grad_(True)
    w, b = (rand(128, dtype=torch.bfloat16, seed=s, shift=1.0).requires_grad_(True) for s in (2, 3))
    g = rand(2, 70, 128, dtype=torch.bfloat16, seed=4)
    seeds = torch.tensor([1, 2, 3], device="cuda")
    args = (ids, table, wqkv, w, b, seeds, g)
    want = {}
    for base in (1, 40, 1):
        seeds.copy_(torch.tensor([base, base + 1, base + 2]))
        want[base] = _step(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(*args)
    for base in (40, 1, 40):
        seeds.copy_(torch.tensor([base, base + 1, base + 2]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[base][0])  # the forward pass is the same bits
        for got, ref in zip(held[1:], want[base][1:]):  # (the query gradient is summed by fp32 atomics)
            assert (got.float() - ref.float()).norm() <= 2 * half(torch.bfloat16) * ref.float().norm()
    _lib.check_status()
    assert not torch.equal(want[1][0], want[40][0])


def test_operators_run_on_the_current_stream():
    x = rand(2000, 768, dtype=torch.bfloat16)
    w = torch.ones(768, dtype=torch.bfloat16, device="cuda")
    want = add_rms_norm(dropout(x * 2, 0.2, 3), x, w, 1e-6, dropout_p=0.1, seed=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            got = add_rms_norm(dropout(x * 2, 0.2, 3), x, w, 1e-6, dropout_p=0.1, seed=4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_compiled_operators_run_the_kernels(backend):
    x, r, g = (rand(2, 130, 128, dtype=torch.bfloat16, seed=i) for i in range(3))
    w = rand(128, dtype=torch.bfloat16, seed=3, shift=1.0).requires_grad_(True)
    tab = rand(512, 128, dtype=torch.bfloat16, seed=4).requires_grad_(True)
    x.requires_grad_(True)
    seed = torch.tensor([7], device="cuda")
    ang = torch.arange(130, device="cuda")[:, None] * torch.ones(64, device="cuda") * 0.1
    cos, sin = ang.cos(), ang.sin()

    def f(x, seed):
        a = disentangled_attention(x, x, x, tab, tab, heads=2, scale_factor=3, bucket_size=256, max_position=512, att_span=256,
                                   dropout_p=0.2, training=True, dropout_seed=seed)
        a = rope_attention(a, x, a, cos, sin, heads=2, rotary_dim=64, dropout_p=0.1, training=True, dropout_seed=12)
        y, total = add_rms_norm(dropout(a, 0.3, seed), r, w, 1e-6, dropout_p=0.2, seed=seed)
        return y + dropout_add(total, x, 0.1, -3)

    want = f(x, seed)
    ref = torch.autograd.grad(want, (x, w, tab), g)
    torch._dynamo.reset()
    before = _lib.LAUNCH_COUNT
    got = torch.compile(f, backend=backend, fullgraph=True)(x, seed)
    grads = torch.autograd.grad(got, (x, w, tab), g)
    assert _lib.LAUNCH_COUNT - before >= 12
    _lib.check_status()
    # (the sum outside the operators and the rotation's own node round at other places; the query gradients use atomics)
    _near(got, want, 0.01)
    for a, b in zip(grads, ref):
        _near(a, b, 0.02)
