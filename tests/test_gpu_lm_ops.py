"""Attention with score modifiers, head norms with rotation, the token embedding and the distillation loss on the GPU, against
plain formulas in 64 bits.

Tolerances, derived before any run.  u = finfo.eps / 2 is half a step of the output's type (bf16 2^-8): every output is rounded
once, so |error| <= u |value| plus what the kernel's arithmetic leaves:
  attention   P and dS are rounded to bf16 in front of their products, and O is, from which delta is formed; scores and
              statistics are fp32 (an exponent off by x 2^-24 for scores |x| < 100, a sum, an exp2, a reciprocal of one ulp
              each: below 2^-12 of P together).  So
                O    within (u + 2^-12) P |V| + u |O|,              dV within (u + 2^-12) P^T |dO| + u |dV|,
                dS   within (u + 2^-12) |dS| + P f scale ((u + 2^-12) |dO| . |O| + 2^-12 |dO| . |V|)   =: E,
                dQ   within E |K| + u |dQ|,                          dK within E^T |Q| + u |dK|,
              f = 1 - tanh^2 <= 1 (1 without a cap; its own error, some 2^-21, is in the last term).
  heads       fp32 from bf16: a rotated channel is a sum of two products, each within 2^-20 of its size after the norm.
  embedding   y is one product rounded once, so exact; n terms added in fp32: within (n + 2) 2^-24 of the sum of their sizes.
  distillation  q within 2^-16 (an exponent |y| < 100 off by 2^-24 relative, the same for the sum's logarithm, plus the sum).
"""
import math

import pytest
import torch

from distributedpytorch_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U16, U32 = 2.0 ** -8, 2.0 ** -24


def _rand(*shape, seed=0, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _within(got, ref, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    over = (got - ref).abs() - tol
    assert (over <= 0).all(), f"{what}: {(over > 0).sum().item()} of {over.numel()} outside, by up to {over.max().item():.3g} (largest value {ref.abs().max().item():.3g})"


# ------------------------------------------------------------------------------------------------------- attention
def _attend_ref(q, k, v, do, causal=True, scale=None, softcap=0.0, slopes=None, documents=None, prefix=None):
    """(value, tolerance) of out, dq, dk, dv in 64 bits on the CPU, one head at a time."""
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    e = 2.0 ** -12
    res = {n: (torch.zeros(s, dtype=torch.float64), torch.zeros(s, dtype=torch.float64)) for n, s in
           (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", k.shape))}
    i = torch.arange(T)
    for b in range(B):
        see = i[None, :] <= i[:, None] if causal else torch.ones(T, T, dtype=torch.bool)
        if prefix is not None:
            see = see | (i[None, :] < int(prefix[b]))
        if documents is not None:
            d = documents[b]
            see = see & (d[:, None] == d[None, :]) & (d >= 0)[:, None]
        any_ = see.any(1, keepdim=True)
        for h in range(Hq):
            kh = h * Hkv // Hq
            Q, K, V, O_ = (t[b, :, n].double() for t, n in ((q, h), (k, kh), (v, kh), (do, h)))
            if documents is not None:
                pad = (documents[b] < 0)[:, None]
                Q, K, V, O_ = (t.masked_fill(pad, 0.0) for t in (Q, K, V, O_))
            x = Q @ K.t() * scale
            f = torch.ones_like(x)
            if softcap:
                x = torch.tanh(x / softcap)
                f = 1 - x * x
                x = x * softcap
            if slopes is not None:
                x = x - slopes[h].double() * (i[:, None] - i[None, :]).abs()
            x = x.masked_fill(~see, -math.inf).masked_fill(~any_, 0.0)
            P = torch.softmax(x, 1) * any_ * see
            out = P @ V
            dP = O_ @ V.t()
            dS = P * (dP - (P * dP).sum(1, keepdim=True)) * f * scale
            E = (U16 + e) * dS.abs() + P * f * scale * ((U16 + e) * (O_.abs() * out.abs()).sum(1, keepdim=True) + e * (O_.abs() @ V.abs().t()))
            for name, n, val, tol in (("out", h, out, (U16 + e) * (P @ V.abs())), ("dq", h, dS @ K, E @ K.abs()),
                                      ("dk", kh, dS.t() @ Q, E.t() @ Q.abs()), ("dv", kh, P.t() @ O_, (U16 + e) * (P.t() @ O_.abs()))):
                res[name][0][b, :, n] += val
                res[name][1][b, :, n] += tol
    return {n: (val, tol + U16 * val.abs() + 1e-30) for n, (val, tol) in res.items()}


def _docs(kind, B, T):
    g = torch.Generator().manual_seed(T)
    if kind == "sorted":          # documents of random lengths, the last row padded at its end
        d = (torch.rand(B, T, generator=g) < 1 / 40).long().cumsum(1)
        d[-1, T - T // 5:] = -1
    elif kind == "ones":          # every token a document of its own
        d = torch.arange(T).expand(B, T).clone()
    elif kind == "shuffled":      # the same numbers again and again, in no order, padding among them
        d = torch.randint(-1, 3, (B, T), generator=g)
    elif kind == "padded":        # one row of nothing but padding
        d = torch.arange(T).expand(B, T) // 50
        d = d.clone()
        d[0] = -5
    return d.to(torch.int32)


ATTEND = [
    # B, T, Hq, Hkv, D, mode
    (1, 1, 1, 1, 64, {}), (2, 2, 3, 1, 128, {}), (1, 31, 2, 2, 64, {}), (1, 33, 2, 1, 8, {}), (2, 63, 2, 2, 40, dict(causal=False)),
    (1, 64, 4, 2, 128, {}), (1, 65, 2, 2, 96, dict(softcap=5.0)), (2, 127, 2, 2, 64, dict(slopes=True)), (1, 128, 2, 2, 64, dict(docs="sorted")),
    (1, 129, 3, 3, 72, dict(docs="shuffled")), (2, 200, 4, 1, 64, dict(docs="sorted", softcap=8.0, slopes=True, prefix=True)),
    (3, 257, 4, 2, 128, dict(docs="padded")), (2, 193, 2, 2, 64, dict(prefix=True)), (2, 300, 6, 2, 128, dict(prefix=True, softcap=20.0)),
    (1, 257, 2, 2, 64, dict(docs="ones")), (2, 256, 2, 1, 128, dict(docs="shuffled", causal=False)), (1, 320, 2, 2, 64, dict(causal=False, slopes=True)),
    (1, 383, 8, 1, 128, dict(slopes=True)), (1, 70, 2, 2, 128, dict(scale=0.5, gain=4.0)), (1, 4300, 1, 1, 64, dict(docs="sorted")),
    (1, 140, 2, 2, 80, dict(docs="sorted", causal=False, softcap=10.0)), (4, 513, 2, 2, 64, dict()), (1, 1000, 4, 4, 128, dict(docs="sorted", prefix=True)),
]


def _attend_inputs(B, T, Hq, Hkv, D, mode):
    kw = dict(mode)
    gain = kw.pop("gain", 1.0)
    q, k, v, do = (_rand(B, T, h, D, seed=s + T, std=gain if s < 2 else 1.0) for s, h in enumerate((Hq, Hkv, Hkv, Hq)))
    if kw.pop("slopes", False):
        kw["slopes"] = torch.tensor([0.3 * (-0.4) ** h for h in range(Hq)])       # of both signs
    docs = kw.pop("docs", None)
    if docs:
        kw["documents"] = _docs(docs, B, T)
    if kw.pop("prefix", False):
        kw["prefix"] = torch.tensor([T // 2, -3, T + 7, T // 3][:B], dtype=torch.int32)
    return q, k, v, do, kw


def _on(kw):
    return {n: x.to(DEV) if torch.is_tensor(x) else x for n, x in kw.items()}


@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention_forward_and_backward(case):
    B, T, Hq, Hkv, D, mode = ATTEND[case]
    q, k, v, do, kw = _attend_inputs(B, T, Hq, Hkv, D, mode)
    ref = _attend_ref(q, k, v, do, **kw)
    leaf = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaf, **_on(kw))
    grads = torch.autograd.grad(out, leaf, do.to(DEV))
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        _within(got, *ref[name], name)
    with torch.no_grad():
        assert torch.equal(ops.attention(*leaf, **_on(kw)), out)                   # alone, and the same bits again


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("softcap,gain,slopes", [(255.0, 2.0, False), (257.0, 2.0, True), (1e3, 2.0, False), (1e5, 2.0, True), (1e7, 2.0, False), (1e11, 2.0, True),
                                                 (300.0, 10.0, False), (2000.0, 10.0, False)])
def test_attention_caps_far_from_the_scores(softcap, gain, slopes, D):
    """Caps up to 256 leave a score 2e-7 of the cap off, wider ones 3e-7 of the score itself; raw scores of deviation gain^2 are off by
    another 2^-23 of their size, and none here is past 700: together below the 2^-12 of P that the bounds count."""
    q, k, v, do, kw = _attend_inputs(1, 200, 4, 2, D, dict(softcap=softcap, gain=gain, slopes=slopes))
    ref = _attend_ref(q, k, v, do, **kw)
    leaf = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaf, **_on(kw))
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaf, do.to(DEV)))):
        _within(got, *ref[name], name)


@pytest.mark.parametrize("softcap,sign", [(2.0, -1), (2.0, 1), (0.5, -1), (1e-11, -1), (1e-11, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_scores_all_at_one_end_of_the_cap(D, softcap, sign):
    """Raw scores around 8 caps of one sign (but for the two smallest caps, where they lie past any exponential): 1 - tanh^2 is some
    1e-7 of 1 and all that the scores' gradients are made of.  Each raw score is within 2^-22 of its size, 8 caps, so 1 - tanh^2 within
    16 2^-22: inside the 2^-12 that the bounds count."""
    B, T, H = 1, 140, 2
    mean = math.sqrt(8 * min(max(softcap, 0.5), 2.0) / math.sqrt(D))
    q, k = ((mean * (1 + 0.1 * _rand(B, T, H, D, seed=s, dtype=torch.float32))).to(torch.bfloat16) for s in (1, 2))
    k = k * sign
    v, do = (_rand(B, T, H, D, seed=s) for s in (3, 4))
    ref = _attend_ref(q, k, v, do, softcap=softcap)
    leaf = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaf, softcap=softcap)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaf, do.to(DEV)))):
        _within(got, *ref[name], name)


def test_attention_reads_strided_views_in_place():
    B, T, Hq, Hkv, D = 2, 150, 4, 2, 64
    pack = _rand(B, T, Hq + 2 * Hkv, D, seed=5).to(DEV)
    do = _rand(B, T, Hq, D, seed=6).to(DEV)
    q, k, v = pack[:, :, :Hq], pack[:, :, Hq:Hq + Hkv], pack[:, :, Hq + Hkv:]
    want = ops.attention(*(t.contiguous() for t in (q, k, v)))

    def grads(ts):
        ts = [t.detach().requires_grad_() for t in ts]
        return torch.autograd.grad(ops.attention(*ts), ts, do)
    base = grads([t.contiguous() for t in (q, k, v)])
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    flat = torch.empty(B * T * Hq * D + 8, dtype=torch.bfloat16, device=DEV)
    odd = flat[1:1 + B * T * Hq * D].view(B, T, Hq, D).copy_(q)                   # off 16 bytes: copied by the call
    last = [torch.stack((t, t), 4)[..., 0] for t in (q, k, v)]                     # last axis not contiguous: copied
    for ts in ((q, k, v), heads_first, (odd, k, v), last):
        assert torch.equal(ops.attention(*ts), want)
        for a, b in zip(grads(ts), base):
            assert torch.equal(a, b)
    one = k[:, :1].expand(B, T, Hkv, D)                                            # stride 0 over the tokens
    assert torch.equal(ops.attention(q, one, one), ops.attention(q, one.contiguous(), one.contiguous()))
    qs, ks, vs = (t.detach().requires_grad_() for t in (q, k, v))                  # an output gradient that is not contiguous
    for a, b in zip(torch.autograd.grad(ops.attention(qs, ks, vs), (qs, ks, vs), do.transpose(1, 2).contiguous().transpose(1, 2)), base):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_padding_holds_anything(D):
    T = 300
    q, k, v, do = (_rand(1, T, 2, D, seed=s).to(DEV) for s in range(4))
    docs = torch.arange(T, dtype=torch.int32)[None] // 90
    docs[0, 100:140] = -1
    docs[0, 290:] = -9
    docs = docs.to(DEV)
    pad = docs[0] < 0

    def go(ts, g):
        ts = [t.clone().requires_grad_() for t in ts]
        out = ops.attention(*ts, documents=docs, softcap=9.0)
        return (out.detach(), *torch.autograd.grad(out, ts, g))
    base = go((q, k, v), do)
    for x in base:
        assert (x[:, pad] == 0).all()
    filled = [t.clone() for t in (q, k, v, do)]
    for t, bad in zip(filled, (math.nan, math.inf, -math.inf, math.nan)):
        t[:, pad] = bad
    for a, b in zip(go(filled[:3], filled[3]), base):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_rows_of_padding_leave_their_neighbours_alone(D):
    """Workgroups that visit no tile end at once; those that take their place on the chip find nothing of theirs."""
    B, T = 96, 200
    q, k, v, do = (_rand(B, T, 2, D, seed=s).to(DEV) for s in range(4))
    docs = torch.zeros(B, T, dtype=torch.int32, device=DEV)
    docs[::2] = -1

    def go(rows):
        ts = [t[rows].detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*ts, documents=docs[rows])
        return (out.detach(), *torch.autograd.grad(out, ts, do[rows]))
    alone = go(slice(1, None, 2))
    for _ in range(3):
        for a, b in zip(go(slice(None)), alone):
            assert torch.equal(a[1::2], b) and (a[::2] == 0).all()


def test_attention_single_visible_key_has_no_score_gradient():
    q, k, v, do = (_rand(3, 1, 2, 128, seed=s, std=3.0).to(DEV) for s in range(4))
    leaf = [t.requires_grad_() for t in (q, k, v)]
    for kw in ({}, dict(softcap=3.0, slopes=torch.ones(2, device=DEV))):
        out = ops.attention(*leaf, **kw)
        dq, dk, dv = torch.autograd.grad(out, leaf, do)
        assert torch.equal(out, v) and torch.equal(dv, do) and (dq == 0).all() and (dk == 0).all()


def test_attention_nan_in_a_seen_row_shows():
    q, k, v = (_rand(1, 70, 1, 64, seed=s).to(DEV) for s in range(3))
    v[0, 10, 0, 3] = math.nan
    out = ops.attention(q, k, v)
    assert torch.isnan(out[0, 10:, 0, 3]).all()


# -------------------------------------------------------------------------------------------------- heads
HEADS = [
    # B, T, Hq, Hkv, D, R, interleaved, norm, positions
    (1, 1, 1, 1, 64, 64, False, True, None), (2, 7, 3, 1, 128, 128, True, True, "batch"), (1, 130, 12, 12, 64, 64, False, True, None),
    (2, 33, 4, 2, 96, 48, False, True, "row"), (1, 5, 2, 2, 8, 0, False, True, None), (3, 9, 8, 1, 256, 256, False, True, "far"),
    (1, 17, 5, 5, 40, 16, True, True, None), (2, 12, 6, 2, 128, 64, False, False, "far"), (1, 40, 2, 1, 32, 32, True, False, "batch"),
    (1, 3000, 2, 1, 64, 64, False, True, None), (1, 20, 17, 3, 80, 80, False, True, "batch"),
]


@pytest.mark.parametrize("case", range(len(HEADS)))
def test_heads_forward_and_backward(case):
    B, T, Hq, Hkv, D, R, inter, norm, pos = HEADS[case]
    eps = 1e-5
    x = _rand(B, T, (Hq + 2 * Hkv) * D, seed=case, std=1.5)
    w = [1 + 0.3 * _rand(D, seed=50 + i, dtype=torch.float32) for i in range(2)] if norm else [None, None]
    freq = ops.rotary_frequencies(R) if R else None
    at = {None: None, "row": torch.arange(T) * 3 + 1, "batch": torch.randint(0, 5000, (B, T), generator=torch.Generator().manual_seed(case)),
          "far": torch.randint(-(1 << 33), 1 << 33, (B, T), generator=torch.Generator().manual_seed(case))}[pos]
    gs = [_rand(B, T, h, D, seed=60 + i) for i, h in enumerate((Hq, Hkv, Hkv))]
    kw = dict(eps=eps, interleaved=inter)
    # 64-bit reference and the sizes its terms have
    X = x.double().view(B, T, Hq + 2 * Hkv, D)
    angle = None if not R else (torch.arange(T).expand(B, T) if at is None else at.expand(B, T)).double()[..., None] * freq

    def pairs():
        i = torch.arange(R // 2)
        return (2 * i, 2 * i + 1) if inter else (i, i + R // 2)

    def turn(t, sign):
        if not R:
            return t, t.abs()
        a, b = pairs()
        c, s = angle.cos()[:, :, None], sign * angle.sin()[:, :, None]
        y, size = t.clone(), t.abs()
        y[..., a], y[..., b] = t[..., a] * c - t[..., b] * s, t[..., b] * c + t[..., a] * s
        size[..., a] = size[..., b] = t[..., a].abs() + t[..., b].abs()
        return y, size
    e = 2.0 ** -20
    want, dwant, dws = [], [], []
    for h, wt, g in ((X[:, :, :Hq], w[0], gs[0]), (X[:, :, Hq:Hq + Hkv], w[1], gs[1])):
        r = (h.square().mean(3, keepdim=True) + eps).rsqrt() if norm else torch.ones(())
        n = h * r
        y, size = turn(n * (wt.double() if norm else 1.0), 1.0)
        want.append((y, U16 * y.abs() + 2 * e * size + 1e-30))
        gr, gsize = turn(g.double(), -1.0)
        if norm:
            gw, gws = gr * wt.double(), gsize * wt.double().abs()
            m = (gw * n).mean(3, keepdim=True)
            dx = r * (gw - n * m)
            dwant.append((dx, U16 * dx.abs() + 4 * e * r * (gws + n.abs() * (gws * n.abs()).mean(3, keepdim=True)) + 1e-30))
            count = B * T * h.shape[2]
            dws.append(((gr * n).sum((0, 1, 2)), (2 * e + count * U32) * (gsize * n.abs()).sum((0, 1, 2))))
        else:
            dwant.append((gr, U16 * gr.abs() + 2 * e * gsize + 1e-30))
    dwant.append((gs[2].double(), torch.zeros_like(gs[2], dtype=torch.float64)))
    leaf = [t.to(DEV).requires_grad_() for t in (x, *w) if t is not None]
    on = dict(kw, inv_freq=None if freq is None else freq.to(DEV), positions=None if at is None else at.to(DEV))
    if norm:
        on.update(q_weight=leaf[1], k_weight=leaf[2])
    q, k, v = ops.qk_norm_rotary(leaf[0], Hq, Hkv, **on)
    _within(q, *want[0], "q")
    _within(k, *want[1], "k")
    assert torch.equal(v.cpu(), x.view(B, T, -1, D)[:, :, Hq + Hkv:])
    grads = torch.autograd.grad((q, k, v), leaf, [g.to(DEV) for g in gs])
    ref = torch.cat([a for a, _ in dwant], 2).view(B, T, -1), torch.cat([b for _, b in dwant], 2).view(B, T, -1)
    _within(grads[0], *ref, "dqkv")
    for name, got, (val, tol) in zip(("dqw", "dkw"), grads[1:], dws):
        _within(got, val, tol, name)


def test_heads_only_one_output_used_and_strided_input():
    x = _rand(2, 6, 5 * 32 + 8, seed=1).to(DEV)[:, :, 8:]                         # a view: copied by the call
    w = torch.ones(32, device=DEV)
    a = x.detach().requires_grad_()
    b = x.detach().contiguous().requires_grad_()
    f = ops.rotary_frequencies(32, device=DEV)
    for n in range(3):
        qa, qb = (ops.qk_norm_rotary(t, 3, 1, q_weight=w, k_weight=w, inv_freq=f)[n] for t in (a, b))
        assert torch.equal(qa, qb)
        (ga,), (gb,) = (torch.autograd.grad(y.float().square().sum(), t) for y, t in ((qa, a), (qb, b)))
        assert torch.equal(ga, gb) and ga.abs().sum() > 0


@pytest.mark.parametrize("Hq,Hkv,D", [(2, 1, 64), (3, 2, 40), (1, 1, 256)])
def test_heads_without_eps(Hq, Hkv, D):
    """eps = 0 divides by a head's own root mean square alone; lanes that hold no such head (values, places past the last one) must
    not bring their 1 / 0 into the gains' gradients.  n is within 2^-20, as with eps; a sum of T H terms within its terms' sizes."""
    T = 9
    x, gs = _rand(1, T, (Hq + 2 * Hkv) * D, seed=5), [_rand(1, T, h, D, seed=6 + i) for i, h in enumerate((Hq, Hkv, Hkv))]
    w = [1 + 0.3 * _rand(D, seed=9 + i, dtype=torch.float32) for i in range(2)]
    xs, ws = x.to(DEV).requires_grad_(), [t.to(DEV).requires_grad_() for t in w]
    got = torch.autograd.grad(ops.qk_norm_rotary(xs, Hq, Hkv, q_weight=ws[0], k_weight=ws[1], eps=0.0), (xs, *ws), [g.to(DEV) for g in gs])
    X = x.double().view(1, T, -1, D)
    n = X / X.square().mean(3, keepdim=True).sqrt()
    for i, (a, b) in enumerate(((0, Hq), (Hq, Hq + Hkv))):
        terms = gs[i].double() * n[:, :, a:b]
        _within(got[1 + i], terms.sum((0, 1, 2)), 2.0 ** -18 * terms.abs().sum((0, 1, 2)), "dw")
        gw = gs[i].double() * w[i].double()
        r = n[:, :, a:b] / X[:, :, a:b]
        d = (gw * n[:, :, a:b]).mean(3, keepdim=True)
        ref = r * (gw - n[:, :, a:b] * d)
        size = r.abs() * (gw.abs() + n[:, :, a:b].abs() * (gw * n[:, :, a:b]).abs().mean(3, keepdim=True))
        _within(got[0].view(1, T, -1, D)[:, :, a:b], ref, U16 * ref.abs() + 2.0 ** -18 * size, "dqkv")
    assert torch.equal(got[0].view(1, T, -1, D)[:, :, Hq + Hkv:].cpu(), gs[2])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_heads_value_gradients_stay_out_of_the_key_gain(bad, interleaved):
    """Whatever the values' gradients hold reaches the projection's gradient alone, where it stands."""
    Hq, Hkv, D = 3, 2, 64
    x = _rand(2, 9, (Hq + 2 * Hkv) * D, seed=1).to(DEV).requires_grad_()
    w = [(1 + 0.3 * _rand(D, seed=2 + i, dtype=torch.float32)).to(DEV).requires_grad_() for i in range(2)]
    gs = [_rand(2, 9, h, D, seed=4 + i).to(DEV) for i, h in enumerate((Hq, Hkv, Hkv))]
    f = ops.rotary_frequencies(D, device=DEV)

    def grads():
        return torch.autograd.grad(ops.qk_norm_rotary(x, Hq, Hkv, q_weight=w[0], k_weight=w[1], inv_freq=f, interleaved=interleaved), (x, *w), gs)
    want = grads()
    gs[2][1, 4, 1, 7] = bad
    dx, dqw, dkw = grads()
    assert torch.equal(dqw, want[1]) and torch.equal(dkw, want[2])
    want[0].view(2, 9, -1, D)[1, 4, Hq + Hkv + 1, 7] = bad
    assert torch.equal(dx.nan_to_num(nan=1e30), want[0].nan_to_num(nan=1e30))


def test_heads_empty():
    w = torch.ones(16, device=DEV, requires_grad=True)
    x = torch.zeros(2, 0, 48, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    q, k, v = ops.qk_norm_rotary(x, 1, q_weight=w, k_weight=w)
    assert q.shape == k.shape == v.shape == (2, 0, 1, 16)
    dx, dw = torch.autograd.grad(q.sum() + v.sum(), (x, w))
    assert dx.shape == x.shape and (dw == 0).all()


# -------------------------------------------------------------------------------------------------- embedding
EMBED = [
    # tokens shape, V, C, kind
    ((1,), 1, 8, "uniform"), ((2, 100), 512, 128, "text"), ((3, 77), 130, 40, "text"), ((700,), 3, 16, "uniform"), ((2000,), 50304, 64, "text"),
    ((5000,), 100, 24, "one"), ((64,), 40000, 8, "uniform"), ((513,), 200000, 8, "uniform"), ((3, 1100), 7, 2056, "pad"), ((0,), 10, 8, "uniform"),
    ((4096,), 600, 520, "text"),
]


def _tokens(shape, V, kind, dtype):
    g = torch.Generator().manual_seed(V)
    n = math.prod(shape)
    if kind == "text":
        t = (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * math.log(V)) - 1).long()
    elif kind == "one":
        t = torch.full((n,), V - 1)
        t[::97] = 3
    else:
        t = torch.randint(0, V, (n,), generator=g)
        if kind == "pad":
            t[::3] = -1
            t[5::11] = V
            t[7::13] = 2 ** 31 - 1
    return t.view(shape).to(dtype)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("case", range(len(EMBED)))
def test_token_embedding_forward_and_backward(case, dtype):
    shape, V, C, kind = EMBED[case]
    tok = _tokens(shape, V, kind, dtype)
    w, dy, scale = _rand(V, C, seed=1, dtype=torch.float32), _rand(*shape, C, seed=2), 3.7
    lp = w.to(torch.bfloat16)
    live = (tok >= 0) & (tok < V)
    at = torch.where(live, tok, 0).long()
    want = torch.where(live[..., None], lp[at].float() * scale, 0.0).to(torch.bfloat16)
    flat, rows = at[live], dy.double()[live]
    ref = torch.zeros(V, C, dtype=torch.float64).index_add_(0, flat, rows) * scale
    size = torch.zeros(V, C, dtype=torch.float64).index_add_(0, flat, rows.abs()) * scale
    count = torch.bincount(flat, minlength=V)[:, None].double()
    wd, td = w.to(DEV).requires_grad_(), tok.to(DEV)
    for shadow in (None, lp.to(DEV)):
        y = ops.token_embedding(td, wd, shadow, scale=scale)
        assert torch.equal(y.detach().cpu(), want)
        (dw,) = torch.autograd.grad(y, wd, dy.to(DEV))
        _within(dw, ref, (count + 2) * U32 * size, "dw")
        (again,) = torch.autograd.grad(ops.token_embedding(td, wd, shadow, scale=scale), wd, dy.to(DEV))
        assert torch.equal(dw, again)


@pytest.mark.parametrize("kind,V,C,n", [("runs", 4000, 16, 0), ("runs", 300, 136, 0), ("one", 90, 8, 30000), ("low", 50304, 8, 40000),
                                        ("low", 20, 24, 20000), ("late", 600, 8, 16384)])
def test_token_embedding_gradient_of_frequent_tokens(kind, V, C, n):
    """Ids that come in every number around 16 and 64, so that their entries end just in front of, on and behind the places where the
    sums are cut, and lists in which a wave meets more of its workgroup's ids than it can note at once.  n terms in fp32, in any order:
    within (n + 2) 2^-24 of the sum of their sizes."""
    g = torch.Generator().manual_seed(V)
    if kind == "runs":
        tok = torch.cat([torch.full((c,), i * 7 % V) for i, c in enumerate((1, 15, 16, 17, 30, 32, 33, 48, 63, 64, 65, 79, 80, 81, 127, 128, 129, 16, 16, 200))])
        tok = tok[torch.randperm(tok.numel(), generator=g)]
    elif kind == "late":                                           # nothing, then a few ids of one workgroup without a pause
        tok = torch.full((n,), -1)
        tok[n // 2:] = torch.randint(0, 8, (n - n // 2,), generator=g)
    elif kind == "one":
        tok = torch.full((n,), 5)
        tok[::1009] = 6
    else:
        tok = (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * math.log(V)) - 1).long()
    dy = _rand(tok.numel(), C, seed=3)
    w = torch.zeros(V, C, device=DEV, requires_grad=True)
    dw, again = (torch.autograd.grad(ops.token_embedding(tok.to(DEV), w), w, dy.to(DEV))[0] for _ in range(2))
    assert torch.equal(dw, again)
    live = tok >= 0
    at, rows = tok[live], dy.double()[live]
    count = torch.bincount(at, minlength=V)[:, None].double()
    zero = torch.zeros(V, C, dtype=torch.float64)
    _within(dw, zero.index_add(0, at, rows), (count + 2) * U32 * zero.index_add(0, at, rows.abs()), "dw")


def test_token_embedding_adds_into_an_installed_gradient_buffer():
    from distributedpytorch_amd.ops import sink
    V, C = 60, 32
    w = torch.nn.Parameter(_rand(V, C, seed=1, dtype=torch.float32).to(DEV))
    tok = _tokens((3, 50), V, "text", torch.int64).to(DEV)
    dy = _rand(3, 50, C, seed=2).to(DEV)
    (want,) = torch.autograd.grad(ops.token_embedding(tok, w, scale=0.5), w, dy)
    buf = torch.full((V * C,), 2.0, device=DEV)
    told = []
    s = sink.GradSink([w], {id(w): buf}, told.append)
    try:
        ops.token_embedding(tok, w, scale=0.5).backward(dy)
    finally:
        s.uninstall()
    assert w.grad is None and len(told) == 1 and told[0] is w
    torch.testing.assert_close(buf.view(V, C), want + 2.0, rtol=2 * U32, atol=0)
    unnamed = torch.ones(V, dtype=torch.bool, device=DEV)
    unnamed[tok.flatten()] = False
    assert unnamed.any() and (buf.view(V, C)[unnamed] == 2.0).all()


# -------------------------------------------------------------------------------------------------- distillation
DISTILL = [
    # N, V, ld, K, dtype, tau, std
    (1, 1, 1, 1, torch.float32, 1.0, 1.0), (3, 500, 512, 8, torch.float32, 1.0, 3.0), (5, 501, 501, 33, torch.bfloat16, 2.0, 3.0),
    (7, 50257, 50304, 32, torch.bfloat16, 2.0, 4.0), (2, 65536, 65536, 1024, torch.bfloat16, 0.5, 1.0), (2, 70001, 70008, 64, torch.bfloat16, 1.0, 2.0),
    (3, 32768, 32768, 5, torch.float32, 4.0, 5.0), (2, 100001, 100001, 200, torch.float32, 1.5, 2.0), (4, 9, 16, 9, torch.bfloat16, 1.0, 30.0),
    (300, 77, 80, 3, torch.float32, 1.0, 1.0), (2, 33000, 33000, 7, torch.float32, 1.0, 2.0), (2, 8191, 8192, 600, torch.bfloat16, 3.0, 2.0),
]


def _teacher(N, V, K, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] if V >= K else torch.randint(0, V, (K,), generator=g) for _ in range(N)])
    t = torch.randn(N, K, generator=g) * 2
    if K > 2:
        ids[0, 1] = ids[0, 0]                       # twice the same
        t[0, 2] = -math.inf                         # a dead entry
    if N > 1:
        ids[1, K // 2:] = -1                        # a short list (or none at all)
        ids[1, K - 1] = V                           # one past the classes
    return ids, t


@pytest.mark.parametrize("ids32", [False, True])
@pytest.mark.parametrize("case", range(len(DISTILL)))
def test_distillation_forward_and_backward(case, ids32):
    N, V, ld, K, dtype, tau, std = DISTILL[case]
    z = _rand(N, ld, seed=case, std=std, dtype=dtype)
    z[:, V:] = math.nan                             # padding columns hold anything
    ids, t = _teacher(N, V, K, case)
    live = (ids >= 0) & (ids < V) & (t > -math.inf)
    rows = live.any(1)
    zz = z[:, :V].double() / tau
    logq = torch.log_softmax(zz, 1)
    logp = torch.log_softmax((t.double() / tau).masked_fill(~live, -math.inf).masked_fill(~rows[:, None], 0.0), 1)
    p = logp.exp() * live
    at = torch.where(live, ids, 0)
    lq = logq.gather(1, at)
    term = torch.where(live, p * (logp - lq), 0.0)
    loss = tau * tau * term.sum() / N
    size = tau * tau * torch.where(live, p * (logp.abs() + lq.abs() + 1), 0.0).sum() / N
    full = torch.zeros(N, V, dtype=torch.float64).scatter_add_(1, at, p)
    q = logq.exp() * rows[:, None]
    d = torch.zeros(N, ld, dtype=torch.float64)
    d[:, :V] = (q - full) * tau / N
    tol = torch.zeros_like(d)
    u = U16 if dtype == torch.bfloat16 else U32
    tol[:, :V] = 2.0 ** -16 * (q + full) * tau / N + u * d[:, :V].abs()
    tol += 1e-38                                    # below the normal numbers
    zd, tt = z.to(DEV).requires_grad_(), t.to(DEV)
    ii = ids.to(torch.int32 if ids32 else torch.int64).to(DEV)
    kw = dict(temperature=tau, n_classes=V)
    got = ops.distillation_loss(zd, ii, tt, **kw)
    _within(got, loss, 2.0 ** -16 * size, "loss")
    with torch.no_grad():
        assert torch.equal(ops.distillation_loss(zd, ii, tt, **kw), got)
    (dz,) = torch.autograd.grad(got, zd, retain_graph=True)
    _within(dz, d, tol, "dlogits")
    (d3,) = torch.autograd.grad(got, zd, torch.tensor(3.0, device=DEV), retain_graph=True)   # another upstream, the same node again
    _within(d3, 3 * d, 3 * tol + 3 * u * d.abs() + tol, "3 dlogits")
    (d1,) = torch.autograd.grad(got, zd)
    assert torch.equal(d1, dz)
    assert torch.equal(z[:, :V], zd.detach().cpu()[:, :V])


@pytest.mark.parametrize("V", [700, 5000, 33000, 110000])
def test_distillation_does_not_feel_a_rows_offset(V):
    """Logits of deviation 2 around 30,000 and -30,000: what is left of each class counts from the row's maximum, so the bounds are those
    of the zero-mean rows (an exponent |y| < 100 off by 2^-24 relative), in all four builds."""
    N, K, tau = 4, 20, 1.5
    z = _rand(N, V, seed=V, std=2.0, dtype=torch.float32) + torch.tensor([0.0, 3e4, -3e4, 1e3])[:, None]
    ids, t = _teacher(N, V, K, V)
    live = (ids >= 0) & (ids < V) & (t > -math.inf)
    at = torch.where(live, ids, 0)
    logq = torch.log_softmax(z.double() / tau, 1)
    logp = torch.log_softmax((t.double() / tau).masked_fill(~live, -math.inf), 1)
    p, lq = logp.exp() * live, logq.gather(1, at)
    loss = tau * tau * torch.where(live, p * (logp - lq), 0.0).sum() / N
    size = tau * tau * torch.where(live, p * (logp.abs() + lq.abs() + 1), 0.0).sum() / N
    full = torch.zeros(N, V, dtype=torch.float64).scatter_add_(1, at, p)
    d = (logq.exp() - full) * tau / N
    zd = z.to(DEV).requires_grad_()
    got = ops.distillation_loss(zd, ids.to(DEV), t.to(DEV), temperature=tau)
    _within(got, loss, 2.0 ** -16 * size, "loss")
    _within(torch.autograd.grad(got, zd)[0], d, 2.0 ** -16 * (logq.exp() + full) * tau / N + U32 * d.abs() + 1e-38, "dlogits")


@pytest.mark.parametrize("V", [40, 700, 5000, 33000, 110000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_rows_of_the_lowest_values(V, dtype):
    """Rows whose classes all hold the type's lowest value, or numbers far below any others, are rows like any: a row of one value is
    uniform, and one of two values far apart is uniform over the higher ones.  q is then a quotient of exact numbers: bounds as for any
    row.  Masked places in an ordinary row are zeros."""
    low = torch.finfo(dtype).min
    z = torch.empty(6, V, dtype=dtype)
    z[0], z[1], z[2], z[3] = low, -2e30, 1e37, low
    z[3, ::4] = -1e35
    z[4] = _rand(V, seed=V, dtype=dtype)
    z[4, 1::3] = low
    z[5] = low
    z[5, 1] = 3.0
    ids = torch.tensor([[0, 4], [4, 8], [8, 12], [0, 16], [0, 6], [1, 1]])
    t = torch.tensor([[0.5, -0.5]]).repeat(6, 1)
    logq = torch.log_softmax(z.double(), 1)
    logp = torch.log_softmax(t.double(), 1)
    p, lq = logp.exp(), logq.gather(1, ids)
    loss = (p * (logp - lq)).sum() / 6
    size = (p * (logp.abs() + lq.abs() + 1)).sum() / 6
    full = torch.zeros(6, V, dtype=torch.float64).scatter_add_(1, ids, p)
    d = (logq.exp() - full) / 6
    zd = z.to(DEV).requires_grad_()
    got = ops.distillation_loss(zd, ids.to(DEV), t.to(DEV))
    _within(got, loss, 2.0 ** -16 * size, "loss")
    _within(torch.autograd.grad(got, zd)[0], d, 2.0 ** -16 * (logq.exp() + full) / 6 + (U16 if dtype == torch.bfloat16 else U32) * d.abs() + 1e-38, "dlogits")


@pytest.mark.parametrize("V", [700, 5000, 110000, 220000])
@pytest.mark.parametrize("weight", [0.3, 1.0, 0.0, -7.0])
def test_distillation_gradient_for_any_upstream_is_rounded_once(V, weight):
    """bf16: half a step of the weighted gradient and the kernel's 2^-16, not a second half step for the weight."""
    N, K, tau = 3, 20, 2.0
    z = _rand(N, V, seed=V, std=2.0)
    ids, t = _teacher(N, V, K, V)
    live = (ids >= 0) & (ids < V) & (t > -math.inf)
    p = torch.softmax((t.double() / tau).masked_fill(~live, -math.inf), 1) * live
    full = torch.zeros(N, V, dtype=torch.float64).scatter_add_(1, torch.where(live, ids, 0), p)
    q = torch.softmax(z.double() / tau, 1)
    d = (q - full) * tau / N * weight
    zd = z.to(DEV).requires_grad_()
    got = ops.distillation_loss(zd, ids.to(DEV), t.to(DEV), temperature=tau)
    g = torch.tensor(weight, device=DEV)
    grads = [torch.autograd.grad(got, zd, g, retain_graph=True)[0] for _ in range(2)]
    assert torch.equal(grads[0], grads[1])
    _within(grads[0], d, 2.0 ** -16 * (q + full) * tau / N * abs(weight) + U16 * d.abs() + 1e-38, "dlogits")


@pytest.mark.parametrize("weight", [1.0, 0.3])
def test_distillation_keeps_its_gradient_where_saved_tensor_hooks_see_it(weight):
    """Offloading moves all that the node keeps, the written gradient among it; hooks that hold on to what they were given find it
    unchanged; a checkpoint forms it again."""
    from torch.utils.checkpoint import checkpoint
    N, V = 64, 4096
    z = _rand(N, V, seed=1, std=2.0).to(DEV).requires_grad_()
    ids, t = (x.to(DEV) for x in _teacher(N, V, 20, 1))
    g = torch.tensor(weight, device=DEV)

    def loss():
        return ops.distillation_loss(z, ids, t, temperature=2.0)
    (want,) = torch.autograd.grad(loss(), z, g)
    held = []

    def hold(x):
        held.append((x, x.detach().clone()))
        return x
    with torch.autograd.graph.saved_tensors_hooks(hold, lambda x: x):
        one = loss()
    assert sum(x.shape == (N, V) for x, _ in held) == 2                            # the logits and the gradient
    for _ in range(2):
        assert torch.equal(torch.autograd.grad(one, z, g, retain_graph=True)[0], want)
    assert all(torch.equal(x, y) for x, y in held)
    held.clear()
    del one
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        one = loss()
    assert torch.cuda.memory_allocated() - before < N * V
    assert torch.equal(torch.autograd.grad(one, z, g)[0], want)
    assert torch.equal(torch.autograd.grad(checkpoint(loss, use_reentrant=False), z, g)[0], want)


@pytest.mark.parametrize("weight", [1.0, 0.3])
def test_distillation_off_16_bytes_and_without_rows(weight):
    """Logits that begin anywhere are copied by the call; no rows give no loss."""
    N, V = 5, 300
    ids, t = (x.to(DEV) for x in _teacher(N, V, 12, 2))
    flat = _rand(N * V + 8, seed=3).to(DEV)
    g = torch.tensor(weight, device=DEV)
    odd = flat[1:1 + N * V].view(N, V).detach().requires_grad_()
    assert odd.data_ptr() % 16 and odd.is_contiguous()
    even = odd.detach().clone().requires_grad_()
    a, b = (ops.distillation_loss(z, ids, t) for z in (odd, even))
    assert torch.equal(a, b)
    for _ in range(2):
        assert torch.equal(*(torch.autograd.grad(y, z, g, retain_graph=True)[0] for y, z in ((a, odd), (b, even))))
    none = torch.zeros(0, V, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    loss = ops.distillation_loss(none, ids[:0], t[:0])
    assert loss.item() == 0.0 and torch.autograd.grad(loss, none, g)[0].shape == (0, V)


def test_distillation_gradient_against_differences():
    N, V, K, tau = 6, 300, 12, 2.0
    z = _rand(N, V, seed=3, std=2.0, dtype=torch.float32).to(DEV).requires_grad_()
    ids, t = (x.to(DEV) for x in _teacher(N, V, K, 5))
    loss = ops.distillation_loss(z, ids, t, temperature=tau)
    (d,) = torch.autograd.grad(loss, z)
    step = _rand(N, V, seed=9, dtype=torch.float32).to(DEV)
    h = 0.05                                        # third-order remainder h^2 / 6 |f'''| against fp32 noise 2^-22 |loss| / h: both under 1e-3 of the slope
    with torch.no_grad():
        up, down = (ops.distillation_loss(z + s * h * step, ids, t, temperature=tau) for s in (1, -1))
    slope = (d.double() * step.double()).sum().item()
    assert abs((up - down).item() / (2 * h) - slope) <= 2e-3 * (d.double().abs() * step.double().abs()).sum().item()


def test_distillation_non_finite_logits_show_in_their_row_only():
    z = _rand(3, 64, seed=1, dtype=torch.float32)
    z[0, 5], z[1, 7] = math.nan, -math.inf
    zd = z.to(DEV).requires_grad_()
    ids, t = torch.tensor([[1, 2], [3, 4], [5, 6]], device=DEV), torch.zeros(3, 2, device=DEV)
    (d,) = torch.autograd.grad(ops.distillation_loss(zd, ids, t), zd)
    assert torch.isnan(d[0]).all() and torch.isfinite(d[1:]).all() and d[1, 7] == 0
    ids[0] = -1                                     # a row without a teacher: whatever it holds
    loss = ops.distillation_loss(zd, ids, t)
    (d,) = torch.autograd.grad(loss, zd)
    assert torch.isfinite(loss) and (d[0] == 0).all()


# -------------------------------------------------------------------------------------------------- all of them
def _passes():
    """One training pass through each operator, as closures over fixed inputs that return every output and gradient."""
    docs = _docs("sorted", 2, 200).to(DEV)
    pre = torch.tensor([20, 130], dtype=torch.int32, device=DEV)
    q, k, v, do = (_rand(2, 200, h, 64, seed=s).to(DEV) for s, h in enumerate((4, 2, 2, 4)))
    q, k, v = (t.requires_grad_() for t in (q, k, v))

    def attend():
        out = ops.attention(q, k, v, documents=docs, prefix=pre, softcap=10.0)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), do))
    x = _rand(2, 200, 8 * 64, seed=7).to(DEV).requires_grad_()
    w1, w2 = (torch.linspace(0.5, 1.5, 64, device=DEV).requires_grad_() for _ in range(2))
    f = ops.rotary_frequencies(64, device=DEV)

    def heads():
        y = ops.qk_norm_rotary(x, 4, 2, q_weight=w1, k_weight=w2, inv_freq=f)
        return (*(t.detach().clone() for t in y), *torch.autograd.grad(y, (x, w1, w2), (do, do[:, :, :2].contiguous(), do[:, :, 2:])))
    tok = _tokens((2, 1200), 900, "text", torch.int64).to(DEV)
    tab = _rand(900, 64, seed=8, dtype=torch.float32).to(DEV).requires_grad_()
    lp = tab.detach().to(torch.bfloat16)
    dy = _rand(2, 1200, 64, seed=9).to(DEV)

    def embed():
        y = ops.token_embedding(tok, tab, lp, scale=8.0)
        return (y.detach(), *torch.autograd.grad(y, tab, dy))
    z = _rand(40, 1000, seed=10).to(DEV).requires_grad_()
    ids, t = (a.to(DEV) for a in _teacher(40, 1000, 20, 11))

    def distil():
        loss = ops.distillation_loss(z, ids, t, temperature=2.0)
        return (loss.detach(), *torch.autograd.grad(loss, z))
    return {"attend": attend, "heads": heads, "embed": embed, "distil": distil}


@pytest.mark.parametrize("which", ["attend", "heads", "embed", "distil"])
def test_pass_on_another_stream_and_in_replayed_graphs(which):
    go = _passes()[which]
    want = [t.clone() for t in go()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = go()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):                              # two graphs, replayed in turn with eager work between
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = go()
        graphs.append((graph, outs))
    for _ in range(3):
        for graph, outs in graphs:
            graph.replay()
        eager = go()
        torch.cuda.synchronize()
        for outs in [o for _, o in graphs] + [eager]:
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
        for _, outs in graphs:
            for t in outs:
                t.fill_(7)                          # a replay has to write everything again


def _large_passes():
    """As `_passes`, through the builds that long and wide inputs take."""
    q, k, v, do = (_rand(1, 1100, h, 128, seed=s).to(DEV) for s, h in enumerate((8, 2, 2, 8)))
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    slopes = torch.linspace(0.01, 0.2, 8, device=DEV)

    def parts():                                    # key heads' gradients by parts
        out = ops.attention(q, k, v, slopes=slopes)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), do))
    tok = torch.zeros(24000, dtype=torch.int32)     # more of one workgroup's tokens than a wave notes at once
    tok[::7] = torch.arange(len(tok[::7]), dtype=torch.int32) % 8
    tok = tok.to(DEV)
    tab = _rand(50, 64, seed=8, dtype=torch.float32).to(DEV).requires_grad_()
    dy = _rand(24000, 64, seed=9).to(DEV)

    def often():
        y = ops.token_embedding(tok, tab, scale=0.5)
        return (y.detach(), *torch.autograd.grad(y, tab, dy))
    passes = {"parts": parts, "often": often}
    for name, V in (("held", 20001), ("lds", 70001), ("again", 110000)):
        z = _rand(5, V, seed=V, dtype=torch.float32).to(DEV).requires_grad_()
        ids, t = (a.to(DEV) for a in _teacher(5, V, 20, 11))

        def distil(z=z, ids=ids, t=t):
            loss = ops.distillation_loss(z, ids, t, temperature=2.0)
            return (loss.detach(), *torch.autograd.grad(loss, z))
        passes[name] = distil
    return passes


@pytest.mark.parametrize("which", ["parts", "often", "held", "lds", "again"])
def test_large_pass_on_two_streams_at_once_and_in_a_replayed_graph(which):
    go = _large_passes()[which]
    want = [t.clone() for t in go()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):                              # nothing waits between the two: each call has its own workspace
        for s in streams:
            with torch.cuda.stream(s):
                got.append(go())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        outs = go()
    for _ in range(3):
        graph.replay()
        eager = go()
        torch.cuda.synchronize()
        got += [[t.clone() for t in outs], eager]
        for t in outs:
            t.fill_(7)
    for one in got:
        for a, b in zip(one, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["attend", "heads", "embed", "distil"])
def test_second_backward_through_a_kept_graph(which):
    """The same gradient again, also after the first one was changed in place."""
    x = {"attend": lambda: _rand(1, 50, 2, 64), "heads": lambda: _rand(1, 5, 192), "embed": lambda: _rand(9, 8, dtype=torch.float32),
         "distil": lambda: _rand(3, 20)}[which]().to(DEV).requires_grad_()
    y = {"attend": lambda: ops.attention(x, x, x), "heads": lambda: ops.qk_norm_rotary(x, 1, inv_freq=ops.rotary_frequencies(64, device=DEV))[0],
         "embed": lambda: ops.token_embedding(torch.tensor([1, 2, 1], device=DEV), x),
         "distil": lambda: ops.distillation_loss(x, torch.tensor([[1], [2], [3]], device=DEV), torch.zeros(3, 1, device=DEV))}[which]()
    g = torch.full_like(y, 0.5)
    (first,) = torch.autograd.grad(y, x, g, retain_graph=True)
    kept = first.clone()
    first.fill_(3)
    for _ in range(2):
        (again,) = torch.autograd.grad(y, x, g, retain_graph=True)
        assert torch.equal(again, kept)


@pytest.mark.parametrize("which", ["attend", "heads", "embed", "distil"])
def test_no_second_derivative(which):
    x = {"attend": lambda: _rand(1, 5, 2, 64), "heads": lambda: _rand(1, 5, 192), "embed": lambda: _rand(9, 8, dtype=torch.float32),
         "distil": lambda: _rand(3, 20)}[which]().to(DEV).requires_grad_()
    y = {"attend": lambda: ops.attention(x, x, x), "heads": lambda: ops.qk_norm_rotary(x, 1, inv_freq=ops.rotary_frequencies(64, device=DEV))[0],
         "embed": lambda: ops.token_embedding(torch.tensor([1, 2], device=DEV), x),
         "distil": lambda: ops.distillation_loss(x, torch.tensor([[1], [2], [3]], device=DEV), torch.zeros(3, 1, device=DEV))}[which]()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(y.float().sum(), x, create_graph=True)


def test_gpu_refusals():
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    for bad in ((b(1, 4, 2, 136),) * 3, (b(1, 4, 2, 12),) * 3):
        with pytest.raises(ValueError):
            ops.attention(*bad)
    with pytest.raises(TypeError):
        ops.attention(*(torch.zeros(1, 4, 2, 64, device=DEV),) * 3)
    with pytest.raises(ValueError):
        ops.attention(b(1, 4, 2, 64), b(1, 4, 2, 64), b(1, 4, 2, 64), documents=torch.zeros(1, 4, dtype=torch.int32))
    w = torch.ones(64, device=DEV)
    with pytest.raises(TypeError):
        ops.qk_norm_rotary(b(1, 4, 192).float(), 1, q_weight=w, k_weight=w)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(b(1, 4, 3 * 264), 1, inv_freq=ops.rotary_frequencies(64, device=DEV))
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(b(1, 4, 192), 1, inv_freq=ops.rotary_frequencies(24, device=DEV))
    tok = torch.zeros(3, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError):
        ops.token_embedding(tok, torch.zeros(4, 12, device=DEV))
    with pytest.raises(TypeError):
        ops.token_embedding(tok, b(4, 16))
    with pytest.raises(ValueError):
        ops.token_embedding(tok, torch.zeros(4, 16, device=DEV), b(4, 8))
    with pytest.raises(ValueError):
        ops.token_embedding(tok.cpu(), torch.zeros(4, 16, device=DEV))
    z, ids = b(2, 2000), torch.zeros(2, 1025, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError):
        ops.distillation_loss(z, ids, torch.zeros(2, 1025, device=DEV))
    with pytest.raises(TypeError):
        ops.distillation_loss(z, ids[:, :3], torch.zeros(2, 3, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        ops.distillation_loss(z.half(), ids[:, :3], torch.zeros(2, 3, device=DEV))


def test_a_small_decoder_trains_through_all_four():
    """Packed rows through embedding, projection, head norms with rotation, attention and the distillation loss: loss and
    gradients against the same composition of the plain paths in fp32 on the CPU.  About 20 roundings to bf16 in a row, each some
    2^-9 of the result at random: under 3 % of a gradient's norm."""
    B, T, V, C, Hq, Hkv, D, K = 2, 160, 400, 128, 4, 2, 32, 6
    table, wqkv, wo = (_rand(*s, seed=i, std=0.05, dtype=torch.float32) for i, s in enumerate(((V, C), ((Hq + 2 * Hkv) * D, C), (C, Hq * D))))
    gains = [1 + 0.1 * _rand(D, seed=5 + i, dtype=torch.float32) for i in range(2)]
    tok = _tokens((B, T), V, "text", torch.int64)
    docs = _docs("sorted", B, T)
    tok[docs < 0] = -1
    ids, teacher = _teacher(B * T, V, K, 1)
    ids[docs.flatten() < 0] = -1
    at = torch.arange(T).expand(B, T).contiguous()

    def run(dev, lp):
        leaf = [t.to(dev).clone().requires_grad_() for t in (table, wqkv, wo, *gains)]
        tb, w1, w2, gq, gk = leaf
        d = docs.to(dev)
        x = ops.token_embedding(tok.to(dev), tb, scale=math.sqrt(C))
        q, k, v = ops.qk_norm_rotary(ops.linear(x, w1, lp(w1), None), Hq, Hkv, q_weight=gq, k_weight=gk,
                                     inv_freq=ops.rotary_frequencies(D, device=dev), positions=at.to(dev))
        a = ops.attention(q, k, v, documents=d, softcap=15.0)
        x = x + ops.linear(a.reshape(B, T, Hq * D), w2, lp(w2), None)
        logits = ops.linear(x, tb, lp(tb), None)
        loss = ops.distillation_loss(logits.reshape(B * T, V), ids.to(dev), teacher.to(dev), temperature=1.5)
        return loss.detach(), torch.autograd.grad(loss, leaf)
    loss, grads = run(DEV, lambda w: w.detach().to(torch.bfloat16))
    ref_loss, ref = run("cpu", lambda w: None)
    assert abs(loss.item() - ref_loss.item()) <= 1e-2 * abs(ref_loss.item())
    for name, a, b in zip(("table", "wqkv", "wo", "q gain", "k gain"), grads, ref):
        err = (a.cpu() - b).norm() / b.norm()
        assert err <= 3e-2, f"{name}: {err:.3g}"
