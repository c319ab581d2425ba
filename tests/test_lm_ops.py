"""Attention with score modifiers, head norms with rotation, the token embedding and the distillation loss off the GPU: the
plain paths (the oracle of the GPU tests) against independent formulas and against differences in 64 bits, and every refusal."""
import math

import pytest
import torch

from distributedpytorch_amd import ops


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _attend_by_loops(q, k, v, causal=True, scale=None, softcap=0.0, slopes=None, documents=None, prefix=None):
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros_like(q)
    for b in range(B):
        for h in range(Hq):
            kh = h * Hkv // Hq
            for i in range(T):
                xs, js = [], []
                for j in range(T):
                    see = not causal or j <= i or (prefix is not None and j < int(prefix[b]))
                    if documents is not None:
                        see = see and int(documents[b, i]) >= 0 and int(documents[b, i]) == int(documents[b, j])
                    if see:
                        x = scale * float(q[b, i, h] @ k[b, j, kh])
                        x = softcap * math.tanh(x / softcap) if softcap else x
                        xs.append(x - (float(slopes[h]) * abs(i - j) if slopes is not None else 0.0))
                        js.append(j)
                if js:
                    w = [math.exp(x - max(xs)) for x in xs]
                    for x, j in zip(w, js):
                        out[b, i, h] += x / sum(w) * v[b, j, kh]
    return out


MODES = [dict(), dict(causal=False), dict(softcap=2.0), dict(slopes=True), dict(documents=True), dict(prefix=True),
         dict(softcap=1.5, slopes=True, documents=True, prefix=True, scale=0.7)]


def _extras(mode, B, T, Hq):
    kw = dict(mode)
    if kw.pop("slopes", False):
        kw["slopes"] = torch.linspace(0.4, -0.1, Hq)
    if kw.pop("documents", False):
        kw["documents"] = torch.tensor([[3, 3, -1, 0, 0, 3, 7][:T], [1] * (T - 1) + [-1]], dtype=torch.int32)[:B]
    if kw.pop("prefix", False):
        kw["prefix"] = torch.tensor([4, -2], dtype=torch.int32)[:B]
    return kw


@pytest.mark.parametrize("mode", range(len(MODES)))
def test_attention_plain_path_against_loops_and_differences(mode):
    B, T, Hq, Hkv, D = 2, 7, 4, 2, 3
    g = _g(mode)
    q, k, v = (torch.randn(B, T, h, D, generator=g, dtype=torch.float64) for h in (Hq, Hkv, Hkv))
    kw = _extras(MODES[mode], B, T, Hq)
    torch.testing.assert_close(ops.attention(q, k, v, **kw), _attend_by_loops(q, k, v, **kw), rtol=1e-12, atol=1e-12)
    for t in (q, k, v):
        t.requires_grad_()
    assert torch.autograd.gradcheck(lambda *a: ops.attention(*a, **kw), (q, k, v))


def test_attention_padding_and_zero_length():
    q, k, v = (torch.randn(1, 4, 2, 8, generator=_g(1), dtype=torch.float64) for _ in range(3))
    docs = torch.tensor([[0, 0, -1, -7]], dtype=torch.int32)
    ref = ops.attention(q, k, v, documents=docs)
    assert (ref[:, 2:] == 0).all()
    for t, bad in ((q, math.nan), (k, math.inf), (v, math.nan)):
        t[:, 2:] = bad
        t.requires_grad_()
    out = ops.attention(q, k, v, documents=docs)
    assert torch.equal(out, ref)
    for d in torch.autograd.grad(out, (q, k, v), torch.ones_like(out)):
        assert torch.isfinite(d).all() and (d[:, 2:] == 0).all()
    for shape in ((2, 0, 2, 8), (0, 5, 2, 8)):
        e = torch.zeros(shape, requires_grad=True)
        out = ops.attention(e, e, e)
        assert out.shape == shape and torch.autograd.grad(out.sum(), e)[0].shape == shape


def test_attention_refusals():
    q, k = torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 2, 8)
    i32 = dict(dtype=torch.int32)
    for bad in (dict(q=q[0]), dict(k=torch.zeros(2, 5, 3, 8)), dict(v=torch.zeros(2, 5, 2, 16)), dict(k=torch.zeros(2, 6, 2, 8), v=torch.zeros(2, 6, 2, 8)),
                dict(k=torch.zeros(2, 5, 3, 8), v=torch.zeros(2, 5, 3, 8)), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
                dict(softcap=-1.0), dict(softcap=math.nan), dict(slopes=torch.zeros(3)), dict(slopes=torch.zeros(4, dtype=torch.float64)),
                dict(slopes=torch.zeros(4, requires_grad=True)), dict(documents=torch.zeros(2, 5)), dict(documents=torch.zeros(2, 5, dtype=torch.int64)),
                dict(documents=torch.zeros(5, **i32)), dict(prefix=torch.zeros(3, **i32)), dict(prefix=torch.zeros(2))):
        kw = dict(q=q, k=k, v=k)
        kw.update(bad)
        with pytest.raises(ValueError):
            ops.attention(kw.pop("q"), kw.pop("k"), kw.pop("v"), **kw)
    with pytest.raises(TypeError):
        ops.attention(q, k.double(), k)
    with pytest.raises(TypeError):
        ops.attention(q.long(), k.long(), k.long())


def test_attention_cap_outside_its_range():
    """A cap that fp32 cannot hold would be no cap at all on the GPU."""
    q = torch.zeros(1, 2, 1, 8)
    for softcap in (1e-46, 1e-13, 1e12, math.inf):
        with pytest.raises(ValueError):
            ops.attention(q, q, q, softcap=softcap)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R", [0, 4, 8])
@pytest.mark.parametrize("norm", [False, True])
def test_heads_plain_path_against_loops_and_differences(norm, R, interleaved):
    if not norm and not R:
        pytest.skip("refused")
    B, T, Hq, Hkv, D = 2, 3, 3, 1, 8
    g = _g(R + norm)
    qkv = torch.randn(B, T, (Hq + 2 * Hkv) * D, generator=g, dtype=torch.float64)
    qw, kw = (torch.randn(D, generator=g, dtype=torch.float64) if norm else None for _ in range(2))
    freq = ops.rotary_frequencies(R, 100.0) if R else None
    pos = torch.tensor([[0, 5, -3], [1 << 40, 2, 9]]) if R else None
    q, k, v = ops.qk_norm_rotary(qkv, Hq, Hkv, q_weight=qw, k_weight=kw, inv_freq=freq, positions=pos, eps=1e-3, interleaved=interleaved)
    x = qkv.view(B, T, Hq + 2 * Hkv, D)
    assert torch.equal(v, x[:, :, Hq + Hkv:])
    for b in range(B):
        for t in range(T):
            for h in range(Hq + Hkv):
                y = x[b, t, h].clone()
                if norm:
                    y = y / math.sqrt(float((y * y).mean()) + 1e-3) * (qw if h < Hq else kw)
                for i in range(R // 2):
                    a, c = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
                    ang = int(pos[b, t]) * float(freq[i])
                    y[a], y[c] = y[a] * math.cos(ang) - y[c] * math.sin(ang), y[c] * math.cos(ang) + y[a] * math.sin(ang)
                got = q[b, t, h] if h < Hq else k[b, t, h - Hq]
                torch.testing.assert_close(got, y, rtol=1e-12, atol=1e-12)
    leaves = [t.requires_grad_() for t in (qkv, qw, kw) if t is not None]

    def f(*a):
        a = list(a) + [None] * (3 - len(a))
        return ops.qk_norm_rotary(a[0], Hq, Hkv, q_weight=a[1], k_weight=a[2], inv_freq=freq, positions=pos, eps=1e-3, interleaved=interleaved)
    assert torch.autograd.gradcheck(f, leaves)


def test_heads_zero_length():
    x = torch.zeros(2, 0, 24, requires_grad=True)
    q, k, v = ops.qk_norm_rotary(x, 1, inv_freq=ops.rotary_frequencies(8))
    assert q.shape == k.shape == v.shape == (2, 0, 1, 8) and torch.autograd.grad(q.sum(), x)[0].shape == x.shape


def test_heads_refusals():
    x, w, f = torch.zeros(2, 3, 5 * 8), torch.ones(8), ops.rotary_frequencies(8)
    ok = dict(q_weight=w, k_weight=w, inv_freq=f)
    ops.qk_norm_rotary(x, 3, 1, **ok)
    for args, kw in (((x[0], 3, 1), ok), ((x, 3, 2), ok), ((x, 0, 1), ok), ((x, 3, 1), {}), ((x, 3, 1), dict(q_weight=w)), ((x, 3, 1), dict(q_weight=w, k_weight=w[:4])),
                     ((x, 3, 1), dict(inv_freq=f.float())), ((x, 3, 1), dict(inv_freq=ops.rotary_frequencies(10))),
                     ((x, 3, 1), dict(inv_freq=f.clone().requires_grad_())), ((x, 3, 1), dict(q_weight=w, k_weight=w, positions=torch.zeros(3, dtype=torch.int64))),
                     ((x, 3, 1), dict(inv_freq=f, positions=torch.zeros(3))), ((x, 3, 1), dict(inv_freq=f, positions=torch.zeros(2, 4, dtype=torch.int64))),
                     ((x, 3, 1), dict(ok, eps=-1.0)), ((x, 3, 1), dict(ok, eps=math.nan))):
        with pytest.raises(ValueError):
            ops.qk_norm_rotary(*args, **kw)
    with pytest.raises(TypeError):
        ops.qk_norm_rotary(x.long(), 3, 1, **ok)
    for bad in (0, 3, -2):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(bad)


def test_token_embedding_plain_path():
    w = torch.randn(6, 3, generator=_g(0), dtype=torch.float64, requires_grad=True)
    tok = torch.tensor([[0, 5, -1, 2], [2, 6, 2, 1 << 40]])
    y = ops.token_embedding(tok, w, scale=2.5)
    for i, row in enumerate(tok.tolist()):
        for j, t in enumerate(row):
            assert torch.equal(y[i, j], 2.5 * w[t] if 0 <= t < 6 else torch.zeros(3, dtype=torch.float64))
    assert torch.autograd.gradcheck(lambda a: ops.token_embedding(tok, a, scale=2.5), (w,))
    assert ops.token_embedding(tok[:0], w).shape == (0, 4, 3)
    assert torch.equal(ops.token_embedding(torch.tensor(5, dtype=torch.int32), w), w[5])
    for bad in ((tok, w[0]), (tok, w.long())):
        with pytest.raises(ValueError):
            ops.token_embedding(*bad)
    with pytest.raises(TypeError):
        ops.token_embedding(tok.float(), w)


def _distill_by_loops(z, ids, t, tau, V):
    total = 0.0
    for r in range(z.shape[0]):
        live = [k for k in range(ids.shape[1]) if 0 <= int(ids[r, k]) < V and float(t[r, k]) != -math.inf]
        if not live:
            continue
        lse = math.log(sum(math.exp(float(x) / tau) for x in z[r, :V]))
        mass = sum(math.exp(float(t[r, k]) / tau) for k in live)
        for k in live:
            p = math.exp(float(t[r, k]) / tau) / mass
            total += tau * tau * p * (math.log(p) - (float(z[r, int(ids[r, k])]) / tau - lse))
    return total / z.shape[0]


@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_distillation_plain_path_against_loops_and_differences(tau):
    g = _g(3)
    z = torch.randn(5, 9, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[0, 3, 6], [2, 2, 5], [-1, -1, -1], [1, 7, 8], [4, -1, 0]])     # twice the same, none, padding columns, short
    t = torch.randn(5, 3, generator=g, dtype=torch.float64)
    t[3, 0] = -math.inf                                                               # ... and so a row whose three entries are all dead
    loss = ops.distillation_loss(z, ids, t, temperature=tau, n_classes=7)
    assert abs(float(loss) - _distill_by_loops(z, ids, t, tau, 7)) < 1e-12
    assert torch.autograd.gradcheck(lambda a: ops.distillation_loss(a, ids, t, temperature=tau, n_classes=7), (z,))
    (d,) = torch.autograd.grad(loss, z)
    assert (d[2:4] == 0).all() and (d[:, 7:] == 0).all()
    with torch.no_grad():
        z[2] = math.nan                                                              # no teacher: whatever the row holds
    assert torch.equal(ops.distillation_loss(z, ids, t, temperature=tau, n_classes=7), loss)
    three = ops.distillation_loss(z.view(1, 5, 9), ids.view(1, 5, 3), t.view(1, 5, 3), temperature=tau, n_classes=7)
    assert torch.equal(three, loss)


def test_distillation_plain_path_does_not_feel_a_rows_offset():
    """fp32 logits around 30,000, where one place is 2^-9, and rows of the lowest value: each term within some places of its own size."""
    z = torch.randn(4, 50, generator=_g(1)) + torch.tensor([0.0, 3e4, -3e4, 0.0])[:, None]
    z[3] = torch.finfo(torch.float32).min
    ids, t = torch.arange(12).view(4, 3), torch.randn(4, 3, generator=_g(2))
    a, b = z.clone().requires_grad_(), z.double().requires_grad_()
    one, two = ops.distillation_loss(a, ids, t), ops.distillation_loss(b, ids, t.double())
    q, p = torch.softmax(z.double(), 1), torch.softmax(t.double(), 1)
    by_hand = (p * (p.log() - q.log().gather(1, ids))).sum() / 4
    assert abs(two.item() - by_hand.item()) < 1e-12
    assert abs(one.item() - by_hand.item()) < 1e-5
    da, db = torch.autograd.grad(one, a)[0], torch.autograd.grad(two, b)[0]
    torch.testing.assert_close(da.double(), db, rtol=0, atol=1e-6)


def test_distillation_refusals():
    z, ids, t = torch.zeros(4, 10), torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    ops.distillation_loss(z, ids, t)
    for args, kw in (((z, ids, t), dict(n_classes=0)), ((z, ids, t), dict(n_classes=11)), ((z, ids, t), dict(temperature=0.0)), ((z, ids, t), dict(temperature=math.nan)),
                     ((z, ids[:3], t), {}), ((z, ids[:, :0], t[:, :0]), {}), ((z[0], ids, t), {}), ((z.long(), ids, t), {}),
                     ((z, ids, t.clone().requires_grad_()), {})):
        with pytest.raises(ValueError):
            ops.distillation_loss(*args, **kw)
    for args in ((z, ids.float(), t), (z, ids, t.long())):
        with pytest.raises(TypeError):
            ops.distillation_loss(*args)
