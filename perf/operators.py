"""Cases for the language-model operators of ``distributedpytorch_amd.ops``: attention with score modifiers, head norms with
rotary positions, the scaled token embedding and the top-logit distillation loss.

Each case is one training pass through one operator: its forward, and the gradients that a training step takes from it.  With
``own`` false ``run`` computes the operators from elementary torch operations in 32 bits (rotation angles in 64), rounded
once at the end; with ``own`` true it calls the framework.
"""
import math
import random

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------- cases
def _attend(name, B, T, Hq, Hkv, D, softcap=0.0, slopes=False, doc=0, prefix=0.0, causal=True, gain=1.0):
    """``doc``: mean length of the documents packed into a row (0: one document per row); ``prefix``: mean share of a row
    that every position sees; ``gain``: standard deviation of the raw scores."""
    return {"name": name, "op": "attend", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "softcap": softcap, "slopes": slopes,
            "doc": doc, "prefix": prefix, "causal": causal, "gain": gain}


def _heads(name, B, T, Hq, Hkv, D, R, interleaved, doc):
    """``R``: rotated channels of a head; ``doc``: mean document length, positions restart at each (0: they run on)."""
    return {"name": name, "op": "heads", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "interleaved": interleaved, "doc": doc}


def _embed(name, B, T, V, C, skew):
    """``skew``: 1 draws tokens with natural text's frequencies (probability ~ 1 / rank), 0 uniformly."""
    return {"name": name, "op": "embed", "B": B, "T": T, "V": V, "C": C, "skew": skew}


def _distill(name, N, V, ld, K, bf16, temperature):
    """``V`` classes in rows of ``ld`` columns; ``K`` teacher entries per row."""
    return {"name": name, "op": "distill", "N": N, "V": V, "ld": ld, "K": K, "bf16": bf16, "temperature": temperature}


def listed():
    return [
        # one short row of packed documents through a two-head model: launch and host time count
        _attend("attend tiny", 1, 128, 2, 2, 64, doc=40),
        # GPT-2 small's heads at its training batch, rows packed with documents of 256 tokens on average
        _attend("attend packed", 16, 1024, 12, 12, 64, doc=256),
        # instruction rows of odd length: the prompt is seen from everywhere, scores capped, four queries heads to a key head
        _attend("attend capped prefix", 4, 2047, 16, 4, 128, softcap=30.0, prefix=0.25, gain=8.0),
        # one long row with a bias that falls with the distance
        _attend("attend far", 1, 8192, 16, 4, 128, slopes=True),
        # GPT-2 small's packed projection, positions running on
        _heads("heads gpt2", 16, 1024, 12, 12, 64, 64, False, 0),
        # grouped heads, neighbouring channels rotated together, odd length, positions restarting at each document
        _heads("heads grouped", 2, 8191, 16, 4, 128, 128, True, 700),
        # a test-sized model's table
        _embed("embed tiny", 2, 100, 512, 128, 1),
        # GPT-2 small's table and training batch, tokens as frequent as in text
        _embed("embed gpt2", 16, 1024, 50304, 768, 1),
        # long batches over the same vocabulary with wider rows
        _embed("embed long", 32, 2048, 50304, 1024, 1),
        # a test-sized vocabulary in 32 bits
        _distill("distill tiny", 64, 500, 512, 8, False, 1.0),
        # GPT-2 small's padded vocabulary at its training batch
        _distill("distill gpt2", 16384, 50257, 50304, 32, True, 2.0),
        # a vocabulary past what one workgroup holds, rows of odd length in 32 bits, many teacher entries
        _distill("distill wide", 2047, 100001, 100001, 200, False, 1.5),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "heads", "embed", "distill"))
    while True:
        if op == "attend":
            D = rng.choice((32, 64, 64, 80, 96, 128, 128))
            Hkv = rng.choice((1, 2, 3, 4, 8, 12))
            group = rng.choice((1, 1, 2, 3, 4, 8))
            T = _log(rng, 1, 8192)
            kind = rng.choice(("doc", "cap", "slopes", "prefix", "all", "both ways"))
            c = _attend("", _log(rng, 1, 16), T, Hkv * group, Hkv, D, doc=_log(rng, 1, 2048) if kind in ("doc", "all", "both ways") else 0,
                        softcap=rng.choice((20.0, 30.0, 50.0)) if kind in ("cap", "all") else 0.0, slopes=kind in ("slopes", "all"),
                        prefix=rng.uniform(0.0, 0.6) if kind in ("prefix", "all") else 0.0, causal=kind != "both ways",
                        gain=rng.choice((1.0, 3.0)))
            whole = 1 if c["causal"] and not c["prefix"] else 2                 # how much of the square may be visible, in halves
            fits = c["B"] * c["Hq"] * T * T * whole <= 16 * 8192 * 8192 and c["Hq"] <= 32 and c["B"] * c["Hq"] * T * D <= 16 * 12 * 1024 * 128
        elif op == "heads":
            D = rng.choice((32, 64, 64, 96, 128, 128))
            Hkv = rng.choice((1, 2, 4, 8, 12))
            c = _heads("", _log(rng, 1, 16), _log(rng, 1, 8192), Hkv * rng.choice((1, 2, 4)), Hkv, D, D if rng.random() < 0.6 else D // 2,
                       rng.random() < 0.5, rng.choice((0, _log(rng, 1, 2000))))
            fits = c["B"] * c["T"] * (c["Hq"] + 2 * Hkv) * D <= 2 * 8191 * 24 * 128
        elif op == "embed":
            c = _embed("", _log(rng, 1, 32), _log(rng, 1, 4096), _log(rng, 100, 60000), 8 * _log(rng, 4, 200), rng.choice((0, 1, 1)))
            fits = c["B"] * c["T"] <= 65536 and c["B"] * c["T"] * c["C"] <= 65536 * 1024 and c["V"] * c["C"] <= 50304 * 1024
        else:
            V = _log(rng, 100, 130000)
            bf16 = rng.random() < 0.6
            c = _distill("", _log(rng, 1, 16384), V, (V + 63) // 64 * 64 if rng.random() < 0.7 else V, min(V, _log(rng, 1, 256)), bf16,
                         rng.choice((1.0, 2.0, 4.0, 0.7)))
            fits = c["N"] * c["ld"] * (2 if bf16 else 4) <= 16384 * 50304 * 2
        if fits:
            c.pop("name")
            return c


# ------------------------------------------------------------------------------------------------------------ inputs
def _documents(rng, B, T, mean):
    """Document numbers [B, T] of rows packed with documents of `mean` tokens on average, and a padded end of the last row."""
    rows = []
    for b in range(B):
        row, n = [], 0
        while len(row) < T:
            k = max(1, int(rng.expovariate(1.0 / mean)) + 1)
            row += [n] * k
            n += 1
        rows.append(row[:T])
    pad = T // 16
    if pad:
        rows[-1][T - pad:] = [-1] * pad
    return rows


def _prefix(rng, B, T, share):
    return [min(T, int(T * share * 2 * rng.random())) for _ in range(B)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    s = {"case": case}
    if case["op"] == "attend":
        B, T, Hq, Hkv, D = (case[k] for k in ("B", "T", "Hq", "Hkv", "D"))
        root = math.sqrt(case["gain"])
        # queries and keys as the head norms leave them, values as a view of the packed projection that they came in
        s["q"] = normal(B, T, Hq, D, std=root).requires_grad_()
        s["k"] = normal(B, T, Hkv, D, std=root).requires_grad_()
        s["v"] = normal(B, T, Hq + 2 * Hkv, D)[:, :, Hq + Hkv:].detach().requires_grad_()
        s["dout"] = normal(B, T, Hq, D)
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=DEV) if case["slopes"] else None
        s["documents"] = torch.tensor(_documents(rng, B, T, case["doc"]), dtype=torch.int32, device=DEV) if case["doc"] else None
        s["prefix"] = torch.tensor(_prefix(rng, B, T, case["prefix"]), dtype=torch.int32, device=DEV) if case["prefix"] else None
    elif case["op"] == "heads":
        B, T, Hq, Hkv, D, R = (case[k] for k in ("B", "T", "Hq", "Hkv", "D", "R"))
        s["qkv"] = normal(B, T, (Hq + 2 * Hkv) * D).requires_grad_()
        s["qw"] = (1.0 + 0.1 * normal(D, dtype=torch.float32)).requires_grad_()
        s["kw"] = (1.0 + 0.1 * normal(D, dtype=torch.float32)).requires_grad_()
        s["inv_freq"] = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R)
        s["positions"] = None
        if case["doc"]:
            at = []
            for row in _documents(rng, B, T, case["doc"]):
                start, line = 0, []
                for t, d in enumerate(row):
                    if t and d != row[t - 1]:
                        start = t
                    line.append(t - start)
                at.append(line)
            s["positions"] = torch.tensor(at, dtype=torch.int64, device=DEV)
        s["dq"], s["dk"], s["dv"] = normal(B, T, Hq, D), normal(B, T, Hkv, D), normal(B, T, Hkv, D)
    elif case["op"] == "embed":
        B, T, V, C = (case[k] for k in ("B", "T", "V", "C"))
        u = torch.rand(B, T, generator=g, device=DEV, dtype=torch.float64)
        rank = (torch.exp(u * math.log(V)) - 1.0 if case["skew"] else u * V).long().clamp_(0, V - 1)
        s["tokens"] = torch.randperm(V, generator=g, device=DEV)[rank]
        s["weight"] = normal(V, C, std=0.02, dtype=torch.float32).requires_grad_()       # the fp32 parameter ...
        s["weight_lp"] = s["weight"].detach().to(torch.bfloat16)                         # ... and the bf16 copy that an optimizer keeps
        s["dout"] = normal(B, T, C, std=0.01)
        s["scale"] = math.sqrt(C)
    else:
        N, V, ld, K = (case[k] for k in ("N", "V", "ld", "K"))
        s["logits"] = normal(N, ld, std=2.0, dtype=torch.bfloat16 if case["bf16"] else torch.float32).requires_grad_()
        # distinct classes per row (a walk through the vocabulary), logits falling; one row of 16 is a prompt's and has no teacher
        first = torch.randint(0, V, (N, 1), generator=g, device=DEV)
        step = V // K if K > 1 else 1
        ids = (first + step * torch.arange(K, device=DEV)) % V
        none = torch.rand(N, 1, generator=g, device=DEV) < 1.0 / 16.0
        s["ids"] = torch.where(none, -1, ids)
        s["teacher"] = (torch.randn(N, K, generator=g, device=DEV) * 2.0 + 4.0).sort(dim=1, descending=True).values
    return s


# ---------------------------------------------------------------------------------------------------- the plain forms
def _visible(case, s):
    B, T = case["B"], case["T"]
    i = torch.arange(T, device=DEV)
    see = (i[None, :] <= i[:, None])[None] if case["causal"] else torch.ones(1, T, T, dtype=torch.bool, device=DEV)
    if s["prefix"] is not None:
        see = see | (i[None, None, :] < s["prefix"][:, None, None])
    if s["documents"] is not None:
        d = s["documents"]
        see = see & (d[:, :, None] == d[:, None, :]) & (d >= 0)[:, :, None]
    return see[:, None]                                                  # [B or 1, 1, T, T]


def _attend_plain(s):
    case = s["case"]
    group, D, T = case["Hq"] // case["Hkv"], case["D"], case["T"]
    q = s["q"].float().transpose(1, 2)
    k = s["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    v = s["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(D)
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    if s["slopes"] is not None:
        i = torch.arange(T, device=DEV, dtype=torch.float32)
        x = x - s["slopes"][:, None, None] * (i[:, None] - i[None, :]).abs()
    x = torch.where(_visible(case, s), x, -math.inf)
    e = torch.exp(x - x.detach().amax(3, keepdim=True).clamp(min=-1e30))
    p = e / e.sum(3, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p, v).transpose(1, 2)
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"].float())
    return {"out": out.detach().to(torch.bfloat16), "dq": dq, "dk": dk, "dv": dv}


def _heads_plain(s):
    case = s["case"]
    B, T, Hq, Hkv, D, R = (case[k] for k in ("B", "T", "Hq", "Hkv", "D", "R"))
    x = s["qkv"].float().view(B, T, Hq + 2 * Hkv, D)
    at = torch.arange(T, device=DEV)[None] if s["positions"] is None else s["positions"]
    angle = at.double()[..., None, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def one(h, w):
        n = h * torch.rsqrt((h * h).mean(3, keepdim=True) + 1e-6) * w
        r = n[..., :R]
        a, b = (r[..., 0::2], r[..., 1::2]) if case["interleaved"] else (r[..., : R // 2], r[..., R // 2:])
        a, b = a * cos - b * sin, b * cos + a * sin
        r = torch.stack((a, b), 4).flatten(3) if case["interleaved"] else torch.cat((a, b), 3)
        return torch.cat((r, n[..., R:]), 3)

    q, k, v = one(x[:, :, :Hq], s["qw"]), one(x[:, :, Hq:Hq + Hkv], s["kw"]), x[:, :, Hq + Hkv:]
    dqkv, dqw, dkw = torch.autograd.grad((q, k, v), (s["qkv"], s["qw"], s["kw"]), (s["dq"].float(), s["dk"].float(), s["dv"].float()))
    q, k, v = (t.detach().to(torch.bfloat16) for t in (q, k, v))
    return {"q": q, "k": k, "v": v, "dqkv": dqkv, "dqw": dqw, "dkw": dkw}


def _embed_plain(s):
    out = (s["weight_lp"][s["tokens"]].float() * s["scale"]).to(torch.bfloat16)
    dw = torch.zeros_like(s["weight"])
    dw.index_add_(0, s["tokens"].flatten(), s["dout"].flatten(0, 1).float() * s["scale"])
    return {"out": out, "dw": dw}


def _distill_plain(s):
    case = s["case"]
    V, N, tau = case["V"], case["N"], case["temperature"]
    z = s["logits"].detach()[:, :V].float() / tau
    m = z.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(1, keepdim=True))
    live = s["ids"] >= 0
    t = torch.where(live, s["teacher"] / tau, -math.inf)
    t = t - t.amax(1, keepdim=True).clamp(min=-1e30)
    mass = torch.exp(t).sum(1, keepdim=True).clamp(min=1e-30)
    p = torch.exp(t) / mass
    logp = torch.where(live, t - torch.log(mass), 0.0)
    at = s["ids"].clamp(min=0)
    loss = tau * tau / N * (p * (logp - z.gather(1, at) + lse)).sum()
    d = torch.zeros_like(s["logits"], dtype=torch.float32)
    d[:, :V] = torch.exp(z - lse) * live.any(1, keepdim=True)
    d.scatter_add_(1, at, -p)
    return {"loss": loss, "dlogits": (d * (tau / N)).to(s["logits"].dtype)}


# --------------------------------------------------------------------------------------------------------------- run
def _attend_own(s):
    from distributedpytorch_amd import ops
    case = s["case"]
    out = ops.attention(s["q"], s["k"], s["v"], causal=case["causal"], softcap=case["softcap"], slopes=s["slopes"],
                        documents=s["documents"], prefix=s["prefix"])
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def _heads_own(s):
    from distributedpytorch_amd import ops
    case = s["case"]
    q, k, v = ops.qk_norm_rotary(s["qkv"], case["Hq"], case["Hkv"], q_weight=s["qw"], k_weight=s["kw"], inv_freq=s["inv_freq"],
                                 positions=s["positions"], interleaved=case["interleaved"])
    dqkv, dqw, dkw = torch.autograd.grad((q, k, v), (s["qkv"], s["qw"], s["kw"]), (s["dq"], s["dk"], s["dv"]))
    return {"q": q.detach(), "k": k.detach(), "v": v.detach(), "dqkv": dqkv, "dqw": dqw, "dkw": dkw}


def _embed_own(s):
    from distributedpytorch_amd import ops
    out = ops.token_embedding(s["tokens"], s["weight"], s["weight_lp"], scale=s["scale"])
    (dw,) = torch.autograd.grad(out, (s["weight"],), s["dout"])
    return {"out": out.detach(), "dw": dw}


def _distill_own(s):
    from distributedpytorch_amd import ops
    case = s["case"]
    loss = ops.distillation_loss(s["logits"], s["ids"], s["teacher"], temperature=case["temperature"], n_classes=case["V"])
    (d,) = torch.autograd.grad(loss, (s["logits"],))
    return {"loss": loss.detach(), "dlogits": d}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attend": _attend_own, "heads": _heads_own, "embed": _embed_own, "distill": _distill_own}[op](state)
    return {"attend": _attend_plain, "heads": _heads_plain, "embed": _embed_plain, "distill": _distill_plain}[op](state)


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "attend":
        B, T, Hq, Hkv, D = (case[k] for k in ("B", "T", "Hq", "Hkv", "D"))
        rng = random.Random(0)
        docs = _documents(rng, B, T, case["doc"]) if case["doc"] else [[0] * T] * B
        share = case["prefix"]
        pairs = 0.0
        for row in docs:
            t = 0
            while t < T:
                e = t
                while e < T and row[e] == row[t]:
                    e += 1
                n = e - t
                if row[t] >= 0:
                    half = n * (n + 1) / 2.0
                    # a prefix of a share of the row shows its keys to the queries in front of them as well
                    pairs += n * n if not case["causal"] else half + share * share / 2.0 * n * n
                t = e
        # forward: two products; backward: the scores again and four more
        return {"bytes": 2.0 * B * T * D * (2 * Hq + 2 * Hkv + 2 * Hq + 2 * Hkv), "flops": 7 * 2.0 * pairs * Hq * D}
    if case["op"] == "heads":
        n = 2.0 * case["B"] * case["T"] * case["D"]
        q, kv = case["Hq"], case["Hkv"]
        # forward reads q and k and writes them (the values stay where they are), backward reads them again beside their
        # gradients and the values', and writes the packed gradient
        return {"bytes": n * ((q + kv) * 2 + (q + kv) + (q + 2 * kv) * 2), "flops": 20.0 * n}
    if case["op"] == "embed":
        rows = case["B"] * case["T"]
        C, V = case["C"], case["V"]
        return {"bytes": rows * (C * 2.0 * 3 + 8) + 4.0 * V * C, "flops": 2.0 * rows * C}
    n = case["N"] * (2.0 if case["bf16"] else 4.0)
    return {"bytes": n * (case["V"] + case["ld"]) + case["N"] * case["K"] * 12.0, "flops": 8.0 * case["N"] * case["V"]}


# ------------------------------------------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attend": _attend_exact, "heads": _heads_exact, "embed": _embed_exact, "distill": _distill_exact}[case["op"]](case, s)


def _attend_exact(case, s):
    """Head by head, gradients from the formulas: dS = P (dP - rowsum(P dP)), through the bias (none), the cap (1 - tanh^2)
    and the scale."""
    B, T, Hq, Hkv, D = (case[k] for k in ("B", "T", "Hq", "Hkv", "D"))
    out, dq = torch.zeros(2, B, T, Hq, D, dtype=torch.float64, device=DEV)
    dk, dv = torch.zeros(2, B, T, Hkv, D, dtype=torch.float64, device=DEV)
    row = torch.arange(T, device=DEV)[:, None]
    col = torch.arange(T, device=DEV)[None, :]
    for b in range(B):
        hidden = col > row if case["causal"] else torch.zeros(T, T, dtype=torch.bool, device=DEV)
        if s["prefix"] is not None:
            hidden = hidden & (col >= int(s["prefix"][b]))
        if s["documents"] is not None:
            d = s["documents"][b]
            hidden = hidden | (d[:, None] != d[None, :]) | (d < 0)[:, None]
        none = hidden.all(1, keepdim=True)
        for h in range(Hq):
            hk = h * Hkv // Hq
            q, k, v, do = s["q"][b, :, h].double(), s["k"][b, :, hk].double(), s["v"][b, :, hk].double(), s["dout"][b, :, h].double()
            x = (q @ k.t().contiguous()) * D ** -0.5
            slope = 1.0
            if case["softcap"]:
                th = torch.tanh(x / case["softcap"])
                x, slope = case["softcap"] * th, 1.0 - th * th
            if s["slopes"] is not None:
                x = x + s["slopes"][h].double() * -(row - col).abs()
            x = x.masked_fill(hidden, -math.inf).masked_fill(none, 0.0)
            x = torch.exp(x - torch.logsumexp(x, 1, keepdim=True)).masked_fill(none, 0.0)
            out[b, :, h] = x @ v
            dp = do @ v.t().contiguous()
            dv[b, :, hk] += x.t().contiguous() @ do
            x = x * (dp - (x * dp).sum(1, keepdim=True)) * slope * D ** -0.5
            dq[b, :, h] = x @ k
            dk[b, :, hk] += x.t().contiguous() @ q
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _heads_exact(case, s):
    """Rotation as a product of complex numbers; the norm's gradient from its formula r (g w - n mean(g w n))."""
    B, T, Hq, Hkv, D, R = (case[k] for k in ("B", "T", "Hq", "Hkv", "D", "R"))
    x = s["qkv"].double().view(B, T, Hq + 2 * Hkv, D)
    at = s["positions"] if s["positions"] is not None else torch.arange(T, device=DEV).expand(B, T)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), at.double()[:, :, None, None] * s["inv_freq"])
    if case["interleaved"]:
        first = torch.arange(0, R, 2, device=DEV)
        second = first + 1
    else:
        first = torch.arange(0, R // 2, device=DEV)
        second = first + R // 2

    def rotate(t, by):
        z = torch.complex(t[..., first], t[..., second]) * by
        t = t.clone()
        t[..., first], t[..., second] = z.real, z.imag
        return t

    def one(h, w, g):
        r = 1.0 / torch.sqrt(h.square().mean(3, keepdim=True) + 1e-6)
        n = h * r
        y = rotate(n * w.double(), turn)
        g = rotate(g.double(), turn.conj())
        gw = g * w.double()
        return y, r * (gw - n * (gw * n).mean(3, keepdim=True)), (g * n).sum((0, 1, 2))

    q, gq, dqw = one(x[:, :, :Hq], s["qw"], s["dq"])
    k, gk, dkw = one(x[:, :, Hq:Hq + Hkv], s["kw"], s["dk"])
    dqkv = torch.cat((gq, gk, s["dv"].double()), 2).view(B, T, -1)
    return {"q": q, "k": k, "v": x[:, :, Hq + Hkv:], "dqkv": dqkv, "dqw": dqw, "dkw": dkw}


def _embed_exact(case, s):
    out = torch.index_select(s["weight_lp"].double(), 0, s["tokens"].reshape(-1)).mul_(s["scale"]).view(case["B"], case["T"], -1)
    dw = torch.zeros(case["V"], case["C"], dtype=torch.float64, device=DEV)
    at = s["tokens"].reshape(-1, 1).expand(-1, case["C"])
    dw.scatter_add_(0, at, s["dout"].double().view(-1, case["C"]))
    return {"out": out, "dw": dw.mul_(s["scale"])}


def _distill_exact(case, s):
    """temperature^2 KL(p || q) per row, p the softmax of the row's teacher entries, q the student's over the vocabulary."""
    N, V, tau = case["N"], case["V"], case["temperature"]
    d = torch.zeros(N, case["ld"], dtype=torch.float64, device=DEV)
    loss = torch.zeros((), dtype=torch.float64, device=DEV)
    for r0 in range(0, N, 2048):
        r = slice(r0, min(N, r0 + 2048))
        logq = torch.log_softmax(s["logits"][r, :V].double() / tau, 1)
        ids = s["ids"][r]
        rows = (ids >= 0).all(1)
        logp = torch.log_softmax(s["teacher"][r].double() / tau, 1)
        full = torch.zeros_like(logq)
        full.scatter_(1, ids.clamp(min=0), logp.exp())
        kl = (logp.exp() * (logp - logq.gather(1, ids.clamp(min=0)))).sum(1)
        loss += tau * tau * kl[rows].sum()
        d[r, :V] = (logq.exp() - full) * rows[:, None] * (tau / N)
    return {"loss": loss / N, "dlogits": d}
