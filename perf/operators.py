"""Performance cases of the serving and distillation operators: what each computes in plain torch operations, what a
caller of ``kubeoperator_amd.ops.functional`` writes for it, and the bytes and operations it cannot do without.

Four operators, used together when one model answers many requests:

* ``prefix``: attention of the newest token(s) of every sequence over a prefix shared by the whole batch and over the
  sequence's own cache (``prefix_attention``);
* ``lora``: low-rank adapters of many requests added to a shared projection's output (``lora_add``);
* ``verify``: drafted tokens accepted or replaced against the target model's distribution (``verify_draft``);
* ``distill``: loss and gradient of a student's logits against a teacher's top logits (``distill_topk``), which is how
  the draft model is trained.

Sizes are those of the model configurations (hidden 4096 / 2048, 32 or 64 query heads over 8 KV heads, 12 heads of 64,
vocabularies of 128256, 50304 and 512) or generic.
"""
import math

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a handful of chats on the smallest model: launch latency
        dict(name="prefix tiny", op="prefix", B=4, T=1, Hq=4, Hkv=2, D=64, P=500, own=60),
        # ordinary decode step behind a 2k-token system prompt, 8B-sized heads
        dict(name="prefix decode", op="prefix", B=64, T=1, Hq=32, Hkv=8, D=128, P=2048, own=500),
        # drafts being checked: five tokens per sequence behind a long shared document
        dict(name="prefix drafts", op="prefix", B=64, T=5, Hq=32, Hkv=8, D=128, P=8192, own=1000),
        # one decode step, most rows on an adapter of their own
        dict(name="lora decode", op="lora", M=64, n=32, r=16, K=4096, N=4096, runs=False),
        # the widest projection at a larger rank, a batch that is no multiple of a tile
        dict(name="lora gate up", op="lora", M=100, n=48, r=64, K=4096, N=28672, runs=False),
        # prompts of several requests in one prefill: long runs of rows on the same adapter
        dict(name="lora prefill", op="lora", M=8100, n=16, r=16, K=4096, N=6144, runs=True),
        # one sequence, three drafted tokens, small vocabulary: latency
        dict(name="verify one", op="verify", B=1, T=3, V=50304, temp=1.0, dtype="float32"),
        # a full batch of sampled drafts on fp32 logits
        dict(name="verify batch", op="verify", B=64, T=4, V=128256, temp=0.8, dtype="float32"),
        # greedy decoding on bf16 logits
        dict(name="verify greedy", op="verify", B=32, T=7, V=128256, temp=0.0, dtype="bfloat16"),
        # the smallest vocabulary: latency
        dict(name="distill tiny", op="distill", N=256, V=512, K=8, temp=1.0),
        # a 50k vocabulary, a whole micro-batch of a small student
        dict(name="distill small vocab", op="distill", N=16384, V=50304, K=32, temp=2.0),
        # the 128k vocabulary, one long sequence
        dict(name="distill large vocab", op="distill", N=8192, V=128256, K=64, temp=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefix", "lora", "verify", "distill"])
    if op == "prefix":
        Hq, Hkv, D = rng.choice([(32, 8, 128), (64, 8, 128), (32, 8, 64), (12, 12, 64), (4, 2, 64), (8, 8, 128), (6, 2, 128)])
        T = rng.choice([1, 1, 1, rng.randint(2, 8)])
        c = dict(op=op, B=_log(rng, 1, 128), T=T, Hq=Hq, Hkv=Hkv, D=D, P=_log(rng, 1, 8192), own=_log(rng, T, 2000))
        while c["B"] > 1 and c["B"] * T * Hq * D * (c["P"] + c["own"]) > 64 * 5 * 32 * 128 * 8000:
            c["B"] -= 1
        return c
    if op == "lora":
        K = rng.choice([4096, 2048, 768, 14336, 8 * rng.randint(8, 1000)])
        N = rng.choice([4096, 6144, 28672, 2048, 8 * rng.randint(8, 1000)])
        M = _log(rng, 1, 8100)
        if M * (K + 2 * N) > 8100 * (4096 + 2 * 6144):
            M = 8100 * (4096 + 2 * 6144) // (K + 2 * N)
        n = rng.randint(1, 64) if M < 2000 else rng.randint(1, 16)
        return dict(op=op, M=M, n=n, r=rng.choice([8, 16, 16, 24, 32, 64]) if M < 2000 else rng.choice([8, 16, 24]), K=K, N=N,
                    runs=M > 300 or rng.random() < 0.3)
    if op == "verify":
        return dict(op=op, B=_log(rng, 1, 64), T=rng.randint(0, 4), V=rng.choice([128256, 50304, 512, _log(rng, 33, 128000)]),
                    temp=rng.choice([0.0, 1.0, round(rng.uniform(0.3, 1.5), 2)]), dtype=rng.choice(["float32", "bfloat16"]))
    V = rng.choice([128256, 50304, 512, _log(rng, 100, 128000)])
    return dict(op=op, N=max(1, min(_log(rng, 1, 16384), 16384 * 50304 // V)), V=V, K=_log(rng, 1, min(V, 128)),
                temp=rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4.0), 2)]))


# ------------------------------------------------------------------------------------------------ inputs
def _spread(lo, hi, count, gen):
    """``count`` lengths evenly spread over [lo, hi], in an order given by the seed: their sum does not depend on it."""
    at = torch.linspace(0, 1, count, device=DEV, dtype=torch.float64) if count > 1 else torch.ones(1, device=DEV, dtype=torch.float64)
    v = (lo + at * (hi - lo)).round().to(torch.int32)
    return v[torch.randperm(count, device=DEV, generator=gen)]


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    if c["op"] == "prefix":
        B, T, Hq, Hkv, D, P = (c[k] for k in ("B", "T", "Hq", "Hkv", "D", "P"))
        Smax = c["own"] + 8
        qkv = normal(B * T, (Hq + 2 * Hkv) * D).bfloat16()  # the fused projection's output: Q is a slice of its columns
        c["q"] = qkv[:, : Hq * D]
        c["kp"], c["vp"] = normal(Hkv, P, D).bfloat16(), normal(Hkv, P, D).bfloat16()
        c["kc"], c["vc"] = normal(B, Hkv, Smax, D).bfloat16(), normal(B, Hkv, Smax, D).bfloat16()
        c["lens"] = _spread(T, c["own"], B, gen)
        c["scale"] = 1.0 / math.sqrt(D)
    elif c["op"] == "lora":
        M, n, r, K, N = (c[k] for k in ("M", "n", "r", "K", "N"))
        c["x"] = normal(M, K).bfloat16()
        c["y"] = normal(M, N).bfloat16()
        c["a"] = (normal(n, r, K) / math.sqrt(K)).bfloat16()
        c["b"] = (normal(n, N, r) / math.sqrt(r)).bfloat16()
        c["alpha"] = torch.rand(n, device=DEV, generator=gen) + 0.5
        if c["runs"]:  # requests one after another; -1: requests without an adapter
            ends = torch.sort(torch.randint(0, M + 1, (2 * n,), device=DEV, generator=gen)).values
            which = torch.randint(-1, n, (2 * n + 1,), device=DEV, generator=gen)
            at = torch.bucketize(torch.arange(M, device=DEV), ends, right=True)
            c["index"] = which[at].to(torch.int32)
        else:
            c["index"] = torch.randint(-1, n, (M,), device=DEV, generator=gen).to(torch.int32)
    elif c["op"] == "verify":
        B, T, V = c["B"], c["T"], c["V"]
        dt = getattr(torch, c["dtype"])
        z = 3.0 * normal(B, T + 1, V)
        c["target"] = z.to(dt)
        c["draft"] = (z[:, :T] + 0.5 * normal(B, T, V)).to(dt)
        # tokens as the draft model picks them: sampled from its own distribution, its best one where decoding is greedy
        if T and c["temp"] > 0:
            cdf = torch.softmax(c["draft"].double() / c["temp"], -1).cumsum(-1)
            pick = torch.rand(B, T, 1, device=DEV, generator=gen, dtype=torch.float64)
            c["tokens"] = torch.searchsorted(cdf, pick).clamp_max(V - 1).squeeze(-1)
        else:
            c["tokens"] = c["draft"].float().argmax(-1) if T else torch.zeros(B, 0, dtype=torch.int64, device=DEV)
        c["u"] = torch.rand(B, T + 1, device=DEV, generator=gen)
    else:
        N, V, K = c["N"], c["V"], c["K"]
        z = 2.0 * normal(N, V)
        c["logits"] = z.bfloat16()
        near = z + normal(N, V)  # the teacher agrees with the student only roughly
        top = torch.topk(near, K, dim=-1)
        c["index"], c["teacher"] = top.indices.to(torch.int32), top.values.contiguous()
        c["weight"] = torch.full((N,), 1.0 / N, device=DEV)
        if N > 8:  # padding rows carry no loss
            c["weight"][torch.randperm(N, device=DEV, generator=gen)[: N // 8]] = 0.0
        del z, near, top
    return c


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        from kubeoperator_amd.ops import functional as kf

        if s["op"] == "prefix":
            return kf.prefix_attention(s["q"], s["kp"], s["vp"], s["kc"], s["vc"], s["lens"], s["own"], s["T"], s["scale"])
        if s["op"] == "lora":
            return kf.lora_add(s["y"], s["x"], s["a"], s["b"], s["index"], s["alpha"])
        if s["op"] == "verify":
            return kf.verify_draft(s["target"], s["draft"], s["tokens"], s["u"], s["temp"])
        return kf.distill_topk(s["logits"], s["index"], s["teacher"], s["temp"], s["weight"])
    return {"prefix": _prefix, "lora": _lora, "verify": _verify, "distill": _distill}[s["op"]](s)


def _prefix(s):
    B, T, Hq, Hkv, D, P = (s[k] for k in ("B", "T", "Hq", "Hkv", "D", "P"))
    G, n = Hq // Hkv, s["own"]
    q = s["q"].float().reshape(B, T, Hkv, G, D) * s["scale"]
    # the prefix: one product for all sequences' rows
    sp = torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(Hkv, B * T * G, D), s["kp"].float().transpose(1, 2))
    sp = sp.reshape(Hkv, B, T, G, P).permute(1, 0, 2, 3, 4)
    # each sequence's own keys: token t of T sees len - (T - 1 - t) of them
    kc, vc = s["kc"][:, :, :n].float(), s["vc"][:, :, :n].float()
    so = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, D), kc.transpose(2, 3)).reshape(B, Hkv, T, G, n)
    seen = s["lens"].view(B, 1) - (T - 1) + torch.arange(T, device=q.device)
    so = so.masked_fill(torch.arange(n, device=q.device) >= seen.view(B, 1, T, 1, 1), float("-inf"))
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    ep, eo = torch.exp(sp - m), torch.exp(so - m)
    den = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    op = torch.matmul(ep.permute(1, 0, 2, 3, 4).reshape(Hkv, B * T * G, P), s["vp"].float())
    op = op.reshape(Hkv, B, T, G, D).permute(1, 0, 2, 3, 4)
    oo = torch.matmul(eo.reshape(B, Hkv, T * G, n), vc).reshape(B, Hkv, T, G, D)
    return ((op + oo) / den).permute(0, 2, 1, 3, 4).reshape(B * T, Hq * D).to(s["q"].dtype)


def _lora(s):
    n, r = s["a"].shape[0], s["r"]
    # every adapter's product with every row, the row's own kept
    h = torch.matmul(s["x"].float(), s["a"].float().reshape(n * r, -1).t()).view(-1, n, r)
    mine = s["index"].view(-1, 1) == torch.arange(n, device=h.device, dtype=torch.int32)
    h = torch.where(mine.unsqueeze(-1), h * s["alpha"].view(1, n, 1), torch.zeros((), device=h.device))
    d = torch.matmul(h.reshape(-1, n * r), s["b"].float().transpose(1, 2).reshape(n * r, -1))
    return (s["y"].float() + d).to(s["y"].dtype)


def _verify(s):
    B, T, V = s["B"], s["T"], s["V"]
    z, row = s["target"], torch.arange(B, device=s["target"].device)
    if s["temp"] == 0:
        best = z.float().argmax(-1)
        ok = s["tokens"] == best[:, :T]
    else:  # probabilities and running sums in 64 bits: the drawn number lies between sums of up to 128k of them
        p = z.double() / s["temp"]
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        q = s["draft"].double() / s["temp"]
        q = torch.exp(q - q.amax(-1, keepdim=True))
        q = q / q.sum(-1, keepdim=True)
        at = s["tokens"].unsqueeze(-1)
        ok = s["u"][:, :T].double() * q.gather(-1, at).squeeze(-1) < p[:, :T].gather(-1, at).squeeze(-1)
    took = ok.long().cumprod(-1).sum(-1) if T else torch.zeros(B, dtype=torch.int64, device=z.device)
    if s["temp"] == 0:
        last = best[row, took]
    else:
        q = torch.cat([q, torch.zeros_like(p[:, :1])], 1)
        rest = (p[row, took] - q[row, took]).clamp_min(0)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p[row, took])
        run_sum = rest.cumsum(-1)
        hit = (run_sum > s["u"][:, T:].double() * run_sum[:, -1:]) & (rest > 0)
        last = hit.to(torch.uint8).argmax(-1)
    col = torch.arange(T + 1, device=z.device)
    tok = torch.cat([s["tokens"], torch.zeros(B, 1, dtype=torch.int64, device=z.device)], 1)
    out = torch.where(col < took.unsqueeze(1), tok, torch.where(col == took.unsqueeze(1), last.unsqueeze(1), -1))
    return out, took.to(torch.int32)


def _distill(s):
    t, at = s["temp"], s["index"].long()
    z = s["logits"].float() / t
    lse = torch.log(torch.exp(z - z.amax(-1, keepdim=True)).sum(-1, keepdim=True)) + z.amax(-1, keepdim=True)
    w = s["teacher"] / t
    w = w - w.amax(-1, keepdim=True)
    logp = w - torch.log(torch.exp(w).sum(-1, keepdim=True))
    p = torch.exp(logp)
    rows = s["weight"].unsqueeze(1)
    loss = (p * (logp - (z.gather(-1, at) - lse))).sum(-1) * s["weight"] * (t * t)
    grad = torch.exp(z - lse).scatter_add_(-1, at, -p) * (rows * t)
    return loss, grad.to(s["logits"].dtype)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(c):
    if c["op"] == "prefix":
        B, T, Hq, Hkv, D = (c[k] for k in ("B", "T", "Hq", "Hkv", "D"))
        total = B * (T + c["own"]) / 2 if B > 1 else c["own"]  # lengths spread evenly over [T, own]
        return {"bytes": 2 * (2 * Hkv * D * (c["P"] + total) + 2 * B * T * Hq * D), "flops": 4.0 * T * Hq * D * (B * c["P"] + total)}
    if c["op"] == "lora":
        M, n, r, K, N = (c[k] for k in ("M", "n", "r", "K", "N"))
        used = n * (1 - (1 - 1 / (n + 1)) ** (2 * n + 1 if c["runs"] else M))  # adapters that some row has
        return {"bytes": 2 * (M * K + 2 * M * N + used * r * (K + N)), "flops": 2.0 * M * r * (K + N)}
    if c["op"] == "verify":
        size = 4 if c["dtype"] == "float32" else 2
        rows = c["B"] * (c["T"] + 1 + (c["T"] if c["temp"] > 0 else 0))
        return {"bytes": rows * c["V"] * size, "flops": 4.0 * rows * c["V"]}
    return {"bytes": c["N"] * (c["V"] * 4 + c["K"] * 8), "flops": 6.0 * c["N"] * c["V"]}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    """The same outputs from the definitions, sequence by sequence and adapter by adapter, in 64 bits."""
    if case["op"] == "verify":
        return None  # whole numbers only
    s = prepare(case, seed)
    if case["op"] == "prefix":
        B, T, Hq, Hkv, D = (s[k] for k in ("B", "T", "Hq", "Hkv", "D"))
        if B * T * Hq > 40000:
            return None
        lens, out = s["lens"].tolist(), torch.zeros(B * T, Hq, D, dtype=torch.float64, device=DEV)
        group = torch.arange(Hq, device=DEV) // (Hq // Hkv)
        for b in range(B):
            k = torch.cat([s["kp"], s["kc"][b, :, : lens[b]]], 1).double()
            v = torch.cat([s["vp"], s["vc"][b, :, : lens[b]]], 1).double()
            for t in range(T):
                seen = k.shape[1] - (T - 1 - t)
                score = (k[group, :seen] @ s["q"][b * T + t].double().view(Hq, D, 1)).squeeze(-1) * s["scale"]
                out[b * T + t] = (torch.softmax(score, -1).unsqueeze(1) @ v[group, :seen]).squeeze(1)
        return out.view(B * T, Hq * D)
    if case["op"] == "lora":
        out = s["y"].double()
        for i in range(case["n"]):
            rows = torch.nonzero(s["index"] == i).flatten()
            if len(rows):
                low = s["x"][rows].double() @ s["a"][i].double().t()
                out[rows] += s["alpha"][i].double() * (low @ s["b"][i].double().t())
        return out
    N, V, t = case["N"], case["V"], case["temp"]
    loss = torch.empty(N, dtype=torch.float64, device=DEV)
    grad = torch.empty(N, V, dtype=torch.float64, device=DEV)
    for at in range(0, N, 1024):
        rows = slice(at, min(N, at + 1024))
        q = torch.log_softmax(s["logits"][rows].double() / t, -1)
        p = torch.log_softmax(s["teacher"][rows].double() / t, -1)
        idx, w = s["index"][rows].long(), s["weight"][rows].double()
        loss[rows] = t * t * w * (p.exp() * (p - q.gather(-1, idx))).sum(-1)
        g = q.exp()
        g.scatter_add_(-1, idx, -p.exp())
        grad[rows] = g * (w * t).unsqueeze(1)
    return loss, grad
