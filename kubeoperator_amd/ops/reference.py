"""Plain-PyTorch fp32 references of every HIP kernel (numerics oracle + CPU plumbing path).

Each function mirrors the semantics of the corresponding gfx950 kernel exactly (layouts, fused residual,
rotate-half RoPE on the first ``nheads`` heads of a row, GQA head mapping, mean cross-entropy with
ignore_index), computing in fp32 and returning the input dtype.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def rms_norm_ref(x, w, eps=1e-5, residual=None):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    sf = s.float()
    y = sf * torch.rsqrt(sf.pow(2).mean(-1, keepdim=True) + eps) * w.float()
    return y.to(x.dtype), s


def layer_norm_ref(x, w, b, eps=1e-5, residual=None):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    y = F.layer_norm(s.float(), (s.shape[-1],), w.float(), b.float(), eps)
    return y.to(x.dtype), s


def rope_cache(S: int, D: int, theta: float, device=None):
    inv = 1.0 / (theta ** (torch.arange(0, D, 2, dtype=torch.float64, device=device) / D))
    t = torch.arange(S, dtype=torch.float64, device=device)
    ang = torch.outer(t, inv)
    return torch.cos(ang).float().contiguous(), torch.sin(ang).float().contiguous()


def rope_ref(x, cos, sin, S: int, nheads: int, D: int, inverse: bool = False, pos=None):
    """Rotate-half RoPE on the first ``nheads`` heads of each row of x [T, >= nheads*D]; returns new tensor."""
    T = x.shape[0]
    out = x.clone()
    p = pos.long() if pos is not None else torch.arange(T, device=x.device) % S
    c = cos[p].unsqueeze(1)  # [T,1,D/2]
    s = sin[p].unsqueeze(1) * (-1.0 if inverse else 1.0)
    h = x[:, : nheads * D].float().view(T, nheads, D)
    a, b = h[..., : D // 2], h[..., D // 2:]
    rot = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    out[:, : nheads * D] = rot.reshape(T, nheads * D).to(x.dtype)
    return out


def swiglu_ref(gu):
    g, u = gu.float().chunk(2, dim=-1)
    return (F.silu(g) * u).to(gu.dtype)


def gelu_ref(x):
    return F.gelu(x.float(), approximate="tanh").to(x.dtype)


def attention_ref(q, k, v, B, S, Hq, Hkv, D, causal=True, scale=None):
    """q [B*S, >=Hq*D], k/v [B*S, >=Hkv*D] row views -> o [B*S, Hq*D], lse [B, Hq, S] (natural log)."""
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    qh = q[:, : Hq * D].float().reshape(B, S, Hq, D).transpose(1, 2)
    kh = k[:, : Hkv * D].float().reshape(B, S, Hkv, D).transpose(1, 2)
    vh = v[:, : Hkv * D].float().reshape(B, S, Hkv, D).transpose(1, 2)
    rep = Hq // Hkv
    kh = kh.repeat_interleave(rep, dim=1)
    vh = vh.repeat_interleave(rep, dim=1)
    s = torch.matmul(qh, kh.transpose(-1, -2)) * scale
    if causal:
        mask = torch.ones(S, S, dtype=torch.bool, device=q.device).triu(1)
        s = s.masked_fill(mask, float("-inf"))
    lse = torch.logsumexp(s, dim=-1)
    p = torch.softmax(s, dim=-1)
    o = torch.matmul(p, vh).transpose(1, 2).reshape(B * S, Hq * D)
    return o.to(q.dtype), lse


def cross_entropy_ref(logits, targets, ignore_index=-100):
    return F.cross_entropy(logits.float(), targets, ignore_index=ignore_index)


def adamw_ref(master, m, v, g, lr, b1, b2, eps, wd, step, gscale=1.0):
    g = g.float() * gscale
    m.mul_(b1).add_(g, alpha=1 - b1)
    v.mul_(b2).addcmul_(g, g, value=1 - b2)
    bc1 = 1 - b1 ** step
    bc2 = 1 - b2 ** step
    master.mul_(1 - lr * wd)
    master.sub_(lr * (m / bc1) / ((v.sqrt() / math.sqrt(bc2)) + eps))
    return master


def decode_attention_ref(q, k_cache, v_cache, lens, scale):
    """One query row per sequence against its cache: q [B, Hq*D], caches [B, Hkv, Smax, D], lens [B] valid keys."""
    B, Hkv, _, D = k_cache.shape
    Hq = q.shape[1] // D
    out = torch.empty(B, Hq * D, dtype=q.dtype, device=q.device)
    for b in range(B):
        n = int(lens[b])
        qh = q[b].float().view(Hq, 1, D)
        kh = k_cache[b, :, :n].float().repeat_interleave(Hq // Hkv, dim=0)  # [Hq, n, D]
        vh = v_cache[b, :, :n].float().repeat_interleave(Hq // Hkv, dim=0)
        p = torch.softmax((qh @ kh.transpose(1, 2)) * scale, dim=-1)
        out[b] = (p @ vh).reshape(Hq * D).to(q.dtype)
    return out


# ---------------------------------------------------------------------------------------------------
# many requests on one model (serving) and the draft model's training
# ---------------------------------------------------------------------------------------------------
def require(ok, message):
    """The CPU path's argument checks raise what the GPU path's (``csrc/bindings.cpp``) do."""
    if not ok:
        raise RuntimeError(message)


def _forward_only(what, *ts):
    require(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)),
            f"{what} is forward only: it has no gradient")


def prefix_attention_ref(q, k_prefix, v_prefix, k_cache, v_cache, lens, max_len, tokens, scale):
    """One softmax per row over the shared prefix [Hkv, P, D] and the row's own keys: token t of ``tokens`` of sequence b
    sees the first lens[b] - (tokens - 1 - t) rows of its cache. Rows that see nothing are 0."""
    _forward_only("prefix_attention", q, k_prefix, v_prefix, k_cache, v_cache)
    require(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "caches must be contiguous [B, Hkv, Smax, D] and equal")
    B, Hkv, Smax, D = k_cache.shape
    for t in (k_prefix, v_prefix):
        require(t.dim() == 3 and t.shape == (Hkv, k_prefix.shape[1], D),
                "prefix must be [Hkv, P, D] with the cache's heads and head dim, K and V alike")
    require(D in (64, 128), "prefix_attention: head dim must be 64 or 128")
    require(Hkv >= 1, "prefix_attention: the cache has no heads")
    require(q.dim() == 2 and tokens >= 1 and q.shape[0] == B * tokens and lens.numel() == B,
            "prefix_attention: q must have B * tokens rows and lens B entries")
    require(lens.dtype == torch.int32, "lens must be contiguous int32")
    require(q.shape[1] > 0 and q.shape[1] % (Hkv * D) == 0, "prefix_attention: q width must be a multiple of Hkv * D")
    require(0 <= max_len <= Smax, "max_len must be in [0, Smax]")
    Hq = q.shape[1] // D
    out = torch.zeros(B * tokens, Hq, D, dtype=q.dtype, device=q.device)
    P, G = k_prefix.shape[1], Hq // Hkv
    for b in range(B):
        n = min(max(int(lens[b]), 0), max_len)
        k = torch.cat([k_prefix, k_cache[b, :, :n]], 1).float()
        v = torch.cat([v_prefix, v_cache[b, :, :n]], 1).float()
        qb = q[b * tokens:(b + 1) * tokens].float().view(tokens, Hkv, G, D).permute(1, 0, 2, 3)  # [Hkv, tokens, G, D]
        seen = P + (n - tokens + 1 + torch.arange(tokens, device=q.device)).clamp(min=0)  # keys each token sees
        top, late = int(seen[-1]), int(seen[0])
        if not top:
            continue
        hidden = torch.arange(top, device=q.device) >= seen.unsqueeze(1)  # [tokens, top]
        # values that only some tokens see: those that are not finite must not reach the others as 0 times NaN
        bad = ~torch.isfinite(v[:, late:top])
        v[:, late:top] = v[:, late:top].masked_fill(bad, 0.0)
        s = torch.matmul(qb.reshape(Hkv, tokens * G, D), k[:, :top].transpose(1, 2)) * scale
        s = s.view(Hkv, tokens, G, top).masked_fill(hidden.view(1, tokens, 1, top), float("-inf"))
        o = torch.matmul(torch.softmax(s, -1).view(Hkv, tokens * G, top), v[:, :top]).view(Hkv, tokens, G, D)
        if bool(bad.any()):
            hit = torch.matmul((~hidden[:, late:]).float(), bad.float()) > 0  # [Hkv, tokens, D]
            o = o.masked_fill(hit.unsqueeze(2), float("nan"))
        o = o.masked_fill((seen == 0).view(1, tokens, 1, 1), 0.0)
        out[b * tokens:(b + 1) * tokens] = o.permute(1, 0, 2, 3).reshape(tokens, Hq, D).to(q.dtype)
    return out.view(B * tokens, Hq * D)


def lora_add_ref(y, x, a, b, index, scale, out=None):
    """out[i] = y[i] + scale[j] b[j] (a[j] x[i]) with j = index[i]; rows whose j is outside [0, n) keep y."""
    _forward_only("lora_add", y, x, a, b, out)
    require(y.dim() == 2 and x.dim() == 2 and a.dim() == 3 and b.dim() == 3, "adapters must be contiguous a [n, r, K] and b [n, N, r]")
    n, r, K = a.shape
    require(x.shape == (y.shape[0], K) and index.shape == (y.shape[0],), "lora_add: x, y and index disagree on the rows")
    require(y.shape[0] <= 32 * (2 ** 24 - 1), "lora_add: too many rows")
    require(b.shape == (n, y.shape[1], r), "lora_add: a must be [n, r, K] and b [n, N, r]")
    require(scale.shape == (n,) and scale.dtype == torch.float32, "lora_add: scale must be [n]")
    require(index.dtype == torch.int32, "index must be contiguous int32")
    require(r >= 8 and r % 8 == 0 and r <= 128, "lora_add: rank must be a multiple of 8 up to 128 (pad a and b with zeros)")
    require(K % 8 == 0 and y.shape[1] % 8 == 0, "lora_add: widths must be multiples of 8")
    require(out is None or out.shape == y.shape, "lora_add: out must have y's shape")
    res = y.float()
    for j in index.unique().tolist():
        if 0 <= j < n:
            rows = torch.nonzero(index == j).flatten()
            res[rows] += scale[j] * (x[rows].float() @ a[j].float().t() @ b[j].float().t())
    res = res.to(y.dtype)
    return res if out is None else out.copy_(res)


def verify_draft_ref(target, draft, tokens, u, temperature, n_draft=None):
    """Accepted prefix of the drafted ``tokens`` [B, T] and the token after it: see ``functional.verify_draft``."""
    _forward_only("verify_draft", target, draft)
    require(target.dim() == 3 and target.shape[1] >= 1 and target.shape[2] >= 1, "target must be [B, T+1, V]")
    require(target.dtype in (torch.float32, torch.bfloat16), "target must be float32 or bfloat16")
    B, T, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    require(T <= 32, "verify_draft: at most 32 drafted tokens")
    require(temperature == 0 or 1e-4 <= temperature <= 1e4, "temperature must be 0 (greedy) or in [1e-4, 1e4]")
    if T > 0 and temperature > 0:
        require(draft is not None, "verify_draft: draft logits are needed unless temperature is 0")
        require(draft.dtype == target.dtype, "draft must have target's dtype")
        require(draft.shape == (B, T, V), "draft must be [B, T, V]")
    require(tokens.dtype == torch.int64 and tokens.shape == (B, T), "tokens must be contiguous int64 [B, T]")
    require(u.dtype == torch.float32 and u.shape == (B, T + 1), "u must be contiguous float32 [B, T+1]")
    require(n_draft is None or (n_draft.shape == (B,) and n_draft.dtype == torch.int32), "n_draft must be [B]")
    out = torch.full((B, T + 1), -1, dtype=torch.int64, device=target.device)
    accepted = torch.zeros(B, dtype=torch.int32, device=target.device)

    def clean(z):
        return torch.nan_to_num(z.float(), nan=float("-inf"), posinf=torch.finfo(torch.float32).max, neginf=float("-inf")).double()

    def probs(z):
        z = clean(z)
        if z.max() == float("-inf"):
            return torch.zeros_like(z)
        e = torch.exp((z - z.max()) / temperature)
        return e / e.sum()

    for b in range(B):
        nd = T if n_draft is None else min(max(int(n_draft[b]), 0), T)
        j, nxt = 0, -1
        while j < nd:
            x = int(tokens[b, j])
            if not 0 <= x < V:
                break
            if temperature == 0:
                z = clean(target[b, j])
                if z.max() == float("-inf") or int(z.argmax()) != x:
                    break
            else:
                if not float(u[b, j]) * float(probs(draft[b, j])[x]) < float(probs(target[b, j])[x]):
                    break
            j += 1
        if temperature == 0:
            z = clean(target[b, j])
            nxt = int(z.argmax()) if z.max() > float("-inf") else -1
        else:
            p = probs(target[b, j])
            r = (p - probs(draft[b, j])).clamp_min(0) if j < nd else p
            if not float(r.sum()) > 0:
                r = p
            if float(r.sum()) > 0:
                c = r.cumsum(0)
                hit = torch.nonzero((c > float(u[b, T]) * float(c[-1])) & (r > 0)).flatten()
                nxt = int(hit[0]) if len(hit) else int(torch.nonzero(r > 0).flatten()[-1])
        out[b, :j] = tokens[b, :j]
        out[b, j] = nxt
        accepted[b] = j
    return out, accepted


def distill_topk_ref(logits, index, teacher, temperature, weight=None, out=None):
    """Loss rows [N] and gradient of the logits [N, V] against a teacher's top logits: see ``functional.distill_topk``."""
    require(logits.dim() == 2 and logits.shape[1] >= 1, "logits must be [N, V] with a contiguous last dimension")
    require(not (logits.requires_grad and torch.is_grad_enabled()),
            "distill_topk returns the gradient itself: detach the logits (distill_topk_lmhead has autograd)")
    N, V = logits.shape
    require(index.dim() == 2 and index.shape == teacher.shape and index.shape[0] == N, "index and teacher must be contiguous [N, K]")
    require(index.dtype == torch.int32 and teacher.dtype == torch.float32, "index must be contiguous int32, teacher float32")
    require(1 <= index.shape[1] <= 512, "distill_topk: 1 to 512 teacher logits per row")
    require(1e-4 <= temperature <= 1e4, "temperature must be in [1e-4, 1e4]")
    require(weight is None or (weight.shape == (N,) and weight.dtype == torch.float32), "weight must be [N]")
    require(out is None or out.shape == logits.shape, "out must have logits' shape, contiguous rows and no overlap")
    w = torch.ones(N, device=logits.device) if weight is None else weight
    real = (index >= 0) & (index < V) & (teacher > float("-inf"))
    live = real.any(-1) & (w != 0)
    at = torch.where(real, index, 0).long()
    lp = torch.log_softmax(torch.where(real, teacher, float("-inf")) / temperature, -1)
    p = torch.where(real & live.unsqueeze(1), torch.exp(lp), 0.0)
    m = logits.float().amax(-1, keepdim=True)
    some = m > float("-inf")  # false: no student probability anywhere, q = 0
    z = (logits.float() - torch.where(some, m, 0.0)) / temperature  # the maximum goes first: m / t takes z's low bits with it
    e = torch.exp(z)
    s = torch.where(some, e.sum(-1, keepdim=True), float("inf"))
    lq = z.gather(-1, at) - torch.log(s)
    loss = torch.where(p > 0, p * (lp - lq), 0.0).sum(-1) * temperature * temperature * w
    grad = (e / s).scatter_add(-1, at, -p) * (temperature * w).unsqueeze(1)
    loss = torch.where(live, loss, 0.0)
    grad = torch.where(live.unsqueeze(1), grad, 0.0).to(logits.dtype)
    return loss, grad if out is None else out.copy_(grad)
