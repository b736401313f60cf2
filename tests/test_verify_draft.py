"""Verification of drafted tokens (``ops.verify_draft``): whole numbers, equal to a plain 64-bit implementation. The
running sums of both are in 64 bits (relative error below 1e-12), so a uniform number would have to lie within 1e-12 of one of
the borders for the two to differ."""
import math

import numpy as np
import pytest
import torch

from kubeoperator_amd.ops import functional as kf

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
FMAX = float(torch.finfo(torch.float32).max)


def plain(target, draft, tokens, u, temp, n_draft):
    def clean(z):
        z = np.where(np.isnan(z), -np.inf, z)
        return np.minimum(z, FMAX)

    def probs(z):
        z = clean(z)
        if z.max() == -np.inf:
            return np.zeros_like(z)
        with np.errstate(over="ignore", under="ignore"):
            e = np.exp((z - z.max()) / temp)
        return e / math.fsum(e)

    tgt = target.float().cpu().double().numpy()
    drf = draft.float().cpu().double().numpy() if draft is not None else None
    tok, uu = tokens.cpu().numpy(), u.cpu().double().numpy()
    B, T1, V = tgt.shape
    out, took = np.full((B, T1), -1, np.int64), np.zeros(B, np.int32)
    for b in range(B):
        nd = T1 - 1 if n_draft is None else min(max(int(n_draft[b]), 0), T1 - 1)
        j = 0
        for j in range(nd + 1):
            p = probs(tgt[b, j]) if temp else None
            best = int(clean(tgt[b, j]).argmax()) if clean(tgt[b, j]).max() > -np.inf else -1
            if j == nd:
                break
            x = int(tok[b, j])
            if not 0 <= x < V:
                break
            if temp == 0:
                if x != best:
                    break
            elif not uu[b, j] * probs(drf[b, j])[x] < p[x]:
                break
        if temp == 0:
            nxt = best
        else:
            r = np.maximum(p - probs(drf[b, j]), 0) if j < nd else p
            if not r.sum() > 0:
                r = p
            c = np.cumsum(r)
            hit = np.nonzero((c > uu[b, -1] * c[-1]) & (r > 0))[0]
            nxt = int(hit[0]) if len(hit) else (int(np.nonzero(r > 0)[0][-1]) if (r > 0).any() else -1)
        out[b, :j] = tok[b, :j]
        out[b, j] = nxt
        took[b] = j
    return torch.from_numpy(out), torch.from_numpy(took)


def make(B, T, V, dev, dtype=torch.float32, seed=0, temp=1.0, spread=3.0, apart=0.5):
    g = torch.Generator().manual_seed(seed)
    z = spread * torch.randn(B, T + 1, V, generator=g)
    target = z.to(dtype)
    draft = (z[:, :T] + apart * torch.randn(B, T, V, generator=g)).to(dtype)
    if T:
        tokens = torch.distributions.Categorical(logits=draft.float().view(-1, V) / (temp or 1.0))
        torch.manual_seed(seed)
        tokens = tokens.sample().view(B, T) if temp else draft.float().argmax(-1)
    else:
        tokens = torch.zeros(B, 0, dtype=torch.int64)
    u = torch.rand(B, T + 1, generator=g)
    return target.to(dev), draft.to(dev), tokens.to(dev), u.to(dev)


def check(target, draft, tokens, u, temp, n_draft=None):
    out, took = kf.verify_draft(target, draft, tokens, u, temp, n_draft)
    want = plain(target, draft, tokens, u, temp, n_draft)
    assert out.dtype == torch.int64 and took.dtype == torch.int32
    assert torch.equal(took.cpu(), want[1]), (took, want[1])
    assert torch.equal(out.cpu(), want[0]), (out, want[0])
    return out, took


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,V,temp", [(1, 0, 1, 1.0), (1, 0, 33, 1.0), (3, 1, 5, 1.0), (5, 3, 511, 0.7), (4, 4, 8192, 1.0),
                                        (2, 2, 8193, 1.3), (2, 8, 50257, 0.3), (2, 3, 128256, 1.0), (3, 32, 300, 1.0),
                                        (4, 3, 1000, 0.0), (2, 5, 50304, 0.0), (1, 0, 128256, 0.0), (3, 3, 4096, 1.0),
                                        (3, 3, 4097, 1.0), (2, 4, 3640, 0.8), (2, 4, 3641, 0.8), (3, 2, 4096, 0.0),
                                        (2, 1, 300001, 1.0), (70, 2, 255, 1.0)])
def test_matches_plain(dev, dtype, B, T, V, temp):
    for seed in range(3):
        check(*make(B, T, V, dev, dtype, seed, temp), temp)


@pytest.mark.parametrize("dev", DEVS)
def test_flat_and_certain_distributions(dev):
    t, d, k, u = make(3, 3, 4000, dev, spread=0.0, apart=0.0)  # equal everywhere: all kept, next one from a flat row
    _, took = check(t, d, k, u, 1.0)
    assert took.tolist() == [3, 3, 3]
    t, d, k, u = make(3, 3, 4000, dev, spread=40.0, apart=30.0)  # one token holds everything
    check(t, d, k, u, 1.0)
    check(t, d, k, u, 1e-3)
    check(t, d, k, u, 100.0)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("temp", [0.0, 0.9])
def test_masks_ties_ragged_drafts_and_bad_tokens(dev, temp):
    B, T, V = 12, 4, 9000
    t, d, k, u = make(B, T, V, dev, temp=1.0)
    t[0, 0] = float("-inf")              # no token possible
    t[1, 0, 1:] = float("-inf")          # only token 0
    k[1, 0] = 5
    t[2, 0, ::3] = float("nan")
    t[3, 1, 100:8800] = float("-inf")
    t[4, 0, 7] = float("inf")
    t[4, 0, 8500] = float("inf")
    d[5, 0] = float("-inf")              # a draft row without any probability
    d[6, 0, k[6, 0]] = float("-inf")     # the drafted token has none
    k[7, 1] = -1
    k[8, 0] = V
    t[9, 0] = 2.0                        # a flat row: ties
    k[9, 0] = 0
    t[10, 0] = torch.finfo(torch.float32).min
    u[11] = torch.tensor([0.0, 0.0, 1.0, float("nan"), 1.0])
    check(t, d if temp else None, k, u, temp)
    n = torch.tensor([0, 1, 2, 3, 4, 9, -2, 1, 4, 4, 0, 2], dtype=torch.int32, device=dev)
    out, took = check(t, d, k, u, temp, n)
    assert (took <= n.clamp(0, T)).all()
    u[:, -1] = torch.linspace(-0.5, 1.5, B)  # outside [0, 1): the first or the last token with any probability
    check(t, d, k, u, temp, n)


@pytest.mark.parametrize("dev", DEVS)
def test_strided_logits(dev):
    t, d, k, u = make(3, 2, 777, dev)
    both = torch.full((3, 5, 800), float("nan"), device=dev)
    both[:, :3, 3:780] = t
    both[:, 3:, 3:780] = d
    a = kf.verify_draft(both[:, :3, 3:780], both[:, 3:, 3:780], k, u)
    b = check(t, d, k, u, 1.0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # the same row for every sequence
    e = t[:1].expand(3, 3, 777)
    check(e, d, k, u, 1.0)


@pytest.mark.parametrize("dev", DEVS)
def test_outputs_follow_the_target(dev):
    """Tokens drawn by the draft and verified are distributed as the target's own samples: 4096 trials of one token over 6;
    each count is binomial, 5 standard deviations apart at most."""
    n = 4096
    p = torch.tensor([0.30, 0.05, 0.25, 0.20, 0.15, 0.05])
    q = torch.tensor([0.05, 0.30, 0.15, 0.30, 0.05, 0.15])
    g = torch.Generator().manual_seed(11)
    k = torch.multinomial(q, n, replacement=True, generator=g).view(n, 1)
    u = torch.rand(n, 2, generator=g)
    t = p.log().view(1, 1, 6).expand(n, 2, 6).contiguous().to(dev)
    out, _ = kf.verify_draft(t, q.log().view(1, 1, 6).expand(n, 1, 6).to(dev), k.to(dev), u.to(dev))
    count = torch.bincount(out[:, 0].cpu(), minlength=6).double()
    sd = (n * p.double() * (1 - p.double())).sqrt()
    assert ((count - n * p.double()).abs() <= 5 * sd).all(), (count, n * p)


@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    t, d, k, u = make(2, 3, 50, dev)
    bad = [
        lambda: kf.verify_draft(t[0], d, k, u),
        lambda: kf.verify_draft(t, None, k, u),
        lambda: kf.verify_draft(t, d[:, :2], k, u),
        lambda: kf.verify_draft(t, d.bfloat16(), k, u),
        lambda: kf.verify_draft(t.double(), d.double(), k, u),
        lambda: kf.verify_draft(t, d, k.int(), u),
        lambda: kf.verify_draft(t, d, k[:, :2], u),
        lambda: kf.verify_draft(t, d, k, u[:, :3]),
        lambda: kf.verify_draft(t, d, k, u.double()),
        lambda: kf.verify_draft(t, d, k, u, -1.0),
        lambda: kf.verify_draft(t, d, k, u, 1e-9),
        lambda: kf.verify_draft(t, d, k, u, float("nan")),
        lambda: kf.verify_draft(t, d, k, u, 1.0, torch.zeros(3, dtype=torch.int32, device=dev)),
        lambda: kf.verify_draft(t.clone().requires_grad_(), d, k, u),
        lambda: kf.verify_draft(*(x.to(dev) for x in make(1, 33, 8, "cpu"))),
    ]
    if dev == "cuda":
        bad += [lambda: kf.verify_draft(t, d.cpu(), k, u), lambda: kf.verify_draft(t[:, :, ::2], d[:, :, ::2], k, u),
                lambda: kf.verify_draft(t, d, k.cpu(), u)]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    out, took = kf.verify_draft(t[:0], d[:0], k[:0], u[:0])
    assert out.shape == (0, 4) and took.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("temp", [0.0, 1.0])
def test_captured_call_replays_and_another_stream(temp):
    t, d, k, u = make(4, 3, 20000, "cuda")
    want = kf.verify_draft(t, d, k, u, temp)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = kf.verify_draft(t, d, k, u, temp)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kf.verify_draft(t, d, k, u, temp)
    for seed in range(3):
        for a, b in zip((t, d, k, u), make(4, 3, 20000, "cuda", seed=seed)):
            a.copy_(b)
        eager = kf.verify_draft(t, d, k, u, temp)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,low,high", [(40, 3, 7), (40, 7, 3), (5000, 3, 7), (5000, 7, 3), (20000, 3, 7), (20000, 7, 3), (20000, 3, 9000)])
def test_infinity_counts_as_the_largest_value(dev, dtype, V, low, high):
    """+inf and the largest fp32 value are a tie, greedy (the lower index) and sampled (half each); bf16 has no such value."""
    t, d, k, u = make(4, 2, V, dev, dtype)
    t[:, :, low], t[:, :, high] = FMAX if dtype == torch.float32 else torch.finfo(dtype).max, float("inf")
    k[0], k[1], k[2] = min(low, high), max(low, high), torch.tensor([low, high])
    check(t, d, k, u, 0.0)
    check(t, d, k, u, 1.0)
