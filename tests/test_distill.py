"""Distillation from a teacher's top logits (``ops.distill_topk``): loss and gradient against the formula in 64 bits, the
gradient against differences of the 64-bit loss, padding / weights / repeated tokens / masked logits, in place, strided
and captured calls, refusals, and the LM-head form's gradients.

Tolerances (u = 2^-24, the fp32 half step; 2^-8 the bf16 one): with R the largest magnitude of an exponent's argument
(in log2 units) the argument carries at most 3 roundings of R u, the exponential 2 u more, and a sum of n terms in chains of
c = max(64, n / 512) plus a 16-step tree (c + 16) u relative -- all terms are positive. So q and p are off by at most
E = (3 R ln 2 + c + 24) u relative, log q and log p by E plus 2 R u absolute, and the loss by
t^2 w sum_k p_k (E |log p_k - log q_k| + 2 E + 4 R u) + (K + 16) u |terms|; the gradient by t w (q + P) E and its
rounding to bf16, 2^-8 of itself."""
import math

import pytest
import torch

from kubeoperator_amd import ops
from kubeoperator_amd.ops import functional as kf

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def oracle(logits, index, teacher, t, weight):
    """(loss, gradient, loss tolerance, gradient tolerance) in 64 bits, row by row."""
    N, V = logits.shape
    z, T = logits.double().cpu() / t, teacher.double().cpu() / t
    loss, grad = torch.zeros(N, dtype=torch.float64), torch.zeros(N, V, dtype=torch.float64)
    ltol, gtol = torch.zeros(N, dtype=torch.float64), torch.zeros(N, V, dtype=torch.float64)
    w = torch.ones(N, dtype=torch.float64) if weight is None else weight.double().cpu()
    for i in range(N):
        idx = index[i].cpu().long()
        ok = (idx >= 0) & (idx < V) & (T[i] > -float("inf"))
        if w[i] == 0 or not ok.any():
            continue
        idx, tl = idx[ok], T[i][ok]
        lp = torch.log_softmax(tl, 0)
        lse = torch.logsumexp(z[i], 0)
        lse = lse if lse > -float("inf") else torch.tensor(float("inf"), dtype=torch.float64)
        q, lq = torch.exp(z[i] - lse), z[i][idx] - lse
        P = torch.zeros(V, dtype=torch.float64).index_add_(0, idx, lp.exp())
        term = torch.where(lp.exp() > 0, lp - lq, torch.zeros_like(lp))
        loss[i] = t * t * w[i] * (lp.exp() * term).sum()
        grad[i] = t * w[i] * (q - P)
        fin = z[i][torch.isfinite(z[i])]
        R = 1.4427 * (2 * max(float(fin.abs().max()) if len(fin) else 0.0, float(tl.abs().max())) + 20)
        E = (3 * R * 0.7 + max(64, V / 512) + 24) * U
        fterm = torch.where(torch.isfinite(term), term, torch.zeros_like(term))
        ltol[i] = t * t * w[i].abs() * (lp.exp() * (E * fterm.abs() + 2 * E + 4 * R * U)
                                       + (len(idx) + 16) * U * lp.exp() * fterm.abs()).sum()
        gtol[i] = t * w[i].abs() * (q + P) * (2 * E) + 2.0 ** -8 * grad[i].abs()
    return loss, grad, ltol, gtol


def make(N, V, K, dev, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (spread * torch.randn(N, V, generator=g)).bfloat16().to(dev)
    index = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)]).to(torch.int32).to(dev)
    teacher = (2.0 * torch.randn(N, K, generator=g)).to(dev)
    weight = (torch.rand(N, generator=g) + 0.25).to(dev)
    return logits, index, teacher, weight


def check(logits, index, teacher, t, weight, out=None):
    want = oracle(logits, index, teacher, t, weight)
    got = kf.distill_topk(logits, index, teacher, t, weight, out)
    for x, y, tol, what in ((got[0], want[0], want[2], "loss"), (got[1], want[1], want[3], "gradient")):
        x = x.double().cpu()
        assert torch.equal(torch.isfinite(x), torch.isfinite(y)), what
        fin = torch.isfinite(y)
        bad = (x - y).abs()[fin] - tol[fin]
        assert bad.max() <= 0, (what, bad.max(), (x - y).abs().max())
    return got


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("N,V,K,t", [(1, 1, 1, 1.0), (3, 7, 7, 1.0), (2, 8, 1, 0.5), (5, 512, 8, 2.0), (4, 1000, 128, 1.0),
                                     (3, 50257, 32, 2.0), (2, 50304, 512, 1.0), (3, 65536, 16, 1.0), (300, 520, 9, 1.0), (2, 1032, 9, 1.0), (2, 2055, 9, 1.0), (2, 4104, 9, 1.0),
                                     (260, 9000, 4, 1.0), (2, 9000, 4, 1.0), (258, 32776, 4, 1.0), (2, 32776, 4, 1.0), (2, 65544, 16, 0.7),
                                     (2, 128256, 64, 1.0), (1, 131072, 8, 1.0), (1, 131080, 8, 4.0), (1, 300001, 5, 1.0)])
def test_matches_the_formula(dev, N, V, K, t):
    check(*make(N, V, K, dev)[:3], t, make(N, V, K, dev)[3])
    check(*make(N, V, K, dev, seed=1)[:3], t, None)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [65545, 128251])
def test_many_long_rows(V):
    """More long rows than the chip has CUs take a form of their own."""
    logits, index, teacher, weight = make(258, V, 8, "cuda")
    weight[3] = 0
    logits[7, 100:] = float("-inf")
    check(logits, index, teacher, 1.5, weight)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("V", [40, 4099, 50304, 128256])
def test_padding_weights_repeats_and_masked_logits(dev, V):
    logits, index, teacher, weight = make(9, V, 12, dev)
    index[0] = -1                       # nothing listed
    index[1, 3:] = -7                   # three entries
    index[2, ::2] = index[2, 1]         # the same token again and again
    index[3, 5] = V                     # outside the vocabulary
    teacher[3, 6:] = float("nan")
    teacher[4, 1:] = float("-inf")      # a teacher that is certain
    weight[5] = 0.0
    logits[6] = float("-inf")           # no student probability at all: infinite loss, finite gradient
    logits[7, : V // 2] = float("-inf")
    index[7] = torch.arange(V - 12, V, dtype=torch.int32)
    teacher[8] = torch.finfo(torch.float32).min  # all at the type's lowest value: uniform
    loss, grad = check(logits, index, teacher, 1.3, weight)
    assert loss[0] == 0 and loss[5] == 0 and not grad[0].any() and not grad[5].any()
    assert loss[6] == float("inf") and torch.isfinite(grad.float()).all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("V", [1001, 4096, 50304, 128256])
def test_strided_rows_other_outputs_and_in_place(dev, V):
    logits, index, teacher, weight = make(4, V, 9, dev)
    wide = torch.full((4, V + 24), float("nan"), dtype=torch.bfloat16, device=dev)
    wide[:, 8:8 + V] = logits
    view = wide[:, 8:8 + V]
    base = check(logits, index, teacher, 1.0, weight)
    a = kf.distill_topk(view, index, teacher, 1.0, weight)
    wout = torch.full((4, V + 3), 7.0, dtype=torch.bfloat16, device=dev)
    b = check(view, index, teacher, 1.0, weight, out=wout[:, 1:1 + V])  # rows that start off the 16-byte grid
    assert b[1].data_ptr() == wout[:, 1:].data_ptr() and (wout[:, 0] == 7).all() and (wout[:, V + 1:] == 7).all()
    c = kf.distill_topk(view, index, teacher, 1.0, weight, out=view)
    assert torch.equal(a[0], base[0]) and torch.equal(a[1], base[1])  # the same rows: the same bits
    assert torch.equal(c[0], base[0]) and torch.equal(view, base[1])
    assert torch.isnan(wide[:, :8]).all() and torch.isnan(wide[:, 8 + V:]).all()


@pytest.mark.parametrize("dev", DEVS)
def test_gradient_matches_differences(dev):
    logits, index, teacher, weight = make(3, 24, 6, dev, spread=1.0)
    index[1, 1] = index[1, 0]
    t = 1.5
    grad = kf.distill_topk(logits, index, teacher, t, weight)[1].double().cpu()
    h = 1e-5
    for i in range(3):
        for v in range(24):
            d = torch.zeros_like(logits, dtype=torch.float64)
            d[i, v] = h
            up = oracle(logits.double() + d, index, teacher, t, weight)[0][i]
            dn = oracle(logits.double() - d, index, teacher, t, weight)[0][i]
            num = float((up - dn) / (2 * h))
            # rounding to bf16, plus h^2 / 6 of a third derivative below t^2 and the differences' own 1e-15 / h
            assert abs(float(grad[i, v]) - num) <= 2.0 ** -8 * abs(num) + 1e-5, (i, v)


@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    logits, index, teacher, weight = make(4, 64, 6, dev)
    bad = [
        lambda: kf.distill_topk(logits.view(2, 2, 64), index, teacher),
        lambda: kf.distill_topk(logits, index.long(), teacher),
        lambda: kf.distill_topk(logits, index, teacher.double()),
        lambda: kf.distill_topk(logits, index[:3], teacher[:3]),
        lambda: kf.distill_topk(logits, index[:, :0], teacher[:, :0]),
        lambda: kf.distill_topk(logits, index[:, :5], teacher),
        lambda: kf.distill_topk(logits, index, teacher, 0.0),
        lambda: kf.distill_topk(logits, index, teacher, float("nan")),
        lambda: kf.distill_topk(logits, index, teacher, 1.0, weight[:3]),
        lambda: kf.distill_topk(logits, index, teacher, 1.0, weight, out=logits[:3]),
        lambda: kf.distill_topk(logits, index.repeat(1, 100), teacher.repeat(1, 100)),
        lambda: kf.distill_topk(logits.clone().requires_grad_(), index, teacher),
    ]
    if dev == "cuda":
        wide = torch.zeros(4, 72, dtype=torch.bfloat16, device=dev)
        bad += [lambda: kf.distill_topk(logits.float(), index, teacher),
                lambda: kf.distill_topk(logits, index.cpu(), teacher),
                lambda: kf.distill_topk(wide[:, :64], index, teacher, out=wide[:, 8:])]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    assert kf.distill_topk(logits[:0], index[:0], teacher[:0])[1].shape == (0, 64)


@pytest.mark.parametrize("dev", DEVS)
def test_teacher_and_weights_have_no_gradient(dev):
    logits, index, teacher, weight = make(4, 64, 6, dev)
    x, w = logits.clone(), torch.zeros(64, 64, dtype=torch.bfloat16, device=dev)
    for f in (lambda t, v: kf.distill_topk(logits, index, t, 1.0, v),
              lambda t, v: kf.distill_topk_lmhead(x, w, index, t, 1.0, v)):
        for t, v in ((teacher.clone().requires_grad_(), weight), (teacher, weight.clone().requires_grad_())):
            with pytest.raises(RuntimeError, match="detach"):
                f(t, v)
            with torch.no_grad():
                f(t, v)
    with pytest.raises(RuntimeError):
        kf.distill_topk(logits, index, teacher, 1.0, weight, out=logits.clone().requires_grad_())


@pytest.mark.parametrize("dev", DEVS)
def test_lmhead_gradients(dev):
    """x and w gradients through the LM head against the 64-bit gradient of the logits that the product gives, and an
    upstream factor; grad_fn of the same leaves may be used for several calls."""
    N, H, V, K = 24, 64, 200, 7
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, N // 2, H, generator=g).bfloat16().to(dev).requires_grad_()
    w = (0.2 * torch.randn(V, H, generator=g)).bfloat16().to(dev).requires_grad_()
    _, index, teacher, weight = make(N, V, K, dev, seed=5)
    for wt in (weight, None):
        x.grad = w.grad = None
        loss = ops.distill_topk_lmhead(x, w, index, teacher, 2.0, wt)
        (loss * 3.0).backward()
        eff = wt if wt is not None else torch.full((N,), 1.0 / N, device=dev)
        logits = torch.mm(x.detach().view(N, H), w.detach().t())
        l64, g64, ltol, _ = oracle(logits, index, teacher, 2.0, eff)
        assert abs(float(loss.detach()) - float(l64.sum())) <= float(ltol.sum()) + 64 * U * float(l64.abs().sum())
        g64 = 3.0 * g64
        X, W = x.detach().double().cpu().view(N, H), w.detach().double().cpu()
        for got, want, mag in ((x.grad.view(N, H), g64 @ W, g64.abs() @ W.abs()), (w.grad, g64.t() @ X, g64.abs().t() @ X.abs())):
            # three bf16 roundings on the way: the gradient of the logits, the upstream factor, the result
            err = (got.double().cpu() - want).abs() - (2.1 * 2.0 ** -8 * mag + 2.0 ** -8 * want.abs() + 1e-6)
            assert err.max() <= 0, err.max()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Logits of more than 2^31 elements, in place: the last rows against the formula."""
    N, V, K = 17000, 128256, 4
    rows, index, teacher, _ = make(3, V, K, "cuda")
    logits = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
    logits[-3:] = rows
    idx, tea = index[:1].repeat(N, 1), teacher[:1].repeat(N, 1)
    idx[-3:], tea[-3:] = index, teacher
    want = oracle(rows, index, teacher, 1.0, None)
    loss, grad = kf.distill_topk(logits, idx, tea, 1.0, None, out=logits)
    assert ((loss[-3:].double().cpu() - want[0]).abs() - want[2]).max() <= 0
    assert ((grad[-3:].double().cpu() - want[1]).abs() - want[3]).max() <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1000, 50304, 128256])
def test_captured_call_replays_and_another_stream(V):
    logits, index, teacher, weight = make(6, V, 9, "cuda")
    want = kf.distill_topk(logits, index, teacher, 1.0, weight)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = kf.distill_topk(logits, index, teacher, 1.0, weight)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    static = logits.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kf.distill_topk(static, index, teacher, 1.0, weight)
    for seed in (0, 4, 5):
        static.copy_(make(6, V, 9, "cuda", seed=seed)[0])
        eager = kf.distill_topk(static, index, teacher, 1.0, weight)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("V", [40, 2055, 50304, 65545, 300001])
@pytest.mark.parametrize("t", [1e-2, 1e-4])
@pytest.mark.parametrize("offset", [0.0, 50.0, -50.0])
def test_low_temperatures(dev, V, t, offset):
    """What the student's logits have in common, and how large it is next to the temperature, takes nothing from the result: only
    differences from the row's maximum enter.

    Tolerance: such a difference d, over t, carries 5 roundings (the difference, t, 1 / t, log2 e, the product); where it counts (a
    weight of 2^-24 of the row's and more) it is at most 24 ln 2 + ln V, so q is off by E = 5 (24 ln 2 + ln V) u, 2 u of the
    exponential and c + 16 of the sum, relative, q smaller than 2^-24 by 2^-24 altogether; P likewise with T's differences (at
    most 40 ln 2 before its weight is nothing); log q_k by 5 u |log q_k| + E. Logits a step of bf16 apart (0.25 at 50) are far
    apart in units of t: the rows get pairs of equal maxima, so that q is not all 0 and 1."""
    N, K = 6, 9
    logits, index, teacher, weight = make(N, V, K, dev, seed=7)
    logits += offset
    teacher = teacher * t  # the teacher's own distribution keeps its shape
    top = logits.float().argmax(-1)
    for i in range(N):
        for j in range(i):  # rows with 1 + i maxima, some of them listed
            logits[i, (int(top[i]) + 3 * j + 1) % V] = logits[i, int(top[i])]
        index[i, 0] = int(top[i])
        index[i, 1] = (int(top[i]) + 1) % V
    loss, grad = kf.distill_topk(logits, index, teacher, t, weight)
    z, T, w = logits.double().cpu() / t, teacher.double().cpu() / t, weight.double().cpu()
    c = max(64, V / 512)
    E = (5 * (24 * 0.7 + math.log(V)) + 2 + c + 16) * U
    EP = (5 * 40 * 0.7 + 2 + K + 16) * U
    lq, lp = torch.log_softmax(z, -1), torch.log_softmax(T, -1)
    q, P = lq.exp(), torch.zeros_like(z).scatter_add_(1, index.cpu().long(), lp.exp())
    g = (q - P) * (t * w).unsqueeze(1)
    slack = (E * q + 2.0 ** -24 * (q < 2.0 ** -24) + EP * P) * (t * w).unsqueeze(1)
    err = (grad.double().cpu() - g).abs() - (2.0 ** -8 * (g.abs() + slack) + slack + 2.0 ** -133)
    assert err.max() <= 0, float(err.max())
    k = lq.gather(1, index.cpu().long())
    want = t * t * w * (lp.exp() * (lp - k)).sum(-1)
    tol = t * t * w * (lp.exp() * (EP * (lp - k).abs() + 5 * U * k.abs() + E + EP + 5 * U * lp.abs())).sum(-1)
    tol += (K + 16) * U * t * t * w * (lp.exp() * (lp - k).abs()).sum(-1)
    assert ((loss.double().cpu() - want).abs() <= tol).all(), ((loss.double().cpu() - want).abs() / tol).max()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("V", [40, 4099, 300001])
@pytest.mark.parametrize("t", [0.5, 1.0])
def test_rows_of_the_lowest_value(dev, V, t):
    """Logits at the type's lowest value (a mask) are finite: a row of nothing else is uniform, beside others they weigh nothing."""
    logits, index, teacher, _ = make(3, V, 5, dev)
    logits[0] = torch.finfo(torch.bfloat16).min
    logits[1, : V // 2] = torch.finfo(torch.bfloat16).min
    index[1] = torch.arange(V - 5, V, dtype=torch.int32)
    logits[2] = torch.finfo(torch.bfloat16).max
    got = kf.distill_topk(logits, index, teacher, t)
    logits[0] = 0.0
    logits[1, : V // 2] = float("-inf")
    logits[2] = 0.0
    want = kf.distill_topk(logits, index, teacher, t)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
