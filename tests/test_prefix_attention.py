"""Attention behind a prefix that the whole batch shares (``ops.prefix_attention``) against one softmax in 64 bits over
prefix and own keys: head layouts, one to many tokens, lengths on and around the 32-key blocks and 128-key steps,
empty prefixes and sequences, stale and non-finite cache rows behind each length, strides, refusals, captured calls.

Tolerance per output, with A = sum_j p_j |v_j|: P is rounded to bf16 (d_j, at most 2^-8 relative) before its product with V
and before its sum, so the quotient is off by sum_j p_j d_j (v_j - o), at most 2^-8 (A + |o|), and the output is rounded once
more (2^-8 |o|); a score is an fp32 sum of D products, scaled (D + 4 roundings of sum |q||k| scale), and the exponential's
argument carries two more roundings of its size, so p is off by e = ((D + 4) max_j sum |q k_j| scale + 4 max |s|) 2^-24 + 2^-22
relative, in the numerator and in the denominator; sums over n keys in fp32 add n 2^-24 to each."""
import math

import pytest
import torch

from kubeoperator_amd.ops import functional as kf

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def make(B, T, Hq, Hkv, D, P, Smax, dev, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16()  # noqa: E731
    qkv = size * rnd(B * T, (Hq + 2 * Hkv) * D)
    return [t.to(dev) for t in (qkv, rnd(Hkv, P, D), rnd(Hkv, P, D), rnd(B, Hkv, Smax, D), rnd(B, Hkv, Smax, D))]


def oracle(q, kp, vp, kc, vc, lens, max_len, T, scale):
    B, Hkv, _, D = kc.shape
    Hq = q.shape[1] // D
    dev = q.device if q.numel() * (kp.shape[1] + max_len) > 1 << 20 else "cpu"
    q, kp, vp, kc, vc = (t.to(dev).double() for t in (q, kp, vp, kc, vc))
    out = torch.zeros(B * T, Hq, D, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = min(max(int(lens[b]), 0), max_len)
        for t in range(T):
            own = max(n - (T - 1 - t), 0)
            k = torch.cat([kp, kc[b, :, :own]], 1).repeat_interleave(Hq // Hkv, 0)
            v = torch.cat([vp, vc[b, :, :own]], 1).repeat_interleave(Hq // Hkv, 0)
            if not k.shape[1]:
                continue
            row = q[b * T + t].view(Hq, D, 1)
            s = (k @ row).squeeze(-1) * scale
            p = torch.softmax(s, -1).unsqueeze(1)
            o, A = (p @ v).squeeze(1), (p @ v.abs()).squeeze(1)
            e = ((D + 4) * (k.abs() @ row.abs()).squeeze(-1).amax(-1) * scale + 4 * s.abs().amax(-1)) * U + 2.0 ** -22 + k.shape[1] * U
            out[b * T + t] = o
            tol[b * T + t] = (2.0 ** -8 + 2 * e.unsqueeze(-1)) * (A + o.abs()) * (1 + 2.0 ** -7) + 2.0 ** -8 * o.abs()
    return out.view(B * T, Hq * D).cpu(), tol.view(B * T, Hq * D).cpu()


def check(q, kp, vp, kc, vc, lens, max_len, T, scale=None):
    D = kc.shape[-1]
    want, tol = oracle(q, kp, vp, kc, vc, lens, max_len, T, scale or 1 / math.sqrt(D))
    got = kf.prefix_attention(q, kp, vp, kc, vc, lens, max_len, T, scale)
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    err = (got.double().cpu() - want).abs() - tol
    assert err.max() <= 0, (err.max(), torch.nonzero(err > 0)[:5])
    return got


def run(B, T, Hq, Hkv, D, P, lens, dev, seed=0, stale=float("nan"), size=1.0):
    Smax = max(max(lens), 1) + 5
    qkv, kp, vp, kc, vc = make(B, T, Hq, Hkv, D, P, Smax, dev, seed, size)
    for b, n in enumerate(lens):
        kc[b, :, max(n, 0):] = stale
        vc[b, :, max(n, 0):] = stale
    return check(qkv[:, : Hq * D], kp, vp, kc, vc, torch.tensor(lens, dtype=torch.int32, device=dev), max(max(lens), 0), T)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (12, 12, 64), (8, 2, 128), (6, 2, 128), (5, 1, 64), (16, 1, 128)])
@pytest.mark.parametrize("P", [0, 1, 33, 200])
@pytest.mark.parametrize("T", [1, 3])
def test_heads_prefixes_and_tokens(dev, Hq, Hkv, D, P, T):
    run(4, T, Hq, Hkv, D, P, [T, 31 + T, 128, 130], dev, seed=P + T)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("T", [1, 2, 5, 8, 40])
@pytest.mark.parametrize("n", [40, 63, 64, 65, 127, 128, 129, 161])
def test_lengths_around_blocks(dev, T, n):
    run(2, T, 8, 2, 64, n, [n, n + 1], dev, seed=n)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("P", [0, 70])
def test_empty_short_and_overlong_sequences(dev, P):
    """Lengths of 0, below the token count (the first tokens see the prefix alone, or nothing: 0) and past max_len."""
    T, Hq, Hkv, D = 4, 8, 4, 64
    qkv, kp, vp, kc, vc = make(6, T, Hq, Hkv, D, P, 90, dev)
    lens = torch.tensor([0, 1, 3, 4, 500, -3], dtype=torch.int32, device=dev)
    got = check(qkv[:, : Hq * D], kp, vp, kc, vc, lens, 77, T)
    if P == 0:
        assert not got[:T].any() and not got[T:2 * T - 1].any() and got[2 * T - 1].any() and not got[-T:].any()
    none = kf.prefix_attention(qkv[:, : Hq * D], kp, vp, kc, vc, lens * 0, 0, T)  # no own keys at all
    if P == 0:
        assert not none.any()
    else:
        check(qkv[:, : Hq * D], kp, vp, kc, vc, lens * 0, 0, T)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_keys_that_are_not_finite(dev, bad):
    """Keys of later tokens hold NaN / inf: earlier tokens' rows are those of a finite cache, bit for bit."""
    T, Hq, Hkv, D, P = 4, 8, 2, 128, 50
    for n in (4, 33, 64, 100):
        qkv, kp, vp, kc, vc = make(2, T, Hq, Hkv, D, P, 128, dev, seed=n)
        q, lens = qkv[:, : Hq * D], torch.full((2,), n, dtype=torch.int32, device=dev)
        want = kf.prefix_attention(q, kp, vp, kc, vc, lens, n, T).view(2, T, -1)
        for what in ("k", "v", "both"):
            k2, v2 = kc.clone(), vc.clone()
            if what != "v":
                k2[:, :, n - 2] = bad
            if what != "k":
                v2[:, :, n - 2] = bad
            got = kf.prefix_attention(q, kp, vp, k2, v2, lens, n, T).view(2, T, -1)
            assert torch.equal(got[:, :2], want[:, :2]), (n, what)  # tokens 0 and 1 do not see key n - 2
            if what == "v":
                assert not torch.isfinite(got[:, 2:].float()).any()


@pytest.mark.parametrize("dev", DEVS)
def test_strided_prefix_and_slots(dev):
    """The prefix as a slot of another cache ([Hkv, Smax, D] cut to P rows), and as rows of a fused [P, Hkv, D] tensor."""
    Hq, Hkv, D, P = 8, 4, 64, 100
    qkv, kp, vp, kc, vc = make(3, 1, Hq, Hkv, D, P, 64, dev)
    lens = torch.tensor([5, 64, 33], dtype=torch.int32, device=dev)
    q = qkv[:, : Hq * D]
    want = check(q, kp, vp, kc, vc, lens, 64, 1)
    slot = torch.full((2, 2, Hkv, P + 28, D), float("nan"), dtype=torch.bfloat16, device=dev)
    slot[0, 1, :, :P], slot[1, 1, :, :P] = kp, vp
    assert torch.equal(kf.prefix_attention(q, slot[0, 1, :, :P], slot[1, 1, :, :P], kc, vc, lens, 64), want)
    rows = torch.stack([kp.transpose(0, 1), vp.transpose(0, 1)], 1).contiguous()  # [P, 2, Hkv, D]
    assert torch.equal(kf.prefix_attention(q, rows[:, 0].transpose(0, 1), rows[:, 1].transpose(0, 1), kc, vc, lens, 64), want)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hkv,D,P,own", [(64, 1, 32, 8, 128, 2048, 500), (24, 5, 32, 8, 128, 3000, 300), (1, 1, 32, 8, 128, 8192, 2000),
                                                (128, 1, 12, 12, 64, 777, 64), (3, 128, 8, 2, 64, 513, 128), (2, 300, 32, 8, 128, 130, 333),
                                                (96, 8, 4, 2, 64, 5000, 40), (2, 1, 64, 8, 128, 1, 3000), (40, 2, 16, 2, 64, 1500, 200),
                                                (33, 7, 6, 2, 128, 999, 77)])
def test_serving_sizes(B, T, Hq, Hkv, D, P, own):
    lens = [T + (b * (own - T)) // max(B - 1, 1) for b in range(B)]
    run(B, T, Hq, Hkv, D, P, lens, "cuda", seed=B)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hkv,D,P", [(64, 24, 8, 2, 64, 130), (64, 25, 8, 2, 128, 64), (130, 96, 2, 2, 64, 0), (1, 1500, 32, 8, 128, 65),
                                            (65, 40, 8, 4, 128, 1), (40, 33, 16, 4, 64, 0), (64, 12, 24, 4, 128, 2000), (22, 50, 20, 4, 64, 300), (3, 700, 6, 6, 128, 0)])
@pytest.mark.parametrize("more", [0, 97])
def test_prompts(B, T, Hq, Hkv, D, P, more):
    """Many rows per sequence: own lengths from the tokens alone up to ``more`` keys before them, stale keys of NaN behind."""
    run(B, T, Hq, Hkv, D, P, [T + (more * b) // max(B - 1, 1) for b in range(B)], "cuda", seed=B)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P", [0, 70])
def test_prompts_empty_short_and_overlong(D, P):
    """As above with lengths of 0, below the token count, past max_len and negative."""
    B, T, Hq, Hkv = 64, 33, 12, 4
    qkv, kp, vp, kc, vc = make(B, T, Hq, Hkv, D, P, 150, "cuda")
    lens = torch.tensor([(0, 1, 32, 33, 34, 500, -3, 96)[b % 8] for b in range(B)], dtype=torch.int32, device="cuda")
    got = check(qkv[:, : Hq * D], kp, vp, kc, vc, lens, 140, T).view(B, T, -1)
    if P == 0:
        assert not got[0].any() and not got[1, :-1].any() and got[1, -1].any() and not got[6].any()
    none = kf.prefix_attention(qkv[:, : Hq * D], kp, vp, kc, vc, lens, 0, T)
    if P == 0:
        assert not none.any()
    else:
        check(qkv[:, : Hq * D], kp, vp, kc, vc, lens, 0, T)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_prompts_with_masked_keys_that_are_not_finite(D, bad):
    """The key of token j holds NaN / inf: the rows of the tokens before it are those of a finite cache, bit for bit."""
    B, T, Hq, Hkv, P, own = 32, 70, 8, 4, 50, 90
    qkv, kp, vp, kc, vc = make(B, T, Hq, Hkv, D, P, own, "cuda", seed=1)
    q, lens = qkv[:, : Hq * D], torch.full((B,), own, dtype=torch.int32, device="cuda")
    want = kf.prefix_attention(q, kp, vp, kc, vc, lens, own, T).view(B, T, -1)
    for j in (1, 31, 32, 44, 69):
        for what in ("k", "v", "both"):
            k2, v2 = kc.clone(), vc.clone()
            if what != "v":
                k2[:, :, own - T + j] = bad
            if what != "k":
                v2[:, :, own - T + j] = bad
            got = kf.prefix_attention(q, kp, vp, k2, v2, lens, own, T).view(B, T, -1)
            assert torch.equal(got[:, :j], want[:, :j]), (j, what)
            if what == "v":
                assert not torch.isfinite(got[:, j:].float()).any()


@pytest.mark.gpu
def test_large_scores():
    """Scores of several hundred: one key holds nearly everything, maxima that move from block to block."""
    run(8, 2, 8, 2, 128, 700, [2, 40, 90, 128, 129, 200, 300, 256], "cuda", size=32.0)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
@pytest.mark.parametrize("B,T", [(3, 2), (20, 9)])
def test_other_scales(dev, scale, B, T):
    """Any sign: maxima are taken before scaling; scale 0 weighs every key that is seen alike."""
    qkv, kp, vp, kc, vc = make(B, T, 4, 2, 64, 70, 90, dev)
    lens = torch.randint(0, 91, (B,), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(dev)
    q = 0.3 * qkv[:, : 4 * 64]
    want, tol = oracle(q, kp, vp, kc, vc, lens, 90, T, scale)
    got = kf.prefix_attention(q, kp, vp, kc, vc, lens, 90, T, scale)
    assert ((got.double().cpu() - want).abs() - tol).max() <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
def test_prompts_with_other_scales(scale):
    test_other_scales("cuda", scale, 130, 30)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A cache and a prefix of more than 2^31 elements each; the queries match keys near the end."""
    Hkv, D, n = 8, 128, (1 << 21) + 4097
    g = torch.Generator(device="cuda").manual_seed(0)
    caches = [torch.zeros(1, Hkv, n, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    at = n - 77
    for t in caches:
        t[:, :, at:] = torch.randn(1, Hkv, n - at, D, device="cuda", generator=g).bfloat16()
    q = 4 * caches[0][0, :, at + 5].reshape(1, Hkv * D)
    for kp, vp, kc, vc, lens in ((caches[0][0], caches[1][0], caches[0][:, :, :64].contiguous(), caches[1][:, :, :64].contiguous(), 0),
                                 (caches[0][0, :, :0], caches[1][0, :, :0], caches[0], caches[1], n)):
        got = kf.prefix_attention(q, kp, vp, kc, vc, torch.tensor([lens], dtype=torch.int32, device="cuda"), kc.shape[2])
        # zero keys have score 0 and value 0: they only add to the normaliser
        s = (caches[0][0, :, at:].double() @ q.view(Hkv, D, 1).double()).squeeze(-1) / math.sqrt(D)
        e = torch.exp(s - s.amax(-1, keepdim=True))
        want = (e.unsqueeze(1) @ caches[1][0, :, at:].double()).squeeze(1) / (
            e.sum(-1) + (at) * torch.exp(-s.amax(-1))).unsqueeze(-1)
        assert (got.double().view(Hkv, D) - want).abs().max() <= 3 * 2.0 ** -8 * float(caches[1].abs().max())


@pytest.mark.gpu
def test_agrees_with_decode_attention():
    """Without a prefix and for one token it is the framework's decode attention; with the prefix copied in front of every
    sequence's own keys, decode attention over the whole cache gives the same."""
    B, Hq, Hkv, D, P = 5, 32, 8, 128, 300
    qkv, kp, vp, kc, vc = make(B, 1, Hq, Hkv, D, P, 200, "cuda")
    lens = torch.tensor([1, 50, 128, 199, 200], dtype=torch.int32, device="cuda")
    q = qkv[:, : Hq * D]
    full_k, full_v = (torch.cat([p.expand(B, Hkv, P, D), c], 2).contiguous() for p, c in ((kp, kc), (vp, vc)))
    for a, b in ((kf.prefix_attention(q, kp[:, :0], vp[:, :0], kc, vc, lens, 200), kf.decode_attention(q, kc, vc, lens, 200)),
                 (kf.prefix_attention(q, kp, vp, kc, vc, lens, 200), kf.decode_attention(q, full_k, full_v, lens + P, 200 + P))):
        # both round P (2^-8 A, A <= max |v|) and the output
        assert (a.float() - b.float()).abs().max() <= 4 * 2.0 ** -8 * float(max(vp.abs().max(), vc.abs().max()))


@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    Hq, Hkv, D, P, B = 4, 2, 64, 20, 3
    qkv, kp, vp, kc, vc = make(B, 1, Hq, Hkv, D, P, 32, dev)
    q, lens = qkv[:, : Hq * D], torch.tensor([1, 2, 3], dtype=torch.int32, device=dev)
    f = kf.prefix_attention
    bad = [
        lambda: f(q, kp, vp[:, :19], kc, vc, lens, 32),
        lambda: f(q, kp[:1], vp[:1], kc, vc, lens, 32),
        lambda: f(q, kp, vp, kc, vc[:, :, :31], lens, 32),
        lambda: f(q, kp, vp, kc, vc, lens, 33),
        lambda: f(q, kp, vp, kc, vc, lens, -1),
        lambda: f(q, kp, vp, kc, vc, lens.long(), 32),
        lambda: f(q, kp, vp, kc, vc, lens[:2], 32),
        lambda: f(q, kp, vp, kc, vc, lens, 32, 2),
        lambda: f(q, kp, vp, kc, vc, lens, 32, 0),
        lambda: f(q[:, :192], kp, vp, kc, vc, lens, 32),
        lambda: f(q[:2], kp, vp, kc, vc, lens, 32),
        lambda: f(q.reshape(B, Hq, D), kp, vp, kc, vc, lens, 32),
        lambda: f(q[:, :64 * 2], kp[..., :32], vp[..., :32], kc[..., :32].contiguous(), vc[..., :32].contiguous(), lens, 32),
        lambda: f(q.clone().requires_grad_(), kp, vp, kc, vc, lens, 32),
    ]
    if dev == "cuda":
        bad += [lambda: f(q.float(), kp, vp, kc, vc, lens, 32), lambda: f(q, kp.cpu(), vp, kc, vc, lens, 32),
                lambda: f(q, kp, vp, kc, vc, lens.cpu(), 32), lambda: f(q, kp, vp, kc[:, :, ::2], vc[:, :, ::2], lens, 16),
                lambda: f(q, kp.transpose(1, 2).contiguous().transpose(1, 2), vp, kc, vc, lens, 32)]
    for g in bad:
        with pytest.raises(RuntimeError):
            g()
    assert f(q[:0], kp, vp, kc[:0], vc[:0], lens[:0], 32).shape == (0, Hq * D)


@pytest.mark.parametrize("dev", DEVS)
def test_a_cache_without_heads_is_refused(dev):
    q = torch.zeros(2, 64, dtype=torch.bfloat16, device=dev)
    kv, cache = torch.zeros(0, 5, 64, dtype=torch.bfloat16, device=dev), torch.zeros(2, 0, 8, 64, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="no heads"):
        kf.prefix_attention(q, kv, kv, cache, cache, torch.zeros(2, dtype=torch.int32, device=dev), 8)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,P", [(4, 1, 500), (48, 4, 700), (130, 20, 30)])
def test_captured_call_replays_and_another_stream(B, T, P):
    Hq, Hkv, D = 8, 2, 128
    qkv, kp, vp, kc, vc = make(B, T, Hq, Hkv, D, P, 200, "cuda")
    lens = torch.randint(T, 201, (B,), dtype=torch.int32, device="cuda")
    args = (qkv[:, : Hq * D], kp, vp, kc, vc, lens, 200, T)
    want = kf.prefix_attention(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = kf.prefix_attention(*args)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kf.prefix_attention(*args)
    for seed in range(3):
        for a, b in zip((qkv, kp, vp, kc, vc), make(B, T, Hq, Hkv, D, P, 200, "cuda", seed=seed)):
            a.copy_(b)
        lens.copy_(torch.randint(0, 201, (B,), dtype=torch.int32, device="cuda"))
        eager = kf.prefix_attention(*args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


FORMS = [pytest.param("cuda", *f, marks=pytest.mark.gpu) for f in (
    (4, 1, 4, 2, 64, 500, 60), (4, 8, 4, 2, 128, 128, 40),          # one launch, 16 and 32 rows by keys
    (64, 1, 32, 8, 128, 2048, 300), (4, 5, 8, 2, 64, 3000, 900),    # ranges: prefix by rows, own keys of 16 and 32 rows by keys
    (4, 1, 16, 4, 128, 3000, 900), (1, 2, 16, 1, 64, 3000, 900),    # ranges: both by keys
    (64, 24, 8, 2, 64, 130, 90), (22, 50, 20, 4, 128, 64, 70))]     # prompts by rows
FORMS += [("cpu", 4, 1, 4, 2, 64, 500, 60), ("cpu", 2, 8, 4, 2, 128, 128, 40)]


@pytest.mark.parametrize("dev,B,T,Hq,Hkv,D,P,own", FORMS)
def test_weights_lose_nothing_to_the_operands_type(dev, B, T, Hq, Hkv, D, P, own):
    """A softmax over six keys (the others' scores are too low to count): what the result may be off by, besides the output's one
    rounding, is the scores' and sums' fp32 and 2^-15 of each weight, not the 2^-8 of a weight in bf16.

    Tolerance, with A = sum_j p_j |v_j| over the six: a weight cut to a bf16 value leaves a remainder below 2^-7 of it, which is
    rounded to bf16 (2^-8) after 2^-20 of the weight went into it: 2^-15 A + 2^-20 A, and as much of |o| for good measure. A score is off by ((D + 4) sum |q||k| scale + 4 |s|) 2^-24 and the
    exponential by 2^-22, e relative together; sums of six terms, in up to 32 parts, add 40 2^-24: (e + 40 2^-24) (A + |o|).
    The other keys' scores are 45 below or lower: 4000 e^-45 < 2^-50. The output's rounding: 2^-8 of what is rounded."""
    qkv, kp, vp, kc, vc = make(B, T, Hq, Hkv, D, P, own + 3, dev, seed=P)
    q = qkv[:, : Hq * D].view(B * T, Hq, D)
    q[:, :, 0] = 8.0
    near = [(kp, [1, 20, P - 1]), (kc, [0, 1, own - T])]  # what every token sees; two at least of a key range each
    for k, at in near:
        rows = k[..., at, :].clone()
        rows[..., 0] = 0.0
        k.zero_()
        k[..., 0] = -8.0 * math.sqrt(D)  # a score of -64
        k[..., at, :] = rows
    lens = torch.full((B,), own, dtype=torch.int32, device=dev)
    got = kf.prefix_attention(qkv[:, : Hq * D], kp, vp, kc, vc, lens, own, T).double().view(B, T, Hq, D)
    pick = lambda p, c: torch.cat([p[:, near[0][1]].expand(B, Hkv, 3, D), c[:, :, near[1][1]]], 2).double().repeat_interleave(Hq // Hkv, 1)  # noqa: E731
    k, v, q = pick(kp, kc), pick(vp, vc), q.double().view(B, T, Hq, D).transpose(1, 2)  # [B, Hq, 6 or T, D]
    s = (k.unsqueeze(2) * q.unsqueeze(3)).sum(-1) / math.sqrt(D)  # [B, Hq, T, 6]
    mag = (k.abs().unsqueeze(2) * q.abs().unsqueeze(3)).sum(-1) / math.sqrt(D)
    p = torch.softmax(s, -1).unsqueeze(-1)
    o, A = (p * v.unsqueeze(2)).sum(3), (p * v.abs().unsqueeze(2)).sum(3)
    e = ((D + 4) * mag.amax(-1) + 4 * s.abs().amax(-1)) * U + 2.0 ** -22 + 40 * U
    tol = (2.0 ** -15 + 2.0 ** -20 + e.unsqueeze(-1)) * (A + o.abs())
    tol = tol + 2.0 ** -8 * (o.abs() + tol)
    err = (got.transpose(1, 2) - o).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dev,B,T,Hq,Hkv,D,P,own", FORMS)
def test_infinite_values_that_every_row_sees(dev, B, T, Hq, Hkv, D, P, own):
    """A value of inf whose weight is not 0 makes its dimension inf, not NaN, in every row that sees it: a weight's remainder is never
    0 times inf, nor of the other sign."""
    for bad in (float("inf"), -float("inf")):
        qkv, kp, vp, kc, vc = make(B, T, Hq, Hkv, D, P, own + 3, dev, seed=P)
        lens = torch.full((B,), own, dtype=torch.int32, device=dev)
        args = (kc, vc, lens, own, T)
        want = kf.prefix_attention(qkv[:, : Hq * D], kp, vp, *args).view(B * T, Hq, D)
        vp[:, 3, 5] = bad
        qkv[:, 0] = 0.0  # a score of 0 against every key of one row: weights that bf16 holds
        kp[:, :, 1:] = 0.0
        got = kf.prefix_attention(qkv[:, : Hq * D], kp, vp, *args).view(B * T, Hq, D)
        assert (got[:, :, 5] == bad).all() and torch.isfinite(got[:, :, [0, 4, 6, D - 1]]).all() and torch.isfinite(want).all()
