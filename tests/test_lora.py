"""Low-rank adapters of many requests beside one projection (``ops.lora_add``) against the formula in 64 bits: ranks, row
counts around the 16-row tiles, mixed / sorted / missing adapters, strided and in-place outputs, adapters that hold NaN,
refusals, captured calls.

Tolerance per output (u = 2^-24): the low-rank value t = a x is an fp32 sum of K bf16 products, K u sum |a||x| off at most;
it enters the second product as a bf16 pair, 2^-16 |t|; that product's fp32 sum of r terms (and the scale) adds
(r + 2) u |b||s t|; the sum with y 2 u, the rounding to bf16 2^-8 of the output."""
import pytest
import torch

from kubeoperator_amd.ops import functional as kf

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def make(M, n, r, K, N, dev, seed=0, order="mixed"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).bfloat16()
    y = torch.randn(M, N, generator=g).bfloat16()
    a = (torch.randn(n, r, K, generator=g) / K ** 0.5).bfloat16()
    b = (torch.randn(n, N, r, generator=g) / r ** 0.5).bfloat16()
    index = torch.randint(-1, n, (M,), generator=g)
    if order == "sorted":
        index = index.sort().values
    if order == "one":
        index[:] = n - 1
    scale = torch.rand(n, generator=g) + 0.5
    return [t.to(dev) for t in (y, x, a, b, index.to(torch.int32), scale)]


def oracle(y, x, a, b, index, scale):
    y, x, a, b, s = (t.double().cpu() for t in (y, x, a, b, scale))
    out, tol = y.clone(), torch.zeros_like(y)
    n, r, K = a.shape
    for i, j in enumerate(index.tolist()):
        if 0 <= j < n:
            t, tm = a[j] @ x[i], a[j].abs() @ x[i].abs()
            out[i] += s[j] * (b[j] @ t)
            tol[i] = s[j].abs() * (b[j].abs() @ (2.0 ** -16 * t.abs() + K * U * tm + (r + 2) * U * t.abs()))
            tol[i] += 2 * U * (y[i].abs() + out[i].abs()) + 2.0 ** -8 * (out[i].abs() + tol[i])
    return out, tol


def check(args, out=None):
    want, tol = oracle(*args)
    got = kf.lora_add(*args, out)
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    err = (got.double().cpu() - want).abs() - tol
    assert err.max() <= 0, (err.max(), torch.nonzero(err > 0)[:5])
    return got


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("M,n,r,K,N", [(1, 1, 8, 8, 8), (1, 3, 16, 4096, 4096), (2, 1, 128, 256, 72), (15, 4, 8, 264, 1000),
                                       (16, 16, 16, 512, 256), (17, 2, 24, 1000, 264), (33, 40, 64, 2048, 520),
                                       (64, 32, 16, 1024, 2048), (100, 5, 104, 136, 8), (257, 3, 40, 520, 328),
                                       (300, 64, 32, 256, 128)])
@pytest.mark.parametrize("order", ["mixed", "sorted", "one"])
def test_matches_the_formula(dev, M, n, r, K, N, order):
    check(make(M, n, r, K, N, dev, seed=M, order=order))


@pytest.mark.gpu
@pytest.mark.parametrize("M,order", [(1100, "mixed"), (2000, "sorted"), (4100, "sorted")])
@pytest.mark.parametrize("r", [16, 64])
def test_many_rows(M, order, r):
    check(make(M, 12, r, 768, 512, "cuda", order=order))


@pytest.mark.parametrize("dev", DEVS)
def test_rows_without_an_adapter_keep_y(dev):
    y, x, a, b, index, scale = make(40, 6, 16, 256, 128, dev)
    index[::3] = torch.tensor(-5, dtype=torch.int32)
    index[1::3] = torch.tensor(6, dtype=torch.int32)  # past the last adapter
    index[2] = 2 ** 31 - 1
    got = check([y, x, a, b, index, scale])
    off = (index < 0) | (index >= 6)
    assert torch.equal(got[off], y[off])
    none = kf.lora_add(y, x, a[:0], b[:0], index, scale[:0])
    assert torch.equal(none, y)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("M", [20, 700])
def test_one_requests_bad_numbers_stay_with_its_rows(dev, M):
    y, x, a, b, index, scale = make(M, 5, 16, 512, 256, dev)
    clean = kf.lora_add(y, x, a, b, index, scale)
    a2, b2, x2 = a.clone(), b.clone(), x.clone()
    a2[1] = float("nan")
    b2[2] = float("inf")
    x2[7] = float("nan")
    got = kf.lora_add(y, x2, a2, b2, index, scale)
    mine = (index != 1) & (index != 2)
    mine[7] = False
    assert mine.any() and torch.equal(got[mine], clean[mine])
    assert not torch.isfinite(got[(index == 1) | (index == 2)].float()).any()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("M", [21, 600])
def test_strided_and_in_place(dev, M):
    y, x, a, b, index, scale = make(M, 4, 24, 264, 136, dev)
    want = check([y, x, a, b, index, scale])
    wide = torch.full((M + 3, 136 + 48), 3.0, dtype=torch.bfloat16, device=dev)
    wide[:M, 24:160] = y
    wx = torch.full((M, 264 + 8), float("nan"), dtype=torch.bfloat16, device=dev)
    wx[:, :264] = x
    view = wide[:M, 24:160]
    got = kf.lora_add(view, wx[:, :264], a, b, index, scale, out=view)  # one slice of a fused projection's output
    assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)
    assert (wide[:, :24] == 3).all() and (wide[:, 160:] == 3).all() and (wide[M:] == 3).all()
    # every row the same x row
    check([y, x[:1].expand(M, 264), a, b, index, scale])


@pytest.mark.parametrize("dev", DEVS)
def test_scale_sign_zero_and_size(dev):
    y, x, a, b, index, scale = make(30, 3, 16, 128, 64, dev)
    scale[0], scale[1], scale[2] = 0.0, -2.5, 3e4
    check([y, x, a, b, index, scale])


@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    y, x, a, b, index, scale = make(8, 3, 16, 64, 40, dev)
    bad = [
        lambda: kf.lora_add(y[:7], x, a, b, index, scale),
        lambda: kf.lora_add(y, x, a, b, index[:7], scale),
        lambda: kf.lora_add(y, x, a, b, index.long(), scale),
        lambda: kf.lora_add(y, x, a, b, index, scale[:2]),
        lambda: kf.lora_add(y, x, a, b, index, scale.double()),
        lambda: kf.lora_add(y, x, a, b[:2], index, scale),
        lambda: kf.lora_add(y, x, a[:, :8], b, index, scale),
        lambda: kf.lora_add(y, x, a[:, :4].contiguous(), b[:, :, :4].contiguous(), index, scale),
        lambda: kf.lora_add(y, x[:, :56], a, b, index, scale),
        lambda: kf.lora_add(y, x, a.repeat(1, 9, 1), b.repeat(1, 1, 9), index, scale),
        lambda: kf.lora_add(y[:, :36], x, a, b[:, :36].contiguous(), index, scale),
        lambda: kf.lora_add(y, x, a, b, index, scale, out=y[:4]),
        lambda: kf.lora_add(y, x, a.clone().requires_grad_(), b, index, scale),
    ]
    if dev == "cuda":
        wide = torch.zeros(8, 64, dtype=torch.bfloat16, device=dev)
        bad += [lambda: kf.lora_add(y, x.float(), a, b, index, scale), lambda: kf.lora_add(y, x.cpu(), a, b, index, scale),
                lambda: kf.lora_add(wide[:, :40], x, a, b, index, scale, out=wide[:, 8:48]),
                lambda: kf.lora_add(wide[:, :40], wide, a, b, index, scale, out=wide[:, :40]),
                lambda: kf.lora_add(y, wide[:, 1:].as_strided((8, 64), (64, 1)), a, b, index, scale),
                lambda: kf.lora_add(y, x, a, b, index, scale, out=y[:1].expand(8, 40))]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    assert kf.lora_add(y[:0], x[:0], a, b, index[:0], scale).shape == (0, 40)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Outputs of more than 2^31 elements, written in place: the last rows against the formula, a row in front untouched."""
    M, N = 280000, 8192
    _, x, a, b, _, scale = make(64, 3, 8, 64, N, "cuda")
    y = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    index = torch.full((M,), -1, dtype=torch.int32, device="cuda")
    index[-64:] = torch.randint(0, 3, (64,), dtype=torch.int32, device="cuda")
    xs = x[:1].expand(M, 64).clone()
    xs[-64:] = x
    kf.lora_add(y, xs, a, b, index, scale, out=y)
    want, tol = oracle(torch.zeros(64, N), x, a, b, index[-64:], scale)
    assert ((y[-64:].double().cpu() - want).abs() - tol).max() <= 0 and not y[:-64].any()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [24, 800])
def test_captured_call_replays_and_another_stream(M):
    args = make(M, 6, 16, 512, 256, "cuda")
    want = kf.lora_add(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = kf.lora_add(*args)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kf.lora_add(*args)
    for seed in range(3):
        for p, q in zip(args, make(M, 6, 16, 512, 256, "cuda", seed=seed)):
            p.copy_(q)
        eager = kf.lora_add(*args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("M", [2 ** 29, 2 ** 31 + 64])
def test_more_rows_than_a_launch_can_have_are_refused(dev, M):
    """Row numbers inside the kernels are 32 bits wide, and a launch has at most 2^32 work-items: refused before anything is allocated
    or launched (rows that are all the same one, so that only the index list takes memory)."""
    row, low = torch.zeros(1, 8, dtype=torch.bfloat16, device=dev), torch.zeros(1, 8, 8, dtype=torch.bfloat16, device=dev)
    index = torch.empty(M, dtype=torch.int32, device=dev) if dev == "cuda" else torch.zeros(1, dtype=torch.int32).expand(M)
    with pytest.raises(RuntimeError, match="too many rows"):
        kf.lora_add(row.expand(M, 8), row.expand(M, 8), low, low, index, torch.ones(1, device=dev))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("M,n", [(1, 700), (64, 700), (130, 1500)])
def test_more_adapters_than_rows(dev, M, n):
    check(make(M, n, 16, 128, 72, dev, seed=n))
