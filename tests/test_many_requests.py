"""One model, many requests: generation behind a shared prefix, with an adapter per request, through drafted tokens, and a draft
model's training -- the operators in a run together, on the CPU references and on the GPU."""
import json

import pytest
import torch

from kubeoperator_amd.models import build_model, get_config
from kubeoperator_amd.ops import functional as kf
from kubeoperator_amd.serve import LlamaGenerator, LoraAdapters

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def model(dev, seed=0, size=0.05, **kw):
    cfg = get_config("tiny_llama", **kw)
    m = build_model(cfg)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.copy_((1 + 0.1 * torch.randn(p.shape, generator=g)) if "norm" in n else size * torch.randn(p.shape, generator=g))
    return m.to(device=dev, dtype=torch.bfloat16)


def adapters(m, n, rank, seed=3, size=0.2):
    """Adapters of different ranks: adapter i uses rank - 8 (i % 2) of the stacked rank (from 16 up)."""
    ad = LoraAdapters(m.cfg, n, rank, m.tok_emb.device)
    g = torch.Generator().manual_seed(seed)
    for li in range(m.cfg.n_layers):
        for t in ad.targets:
            A, B = ad.layers[li][t]
            for i in range(n):
                r = rank - 8 * (i % 2) if rank >= 16 else rank
                ad.set(i, li, t, size * torch.randn(r, A.shape[2], generator=g) / A.shape[2] ** 0.5 * 4,
                       size * torch.randn(B.shape[1], r, generator=g))
    ad.scale.copy_(torch.rand(n, generator=g) + 0.5)
    return ad


def merged(m, ad, i):
    """A copy of the model with adapter i added into its weights (in fp32, rounded once)."""
    out = model(m.tok_emb.device, **{k: getattr(m.cfg, k) for k in ("hidden", "n_heads", "n_kv_heads", "ffn_hidden")})
    out.load_state_dict(m.state_dict())
    with torch.no_grad():
        for blk, layer in zip(out.layers, ad.layers):
            for t, (a, b) in layer.items():
                w = getattr(blk, t)
                w.copy_(w.float() + float(ad.scale[i]) * (b[i].float() @ a[i].float()))
    return out


def ids_of(m, B, S, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, m.cfg.vocab_size, (B, S), generator=g).to(m.tok_emb.device)


def close(a, b, tol=3e-2):
    """Two bf16 paths through the same network: the bound test_serve.py holds decode against a fresh prefill to."""
    err = (a - b).abs().max().item() / b.abs().max().item()
    assert err < tol, err


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("P", [1, 77, 128, 200])
def test_prefix_is_the_same_as_prompts_that_start_with_it(dev, graph, P):
    m = model(dev)
    pre, own = ids_of(m, 1, P, seed=9)[0], ids_of(m, 3, 33)
    gen = LlamaGenerator(m, max_batch=3, max_seq=64, graph=graph)
    gen.set_prefix(pre)
    whole = LlamaGenerator(m, max_batch=3, max_seq=P + 64)
    lengths = [33, 5, 20]
    full = torch.zeros(3, P + 33, dtype=torch.long, device=dev)
    full[:, :P], full[:, P:] = pre, own
    a, b = gen.prefill(own, lengths=lengths), whole.prefill(full, lengths=[P + n for n in lengths])
    close(a, b)
    for step in range(4):
        tok = ids_of(m, 3, 1, seed=20 + step)[:, 0]
        close(gen.decode(tok), whole.decode(tok))
    assert gen.cache.host_lens == [n + 4 for n in lengths] and gen.cache.lens.tolist() == gen.cache.host_lens
    # another prefix, then none: nothing of the old one is left
    gen.set_prefix(pre.flip(0))
    full[:, :P] = pre.flip(0)
    close(gen.prefill(own), whole.prefill(full))
    gen.set_prefix(None)
    close(gen.prefill(own), LlamaGenerator(m, 3, 64).prefill(own))
    tok = own[:, 0]
    close(gen.decode(tok), LlamaGenerator(m, 3, 64).prefill(torch.cat([own, tok.unsqueeze(1)], 1)))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("prefix", [0, 50])
def test_extend_is_the_same_as_steps(dev, prefix):
    m = model(dev)
    gens = [LlamaGenerator(m, max_batch=3, max_seq=80) for _ in range(2)]
    prompt, more = ids_of(m, 3, 17), ids_of(m, 3, 5, seed=2)
    for g in gens:
        if prefix:
            g.set_prefix(ids_of(m, 1, prefix, seed=9)[0])
        g.prefill(prompt, lengths=[17, 3, 9])
    many = gens[0].extend(more)
    steps = torch.stack([gens[1].decode(more[:, t]) for t in range(5)], 1)
    close(many, steps)
    assert gens[0].cache.host_lens == gens[1].cache.host_lens == [22, 8, 14]
    for g in gens:  # two tokens taken back, then on
        g.cache.truncate([20, 6, 12])
    close(gens[0].extend(more[:, 3:]), torch.stack([gens[1].decode(more[:, t]) for t in (3, 4)], 1))
    with pytest.raises(ValueError):
        gens[0].cache.truncate([100])
    with pytest.raises(ValueError):
        gens[0].extend(ids_of(m, 3, 70))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("graph", [False, True])
def test_each_request_gets_its_adapter(dev, graph):
    m = model(dev)
    ad = adapters(m, 3, 16)
    gen = LlamaGenerator(m, max_batch=5, max_seq=48, graph=graph)
    base = LlamaGenerator(m, max_batch=5, max_seq=48)
    prompt = ids_of(m, 5, 21)
    plain = base.prefill(prompt)
    gen.set_adapters(ad)
    which = [2, -1, 0, 1, 2]
    got = gen.prefill(prompt, adapters=which)
    tok = ids_of(m, 5, 3, seed=4)
    steps = [gen.decode(tok[:, 0]), gen.decode(tok[:, 1])]
    last = gen.extend(tok[:, 2:])[:, 0]
    for i in range(-1, 3):
        rows = [b for b in range(5) if which[b] == i]
        own = LlamaGenerator(m if i < 0 else merged(m, ad, i), max_batch=len(rows), max_seq=48)
        close(got[rows], own.prefill(prompt[rows]))
        for t in range(2):
            close(steps[t][rows], own.decode(tok[rows, t]))
        close(last[rows], own.decode(tok[rows, 2]))
    assert (got[0] - plain[0]).abs().max() > 0.1 * plain.abs().max()  # the adapters do something
    close(gen.prefill(prompt), plain)  # no adapter named: none
    with pytest.raises(ValueError):
        gen.prefill(prompt, adapters=[0, 1, 2, 3, 0])
    with pytest.raises(ValueError):
        base.prefill(prompt, adapters=[0] * 5)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("drafts", [1, 4])
def test_speculative_greedy_is_the_targets_own(dev, drafts):
    """The tokens are the target's greedy ones. On the CPU both paths are the same arithmetic; on the GPU steps of one and of
    several tokens differ in rounding, and a token may differ where the target's two best logits are that close."""
    m = model(dev, size=0.08)
    near = model(dev, size=0.08)
    with torch.no_grad():
        for p in near.parameters():
            p.add_(0.004 * torch.randn(p.shape, generator=torch.Generator().manual_seed(5)).to(p))
    ids, n = ids_of(m, 3, 12), 15
    gens = [LlamaGenerator(x, max_batch=3, max_seq=12 + n + drafts) for x in (m, near)]
    got, rounds = gens[0].speculate(gens[1], ids, n, drafts=drafts)
    assert got.shape == (3, 12 + n) and torch.equal(got[:, :12], ids)
    assert all(0 <= k <= drafts for r in rounds for k in r) and any(k > 0 for r in rounds for k in r)
    fresh = LlamaGenerator(m, max_batch=3, max_seq=12 + n + 1)
    logits = fresh.prefill(ids)
    for t in range(n):  # every token is the best one after the tokens before it, up to the two paths' rounding
        top = logits.max(-1).values - logits.gather(1, got[:, 12 + t].unsqueeze(1)).squeeze(1)
        assert (top <= (0.0 if dev == "cpu" else 3e-2) * logits.abs().max()).all(), (t, top)
        logits = fresh.decode(got[:, 12 + t])


@pytest.mark.parametrize("dev", DEVS)
def test_speculative_sampling_with_itself_keeps_nearly_everything(dev):
    """A draft that is the target itself: acceptance fails only where the two paths' roundings differ."""
    m = model(dev)
    ids = ids_of(m, 4, 9)
    a, b = (LlamaGenerator(m, max_batch=4, max_seq=64) for _ in range(2))
    pre = ids_of(m, 1, 40, seed=9)[0]
    a.set_prefix(pre)
    with pytest.raises(ValueError):
        a.speculate(b, ids, 8)
    b.set_prefix(pre)
    g = torch.Generator(device=dev).manual_seed(0)
    out, rounds = a.speculate(b, ids, 20, drafts=3, temperature=0.9, generator=g)
    kept = [k for r in rounds for k in r]
    assert out.shape == (4, 29) and sum(kept) >= 0.9 * 3 * len(kept)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_speculation_with_broken_logits(dev, temperature):
    """A draft whose logits are all NaN proposes nothing that is kept (and no token outside the vocabulary reaches a model); a
    target like that is an error, as is a draft that shares the target's cache."""
    m, bad = model(dev), model(dev)
    with torch.no_grad():
        bad.final_norm.fill_(float("nan"))
    ids = ids_of(m, 2, 10)
    gen, broken = (LlamaGenerator(x, max_batch=2, max_seq=32) for x in (m, bad))
    out, rounds = gen.speculate(broken, ids, 6, drafts=3, temperature=temperature)
    assert out.shape == (2, 16) and rounds == [[0, 0]] * 5
    assert ((out >= 0) & (out < m.cfg.vocab_size)).all()
    with pytest.raises(RuntimeError, match="probability"):
        broken.speculate(gen, ids, 6, drafts=3, temperature=temperature)
    with pytest.raises(ValueError, match="of its own"):
        gen.speculate(gen, ids, 6)


@pytest.mark.parametrize("dev", DEVS)
def test_draft_training_gradients(dev):
    """Llama.distill against the logits' formula: the gradient of every parameter against differences of the loss along a
    direction (fp32 master copy, so the differences are those of the same network)."""
    m = model("cpu").float() if dev == "cpu" else model(dev)
    B, S, K = 2, 128, 8
    ids = ids_of(m, B, S)
    g = torch.Generator().manual_seed(8)
    index = torch.randint(0, m.cfg.vocab_size, (B, S, K), generator=g).to(torch.int32).to(dev)
    teacher = torch.randn(B, S, K, generator=g).to(dev)
    weight = (torch.rand(B, S, generator=g) / (B * S)).to(dev)
    weight[0, ::3] = 0
    loss = m.distill(ids, index, teacher, 1.5, weight)
    loss.backward()
    if dev == "cuda":  # the same network on the CPU, fp32 weights: bf16 activations differ by a few percent of the norm
        ref = model("cpu").float()
        want = ref.distill(ids.cpu(), index.cpu(), teacher.cpu(), 1.5, weight.cpu())
        want.backward()
        assert abs(float(loss.detach()) - float(want.detach())) < 2e-2 * abs(float(want.detach()))
        for (n, p), q in zip(m.named_parameters(), ref.parameters()):
            assert (p.grad.float().cpu() - q.grad).norm() <= 0.06 * q.grad.norm(), n
        return
    for name, p in m.named_parameters():
        if name not in ("lm_head", "layers.1.w_down", "layers.0.wqkv", "tok_emb", "final_norm"):
            continue
        d = p.grad / p.grad.norm()
        h = 2e-3
        vals = []
        with torch.no_grad():
            for sgn in (1, -1):
                p.add_(sgn * h * d)
                vals.append(float(m.distill(ids, index, teacher, 1.5, weight).double()))
                p.add_(-sgn * h * d)
        num, ana = (vals[0] - vals[1]) / (2 * h), float(p.grad.norm())
        # logits reach the loss in fp32: 1e-6 of it over the step, and h^2 of the third derivative
        assert abs(num - ana) <= 0.02 * ana + 1e-3, (name, num, ana)


def test_server_prefix_and_adapters(tmp_path):
    from fastapi.testclient import TestClient

    from kubeoperator_amd.serve.server import build_parser, create_app

    m = model("cpu")
    ad = adapters(m, 2, 8)
    torch.save(ad.state_dict(), tmp_path / "ad.pt")
    again = LoraAdapters.load(m.cfg, str(tmp_path / "ad.pt"), "cpu")
    assert again.n == 2 and again.rank == 8 and torch.equal(again.layers[1]["wo"][1], ad.layers[1]["wo"][1])
    with pytest.raises(ValueError):
        LoraAdapters.load(get_config("tiny_llama", ffn_hidden=256), str(tmp_path / "ad.pt"), "cpu")
    prefix = ids_of(m, 1, 30, seed=9)[0].tolist()
    (tmp_path / "p.json").write_text(json.dumps(prefix))
    assert build_parser().parse_args(["--prefix", str(tmp_path / "p.json")]).prefix
    c = TestClient(create_app(m, max_batch=2, max_seq=48, prefix=prefix, adapters=again))
    info = c.get("/v1/model").json()
    assert info["prefix_tokens"] == 30 and info["adapters"] == 2
    prompts = [[1, 2, 3, 4], [9, 8, 7]]
    for which, net in ((-1, m), (1, merged(m, ad, 1))):
        r = c.post("/v1/generate", json={"tokens": prompts, "max_new_tokens": 4, "adapter": which})
        assert r.status_code == 200, r.text
        for p, got in zip(prompts, r.json()["tokens"]):
            gen = LlamaGenerator(m, 1, 48)
            gen.set_prefix(torch.tensor(prefix))
            gen.set_adapters(ad)
            logits = gen.prefill(torch.tensor([p]), adapters=[which])
            for t in got:
                assert int(logits.argmax(-1)) == t
                logits = gen.decode(torch.tensor([t]))
    assert c.post("/v1/generate", json={"tokens": prompts, "adapter": 2}).status_code == 400
    assert c.post("/v1/generate", json={"tokens": prompts, "adapter": -2}).status_code == 400
    with pytest.raises(ValueError):
        create_app(m, 2, 48, prefix=[m.cfg.vocab_size])


def test_adapter_refusals():
    m = model("cpu")
    for kw in (dict(n=0, rank=8), dict(n=1, rank=4), dict(n=1, rank=12), dict(n=1, rank=136), dict(n=1, rank=8, targets=("lm_head",))):
        with pytest.raises(ValueError):
            LoraAdapters(m.cfg, device="cpu", **kw)
    ad = LoraAdapters(m.cfg, 2, 16, "cpu")
    a, b = ad.layers[0]["wo"]
    for i, x, y in ((2, a[0], b[0]), (0, a[0, :8], b[0]), (0, a[0, :, :64], b[0]), (-1, a[0], b[0])):
        with pytest.raises(ValueError):
            ad.set(i, 0, "wo", x, y)


def is_greedy(dev, gen, ids, got, n, adapters=None):
    """Every one of the n tokens behind ``ids`` is the best one after those before it, up to the rounding of two paths on the GPU."""
    S = ids.shape[1]
    logits = gen.prefill(ids, adapters=adapters)
    for t in range(n):
        top = logits.max(-1).values - logits.gather(1, got[:, S + t].unsqueeze(1)).squeeze(1)
        assert (top <= (0.0 if dev == "cpu" else 3e-2) * logits.abs().max()).all(), (t, top)
        logits = gen.decode(got[:, S + t])


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("graph", [False, True])
def test_speculation_and_generation_with_an_adapter_per_request(dev, graph):
    """Requests bring adapters and speculate together: the tokens are those of step-by-step decoding with the same adapters, a
    captured draft (and target) included, and not the base model's."""
    m = model(dev, size=0.08)
    ad, which = adapters(m, 3, 16), [2, -1, 0]
    ids, n = ids_of(m, 3, 11), 10
    new = lambda g: LlamaGenerator(m, max_batch=3, max_seq=40, graph=g)  # noqa: E731
    gen, draft, steps = new(graph), new(graph), new(False)
    for g in (gen, steps):
        g.set_adapters(ad)
    for _ in range(2):  # the second time on captured graphs
        got, _ = gen.speculate(draft, ids, n, drafts=3, adapters=which)
        assert gen.slot_adapter.tolist() == which
        is_greedy(dev, steps, ids, got, n, which)
    got = gen.generate(ids, n, adapters=which)
    is_greedy(dev, steps, ids, got, n, which)
    base, _ = gen.speculate(draft, ids, n, drafts=3)  # none named: none
    is_greedy(dev, new(False), ids, base, n)
    assert not torch.equal(base[0], got[0])
    with pytest.raises(ValueError):
        gen.speculate(draft, ids, n, adapters=[0, 1])
    with pytest.raises(ValueError):
        gen.generate(ids, n, adapters=[0, 1, 3])
    with pytest.raises(ValueError):
        draft.generate(ids, n, adapters=which)


def test_a_finished_sequence_cannot_stop_the_others(monkeypatch):
    """A row that has all its tokens goes on computing rows that are thrown away: one without any probability there (-1), or right
    behind the last token, is not an error, and no -1 reaches the embedding."""
    from kubeoperator_amd.serve import generate

    m = model("cpu")
    gen, draft = (LlamaGenerator(m, max_batch=2, max_seq=40) for _ in range(2))
    ids, n, verify, calls = ids_of(m, 2, 10), 8, kf.verify_draft, []

    def stub(target, d, tokens, u, temperature=1.0, n_draft=None):
        """Checks of drafts: row 0 keeps all three, row 1 none; row 0 finds no token behind its eighth (the second round)
        and later."""
        if tokens.shape[1] == 0:
            return verify(target, d, tokens, u, temperature, n_draft)
        calls.append(0)
        best = target.argmax(-1)
        out = torch.full((2, 4), -1)
        out[0, :3], out[0, 3], out[1, 0] = tokens[0], best[0, 3] if len(calls) < 2 else -1, best[1, 0]
        return out, torch.tensor([3, 0], dtype=torch.int32)

    monkeypatch.setattr(generate.kf, "verify_draft", stub)
    out, rounds = gen.speculate(draft, ids, n, drafts=3)
    assert len(rounds) == 7 and ((out >= 0) & (out < m.cfg.vocab_size)).all()
    monkeypatch.undo()
    is_greedy("cpu", LlamaGenerator(m, 2, 40), ids, out, n)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("n", [1, 2, 13])
@pytest.mark.parametrize("prefix", [0, 30])
def test_caches_after_speculation(dev, n, prefix):
    """They hold what generate() leaves there, everything but the last token returned, for each sequence and in both models: decoding
    goes on from it."""
    m, other = model(dev, size=0.08), model(dev, size=0.08, seed=1)
    with torch.no_grad():  # sequences that keep different numbers of drafts
        for p, q in zip(other.parameters(), m.parameters()):
            p.copy_(0.97 * q + 0.03 * p)
    ids = ids_of(m, 3, 12)
    new = lambda x: LlamaGenerator(x, max_batch=3, max_seq=40)  # noqa: E731
    gens = [new(m), new(other)]
    for g in gens:
        if prefix:
            g.set_prefix(ids_of(m, 1, prefix, seed=9)[0])
    got, _ = gens[0].speculate(gens[1], ids, n, drafts=3)
    for g, x in zip(gens, (m, other)):
        assert g.cache.host_lens == [12 + n - 1] * 3 == g.cache.lens.tolist()
        fresh = new(x)
        if prefix:
            fresh.set_prefix(ids_of(m, 1, prefix, seed=9)[0])
        close(g.decode(got[:, -1]), fresh.prefill(got))
