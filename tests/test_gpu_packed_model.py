"""Packed steps in the model: requests of any lengths in one batch, their prompts in
chunks, with and without adapters, against each request alone. Exact equality."""

import numpy as np
import pytest
import torch

import packedcases as pc
from idempotent_llm_amd import artifact as art

pytestmark = pytest.mark.gpu
I64 = torch.int64


@pytest.fixture(scope="module")
def artifact(tmp_path_factory):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    d = str(tmp_path_factory.mktemp("a"))
    art.make_artifact(d, art.MID, 7)
    return d


@pytest.fixture(scope="module")
def model(artifact):
    from idempotent_llm_amd.model import IntQwen3
    return IntQwen3(artifact, backend="rocm")


def _prompts(m, lens, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, m.vocab, (n,), generator=g) for n in lens]


def _alone(m, ids):
    """Logits of every token of one request, its tokens in one piece."""
    n = ids.numel()
    return m.forward(ids[None], torch.arange(n)[None])[0][0]


STEPS = {
    "chunks": ((70, 5, 130), ([64, 1, 0], [0, 1, 129], [1, 1, 1], [5, 2, 0])),
    "decode": ((40, 1, 300), ([39, 0, 299], [1, 1, 1])),
    "one_row": ((200,), ([1], [127], [1], [71])),
    "idle": ((3, 20, 4, 9), ([0, 20, 0, 0], [3, 0, 0, 8], [0, 0, 4, 1])),
}


@pytest.mark.parametrize("name", list(STEPS))
def test_steps_are_the_requests_alone(model, name):
    from idempotent_llm_amd.packed import PackedCache
    print(f"[packed steps {name}]", flush=True)
    lens, steps = STEPS[name]
    ids = _prompts(model, lens, 1)
    want = [_alone(model, x) for x in ids]
    cache = PackedCache(model, len(lens), max(lens))
    at = [0] * len(lens)
    for i, new in enumerate(steps):
        step = torch.cat([x[p:p + n] for x, p, n in zip(ids, at, new)])
        got = model.forward_packed(step.cuda() if i % 2 else step, new, cache)
        at = [p + n for p, n in zip(at, new)]
        last = torch.stack([w[p - 1] for w, p, n in zip(want, at, new) if n])
        assert torch.equal(got, last)
        assert cache.lens == at and cache.past.tolist() == at
    model.raise_if_device_error()


def test_rows_are_taken_up_again(model):
    """Released rows, rows cut back to a prefix (a rejected draft), and a step that
    only gives pages back."""
    from idempotent_llm_amd.packed import OutOfPages, PackedCache
    print("[packed rows taken up again]", flush=True)
    m, (a, b, c) = model, _prompts(model, (300, 200, 260), 2)
    cache = PackedCache(m, 2, 512, pages=5)
    m.forward_packed(torch.cat([a, b]), (300, 200), cache)
    with pytest.raises(OutOfPages):
        m.forward_packed(c[:100], (100, 0), cache)
    assert cache.lens == [300, 200] and cache.pages_left() == 0
    cache.release(0, 150)
    got = m.forward_packed(torch.cat([c[:20], b[:1]]), (20, 1), cache)
    assert torch.equal(got[0], _alone(m, torch.cat([a[:150], c[:20]]))[-1])
    assert torch.equal(got[1], _alone(m, torch.cat([b, b[:1]]))[-1])
    cache.release(0)
    cache.release(1)
    assert m.forward_packed(torch.empty(0, dtype=I64), (0, 0), cache).shape == (0, m.vocab)
    assert int(cache.n_free) == 5 and sorted(cache.free.tolist()) == list(range(5))
    assert torch.equal(m.forward_packed(c, (0, 260), cache)[0], _alone(m, c)[-1])
    m.raise_if_device_error()


@pytest.mark.parametrize("rows,step_tokens,pages", [(5, 512, None), (2, 40, None), (3, 64, 4)])
def test_generate_packed(model, rows, step_tokens, pages):
    from idempotent_llm_amd.packed import generate_packed
    print(f"[generate packed {rows} {step_tokens} {pages}]", flush=True)
    m = model
    prompts = _prompts(m, (30, 1, 150, 64, 9), 3)
    most = [6, 3, 1, 0, 9]
    got = generate_packed(m, prompts, most, rows=rows, step_tokens=step_tokens, pages=pages)
    for p, n, g in zip(prompts, most, got):
        want = m.generate(p[None], n)[0][0].cpu() if n else torch.empty(0, dtype=I64)
        assert torch.equal(g, want)


def _bank(m, n, rank, modules, seed):
    from idempotent_llm_amd.lora import AdapterBank
    bank = AdapterBank(m, n, rank)
    g = torch.Generator().manual_seed(seed)
    site = {"q": "qkv", "k": "qkv", "v": "qkv", "o": "o", "gate": "gu", "up": "gu", "down": "d"}
    for i in range(n):
        bank.set(i, {(li, mod): (torch.randn(rank - i % 2, bank.depth[site[mod]], generator=g),
                                 torch.randn(bank.cols[mod], rank - i % 2, generator=g) * 1e-3)
                     for li in range(m.n_layers) for mod in modules})
    return bank


@pytest.mark.parametrize("modules", [("q", "v"), ("q", "k", "v", "o", "gate", "up", "down")])
def test_adapters_per_row(model, artifact, modules):
    """Rows of three adapters and none in one step, against a model whose products
    get the adapters in 64 bits on the host."""
    from idempotent_llm_amd.model import IntQwen3
    from idempotent_llm_amd.packed import PackedCache, generate_packed
    print(f"[adapters {modules}]", flush=True)
    bank = _bank(model, 3, 5, modules, 4)

    class Host(IntQwen3):
        which = -1

        def _gemm(self, x, w, *args, **kw):
            P, ns, st = super()._gemm(x, w, *args, **kw)
            for li, L in enumerate(self.layers):
                for site, p in (("qkv", L.wqkv), ("o", L.wo), ("gu", L.wgu), ("d", L.wd)):
                    if w is p:
                        part = [t.cpu().numpy() for t in bank.sites[li][site]]
                        P[0] = torch.from_numpy(pc.lora(
                            P[0].cpu().numpy(), x.cpu().numpy(), *part,
                            np.full(x.shape[0], self.which))).cuda()
            return P, ns, st

    host = Host(artifact, backend="rocm")
    lens, which = (40, 70, 9, 5), (2, -1, 0, 2)
    ids = _prompts(model, lens, 5)
    want = []
    for x, a in zip(ids, which):
        host.which = a
        want.append(_alone(host, x))
    assert torch.equal(want[1], _alone(model, ids[1]))
    assert not torch.equal(want[0], _alone(model, ids[0]))
    cache = PackedCache(model, 4, 70)
    at = [0] * 4
    for new in ([39, 70, 0, 4], [1, 0, 8, 1], [0, 0, 1, 0]):
        step = torch.cat([x[p:p + n] for x, p, n in zip(ids, at, new)])
        got = model.forward_packed(step, new, cache, bank, which)
        at = [p + n for p, n in zip(at, new)]
        assert torch.equal(got, torch.stack([w[p - 1] for w, p, n in zip(want, at, new) if n]))
    # a scheduler's run: each reply begins with the host model's choice
    got = generate_packed(model, ids, 2, rows=3, step_tokens=50, adapters=bank,
                          adapter_of=[a if a >= 0 else None for a in which])
    for g, w in zip(got, want):
        assert int(g[0]) == int(model.greedy_pick(w[-1:])[0])
    model.raise_if_device_error()


def test_refusals(model, artifact, tmp_path):
    from types import SimpleNamespace

    from idempotent_llm_amd.lora import AdapterBank
    from idempotent_llm_amd.model import IntQwen3
    from idempotent_llm_amd.packed import PackedCache
    print("[packed refusals]", flush=True)
    m = model
    cache, ids = PackedCache(m, 2, 3000), torch.zeros(3, dtype=I64)
    bank = AdapterBank(m, 2, 4)
    for args in ((ids, (1, 1)), (ids[None], (1, 2)), (ids, (1, 2, 0)), (ids, (4, -1)),
                 (ids, (1, 2), cache, bank), (ids, (1, 2), cache, bank, (0,)),
                 (ids, (1, 2), cache, bank, (0, 2)), (ids, (1, 2), cache, bank, (-2, 0))):
        with pytest.raises(ValueError):
            m.forward_packed(*args[:2], cache, *args[3:])
    with pytest.raises(IndexError):                    # past the rotation tables
        m.forward_packed(torch.zeros(2500, dtype=I64), (2500, 0), cache)
    with pytest.raises(IndexError):
        m.forward_packed(torch.tensor([0, m.vocab, 0]), (1, 2), cache)
    shape = dict(n_layers=m.n_layers, n_kv=m.n_kv, device=m.device)
    for kw in (dict(n_layers=1), dict(n_kv=4)):
        with pytest.raises(ValueError, match="kv heads"):
            m.forward_packed(ids, (1, 2), PackedCache(SimpleNamespace(**{**shape, **kw}), 2, 100))
    bank.cols = dict(bank.cols, q=128)
    with pytest.raises(ValueError, match="adapters"):
        m.forward_packed(ids, (1, 2), cache, bank, (0, 0))

    class Seams(IntQwen3):
        def _attn_context(self, probs, V8r, L, aux=None):
            return super()._attn_context(probs, V8r, L, aux)

    with pytest.raises(NotImplementedError):
        Seams(artifact, backend="rocm").forward_packed(ids, (1, 2), cache)
    assert cache.lens == [0, 0] and int(cache.n_free) == cache.pages
    # a device token id out of range is flagged, as forward's are
    m.forward_packed(torch.tensor([0, m.vocab, 0]).cuda(), (1, 2), cache)
    with pytest.raises(IndexError):
        m.raise_if_device_error()
