"""The long-context cache in the model: weights tracked over a prompt and its
reply, eviction between steps, and rows forked from one prefix. Exact equality
throughout; the references are the model's own seams (probabilities), masks in
place of compaction, and a batch of equal prompts in place of a fork."""

import pytest
import torch

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


def _prompt(m, B, T, seed, lens=None):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, m.vocab, (B, T), generator=g).cuda()
    valid = torch.ones(B, T, dtype=torch.bool, device="cuda")
    if lens is not None:
        valid = torch.arange(T, device="cuda")[None] < torch.tensor(lens, device="cuda")[:, None]
    return ids, torch.arange(T, device="cuda").expand(B, T).contiguous(), valid


def _step(m, cache, cur, pos):
    logits, _, _, _ = m.forward(cur[:, None], pos[:, None], cache)
    return logits[:, 0]


def test_tracked_prompt_adds_the_seams_probabilities(model, artifact):
    """acc after a ragged prompt: the probabilities that reach the context
    seam, summed over layers, query heads and the queries of real tokens."""
    from idempotent_llm_amd.kvcache import KVCache
    from idempotent_llm_amd.model import IntQwen3
    print("[tracked prompt]", flush=True)
    seen = []

    class Probe(IntQwen3):
        def _attn_context(self, probs, V8r, L, aux=None):
            seen.append(probs.to(I64))
            return super()._attn_context(probs, V8r, L, aux)

    B, T = 3, 70
    ids, pos, valid = _prompt(model, B, T, 1, (70, 41, 66))
    plain, _, _, _ = Probe(artifact).forward(ids, pos, None, valid)
    cache = KVCache().track_weights()
    logits, _, _, _ = model.forward(ids, pos, cache, valid)
    assert torch.equal(logits, plain)
    p = sum(torch.where(valid[:, None, :, None], x, 0) for x in seen)   # [B, n_q, T, S]
    want = p.view(B, model.n_kv, -1, T).sum(2)
    assert len(seen) == model.n_layers and torch.equal(cache.acc[:, :, :T], want)
    assert not cache.acc[:, :, T:].any()
    with pytest.raises(NotImplementedError):
        Probe(artifact).forward(ids, pos, KVCache().track_weights(), valid)


@pytest.mark.parametrize("B", [1, 3])
def test_tracked_decode_eager_and_graphed(model, B):
    """Tracking changes no logit; the graphed steps add what the eager ones
    do (each once: the capture's warm-up is taken back), and each step of a
    row adds about 2^14 per query head and layer."""
    from idempotent_llm_amd.graphed import GraphedDecode
    from idempotent_llm_amd.kvcache import KVCache
    print(f"[tracked decode B={B}]", flush=True)
    m, T, steps = model, 40, 5
    lens = torch.tensor((40, 25, 31)[:B], device="cuda")
    ids, pos, valid = _prompt(m, B, T, 2, lens.tolist())
    caches = [KVCache(), KVCache().track_weights(), KVCache().track_weights()]
    for c in caches:
        m.forward(ids, pos, c, valid)
    gd = GraphedDecode(m, caches[2], lens)
    cur = ids[:, 0].clone()
    for s in range(steps):
        want = _step(m, caches[0], cur, lens + s)
        before = caches[1].acc.sum((1, 2))
        assert torch.equal(_step(m, caches[1], cur, lens + s), want)
        assert torch.equal(gd.step(cur), want)
        a, b = caches[1].acc, caches[2].acc
        n = min(a.shape[2], b.shape[2])
        assert torch.equal(a[:, :, :n], b[:, :, :n])
        grown = a.sum((1, 2)) - before
        rows, slots = m.n_layers * m.n_q, T + s + 1
        assert bool(((grown - rows * (1 << 14)).abs() <= rows * slots / 2).all())
        cur = want.argmax(-1)


@pytest.mark.parametrize("lens,budget,recent,sinks", [((150, 90, 131), 64, 16, 4),
                                                      ((150, 150, 150), 140, 0, 0),
                                                      ((300, 20, 290), 129, 40, 1)])
def test_evicted_cache_answers_as_a_masked_one(model, lens, budget, recent, sinks):
    """After eviction the model's logits are those of the same cache with the
    evicted slots masked, eager steps and a graphed decode behind them; a
    second eviction and new tokens work on the pages handed back."""
    from idempotent_llm_amd.graphed import GraphedDecode
    from idempotent_llm_amd.kvcache import KVCache
    print(f"[evict {lens} {budget}]", flush=True)
    m, B, T = model, len(lens), max(lens)
    at = torch.tensor(lens, device="cuda")
    ids, pos, valid = _prompt(m, B, T, 3, lens)
    full, cut = KVCache(), KVCache().track_weights()
    for c in (full, cut):
        m.forward(ids, pos, c, valid)
    cur = ids[:, 1].clone()
    for round_ in range(2):
        keep, kept = torch.ops.detllm_rocm.kv_select(cut.acc, cut.valid_buf, cut.length, budget,
                                                     recent, sinks)
        # the same slots by their place in the cache that keeps everything
        where = full_slots if round_ else torch.arange(T, device="cuda").expand(B, T)
        full_slots = torch.where(keep >= 0, where.gather(1, keep.clamp(min=0).long()), -1)
        mask = torch.zeros_like(full.valid_buf)
        for b in range(B):
            mask[b, full_slots[b][full_slots[b] >= 0]] = True
        pool = cut.k_pools[0].data_ptr()
        cut.evict(budget, recent, sinks)
        assert cut.length == budget and cut.k_pools[0].data_ptr() == pool
        assert torch.equal(cut.valid, keep >= 0) and torch.equal(cut.acc[:, :, :budget], kept)
        used = cut._table_host[cut._table_host >= 0]
        assert len(set(used.tolist())) == used.size and not set(used.tolist()) & set(cut._free)
        full.valid_buf.copy_(mask)
        for s in range(3):
            a, b = _step(m, full, cur, at), _step(m, cut, cur, at)
            assert torch.equal(a, b)
            new = torch.full((B, 1), full.length - 1, device="cuda")
            full_slots = torch.cat([full_slots, new], dim=1)
            cur, at = b.argmax(-1), at + 1
    gd = GraphedDecode(m, cut, at)
    for s in range(3):
        a, b = _step(m, full, cur, at), gd.step(cur)
        assert torch.equal(a, b)
        cur, at = a.argmax(-1), at + 1


@pytest.mark.parametrize("T,rows", [(200, 3), (256, 2), (1950, 14)])
def test_forked_rows_answer_as_equal_prompts(model, T, rows):
    """Rows forked from one prompt give the logits of as many equal prompts,
    eager (the longest case reads its prefix once for the batch), graphed and
    as a chunk; evicting them copies what they share."""
    from idempotent_llm_amd.graphed import GraphedDecode
    from idempotent_llm_amd.kvcache import KVCache
    print(f"[fork T={T} rows={rows}]", flush=True)
    m = model
    ids, pos, _ = _prompt(m, 1, T, 4)
    one, many = KVCache().track_weights(), KVCache()
    m.forward(ids, pos, one)
    m.forward(ids.expand(rows, T).contiguous(), pos.expand(rows, T).contiguous(), many)
    one.fork(rows)
    one.tracking, acc, one.acc = False, one.acc, None      # (the shared form tracks no weights)
    assert m._joint(rows, T + 1, one.shared) == (rows == 14)
    at = torch.full((rows,), T, device="cuda")
    cur = torch.arange(rows, device="cuda") + 5            # the rows part here
    for s in range(3):
        a, b = _step(m, many, cur, at), _step(m, one, cur, at)
        assert torch.equal(a, b)
        cur, at = a.argmax(-1), at + 1
    chunk = torch.arange(rows * 9, device="cuda").view(rows, 9) + 3
    where = at[:, None] + torch.arange(9, device="cuda")
    a, b = (m.forward(chunk, where, c)[0] for c in (many, one))
    assert torch.equal(a, b)
    cur, at = a[:, -1].argmax(-1), at + 9
    # eviction: weights of the prompt's slots, none of the rest
    one.tracking, one.acc = True, torch.zeros(rows, m.n_kv, one.cap, dtype=I64, device="cuda")
    one.acc[:, :, :T] = acc[:, :, :T]
    keep, _ = torch.ops.detllm_rocm.kv_select(one.acc, one.valid_buf, one.length, 160, 30, 4)
    mask = torch.zeros_like(many.valid_buf)
    for r in range(rows):
        mask[r, keep[r].long()] = True
    one.evict(160, 30, 4)
    many.valid_buf.copy_(mask)
    assert one.shared == 0
    assert torch.equal(_step(m, many, cur, at), _step(m, one, cur, at))
    at = at + 1
    one.tracking, one.acc = False, None
    # a graphed decode of a fork
    two = KVCache()
    m.forward(ids, pos, two)
    two.fork(rows)
    ref = KVCache()
    m.forward(ids.expand(rows, T).contiguous(), pos.expand(rows, T).contiguous(), ref)
    at = torch.full((rows,), T, device="cuda")
    gd = GraphedDecode(m, two, at)
    for s in range(4):
        a, b = _step(m, ref, cur, at), gd.step(cur)
        assert torch.equal(a, b)
        cur, at = a.argmax(-1), at + 1
