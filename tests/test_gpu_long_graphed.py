"""Long-context caches under the graphed decode: what form its steps take and
that they answer as eager ones. Exact equality."""

import pytest
import torch

from idempotent_llm_amd import artifact as art

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from idempotent_llm_amd.model import IntQwen3
    d = str(tmp_path_factory.mktemp("a"))
    art.make_artifact(d, dict(art.MID, max_pos=8192), 7)
    return IntQwen3(d, backend="rocm")


def _prompt(m, T, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, m.vocab, (1, T), generator=g).cuda(),
            torch.arange(T, device="cuda").view(1, T))


def _step(m, cache, cur, pos):
    return m.forward(cur[:, None], pos[:, None], cache)[0][:, 0]


@pytest.mark.parametrize("mode,greedy", [("capture", False), ("capture", True), ("layers", False)])
@pytest.mark.parametrize("T,rows,joint_steps", [(2060, 14, 9), (2170, 14, 6), (4350, 20, 9)])
def test_graphed_forks_read_the_prefix_once(model, monkeypatch, T, rows, joint_steps, mode, greedy):
    """The capacity (the next bucket) leaves more room behind the prefix than
    the joint form is for; the steps take it by their own slots, and give it up
    where these become too many."""
    from idempotent_llm_amd import model as module
    from idempotent_llm_amd.graphed import GraphedDecode
    from idempotent_llm_amd.kvcache import KVCache
    print(f"[graphed fork T={T} rows={rows} {mode} {greedy}]", flush=True)
    m, steps = model, 9
    ids, pos = _prompt(m, T, 4)
    caches = []
    for _ in range(2):
        c = KVCache()
        m.forward(ids, pos, c)
        caches.append(c.fork(rows))
    at = torch.full((rows,), T, device="cuda")
    cur = torch.arange(rows, device="cuda") + 5
    real, names = module.call, []
    monkeypatch.setattr(module, "call", lambda name, *a: (names.append(name), real(name, *a))[1])
    gd = GraphedDecode(m, caches[1], at, mode=mode)
    assert caches[1].static_cap > T + 1000
    for s in range(steps):
        del names[:]
        pools = caches[1].pool_generation
        got = gd.step_greedy(cur).clone() if greedy else gd.step(cur).clone()
        now = "detllm_attn_decode_shared" in names
        if names:       # (a replay calls nothing)
            assert now == (s < joint_steps), s
        grown = caches[1].pool_generation != pools
        assert bool(names) == (mode == "layers" or s in (0, joint_steps) or grown), s
        del names[:]
        want = _step(m, caches[0], cur, at + s)
        assert ("detllm_attn_decode_shared" in names) == (s < joint_steps), s
        if greedy:
            assert torch.equal(gd.out_pick[:, 0], want) and torch.equal(got, m.greedy_pick(want))
        else:
            assert torch.equal(got, want)
        cur = m.greedy_pick(want)
    m.raise_if_device_error()


@pytest.mark.parametrize("greedy", [False, True])
def test_weights_of_graphed_steps_drive_an_eviction(model, greedy):
    """decode, evict, decode with the steps graphed: the cache is released for
    the eviction, and tokens, weights and pages are those of eager steps."""
    from idempotent_llm_amd.graphed import GraphedDecode
    from idempotent_llm_amd.kvcache import KVCache
    print(f"[graphed evict {greedy}]", flush=True)
    m, B, T = model, 3, 200
    g = torch.Generator().manual_seed(9)
    ids = torch.randint(0, m.vocab, (B, T), generator=g).cuda()
    pos = torch.arange(T, device="cuda").expand(B, T).contiguous()
    lens = torch.tensor((200, 150, 180), device="cuda")
    valid = torch.arange(T, device="cuda")[None] < lens[:, None]
    eager, graphed = KVCache().track_weights(), KVCache().track_weights()
    for c in (eager, graphed):
        m.forward(ids, pos, c, valid)
    cur, at = ids[:, 0].clone(), lens
    for turn in range(3):
        gd = GraphedDecode(m, graphed, at)
        with pytest.raises(ValueError, match="graphed"):
            graphed.evict(128, 30, 4)
        for s in range(4):
            want = _step(m, eager, cur, at)
            if greedy:
                got = gd.step_greedy(cur).clone()
                assert torch.equal(gd.out_pick[:, 0], want)
                assert torch.equal(got, m.greedy_pick(want))
            else:
                assert torch.equal(gd.step(cur), want)
            cur, at = m.greedy_pick(want), at + 1
        assert gd.release() is graphed and graphed.length == eager.length
        for f in (lambda: gd.step(cur), lambda: gd.step_greedy(cur), gd.release):
            with pytest.raises(ValueError, match="released"):
                f()
        n = eager.length
        assert torch.equal(graphed.acc[:, :, :n], eager.acc[:, :, :n])
        assert torch.equal(graphed.valid, eager.valid)
        for c in (eager, graphed):
            c.evict(128, 30, 4)
        assert torch.equal(graphed.acc[:, :, :128], eager.acc[:, :, :128])
        assert all(torch.equal(x, y) for x, y in zip(graphed.k8 + graphed.v8, eager.k8 + eager.v8))
    # eager chunks work on it as well
    chunk = ids[:, :7].contiguous()
    where = at[:, None] + torch.arange(7, device="cuda")
    assert torch.equal(m.forward(chunk, where, eager)[0], m.forward(chunk, where, graphed)[0])


def test_release_leaves_a_cache_that_another_decode_took(model):
    from idempotent_llm_amd.graphed import GraphedDecode
    from idempotent_llm_amd.kvcache import KVCache
    print("[release of a cache taken over]", flush=True)
    m = model
    ids, pos = _prompt(m, 50, 3)
    one, ref = KVCache(), KVCache()
    for c in (one, ref):
        m.forward(ids, pos, c)
    at, cur = torch.tensor([50], device="cuda"), ids[:, 0].clone()
    first = GraphedDecode(m, one, at)
    assert torch.equal(first.step(cur), _step(m, ref, cur, at))
    second = GraphedDecode(m, one, at + 1)
    first.release()
    assert one.static_cap
    for s in (1, 2):
        assert torch.equal(second.step(cur), _step(m, ref, cur, at + s))
    second.release()
    assert not one.static_cap and one.length == ref.length
