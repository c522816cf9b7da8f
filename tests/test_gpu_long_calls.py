"""GPU checks of calls that the long-cache operators' contracts allow beside
the ordinary ones of test_gpu_long.py. Integer arithmetic: exact equality."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from pagedcache import PAGE, paged, unpaged

pytestmark = pytest.mark.gpu
I64 = torch.int64


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from idempotent_llm_amd import _lib, torch_ops  # noqa: F401
    _lib.load()


def _ops():
    return torch.ops.detllm_rocm


# B, n_kv, slots, kept (the budget), pages of dst
WIDER = {
    "one_more": (2, 2, 300, 100, 2),
    "whole_page": (1, 1, 300, 128, 2),
    "many": (3, 2, 900, 200, 7),
    "all_zero": (2, 1, 300, 0, 2),
    "parts": (1, 1, 5000, 3000, 40),
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", list(WIDER))
def test_compact_to_more_pages_than_the_budget(name, in_place):
    """Pages of dst behind the budget's become 0 like the slots behind the
    last kept one."""
    B, n_kv, S, budget, wide = WIDER[name]
    print(f"[compact wider {name} in_place={in_place}]", flush=True)
    rng = np.random.default_rng(wide)
    kc = rng.integers(-128, 128, (B, n_kv, S, 128), dtype=np.int8)
    vc = rng.integers(-128, 128, (B, n_kv, 128, S), dtype=np.int8)
    kp, vp, table, w = paged(kc, vc, seed=5)
    keep = np.stack([np.sort(rng.choice(S, budget, replace=False)) for _ in range(B)])
    keep = keep.astype(np.int32)
    fresh = torch.arange(B * w, B * (w + wide), dtype=torch.int32, device="cuda").view(B, wide)
    dst = fresh.clone()
    if in_place:
        dst[:, :min(w, wide)] = table[:, :min(w, wide)]
    kp, vp = (torch.cat([x, torch.full((B * wide,) + x.shape[1:], 77, dtype=torch.int8,
                                       device="cuda")]) for x in (kp, vp))
    before = kp.clone(), vp.clone()
    _ops().kv_compact([kp], [vp], table, dst, torch.from_numpy(keep).cuda())
    k, v = (x.cpu().numpy() for x in unpaged(kp, vp, dst, wide * PAGE))
    for b in range(B):
        assert np.array_equal(k[b, :, :budget], kc[b][:, keep[b]])
        assert np.array_equal(v[b, :, :budget], vc[b].transpose(0, 2, 1)[:, keep[b]])
    assert not k[:, :, budget:].any() and not v[:, :, budget:].any()
    others = torch.ones(kp.shape[0], dtype=torch.bool, device="cuda")
    others[dst.reshape(-1).long()] = False
    assert torch.equal(kp[others], before[0][others]) and torch.equal(vp[others], before[1][others])


def test_select_with_the_largest_budget():
    """2^31 - 2 places for 300 slots: everything stays, -1 and 0 behind it."""
    print("[select largest budget]", flush=True)
    S, budget = 300, 2**31 - 2
    acc = torch.arange(1, S + 1, dtype=I64, device="cuda").view(1, 1, S)
    valid = torch.arange(S, device="cuda")[None] % 3 != 1
    live = valid[0].nonzero()[:, 0]
    n = len(live)
    keep, kept = _ops().kv_select(acc, valid, S, budget, 0, 0)
    torch.cuda.synchronize()
    assert keep.shape == (1, budget) and kept.shape == (1, 1, budget)
    assert torch.equal(keep[0, :n].long(), live) and torch.equal(kept[0, 0, :n], acc[0, 0, live])
    assert int(keep[0, n:].max()) == -1 and int(keep[0, n:].min()) == -1
    assert int(kept[0, 0, n:].max()) == 0 and int(kept[0, 0, n:].min()) == 0


@pytest.mark.parametrize("slots,pages", [((70000, 70100), 1094), ((131071,), 1024),
                                         ((66000, 66049), 1032)])
def test_evict_of_long_caches(slots, pages):
    """Caches whose table doubled past 1024 pages, and the longest one."""
    from idempotent_llm_amd.kvcache import KVCache
    print(f"[evict long {slots}]", flush=True)
    model = SimpleNamespace(n_layers=2, n_kv=1, hd=128, device=torch.device("cuda"))
    c = KVCache().track_weights()
    for n in slots:
        c.reserve(model, 2, n)
    S = c.length = slots[-1]
    assert c.width == pages
    g = torch.Generator(device="cuda").manual_seed(S)
    for pool in c.k_pools + c.v_pools:
        pool.copy_(torch.randint(-128, 128, pool.shape, dtype=torch.int8, device="cuda",
                                 generator=g))
    c.valid_buf[:, :S] = torch.rand(2, S, device="cuda", generator=g) < 0.9
    c.acc[:, :, :S] = torch.randint(0, 1 << 40, (2, 1, S), device="cuda", generator=g)
    keep, kept = _ops().kv_select(c.acc, c.valid_buf, S, 900, 50, 4)
    at = keep.long()[:, None, :, None].expand(2, 1, 900, 128)
    want = [x.gather(2, at) for x in c.k8 + c.v8]
    c.evict(900, 50, 4)
    assert c.length == 900 and bool(c.valid.all()) and torch.equal(c.acc[:, :, :900], kept)
    assert all(torch.equal(x, y) for x, y in zip(c.k8 + c.v8, want))


# B, n_q, n_kv, S, window and sinks or None: the forms that need scratch
SCRATCH = {
    "window_cut": (1, 16, 8, 5000, (4000, 4)),
    "window_cut_rows": (40, 4, 2, 9000, (8000, 4)),
    "window_scores": (2, 8, 1, 8000, (300, 4)),
    "acc_cut": (3, 16, 8, 5000, None),
    "acc_cut_8": (1, 8, 1, 2500, None),
    "shared_cut": (2, 16, 8, 4500, 4352),
    "shared_once": (33, 16, 8, 2640, 2560),
    "shared_once_few": (8, 4, 1, 4200, 4096),
    "shared_once_many": (20, 64, 8, 4240, 4096),
}


@pytest.mark.parametrize("name", list(SCRATCH))
def test_scratch_is_enough(name):
    """Every form writes the bytes that its planner names and none behind."""
    import ctypes
    from idempotent_llm_amd._lib import attn_acc_work, attn_shared_work, call, load
    B, n_q, n_kv, S, extra = SCRATCH[name]
    print(f"[scratch {name}]", flush=True)
    g = torch.Generator(device="cuda").manual_seed(S)
    w = -(-S // PAGE)
    rnd = lambda *s: torch.randint(-128, 128, s, dtype=torch.int8, device="cuda", generator=g)
    kp, vp, q8 = rnd(B * w, n_kv, 128, 128), rnd(B * w, n_kv, 128, 128), rnd(B, n_q, 128)
    tpos = torch.randint(1500, 24000, (B, n_q), dtype=I64, device="cuda", generator=g)
    table = torch.randperm(B * w, device="cuda", generator=g).view(B, w).to(torch.int32)
    valid = torch.rand(B, w * PAGE, device="cuda", generator=g) < 0.9
    if name.startswith("shared"):
        table[:, :extra // PAGE] = table[:1, :extra // PAGE].clone()
        n, joint = attn_shared_work(B, S, n_q, n_kv, extra)
        assert joint == ("once" in name)
        entry, tail = "detllm_attn_decode_shared", (extra,)
    elif name.startswith("acc"):
        acc = torch.zeros(B, n_kv, S, dtype=I64, device="cuda")
        n, entry, tail = attn_acc_work(B, S, n_q, n_kv), "detllm_attn_decode_acc", (acc, S)
    else:
        bytes_ = ctypes.c_int64(0)
        assert load().detllm_attn_window_decode_work(B, S, n_q, n_kv, *extra,
                                                     ctypes.byref(bytes_)) == 0
        n, entry, tail = bytes_.value, "detllm_attn_window_decode", extra
    assert n > 0
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = _ops().attn_decode(q8, tpos, kp, vp, table, valid, S, err)
    if name.startswith("window"):
        want = _ops().attn_window_decode(q8, tpos, kp, vp, table, valid, S, *extra)
    out = torch.zeros(B, n_q * 128, dtype=I64, device="cuda")
    work = torch.full((2 * n + (1 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    call(entry, q8, tpos, kp, vp, table, w, valid.view(torch.uint8), w * PAGE, B, S, n_q, n_kv,
         None, *tail, work, n, out, err)
    assert torch.equal(out, want) and int(err) == 0
    assert bool((work[n:] == 0xA5).all())
