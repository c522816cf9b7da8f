"""GPU checks of the long-cache operators (windowed attention with sinks,
attention that accumulates its weights, eviction by those weights, decode
attention of a shared prefix) against 64-bit loops over the CPU oracle
(longcases.py). Everything is integer arithmetic: exact equality."""

import numpy as np
import pytest
import torch

import longcases as lc
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


def _dev(c, seed=0):
    """The operators' leading operands (q8, tpos, kpool, vpool, table, valid)."""
    kp, vp, table, _, valid = paged(c["kc"], c["vc"], c["valid"], seed=seed)
    return (torch.from_numpy(c["q8"]).cuda(), torch.from_numpy(c["tpos"]).cuda(), kp, vp, table,
            valid)


def _eq(got, want):
    assert np.array_equal(got.cpu().numpy(), want)


# ------------------------------------------------------------ windowed attention

# B, n_q, n_kv, S, window, sinks, extras of longcases.make
WINDOW_DECODE = {
    "one_slot": (1, 2, 1, 1, 1, 0, {}),
    "one_slot_sinks": (2, 2, 2, 1, 5, 9, {}),
    "window_1": (2, 4, 2, 300, 1, 0, {}),
    "window_1_sink_1": (2, 4, 2, 300, 1, 1, dict(p_valid=0.5)),
    "page_edges": (2, 2, 2, 512, 128, 128, {}),
    "one_off_edges": (2, 2, 2, 513, 129, 127, {}),
    "gapless_all": (2, 8, 2, 260, 4096, 4, {}),
    "wide_window": (1, 2, 1, 200, 2**31 - 1, 2**31 - 1, {}),
    "padding": (4, 4, 2, 700, 150, 4, dict(gaps=((0, 50, 600), (1, 0, 699), (2, 100, 101),
                                                 (3, 300, 700)))),
    "sparse": (3, 16, 8, 1500, 200, 3, dict(p_valid=0.1)),
    "dead_row": (3, 2, 2, 400, 64, 4, dict(dead_rows=(1,))),
    "group_8": (2, 8, 1, 600, 100, 4, dict(p_valid=0.9)),
    "group_8_long": (1, 8, 1, 3000, 1800, 4, dict(p_valid=0.9)),
    "group_4_long": (2, 32, 8, 2000, 1200, 64, dict(p_valid=0.95)),
    "long": (1, 4, 2, 5000, 2500, 4, dict(p_valid=0.98)),
    "long_gap": (2, 4, 2, 6000, 900, 4, dict(gaps=((0, 1000, 5600), (1, 3, 5990)))),
    "long_gap_split": (2, 4, 2, 9000, 2000, 4, dict(gaps=((0, 500, 8600), (1, 2500, 8000)))),
    "long_gap_8": (1, 8, 1, 8000, 300, 4, dict(gaps=((0, 200, 7900),))),
    "sparse_scratch": (2, 8, 1, 8000, 600, 4, dict(p_valid=0.08)),
    "sparse_scratch_2": (3, 4, 2, 9000, 100, 4, dict(p_valid=0.01)),
    "sparse_split": (1, 4, 2, 9000, 1500, 70, dict(p_valid=0.2)),
    "wide_tpos": (2, 4, 2, 400, 120, 4, dict(tpos=(0, 62), p_valid=0.8)),
    "wide_tpos_long": (1, 4, 2, 3000, 1500, 4, dict(tpos=(0, 62), p_valid=0.8)),
    "flat": (1, 2, 1, 4000, 3000, 4, dict(flat_heads=(0, 1), tpos=(38, 39))),
    "extreme": (1, 2, 2, 500, 300, 4, dict(extreme=(0,), tpos=(28, 40))),
}


@pytest.mark.parametrize("name", list(WINDOW_DECODE))
def test_window_decode(name):
    B, n_q, n_kv, S, window, sinks, extra = WINDOW_DECODE[name]
    print(f"[window decode {name}]", flush=True)
    c = lc.make(B, n_q, n_kv, S, seed=len(name), **extra)
    want, _ = lc.attend(c, S=S, window=window, sinks=sinks)
    _eq(_ops().attn_window_decode(*_dev(c, S), S, window, sinks), want)


def test_window_decode_of_no_slots_and_no_rows():
    print("[window decode empty]", flush=True)
    c = lc.make(2, 4, 2, 130, seed=3)
    args = _dev(c)
    _eq(_ops().attn_window_decode(*args, 0, 4, 4), np.zeros((2, 512), dtype=np.int64))
    none = [x[:0] if i in (0, 1, 4, 5) else x for i, x in enumerate(args)]
    assert _ops().attn_window_decode(*none, 100, 4, 4).shape == (0, 512)


# B, n_q, n_kv, T, past, window, sinks, extras
WINDOW_PREFILL = {
    "one_query": (1, 2, 1, 1, 0, 1, 0, {}),
    "one_query_past": (2, 4, 2, 1, 333, 100, 4, dict(p_valid=0.7)),
    "window_1": (1, 2, 2, 70, 0, 1, 0, {}),
    "window_1_sink_1": (1, 2, 2, 70, 60, 1, 1, {}),
    "tile_edges": (1, 2, 1, 128, 0, 64, 0, {}),
    "odd": (2, 4, 2, 150, 37, 33, 3, dict(p_valid=0.8)),
    "three_pages": (1, 2, 2, 330, 0, 100, 1, {}),
    "window_of_all": (2, 4, 2, 150, 37, 4096, 4, dict(p_valid=0.8)),
    "wide_window": (1, 2, 1, 65, 64, 2**31 - 1, 2**31 - 1, {}),
    "sinks_past_window": (1, 2, 1, 200, 300, 50, 300, {}),
    "long_past": (1, 4, 2, 65, 1500, 300, 4, dict(p_valid=0.95)),
    "padding": (3, 2, 2, 200, 900, 150, 4, dict(gaps=((0, 100, 900), (1, 0, 1000),
                                                      (2, 1000, 1100)))),
    "sparse": (2, 2, 1, 100, 1500, 60, 3, dict(p_valid=0.08)),
    "dead_row": (2, 2, 2, 100, 200, 64, 4, dict(dead_rows=(1,))),
    "group_8": (1, 8, 1, 96, 200, 90, 5, dict(p_valid=0.9)),
    "group_3": (1, 6, 2, 96, 200, 90, 5, dict(p_valid=0.9)),
    "wide_tpos": (2, 4, 2, 150, 300, 90, 4, dict(tpos=(0, 62), p_valid=0.8)),
    "flat": (1, 2, 1, 64, 2000, 1500, 4, dict(flat_heads=(0, 1), tpos=(38, 39))),
    "extreme": (1, 2, 2, 96, 100, 90, 4, dict(extreme=(0,), tpos=(28, 40))),
}


@pytest.mark.parametrize("name", list(WINDOW_PREFILL))
def test_window_prefill(name):
    B, n_q, n_kv, T, past, window, sinks, extra = WINDOW_PREFILL[name]
    print(f"[window prefill {name}]", flush=True)
    c = lc.make(B, n_q, n_kv, past + T, seed=len(name), T=T, **extra)
    want, _ = lc.attend(c, T, past, window, sinks)
    _eq(_ops().attn_window_prefill(*_dev(c, T), past, window, sinks), want)


def test_window_over_everything_is_ordinary_attention():
    """A window as wide as the cache gives attn_prefill's and attn_decode's
    contexts (many query tiles, several chunks)."""
    print("[window as wide as the cache]", flush=True)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    c = lc.make(2, 4, 2, 1700, seed=5, T=700, p_valid=0.9)
    args = _dev(c)
    assert torch.equal(_ops().attn_window_prefill(*args, 1000, 1700, 0),
                       _ops().attn_prefill(*args, 1000))
    c = lc.make(2, 4, 2, 7000, seed=6, p_valid=0.9)
    args = _dev(c)
    assert torch.equal(_ops().attn_window_decode(*args, 7000, 7000, 0),
                       _ops().attn_decode(*args, 7000, err))


def test_window_rows_do_not_depend_on_padding():
    """The same tokens with and without padding between them: the same
    contexts (the window counts tokens, not slots)."""
    print("[window padding]", flush=True)
    S, pad = 400, 300
    c = lc.make(1, 4, 2, S, seed=8)
    wide = lc.make(1, 4, 2, S + pad, seed=9)
    at = np.concatenate([np.arange(150), np.arange(150 + pad, S + pad)])
    for n, axis in (("kc", 2), ("vc", 3)):
        idx = [slice(None)] * 4
        idx[axis] = at
        wide[n][tuple(idx)] = c[n]
    wide["valid"][:] = False
    wide["valid"][:, at] = True
    for n in ("q8", "tpos"):
        wide[n] = c[n]
    a = _ops().attn_window_decode(*_dev(c), S, 200, 4)
    assert torch.equal(a, _ops().attn_window_decode(*_dev(wide), S + pad, 200, 4))


# ------------------------------------------------------- accumulated weights

ACC_DECODE = {
    "one_slot": (1, 2, 1, 1, {}),
    "small": (3, 8, 8, 17, dict(p_valid=0.7)),
    "typical": (2, 4, 2, 320, dict(p_valid=0.8)),
    "group_4": (2, 32, 8, 1000, dict(p_valid=0.9)),
    "group_8": (2, 8, 1, 600, dict(p_valid=0.9)),
    "group_8_long": (1, 8, 1, 2500, dict(p_valid=0.9)),
    "long": (1, 4, 2, 3333, dict(p_valid=0.9)),
    "many_rows_long": (33, 8, 4, 1300, dict(p_valid=0.9)),
    "group_8_rows": (17, 64, 8, 1700, dict(p_valid=0.9)),
    "group_1_rows": (130, 1, 1, 12300, dict(p_valid=0.9)),
    "dead_rows": (3, 2, 2, 300, dict(dead_rows=(0, 2))),
    "last_slot_dead": (2, 2, 1, 300, dict(gaps=((1, 290, 300),))),
    "wide_tpos": (2, 4, 2, 400, dict(tpos=(0, 40), p_valid=0.8)),
    "flat": (1, 2, 1, 3000, dict(flat_heads=(0, 1), tpos=(38, 39))),
}


@pytest.mark.parametrize("name", list(ACC_DECODE))
def test_acc_decode(name):
    """The context is attn_decode's, the accumulators grow by the weights, and
    words past the slots stay. A second call adds the same again."""
    B, n_q, n_kv, S, extra = ACC_DECODE[name]
    print(f"[acc decode {name}]", flush=True)
    c = lc.make(B, n_q, n_kv, S, seed=len(name), **extra)
    rows = range(B) if B < 10 else (0, 1, B - 1)     # the loops' time
    sub = {k: (v[list(rows)] if isinstance(v, np.ndarray) else v) for k, v in c.items()}
    want, add = lc.attend(sub, S=S)
    args = _dev(c, S)
    acc = torch.randint(-(1 << 40), 1 << 40, (B, n_kv, S + 5), dtype=I64, device="cuda")
    start = acc.clone()
    for k in (1, 2):
        out = _ops().attn_decode_acc(*args, S, acc)
        _eq(out[list(rows)], want)
        _eq((acc - start)[list(rows), :, :S], k * add)
        assert torch.equal(acc[:, :, S:], start[:, :, S:])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(out, _ops().attn_decode(*args, S, err))


ACC_PREFILL = {
    "one_query": (1, 2, 1, 1, 0, {}),
    "small": (3, 8, 8, 17, 0, dict(p_valid=0.7)),
    "odd": (2, 4, 2, 150, 37, dict(p_valid=0.8)),
    "pages": (1, 4, 1, 300, 100, dict(p_valid=0.9)),
    "group_3": (1, 6, 2, 96, 20, {}),
    "padding": (2, 2, 2, 130, 200, dict(gaps=((0, 250, 330), (1, 0, 100)))),
    "dead_row": (2, 2, 2, 70, 10, dict(dead_rows=(1,))),
    "wide_tpos": (2, 4, 2, 150, 100, dict(tpos=(0, 40), p_valid=0.8)),
    "flat": (1, 2, 1, 64, 1500, dict(flat_heads=(0, 1), tpos=(38, 39))),
}


@pytest.mark.parametrize("name", list(ACC_PREFILL))
def test_acc_prefill(name):
    B, n_q, n_kv, T, past, extra = ACC_PREFILL[name]
    print(f"[acc prefill {name}]", flush=True)
    S = past + T
    c = lc.make(B, n_q, n_kv, S, seed=len(name), T=T, **extra)
    want, add = lc.attend(c, T, past)
    args = _dev(c, T)
    acc = torch.randint(-(1 << 40), 1 << 40, (B, n_kv, S + 5), dtype=I64, device="cuda")
    start = acc.clone()
    for k in (1, 2):
        _eq(_ops().attn_prefill_acc(*args, past, acc), want)
        _eq((acc - start)[:, :, :S], k * add)
        assert torch.equal(acc[:, :, S:], start[:, :, S:])


# ------------------------------------------------------------------ eviction

# B, n_kv, S, budget, recent, sinks, p_valid, weights
SELECT = {
    "nothing_to_do": (2, 2, 50, 60, 4, 4, 0.9, "random"),
    "exactly_full": (1, 2, 64, 64, 4, 4, 1.0, "random"),
    "one_too_many": (1, 2, 65, 64, 4, 4, 1.0, "random"),
    "budget_1": (3, 2, 500, 1, 0, 0, 0.9, "random"),
    "all_recent": (2, 2, 500, 40, 40, 0, 0.9, "random"),
    "all_sinks": (2, 2, 500, 40, 0, 40, 0.9, "random"),
    "protected_only": (2, 2, 500, 40, 30, 10, 0.9, "random"),
    "ties": (3, 1, 700, 100, 7, 3, 0.9, "ties"),
    "all_equal": (2, 8, 3000, 333, 16, 4, 1.0, "zero"),
    "typical": (4, 8, 4000, 1024, 256, 4, 0.95, "random"),
    "long": (1, 8, 20000, 5000, 100, 4, 0.9, "random"),
    "mid": (2, 8, 9000, 2000, 100, 4, 0.9, "random"),
    "ranked_ties": (2, 1, 900, 300, 5, 2, 1.0, "few"),
    "one_heavy": (2, 2, 3000, 8, 4, 3, 1.0, "one"),
    "long_ties": (1, 1, 17000, 3000, 10, 4, 0.9, "ties"),
    "wide": (3, 8, 2500, 600, 50, 4, 0.9, "wide"),
    "sparse": (3, 4, 3000, 100, 20, 4, 0.06, "random"),
    "dead": (2, 4, 300, 100, 20, 4, 0.0, "random"),
    "no_slots": (2, 4, 0, 10, 2, 2, 1.0, "random"),
}


def _weights(kind, B, n_kv, S, rng):
    if kind == "ties":
        return rng.integers(0, 5, (B, n_kv, S), dtype=np.int64)
    if kind == "few":      # groups of equal weights of about a hundred slots
        return rng.integers(0, 9, (B, n_kv, S), dtype=np.int64) << 30
    if kind == "one":      # one slot holds nearly everything
        w = np.ones((B, n_kv, S), dtype=np.int64)
        w[..., S // 3] = 1 << 50
        return w
    if kind == "zero":
        return np.zeros((B, n_kv, S), dtype=np.int64)
    if kind == "wide":     # sums that wrap, negative ones among them
        return rng.integers(-(1 << 62), 1 << 62, (B, n_kv, S), dtype=np.int64)
    return (2.0 ** rng.uniform(0, 30, (B, n_kv, S))).astype(np.int64)


@pytest.mark.parametrize("name", list(SELECT))
def test_select(name):
    B, n_kv, S, budget, recent, sinks, p_valid, weights = SELECT[name]
    print(f"[select {name}]", flush=True)
    rng = np.random.default_rng(len(name))
    acc = _weights(weights, B, n_kv, S + 3, rng)
    valid = rng.random((B, S + 7)) < p_valid
    keep, kept = _ops().kv_select(torch.from_numpy(acc).cuda(), torch.from_numpy(valid).cuda(), S,
                                  budget, recent, sinks)
    want_keep, want_kept = lc.select(acc[:, :, :S], valid[:, :S], budget, recent, sinks)
    _eq(keep, want_keep)
    _eq(kept, want_kept)


def _compacted(kc, vc, keep):
    """K [B, n_kv, slots, 128] and V of the kept slots, zeros behind them."""
    B, n_kv = kc.shape[:2]
    n = keep.shape[1]
    slots = -(-n // PAGE) * PAGE
    k, v = (np.zeros((B, n_kv, slots, 128), dtype=np.int8) for _ in range(2))
    for b in range(B):
        live = keep[b][keep[b] >= 0]
        k[b, :, :len(live)] = kc[b][:, live]
        v[b, :, :len(live)] = vc[b].transpose(0, 2, 1)[:, live]
    return k, v


# B, n_kv, S, budget, kept share, layers
COMPACT = {
    "one_slot": (1, 1, 1, 1, 1.0, 1),
    "few": (2, 2, 100, 7, 0.05, 2),
    "odd": (3, 2, 500, 150, 0.25, 2),
    "dense": (2, 8, 700, 640, 0.9, 1),
    "sparse_pages": (1, 2, 6000, 140, 0.02, 1),
    "whole_pages": (2, 1, 512, 256, 0.5, 3),
    "many_layers": (1, 1, 300, 130, 0.4, 35),
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", list(COMPACT))
def test_compact(name, in_place):
    """Kept slots move to fresh pages, or to the row's own first pages; every
    other page keeps its bytes."""
    B, n_kv, S, budget, share, layers = COMPACT[name]
    print(f"[compact {name} in_place={in_place}]", flush=True)
    rng = np.random.default_rng(len(name))
    keep = np.full((B, budget), -1, dtype=np.int32)
    for b in range(B):
        live = np.flatnonzero(rng.random(S) < share)[:budget]
        keep[b, :len(live)] = live
    if B > 1:
        keep[-1] = -1                                   # a row that keeps nothing
    wb = -(-budget // PAGE)
    kps, vps, want = [], [], []
    for i in range(layers):
        kc = rng.integers(-128, 128, (B, n_kv, S, 128), dtype=np.int8)
        vc = rng.integers(-128, 128, (B, n_kv, 128, S), dtype=np.int8)
        kp, vp, table, w = paged(kc, vc, seed=7)
        extra = torch.full((B * wb,) + kp.shape[1:], 77, dtype=torch.int8, device="cuda")
        kps.append(torch.cat([kp, extra]))
        vps.append(torch.cat([vp, extra]))
        want.append(_compacted(kc, vc, keep))
    fresh = torch.arange(B * w, B * (w + wb), dtype=torch.int32, device="cuda").view(B, wb)
    dst = table[:, :wb].contiguous() if in_place else fresh.flip(0).contiguous()
    before = [(k.clone(), v.clone()) for k, v in zip(kps, vps)]
    _ops().kv_compact(kps, vps, table, dst, torch.from_numpy(keep).cuda())
    others = torch.ones(kps[0].shape[0], dtype=torch.bool, device="cuda")
    others[dst.reshape(-1).long()] = False
    for (k, v), kp, vp, (k0, v0) in zip(want, kps, vps, before):
        got_k, got_v = unpaged(kp, vp, dst, wb * PAGE)
        _eq(got_k, k)
        _eq(got_v, v)
        assert torch.equal(kp[others], k0[others]) and torch.equal(vp[others], v0[others])


@pytest.mark.parametrize("n_kv, layers, S, budget", [(2, 1, 2000, 900), (8, 2, 4300, 3000)])
def test_compact_mixed_rows(n_kv, layers, S, budget):
    """Rows of one call whose pages are their own, their own behind a new one,
    new, and their own but for the first."""
    print(f"[compact mixed {n_kv} {layers} {S} {budget}]", flush=True)
    B, rng, wb = 4, np.random.default_rng(budget), -(-budget // PAGE)
    keep = np.stack([np.sort(rng.choice(S, budget, replace=False)) for _ in range(B)])
    keep[3, budget // 2:] = -1
    keep = keep.astype(np.int32)
    kps, vps, want = [], [], []
    for i in range(layers):
        kc = rng.integers(-128, 128, (B, n_kv, S, 128), dtype=np.int8)
        vc = rng.integers(-128, 128, (B, n_kv, 128, S), dtype=np.int8)
        kp, vp, table, w = paged(kc, vc, seed=3)
        extra = torch.full((B * wb,) + kp.shape[1:], 77, dtype=torch.int8, device="cuda")
        kps.append(torch.cat([kp, extra]))
        vps.append(torch.cat([vp, extra]))
        want.append(_compacted(kc, vc, keep))
    dst = torch.arange(B * w, B * (w + wb), dtype=torch.int32, device="cuda").view(B, wb)
    dst[0] = table[0, :wb]
    dst[1, 1:] = table[1, :wb - 1]
    dst[3, 1:] = table[3, 1:wb]
    _ops().kv_compact(kps, vps, table, dst, torch.from_numpy(keep).cuda())
    for (k, v), kp, vp in zip(want, kps, vps):
        got_k, got_v = unpaged(kp, vp, dst, wb * PAGE)
        _eq(got_k, k)
        _eq(got_v, v)


def test_compact_skips_unmapped_pages():
    """dst -1: nothing is written; a kept slot whose page is not mapped
    becomes 0."""
    print("[compact unmapped]", flush=True)
    c = lc.make(1, 1, 1, 400, seed=2)
    kp, vp, table, w = paged(c["kc"], c["vc"], seed=1)
    keep = np.arange(0, 400, 2, dtype=np.int32)[None]
    table[0, 1] = -1
    kp, vp = (torch.cat([x, torch.full_like(x[:2], 9)]) for x in (kp, vp))
    dst = torch.tensor([[w, -1]], dtype=torch.int32, device="cuda")
    kc, vc = c["kc"].copy(), c["vc"].copy()
    kc[:, :, 128:256] = 0
    vc[:, :, :, 128:256] = 0
    k, v = _compacted(kc, vc, keep)
    _ops().kv_compact([kp], [vp], table, dst, torch.from_numpy(keep).cuda())
    got_k, got_v = unpaged(kp, vp, dst[:, :1], PAGE)
    _eq(got_k, k[:, :, :PAGE])
    _eq(got_v, v[:, :, :PAGE])
    assert bool((kp[w + 1] == 9).all()) and bool((vp[w + 1] == 9).all())


# ------------------------------------------------------------- shared prefix

# B, n_q, n_kv, shared, suffix slots, extras
SHARED = {
    "one_row": (1, 2, 1, 128, 1, {}),
    "no_prefix": (3, 4, 2, 0, 200, dict(p_valid=0.8)),
    "no_suffix": (3, 4, 2, 256, 0, {}),
    "nothing": (2, 4, 2, 0, 0, {}),
    "few": (4, 32, 8, 512, 40, {}),
    "group_1": (20, 8, 8, 384, 77, dict(p_valid=0.9)),
    "group_8": (3, 8, 1, 256, 300, dict(p_valid=0.9)),
    "odd_rows": (9, 4, 2, 640, 65, dict(p_valid=0.9)),
    "two_blocks": (70, 4, 2, 1280, 10, {}),
    "long": (5, 4, 2, 2048, 130, dict(p_valid=0.95)),
    # (from here to flat_joint: prefixes read once for the batch)
    "one_group": (8, 2, 1, 3584, 40, dict(p_valid=0.9)),
    "two_groups": (13, 4, 2, 2048, 70, dict(p_valid=0.9)),
    "one_group_8": (2, 16, 2, 24576, 200, dict(p_valid=0.9)),
    "four_groups_1": (50, 2, 2, 1792, 1, dict(p_valid=0.9)),
    "no_suffix_joint": (40, 4, 2, 2176, 0, dict(p_valid=0.9)),
    "long_suffix": (18, 4, 2, 4864, 1000, dict(p_valid=0.9)),
    "many_chunks": (5, 8, 1, 19968, 3, dict(p_valid=0.9)),
    "dead_joint": (40, 4, 2, 2176, 20, dict(gaps=((0, 0, 2196), (39, 0, 2176), (1, 2170, 2196)))),
    "wide_tpos_joint": (33, 4, 2, 2560, 40, dict(tpos=(0, 62), p_valid=0.8)),
    "mixed_tpos_joint": (33, 4, 2, 2560, 40, dict(tpos=(30, 48), p_valid=0.8)),
    "extreme_joint": (33, 2, 2, 2560, 70, dict(extreme=(0,), tpos=(28, 40))),
    "flat_joint": (5, 4, 2, 6144, 20, dict(flat_heads=(0, 1), tpos=(38, 39))),
    "dead_prefix": (3, 4, 2, 256, 50, dict(gaps=((1, 0, 256),))),
    "dead_row": (3, 4, 2, 256, 50, dict(dead_rows=(1,))),
    "wide_tpos": (3, 4, 2, 256, 100, dict(tpos=(0, 62), p_valid=0.8)),
    "flat": (2, 2, 1, 2560, 20, dict(flat_heads=(0, 1), tpos=(38, 39))),
    "extreme": (2, 2, 2, 256, 70, dict(extreme=(0,), tpos=(28, 40))),
}


def _shared_case(B, n_q, n_kv, shared, suffix, seed, extra):
    """longcases.make with the rows' first `shared` slots the same in all,
    and a table whose first pages are row 0's."""
    c = lc.make(B, n_q, n_kv, max(1, shared + suffix), seed, **extra)
    c["kc"][:, :, :shared] = c["kc"][:1, :, :shared]
    c["vc"][:, :, :, :shared] = c["vc"][:1, :, :, :shared]
    args = list(_dev(c, seed))
    args[4][:, :shared // PAGE] = args[4][:1, :shared // PAGE].clone()
    return c, args


@pytest.mark.parametrize("name", list(SHARED))
def test_shared_decode(name):
    B, n_q, n_kv, shared, suffix, extra = SHARED[name]
    print(f"[shared decode {name}]", flush=True)
    S = shared + suffix
    c, args = _shared_case(B, n_q, n_kv, shared, suffix, len(name), extra)
    rows = range(B) if B < 10 else (0, 1, B - 1)
    sub = {k: (v[list(rows)] if isinstance(v, np.ndarray) else v) for k, v in c.items()}
    want, _ = lc.attend(sub, S=S)
    out = _ops().attn_decode_shared(*args, S, shared)
    _eq(out[list(rows)], want)
    if S:
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        assert torch.equal(out, _ops().attn_decode(*args, S, err))
    from idempotent_llm_amd._lib import attn_shared_work
    names = list(SHARED)
    joint = names.index("one_group") <= names.index(name) <= names.index("flat_joint")
    assert attn_shared_work(B, S, n_q, n_kv, shared)[1] == (joint or name == "two_blocks")


def test_shared_decode_takes_row_0s_pages():
    """The other rows' entries for the prefix are not read."""
    print("[shared decode row 0]", flush=True)
    c, args = _shared_case(4, 4, 2, 256, 30, 5, {})
    want = _ops().attn_decode_shared(*args, 286, 256)
    args[4][1:, :2] = -1
    assert torch.equal(_ops().attn_decode_shared(*args, 286, 256), want)


# ------------------------------------------------- the operators as they are used

# every attention form once: (operator, arguments behind the cache)
def _forms(S, T, past, acc):
    return {"window_decode": lambda a, c: _ops().attn_window_decode(*a, S, 100, 4),
            "window_decode_split": lambda a, c: _ops().attn_window_decode(*a, S, S, 4),
            "acc_decode": lambda a, c: _ops().attn_decode_acc(*a, S, acc),
            "shared_decode": lambda a, c: _ops().attn_decode_shared(*a, S, (S - 1) // PAGE * PAGE),
            "shared_decode_rows": lambda a, c: _ops().attn_decode_shared(*a, S, 128),
            "window_prefill": lambda a, c: _ops().attn_window_prefill(*c, past, 100, 4),
            "acc_prefill": lambda a, c: _ops().attn_prefill_acc(*c, past, acc)}


def _both(B, n_q, n_kv, S, T, seed):
    """A decode and a chunk's operands over one cache of S slots."""
    c = lc.make(B, n_q, n_kv, S, seed, T=T, p_valid=0.9)
    chunk = _dev(c, seed)
    one = (chunk[0][:, :, -1].contiguous(), chunk[1][:, :, -1].contiguous()) + chunk[2:]
    return one, chunk


def test_captured_calls_replay():
    """All forms in one graph, with selection and compaction behind them: each
    replay, with other queries and eager work in between, gives the eager
    results."""
    print("[captured calls]", flush=True)
    B, n_q, n_kv, S, T = 40, 4, 2, 2400, 70
    one, chunk = _both(B, n_q, n_kv, S, T, 11)
    acc = torch.zeros(B, n_kv, S, dtype=I64, device="cuda")
    wb = 3
    fresh = torch.arange(one[2].shape[0], one[2].shape[0] + B * wb, dtype=torch.int32,
                         device="cuda").view(B, wb)
    one, chunk = (list(a) for a in (one, chunk))
    for a in (one, chunk):
        for i in (2, 3):
            a[i] = torch.cat([a[i], torch.zeros(B * wb, *a[i].shape[1:], dtype=torch.int8,
                                                device="cuda")])
    chunk[2], chunk[3] = one[2], one[3]
    forms = _forms(S, T, S - T, acc)

    def run():
        out = [f(one, chunk) for f in forms.values()]
        keep, kept = _ops().kv_select(acc, one[5], S, 300, 30, 4)
        _ops().kv_compact([one[2]], [one[3]], one[4], fresh, keep)
        cut = (keep >= 0)
        left = torch.zeros(B, wb * PAGE, dtype=torch.bool, device="cuda")
        left[:, :300] = cut
        out.append(_ops().attn_window_decode(one[0], one[1], one[2], one[3], fresh, left, 300,
                                             128, 4))
        return out + [keep, kept]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for k in range(4):
        acc.fill_(k)
        for a in (one, chunk):
            a[0].copy_(torch.randint(-128, 128, a[0].shape, dtype=torch.int8, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        got_k, acc_k = [x.clone() for x in got], acc.clone()
        acc.fill_(k)
        want = run()
        for name, x, y in zip(list(forms) + ["cut", "keep", "kept"], got_k, want):
            assert torch.equal(x, y), (k, name)
        assert torch.equal(acc_k, acc)


def test_other_streams_and_two_at_once():
    """The operators run on torch's current stream: two streams with their own
    operands, interleaved, give what each gives alone."""
    print("[streams]", flush=True)
    cases = []
    for seed in (3, 4):
        one, chunk = _both(36, 4, 2, 2500, 40, seed)
        acc = torch.zeros(36, 2, 2500, dtype=I64, device="cuda")
        cases.append((one, chunk, acc, _forms(2500, 40, 2460, acc)))
    alone = [[f(one, chunk) for f in forms.values()] for one, chunk, _, forms in cases]
    accs = [acc.clone() for _, _, acc, _ in cases]
    for _, _, acc, _ in cases:
        acc.zero_()
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for name in cases[0][3]:
        for i, (one, chunk, _, forms) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(forms[name](one, chunk))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for x, y in zip(got[i], alone[i]))
        assert torch.equal(cases[i][2], accs[i])


def test_strided_queries_and_masks():
    """Queries and constants in another order, and a mask that is a slice at
    an odd address with rows further apart than the slots."""
    print("[strides]", flush=True)
    S, T = 2560, 50
    one, chunk = _both(35, 4, 2, S, T, 21)
    B, w = one[4].shape
    acc = torch.zeros(B, 2, S, dtype=I64, device="cuda")
    forms = _forms(S, T, S - T, acc)
    wide = torch.ones(B, w * PAGE + 37, dtype=torch.bool, device="cuda")
    wide[:, 5:5 + S] = one[5][:, :S]
    mask = wide[:, 5:5 + S]

    def other(a):
        q = a[0].transpose(1, 0).contiguous().transpose(1, 0)
        t = a[1].transpose(1, 0).contiguous().transpose(1, 0)
        assert not q.is_contiguous() and not t.is_contiguous()
        return (q, t) + tuple(a[2:5]) + (mask,)

    for name, f in forms.items():
        acc.zero_()
        want, add = f(one, chunk), acc.clone()
        acc.zero_()
        got = f(other(one), other(chunk))
        assert torch.equal(got, want) and torch.equal(acc, add), name
    acc.random_(0, 1000)
    a = _ops().kv_select(acc, one[5][:, :S].contiguous(), S, 200, 20, 4)
    b = _ops().kv_select(acc, mask, S, 200, 20, 4)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_broadcast_masks():
    """One mask for all rows (stride 0), and one row whose stride is anything."""
    print("[broadcast masks]", flush=True)
    S, T = 300, 40
    one, chunk = _both(34, 4, 2, S, T, 22)
    acc = torch.zeros(34, 2, S, dtype=I64, device="cuda")
    row = one[5][:1, :S].contiguous()
    for name, f in _forms(S, T, S - T, acc).items():
        want = f(one[:5] + (row.repeat(34, 1),), chunk[:5] + (row.repeat(34, 1),))
        got = f(one[:5] + (row.expand(34, S),), chunk[:5] + (row.expand(34, S),))
        assert torch.equal(got, want), name
    odd = torch.as_strided(row, (1, S), (1, 1))
    first = lambda a: tuple(x[:1] if i in (0, 1, 4) else x for i, x in enumerate(a[:5]))
    a = _ops().attn_window_decode(*first(one), row, S, 100, 4)
    assert torch.equal(_ops().attn_window_decode(*first(one), odd, S, 100, 4), a)
    a, b = (_ops().kv_select(acc, m, S, 90, 9, 4) for m in (row.repeat(34, 1), row.expand(34, S)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_empty_calls():
    """No rows, and a chunk of no queries."""
    print("[empty calls]", flush=True)
    one, chunk = _both(2, 4, 2, 200, 5, 23)
    none = lambda a: tuple(x[:0] if i in (0, 1, 4, 5) else x for i, x in enumerate(a))
    acc = torch.zeros(2, 2, 200, dtype=I64, device="cuda")
    assert _ops().attn_window_decode(*none(one), 200, 9, 4).shape == (0, 512)
    assert _ops().attn_decode_acc(*none(one), 200, acc[:0]).shape == (0, 512)
    assert _ops().attn_decode_shared(*none(one), 200, 128).shape == (0, 512)
    assert _ops().attn_window_prefill(*none(chunk), 195, 9, 4).shape == (0, 5, 512)
    assert _ops().attn_prefill_acc(*none(chunk), 195, acc[:0]).shape == (0, 5, 512)
    short = (chunk[0][:, :, :0], chunk[1][:, :, :0]) + chunk[2:]
    assert _ops().attn_window_prefill(*short, 195, 9, 4).shape == (2, 0, 512)
    assert _ops().attn_prefill_acc(*short, 195, acc).shape == (2, 0, 512)
    keep, kept = _ops().kv_select(acc[:0], one[5][:0], 200, 50, 5, 4)
    assert keep.shape == (0, 50) and kept.shape == (0, 2, 50)
    before = one[2].clone()
    _ops().kv_compact([one[2]], [one[3]], one[4][:0], one[4][:0], keep)
    assert not acc.any() and torch.equal(one[2], before)


def test_compact_ignores_pages_that_are_not_the_pools():
    """Ids past the pools, in dst or the table, count as not mapped."""
    print("[compact foreign pages]", flush=True)
    c = lc.make(1, 1, 1, 256, seed=6)
    kp, vp, table, w = paged(c["kc"], c["vc"], seed=1)
    keep = torch.arange(0, 256, 2, dtype=torch.int32, device="cuda")[None]
    before = kp.clone(), vp.clone()
    _ops().kv_compact([kp], [vp], table, torch.tensor([[w]], dtype=torch.int32, device="cuda"), keep)
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])
    kp, vp = (torch.cat([x, torch.full_like(x[:1], 9)]) for x in (kp, vp))
    table[0, 1] = 1 << 20
    _ops().kv_compact([kp], [vp], table, torch.tensor([[w]], dtype=torch.int32, device="cuda"), keep)
    _eq(kp[w, 0, :64], c["kc"][0, 0, 0:128:2])
    assert not kp[w, 0, 64:].any() and not vp[w, 0, :, 64:].any()


def test_pages_past_4_gib():
    """Pages whose bytes lie past 2^32 of their pool."""
    print("[far pages]", flush=True)
    one, chunk = _both(33, 16, 8, 2640, 20, 31)
    n = one[2].shape[0]
    far = (1 << 32) // (8 * PAGE * 128) + 100
    acc = torch.zeros(33, 8, 2640, dtype=I64, device="cuda")
    forms = _forms(2640, 20, 2620, acc)
    want = [f(one, chunk) for f in forms.values()]
    add = acc.clone()
    acc.zero_()
    keep = torch.arange(0, 600, 3, dtype=torch.int32, device="cuda").expand(33, 200).contiguous()
    kp, vp = (torch.empty(far + n + 66, 8, PAGE, 128, dtype=torch.int8, device="cuda")
              for _ in range(2))
    kp[far:far + n], vp[far:far + n] = one[2], one[3]
    table = one[4] + far
    move = lambda a: a[:2] + (kp, vp, table, a[5])
    got = [f(move(one), move(chunk)) for f in forms.values()]
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(acc, add)
    dst = torch.arange(far + n, far + n + 66, dtype=torch.int32, device="cuda").view(33, 2)
    _ops().kv_compact([kp], [vp], table, dst, keep)
    k, v = unpaged(kp, vp, dst, 200)
    k0, v0 = unpaged(one[2], one[3], one[4], 600)
    assert torch.equal(k, k0[:, :, ::3]) and torch.equal(v, v0[:, :, ::3])


def test_longest_row():
    """131071 slots, the most a row may have."""
    print("[longest row]", flush=True)
    S = 131071
    c = lc.make(1, 2, 1, S, seed=41, p_valid=0.9)
    args = _dev(c, 1)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = _ops().attn_decode(*args, S, err)
    live = int(c["valid"].sum())
    assert torch.equal(_ops().attn_window_decode(*args, S, live, 0), want)
    acc = torch.zeros(1, 1, S, dtype=I64, device="cuda")
    assert torch.equal(_ops().attn_decode_acc(*args, S, acc), want)
    out, add = lc.attend(c, S=S)
    _eq(want, out)
    _eq(acc, add)
    want, _ = lc.attend(c, S=S, window=5000, sinks=100)
    _eq(_ops().attn_window_decode(*args, S, 5000, 100), want)
    keep, kept = _ops().kv_select(acc, args[5], S, 9000, 300, 50)
    want_keep, want_kept = lc.select(add, c["valid"], 9000, 300, 50)
    _eq(keep, want_keep)
    _eq(kept, want_kept)
    dst = torch.arange(args[2].shape[0], args[2].shape[0] + 71, dtype=torch.int32,
                       device="cuda")[None]
    kp, vp = (torch.cat([x, torch.zeros_like(x[:71])]) for x in args[2:4])
    _ops().kv_compact([kp], [vp], args[4], dst, keep)
    k, v = unpaged(kp, vp, dst, 9000)
    _eq(k[0, 0], c["kc"][0, 0][want_keep[0]])
    _eq(v[0, 0], c["vc"][0, 0].T[want_keep[0]])
    two = [x.expand(2, *x.shape[1:]).contiguous() if i in (0, 1, 4, 5) else x
           for i, x in enumerate(args)]
    shared = S // PAGE * PAGE
    both = _ops().attn_decode_shared(*two, S, shared)
    _eq(both[0], out[0])
    _eq(both[1], out[0])
    # a chunk at the end of such a row
    q = torch.randint(-128, 128, (1, 2, 3, 128), dtype=torch.int8, device="cuda")
    t = torch.randint(1000, 9000, (1, 2, 3), dtype=I64, device="cuda")
    want = _ops().attn_prefill(q, t, *args[2:], S - 3)
    assert torch.equal(_ops().attn_window_prefill(q, t, *args[2:], S - 3, live, 0), want)
    acc.zero_()
    assert torch.equal(_ops().attn_prefill_acc(q, t, *args[2:], S - 3, acc), want)


@pytest.mark.parametrize("count", [0, 100, 2176, 2300, 2560])
def test_device_slot_counts(count):
    """The entry points bound the scanned slots by a device word (a captured
    step's): the same as that many slots; one above the launch's bound sets
    bit 4 of the error word and scans the bound."""
    print(f"[device count {count}]", flush=True)
    from idempotent_llm_amd._lib import attn_acc_work, attn_shared_work, call
    B, n_q, n_kv, S, cap = 40, 4, 2, 2400, 2560
    one, _ = _both(B, n_q, n_kv, cap, 3, 51)
    q8, tpos, kp, vp, table, valid = one
    n = min(count, S)
    word = torch.tensor([count], dtype=I64, device="cuda")
    cache = (q8, tpos, kp, vp, table, table.shape[1], valid.view(torch.uint8), valid.shape[1], B)
    work = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    assert attn_shared_work(B, S, n_q, n_kv, 2176)[1]
    for name, tail, want in (
            ("detllm_attn_window_decode", (100, 4), lambda: _ops().attn_window_decode(*one, n, 100, 4)),
            ("detllm_attn_window_decode", (10**6, 0),
             lambda: _ops().attn_window_decode(*one, n, 10**6, 0)),
            ("detllm_attn_decode_acc", "acc", lambda: _ops().attn_decode_acc(*one, n, other)),
            ("detllm_attn_decode_shared", (2176,), lambda: _ops().attn_decode_shared(*one, n, 0)),
            ("detllm_attn_decode_shared", (0,), lambda: _ops().attn_decode_shared(*one, n, 0))):
        if tail == (2176,):
            table[:, :17] = table[:1, :17].clone()
        acc, other = (torch.zeros(B, n_kv, cap, dtype=I64, device="cuda") for _ in range(2))
        args = (acc, cap) if tail == "acc" else tail
        out = torch.full((B, n_q * 128), 7, dtype=I64, device="cuda")
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        call(name, *cache, S, n_q, n_kv, word, *args, work, work.numel(), out, err)
        assert torch.equal(out, want()), (name, tail)
        assert torch.equal(acc, other)
        assert int(err) == (4 if count > S else 0), (name, tail)
