"""Calls of the long-cache operators and of the KV cache that keeps them, as
far as they show without a GPU."""

from types import SimpleNamespace

import pytest
import torch

from idempotent_llm_amd import torch_ops  # noqa: F401  (registers the operators)
from idempotent_llm_amd.kvcache import PAGE, KVCache

KEY = torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA)
I8, I32, I64 = torch.int8, torch.int32, torch.int64


def _call(name, *args):
    """The operator's native kernel on host tensors (checks run first)."""
    return getattr(torch.ops.detllm_rocm, name).default.redispatch(KEY, *args)


def test_compact_refuses_a_dst_whose_slots_pass_32_bits():
    pool = lambda: torch.zeros(3, 1, 128, 128, dtype=I8)
    dst = torch.full((1, (1 << 23) + 1), -1, dtype=I32)
    with pytest.raises(ValueError, match="kv_compact"):
        _call("kv_compact", [pool()], [pool()], torch.zeros(1, 2, dtype=I32), dst,
              torch.zeros(1, 9, dtype=I32))


# ------------------------------------------------------------------ KVCache

def _model():
    return SimpleNamespace(n_layers=1, n_kv=1, hd=128, device=torch.device("cpu"))


def _tracked(*reserved):
    """A tracked cache of two rows that grew to each of `reserved` slots."""
    c = KVCache().track_weights()
    for n in reserved:
        c.reserve(_model(), 2, n)
        c.valid_buf[:, c.length:n] = True
        c.length = n
    return c


@pytest.fixture
def eviction(monkeypatch):
    """The eviction's operators without a GPU: kv_select keeps each row's last
    `budget` slots; kv_compact refuses what it refuses, and `seen` gets its table."""
    seen = []

    def kv_select(acc, valid, S, budget, recent, sinks):
        keep = torch.arange(S - budget, S, dtype=I32).expand(acc.shape[0], budget).contiguous()
        return keep, acc[:, :, S - budget:S].clone()

    def kv_compact(kpools, vpools, table, dst, keep):
        if table.shape[1] > 1024 or not table.is_contiguous():
            raise ValueError("kv_compact")
        seen.append(table)

    monkeypatch.setattr(torch.ops.detllm_rocm, "kv_select", kv_select)
    monkeypatch.setattr(torch.ops.detllm_rocm, "kv_compact", kv_compact)
    return seen


def test_evict_of_a_table_past_1024_pages(eviction):
    """A cache of 70100 slots whose table doubled from 547 to 1094 pages."""
    c = _tracked(70000, 70100)
    assert c.width > 1024
    table = c.table.clone()
    c.evict(500, 10, 4)
    assert torch.equal(eviction[0], table[:, :548]) and c.length == 500
    assert (c._table_host[:, :4] >= 0).all() and (c._table_host[:, 4:] == -1).all()


def _books(c):
    return sorted(c._free), c.n_pages, c._table_host.tolist(), c.table.tolist(), c.length, c.shared


def test_a_failed_eviction_keeps_its_pages(eviction, monkeypatch):
    """Pages taken for a move that is refused are not lost, whether they were
    free ones or new, and the cache evicts once the cause is gone."""
    for free in ((), (0, 3)):
        c = _tracked(1000, 1100)
        c._free += [c.n_pages + i for i in range(len(free))]
        c.n_pages += len(free)
        c._ensure_pool(c.n_pages + 40)
        before = _books(c)
        good = torch.ops.detllm_rocm.kv_compact

        def refuse(*args):
            raise ValueError("kv_compact")

        monkeypatch.setattr(torch.ops.detllm_rocm, "kv_compact", refuse)
        for _ in range(3):
            with pytest.raises(ValueError):
                c.evict(300, 10, 4)
            assert _books(c) == before
        monkeypatch.setattr(torch.ops.detllm_rocm, "kv_compact", good)
        c.evict(300, 10, 4)
        assert c.length == 300
        used = c._table_host[c._table_host >= 0].tolist()
        assert sorted(used + c._free) == list(range(c.n_pages))


def test_a_failed_fork_keeps_its_pages(monkeypatch):
    """No memory for the pages begun: the cache stays the one row it was."""
    c = KVCache()
    c.reserve(_model(), 1, 700)
    c.length = 200                          # pages behind the one begun are handed back
    before = _books(c)

    def no_memory(need):
        raise MemoryError

    monkeypatch.setattr(c, "_ensure_pool", no_memory)
    with pytest.raises(MemoryError):
        c.fork(9)
    assert _books(c) == before
    monkeypatch.undo()
    v_pools, c.v_pools = c.v_pools, [None]              # ... or fails behind the pages taken
    with pytest.raises(TypeError):
        c.fork(3)
    assert _books(c) == before
    c.v_pools = v_pools
    c.fork(9)
    used = set(c._table_host[c._table_host >= 0].tolist())
    assert not used & set(c._free) and used | set(c._free) == set(range(c.n_pages))


def test_free_pages_stay_free_when_the_pool_cannot_grow(monkeypatch):
    c = _tracked(300)
    c._ensure_width(2, 9)
    c._free += [c.n_pages]
    c.n_pages += 1

    def no_memory(need):
        raise MemoryError

    monkeypatch.setattr(c, "_ensure_pool", no_memory)
    before = _books(c)
    with pytest.raises(MemoryError):
        c.map_slots(c.cap)
    assert _books(c) == before


def test_a_table_that_cannot_grow_keeps_its_accumulators(monkeypatch):
    """acc is as wide as the table, also where the wider table fails."""
    c = _tracked(300)

    def no_memory(x):
        raise MemoryError

    with monkeypatch.context() as m:
        m.setattr(torch, "from_numpy", no_memory)
        with pytest.raises(MemoryError):
            c._ensure_width(2, 9)
    assert c.acc.shape[2] == c.valid_buf.shape[1] == c.cap == c._table_host.shape[1] * PAGE
    c._ensure_width(2, 9)
    assert c.acc.shape[2] == c.valid_buf.shape[1] == c.cap == 9 * PAGE


def test_a_prefix_that_16_rows_read_once_17_do_too():
    """The shared form's rule at prefixes where it pays on both sides of 16
    rows, and few slots behind them hold it where more do."""
    from idempotent_llm_amd._lib import attn_shared_work
    joint = lambda B, S, P, n_q=16, n_kv=8: attn_shared_work(B, S, n_q, n_kv, P)[1]
    for n_q, n_kv in ((16, 8), (8, 8), (32, 8), (64, 8), (8, 1)):
        for P in (2560, 4096, 8192, 130944):
            rows = [joint(B, P + 40, P, n_q, n_kv) for B in range(1, 80)]
            assert rows == sorted(rows) and rows[16], (n_q, n_kv, P)
    for B in (2, 8, 16, 17, 24, 64, 300):
        for P in (128, 1024, 1536, 2048, 4096, 24576):
            own = [joint(B, P + n, P) for n in range(0, P + 1, 8)]
            assert own == sorted(own, reverse=True), (B, P)


# ------------------------------------------------------------------ scratch

def _cdiv(a, b):
    return -(-a // b)


def _split_bytes(B, S, n_q, chunk):
    """Scores [B][n_q][ns * chunk] and chunk maxima [B][n_q][ns], int32."""
    ns = _cdiv(S, chunk)
    return B * n_q * ns * chunk * 4 + _cdiv(B * n_q * ns * 4, 16) * 16


HEADS = ((8, 8), (16, 8), (32, 8), (64, 8), (8, 1), (4, 2))
LDS = 48 * 1024     # of scores in the one-block kernels


@pytest.mark.parametrize("n_q,n_kv", HEADS)
def test_scratch_holds_what_the_forms_write(n_q, n_kv):
    """Each planner's bytes are those of one of the forms that the size may
    take: none where the scores fit a block's LDS, else the scores (and what
    the cut form adds)."""
    import ctypes
    from idempotent_llm_amd._lib import attn_acc_work, attn_split_plan, load
    G = n_q // n_kv
    out = ctypes.c_int64(0)
    for B in (1, 3, 16, 64, 300):
        for S in (1, 127, 700, 960, 1700, 5000, 12289, 40000, 131071):
            spad = _cdiv(S, 16) * 16
            chunk, ns = attn_split_plan(B, S, n_q, n_kv)
            forms = [_split_bytes(B, S, n_q, chunk)] if ns > 1 else []
            if G * spad * 4 <= LDS:
                forms.append(0)
            assert attn_acc_work(B, S, n_q, n_kv) in forms, (B, S)
            for window, sinks in ((1, 0), (200, 4), (3000, 64), (2**31 - 1, 2**31 - 1)):
                assert load().detllm_attn_window_decode_work(B, S, n_q, n_kv, window, sinks,
                                                             ctypes.byref(out)) == 0
                chunk, ns = attn_split_plan(B, min(S, window + sinks + 6 * PAGE), n_q, n_kv)
                forms = [0 if G * spad * 4 <= LDS else B * n_q * spad * 4]
                if ns > 1:      # + the rows' ranges (16 bytes) and page lists
                    forms.append(_split_bytes(B, S, n_q, chunk) + B * (16 + 2 * _cdiv(S, PAGE)))
                assert out.value in forms, (B, S, window)


@pytest.mark.parametrize("n_q,n_kv", HEADS)
def test_scratch_of_a_prefix_read_once(n_q, n_kv):
    """For each query maxima (4 bytes) and denominators (8) of every part, and
    the prefix's partial contexts (512): the parts of the launches' plan."""
    from idempotent_llm_amd._lib import attn_shared_work
    G, seen = n_q // n_kv, 0
    for B in (2, 5, 9, 17, 40, 64, 200):
        for P in (1536, 2048, 4096, 8192, 24576, 130944):
            n, joint = attn_shared_work(B, P + 40, n_q, n_kv, P)
            if not joint:
                continue
            seen += 1
            M = B * G
            ng = 1 if M <= 16 else 2 if M <= 32 else 4
            blocks = _cdiv(M, 16 * ng) * n_kv
            chunk = _cdiv(_cdiv(P // 64, max(512 // blocks, 1)), 4) * 4 * 64
            parts = _cdiv(P, chunk) + 1
            pages = min(max(_cdiv(P // PAGE, max(256 // blocks, 1)), 1), 8)
            parts2 = _cdiv(P // PAGE, pages) * (4 // ng)
            rows = n_kv * M
            assert n >= _cdiv(rows * parts * 12, 64) * 64 + rows * parts2 * 512, (B, P)
    assert seen > 10
