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
