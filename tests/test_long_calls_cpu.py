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
