"""Calls of the long-cache operators and of the KV cache that keeps them, as
far as they show without a GPU."""

import pytest
import torch

from idempotent_llm_amd import torch_ops  # noqa: F401  (registers the operators)

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
