"""Packed steps: requests of any lengths in one batch without padding (no
counterpart in the reference, whose batches are right-padded rows that all stand
at one slot).

* ``PackedCache`` is a paged int8 KV cache (kvcache.py's pages) whose rows have
  lengths of their own. The page table and the free list live on the device;
  ``packed_plan`` maps and gives back pages there, so a step needs nothing from
  the device.
* ``IntQwen3.forward_packed`` runs one step of it: each row's new tokens (none,
  one, a chunk of its prompt) follow each other in ``ids``, and each row's last
  one gets logits.
* ``generate_packed`` is a scheduler on top: prompts are admitted as rows and
  pages allow, fed in chunks beside the running replies, and leave when done.

Every integer of a request is what the request gets alone (``generate``): a
token's row of every product, its attention over its own slots and its positions
do not depend on what else is in the step.
"""

from __future__ import annotations

import torch

from . import torch_ops  # noqa: F401  (registers the operators)
from .kvcache import PAGE

I32 = torch.int32
MAX_SLOTS = 131071      # of a row (int32 accumulators of P.V)
MAX_ROWS = 2048         # of a batch (packed_plan)


class OutOfPages(RuntimeError):
    """A step that needs more pages than the pools have left. Raised before
    anything is launched: the cache is as it was."""


class PackedCache:
    """Pools of ``pages`` pages per layer for ``rows`` rows of up to ``slots``
    tokens. ``past`` [rows] int32 (device) and ``lens`` (host) count each row's
    tokens."""

    def __init__(self, model, rows: int, slots: int, pages: int | None = None):
        width = -(-int(slots) // PAGE)
        if not 1 <= rows <= MAX_ROWS or not 1 <= slots <= MAX_SLOTS:
            raise ValueError(f"PackedCache: {rows} rows of {slots} slots (at most {MAX_ROWS} of "
                             f"{MAX_SLOTS})")
        pages = rows * width if pages is None else int(pages)
        if pages < 1:
            raise ValueError(f"PackedCache: {pages} pages")
        dev = model.device
        self.rows, self.slots, self.pages = rows, int(slots), pages
        shape = (pages, model.n_kv, PAGE, PAGE)
        self.k_pools = [torch.empty(shape, dtype=torch.int8, device=dev)
                        for _ in range(model.n_layers)]
        self.v_pools = [torch.empty(shape, dtype=torch.int8, device=dev)
                        for _ in range(model.n_layers)]
        self.table = torch.full((rows, width), -1, dtype=I32, device=dev)
        self.free = torch.arange(pages - 1, -1, -1, dtype=I32, device=dev)
        self.n_free = torch.full((1,), pages, dtype=I32, device=dev)
        self.past = torch.zeros(rows, dtype=I32, device=dev)
        self.lens = [0] * rows

    def pages_left(self) -> int:
        """Pages that no row's tokens need (a released row's come back with
        the next step, before that step takes any)."""
        return self.pages - sum(-(-n // PAGE) for n in self.lens)

    def release(self, row: int, keep: int = 0) -> None:
        """Row ``row`` keeps its first ``keep`` tokens (0: the row is free for
        another request); the pages behind them come back with the next step."""
        if not 0 <= row < self.rows or not 0 <= keep <= self.lens[row]:
            raise ValueError(f"release: row {row} down to {keep} tokens")
        self.past[row] = keep
        self.lens[row] = keep

    def check_model(self, model) -> None:
        """ValueError for a model whose layers or heads are not the cache's."""
        have = (len(self.k_pools), self.k_pools[0].shape[1], self.k_pools[0].device)
        want = (model.n_layers, model.n_kv, self.k_pools[0].new_empty(0).to(model.device).device)
        if have != want:
            raise ValueError(f"packed step: a cache of {have[0]} layers of {have[1]} kv heads on "
                             f"{have[2]}, a model of {want[0]} of {want[1]} on {want[2]}")

    def check(self, new) -> None:
        """ValueError for counts that do not fit the rows, OutOfPages."""
        if len(new) != self.rows or any(n < 0 for n in new):
            raise ValueError(f"packed step: {self.rows} counts of new tokens, none negative")
        for b, (n, have) in enumerate(zip(new, self.lens)):
            if have + n > self.slots:
                raise ValueError(f"packed step: row {b} of {have} tokens and {n} new ones has "
                                 f"{self.slots} slots")
        need = sum(-(-(n + have) // PAGE) for n, have in zip(new, self.lens))
        if need > self.pages:
            raise OutOfPages(f"packed step: {need} pages of {self.pages}")


def generate_packed(model, prompts, max_new, rows: int = 32, step_tokens: int = 512,
                    pages: int | None = None, stop_at_eos: bool = False, adapters=None,
                    adapter_of=None):
    """Greedy replies to ``prompts`` (1-D int64 tensors) of at most ``max_new``
    tokens each (a number, or one per prompt), at most ``rows`` at a time and
    ``step_tokens`` token rows a step; adapter_of: per prompt, its adapter in
    ``adapters`` (None or -1: none). Returns a list of token tensors."""
    n = len(prompts)
    prompts = [p.reshape(-1).to("cpu", torch.int64) for p in prompts]
    most = [int(max_new)] * n if not hasattr(max_new, "__len__") else [int(m) for m in max_new]
    if adapter_of is not None and len(adapter_of) != n:
        raise ValueError(f"generate_packed: {len(adapter_of)} adapters of {n} prompts")
    which = [-1 if adapter_of is None or adapter_of[i] is None else int(adapter_of[i])
             for i in range(n)]
    if len(most) != n or any(m < 0 for m in most) or any(p.numel() < 1 for p in prompts):
        raise ValueError("generate_packed: prompts of at least one token, as many reply lengths")
    if step_tokens < 1 or rows < 1:
        raise ValueError(f"generate_packed: {rows} rows, {step_tokens} token rows a step")
    out = [[] for _ in range(n)]
    todo = [i for i in range(n) if most[i] > 0]
    if not todo:
        return [torch.empty(0, dtype=torch.int64) for _ in range(n)]
    # (the last token of a reply is not fed back)
    total = [prompts[i].numel() + most[i] - 1 for i in range(n)]
    for i in todo:
        if total[i] > model.max_pos:
            raise IndexError(f"generate_packed: request {i} reaches position {total[i] - 1}, outside "
                             f"the RoPE tables (size {model.max_pos})")
    # every request before the first step: one that the model refuses would end the
    # run with the replies of the others (a stand-in for a model may take any)
    check = getattr(model, "check_requests", None)
    if check is not None:
        check(prompts, adapters, which)
    rows = min(rows, len(todo))
    cache = PackedCache(model, rows, max(total[i] for i in todo), pages)
    for i in todo:
        if -(-total[i] // PAGE) > cache.pages:
            raise OutOfPages(f"generate_packed: request {i} alone needs more than {cache.pages} pages")
    at = [None] * rows          # the request of each row
    fed = [0] * n               # prompt tokens fed
    eos = model.cfg.get("eos_token_id") if stop_at_eos else None
    while todo or any(r is not None for r in at):
        # a request is admitted with the pages of its whole reply set aside
        kept = sum(-(-total[r] // PAGE) for r in at if r is not None)
        for b in range(rows):
            if at[b] is None and todo and kept + -(-total[todo[0]] // PAGE) <= cache.pages:
                at[b] = todo.pop(0)
                kept += -(-total[at[b]] // PAGE)
        new, parts, left = [0] * rows, [None] * rows, step_tokens
        for b, r in enumerate(at):      # running replies first, then the prompts' chunks
            if r is not None and fed[r] == prompts[r].numel() and left > 0:
                new[b], parts[b], left = 1, torch.tensor([out[r][-1]]), left - 1
        for b, r in enumerate(at):
            if r is not None and fed[r] < prompts[r].numel() and left > 0:
                k = min(left, prompts[r].numel() - fed[r])
                new[b], parts[b], left = k, prompts[r][fed[r]:fed[r] + k], left - k
                fed[r] += k
        ids = torch.cat([p for p in parts if p is not None])
        logits = model.forward_packed(ids, new, cache, adapters,
                                      [-1 if r is None else which[r] for r in at])
        picked = model.greedy_pick(logits).tolist()
        model.raise_if_device_error()
        live = [b for b in range(rows) if new[b] > 0]
        for b, tok in zip(live, picked):
            r = at[b]
            if fed[r] < prompts[r].numel():
                continue                # a chunk inside the prompt
            out[r].append(tok)
            if len(out[r]) == most[r] or tok == eos:
                cache.release(b)
                at[b] = None
    return [torch.tensor(o, dtype=torch.int64) for o in out]
