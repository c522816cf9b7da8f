"""Paged int8 KV cache of the rocm runtime (the contract of the reference's
KVCache, src/detllm/model.py:67-102, with paged storage).

The reference keeps, per layer, one contiguous [B, n_kv, CAP, hd] K and V
buffer and grows them by reallocating and copying the filled prefix. Here
each layer owns a page pool and every row a page table:

* a page holds PAGE = 128 slots of all kv heads: K as [n_kv, 128 slots, 128]
  and V transposed as [n_kv, 128 channels, 128 slots] (the attention kernels
  read slot-contiguous bytes from both);
* ``table[b, j]`` (int32, device) is the page of row b's slots
  [128 j, 128 j + 128), -1 when not mapped; the same page ids serve every
  layer (each layer indexes its own pool with them);
* growing the cache maps free pages of the pool into the tables, so filled
  slots are never copied; only when a pool runs out of pages is it
  reallocated at twice the size (the pages keep their ids, and
  ``pool_generation`` tells a captured graph to capture again).

Slot semantics are the reference's: slot order is call order for every row,
``valid`` marks real tokens, ``length`` counts filled slots. Slots that are
not valid are never read as data by the kernels (their K/V bytes are
unspecified), which is why pools are not zero-filled.

For long contexts (no counterpart in the reference):

* ``track_weights()`` makes the model's attention add each slot's weight, over
  all layers, to ``acc`` [B, n_kv, slots], and ``evict(budget, recent, sinks)``
  keeps the slots that kv_select picks by it, moves them together in every
  layer and returns the other pages. Positions are the caller's, so decoding
  goes on where it was. A graphed decode hands its cache back for it
  (GraphedDecode.release);
* ``fork(rows)`` makes a one-row cache one of ``rows`` rows that share its full
  pages (``shared`` slots); decode attention reads these once for the batch
  where that pays and the cache does not track its weights.
"""

from __future__ import annotations

from contextlib import contextmanager

import numpy as np
import torch

PAGE = 128   # slots per page (csrc/common.h DI_PAGE)


class CacheRowsMismatch(RuntimeError, ValueError):
    """A batch whose row count differs from the rows the cache holds. The
    reference fails the same call in ``torch.cat([cache.valid, chunk_valid])``
    (a RuntimeError); here the check runs on the host before any kernel
    would index the page tables past their rows."""


class KVCache:
    def __init__(self):
        self.k_pools: list = []     # per layer [n_pages, n_kv, PAGE, hd] int8
        self.v_pools: list = []     # per layer [n_pages, n_kv, hd, PAGE] int8
        self.table = None           # [B, width] int32 device
        self._table_host = None     # numpy mirror of ``table``
        self.n_pages = 0            # pages handed out (ids 0 .. n_pages - 1)
        self.mapped = 0             # slots [0, mapped) are mapped on every row
        self.valid_buf = None       # [B, width * PAGE] bool
        self.length = 0
        self.static_cap = 0         # slots of a graphed decode's tables (0: eager)
        self.static_scan = 0        # slots its steps' attention is sized for
        self.len_idx = None         # [1] int64 device: slot written by a graphed step
        self.nslots = None          # [1] int64 device: slots visible to a graphed step
        self.pool_generation = 0
        self._dims = None           # (n_layers, n_kv, hd, device)
        self._free: list = []       # page ids handed back by evict
        self.tracking = False
        self.acc = None             # [B, n_kv, width * PAGE] int64 (track_weights)
        self.shared = 0             # slots whose pages all rows share (fork)

    # -- reference-compatible surface ------------------------------------------
    @property
    def width(self) -> int:
        return 0 if self.table is None else int(self.table.shape[1])

    @property
    def cap(self) -> int:
        return self.width * PAGE

    @property
    def valid(self):
        return None if self.valid_buf is None else self.valid_buf[:, :self.length]

    def seq_len(self) -> int:
        return self.length

    @property
    def k8(self) -> list:
        """Per layer K in the reference layout [B, n_kv, length, hd] (a
        gathered copy, for inspection)."""
        return [self._gather(li, "k") for li in range(len(self.k_pools))]

    @property
    def v8(self) -> list:
        """Per layer V in the reference layout [B, n_kv, length, hd]."""
        return [self._gather(li, "v") for li in range(len(self.v_pools))]

    def _gather(self, li: int, which: str, S: int | None = None) -> torch.Tensor:
        """[B, n_kv, S, hd] of layer li (S defaults to ``length``); slots of
        pages that are not mapped read as 0."""
        S = self.length if S is None else S
        w = -(-S // PAGE)
        B = self.table.shape[0]
        tb = self.table[:, :w].long()
        ids = tb.clamp(min=0)
        if which == "k":
            pages = self.k_pools[li][ids]                       # [B, w, n_kv, PAGE, hd]
            out = pages.permute(0, 2, 1, 3, 4)
        else:
            pages = self.v_pools[li][ids]                       # [B, w, n_kv, hd, PAGE]
            out = pages.permute(0, 2, 1, 4, 3)
        n_kv, hd = out.shape[1], out.shape[-1]
        out = out.reshape(B, n_kv, w * PAGE, hd)[:, :, :S]
        live = (tb >= 0).repeat_interleave(PAGE, dim=1)[:, None, :S, None]
        return torch.where(live, out, torch.zeros_like(out))

    # -- storage ------------------------------------------------------------------
    def _ensure_pool(self, need_pages: int):
        n_layers, n_kv, hd, dev = self._dims
        have = self.k_pools[0].shape[0] if self.k_pools else 0
        if need_pages <= have:
            return
        new = max(need_pages, 2 * have)
        kp = [torch.empty(new, n_kv, PAGE, hd, dtype=torch.int8, device=dev)
              for _ in range(n_layers)]
        vp = [torch.empty(new, n_kv, hd, PAGE, dtype=torch.int8, device=dev)
              for _ in range(n_layers)]
        for li in range(len(self.k_pools)):
            kp[li][:self.n_pages] = self.k_pools[li][:self.n_pages]
            vp[li][:self.n_pages] = self.v_pools[li][:self.n_pages]
        self.k_pools, self.v_pools = kp, vp
        self.pool_generation += 1

    def _ensure_width(self, B: int, width: int):
        if self.table is not None and width <= self.width:
            return
        host = np.full((B, width), -1, dtype=np.int32)
        dev = self._dims[3]
        valid = torch.zeros(B, width * PAGE, dtype=torch.bool, device=dev)
        if self.table is not None:
            host[:, :self.width] = self._table_host
            valid[:, :self.valid_buf.shape[1]] = self.valid_buf
        acc = self.acc
        if self.tracking:
            acc = torch.zeros(B, self._dims[1], width * PAGE, dtype=torch.int64, device=dev)
            if self.acc is not None:
                acc[:, :, :self.acc.shape[2]] = self.acc
        table = torch.from_numpy(host).to(dev)
        # (together: the attention takes acc's row stride from the table's width)
        self._table_host, self.table, self.valid_buf, self.acc = host, table, valid, acc

    def map_slots(self, upto: int):
        """Map pages so every row's slots [0, upto) have one. Only new pages
        are written into the tables (in place: a captured graph keeps
        reading the same table buffer)."""
        if upto <= self.mapped:
            return
        need_w = -(-upto // PAGE)
        B = self._table_host.shape[0]
        assert need_w <= self.width, "map_slots beyond the table width"
        missing = np.argwhere(self._table_host[:, :need_w] < 0)
        if len(missing):
            self._table_host[missing[:, 0], missing[:, 1]] = self._take_pages(len(missing))
            self.table.copy_(torch.from_numpy(self._table_host))
        self.mapped = need_w * PAGE

    def _take_pages(self, n: int) -> np.ndarray:
        """Ids of n pages of the pool: those handed back first, then new ones."""
        new = max(0, n - len(self._free))
        self._ensure_pool(self.n_pages + new)      # (may raise: before any page is taken)
        old = [self._free.pop() for _ in range(n - new)]
        ids = np.arange(self.n_pages, self.n_pages + new, dtype=np.int32)
        self.n_pages += new
        return np.concatenate([np.array(old, dtype=np.int32), ids])

    @contextmanager
    def _pages_as_before_if_it_raises(self):
        free, n_pages = list(self._free), self.n_pages
        try:
            yield
        except BaseException:
            self._free, self.n_pages = free, n_pages
            raise

    def check_rows(self, B: int):
        """Raise CacheRowsMismatch unless the cache is empty or holds B rows."""
        if self._table_host is not None and self._table_host.shape[0] != B:
            raise CacheRowsMismatch(
                f"a batch of {B} rows cannot use a KV cache of "
                f"{self._table_host.shape[0]} rows")

    def _init(self, model, B: int):
        self.check_rows(B)
        if self._dims is None:
            self._dims = (model.n_layers, model.n_kv, model.hd, model.device)
            self._ensure_width(B, 1)

    def plan(self, model, B: int, slots: int) -> "KVCache":
        """Size the tables and the page pools for ``slots`` slots per row up
        front (a caller that knows its longest sequence, e.g. generate with
        max_new): growth up to that length then only maps pages — nothing is
        reallocated or copied and a captured decode graph is never
        captured again."""
        self._init(model, B)
        w = max(1, -(-slots // PAGE))
        self._ensure_width(B, w)
        self._ensure_pool(B * w)
        return self

    def reserve(self, model, B: int, need: int):
        """Dynamic (prefill / eager decode) growth: table width at least
        ``need`` slots (doubling), pages mapped for slots [0, need)."""
        self._init(model, B)
        if need > self.cap:
            self._ensure_width(B, max(-(-need // PAGE), 2 * self.width))
        self.map_slots(need)

    def resize(self, cap: int):
        """Static (graphed) capacity: the table covers ``cap`` slots; pages
        are mapped as the steps reach them (graphed.py)."""
        assert cap % PAGE == 0
        B = self._table_host.shape[0]
        self._ensure_width(B, cap // PAGE)

    # -- long contexts ------------------------------------------------------------
    def _no_graph(self, what: str):
        if self.static_cap:
            raise ValueError(f"{what}: a graphed decode holds this cache's tables "
                             "(GraphedDecode.release gives them back)")

    def track_weights(self) -> "KVCache":
        """From now on the model adds each slot's attention weight (p in
        [0, 2^14], over the query heads of a kv head, the layers and the
        queries at valid slots) to ``acc``."""
        self._no_graph("track_weights")
        if not self.tracking:
            self.tracking = True
            if self.table is not None:
                self.acc = torch.zeros(self.table.shape[0], self._dims[1], self.cap,
                                       dtype=torch.int64, device=self._dims[3])
        return self

    def evict(self, budget: int, recent: int = 0, sinks: int = 0) -> "KVCache":
        """At most ``budget`` slots per row stay: the first ``sinks`` and the
        last ``recent`` valid ones and the heaviest others by ``acc``
        (kv_select), in their order, at slots 0, 1, ...; the cache is then
        ``budget`` slots long (rows that keep fewer end in slots that are not
        valid) and the pages behind them are free. A cache of at most
        ``budget`` slots stays as it is."""
        self._no_graph("evict")
        if not self.tracking:
            raise ValueError("evict: no weights (call track_weights before the prompt)")
        if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
            raise ValueError(f"evict: recent {recent} and sinks {sinks} of a budget of {budget}")
        if self.length <= budget:
            return self
        from . import torch_ops  # noqa: F401  (registers the operators)
        ops = torch.ops.detllm_rocm
        keep, kept = ops.kv_select(self.acc, self.valid_buf, self.length, budget, recent, sinks)
        # pages of the pool that no row uses take the slots where there are
        # enough (kv_compact then works on a row's pages at once: 2 x 4000 slots
        # to 1024, 8 layers, 30 us against 71); else a row's own first pages do,
        # and new ones for those that rows share
        wb = -(-budget // PAGE)
        host = self._table_host
        ids, n = np.unique(host[host >= 0], return_counts=True)
        dst = host[:, :wb].copy()
        spare = len(self._free) + self.k_pools[0].shape[0] - self.n_pages
        fresh = np.argwhere(np.isin(dst, ids[n > 1]) | (spare >= dst.size))
        with self._pages_as_before_if_it_raises():
            if len(fresh):
                dst[fresh[:, 0], fresh[:, 1]] = self._take_pages(len(fresh))
            dst_dev = torch.from_numpy(dst).to(self._dims[3])
            there = keep >= 0
            # (the columns that hold the slots: a table grown by doubling may have
            # more than kv_compact's 1024)
            table = self.table[:, :-(-self.length // PAGE)].contiguous()
            ops.kv_compact(self.k_pools, self.v_pools, table, dst_dev, keep)
        self._free += [int(i) for i in np.setdiff1d(ids, dst)][::-1]
        host[:] = -1
        host[:, :wb] = dst
        self.table.copy_(torch.from_numpy(host))
        self.valid_buf.zero_()
        self.valid_buf[:, :budget] = there
        self.acc.zero_()
        self.acc[:, :, :budget] = kept
        self.length, self.mapped, self.shared = budget, wb * PAGE, 0
        return self

    def fork(self, rows: int) -> "KVCache":
        """This one-row cache with ``rows`` rows that begin alike: its full
        pages are shared (``shared`` slots), the page begun is copied."""
        self._no_graph("fork")
        if self.table is None or self.table.shape[0] != 1 or rows < 1:
            raise ValueError("fork: a cache of one row, into one row or more")
        full, part = self.length // PAGE, self.length % PAGE
        row = self._table_host[0]
        begun = int(row[full]) if part else -1
        host = np.full((rows, self.width), -1, dtype=np.int32)
        host[:, :full] = row[:full]
        with self._pages_as_before_if_it_raises():
            self._free += [int(i) for i in row[full + (1 if part else 0):] if i >= 0]
            if part:
                host[0, full] = begun
                host[1:, full] = self._take_pages(rows - 1)
                to = torch.from_numpy(host[1:, full].copy()).to(self._dims[3]).long()
                for kp, vp in zip(self.k_pools, self.v_pools):
                    kp[to] = kp[begun].clone()
                    vp[to] = vp[begun].clone()
            table = torch.from_numpy(host).to(self._dims[3])
            valid = self.valid_buf.repeat(rows, 1)
            acc = None if self.acc is None else self.acc.repeat(rows, 1, 1)
        self._table_host, self.table, self.valid_buf, self.acc = host, table, valid, acc
        self.mapped, self.shared = (full + (1 if part else 0)) * PAGE, full * PAGE
        return self

    def layer_args(self, li: int):
        """(K pool, V pool, table, width) of layer li for the C ABI."""
        return self.k_pools[li], self.v_pools[li], self.table, self.width


def pages_from_contiguous(kc: torch.Tensor, vc: torch.Tensor, seed: int | None = None):
    """Paged copy of a contiguous cache: kc [B, n_kv, cap, hd], vc (V^T)
    [B, n_kv, hd, cap] with cap % PAGE == 0 -> (k_pool, v_pool, table). With
    ``seed`` the page ids are a seeded permutation (rows interleaved, so
    lookups must go through the table)."""
    B, n_kv, cap, hd = kc.shape
    w = cap // PAGE
    n = B * w
    order = np.arange(n, dtype=np.int32)
    if seed is not None:
        order = np.random.default_rng(seed).permutation(n).astype(np.int32)
    table = torch.from_numpy(order.reshape(B, w)).to(kc.device)
    kp = torch.empty(n, n_kv, PAGE, hd, dtype=torch.int8, device=kc.device)
    vp = torch.empty(n, n_kv, hd, PAGE, dtype=torch.int8, device=kc.device)
    kpages = kc.reshape(B, n_kv, w, PAGE, hd).permute(0, 2, 1, 3, 4).reshape(n, n_kv, PAGE, hd)
    vpages = vc.reshape(B, n_kv, hd, w, PAGE).permute(0, 3, 1, 2, 4).reshape(n, n_kv, hd, PAGE)
    idx = table.reshape(-1).long()
    kp[idx] = kpages
    vp[idx] = vpages
    return kp, vp, table
