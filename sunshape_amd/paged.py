"""vLLM-style paged KV cache for SunShape-compressed keys.

No counterpart in the reference: its quantized keys are one contiguous [T, nb] code
tensor per (batch, KV head) (sunshape/vllm_attn_backend.py:99-123), and it has no paged
layout.  This is the caller on the write side of the decode kernel:

* key pages   [P, Hkv, page, nb] codes (uint8, or int16 / int32 past 256 codewords), filled by the encode kernel through
  a slot mapping (token slot = page * page_size + offset), no dense key tensor;
* passthrough [P, Hkv, page, n_heavy, bd] for SunShape-Mixed heavy blocks;
* value pages [P, Hkv, Dv, page] -- vLLM's dim-major value layout, which the
  MFMA decode kernel reads as B-operand fragments directly; 16 bits, or 8 (float8_e4m3fn) with a scale per
  page and KV head [P, Hkv];
* per-sequence block tables and lengths, with a simple free-page allocator;
* sequences that continue a shared one (``fork``): its pages are held once, and decode reads them once
  for the whole batch; or, with 8-bit values or a window, sequences that share whole pages and go on by themselves;
* a sliding window with first tokens that stay visible, whose dead pages ``release`` gives back;
* ``compact`` and ``resize``, which move pages.

``attend`` is one layer's step of a serving loop: norm and rotation of the queries, the append of raw keys
and values with the same for the keys, and the attention.
"""

from __future__ import annotations

import contextlib
from typing import Optional

import torch

from . import hip_ops


class PagedSunShapeCache:
    def __init__(self, codec, *, num_pages: int, num_kv_heads: int, value_dim: int, page_size: int = 16,
                 value_dtype: torch.dtype = torch.bfloat16, passthrough_dtype: torch.dtype = torch.bfloat16,
                 device: Optional[torch.device] = None, window: Optional[int] = None, sinks: int = 0):
        """value_dtype float8_e4m3fn: values in 8 bits (hip_ops.append_values).  window, sinks: every token sees the
        window's newest tokens up to itself and the first `sinks` ones.  Either takes hip_ops.decode_window,
        which is causal and serves fewer codecs: others are refused here."""
        reason = codec.unsupported_reason()
        if reason is not None:
            raise RuntimeError(reason)
        self.window, self.sinks = window, int(sinks)
        self.causal = window is not None or value_dtype == torch.float8_e4m3fn  # decode_window serves decode
        if self.causal:
            reason = self._causal_unsupported(codec, value_dim, page_size, value_dtype, window, sinks)
            if reason is not None:
                raise RuntimeError(reason)
        elif sinks:
            raise RuntimeError("sinks go with a window")
        self.codec = codec
        self.device = torch.device(device) if device is not None else codec.device
        self.page_size = int(page_size)
        self.num_pages = int(num_pages)
        self.num_kv_heads = int(num_kv_heads)
        self.value_dim = int(value_dim)
        nb, bd = codec.n_blocks, codec.block_dim
        self.code_pages = torch.zeros(num_pages, num_kv_heads, page_size, nb, device=self.device,
                                      dtype=hip_ops.index_dtype(self.codec.n_centroids))
        self.v_pages = torch.zeros(num_pages, num_kv_heads, value_dim, page_size, dtype=value_dtype, device=self.device)
        self.v_scale = None
        if value_dtype == torch.float8_e4m3fn:
            self.v_scale = torch.zeros(num_pages, num_kv_heads, device=self.device)
        heavy = codec.heavy_blocks()
        self.heavy = heavy
        self.pt_pages = None
        if heavy is not None:
            self.pt_pages = torch.zeros(num_pages, num_kv_heads, page_size, sum(heavy), bd, dtype=passthrough_dtype,
                                        device=self.device)
        self._free = list(range(num_pages - 1, -1, -1))
        self.block_tables: dict[int, list[int]] = {}
        self.seq_lens: dict[int, int] = {}
        self.prefix_of: dict[int, int] = {}  # forked sequence -> the sequence it continues
        self._refs: dict[int, int] = {}      # page -> the sequences that hold it, where several do
        self._released: dict[int, int] = {}  # sequence -> the token that pages given back end at

    @staticmethod
    def _causal_unsupported(codec, value_dim, page_size, value_dtype, window, sinks) -> Optional[str]:
        """Why decode_window does not serve a cache (None: it does)."""
        D, bd = codec.n_blocks * codec.block_dim, codec.block_dim
        if window is not None and window < 1:
            return "window must be at least 1 (None: no window)"
        if sinks < 0 or (sinks and window is None):
            return "sinks go with a window, and are not negative"
        if codec.heavy_blocks() is not None:
            return "8-bit values and windows take codecs without passthrough blocks"
        if D not in (64, 128) or value_dim != D:
            return f"8-bit values and windows take head_dim 64 or 128 with value_dim the same, not {D} and {value_dim}"
        if bd not in (2, 4, 8) or codec.n_centroids > 256:
            return "8-bit values and windows take byte codes of block_dim 2, 4 or 8"
        if page_size not in (16, 32, 64, 128, 256):
            return f"8-bit values and windows take pages of 16, 32, 64, 128 or 256 tokens, not {page_size}"
        if value_dtype not in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
            return f"a window takes values of 8 or 16 bits, not {value_dtype}"
        return None

    # ------------------------------------------------------------------ pages
    def _pages(self, length: int) -> int:
        return (length + self.page_size - 1) // self.page_size

    @contextlib.contextmanager
    def _undone_if_refused(self, seq_ids: list[int]):
        """Gives the sequences' new pages and tokens back if the body raises: a refused step leaves no unwritten
        tokens behind."""
        before = {s: (self.seq_lens.get(s), len(self.block_tables.get(s, ()))) for s in seq_ids}
        try:
            yield
        except BaseException:
            for s, (length, pages) in reversed(before.items()):
                table = self.block_tables.get(s, [])
                while len(table) > pages:
                    self._free.append(table.pop())
                if length is None:
                    self.seq_lens.pop(s, None)
                    if not pages:
                        self.block_tables.pop(s, None)
                else:
                    self.seq_lens[s] = length
            raise

    def free(self, seq_id: int) -> None:
        if seq_id in self.prefix_of.values():
            raise RuntimeError(f"sequence {seq_id} is the prefix of others; free them first")
        self.prefix_of.pop(seq_id, None)
        for pg in self.block_tables.pop(seq_id, []):
            self._drop(pg)
        self.seq_lens.pop(seq_id, None)
        self._released.pop(seq_id, None)

    def _drop(self, page: int) -> None:
        """One holder less of a page (-1: released before)."""
        if page < 0:
            return
        left = self._refs.get(page, 1) - 1
        if left == 0:
            self._free.append(page)
        elif left == 1:
            del self._refs[page]
        else:
            self._refs[page] = left

    def fork(self, prefix_id: int, seq_ids: list[int]) -> None:
        """Start sequences that continue prefix_id's tokens.  They start empty, and the prefix takes no more tokens while
        any of them lives, and decode reads them once for all; in a cache with 8-bit values or a window they start as copies
        of it, which share its whole pages, copy its last one if that is not full and go on by themselves, and decode reads
        the shared pages once for each."""
        if self.causal:
            return self._fork_copies(prefix_id, seq_ids)
        if not self.seq_lens.get(prefix_id) or prefix_id in self.prefix_of:
            raise RuntimeError(f"sequence {prefix_id} cannot be a prefix: it holds no tokens or continues another")
        if len(set(seq_ids)) != len(seq_ids) or any(s == prefix_id or s in self.seq_lens or s in self.prefix_of
                                                    for s in seq_ids):
            raise RuntimeError("fork starts new, distinct sequences")
        for s in seq_ids:
            self.prefix_of[s] = prefix_id

    def _fork_copies(self, prefix_id: int, seq_ids: list[int]) -> None:
        length = self.seq_lens.get(prefix_id)
        if not length:
            raise RuntimeError(f"sequence {prefix_id} cannot be a prefix: it holds no tokens")
        if len(set(seq_ids)) != len(seq_ids) or any(s in self.seq_lens or s in self.block_tables for s in seq_ids):
            raise RuntimeError("fork starts new, distinct sequences")
        table = self.block_tables[prefix_id]
        whole = length // self.page_size
        part = length % self.page_size != 0
        if part and len(seq_ids) > len(self._free):
            raise RuntimeError("PagedSunShapeCache is out of pages")
        if part and seq_ids:
            own = self._free[-len(seq_ids):][::-1]
            hip_ops.copy_pages(self._pools(), self._index([table[whole]] * len(own)), self._index(own))
            del self._free[-len(own):]
        for i, s in enumerate(seq_ids):
            for pg in table[:whole]:
                if pg >= 0:
                    self._refs[pg] = self._refs.get(pg, 1) + 1
            self.block_tables[s] = table[:whole] + ([own[i]] if part else [])
            self.seq_lens[s] = length
            if prefix_id in self._released:
                self._released[s] = self._released[prefix_id]

    def _pools(self) -> list[torch.Tensor]:
        return [p for p in (self.code_pages, self.v_pages, self.v_scale, self.pt_pages) if p is not None]

    def _index(self, pages: list[int]) -> torch.Tensor:
        return torch.tensor(pages, dtype=torch.int64, device=self.device)

    def release(self, seq_ids: list[int]) -> int:
        """Give back the pages whose tokens have left the window (and are no sinks) of each sequence's newest token;
        returns how many are free again.  decode refuses queries older than that token, where they would see one."""
        if self.window is None:
            return 0
        before = len(self._free)
        for s in seq_ids:
            first = (self.sinks + self.page_size - 1) // self.page_size
            end = (self.seq_lens.get(s, 0) - self.window) // self.page_size  # pages [first, end) are dead
            table = self.block_tables.get(s, [])
            for i in range(max(first, self._released.get(s, 0) // self.page_size), end):
                self._drop(table[i])
                table[i] = -1
            if end > first:
                self._released[s] = max(self._released.get(s, 0), end * self.page_size)
        return len(self._free) - before

    def _held(self) -> list[int]:
        return sorted({pg for t in self.block_tables.values() for pg in t if pg >= 0})

    def _renumber(self, to: dict[int, int], num_pages: int) -> None:
        for table in self.block_tables.values():
            table[:] = [to.get(pg, pg) for pg in table]
        self._refs = {to.get(pg, pg): n for pg, n in self._refs.items()}
        used = set(self._held())
        self._free = [pg for pg in range(num_pages - 1, -1, -1) if pg not in used]

    def compact(self) -> int:
        """Move the pages that sequences hold to the front of the pools, in place; returns how many there are.  Tables made
        before are out of date."""
        held = self._held()
        n = len(held)
        behind = [pg for pg in held if pg >= n]
        room = sorted(set(range(n)) - set(held))
        if behind:
            hip_ops.copy_pages(self._pools(), self._index(behind), self._index(room))
        self._renumber(dict(zip(behind, room)), self.num_pages)
        return n

    def resize(self, num_pages: int) -> None:
        """New pools of num_pages pages with what the sequences hold at the front.  Tables and pools taken before are
        out of date."""
        held = self._held()
        if num_pages < len(held):
            raise RuntimeError(f"{len(held)} pages are held, more than {num_pages}")
        old = self._pools()
        new = [torch.zeros(num_pages, *p.shape[1:], dtype=p.dtype, device=p.device) for p in old]
        if held:
            hip_ops.copy_pages(old, self._index(held), self._index(list(range(len(held)))), into=new)
        pools = iter(new)
        self.code_pages, self.v_pages = next(pools), next(pools)
        self.v_scale = None if self.v_scale is None else next(pools)
        self.pt_pages = None if self.pt_pages is None else next(pools)
        self.num_pages = int(num_pages)
        self._renumber({pg: i for i, pg in enumerate(held)}, self.num_pages)

    def _shared_prefix(self, seq_ids: list[int]) -> Optional[int]:
        found = {self.prefix_of.get(s) for s in seq_ids}
        if len(found) > 1:
            raise RuntimeError("the sequences of one call must continue the same prefix, or none")
        return found.pop() if found else None

    def positions(self, seq_ids: list[int], num_new: int) -> torch.Tensor:
        """int64 positions [len(seq_ids), num_new] of the next num_new tokens of (distinct) sequences, their
        prefix counted."""
        first = [self.seq_lens.get(s, 0) + self.seq_lens.get(self.prefix_of.get(s), 0) for s in seq_ids]
        return torch.tensor([[f + i for i in range(num_new)] for f in first], dtype=torch.int64,
                            device=self.device).view(len(seq_ids), num_new)

    def _within(self, seq_ids: list[int], num_new: int, cos: torch.Tensor) -> None:
        """The next tokens' positions lie inside the rotation's tables (past them a key would be NaN, and its codes
        those of some other key)."""
        end = max((self.seq_lens.get(s, 0) + self.seq_lens.get(self.prefix_of.get(s), 0) for s in seq_ids), default=0) + num_new
        if num_new and cos.dim() == 2 and end > cos.shape[0]:
            raise RuntimeError(f"position {end - 1} is outside the rotation's tables ({cos.shape[0]} rows)")

    def slot_mapping(self, seq_ids: list[int], num_new: int) -> torch.Tensor:
        """Allocate room for num_new tokens per sequence, for all or for none; return int64 slots
        [len(seq_ids), num_new]."""
        shared = set(self.prefix_of.values())
        if any(s in shared for s in seq_ids):
            raise RuntimeError("a sequence that others continue takes no more tokens")
        lengths: dict[int, int] = {}
        for sid in seq_ids:
            lengths[sid] = lengths.get(sid, self.seq_lens.get(sid, 0)) + num_new
        missing = sum(max(0, self._pages(n) - len(self.block_tables.get(sid, ()))) for sid, n in lengths.items())
        if missing > len(self._free):
            raise RuntimeError("PagedSunShapeCache is out of pages")
        rows = []
        for sid in seq_ids:
            start = self.seq_lens.get(sid, 0)
            table = self.block_tables.setdefault(sid, [])
            while len(table) < self._pages(start + num_new):
                table.append(self._free.pop())
            rows.append([table[(start + i) // self.page_size] * self.page_size + (start + i) % self.page_size
                         for i in range(num_new)])
            self.seq_lens[sid] = start + num_new
        return torch.tensor(rows, dtype=torch.int64, device=self.device)

    # ------------------------------------------------------------------ append / decode
    def append(self, seq_ids: list[int], key_states: torch.Tensor, value_states: torch.Tensor, *,
               cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
               k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
        """Encode keys [B, Hkv, S, D] into the code pages and write values [B, Hkv, S, Dv]; returns the slots.

        With cos and sin (tables, hip_ops.rope_table) or k_weight the keys are raw: they are normed and
        rotated on the way, each token at its position in its sequence (its prefix counted), which the tables
        have to reach."""
        B, Hkv, S, _ = key_states.shape
        if Hkv != self.num_kv_heads or value_states.shape[:3] != key_states.shape[:3]:
            raise RuntimeError("key/value shapes do not match the cache")
        if (cos is None) != (sin is None):
            raise RuntimeError("cos and sin come together")
        if self.v_scale is not None and len(set(seq_ids)) != len(seq_ids):
            raise RuntimeError("an append of 8-bit values takes each sequence once")
        if cos is not None or k_weight is not None:
            if len(seq_ids) != B:
                raise RuntimeError(f"{B} rows of keys for {len(seq_ids)} sequences")
            if len(set(seq_ids)) != len(seq_ids):
                raise RuntimeError("an append with rotation takes each sequence once")
            if cos is not None:
                self._within(seq_ids, S, cos)
            return self._append_raw(seq_ids, key_states, value_states, self.positions(seq_ids, S) if cos is not None else None,
                                    cos=cos, sin=sin, k_weight=k_weight, eps=eps, interleaved=interleaved)
        with self._undone_if_refused(seq_ids):
            slots = self.slot_mapping(seq_ids, S)
            perm = self.codec.effective_permutation()
            # as quantize_key_states: one reference cdist per (sequence, KV head) over its S new keys
            hip_ops.encode(key_states.to(self.device), perm, self.codec.centroids, heavy=self.heavy,
                           codes_out=self.code_pages, pt_out=self.pt_pages, slot_mapping=slots,
                           metric=self.codec.encode_metric(), grid=self.codec.encode_search_grid(self.codec.centroids),
                           direct=hip_ops.cdist_direct(S, self.codec.n_centroids),
                           rotation=self.codec.rotation_matrix())
            if self.v_scale is not None:
                hip_ops.append_values(value_states.to(self.device), self.v_pages, self.v_scale, slots)
                return slots
            flat = slots.reshape(-1)
            page, off = flat // self.page_size, flat % self.page_size
            vals = value_states.to(self.device, self.v_pages.dtype).permute(0, 2, 1, 3).reshape(B * S, Hkv, self.value_dim)
            self.v_pages[page, :, :, off] = vals
        return slots

    def _scales(self) -> dict:
        return {} if self.v_scale is None else {"v_scale": self.v_scale}

    def _append_raw(self, seq_ids, key_states, value_states, positions, **turn) -> torch.Tensor:
        S = key_states.shape[2]
        with self._undone_if_refused(seq_ids):
            slots = self.slot_mapping(seq_ids, S)
            hip_ops.append_kv(key_states.to(self.device), value_states.to(self.device), self.codec.effective_permutation(),
                              self.codec.centroids, codes_out=self.code_pages, v_out=self.v_pages, slot_mapping=slots,
                              positions=positions, heavy=self.heavy, pt_out=self.pt_pages, metric=self.codec.encode_metric(),
                              grid=self.codec.encode_search_grid(self.codec.centroids),
                              direct=hip_ops.cdist_direct(S, self.codec.n_centroids),
                              rotation=self.codec.rotation_matrix(), **turn, **self._scales())
        return slots

    def tables(self, seq_ids: list[int]) -> tuple[torch.Tensor, torch.Tensor]:
        """(block_table [B, max_pages] int32, seq_lens [B] int32) for these sequences."""
        width = max(len(self.block_tables.get(s, [])) for s in seq_ids) or 1
        bt = torch.zeros(len(seq_ids), width, dtype=torch.int32)
        for i, s in enumerate(seq_ids):
            t = self.block_tables.get(s, [])
            bt[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        lens = torch.tensor([self.seq_lens.get(s, 0) for s in seq_ids], dtype=torch.int32)
        return bt.to(self.device), lens.to(self.device)

    def decode(self, seq_ids: list[int], query: torch.Tensor, *, scale: Optional[float] = None,
               return_lse: bool = False, mask: Optional[torch.Tensor] = None):
        """Fused decode of query [B, Hq, Lq, D] against the cached sequences; forked ones attend their shared
        prefix's tokens first (the sequences of one call continue the same one, or none).  mask: additive,
        broadcastable to [B, Hq, Lq, T], T the sequences' own table width times the page size.  In a cache with 8-bit
        values or a window the queries are those of each sequence's Lq newest tokens, each of which sees the tokens up
        to itself (in its window); no mask."""
        if self.causal:
            if mask is not None:
                raise RuntimeError("a cache with 8-bit values or a window takes no mask")
            self._still_seen(seq_ids, query.shape[2])
            bt, lens = self.tables(seq_ids)
            return hip_ops.decode_window(query, self.code_pages, self.v_pages, self.codec.effective_permutation(),
                                         self.codec.centroids, block_table=bt, seq_lens=lens, scale=scale,
                                         window=self.window, sinks=self.sinks, return_lse=return_lse,
                                         rotation=self.codec.rotation_matrix(), **self._scales())
        prefix = self._shared_prefix(seq_ids)
        bt, lens = self.tables(seq_ids)
        if prefix is None:
            return hip_ops.decode(query, self.code_pages, self.v_pages, self.codec.effective_permutation(),
                                  self.codec.centroids, scale=scale, mask=mask, heavy=self.heavy, pt=self.pt_pages,
                                  pt_dense=False, block_table=bt, seq_lens=lens, return_lse=return_lse,
                                  rotation=self.codec.rotation_matrix())
        ptab, plen = self.tables([prefix])
        return hip_ops.decode_prefix(query, self.code_pages, self.v_pages, self.codec.effective_permutation(),
                                     self.codec.centroids, prefix_table=ptab[0], prefix_len=plen, block_table=bt,
                                     seq_lens=lens, scale=scale, mask=mask, heavy=self.heavy, pt=self.pt_pages,
                                     return_lse=return_lse, rotation=self.codec.rotation_matrix())

    def _still_seen(self, seq_ids: list[int], num_rows: int) -> None:
        """No token that the oldest of num_rows queries sees is in a released page."""
        for s, end in self._released.items():
            if s in seq_ids and self.seq_lens[s] - num_rows - self.window + 1 < end:
                raise RuntimeError(f"pages that the oldest query of sequence {s} sees are released")

    def attend(self, seq_ids: list[int], query: torch.Tensor, key_states: torch.Tensor, value_states: torch.Tensor, *,
               cos: torch.Tensor, sin: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
               k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
               scale: Optional[float] = None) -> torch.Tensor:
        """One step over raw projections: query [B, Hq, S, D], keys and values [B, Hkv, S, ..] of the S next
        tokens of each sequence.  Norms and rotates them, appends keys and values, and attends causally;
        returns [B, Hq, S, Dv].  scale as in decode (None: the query as it is).  A step that is refused leaves the
        sequences as they were (8-bit values of a last page may have been rounded to a larger scale).  With S > 1 the causal
        mask takes 4 B S times the longest own table's tokens in bytes (none in a cache with 8-bit values or a window, whose
        pages that left the window are given back after the step)."""
        B, _, S, _ = query.shape
        if len(set(seq_ids)) != len(seq_ids):
            raise RuntimeError("attend takes each sequence once")
        if len(seq_ids) != B or key_states.shape[0] != B or key_states.shape[2] != S:
            raise RuntimeError("query, keys and values must hold the same new tokens of each sequence")
        if key_states.shape[1] != self.num_kv_heads or value_states.shape[:3] != key_states.shape[:3]:
            raise RuntimeError("key/value shapes do not match the cache")
        if query.shape[1] % self.num_kv_heads:  # (decode would find it behind the append)
            raise RuntimeError("Query head count must be divisible by kv-head count.")
        self._shared_prefix(seq_ids)
        self._within(seq_ids, S, cos)
        positions = self.positions(seq_ids, S)
        q, _ = hip_ops.qk_norm_rope(query, None, cos, sin, positions, q_weight=q_weight, eps=eps, interleaved=interleaved)
        with self._undone_if_refused(seq_ids):
            self._append_raw(seq_ids, key_states, value_states, positions, cos=cos, sin=sin, k_weight=k_weight, eps=eps,
                             interleaved=interleaved)
            mask = None
            if S > 1 and not self.causal:  # new token i sees its sequence up to itself
                width = max(len(self.block_tables[s]) for s in seq_ids) * self.page_size
                last = torch.tensor([self.seq_lens[s] - S for s in seq_ids], device=self.device)[:, None] + \
                    torch.arange(S, device=self.device)[None]
                mask = torch.zeros(B, 1, S, width, device=self.device)
                mask.masked_fill_(torch.arange(width, device=self.device) > last[:, None, :, None], float("-inf"))
            out = self.decode(seq_ids, q, scale=scale, mask=mask)
        self.release(seq_ids)
        return out
