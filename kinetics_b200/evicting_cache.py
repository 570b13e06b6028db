"""KV manager of bounded size: eviction by accumulated attention weight.

The surface of ``BatchKVManager`` (``compute_attention``, ``begin_step``, ``prepare_step`` / ``end_step``, ``clear_cache``,
``check_status``; counterpart of ``LiteSys/litesys/attention/batch_cache.py:10-168``), over caches that hold at most
``keep + max(room, portion)`` tokens per slot whatever the length of the sequence.  The reference has no such cache: its
masks choose among tokens that all stay.

* Every attention also adds up, per kv head, the weights that it gives each cached token (``ops.dense_decode_mass``,
  ``ops.prefill_attention_mass``: of a portion of a prompt those of the last ``window`` tokens).
* A slot that has grown ``room`` tokens beyond ``keep`` is cut back to ``keep`` (``ops.evict``): the first ``sink``
  positions and the last ``recent`` ones stay, and of the others the tokens that were paid most.
* Prompts run in portions of ``portion`` tokens, cut back in between, so that a prompt of any length fits.

The keys in the cache carry their rotary positions, so a token's place in the cache does not matter, and the model counts
positions as if nothing had been evicted.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence

import numpy as np
import torch

from . import ops

PAGE = ops.PAGE_SIZE


class EvictingKVManager:
    def __init__(self, config, max_batch_size: int, max_seq_len: int, device, dtype, keep: int, sink: int = 4,
                 recent: int = 64, window: int = 64, room: int = 256, portion: int = 1024, decay: float = 1.0):
        """keep: tokens of a slot behind an eviction; decay: factor of the accumulated weights per attention."""
        if keep < 1 or sink < 0 or recent < 0 or sink + recent > keep:
            raise ValueError(f"keep {keep}, sink {sink}, recent {recent}: 1 <= keep and sink + recent <= keep")
        if room < 1 or portion < 1 or window < 0:
            raise ValueError(f"room {room} and portion {portion} are at least 1, window {window} at least 0")
        self.config = config
        self.max_length = max_seq_len
        self.device = torch.device(device)
        self.dtype = dtype
        self.max_batch_size = max_batch_size
        self.head_dim = getattr(config, "head_dim", config.hidden_size // config.num_attention_heads)
        if self.head_dim != ops.HEAD_DIM:
            raise ValueError(f"only head_dim={ops.HEAD_DIM} is built")
        self.world_size = torch.distributed.get_world_size() if torch.distributed.is_available() and \
            torch.distributed.is_initialized() else 1
        self.num_layers = config.num_hidden_layers
        self.hidden_size = self.head_dim * config.num_attention_heads // self.world_size
        self.num_key_value_heads = config.num_key_value_heads // self.world_size
        self.num_attention_heads = config.num_attention_heads // self.world_size
        self.keep, self.sink, self.recent, self.window, self.decay = keep, sink, recent, window, decay
        self.room, self.portion = room, portion
        self.capacity = keep + max(room, portion)
        self.pages_per_slot = (self.capacity + PAGE - 1) // PAGE
        self.sm_scale = 1.0 / math.sqrt(self.head_dim)

        # slot b owns pages [b * pages_per_slot, (b + 1) * pages_per_slot)
        n, heads, places = max_batch_size * self.pages_per_slot, self.num_key_value_heads, self.pages_per_slot * PAGE
        self.kv_pages = [torch.zeros(n, 2, PAGE, heads, self.head_dim, device=self.device, dtype=dtype)
                         for _ in range(self.num_layers)]
        self.kv_indices = torch.arange(n, device=self.device, dtype=torch.int32)
        self.mass = [torch.zeros(max_batch_size, heads, places, device=self.device) for _ in range(self.num_layers)]
        self.positions = [torch.zeros(max_batch_size, heads, places, device=self.device, dtype=torch.int32)
                          for _ in range(self.num_layers)]
        self.status = ops.new_status(self.device)
        # per layer and slot: tokens in the cache, those whose positions are stored, tokens given in all
        self._held = np.zeros((self.num_layers, max_batch_size), dtype=np.int64)
        self._stored = np.zeros_like(self._held)
        self._seen = np.zeros_like(self._held)
        self._active: Optional[List[int]] = None
        self._table_key = self._table_val = None
        self._step_table = None
        self._static = None
        self._workspace = None
        self.evictions = 0               # of (layer, slot)

    # ---- page table: starts, page counts, tokens in the last page, slots
    @staticmethod
    def _rows(slots, lengths, pages_per_slot):
        s, n = np.asarray(slots, dtype=np.int64), np.asarray(lengths, dtype=np.int64)
        count = (n + PAGE - 1) // PAGE
        return np.stack((s * pages_per_slot, count, n - (count - 1) * PAGE, s)).astype(np.int32)

    def _table(self, slots, lengths):
        key = (tuple(slots), tuple(lengths), torch.cuda.current_stream(self.device).cuda_stream)
        if key != self._table_key:
            rows = torch.from_numpy(self._rows(slots, lengths, self.pages_per_slot)).pin_memory().to(self.device, non_blocking=True)
            self._table_key, self._table_val = key, (rows[0], rows[2], ops.PageView(0, 0, rows[1], rows[3]))
        return self._table_val

    def _checked(self, slots) -> List[int]:
        """A row each: two rows of one slot would append to and count the same places."""
        slots = [int(s) for s in slots]
        if len(set(slots)) != len(slots) or any(not 0 <= s < self.max_batch_size for s in slots):
            raise ValueError(f"slots {slots}: different ones of {self.max_batch_size}")
        return slots

    def _slots_of(self, batch_idx) -> List[int]:
        if self._active is not None and len(self._active) == batch_idx.numel():
            return self._active
        return self._checked(batch_idx.tolist())

    def cached(self, slot: int, layer_idx: int = 0) -> int:
        """Tokens that the slot's cache holds."""
        return int(self._held[layer_idx, slot])

    # ---- eviction
    def _evict(self, layer_idx: int, slots: Sequence[int]) -> None:
        slots = [s for s in slots if self._held[layer_idx, s] > self.keep]
        if not slots:
            return
        lengths = [int(self._held[layer_idx, s]) for s in slots]
        start, last, view = self._table(slots, lengths)
        counts = torch.from_numpy(np.stack((self._stored[layer_idx], self._seen[layer_idx])).astype(np.int32))
        stored, seen = counts.pin_memory().to(self.device, non_blocking=True).unbind(0)
        ops.evict(self.kv_pages[layer_idx], self.kv_indices, start, last, self.pages_per_slot, self.mass[layer_idx],
                  self.positions[layer_idx], stored, seen, self.keep, self.sink, self.recent, status=self.status, view=view)
        self._held[layer_idx, slots] = self._stored[layer_idx, slots] = self.keep
        self.evictions += len(slots)

    def _full(self, layer_idx: int, slots: Sequence[int]) -> List[int]:
        """Slots without room for another token of theirs."""
        return [s for s in slots if self._held[layer_idx, s] + 1 > self.keep + self.room]

    # ---- attention
    def compute_attention(self, query_states, key_states, value_states, layer_idx, batch_idx):
        """q [B, Hq, S, D], k/v [B, Hkv, S, D] -> [B, S, Hq * D] (batch_cache.py:86-110)."""
        bsz, seq_len = query_states.shape[0], query_states.shape[2]
        if seq_len > 1:
            return self.prefill_or_append(query_states, key_states, value_states, layer_idx, batch_idx)
        return self.decode(query_states, key_states, value_states, batch_idx, layer_idx).reshape(bsz, seq_len, self.hidden_size)

    def _decode_workspace(self):
        """Sized once for any number of active slots: captured steps keep its address."""
        if self._workspace is None:
            need = ops.decode_mass_workspace_bytes(self.max_batch_size, self.num_key_value_heads,
                                                   self.num_attention_heads // self.num_key_value_heads, self.pages_per_slot, self.dtype,
                                                   fewer=True)
            self._workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
        return self._workspace

    def decode(self, query, key, value, batch_idx, layer_idx):
        """One token of every active slot: append, attend, accumulate."""
        B, workspace = batch_idx.numel(), self._decode_workspace()           # before the slots count the token
        if self._step_table is None:
            slots = self._slots_of(batch_idx)
            self._evict(layer_idx, self._full(layer_idx, slots))
            self._held[layer_idx, slots] += 1
            self._seen[layer_idx, slots] += 1
            table = self._table(slots, [int(self._held[layer_idx, s]) for s in slots])
        else:
            table = self._step_table
        start, last, view = table
        rows = lambda t, heads: t.reshape(B, heads, self.head_dim).to(self.dtype).contiguous()
        pages = self.kv_pages[layer_idx]
        ops.append_kv(rows(key, self.num_key_value_heads), rows(value, self.num_key_value_heads), pages, None, self.kv_indices, start,
                      last, status=self.status, view=view)
        out, _ = ops.dense_decode_mass(rows(query, self.num_attention_heads), pages, self.kv_indices, start, last, self.pages_per_slot,
                                       self.mass[layer_idx], self.decay, self.sm_scale, workspace=workspace,
                                       status=self.status, view=view)
        return out

    def prefill_or_append(self, query_states, key_states, value_states, layer_idx, batch_idx):
        """One sequence's next tokens, portion by portion: append, attend causally, accumulate, and cut back where the next
        portion would not fit."""
        bsz, seq_len = query_states.shape[0], query_states.shape[2]
        assert bsz == 1, "prefill handles one sequence at a time, like the reference"
        slot = self._slots_of(batch_idx)[0]
        # [tokens, heads, D]
        q, k, v = (t[0].transpose(0, 1).to(self.dtype).contiguous() for t in (query_states, key_states, value_states))
        pages, outs, at = self.kv_pages[layer_idx], [], 0
        while at < seq_len:
            n = min(seq_len - at, self.portion)
            if self._held[layer_idx, slot] + n > self.capacity:
                self._evict(layer_idx, [slot])
            n = min(n, self.capacity - int(self._held[layer_idx, slot]))
            self._held[layer_idx, slot] += n
            self._seen[layer_idx, slot] += n
            start, last, view = self._table([slot], [int(self._held[layer_idx, slot])])
            indptr = torch.tensor([0, n], device=self.device, dtype=torch.int32)
            ops.append_tokens(k[at:at + n], v[at:at + n], indptr, pages, None, self.kv_indices, start, last, status=self.status,
                              view=view)
            out, _ = ops.prefill_attention_mass(q[at:at + n], indptr, n, pages, self.kv_indices, start, last, self.mass[layer_idx],
                                                self.window, self.decay, self.sm_scale, status=self.status, view=view)
            outs.append(out)
            at += n
        out = outs[0] if len(outs) == 1 else torch.cat(outs)
        return out.reshape(bsz, seq_len, self.hidden_size)

    # ---- a decode step whose device work can sit in a CUDA graph (Engine.decode_graphed)
    def begin_step(self, slots: Sequence[int]) -> None:
        """The slots of the calls that follow, in the order of their batch_idx, which is then not read."""
        self._active = self._checked(slots)

    def prepare_step(self, slots: Sequence[int]) -> None:
        """The host work of one decode step over `slots`, and the evictions it needs, of all layers: the step itself is then the
        same launches whatever the lengths, with the page table in buffers whose addresses never change.  `end_step()` closes
        the step."""
        slots = self._checked(slots)
        n = len(slots)
        for layer in range(self.num_layers):
            self._evict(layer, self._full(layer, slots))
        self._held[:, slots] += 1
        self._seen[:, slots] += 1
        if self._static is None:
            mk = lambda: torch.empty(4, self.max_batch_size, dtype=torch.int32)
            self._static = (mk().pin_memory(), mk().to(self.device), torch.cuda.Event())
        else:
            self._static[2].synchronize()        # the last step's copy has read the pinned rows
        pinned, rows, copied = self._static
        pinned[:, :n] = torch.from_numpy(self._rows(slots, self._held[0, slots], self.pages_per_slot))
        rows.copy_(pinned, non_blocking=True)
        copied.record()
        self._step_table = (rows[0, :n], rows[2, :n], ops.PageView(0, 0, rows[1, :n], rows[3, :n]))
        self._active = slots

    def end_step(self) -> None:
        self._step_table = None

    def clear_cache(self, batch_idx: int):
        """The slot is free; what its pages and masses hold is never read again."""
        for a in (self._held, self._stored, self._seen):
            a[:, batch_idx] = 0

    def check_status(self):
        ops.raise_on_status(self.status)
