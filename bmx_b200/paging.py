"""Page-slot allocator and a multi-sequence k2b layer state on top of it.

bmx keeps one cache object per sequence and measures the steady-state cost of a sequence by running several of them side
by side (bmx: scripts/batch_oom_sweep.py:112-178).  On the B200 path all sequences of a layer share ONE page pool: a
sequence owns whatever slots the allocator handed it, its row of the page table lists them in order, and the decode and
append kernels only ever see (pool, page table, page counts).  Sequences of different lengths join and leave; freed slots
are reused.  Memory per sequence comes from the allocator's own statistics, never from exhausting the device.
"""

from __future__ import annotations

import math

import torch

from . import kernels as K
from .schedule import compute_flush_schedule

HEAD_DIM = K.HEAD_DIM


class PageAllocator:
    """Free list over `n_slots` page slots (pure host code).  Slots of a sequence are returned in allocation order.  A slot may belong
    to several sequences (share) and is free again when the last of them gives it back."""

    def __init__(self, n_slots: int):
        assert n_slots > 0
        self.n_slots = n_slots
        self._free = list(range(n_slots - 1, -1, -1))  # pop() hands out low slots first
        self._owned: dict[object, list[int]] = {}
        self._refs: dict[int, int] = {}                # slot -> sequences that hold it
        self.peak_in_use = 0
        self.version = 0                               # changes with every change of who holds what

    def alloc(self, seq, n: int, places: list[int] | None = None, pages: int | None = None) -> list[int]:
        """n more slots for sequence `seq`; raises MemoryError (and changes nothing) if the pool cannot hold them.  With places, the
        sequence grows by `pages` pages of which only those at `places` (ascending, n of them) get a slot, the others -1."""
        if n > len(self._free):
            raise MemoryError(f"page pool exhausted: {n} slots wanted, {len(self._free)} of {self.n_slots} free")
        got = [self._free.pop() for _ in range(n)]
        self.version += bool(got or pages)
        for s in got:
            self._refs[s] = 1
        held = got
        if places is not None:
            held = [-1] * pages
            for p, s in zip(places, got):
                held[p] = s
        self._owned.setdefault(seq, []).extend(held)
        self.peak_in_use = max(self.peak_in_use, self.in_use)
        return got

    def _give_back(self, slots: list[int]) -> int:
        """One holder less for each slot, in order; returns how many are free again."""
        n = 0
        self.version += bool(slots)
        for s in slots:
            self._refs[s] -= 1
            if self._refs[s] == 0:
                del self._refs[s]
                self._free.append(s)
                n += 1
        return n

    def free(self, seq) -> int:
        """Gives back every slot of `seq`; returns how many of them nobody holds any more."""
        slots = self._owned.pop(seq, [])
        self.version += bool(slots)  # entries of pages given back before count too: they were part of a page table
        return self._give_back([s for s in reversed(slots) if s >= 0])

    def share(self, seq, other) -> list[int]:
        """`other`, which holds nothing yet, holds all slots of `seq` too (a fork: committed pages never change)."""
        if self._owned.get(other):
            raise ValueError(f"sequence {other!r} holds slots already")
        slots = self._owned.get(seq, [])
        self.version += 1
        for s in slots:
            if s >= 0:
                self._refs[s] += 1
        self._owned[other] = list(slots)
        return list(slots)

    def release(self, seq, first: int, end: int) -> int:
        """Gives back the slots of pages first .. end - 1 of `seq`, whose entries become -1 (pages that no query sees any more)."""
        slots = self._owned.get(seq, [])
        if not 0 <= first <= end <= len(slots):
            raise ValueError(f"pages {first}..{end} of a sequence of {len(slots)}")
        gone = [s for s in reversed(slots[first:end]) if s >= 0]
        slots[first:end] = [-1] * (end - first)
        return self._give_back(gone)

    def available(self, seq, first: int, end: int) -> int:
        """Slots that are free once release(seq, first, end) has been called."""
        mine = self._owned.get(seq, [])[first:end]
        return len(self._free) + sum(s >= 0 and self._refs[s] == 1 for s in mine)

    def compact(self) -> tuple[list[int], list[int]]:
        """Renumbers the held slots to 0 .. in_use - 1 and returns the (from, to) lists of those that have to be copied: the ones
        beyond, into the holes below, so that no slot is both read and written."""
        m = self.in_use
        self.version += 1
        holes = sorted(s for s in self._free if s < m)
        moved = sorted(s for s in self._refs if s >= m)
        new = dict(zip(moved, holes))
        for slots in self._owned.values():
            slots[:] = [new.get(s, s) for s in slots]
        self._refs = {new.get(s, s): r for s, r in self._refs.items()}
        self._free = list(range(self.n_slots - 1, m - 1, -1))
        return moved, holes

    def slots(self, seq) -> list[int]:
        """Slots of `seq` in page order; -1 for pages that were given back."""
        return list(self._owned.get(seq, ()))

    @property
    def in_use(self) -> int:
        return self.n_slots - len(self._free)

    def grow(self, n_more: int) -> None:
        """The pool behind this allocator was enlarged by n_more slots (existing slots keep their numbers)."""
        self._free = list(range(self.n_slots + n_more - 1, self.n_slots - 1, -1)) + self._free
        self.n_slots += n_more

    def shrink(self, n_slots: int) -> None:
        """The pool behind this allocator was cut to its first n_slots slots, the others being free (see compact)."""
        if any(s >= n_slots for s in self._refs):
            raise ValueError(f"slots beyond {n_slots} are held")
        self._free = [s for s in self._free if s < n_slots]
        self.n_slots = n_slots


def _runs(numbers: list[int]) -> list[tuple[int, int]]:
    """Ascending integers -> their runs of consecutive ones as (begin, end)."""
    out: list[tuple[int, int]] = []
    for p in numbers:
        if out and out[-1][1] == p:
            out[-1] = (out[-1][0], p + 1)
        else:
            out.append((p, p + 1))
    return out


class PagedK2bLayer:
    """One attention layer's k2b cache for a changing set of sequences over one shared page pool.

    Each sequence has its own length, its own fp16 window row and its own run of page slots; all sequences share the frozen
    key basis of the layer (set with set_basis, or fitted on the first page that is ever committed).  `decode` runs one
    fused step over any subset of the live sequences.

    `fork` makes sequences that share all committed pages of another one; a decode step that meets several sequences with a common
    prefix reads it once for all of them.  With sliding_window, a token sees the last sliding_window tokens and the first `sinks`; pages
    that fall between the two are freed as sequences grow.  `compact` and `resize` close the holes that finished sequences leave.
    A sequence's length is limited by max_pages_per_seq pages, freed ones among them (its page table keeps their places), and by the
    rotation tables.
    """

    # 128-token tiles per SM that attending shared prefixes once has to save over streaming them for every sequence; its launch and the set-up of
    # its blocks cost the time of about one.  Measured at 8 KV heads and up to 3 pages behind the prefixes, steps in a replayed graph, shared
    # against streamed, in us.  Shared by this rule: 4 query heads per KV head, 2 sequences x 20 pages (1.1 tiles per SM saved) 15.7 / 15.7,
    # 8 x 4 (1.5) 16.7 / 18.3, 32 x 4 (6.7) 22.2 / 42.5, 32 x 256 49 / 402; 1 query head, 3 x 16 (1.7) 15.5 / 14.9, 6 x 8 (2.2) 15.6 / 17.1, 8 x 8
    # (3.0) 17.0 / 18.1.  Streamed: 1 query head, 4 x 4 (0.6) 14.9 / 12.5, 2 x 16 (0.9) 15.3 / 13.9; 4 query heads, 4 x 4 (0.6) 15.0 / 16.0, 3 x 8
    # (0.9) 15.1 / 16.6; 8 query heads, 4 x 1 (0.2) 15.9 / 18.1, 2 x 8 (0.4) 15.9 / 19.4.  The border lies higher with one query head and lower with
    # eight; one number for all of them is off by at most 0.6 us above it and 3.5 us below.
    SHARED_MIN_TILES = 1

    def __init__(self, geom, n_slots: int, max_seqs: int, recent_window: int, device, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
                 *, v_seed: int = 0, max_pages_per_seq: int = 1024, sliding_window: int | None = None, sinks: int = 0):
        if sliding_window is not None and (sliding_window < 1 or sinks < 0 or geom.layout != 1):
            raise ValueError(f"sliding_window={sliding_window}, sinks={sinks}: a window of at least one token over 128-token pages of layout 1")
        if sliding_window is None and sinks:
            raise ValueError("sinks without a sliding_window: every token is visible already")
        self.sliding_window, self.sinks = sliding_window, sinks
        self.geom, self.device, self.page, self.W = geom, torch.device(device), geom.page, recent_window
        self.pool = K.K2bPool(geom, n_slots, self.device)
        self.alloc = PageAllocator(n_slots)
        self.max_seqs, self.max_pages = max_seqs, max_pages_per_seq
        self.tail_cap = recent_window + geom.page
        shape = (max_seqs, geom.h_kv, self.tail_cap, HEAD_DIM)
        self.k_win = torch.zeros(shape, dtype=torch.float16, device=self.device)
        self.v_win = torch.zeros(shape, dtype=torch.float16, device=self.device)
        self.k_pre_win = torch.zeros(shape, dtype=torch.float16, device=self.device)
        self.rope_cos, self.rope_sin = rope_cos, rope_sin
        cb = K.GAUSSIAN_CODEBOOK[geom.vbits]
        self.codebook = torch.tensor(cb, dtype=torch.float32, device=self.device)
        self.v_lut = K.v_lut_tensor(cb, self.device)
        self.signs = K.hadamard_signs(HEAD_DIM, v_seed).to(self.device)
        self.basis_f32 = self.basis_f16 = None
        self.sm_scale = 1.0 / math.sqrt(HEAD_DIM)
        self._rows: dict[object, int] = {}          # sequence -> row of the window buffers
        self._free_rows = list(range(max_seqs - 1, -1, -1))
        self._committed: dict[object, int] = {}
        self._tail: dict[object, int] = {}
        self._ws: dict[tuple[int, int], torch.Tensor] = {}  # decode workspaces by batch size and stream
        self._plan: tuple | None = None             # (what it holds for, page table, page counts, window rows, prefix groups, workspace) of a step
        self._rope_frag: tuple | None = None        # (stream, rotation tables in the prefill kernel's order, as far as prefixes reach)

    # ---- bookkeeping ------------------------------------------------------------------------
    def set_basis(self, basis_f32: torch.Tensor) -> None:
        self.basis_f32 = basis_f32.to(self.device, torch.float32).contiguous()
        self.basis_f16 = self.basis_f32.half().contiguous()

    def add_sequence(self, seq) -> None:
        assert seq not in self._rows, f"sequence {seq!r} is live already"
        if not self._free_rows:
            raise MemoryError(f"all {self.max_seqs} sequence rows are in use")
        self._rows[seq], self._committed[seq], self._tail[seq] = self._free_rows.pop(), 0, 0

    def drop_sequence(self, seq) -> int:
        """Ends a sequence: its page slots and its window row can be reused at once.  Returns the slots freed."""
        self._free_rows.append(self._rows.pop(seq))
        del self._committed[seq], self._tail[seq]
        return self.alloc.free(seq)

    def seq_len(self, seq) -> int:
        return self._committed[seq] + self._tail[seq]

    def fork(self, seq, *children) -> None:
        """New sequences that begin with everything `seq` holds: its committed pages are shared (they never change, and are free again
        when the last holder ends), its row of the fp16 windows is copied, in one launch for all children."""
        row, t, h = self._rows[seq], self._tail[seq], self.geom.h_kv
        if len(set(children)) != len(children) or any(c in self._rows for c in children):
            raise ValueError(f"fork: {children} are live already or named twice")
        if len(children) > len(self._free_rows):
            raise MemoryError(f"{len(children)} sequence rows wanted, {len(self._free_rows)} of {self.max_seqs} free")
        to = []
        for c in children:
            self.add_sequence(c)
            self.alloc.share(seq, c)
            self._committed[c], self._tail[c] = self._committed[seq], t
            to += [self._rows[c] * h + i for i in range(h)]
        if t and to:
            wins = [w.flatten(0, 1)[:, :t] for w in (self.k_win, self.v_win, self.k_pre_win)]
            K.copy_slots(wins, wins, [row * h + i for _ in children for i in range(h)], to)

    def compact(self) -> int:
        """Moves the pages in use to the lowest slots of the pool, in one launch; returns how many moved."""
        moved, holes = self.alloc.compact()
        K.copy_slots([self.pool.pages, self.pool.coefs], [self.pool.pages, self.pool.coefs], moved, holes)
        return len(moved)

    def resize(self, n_slots: int) -> None:
        """A pool of n_slots slots takes this one's place, with the pages in use (MemoryError if they do not fit) in its lowest slots."""
        m = self.alloc.in_use
        if n_slots < max(1, m):
            raise MemoryError(f"{m} slots are in use, {n_slots} wanted")
        old, live = self.pool, sorted(self.alloc._refs)
        pool = K.K2bPool(self.geom, n_slots, self.device)
        moved, holes = self.alloc.compact()
        now = dict(zip(moved, holes))
        K.copy_slots([old.pages, old.coefs], [pool.pages, pool.coefs], live, [now.get(s, s) for s in live])
        for t in (old.pages, old.coefs):  # their memory may belong to another stream, which must not hand it out while this one copies
            if t.is_cuda:
                t.record_stream(torch.cuda.current_stream(self.device))
        self.pool = pool
        if n_slots > self.alloc.n_slots:
            self.alloc.grow(n_slots - self.alloc.n_slots)
        else:
            self.alloc.shrink(n_slots)

    # ---- append -----------------------------------------------------------------------------
    def append(self, seq, k_pre: torch.Tensor, k_post: torch.Tensor, v: torch.Tensor) -> None:
        """n new tokens of one sequence, (h_kv, n, 128) each (fp16 or bf16): whole pages beyond the recent window are
        quantized into freshly allocated slots, the rest stays in the sequence's fp16 window (bmx's flush schedule)."""
        from .engine import fit_basis

        row, t, n = self._rows[seq], self._tail[seq], k_post.shape[1]
        src_k = torch.cat([self.k_pre_win[row, :, :t].to(k_pre.dtype), k_pre], 1) if t else k_pre
        post = torch.cat([self.k_win[row, :, :t].to(k_post.dtype), k_post], 1) if t else k_post
        val = torch.cat([self.v_win[row, :, :t].to(v.dtype), v], 1) if t else v
        total = self._committed[seq] + t + n
        p0 = self._committed[seq] // self.page
        n_flush = (compute_flush_schedule(total, self.W, self.page) - self._committed[seq]) // self.page
        # sliding_window: the next query is the newest token or a later one, so the pages behind the sinks' and in front of the newest
        # token's window are given back, and those among the new ones are never quantized
        keep, first = p0 + n_flush, 0
        if self.sliding_window is not None:
            keep, first = -(-self.sinks // self.page), max(0, total - self.sliding_window) // self.page
        kept = [p for p in range(p0, p0 + n_flush) if p < keep or p >= first]
        old = self.alloc.slots(seq)
        gone = (min(keep, p0), max(min(keep, p0), min(p0, first)))
        if len(kept) > self.alloc.available(seq, *gone):
            raise MemoryError(f"page pool exhausted: {len(kept)} slots wanted, {self.alloc.available(seq, *gone)} of {self.alloc.n_slots} free")
        if n_flush > 0:
            assert len(old) + n_flush <= self.max_pages, "sequence longer than max_pages_per_seq pages"
            if self.basis_f32 is None:
                self.set_basis(fit_basis(self.geom, src_k[:, : self.page]))
        if gone[0] < gone[1]:
            self.alloc.release(seq, *gone)
        if n_flush > 0:
            got = dict(zip(kept, self.alloc.alloc(seq, len(kept), [p - p0 for p in kept], n_flush)))
            k_all, v_all = src_k[None], val[None].to(src_k.dtype)
            for a, b in _runs(kept):
                slots = torch.tensor([got[p] for p in range(a, b)], dtype=torch.int32, device=self.device)
                tok = slice((a - p0) * self.page, (b - p0) * self.page)
                K.k2b_append(self.pool, k_all[:, :, tok].contiguous(), v_all[:, :, tok].contiguous(), self.basis_f32, self.signs, self.codebook,
                             slots, b - a)
            self._committed[seq] += n_flush * self.page
        off = n_flush * self.page
        rest = post.shape[1] - off
        assert rest <= self.tail_cap
        self.k_win[row, :, :rest], self.v_win[row, :, :rest], self.k_pre_win[row, :, :rest] = post[:, off:], val[:, off:], src_k[:, off:]
        self._tail[seq] = rest

    # ---- decode -----------------------------------------------------------------------------
    def _prefix_groups(self, slots: list) -> tuple[list, list]:
        """(members, prefix pages) of the sequences that begin with the same slots, where attending their prefixes once pays."""
        if len(slots) > K.SHARED_MAX_BATCH or (self.geom.n_q_groups > 4 and self.k_win.shape[2] > K.SHARED_MAX_WINDOW_G8):
            return [], []
        first: dict[int, list[int]] = {}
        for i, s in enumerate(slots):
            if s:
                first.setdefault(s[0], []).append(i)
        members, pages = [], []
        for rows in first.values():
            if len(rows) < 2:
                continue
            a, n = slots[rows[0]], min(len(slots[r]) for r in rows)
            for r in rows[1:]:
                s = slots[r]
                if s[:n] != a[:n]:
                    n = next(j for j in range(n) if s[j] != a[j])
            members.append(rows)
            pages.append(n)
        saved = sum((len(m) - 1) * n for m, n in zip(members, pages)) * self.geom.h_kv
        return (members, pages) if saved >= self.SHARED_MIN_TILES * K.sm_count(self.device) else ([], [])

    def decode(self, seqs: list, q: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """q (len(seqs), heads, 128) fp16: one fused decode step over those sequences, each with its own pages and window; a prefix
        that several of them share is read once."""
        n = len(seqs)
        # what a step keeps for the next belongs to the stream it was made on: another stream's step makes its own, so that nothing is read
        # before it is written or reused while a kernel still reads it
        stream = torch.cuda.current_stream(self.device).cuda_stream
        holds = (tuple(self._rows[s] for s in seqs), tuple(seqs), self.alloc.version, self.SHARED_MIN_TILES, stream)
        if self._plan is None or self._plan[0] != holds:
            slots = [self.alloc.slots(s) for s in seqs]
            counts = [len(s) for s in slots]
            max_pg = max(1, max(counts))
            table = torch.tensor([s + [0] * (max_pg - len(s)) for s in slots], dtype=torch.int32).to(self.device)
            ints = torch.tensor(counts, dtype=torch.int32).to(self.device)
            groups = ws = None
            if self.sliding_window is None and self.geom.layout == 1:
                members, pages = self._prefix_groups(slots)
                if members:
                    own = sum(counts) - sum(len(m) * p for m, p in zip(members, pages))
                    groups = K.PrefixGroups(self.geom, n, members, pages, self.device, own_pages=own)
                    ws = K.decode_shared_workspace(self.geom, n, groups, self.device)
                    if self._rope_frag is None or self._rope_frag[0] != stream or self._rope_frag[1].shape[0] < groups.max_prefix:
                        most = self.rope_cos.shape[0] // 128
                        self._rope_frag = (stream, K.rope_fragments(self.rope_cos, self.rope_sin, min(most, 2 * groups.max_prefix)))
            self._plan = (holds, table, ints, torch.tensor(holds[0], device=self.device), groups, ws, max_pg if any(counts) else 0)
        _, table, n_pages, rows, groups, ws, max_walk = self._plan
        tail = torch.tensor([self._tail[s] for s in seqs], dtype=torch.int32).to(self.device)
        basis16 = self.basis_f16 if self.basis_f16 is not None else torch.zeros(self.geom.h_kv * HEAD_DIM, self.geom.rank, dtype=torch.float16,
                                                                                 device=self.device)
        tails = (self.k_win[rows].contiguous(), self.v_win[rows].contiguous(), tail)
        last = (self.v_lut, self.signs, self.sm_scale)
        if groups is not None:
            return K.k2b_decode_shared(self.pool, q, basis16, table, n_pages, max_walk, groups, self.rope_cos, self.rope_sin, self._rope_frag[1], *tails, *last,
                                       ws, out=out)
        if (n, stream) not in self._ws:
            self._ws[n, stream] = K.decode_workspace(self.geom, n, table.shape[1], self.device)
        ws = self._ws[n, stream]
        if self.sliding_window is not None:
            return K.k2b_decode_sliding(self.pool, q, basis16, table, n_pages, max_walk, self.rope_cos, self.rope_sin, *tails, *last, ws,
                                        self.sliding_window, self.sinks, out=out)
        return K.k2b_decode(self.pool, q, basis16, table, n_pages, max_walk, self.rope_cos, self.rope_sin, *tails, *last, ws, out=out)

    # ---- accounting -------------------------------------------------------------------------
    def bytes_per_slot(self) -> int:
        g = self.geom
        return g.h_kv * K.page_block_bytes(g) + g.n_coef_heads * K.coef_block_bytes(g)

    def memory_stats(self) -> dict:
        """Bytes held for the live sequences, from the allocator's own counts: packed pages actually owned, plus each
        sequence's three fp16 window rows.  `per_sequence_bytes` is the steady-state marginal cost of one more sequence of
        the mean live length (bmx measures the same quantity by co-residency, scripts/batch_oom_sweep.py:112-178)."""
        n = len(self._rows)
        window = 3 * self.geom.h_kv * self.tail_cap * HEAD_DIM * 2
        pages = self.alloc.in_use * self.bytes_per_slot()
        tokens = sum(self.seq_len(s) for s in self._rows)
        dense = 2 * self.geom.h_kv * HEAD_DIM * 2  # fp16 K and V per token
        return {"sequences": n, "slots_in_use": self.alloc.in_use, "slots_total": self.alloc.n_slots, "peak_slots_in_use": self.alloc.peak_in_use,
                "packed_page_bytes": pages, "window_bytes": n * window, "per_sequence_bytes": (pages + n * window) / n if n else 0.0,
                "tokens": tokens, "bytes_per_token": (pages + n * window) / tokens if tokens else 0.0, "dense_fp16_bytes_per_token": dense}
