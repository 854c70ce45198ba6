"""Serving: the caches of many sequences in pages, and layers with weights of 4 bits.

The reference decodes one batch whose sequences are all of one length, from caches that it concatenates
(lookahead_keys_attention/lookahead_keys_attention.py:166-203).  A server has sequences that come and go, of different lengths,
several of them continuing one prompt.  `PagedCache` holds their rows in pages and does the bookkeeping on the host; the work on
the device is `castle_paged_decode_step`, `castle_write_pages` and `castle_copy_pages`.

    cache = PagedCache(layers=len(model), pages=4096, heads=8, dim_head=64, dtype=torch.bfloat16)
    seq = cache.add()
    for i, layer in enumerate(model):                  # the prompt
        x, c = layer(x, return_next_cache=True)
        cache.write([seq], i, c)
    others = cache.fork(seq, 3)                        # three more continuations of it
    batch = cache.batch([seq, *others])
    for token in range(n):
        for i, layer in enumerate(model):
            x, _ = layer(x, cache=batch.layer(i))      # x (4, 1, dim)
        batch.advance()
    cache.free(seq)
"""
from __future__ import annotations

import weakref

import torch
from torch import nn

from . import ops


class _Pool:
    """Which pages of a pool are free, and how many sequences hold each of the others."""

    __slots__ = ("free", "held")

    def __init__(self, pages):
        self.free = list(range(pages - 1, -1, -1))   # the lowest numbers are taken first
        self.held = [0] * pages

    def take(self):
        page = self.free.pop()
        self.held[page] = 1
        return page

    def drop(self, page):
        self.held[page] -= 1
        if self.held[page] == 0:
            self.free.append(page)

    def moves(self):
        """(source, target) pages that leave the pages in use without gaps."""
        used = [p for p, h in enumerate(self.held) if h]
        gaps = [p for p in range(len(used)) if not self.held[p]]
        high = used[len(used) - len(gaps):]
        return high, gaps

    def moved(self, source, target):
        for s, t in zip(source, target):
            self.held[t], self.held[s] = self.held[s], 0
        self.free = sorted((p for p, h in enumerate(self.held) if h == 0), reverse=True)


class _Sequence:
    __slots__ = ("length", "pages", "u_pages", "batch")

    def __init__(self, length=0, pages=(), u_pages=()):
        self.length, self.pages, self.u_pages = length, list(pages), list(u_pages)
        self.batch = None     # a weak reference to the batch that it is in


class PagedCache:
    """The caches of up to some number of positions, for all layers of a model, in pages of `page_size` positions (a power of two from
    16 to 1024).  Rows of qu, kc and vc never change once they are written, so sequences that continue one prompt share the
    prompt's pages of them; a lookahead key U is rewritten by every token, so U's pages are one sequence's, from a pool of
    `u_pages` (as many as the others' unless given).  A page number stands for that page in every layer.  The host keeps the books; calls on the device go to
    the current stream, in order, and none waits for it.  For one thread and one stream at a time."""

    def __init__(self, layers, pages, heads, dim_head=64, page_size=64, u_pages=None, dtype=torch.bfloat16, device="cuda"):
        u_pages = pages if u_pages is None else u_pages
        if layers < 1 or pages < 1 or u_pages < 1:
            raise ValueError("PagedCache: at least one layer and one page of each kind expected")
        if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError(f"PagedCache: page_size {page_size} is not a power of two from 16 to 1024")
        if dim_head not in (16, 32, 64, 128):
            raise ValueError(f"PagedCache: dim_head {dim_head} not supported (16, 32, 64, 128)")
        self.layers, self.heads, self.dim_head, self.page_size = layers, heads, dim_head, page_size
        self.dtype, self.device = dtype, torch.empty(0, device=device).device
        self._allocate(pages, u_pages)
        self._kv, self._u = _Pool(pages), _Pool(u_pages)
        self._sequences, self._next, self._batches = {}, 0, weakref.WeakSet()

    @torch.inference_mode(False)   # (what a cache made in inference mode holds is written outside it as well)
    def _allocate(self, pages, u_pages):
        new = lambda n: torch.empty(self.layers, n, self.heads, self.page_size, self.dim_head, dtype=self.dtype, device=self.device)  # noqa: E731
        self.U, self.qu, self.kc, self.vc = new(u_pages), new(pages), new(pages), new(pages)

    # ---- the books
    def _of(self, seq) -> _Sequence:
        try:
            return self._sequences[seq]
        except KeyError:
            raise ValueError(f"PagedCache: there is no sequence {seq}") from None

    def length(self, seq) -> int:
        return self._of(seq).length

    def free_pages(self):
        """(pages of qu, kc and vc, pages of U) that no sequence holds."""
        return len(self._kv.free), len(self._u.free)

    def _missing(self, wanted):
        """How many pages each of `wanted` = [(sequence, positions)] lacks."""
        return [max(0, -(-n // self.page_size) - len(s.pages)) for s, n in wanted]

    def _reserve(self, wanted):
        """Pages for `wanted` = [(sequence, positions)]: all of them, or none and an error.  How many each got."""
        need = self._missing(wanted)
        if sum(need) > min(len(self._kv.free), len(self._u.free)):
            raise RuntimeError(f"PagedCache: {sum(need)} more pages needed, {len(self._kv.free)} and {len(self._u.free)} (U) are free")
        for (s, _), k in zip(wanted, need):
            for _ in range(k):
                s.pages.append(self._kv.take())
                s.u_pages.append(self._u.take())
        return need

    def add(self) -> int:
        """A sequence without positions."""
        self._sequences[self._next] = _Sequence()
        self._next += 1
        return self._next - 1

    def free(self, seq):
        """Give a sequence's pages back (those that others share stay theirs).  Its row of a batch takes no part from then on."""
        s = self._of(seq)
        batch = s.batch() if s.batch else None
        del self._sequences[seq]
        if batch is not None:
            batch._drop(seq)
        for p in reversed(s.pages):
            self._kv.drop(p)
        for p in reversed(s.u_pages):
            self._u.drop(p)

    # ---- the device
    def _pools(self, layer):
        if not 0 <= layer < self.layers:
            raise ValueError(f"PagedCache: there is no layer {layer}")
        return self.U[layer], self.qu[layer], self.kc[layer], self.vc[layer]

    @torch.inference_mode(False)
    def _to_device(self, values):
        t = torch.tensor(values, dtype=torch.int32, device="cpu")   # (whatever the default device is)
        return (t.pin_memory() if self.device.type == "cuda" else t).to(self.device, non_blocking=True)

    def _tables(self, sequences, width):
        """(U's table, the others', lengths); a row of length -1 for None."""
        u = [s.u_pages + [-1] * (width - len(s.u_pages)) if s else [-1] * width for s in sequences]
        kv = [s.pages + [-1] * (width - len(s.pages)) if s else [-1] * width for s in sequences]
        return self._to_device(u), self._to_device(kv), self._to_device([s.length if s else -1 for s in sequences])

    def write(self, seqs, layer, cache):
        """A prompt's cache (the one that `Castle(..., return_next_cache=True)` returned for a batch of len(seqs) prompts of one length) as
        layer `layer` of sequences that have no positions, or (the other layers of the same prompt) exactly as many."""
        U, qu, kc, vc = cache
        n = U.shape[2]
        if U.shape[0] != len(seqs) or len(set(seqs)) != len(seqs):
            raise ValueError("PagedCache: a sequence of its own for each of the cache's batch expected")
        pools, sequences = self._pools(layer), [self._of(q) for q in seqs]
        if any(s.length not in (0, n) for s in sequences) or any(s.batch and s.batch() for s in sequences):
            raise ValueError("PagedCache: a prompt can be written only to a sequence without positions that is in no batch")
        if any(self._kv.held[p] > 1 for s in sequences for p in s.pages):
            raise ValueError("PagedCache: a prompt cannot be written to pages that a fork shares")
        if n == 0 or not seqs:
            return
        self._reserve([(s, n) for s in sequences])
        before = [s.length for s in sequences]
        for s in sequences:
            s.length = n
        try:
            u, kv, lengths = self._tables(sequences, max(len(s.pages) for s in sequences))
            ops.castle_write_pages(U, qu, kc, vc, *pools, u, kv, lengths)
        except BaseException:
            for s, k in zip(sequences, before):   # (the pages stay theirs)
                s.length = k
            raise

    def fork(self, seq, count: int = 1):
        """`count` more sequences with the positions of `seq` (between two tokens of all layers): its full pages of qu, kc and vc are shared, the last one, if it is not full, and U's are copied,
        in all layers."""
        s = self._of(seq)
        full, every = s.length // self.page_size, -(-s.length // self.page_size)
        if count * (every - full) > len(self._kv.free) or count * every > len(self._u.free):
            raise RuntimeError(f"PagedCache: {count * (every - full)} and {count * every} (U) more pages needed, {len(self._kv.free)} and {len(self._u.free)} (U) are free")
        new, kv_copies, u_copies = [], ([], []), ([], [])
        for _ in range(count):
            for p in s.pages[:full]:
                self._kv.held[p] += 1
            tail = [self._kv.take() for _ in range(every - full)]
            u = [self._u.take() for _ in range(every)]
            kv_copies[0].extend(s.pages[full:every])
            kv_copies[1].extend(tail)
            u_copies[0].extend(s.u_pages[:every])
            u_copies[1].extend(u)
            q = self.add()
            self._sequences[q] = _Sequence(s.length, s.pages[:full] + tail, u)
            new.append(q)
        try:
            self._copy(kv_copies, u_copies)
        except BaseException:
            for q in new:
                self.free(q)
            raise
        return new

    def _copy(self, kv, u):
        if kv[0]:
            ops.castle_copy_pages([t[i] for t in (self.qu, self.kc, self.vc) for i in range(self.layers)], *kv)
        if u[0]:
            ops.castle_copy_pages(list(self.U), *u)

    def compact(self):
        """Move pages so that those in use are the first ones; returns how many they are (qu, kc and vc; U).  Batches' tables follow."""
        kv, u = self._kv.moves(), self._u.moves()
        self._copy(kv, u)
        new_kv, new_u = dict(zip(*kv)), dict(zip(*u))
        for s in self._sequences.values():
            s.pages = [new_kv.get(p, p) for p in s.pages]
            s.u_pages = [new_u.get(p, p) for p in s.u_pages]
        self._kv.moved(*kv)
        self._u.moved(*u)
        if new_kv or new_u:
            for batch in self._batches:
                batch._upload()
        return len(self._kv.held) - len(self._kv.free), len(self._u.held) - len(self._u.free)

    def resize(self, pages, u_pages=None):
        """Other numbers of pages, in new memory (what was captured with the old one is void); compacts first."""
        u_pages = pages if u_pages is None else u_pages
        used = self.compact()
        if pages < max(1, used[0]) or u_pages < max(1, used[1]):
            raise ValueError(f"PagedCache: {used[0]} and {used[1]} (U) pages are in use")
        old = self.U, self.qu, self.kc, self.vc
        self._allocate(pages, u_pages)
        for new, was, n in zip((self.U, self.qu, self.kc, self.vc), old, (used[1], used[0], used[0], used[0])):
            new[:, :n].copy_(was[:, :n])
        for pool, n in ((self._kv, pages), (self._u, u_pages)):
            pool.held = (pool.held + [0] * n)[:n]
            pool.free = sorted((p for p, h in enumerate(pool.held) if h == 0), reverse=True)

    def batch(self, seqs, size=None, width=None) -> "PagedBatch":
        """Sequences that take their next tokens together; `size` and `width`: rows and pages of a row that the batch's tables have at least (fixed
        addresses for a captured step; rows without a sequence take no part)."""
        return PagedBatch(self, seqs, size, width)


class PagedBatch:
    """Sequences of a `PagedCache` that take tokens together: row i of a step's input is the next token of `seqs[i]` (None: a row without a sequence, which
    takes no part).  `layer(i)` is the `cache=` of the i-th layer's `Castle`; after all layers, `advance()` counts the token.  `u_table`, `table` and
    `lengths` are the tensors that the steps read; they keep their addresses unless a sequence outgrows the width (then new ones take their place, and a
    captured step is void)."""

    def __init__(self, cache: PagedCache, seqs, size=None, width=None):
        self.cache, self.seqs, self._size, self._width = cache, [], size or 0, width or 1
        self.u_table = self.table = self.lengths = self._taking = None
        cache._batches.add(self)
        self.replace(seqs)

    def replace(self, seqs):
        """Other sequences from the next token on, in the same tensors where they fit."""
        seqs, known = list(seqs), [q for q in seqs if q is not None]
        size = max(len(seqs), self._size)
        if size == 0:
            raise ValueError("PagedBatch: at least one sequence, or a size, expected")
        sequences = [self.cache._of(q) for q in known]
        if len(set(known)) != len(known) or any(s.batch and s.batch() not in (None, self) for s in sequences):
            raise ValueError("PagedBatch: a sequence can take one token at a time")
        self.cache._reserve([(s, s.length + 1) for s in sequences])
        for q in self.seqs:
            if q is not None:
                self.cache._of(q).batch = None
        for s in sequences:
            s.batch = weakref.ref(self)
        self.seqs, self._size = seqs + [None] * (size - len(seqs)), size
        self._upload()

    def _sequences(self):
        return [None if q is None else self.cache._of(q) for q in self.seqs]

    @torch.inference_mode(False)
    def _upload(self):
        sequences = self._sequences()
        self._width = max([self._width] + [len(s.pages) for s in sequences if s])
        new = self.cache._tables(sequences, self._width)
        if self.table is not None and self.table.shape == (self._size, self._width):
            for t, n in zip((self.u_table, self.table, self.lengths), new):
                t.copy_(n)
        else:
            self.u_table, self.table, self.lengths = new
        self._taking = (self.lengths >= 0).to(torch.int32)

    def _drop(self, seq):
        self.seqs[self.seqs.index(seq)] = None
        self._upload()

    def layer(self, index) -> "PagedLayer":
        return PagedLayer(self, index)

    def advance(self, leave: bool = False):
        """Every sequence has its token in all layers: count it, and have a place for the next.  Where no page is free for one nothing is counted: free a
        sequence and advance again.  With `leave` every token is counted, one that fills the last free page too, and the sequences that no page is free for leave
        the batch: they stay the cache's, their rows take no part from then on, and `replace` takes them back once there are pages.  Returns those that left."""
        sequences = self._sequences()
        rows = [i for i, s in enumerate(sequences) if s]
        stay, left = rows, []
        if leave:
            stay, room = [], min(self.cache.free_pages())
            for i, k in zip(rows, self.cache._missing([(sequences[i], sequences[i].length + 2) for i in rows])):
                (stay if k <= room else left).append(i)
                room -= k if k <= room else 0
        grown = self.cache._reserve([(sequences[i], sequences[i].length + 2) for i in stay])
        for i in rows:
            sequences[i].length += 1
        gone = [self.seqs[i] for i in left]
        for i in left:
            sequences[i].batch = self.seqs[i] = None
        grown = [i for i, k in zip(stay, grown) if k]
        if any(len(sequences[i].pages) > self._width for i in grown):
            self._upload()
            return gone
        self.lengths += self._taking
        if grown:   # the new pages alone
            at, column, u, kv = self.cache._to_device([grown, [len(sequences[i].pages) - 1 for i in grown], [sequences[i].u_pages[-1] for i in grown],
                                                       [sequences[i].pages[-1] for i in grown]])
            self.u_table[at, column] = u
            self.table[at, column] = kv
        if left:
            at = self.cache._to_device(left)
            self.lengths[at], self._taking[at] = -1, 0
        return gone


class PagedLayer:
    """A layer's share of a batch: the `cache=` of its `Castle`."""

    __slots__ = ("batch", "index")

    def __init__(self, batch, index):
        batch.cache._pools(index)
        self.batch, self.index = batch, index

    @property
    def pools(self):
        return self.batch.cache._pools(self.index)


class Linear4bit(nn.Module):
    """A linear layer with frozen weights of 4 bits (`castle_linear_4bit`); `Linear4bit.from_linear(m)` quantises an `nn.Linear`.  It can take the place
    of any, a `Castle`'s projections among them (`Castle.quantize_4bit`).  Under autocast it takes its rows in autocast's type, as a linear layer does."""

    def __init__(self, in_features, out_features, bias=False, group_size=64, zeros=False, device=None, dtype=None):
        super().__init__()
        if group_size < 32 or group_size & (group_size - 1):
            raise ValueError(f"Linear4bit: group_size {group_size} is not a power of two from 32 up")
        self.in_features, self.out_features, self.group_size = in_features, out_features, group_size
        groups = -(-in_features // group_size)
        self.register_buffer("codes", torch.full((-(-out_features // 16), -(-in_features // 256) * 512), -0x77777778, dtype=torch.int32, device=device))   # (eights)
        self.register_buffer("scales", torch.ones(out_features, groups, device=device, dtype=dtype))
        self.register_buffer("zeros", torch.full((out_features, groups), 8.0, device=device, dtype=dtype) if zeros else None)
        self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype)) if bias else None

    @classmethod
    def from_linear(cls, linear: nn.Linear, group_size=64, zeros=False):
        w = linear.weight.detach()
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, group_size, zeros, device=w.device, dtype=w.dtype)
        m.codes, m.scales, m.zeros = ops.castle_quantize_4bit(w, group_size, zeros)
        if linear.bias is not None:
            m.bias = nn.Parameter(linear.bias.detach().clone(), requires_grad=linear.bias.requires_grad)
        return m.train(linear.training)

    def forward(self, x):
        if x.is_cuda and torch.is_autocast_enabled("cuda") and x.is_floating_point() and x.dtype is not torch.float64:
            x = x.to(torch.get_autocast_dtype("cuda"))
        y = ops.castle_linear_4bit(x, self.codes, self.scales, self.zeros, self.group_size)
        return y if self.bias is None else y + self.bias.to(y.dtype)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, group_size={self.group_size}, zeros={self.zeros is not None}"
