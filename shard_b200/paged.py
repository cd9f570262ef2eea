"""`PagedCache`: keys and values of many sequences at once, in pages of 4-bit codes.

Where `Cache` holds one sequence and compresses it after its prefill, this one holds every token in 4.25 bits a
value from the moment it arrives, and hands memory out in pages of a few tokens, so that sequences of any length
come, grow and go independently.  It keeps the pages' books on the host; the arithmetic is in `ops.paged_append`,
`ops.paged_attn` and `ops.paged_read_back`.

    cache = PagedCache(num_layers, n_kv_heads, n_pages, max_seqs, max_len, rope_inv_freq)
    a, b = cache.add(), cache.add()
    cache.begin({a: 700, b: 90})                      # two prompts, one behind the other
    for i, layer in enumerate(layers):                # q (790, n_q, 128), k and v (790, n_kv_heads, 128)
        out = cache.attend(i, q, k, v)
    cache.begin({a: 1, b: 5})                         # the next token of one, five drafted ones of the other
    ...
    cache.truncate(b, cache.length(b) - 3)            # of which two were accepted
    cache.remove(a)
"""
from __future__ import annotations

import torch

from . import ops
from ._lib import PAGED_MAX_SEQS, ShardError
from .rope import rope_table

_PROBLEMS = ((1, "a token had no page"), (2, "a position lies behind the rotation table"),
             (4, "a sequence had more new tokens than the call allowed"), (8, "a launch gave up on a bounded wait; its output is undefined"))


class PagedCache:
    """num_layers layers of n_pages pages, for up to max_seqs sequences of up to max_len tokens.  Positions
    are rotated by `rope_inv_freq` (64 frequencies), or by `rope` (max_len, 128), a table as `rope.rope_table`
    makes it.  All calls of a step go to the current stream."""

    def __init__(self, num_layers, n_kv_heads, n_pages, max_seqs, max_len, rope_inv_freq=None, *, rope=None, page_size=64,
                 device=None):
        if num_layers < 1 or n_pages < 1 or max_seqs < 1 or max_len < 1:
            raise ShardError("a paged cache needs at least one layer, page, sequence and token")
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.page_size, self.max_len, self.n_pages = page_size, max_len, n_pages
        self.width = -(-max_len // page_size)
        one = ops.paged_pool(n_pages, n_kv_heads, page_size, self.device) if num_layers == 1 else None
        if one is None:
            shape = ops.paged_pool(1, n_kv_heads, page_size, self.device).shape
            self.pools = torch.zeros(num_layers, n_pages, *shape[1:], dtype=torch.uint8, device=self.device)
        else:
            self.pools = one.unsqueeze(0)
        if rope is None:
            if rope_inv_freq is None:
                raise ShardError("a paged cache needs rope_inv_freq or a rotation table")
            rope = rope_table(max_len, rope_inv_freq.float().to(self.device))
        if tuple(rope.shape) != (rope.shape[0], ops.HD) or rope.shape[0] < max_len:
            raise ShardError(f"the rotation table must have {max_len} rows of 128")
        self.rope = rope.to(self.device, torch.float32).contiguous()
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._free = list(range(n_pages - 1, -1, -1))
        self._slots = [None] * max_seqs             # pages of the sequence in each slot
        self._lens = [0] * max_seqs
        self._batch = None

    # ---- sequences ----------------------------------------------------------------------------
    def add(self):
        """A new, empty sequence; returns its number."""
        for i, pages in enumerate(self._slots):
            if pages is None:
                self._slots[i], self._lens[i] = [], 0
                return i
        raise ShardError(f"all {len(self._slots)} sequences are in use")

    def remove(self, seq):
        """Forgets a sequence; its pages are free for calls that are made from now on."""
        self._free.extend(reversed(self._pages(seq)))
        self._slots[seq], self._lens[seq], self._batch = None, 0, None

    def truncate(self, seq, tokens):
        """Keeps a sequence's first `tokens` tokens and forgets the others (drafted ones that were not accepted); pages
        that hold none of the first are free for calls that are made from now on.  begin() comes before the next step."""
        pages, tokens = self._pages(seq), int(tokens)
        if not 0 <= tokens <= self._lens[seq]:
            raise ShardError(f"sequence {seq} has {self._lens[seq]} tokens and cannot keep {tokens}")
        kept = -(-tokens // self.page_size)
        self._free.extend(reversed(pages[kept:]))
        del pages[kept:]
        self._lens[seq], self._batch = tokens, None

    def length(self, seq):
        self._pages(seq)
        return self._lens[seq]

    def _pages(self, seq):
        if not 0 <= seq < len(self._slots) or self._slots[seq] is None:
            raise ShardError(f"there is no sequence {seq}")
        return self._slots[seq]

    @property
    def free_pages(self):
        return len(self._free)

    # ---- a step -------------------------------------------------------------------------------
    def begin(self, new):
        """The next calls deal with new[seq] new tokens of each sequence, whose rows follow one another in
        the dictionary's order.  Takes the pages that they need; if those are not there, nothing has changed."""
        new = {seq: int(n) for seq, n in new.items()}
        if len(new) > PAGED_MAX_SEQS:
            raise ShardError(f"a call takes up to {PAGED_MAX_SEQS} sequences (got {len(new)})")
        self._not_capturing("begin")
        need = 0
        for seq, n in new.items():
            pages, total = self._pages(seq), self._lens[seq] + n
            if n < 0 or total > self.max_len:
                raise ShardError(f"sequence {seq} cannot have {n} more tokens: it has {self._lens[seq]} of at most {self.max_len}")
            need += max(0, -(-total // self.page_size) - len(pages))
        if need > len(self._free):
            raise ShardError(f"{need} pages are needed and {len(self._free)} are free")
        for seq, n in new.items():
            pages = self._slots[seq]
            self._lens[seq] += n
            while len(pages) * self.page_size < self._lens[seq]:
                pages.append(self._free.pop())
        self._batch = self._tables(list(new), list(new.values()))

    def _not_capturing(self, what):
        # (a replay would copy these tables from memory that has long been something else)
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise ShardError(f"{what}() copies tables from the host: call it outside a graph's capture (ops.paged_* follow tables of your own)")

    def _tables(self, seqs, new):
        """(page_table, cu, lens, rows, max_new) on the device, by one copy."""
        n, width = len(seqs), max([len(self._slots[s]) for s in seqs], default=0)
        rows = sum(new)
        flat = [0]
        for k in new:
            flat.append(flat[-1] + k)
        flat += [self._lens[s] for s in seqs]
        for s in seqs:
            flat += self._slots[s] + [-1] * (width - len(self._slots[s]))
        host = torch.tensor(flat, dtype=torch.int32)
        dev = (host.pin_memory() if self.device.type == "cuda" else host).to(self.device, non_blocking=True)
        cu, lens, table = dev.split([n + 1, n, n * width])
        return table.view(n, width), cu, lens, rows, max(new, default=0)

    def _current(self):
        if self._batch is None:
            raise ShardError("begin() says which tokens a call deals with")
        return self._batch

    def append(self, layer, k, v, q=None):
        """Rotates and stores the new tokens' keys and values (rows, heads, 128) of a layer; returns the
        queries, rotated, if there are any."""
        table, cu, lens, rows, _ = self._current()
        if k.shape[0] != rows:
            raise ShardError(f"begin() announced {rows} tokens (got {k.shape[0]})")
        return ops.paged_append(k, v, self.pools[layer], table, cu, lens, self.rope, q=q, status=self.status)

    def attend(self, layer, q, k, v, scale=None, lse=None):
        """`append`, and the attention of the new tokens over their sequences: (rows, n_q, 128)."""
        q = self.append(layer, k, v, q)
        table, cu, lens, _, max_new = self._batch
        return ops.paged_attn(q, self.pools[layer], table, cu, lens, scale=scale, max_new=max_new, lse=lse, status=self.status)

    def read_back(self, layer, seq, dtype=torch.float16):
        """Keys (rotated) and values of a sequence as the cache holds them, (1, n_kv_heads, tokens, 128) like
        `Cache.layers[i].keys`."""
        n = self.length(seq)
        self._not_capturing("read_back")
        table, cu, lens, rows, _ = self._tables([seq], [n])
        k, v = ops.paged_read_back(self.pools[layer], table, cu, lens, rows, dtype, status=self.status)
        return k.transpose(0, 1).unsqueeze(0), v.transpose(0, 1).unsqueeze(0)

    def check(self):
        """Raises what a kernel of an earlier call found wrong with its tables (waits for the current stream)."""
        word = int(self.status)
        if word:
            self.status.zero_()
            raise ShardError("paged cache: " + "; ".join(text for bit, text in _PROBLEMS if word & bit))

    def memory_bytes(self):
        """Bytes of the pages that sequences hold."""
        used = self.n_pages - len(self._free)
        return used * self.pools[:, 0].numel()

    def fp16_equivalent_bytes(self):
        """What the sequences' tokens would take as fp16 keys and values."""
        tokens = sum(n for n, pages in zip(self._lens, self._slots) if pages is not None)
        return tokens * self.pools.shape[0] * self.pools.shape[2] * 2 * ops.HD * 2
