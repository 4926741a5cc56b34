"""A decoder's self-attention keys and values in pages (the dense counterpart: TransformerDecoder.create_decoding_internal_cache; the reference
concatenates per-layer tensors, neurst/layers/attentions/multi_head_attention.py:254-290, and gathers all of them behind every step of a
beam search, neurst/layers/search/beam_search.py:409-410).

Rows (hypotheses, requests) may have different lengths.  Which pages a row holds, how long it is and which pages are free lives on the device
and is brought forward by kernels: nothing of a step depends on a value the host reads back.  Behind a re-ordering rows SHARE the pages they have
in common and only their partly filled last pages are copied, where the dense cache gathers every position of every layer.
"""
import torch

from neurst_amd import kernels as K


class PagedKVCache(object):
    """extend() once per step (pages and slots for the new tokens of every row), then per layer append() and attend(); reorder() between
    steps.  static: the state stays in the same buffers (what a captured graph needs)."""

    def __init__(self, num_layers, rows, num_heads, head_dim, max_length, page_size, dtype, device, static=False):
        if page_size < 1 or max_length < 1:
            raise ValueError(f"a paged cache needs pages and rows of at least one token, got {page_size} and {max_length}")
        if head_dim > 256:
            raise ValueError(f"the attention over pages takes heads of up to 256 elements, got {head_dim}")
        self.rows, self.page_size, self.max_length, self.static = rows, int(page_size), int(max_length), bool(static)
        self.width = -(-self.max_length // self.page_size)             # pages of a row
        pages = rows * (self.width + 1)                                # every row filled to the end, and one spare page each
        self.pool = torch.zeros(2 * num_layers, pages, self.page_size, num_heads * head_dim, dtype=dtype, device=device)
        heads = self.pool.view(2 * num_layers, pages, self.page_size, num_heads, head_dim)
        self.layers = [(heads[2 * i], heads[2 * i + 1]) for i in range(num_layers)]
        self.num_heads, self.head_dim = num_heads, head_dim
        self._pages = torch.arange(pages, dtype=torch.int32, device=device)
        self._one_each = torch.ones(rows, dtype=torch.int32, device=device)
        self.free = self._pages[rows:]
        self.table = torch.full((rows, self.width), -1, dtype=torch.int32, device=device)
        self.spare = self._pages[:rows].clone()
        self.seq_lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.cursor = torch.zeros(1, dtype=torch.int32, device=device)
        self.slots = None
        self.len = 0                                                   # the host's bound of the longest row; exact while all rows grow alike

    def reset(self):
        """Every page free again, every row empty."""
        self.table.fill_(-1)
        self.spare.copy_(self._pages[:self.rows])
        self.rewind(0)

    def rewind(self, length):
        """Takes back the last extend() of a cache whose rows are all equally long (and were not re-ordered since): every row has
        `length` tokens.  The pages that were taken are taken again by the next extend()."""
        self.seq_lens.fill_(length)
        self.cursor.fill_(self.rows * -(-length // self.page_size))
        self.len = length

    def _keep(self, name, value):
        if self.static:
            getattr(self, name).copy_(value)
        else:
            setattr(self, name, value)

    def extend(self, new_lens=None, longest=1, max_tokens=None, length=None):
        """One new token for every row; or new_lens [rows] int32 on the device, of which none is larger than `longest` and whose sum is at
        most max_tokens (rows * longest).  The tokens' rows follow each other row after row in append().
        length: what no row is longer than afterwards, where the host knows.  The lengths live on the device, so without it every call is
        taken to lengthen the longest row by `longest`: rows that grow in turn then seem full before they are (tokens that pass the
        pages of a row, because `length` was too small, are dropped: nst_paged_plan)."""
        after = self.len + longest if length is None else length
        if after < 0:
            raise ValueError(f"rows of at most {after} tokens")
        if after > self.max_length:
            raise RuntimeError(f"attention cache of {self.max_length} positions is full")
        self.slots, seq_lens, _, cursor = K.paged_plan(self.seq_lens, self._one_each if new_lens is None else new_lens, self.table, self.free,
                                                       self.cursor, self.page_size, self.rows * longest if max_tokens is None else max_tokens)
        self._keep("seq_lens", seq_lens)
        self._keep("cursor", cursor)
        self.len = after

    def append(self, layer, k, v):
        """k, v [tokens, num_heads, head_dim] of the step's tokens into their slots."""
        K.paged_append(k, v, *self.layers[layer], self.slots)

    def attend(self, layer, q):
        """q [rows, num_heads, head_dim] over everything appended so far -> [rows, num_heads, head_dim]."""
        return K.paged_attention(q, *self.layers[layer], self.table, self.seq_lens, max_len=self.len)

    def reorder(self, parents):
        """Row r continues row parents[r] (int64), which is as long."""
        table, spare = K.paged_reorder(self.pool, self.table, self.seq_lens, parents, self.spare)
        self._keep("table", table)
        self._keep("spare", spare)
