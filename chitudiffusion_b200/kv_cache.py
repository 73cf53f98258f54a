"""A paged key/value cache with its bookkeeping: pools, page tables and lengths of a batch of sequences.

The arithmetic is in ``ops.kv_cache_append`` and ``ops.attn_fwd_cache``; this class allots pages, keeps the tables on the GPU up to
date and hands both operators what they need; no call waits for the GPU.  Generation frame by frame (the frames made so far are the
keys of the next chunk), a prompt taken in chunks and single tokens are the same two calls::

    cache = PagedKVCache(batch=2, num_heads=8, max_tokens=4096, device="cuda")
    q = cache.append(k, v, q=q, rope_table=table)        # [B, S, H, 128], or packed tokens and new_lens=[...]
    out, lse = cache.attend(q, causal=True)

Pages of 8 bits (the default) hold e4m3 codes with a power-of-two scale per page and head: half the memory of 16-bit ones and
about half the time of a single-token step (64 sequences of up to 16300 keys, 8 key heads: 205 us against 368).  (The reference
keeps the gathered keys of a layer as 16-bit tensors, modules/attention/image_cp_attention.py:131-205.)
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from . import ops


class PagedKVCache:
    """Keys and values of ``batch`` sequences in pages of ``page_size`` tokens.

    ``max_tokens`` bounds each sequence; ``num_pages`` (default: enough for all of them at that length) the pool they share.
    ``dtype`` is ``torch.float8_e4m3fn``, bf16 or fp16.  An append that raises, for want of a free page or anything else, leaves the cache
    holding what it held.
    Calls that are to be captured into a graph use the operators directly, on :attr:`tensors` (allotting pages is host work).
    """

    def __init__(self, batch: int, num_heads: int, max_tokens: int, *, page_size: int = 64, dtype: torch.dtype = torch.float8_e4m3fn,
                 num_pages: Optional[int] = None, device=None):
        if batch < 1 or num_heads < 1 or max_tokens < 1:
            raise ValueError("PagedKVCache: batch, num_heads and max_tokens must be positive")
        if page_size not in ops._CACHE_PAGES:
            raise NotImplementedError(f"PagedKVCache: page_size must be one of {ops._CACHE_PAGES} (got {page_size})")
        if dtype not in (torch.float8_e4m3fn, torch.bfloat16, torch.float16):
            raise NotImplementedError(f"PagedKVCache: pages hold float8_e4m3fn, bf16 or fp16 (got {dtype})")
        width = -(-max_tokens // page_size)
        num_pages = batch * width if num_pages is None else int(num_pages)
        if num_pages < 1:
            raise ValueError("PagedKVCache: num_pages must be positive")
        device = torch.device("cuda" if device is None else device)
        self.batch, self.num_heads, self.page_size, self.max_tokens, self.dtype = batch, num_heads, page_size, max_tokens, dtype
        shape = (num_pages, num_heads, page_size, ops._CACHE_HEAD_DIM)  # a head's page is contiguous
        self._k, self._v = (torch.empty(shape, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
        self._k_scale = self._v_scale = None
        if dtype == torch.float8_e4m3fn:
            self._k_scale, self._v_scale = (torch.ones(num_pages, num_heads, dtype=torch.float32, device=device) for _ in range(2))
        self._table = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        self._lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self._cu = torch.zeros(batch + 1, dtype=torch.int32, device=device)
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(batch)]
        self._host_lens = [0] * batch
        self._new = [0] * batch

    # ------------------------------------------------------------------ what the operators take
    @property
    def tensors(self) -> dict:
        """Arguments of the operators that belong to the cache."""
        return dict(k_cache=self._k, v_cache=self._v, block_table=self._table, kv_lens=self._lens, cu_seqlens=self._cu,
                    k_scale=self._k_scale, v_scale=self._v_scale)

    @property
    def lens(self) -> List[int]:
        return list(self._host_lens)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    # ------------------------------------------------------------------ bookkeeping
    def _allot(self, new: Sequence[int]) -> None:
        after = [a + n for a, n in zip(self._host_lens, new)]
        if any(n < 0 for n in new) or max(after) > self.max_tokens:
            raise ValueError(f"PagedKVCache: sequences of {after} tokens, at most {self.max_tokens} fit")
        want = [-(-n // self.page_size) - len(pages) for n, pages in zip(after, self._pages)]
        if sum(w for w in want if w > 0) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {sum(w for w in want if w > 0)} pages are needed, {len(self._free)} are free")
        rows, cols, ids = [], [], []
        for b, w in enumerate(want):
            for _ in range(w):
                rows.append(b)
                cols.append(len(self._pages[b]))
                ids.append(self._free.pop())
                self._pages[b].append(ids[-1])
        if ids:
            rows, cols, ids = self._on_device(rows + cols + ids).view(3, -1)
            self._table[rows, cols] = ids
        self._set_new(list(new))
        if len(set(new)) == 1:
            self._lens += new[0]
        else:
            self._lens.copy_(self._on_device(after))
        self._host_lens = after

    def _on_device(self, values: List[int]) -> torch.Tensor:
        """``values`` where the cache is, without a wait for the GPU: from pinned memory, which torch uses again once the
        copy is through."""
        if self._table.device.type == "cpu":
            return torch.tensor(values, dtype=torch.int32)
        return torch.tensor(values, dtype=torch.int32, pin_memory=True).to(self._table.device, non_blocking=True)

    def _set_new(self, new: List[int]) -> None:
        if new != self._new:
            self._new = []  # (nothing that another call could match, should the copy fail)
            self._cu.copy_(self._on_device(self._ends(new)))
            self._new = new

    @staticmethod
    def _ends(lens: Sequence[int]) -> List[int]:
        ends = [0]
        for n in lens:
            ends.append(ends[-1] + n)
        return ends

    def truncate(self, sequence: int, tokens: int = 0) -> None:
        """Forget what ``sequence`` holds behind its first ``tokens`` tokens; its pages behind them are free again."""
        if not 0 <= sequence < self.batch or not 0 <= tokens <= self._host_lens[sequence]:
            raise ValueError("PagedKVCache: no such sequence, or it holds fewer tokens")
        pages, keep = self._pages[sequence], -(-tokens // self.page_size)
        if len(pages) > keep:
            # (they may soon be another sequence's: a caller that advances kv_lens by itself finds no page here)
            self._table[sequence, keep:len(pages)].fill_(-1)
        while len(pages) > keep:
            self._free.append(pages.pop())
        self._host_lens[sequence] = tokens
        self._lens[sequence].fill_(tokens)  # (assigning a number copies it from the host, with a wait)

    # ------------------------------------------------------------------ the two calls
    def _packed(self, t: torch.Tensor) -> torch.Tensor:
        return t.flatten(0, 1) if t.dim() == 4 else t

    def append(self, k: torch.Tensor, v: torch.Tensor, new_lens: Optional[Sequence[int]] = None, *, q: Optional[torch.Tensor] = None,
               rope_table: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
               interleaved: bool = True) -> Optional[torch.Tensor]:
        """Append ``k, v``: ``[B, S, H, 128]``, ``S`` tokens each, or packed ``[T, H, 128]`` with ``new_lens`` tokens of every
        sequence.  Returns ``q`` rotated (in its own shape) where it is given; see ``ops.kv_cache_append``."""
        if k.dim() == 4:
            if k.shape[0] != self.batch or new_lens is not None:
                raise ValueError(f"PagedKVCache: [B, S, H, 128] has one row per sequence (B = {self.batch}) and takes no new_lens")
            new = [k.shape[1]] * self.batch
        else:
            new = [int(n) for n in new_lens] if new_lens is not None else []
            if len(new) != self.batch or sum(new) > k.shape[0]:
                raise ValueError("PagedKVCache: packed tokens need new_lens, one per sequence, of no more tokens than there are")
        before, before_new = list(self._host_lens), list(self._new)
        try:
            self._allot(new)
            turned = ops.kv_cache_append(self._packed(k), self._packed(v), **self.tensors, positions=positions, rope_table=rope_table,
                                         interleaved=interleaved, q=None if q is None else self._packed(q), max_new=max(new))
        except BaseException:  # (an interrupt or a wrong argument's TypeError leaves no tokens behind either)
            for b, n in enumerate(before):
                self.truncate(b, n)
            self._set_new(before_new)
            raise
        return turned if turned is None or q.dim() == 3 else turned.view(q.shape)

    def attend(self, q: torch.Tensor, *, causal: bool = False, softmax_scale: Optional[float] = None, return_lse: bool = False,
               out: Optional[torch.Tensor] = None, q_lens: Optional[Sequence[int]] = None
               ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """Attention of ``q`` over what the cache holds: the queries of the last :meth:`append`, in its shape, or others
        (``q_lens`` of each sequence, packed; ``[B, S, H, 128]``); see ``ops.attn_fwd_cache``.  The log-sum-exp is ``[Hq, T]``, of
        ``[B, S, H, 128]`` queries ``[B, Hq, S]``."""
        if q.dim() == 4:
            if q.shape[0] != self.batch or q_lens is not None:
                raise ValueError(f"PagedKVCache: [B, S, H, 128] has one row per sequence (B = {self.batch}) and takes no q_lens")
            lens = [q.shape[1]] * self.batch
        else:
            lens = self._new if q_lens is None else [int(n) for n in q_lens]
            if len(lens) != self.batch or min(lens) < 0 or sum(lens) > q.shape[0]:
                raise ValueError("PagedKVCache: packed queries need q_lens, one per sequence, of no more tokens than there are")
        if out is not None and (out.shape != q.shape or not out.is_contiguous()):
            raise ValueError(f"PagedKVCache: out must be contiguous, of q's shape {tuple(q.shape)}")
        args = self.tensors
        if lens != self._new:
            args["cu_seqlens"] = self._on_device(self._ends(lens))
        got, lse = ops.attn_fwd_cache(self._packed(q), **args, softmax_scale=softmax_scale, causal=causal, return_lse=return_lse,
                                      out=None if out is None else self._packed(out), max_q=max(lens), max_kv=max(self._host_lens))
        if q.is_cuda:
            ops.poll_status(q.device)
        if q.dim() == 4:
            B, S, H, _ = q.shape
            got = got.view(q.shape)
            lse = None if lse is None else lse.view(H, B, S).transpose(0, 1).contiguous()
        return got, lse
