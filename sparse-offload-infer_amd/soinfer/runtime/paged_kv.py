"""Several sequences at once over a paged KV cache held in 4 bits.

PagedKV4 owns the pages of every layer, hands them out to sequences, and turns "these sequences get so many new tokens"
into the block table, lengths and offsets that the operators take (soinfer.ops.kv4_append, kv4_read,
kv4_decode_attention, prompt_attention). No reference counterpart: the reference keeps one sequence's binary16 cache of
a fixed length per layer (python/soinfer/runtime/generate.py:276-310).

    cache = PagedKV4(layers, pages, NKV, hd, max_len=4096)
    a, b = cache.add(), cache.add()
    step = cache.step({a: 100, b: 37})                       # two prompts, packed
    q, k = cache.append(layer, step, qkv, qn, kn, cos, sin, NQ, keep_k=True)
    out = cache.prompt(layer, step, q, k, v)                 # causal attention of the packed prompts
    step = cache.step({a: 1, b: 1})                          # a decode step
    out = cache.attend(layer, step, cache.append(layer, step, qkv, qn, kn, cos, sin, NQ))

One page number stands for the same page in every layer, so a step's tables serve them all.
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from .. import ops


@dataclass
class Step:
    """What one batch of new tokens is to the operators. Sequence i of the batch is sequences[i]."""
    sequences: tuple[int, ...]
    new: tuple[int, ...]        # new tokens of each
    lens: tuple[int, ...]       # tokens of each with the new ones
    block_table: torch.Tensor   # int32 [B, blocks of the longest]
    seq_lens: torch.Tensor      # int32 [B]
    cu_seqlens: torch.Tensor    # int32 [B + 1]: the new tokens' rows
    tokens: int                 # rows of all sequences
    max_new: int
    max_len: int


class PagedKV4:
    """num_pages pages of page_size tokens for each of `layers` layers; at most max_len tokens a sequence. group_size:
    dimensions that share a scale (32, 64 or 128, at most head_dim); page_size: a power of two from 16 up (from 64 up the
    attention's addresses are cheaper)."""

    def __init__(self, layers: int, num_pages: int, num_kv_heads: int, head_dim: int, *, max_len: int, group_size: int = 64,
                 page_size: int = 64, device="cuda"):
        if head_dim not in (64, 128, 256) or group_size not in (32, 64, 128) or group_size > head_dim:
            raise ValueError("PagedKV4: head_dim 64, 128 or 256 and group_size 32, 64 or 128, at most head_dim")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError("PagedKV4: page_size must be a power of two from 16 up")
        if layers < 1 or num_pages < 1 or num_kv_heads < 1 or max_len < 1:
            raise ValueError("PagedKV4: layers, num_pages, num_kv_heads and max_len must be positive")
        self.page_size, self.max_len, self.num_pages = page_size, max_len, num_pages
        self.num_kv_heads, self.head_dim, self.group_size = num_kv_heads, head_dim, group_size
        self.device = torch.device(device)

        def pages(shape, dtype):
            return [torch.zeros((num_pages, num_kv_heads, *shape), dtype=dtype, device=self.device) for _ in range(layers)]

        self.k_pages = pages((page_size, head_dim // 2), torch.uint8)
        self.v_pages = pages((page_size, head_dim // 2), torch.uint8)
        self.k_scale = pages((head_dim // group_size, page_size), torch.float16)
        self.v_scale = pages((head_dim // group_size, page_size), torch.float16)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._lens: dict[int, int] = {}
        self._next = 0

    # ---- sequences ------------------------------------------------------------------------------

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        return self._lens[sequence]

    def add(self) -> int:
        """A new, empty sequence."""
        s = self._next
        self._next += 1
        self._pages[s], self._lens[s] = [], 0
        return s

    def free(self, sequence: int) -> None:
        """Gives a sequence's pages back. Work already on the stream still reads them; the pages are written again only by
        later appends on it."""
        self._free.extend(reversed(self._pages.pop(sequence)))
        del self._lens[sequence]

    def step(self, new: dict[int, int]) -> Step:
        """Room for `new` tokens of each sequence (0: attend or read only). Raises RuntimeError, and changes nothing, where
        the pages or max_len do not reach."""
        if not new:
            raise ValueError("PagedKV4.step: no sequences")
        need = 0
        for s, n in new.items():
            if n < 0:
                raise ValueError("PagedKV4.step: token counts must not be negative")
            if self._lens[s] + n > self.max_len:
                raise RuntimeError(f"PagedKV4.step: sequence {s} would hold {self._lens[s] + n} tokens, max_len is {self.max_len}")
            need += -(-(self._lens[s] + n) // self.page_size) - len(self._pages[s])
        if need > len(self._free):
            raise RuntimeError(f"PagedKV4.step: {need} pages needed, {len(self._free)} free")
        for s, n in new.items():
            self._lens[s] += n
            while len(self._pages[s]) * self.page_size < self._lens[s]:
                self._pages[s].append(self._free.pop())
        seqs = tuple(new)
        lens = tuple(self._lens[s] for s in seqs)
        table = np.zeros((len(seqs), max(1, max(len(self._pages[s]) for s in seqs))), np.int32)
        for i, s in enumerate(seqs):
            table[i, :len(self._pages[s])] = self._pages[s]
        cu = np.concatenate([[0], np.cumsum(list(new.values()))]).astype(np.int32)
        # one copy for the three tables
        flat = torch.from_numpy(np.concatenate([table.ravel(), np.asarray(lens, np.int32), cu])).to(self.device)
        t, ln, c = flat.split([table.size, len(seqs), len(seqs) + 1])
        return Step(seqs, tuple(new.values()), lens, t.view(table.shape), ln, c, int(cu[-1]), max(new.values()), max(lens))

    # ---- the operators --------------------------------------------------------------------------

    def _layer(self, layer: int):
        return self.k_pages[layer], self.k_scale[layer], self.v_pages[layer], self.v_scale[layer]

    @staticmethod
    def _need_rows(what: str, step: Step, *rows: torch.Tensor) -> None:
        for x in rows:
            if x.shape[0] < step.tokens:
                raise ValueError(f"PagedKV4.{what}: the step has {step.tokens} rows, got {x.shape[0]}")

    def append(self, layer: int, step: Step, qkv: torch.Tensor, q_norm, k_norm, cos_table: torch.Tensor,
               sin_table: torch.Tensor, num_q_heads: int, eps: float = 1e-6, keep_k: bool = False):
        """ops.kv4_append of the step's rows: the rotated q, or (q, rotated k) with keep_k. Rows past the step's are left out;
        ValueError where rows are missing or a new position is past the tables, as the step's tokens count as cached."""
        self._need_rows("append", step, qkv)
        last = max((ln for n, ln in zip(step.new, step.lens) if n), default=0)
        if min(cos_table.shape[0], sin_table.shape[0]) < last:
            raise ValueError(f"PagedKV4.append: the step needs {last} positions of the RoPE tables, got "
                             f"{cos_table.shape[0]} and {sin_table.shape[0]}")
        k_out = None
        if keep_k:
            k_out = torch.empty((qkv.shape[0], self.num_kv_heads, self.head_dim), dtype=torch.float16, device=qkv.device)
        q = ops.kv4_append(qkv, q_norm, k_norm, cos_table, sin_table, *self._layer(layer), step.block_table, step.seq_lens,
                           step.cu_seqlens, num_q_heads, eps, k_out)
        return (q, k_out) if keep_k else q

    def read(self, layer: int, step: Step):
        """The sequences' whole contexts as binary16, packed: (k, v, cu_k)."""
        cu = np.concatenate([[0], np.cumsum(step.lens)]).astype(np.int32)
        cu_k = torch.from_numpy(cu).to(self.device)
        k, v = ops.kv4_read(*self._layer(layer), step.block_table, step.seq_lens, cu_k, int(cu[-1]))
        return k, v, cu_k

    def attend(self, layer: int, step: Step, q: torch.Tensor, scale: float | None = None) -> torch.Tensor:
        """ops.kv4_decode_attention: one query token of each sequence, q [B, NQ, hd], over its cached tokens."""
        return ops.kv4_decode_attention(q, *self._layer(layer), step.block_table, step.seq_lens, step.max_len, scale)

    def prompt(self, layer: int, step: Step, q: torch.Tensor, k: torch.Tensor | None = None, v: torch.Tensor | None = None,
               scale: float | None = None) -> torch.Tensor:
        """Causal attention of the step's rows. With k and v, the new rows' own (sequences that begin with this step);
        without, over everything cached, read back from the pages (prompts that continue a context)."""
        if k is not None:
            if any(n != ln for n, ln in zip(step.new, step.lens)):
                raise ValueError("PagedKV4.prompt: k and v of the new rows only serve sequences that begin with them")
            self._need_rows("prompt", step, q, k, v)
            cu_k = step.cu_seqlens
        else:
            self._need_rows("prompt", step, q)
            k, v, cu_k = self.read(layer, step)
        return ops.prompt_attention(q, k, v, step.cu_seqlens, cu_k, step.max_new, scale)
