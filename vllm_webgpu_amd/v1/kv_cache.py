"""``PagedKVCache``: the keys and values that a target's layers keep of running requests, in pages.

The reference keeps one contiguous cache a request (``vllm_webgpu/models/llama.py:222-237`` passes positions into
it).  Here every layer has ``num_pages`` pages of ``page_size`` tokens, a request owns pages by number (the same in
every layer), and the kernels read and write them through a block table: ``append`` (with the position
rotation), ``attend`` (drafted trees, prompts' chunks as chains, single tokens), ``keep`` (a verified tree's accepted
nodes move up behind the context).  Values are stored by dimension, [pages, kv_heads, head_dim, page_size]: the order in
which the attention's second product reads them.
"""
from __future__ import annotations

import torch

from .. import ops
from .sample.tree_sampler import DraftTree


class PagedKVCache:
    def __init__(self, num_layers: int, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda") -> None:
        self.page_size, self.num_pages = page_size, num_pages
        self.k = [torch.empty((num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(num_layers)]
        self.v = [torch.empty((num_pages, kv_heads, head_dim, page_size), dtype=dtype, device=device) for _ in range(num_layers)]
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[str, list[int]] = {}

    # ---- pages, on the host

    def reserve(self, req_id: str, num_tokens: int) -> None:
        """Gives a request pages for its first ``num_tokens`` positions."""
        pages = self._pages.get(req_id, [])
        need = (num_tokens + self.page_size - 1) // self.page_size - len(pages)
        if need > len(self._free):
            raise RuntimeError(f"the cache is full: {need} more pages for request {req_id!r}, {len(self._free)} free")
        self._pages[req_id] = pages + [self._free.pop() for _ in range(max(need, 0))]

    def release(self, req_id: str) -> None:
        self._free += reversed(self._pages.pop(req_id, []))

    def block_table(self, req_ids: list[str]) -> torch.Tensor:
        """int32 [B, pages of the longest]; -1 behind a request's last page."""
        pages = [self._pages[r] for r in req_ids]
        width = max((len(p) for p in pages), default=0) or 1
        return torch.tensor([p + [-1] * (width - len(p)) for p in pages], dtype=torch.int32).view(len(pages), width).to(self.k[0].device)

    def slots(self, block_table: torch.Tensor, context_lens: torch.Tensor, tree: DraftTree) -> torch.Tensor:
        """int32 [T]: where the nodes' keys and values go, behind their contexts; -1 (nowhere) past a request's pages."""
        B = len(tree.num_nodes)
        if block_table.dim() != 2 or block_table.shape[0] != B or context_lens.shape != (B,):  # (a device would index past its end)
            raise ValueError(f"block_table must be [{B}, pages] and context_lens [{B}], one row for each tree (got {tuple(block_table.shape)} "
                             f"and {tuple(context_lens.shape)})")
        at = context_lens.long()[tree.requests] + tree.numbers
        i = at // self.page_size
        held = (i >= 0) & (i < block_table.shape[1])
        page = block_table[tree.requests, i.clamp(0, block_table.shape[1] - 1)]
        return torch.where(held & (page >= 0), page * self.page_size + at % self.page_size, -1).int()

    # ---- a layer's step, on the device

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, **rotation) -> torch.Tensor | None:
        """``ops.append_kv`` on the layer's pages (``q``, ``positions``, ``inv_freq``, ...): the rotated queries."""
        return ops.append_kv(k, v, self.k[layer], self.v[layer], slots, **rotation)

    def attend(self, layer: int, q: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor, tree: DraftTree,
               scale: float | None = None) -> torch.Tensor:
        """``ops.tree_attention`` of the nodes, whose keys and values have been appended, over the layer's pages."""
        return ops.tree_attention(q, self.k[layer], self.v[layer], block_table, context_lens, tree.cu_nodes, tree.max_nodes,
                                  visible=tree.visible, scale=scale)

    def keep(self, block_table: torch.Tensor, context_lens: torch.Tensor, path: torch.Tensor) -> None:
        """Moves the visited nodes of ``path`` (``TreeSamplerOutput.path``) up behind their contexts, in every layer: the
        contexts then end ``num_accepted + 1`` positions further."""
        for k, v in zip(self.k, self.v):
            ops.compact_kv(k, v, block_table, context_lens, path)
