"""The caller side of the sparse layer-step.

``Attention`` routes a layer's post-RoPE q/k/v the way the reference's
``Attention.forward`` does in sparse mode (nanovllm/layers/attention.py:
64-99): verify mode -> ``verify_tokens``; the first prefill chunk -> dense
causal attention within the chunk, then ``prefill_first``; later prefill
chunks -> ``prefill_chunk``; one decode token -> ``decode``.  The reference
runs the first chunk through flash-attention; here it is
``M12LayerRuntime.dense_prefill`` on this library's matrix-core kernel.

``attach_m12_runtimes`` is the wiring of ``ModelRunner.allocate_kv_cache``
for the M12 runtime (nanovllm/engine/model_runner.py:125-183): every module
that has ``k_cache`` / ``v_cache`` gets a layer id, zero paged blocks and an
``M12LayerRuntime``.  All layers share one HBM store.

``Context`` / ``get_context`` / ``set_context`` / ``reset_context`` carry the
per-step batch description with the fields of nanovllm/utils/context.py, so a
model runner that sets the context before each forward drives both.

Without an enabled runtime a layer attends densely over its paged cache, if
``attach_paged_cache`` gave it one (the reference's path with the feature off,
attention.py:100-119): several sequences at once, whose tokens are written to
``slot_mapping`` and attend to all keys of their sequence (``block_tables``,
``context_lens``), one token each, several in order (``cu_seqlens_q``), or drafted trees
(``tree_masks``).  A layer with neither raises.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import nn

from .paged import PagedKV, append_paged, attend_paged, new_paged_kv
from .sparse.m12_runtime import M12Config, M12LayerRuntime
from .store import SparseKVStore


@dataclass(slots=True)
class Context:
    """Per-step batch description (field names of nanovllm/utils/context.py:5-14)."""
    is_prefill: bool = False
    cu_seqlens_q: torch.Tensor | None = None
    cu_seqlens_k: torch.Tensor | None = None
    max_seqlen_q: int = 0
    max_seqlen_k: int = 0
    slot_mapping: torch.Tensor | None = None
    context_lens: torch.Tensor | None = None
    block_tables: torch.Tensor | None = None


@dataclass(slots=True)
class TreeContext(Context):
    """A step of drafted trees: the masks of their tokens (paged.tree_masks)."""
    tree_masks: torch.Tensor | None = None


_CONTEXT = Context()


def get_context() -> Context:
    return _CONTEXT


def set_context(is_prefill, cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q=0, max_seqlen_k=0,
                slot_mapping=None, context_lens=None, block_tables=None, tree_masks=None) -> None:
    global _CONTEXT
    fields = (is_prefill, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, slot_mapping, context_lens,
              block_tables)
    _CONTEXT = Context(*fields) if tree_masks is None else TreeContext(*fields, tree_masks)


def reset_context() -> None:
    global _CONTEXT
    _CONTEXT = Context()


class Attention(nn.Module):
    """One attention layer's entry point (constructor of nanovllm/layers/attention.py:47-61)."""

    def __init__(self, num_heads: int, head_dim: int, scale: float, num_kv_heads: int):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.k_cache = self.v_cache = torch.tensor([])
        self.layer_id = None
        self.sparse_rt = None
        self.paged_cache: PagedKV | None = None

    def dense(self) -> PagedKV | None:
        """The paged cache that this step's tokens attend over, or None in sparse mode."""
        rt = self.sparse_rt
        return None if rt is not None and rt.enabled else self.paged_cache

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """q [T, Hq, D], k/v [T, Hkv, D] bf16 -> [T, Hq, D] bf16."""
        context = get_context()
        rt = self.sparse_rt
        if rt is None or not rt.enabled:
            if self.paged_cache is None:
                raise NotImplementedError(
                    "the layer has neither an enabled sparse runtime nor a paged cache: attach an M12LayerRuntime "
                    "as sparse_rt (attach_m12_runtimes) or a cache (attach_paged_cache)")
            append_paged(self.paged_cache, k, v, self.slots(context))
            return self.attend(q, context)
        if rt.verify_mode:
            return rt.verify_tokens(q, k, v, q.device)
        assert q.shape[0] == (context.max_seqlen_q or q.shape[0]) or context.is_prefill
        if context.is_prefill:
            if rt.prefill_len == 0:
                o = rt.dense_prefill(q, k, v, scale=self.scale)
                rt.prefill_first(q, k, v)
                return o
            return rt.prefill_chunk(q, k, v, q.device)
        assert q.shape[0] == 1, "sparse decode supports a single query token"
        assert context.block_tables is None, "sparse decode must not use paged block tables"
        assert self.k_cache.numel() == 0, "sparse mode must allocate zero paged blocks"
        return rt.decode(q, k, v, q.device)


    @staticmethod
    def slots(context: Context) -> torch.Tensor:
        if context.slot_mapping is None:
            raise ValueError("dense attention needs the step's slot_mapping (set_context)")
        return context.slot_mapping

    def attend(self, q: torch.Tensor, context: Context) -> torch.Tensor:
        """Attention over the paged cache, this step's keys and values among it."""
        c = context
        lengths = c.context_lens
        if lengths is None and c.cu_seqlens_k is not None:
            lengths = c.cu_seqlens_k[1:] - c.cu_seqlens_k[:-1]
        if c.block_tables is None or lengths is None:
            raise ValueError("dense attention needs the step's block_tables and context_lens (set_context)")
        ragged = c.cu_seqlens_q is not None
        return attend_paged(q, self.paged_cache, c.block_tables, lengths, starts=c.cu_seqlens_q,
                            max_new=(c.max_seqlen_q or None) if ragged else None,
                            tree=getattr(c, "tree_masks", None), scale=self.scale)


def attach_paged_cache(model: nn.Module, pages: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16,
                       device=None) -> list[PagedKV]:
    """Give every Attention of `model` a layer id and a paged cache of bf16 values or int8
    codes, and no sparse runtime (the paged blocks of model_runner.py:125-175).
    The caches of a model are pieces of one pair of allocations."""
    layers = [m for m in model.modules() if isinstance(m, Attention)]
    if not layers:
        raise ValueError("model has no attention modules")
    if len({(m.num_kv_heads, m.head_dim) for m in layers}) > 1:
        raise ValueError("the model's attention modules differ in their heads")
    if device is None:
        device = next((p.device for p in model.parameters()), torch.device("cuda"))
    held = new_paged_kv(len(layers) * pages, layers[0].num_kv_heads, page_size, layers[0].head_dim, dtype, device)
    caches = []
    for layer_id, module in enumerate(layers):
        mine = PagedKV(*(None if t is None else t[layer_id * pages:(layer_id + 1) * pages] for t in held))
        module.layer_id = layer_id
        module.paged_cache = mine
        module.k_cache, module.v_cache = mine.k, mine.v
        module.sparse_rt = None
        caches.append(mine)
    return caches


def attach_m12_runtimes(model: nn.Module, cfg: M12Config, device=None) -> list[M12LayerRuntime]:
    """Give every attention module of `model` its layer id, zero paged blocks and an
    M12LayerRuntime over one shared HBM store (model_runner.py:125-183)."""
    layers = [m for m in model.modules() if hasattr(m, "k_cache") and hasattr(m, "v_cache")]
    if not layers:
        raise ValueError("model has no attention modules (nothing with k_cache / v_cache)")
    B = cfg.block_size
    store = SparseKVStore(
        len(layers), num_heads=cfg.num_heads, num_kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim,
        block_size=B, r=cfg.r, cap_blocks=(cfg.max_model_len + B - 1) // B,
        sink_tokens=cfg.sink_tokens, recent_tokens=cfg.recent_tokens, kv_format=cfg.kv_format,
        device=device, history_tier=cfg.history_tier)
    runtimes = []
    for layer_id, module in enumerate(layers):
        module.layer_id = layer_id
        module.k_cache = torch.empty(0)
        module.v_cache = torch.empty(0)
        module.paged_cache = None
        module.sparse_rt = M12LayerRuntime(layer_id, cfg, store=store)
        runtimes.append(module.sparse_rt)
    return runtimes


__all__ = ["Attention", "Context", "TreeContext", "attach_m12_runtimes", "attach_paged_cache", "get_context",
           "reset_context", "set_context"]
