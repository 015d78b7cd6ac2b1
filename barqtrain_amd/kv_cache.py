"""Paged KV-cache objects with the Python surface of the reference's python/barqtrain/kv_cache.py.

``BarqPagedKVCacheLayer`` keeps the reference's names, signatures and value semantics
(kv_cache.py:37-194): ``update`` appends new K/V at each row's current length and returns
``[batch, kv_heads, max_len, head_dim]`` K and V whose slot s of row b is the value last
appended at s, or zero where nothing was written.  The storage behind it is a page pool
(``barqtrain_amd.paged.PagePool``): a block table maps each row's blocks to pages taken from a
free stack on the device, and the returned K/V are materialised contiguously by the gfx950
kernels in one pass that also stores the new tokens.  Lengths are shadowed on the host, so no
call reads the device.

Beyond the reference surface: ``get_max_length`` and the two-argument ``lazy_initialization``
that transformers 5.x declares abstract, ``get_mask_sizes`` accepting an int, an optional
``num_pages`` to size the pool below the dense reservation, ``free_rows``, and
``fused_attention``: ``update`` then only appends and returns views naming the layer, which the
``"barq_paged"`` attention implementation (barqtrain_amd.attention) reads through the block
table instead of a gathered copy.
"""

from __future__ import annotations

import math
import os
from typing import Any, Optional

import torch

from barqtrain_amd._ffi import load_cuda_backend
from barqtrain_amd.attention import paged_kv_view
from barqtrain_amd.paged import (
    KV_QUANT_FP8,
    PagedKVCapacityError,
    PagedKVPoolExhausted,
    PagePool,
    QuantPagePool,
    SlotMap,
    crop_layers,
    map_slots_layers,
    reset_layers,
    select_rows_layers,
)

try:
    from transformers.cache_utils import Cache, CacheLayerMixin
except ImportError:  # pragma: no cover - transformers is a required dependency
    Cache = object  # type: ignore[assignment,misc]
    CacheLayerMixin = object  # type: ignore[assignment,misc]


def _get_cuda_backend():
    """The HIP backend module (kv_cache.py:20-21); a monkeypatch point of the reference tests."""
    return load_cuda_backend()


def _env_enabled(name: str, default: str = "1") -> bool:
    value = os.environ.get(name, default).strip().lower()
    return value not in {"0", "false", "no", "off"}


def _decoder_config(config):
    return config.get_text_config(decoder=True) if hasattr(config, "get_text_config") else config


def _min_paged_kv_cache_len() -> int:
    return int(os.environ.get("BARQTRAIN_PAGED_KV_MIN_CACHE_LEN", "256"))


# Calls that go past a layer's and its pool's methods, straight to the binding or to all layers' pools at
# once, are for these classes: a method that a subclass overrides is called as ever.
_POOL_TYPES = (PagePool, QuantPagePool)


class BarqPagedKVCacheLayer(CacheLayerMixin):
    """A fixed-capacity paged KV-cache layer (reference: kv_cache.py:37-194)."""

    is_sliding = False
    is_compileable = False

    def __init__(self, max_batch_size: int, max_cache_len: int, page_size: int = 16,
                 num_pages: Optional[int] = None, fused_attention: bool = False,
                 kv_quant: Optional[str] = None, residual_window: int = 128):
        super().__init__()
        self.fused_attention = fused_attention
        self.kv_quant = _quant_mode(kv_quant)
        self.residual_window = int(residual_window)
        self.max_batch_size = max_batch_size
        self.max_cache_len = max_cache_len
        self.page_size = page_size
        self.max_blocks = math.ceil(max_cache_len / page_size)
        self.num_pages = num_pages
        self.pool: Optional[PagePool] = None
        self.seq_lens: Optional[torch.Tensor] = None
        self.device: Optional[torch.device] = None
        self.dtype: Optional[torch.dtype] = None
        self.current_batch_size = 0

    # kv_cache.py:53-73.  transformers 5.x passes (key_states, value_states); the reference one.
    def lazy_initialization(self, key_states: torch.Tensor, value_states: Optional[torch.Tensor] = None):
        if key_states.dim() != 4:
            raise ValueError("key_states must have shape [batch, kv_heads, seq, head_dim]")
        batch_size, num_kv_heads, _, head_dim = key_states.shape
        if batch_size > self.max_batch_size:
            raise ValueError(
                f"batch_size={batch_size} exceeds max_batch_size={self.max_batch_size} for paged KV cache"
            )
        self.device = key_states.device
        self.dtype = key_states.dtype
        self.current_batch_size = batch_size
        geometry = dict(max_batch=self.max_batch_size, max_blocks=self.max_blocks, page_size=self.page_size,
                        kv_heads=num_kv_heads, head_dim=head_dim, dtype=self.dtype, device=self.device,
                        num_pages=self.num_pages)
        if self.kv_quant:
            self.pool = QuantPagePool(window=self.residual_window, **geometry)
        else:
            self.pool = PagePool(**geometry)
        self._bind_pool()
        self.is_initialized = True

    def _bind_pool(self) -> None:
        self.keys = self.pool.key_pages
        self.values = self.pool.value_pages
        self.seq_lens = self.pool.seq_lens
        self.block_table = self.pool.block_table
        self.high_water = self.pool.high_water

    # kv_cache.py:93-104
    def _check_append(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        if key_states.shape != value_states.shape:
            raise ValueError("key_states and value_states must have identical shapes")
        if key_states.device != self.device or value_states.device != self.device:
            raise ValueError("key_states and value_states must stay on the cache device")
        if key_states.dtype != self.dtype or value_states.dtype != self.dtype:
            raise ValueError("key_states and value_states must stay in the cache dtype")
        if key_states.size(0) > self.max_batch_size:
            raise ValueError("batch size exceeds the configured paged KV cache capacity")

    def append(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        """Store the new tokens of rows [0, batch) (kv_cache.py:93-118).  A call that would pass
        max_cache_len raises PagedKVCapacityError and changes nothing."""
        self._check_append(key_states, value_states)
        self.pool.append(key_states, value_states, max_length=self.max_cache_len)
        self.current_batch_size = key_states.size(0)

    def current_tensors(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Contiguous ``[current_batch, kv_heads, get_seq_length(), head_dim]`` K and V
        (kv_cache.py:120-133, materialised)."""
        batch = self.current_batch_size or self.max_batch_size
        return self.pool.gather(batch, self.get_seq_length())

    def update(
        self,
        key_states: torch.Tensor,
        value_states: torch.Tensor,
        cache_kwargs: Optional[dict[str, Any]] = None,
        *args,
        **kwargs,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """append + current_tensors (kv_cache.py:135-142), one kernel pass on the GPU.  With
        fused_attention: append, then page views for the "barq_paged" attention."""
        # The usual step: planned and checked in the binding; a call it does not take is checked below,
        # as is one of a subclass or of an object whose append was replaced.
        pool = self.pool
        if (type(pool) in _POOL_TYPES and type(self) is BarqPagedKVCacheLayer and "append" not in self.__dict__
                and self.is_initialized and key_states.dim() == 4 and key_states.size(0) <= self.max_batch_size):
            got = pool.step(key_states, value_states, self.max_cache_len, not self.fused_attention)
            if got is not None:
                self.current_batch_size = key_states.size(0)
                if not self.fused_attention:
                    return got[:2]
                return paged_kv_view(self, key_states, got[2]), paged_kv_view(self, value_states, got[2])
        if self.fused_attention:
            self.append(key_states, value_states)
            seq = self.get_seq_length()
            return paged_kv_view(self, key_states, seq), paged_kv_view(self, value_states, seq)
        self._check_append(key_states, value_states)
        out = self.pool.update(key_states, value_states, max_length=self.max_cache_len)
        self.current_batch_size = key_states.size(0)
        return out

    # kv_cache.py:144-148; transformers 5.x passes the query length as an int
    def get_mask_sizes(self, cache_position) -> tuple[int, int]:
        query_length = cache_position if isinstance(cache_position, int) else cache_position.shape[0]
        return self.get_seq_length() + int(query_length), 0

    # kv_cache.py:150-153, served from the host shadow (no device read)
    def get_seq_length(self) -> int:
        if not self.is_initialized or self.pool is None or self.current_batch_size == 0:
            return 0
        return self.pool.max_len(self.current_batch_size)

    def get_max_cache_shape(self) -> int:
        return self.max_cache_len

    def get_max_length(self) -> int:
        return self.max_cache_len

    # kv_cache.py:158-164
    def crop(self, max_length: int) -> None:
        if not self.is_initialized or self.pool is None:
            return
        if max_length < 0:
            max_length = self.get_seq_length() - abs(max_length)
        max_length = max(max_length, 0)
        self.pool.crop(self.current_batch_size, max_length)

    def _select_rows(self, rows: list[int]) -> None:
        # kv_cache.py:166-183: the cache becomes len(rows) rows, row i a copy of rows[i].  In
        # place with shared pages when the rows fit the pool; else into a larger pool.
        if len(rows) <= self.pool.max_batch:
            self.pool.select_rows(rows)
        else:
            self.pool = self.pool.copy_rows(rows)
            self._bind_pool()
        self.current_batch_size = len(rows)
        self.max_batch_size = self.current_batch_size

    def batch_repeat_interleave(self, repeats: int) -> None:
        if not self.is_initialized or self.current_batch_size == 0:
            return
        self._select_rows([b for b in range(self.current_batch_size) for _ in range(int(repeats))])

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        if not self.is_initialized or self.current_batch_size == 0:
            return
        self._select_rows(_selected_rows(indices, self.current_batch_size))

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        self.batch_select_indices(beam_idx)

    # kv_cache.py:188-194 -- O(metadata): pages are returned, nothing is cleared
    def reset(self) -> None:
        if not self.is_initialized:
            return
        self.pool.reset()
        self.current_batch_size = 0

    def free_rows(self, rows) -> None:
        """Release rows (finished sequences) back to the page pool; they restart empty."""
        if self.is_initialized:
            self.pool.free_rows(rows)

    def write_slots(self, slots: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                    index: Optional[torch.Tensor] = None) -> None:
        """Store packed tokens, or the accepted nodes of drafted trees, in slots of this layer
        (PagePool.write_slots; the slots come from the cache's map_slots)."""
        self.pool.write_slots(slots, key, value, index)

    def attend_tree(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                    mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
        """Attention of drafted tokens over this layer's rows and over one another (PagePool.attend_tree)."""
        return self.pool.attend_tree(query, key, value, mask, scale)

    def offload(self):
        if self.is_initialized:
            self.pool.to("cpu")
            self._bind_pool()

    def prefetch(self):
        if self.is_initialized and self.pool.device != self.device:
            self.pool.to(self.device)
            self._bind_pool()


def _quant_mode(kv_quant: Optional[str]) -> Optional[str]:
    """None for full-precision pages, else KV_QUANT_FP8 ("fp8" and "fp8_e4m3" name it)."""
    if kv_quant is None or str(kv_quant).strip().lower() in {"", "0", "none", "off", "false"}:
        return None
    if str(kv_quant).strip().lower() in {"fp8", "fp8_e4m3", "e4m3", "1", "on", "true"}:
        return KV_QUANT_FP8
    raise ValueError(f"unknown kv_quant {kv_quant!r}: use None or 'fp8_e4m3'")


def _selected_rows(indices, current_batch_size: int) -> list[int]:
    """Row indices of a batch selection (negative ones count from the end), checked."""
    cur = int(current_batch_size)
    rows = [int(i) + cur if int(i) < 0 else int(i) for i in torch.as_tensor(indices).reshape(-1).tolist()]
    if any(r < 0 or r >= cur for r in rows):
        raise IndexError("batch_select_indices: index out of range")
    return rows


class BarqPagedKVCache(Cache):
    """A paged KV cache with one page pool per decoder layer (kv_cache.py:197-223)."""

    def __init__(
        self,
        config,
        max_batch_size: int,
        max_cache_len: int,
        page_size: int = 16,
        num_pages: Optional[int] = None,
        fused_attention: bool = False,
        kv_quant: Optional[str] = None,
        residual_window: int = 128,
    ):
        decoder_config = _decoder_config(config)
        num_layers = decoder_config.num_hidden_layers
        if hasattr(decoder_config, "num_kv_shared_layers"):
            num_layers -= decoder_config.num_kv_shared_layers
        layers = [
            BarqPagedKVCacheLayer(
                max_batch_size=max_batch_size,
                max_cache_len=max_cache_len,
                page_size=page_size,
                num_pages=num_pages,
                fused_attention=fused_attention,
                kv_quant=kv_quant,
                residual_window=residual_window,
            )
            for _ in range(num_layers)
        ]
        super().__init__(layers=layers)
        self.page_size = page_size
        self.barqtrain_max_cache_len = max_cache_len
        self.barqtrain_max_batch_size = max_batch_size

    def free_rows(self, rows) -> None:
        for layer in self.layers:
            layer.free_rows(rows)

    def map_slots(self, lengths, rows=None) -> SlotMap:
        """Take lengths[i] new tokens into row rows[i] of every layer (paged.map_slots_layers): block tables and
        slots [layers, total] of the packed tokens, which each layer's write_slots stores.  The layers must be
        initialised (have taken a first update, or lazy_initialization)."""
        layers = self.layers
        if not layers or not all(l.is_initialized for l in layers):
            raise ValueError("map_slots: the cache's layers hold no pages yet")
        got = map_slots_layers([l.pool for l in layers], lengths, rows, layers[0].max_cache_len)
        last = 1 + max(range(len(lengths)) if rows is None else [int(r) for r in rows], default=-1)
        for l in layers:
            l.current_batch_size = max(l.current_batch_size, last)
        return got

    # Cache.crop and Cache.reset, layer by layer in transformers: one launch for every layer's pool.
    def _pools(self):
        """The layers' pools when every layer is a GPU paged one holding the same rows, else None."""
        layers = self.layers
        if not layers or not all(type(l) is BarqPagedKVCacheLayer and l.is_initialized and type(l.pool) in _POOL_TYPES
                                 and "crop" not in l.__dict__ and "reset" not in l.__dict__ for l in layers):
            return None
        cur = layers[0].current_batch_size
        if any(l.current_batch_size != cur or not l.pool.on_gpu for l in layers):
            return None
        return [l.pool for l in layers]

    def crop(self, tokens_to_remove: Optional[int] = None, *, max_length: Optional[int] = None) -> None:
        """Cache.crop under its own parameter name (a length, or a negative count of tokens to remove),
        or under its former one."""
        if (tokens_to_remove is None) == (max_length is None):
            raise TypeError("crop() takes tokens_to_remove, or max_length")
        to = tokens_to_remove if max_length is None else max_length
        pools = self._pools()
        if pools is not None and to < 0:
            lengths = {l.get_seq_length() for l in self.layers}
            if len(lengths) > 1:  # a length of its own for each layer
                pools = None
            else:
                to = max(lengths.pop() + to, 0)
        if pools is None:
            super().crop(to)
        else:
            crop_layers(pools, self.layers[0].current_batch_size, to)

    def reset(self) -> None:
        pools = self._pools()
        if pools is None:
            super().reset()
            return
        reset_layers(pools)
        for l in self.layers:
            l.current_batch_size = 0

    # Cache.batch_select_indices / reorder_cache / batch_repeat_interleave apply one selection to
    # every layer, one layer at a time; here every layer's pool takes it in one set of launches
    # (barq_kv_select_rows_layers) and the indices cross to the host once.
    def _select_all_layers(self, rows_of) -> bool:
        layers = self.layers
        if not layers or not all(isinstance(l, BarqPagedKVCacheLayer) and l.is_initialized for l in layers):
            return False
        cur = layers[0].current_batch_size
        if any(l.current_batch_size != cur for l in layers):
            return False
        if cur == 0:
            return True
        rows = rows_of(cur)
        if len(rows) > min(l.pool.max_batch for l in layers):
            return False
        select_rows_layers([l.pool for l in layers], rows)
        for l in layers:
            l.current_batch_size = l.max_batch_size = len(rows)
        return True

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        if not self._select_all_layers(lambda cur: _selected_rows(indices, cur)):
            super().batch_select_indices(indices)

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        if not self._select_all_layers(lambda cur: _selected_rows(beam_idx, cur)):
            super().reorder_cache(beam_idx)

    def batch_repeat_interleave(self, repeats: int) -> None:
        if not self._select_all_layers(lambda cur: [b for b in range(cur) for _ in range(int(repeats))]):
            super().batch_repeat_interleave(repeats)


def create_paged_kv_cache(
    model_or_config,
    *,
    max_batch_size: int,
    max_cache_len: int,
    page_size: int = 16,
    num_pages: Optional[int] = None,
    fused_attention: Optional[bool] = None,
    kv_quant: Optional[str] = None,
    residual_window: Optional[int] = None,
) -> BarqPagedKVCache:
    """Create a paged KV cache for a model or decoder config (kv_cache.py:226-240).
    fused_attention defaults to whether the model was routed through "barq_paged".  kv_quant
    ("fp8_e4m3"; default: the BARQTRAIN_KV_QUANT switch, off) keeps blocks older than the last
    residual_window tokens (default: BARQTRAIN_KV_QUANT_WINDOW, else 128) of every row as fp8
    codes, dequantised on every read -- not bit-exact, by design."""
    config = getattr(model_or_config, "config", model_or_config)
    if fused_attention is None:
        fused_attention = bool(getattr(model_or_config, "_barqtrain_paged_attention", False))
    if kv_quant is None:
        kv_quant = os.environ.get("BARQTRAIN_KV_QUANT")
    if residual_window is None:
        residual_window = int(os.environ.get("BARQTRAIN_KV_QUANT_WINDOW", "128"))
    return BarqPagedKVCache(
        config=config,
        max_batch_size=max_batch_size,
        max_cache_len=max_cache_len,
        page_size=page_size,
        num_pages=num_pages,
        fused_attention=fused_attention,
        kv_quant=kv_quant,
        residual_window=residual_window,
    )


def _prompt_geometry(args, kwargs):
    """(batch, prompt_length, device) of a generate() call, taken from the first present of
    input_ids (keyword, else first positional), inputs_embeds, attention_mask."""
    input_ids = kwargs.get("input_ids")
    if input_ids is None and args:
        input_ids = args[0]
    for source in (input_ids, kwargs.get("inputs_embeds"), kwargs.get("attention_mask")):
        if source is not None:
            batch, length = source.shape[:2]
            return int(batch), int(length), source.device
    return None


def _cache_length_budget(model, kwargs, prompt_length: int) -> Optional[int]:
    """prompt + max_new_tokens, else max(max_length, prompt); call kwargs before the model's
    generation_config."""
    config = kwargs.get("generation_config") or getattr(model, "generation_config", None)

    def setting(name):
        value = kwargs.get(name)
        return getattr(config, name, None) if value is None and config is not None else value

    new_tokens = setting("max_new_tokens")
    if new_tokens is not None:
        return prompt_length + int(new_tokens)
    total = setting("max_length")
    return None if total is None else int(max(total, prompt_length))


def maybe_prepare_paged_kv_generate_kwargs(model: torch.nn.Module, args, kwargs):
    """Return ``(kwargs, used)``: kwargs with a fresh paged cache as ``past_key_values`` when
    every gate of the reference passes (kv_cache.py:243-303) -- no cache given, the
    ``BARQTRAIN_ENABLE_PAGED_KV`` switch on, the model marked supported, the GPU backend
    present, a GPU prompt, and a budget of at least ``BARQTRAIN_PAGED_KV_MIN_CACHE_LEN``."""
    declined = (kwargs, False)
    if kwargs.get("past_key_values") is not None or not _env_enabled("BARQTRAIN_ENABLE_PAGED_KV", "1"):
        return declined
    if not getattr(model, "_barqtrain_paged_kv_supported", False) or _get_cuda_backend() is None:
        return declined
    geometry = _prompt_geometry(args, kwargs)
    if geometry is None or geometry[2].type != "cuda":
        return declined
    batch, prompt_length, _ = geometry
    budget = _cache_length_budget(model, kwargs, prompt_length)
    if budget is None or budget < _min_paged_kv_cache_len():
        return declined
    cache = create_paged_kv_cache(
        model,
        max_batch_size=batch,
        max_cache_len=budget,
        page_size=int(os.environ.get("BARQTRAIN_PAGED_KV_PAGE_SIZE", "16")),
    )
    return {**kwargs, "past_key_values": cache, "use_cache": True}, True


def paged_kv_supported_for_model(model: torch.nn.Module) -> bool:
    """True when paged KV-cache injection can run for this model (kv_cache.py:306-308)."""
    return torch.cuda.is_available() and _get_cuda_backend() is not None and hasattr(model, "generate")


__all__ = [
    "BarqPagedKVCache",
    "BarqPagedKVCacheLayer",
    "PagedKVCapacityError",
    "PagedKVPoolExhausted",
    "create_paged_kv_cache",
    "maybe_prepare_paged_kv_generate_kwargs",
    "paged_kv_supported_for_model",
]
