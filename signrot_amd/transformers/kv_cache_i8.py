"""Paged int8 KV cache, beside the int4 one (kv_cache.py), for layers whose
attention 4 bits hurt and for models with query / key norms.

  pages  i8  [pages, n_layers, 2, num_heads, page_size, 128]      (K, V)
  scales f32 [pages, n_layers, 2, num_heads, page_size / 16]

value = code * scale, one scale for each block of 16 tokens and head: 256.5 bytes a
token and head for K and V together against the int4 cache's 136.  Tokens that come
one at a time are kept less exactly than a prompt's: each growth of the open block's
scale rounds its older codes again (normal values: 25% more rms error than in one
piece), so what the cache holds depends on how the tokens were cut into calls.  The
page table is the int4 cache's (request b's page j is page j * B + b), and so are the
protocol of update() and that of graph capture.  Differences:
  * update() takes any number of tokens after the prefill (a prompt's next piece,
    tokens to be verified), and its attention as many queries, causally.
  * update_qkv() is update() from the q/k/v projection output with the q/k norms
    and the rotary embedding in the same launch.
  * Keys are stored as they come: there is no head-dim Hadamard, which int4 needs.
"""
import math
from typing import Any, Dict, Optional

import torch
from transformers.cache_utils import Cache

from .. import _CUDA
from .kv_cache import _PageTable, _init_hf_cache, _pages_for


class _LayerAttentionI8:
    """What update() returns after an append: q [B, T, Hq, 128] of the appended
    tokens -> attention over this layer's cache, same shape.  `live`: the rows of
    [B T] that came in where the mask left some out, whose outputs are 0."""

    def __init__(self, cache, layer_idx, tokens, starts, live=None):
        self.cache, self.layer_idx, self.tokens, self.starts = cache, layer_idx, tokens, starts
        self.live = live

    def __call__(self, q):
        B, T, Hq, D = q.shape
        if T != self.tokens:
            raise ValueError(f"attention takes the {self.tokens} appended tokens, got {T}")
        q = q.reshape(B * T, Hq, D)
        if self.live is None:
            o = self.cache._attend(q.contiguous(), self.layer_idx, T, self.starts)
        else:
            o = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
            o[self.live] = self.cache._attend(q[self.live], self.layer_idx, T, self.starts)
        return o.view(B, T, Hq, D)


class MultiLayerPagedKVCache8Bit(Cache):
    """Paged int8 KV cache for all layers of a model.  `num_heads` is the number
    of KV heads; `softmax_scale` defaults to 1 / sqrt(128)."""

    batch_size = None   # ahead of the read-only property of transformers' Cache

    def __init__(self, batch_size, page_size, max_seq_len, device, n_layers, num_heads, head_dim,
                 softmax_scale=None):
        if head_dim != 128:
            raise ValueError("head_dim must be 128")
        if page_size <= 0 or page_size % _CUDA.I8_BLOCK:
            raise ValueError(f"page_size must be a multiple of {_CUDA.I8_BLOCK}")
        if softmax_scale and not 2.0 ** -20 <= abs(softmax_scale) <= 2.0 ** 60:
            raise ValueError(f"softmax_scale={softmax_scale} must be 0, or 2^-20 to 2^60 in "
                             "magnitude")
        _init_hf_cache(self)
        self.batch_size = batch_size
        self.page_size = page_size
        self.max_seq_len = max_seq_len
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.softmax_scale = 1 / math.sqrt(head_dim) if softmax_scale is None else softmax_scale
        self.device = device
        self.length = 0
        pool = max(1, _pages_for(max_seq_len, page_size) * batch_size)
        self.pages = torch.empty((pool, n_layers, 2, num_heads, page_size, head_dim),
                                 dtype=torch.int8, device=device)
        self.scales = torch.empty((pool, n_layers, 2, num_heads, page_size // _CUDA.I8_BLOCK),
                                  dtype=torch.float32, device=device)
        self._filled = [False] * n_layers
        self._table = _PageTable(batch_size, pool, device)
        self._frozen = False
        self._spec = {}
        self._point_spec()
        self._held = 0
        self._set_table(0)

    def _set_table(self, held, beside=None):
        """Index tensors of `held` tokens per request: one number, or int32 [B] (which
        the host reads and returns, and `beside` with them).  They stay as they were
        where that is refused."""
        was, self._held = self._held, held
        try:
            if isinstance(held, int):
                return self._table.set_uniform(held, self.page_size)
            host = self._table.set_lengths(held, self.page_size, beside)
            if (host[0] == self.length).all():   # no padding: as without a mask
                self._held = self.length
            return host
        except BaseException:
            if self._held is not was:
                self._set_table(was)
            raise

    def _point_spec(self):
        self._spec.update(kv_data=self.pages, kv_scale=self.scales, kv_indptr=self._table.indptr,
                          kv_indices=self._table.indices, last_page_offset=self._table.last)

    @property
    def seen_tokens(self):
        return self.length

    def _reserve(self, tokens):
        """Room for `tokens` per request, the pool doubled when it runs out."""
        need, have = _pages_for(tokens, self.page_size) * self.batch_size, self.pages.shape[0]
        if need <= have:
            return
        total = max(need, 2 * have)
        self.pages, self.scales = (torch.cat([t, t.new_empty((total - have, *t.shape[1:]))])
                                   for t in (self.pages, self.scales))
        self._table.grow(total)
        self._point_spec()

    def _step(self, tokens, layer_idx, mask):
        """Count the new tokens (with the first layer), write the index tensors and
        return whether the mask counts all of the new ones.  Frozen index tensors say
        themselves where the tokens go, within the pool that they were made for: it
        keeps its place then, as a captured step needs."""
        if mask is None and not self._frozen and self.length and not isinstance(self._held, int):
            raise ValueError("the cache holds padded requests: their attention_mask is needed")
        if layer_idx == 0:
            if not self._frozen:
                self._reserve(self.length + tokens)
            self.length += tokens
        if mask is None:
            self.get_cache_specs_for_flash_infer(None)
            return True
        new = mask[:, mask.shape[1] - tokens:].sum(dim=-1, dtype=torch.int32)
        return bool((self._set_table(mask.sum(dim=-1, dtype=torch.int32), new)[1] == tokens).all())

    def _undone(self, length, held):
        """After a refused call: length and index tensors as before it."""
        self.length = length
        if self._held is not held or self._table.unwritten():
            self._set_table(held)

    def _starts(self, tokens):
        """Row index of `tokens` rows per request, None for one each."""
        return None if tokens == 1 else self._table._row * tokens

    def _check_mask(self, mask, tokens, layer_idx):
        """The mask covers the new tokens, and behind the prefill those before them too
        (the first layer counts the new ones)."""
        B, first = self.batch_size, not self._filled[layer_idx]
        want = tokens if first else self.length + (tokens if layer_idx == 0 else 0)
        if mask.dim() != 2 or mask.shape[0] != B or mask.shape[1] < max(want, tokens) or \
                (first and mask.shape[1] != want):
            raise ValueError(f"attention_mask must be [{B}, {want}], got {tuple(mask.shape)}")

    def _live_rows(self, mask, tokens):
        """The rows of [B tokens] that the mask's last columns count as tokens, and
        their index by request."""
        live = mask[:, mask.shape[1] - tokens:] != 0
        starts = torch.zeros(self.batch_size + 1, device=self.device, dtype=torch.int32)
        torch.cumsum(live.sum(dim=-1, dtype=torch.int32), dim=0, out=starts[1:])
        return live.flatten().nonzero().flatten(), starts

    def update(self, key_states, value_states, layer_idx,
               cache_kwargs: Optional[Dict[str, Any]] = None):
        """Store K/V fp16 [B, T, H, 128] of one layer.  The first call for a layer
        is its prefill and returns the inputs for the prefill attention; later calls
        append T tokens per request and return the attention over the cache, a
        callable that takes their queries [B, T, Hq, 128].  With an attention_mask (in
        later calls the one of all tokens so far, its last T columns the new ones)
        only its 1-positions are stored; a 0-position's attention is 0.  Padded requests
        go on with their mask."""
        B, T, H, D = key_states.shape
        if H != self.num_heads:
            raise ValueError(f"update() takes the {self.num_heads} KV heads, got {H}")
        if B != self.batch_size:
            raise ValueError(f"batch {B} != the cache's {self.batch_size}")
        mask = (cache_kwargs or {}).get("attention_mask")
        first = not self._filled[layer_idx]
        length, held = self.length, self._held
        try:
            k, v = (t.reshape(B * T, H, D) for t in (key_states, value_states))
            if mask is not None:
                self._check_mask(mask, T, layer_idx)
            if self._step(T, layer_idx, mask):
                live, starts = None, self._starts(T)
            else:
                live, starts = self._live_rows(mask, T)
                k, v = k[live], v[live]
            _CUDA.append_kv_i8(**self._spec, layer_idx=layer_idx, k=k, v=v, new_indptr=starts,
                               max_new=T)
        except BaseException:   # refused: no tokens came in
            self._undone(length, held)
            raise
        self._filled[layer_idx] = True
        if first:
            return key_states, value_states
        return _LayerAttentionI8(self, layer_idx, T, starts, live)

    def update_qkv(self, qkv, cos, sin, layer_idx, num_q_heads, q_weight=None, k_weight=None,
                   eps=None, attention_mask=None):
        """update() of T tokens per request from their q/k/v projection output
        qkv fp16 [B, T, (Hq + 2 H) 128], one launch: RMSNorm of each q and k head
        (eps given; weights [128] or None), rotary embedding (cos / sin [1 or B, T,
        128]), k and v into the cache.  Returns q [B, T, Hq, 128], for attend().
        It may be a layer's first update too (of a prompt without padding: attend()
        then is the prefill attention, over the cache's values).  attention_mask: the
        extended mask after a left-padded prefill, as for update(), all of its last T
        columns 1."""
        B, T = qkv.shape[:2]
        if B != self.batch_size:
            raise ValueError(f"batch {B} != the cache's {self.batch_size}")
        if attention_mask is not None and not self._filled[layer_idx]:
            raise ValueError("update_qkv() takes a prompt without padding")
        if attention_mask is not None:
            self._check_mask(attention_mask, T, layer_idx)
        if tuple(cos.shape) not in ((1, T, 128), (B, T, 128)) or cos.shape != sin.shape:
            raise ValueError(f"cos / sin must be [1 or {B}, {T}, 128]")
        rows = [t.reshape(T, 128) if B == 1 or (T == 1 and t.shape[0] == 1)
                else t.expand(B, T, 128).reshape(B * T, 128) for t in (cos, sin)]
        length, held = self.length, self._held
        try:
            if not self._step(T, layer_idx, attention_mask):
                raise ValueError("update_qkv() takes new tokens without padding")
            q = _CUDA.qkv_norm_rope_append_i8(
                **self._spec, layer_idx=layer_idx, qkv=qkv.reshape(B * T, -1),
                cos=rows[0].contiguous(), sin=rows[1].contiguous(), n_q_heads=num_q_heads,
                q_weight=q_weight, k_weight=k_weight, eps=eps, new_indptr=self._starts(T),
                max_new=T)
        except BaseException:
            self._undone(length, held)
            raise
        self._filled[layer_idx] = True
        return q.view(B, T, num_q_heads, 128)

    def attend(self, q, layer_idx):
        """Causal attention of each request's last T tokens q [B, T, Hq, 128] over
        this layer's cache."""
        return _LayerAttentionI8(self, layer_idx, q.shape[1], self._starts(q.shape[1]))(q)

    def _attend(self, q, layer_idx, tokens, starts):
        # a captured step is replayed for longer contexts: the split is planned
        # for the longest
        longest = self.max_seq_len if self._frozen else max(1, self.length)
        return _CUDA.batch_attention_i8(torch.empty_like(q), q, **self._spec,
                                        layer_idx=layer_idx, q_indptr=starts, max_q_len=tokens,
                                        max_kv_len=longest, softmax_scale=self.softmax_scale)

    def update_qkv_decode_quant(self, qkv, cos, sin, layer_idx, num_q_heads, scale,
                                attention_mask=None, q_weight=None, k_weight=None, eps=None):
        """A decode step's attention and the o_proj input (codes [B, Hq 64], scales
        [B, 1]): update_qkv() of one token per request, attend(), then the head-axis
        Hadamard (times scale) and the per-token quantizer.  qkv [B, (Hq + 2 H) 128]."""
        if not self._filled[layer_idx]:
            raise RuntimeError("update_qkv_decode_quant: the layer has no prefill yet")
        if not 0 < num_q_heads <= 64 or num_q_heads & (num_q_heads - 1) or \
                num_q_heads % self.num_heads:
            raise RuntimeError(f"update_qkv_decode_quant: {num_q_heads} query heads must be a "
                               f"power of two <= 64, a multiple of the {self.num_heads} KV heads")
        B = qkv.shape[0]
        q = self.update_qkv(qkv.view(B, 1, -1), cos, sin, layer_idx, num_q_heads, q_weight,
                            k_weight, eps, attention_mask)
        o = self._attend(q.view(B, num_q_heads, 128), layer_idx, 1, None)
        return _CUDA.head_had_quant(o, scale)

    # ---------------------------------------------------------- index specs
    def specs(self):
        """The op keyword arguments (kv_data, kv_scale, kv_indptr, kv_indices,
        last_page_offset) as they stand."""
        return self._spec

    def refresh_specs(self, length: Optional[int] = None):
        """Rewrite the index tensors in place for `length` tokens per request
        (default: the current length), before a replay of a captured step."""
        self._set_table(self.length if length is None else int(length))
        return self._spec

    def freeze_specs(self, frozen=True):
        """While frozen, update() uses the index tensors as they are and the pool does
        not grow, so it can be captured in a graph."""
        self._frozen = frozen

    def get_cache_specs_for_flash_infer(self, attention_mask):
        if attention_mask is not None:
            self._set_table(attention_mask.sum(dim=-1, dtype=torch.int32))
        elif not self._frozen:
            self._set_table(self.length)
        return self._spec

    def mark_prefilled(self, length: int):
        """Declare that every layer holds `length` tokens per request, written into
        `pages` / `scales` directly; the next update() of each layer appends."""
        self._reserve(length)
        self.length = length
        self._filled = [True] * len(self._filled)
        if not self._frozen:
            self._set_table(length)

    def clone(self):
        """An independent copy: own pages, scales and index tensors, same state."""
        c = object.__new__(type(self))
        c.__dict__.update(self.__dict__)
        c.pages, c.scales = self.pages.clone(), self.scales.clone()
        c._filled = list(self._filled)
        c._table = self._table.clone()
        c._spec = {}
        c._point_spec()
        return c

    def reset(self):
        self.length = 0
        self._filled = [False] * len(self._filled)
        if not self._frozen:
            self._set_table(0)

    def get_seq_length(self, layer_idx: Optional[int] = 0) -> int:
        return self.length

    def get_max_length(self) -> Optional[int]:
        return None

    def __len__(self):
        return len(self._filled)

    def get_usable_length(self, new_seq_length: int, layer_idx: Optional[int] = 0) -> int:
        return self.length

    def to_legacy_cache(self):
        return self
