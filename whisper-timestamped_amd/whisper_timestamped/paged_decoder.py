"""The backend decoder's self-attention over paged caches, for the B-stream driver (streams.py).

The backend keeps every layer's text keys and values by concatenation: per layer and token it copies all of them once more
(openai-whisper's ``install_kv_cache_hooks``; the reference drives that cache as it is,
/root/reference/whisper_timestamped/transcribe.py:783-793 only observes it).  Inside ``with PagedText(...).attached():`` the
decoder's self-attention modules write a token's keys and values into a ``PagedKVCache`` per layer and attend over it:
two launches a layer and token, nothing that is there moves.  The backend is instrumented, not modified: the modules'
``forward`` and the model's ``install_kv_cache_hooks`` are shadowed on the instances for the duration of the block;
cross-attention, projections, hooks and everything else stay the backend's own.
"""
from __future__ import annotations

from contextlib import contextmanager

import torch

from ._lib import WtError
from .kvcache import HEAD_DIMS, PagedKVCache

PAGE = 32


def _replaced(model) -> bool:
    return any("forward" in vars(b.attn) for b in model.decoder.blocks) or "install_kv_cache_hooks" in vars(model)


def supported(model, dtype) -> bool:
    dims = model.dims
    return dims.n_text_state // dims.n_text_head in HEAD_DIMS and dtype in (torch.float16, torch.float32, torch.bfloat16) and \
        not _replaced(model) and all(hasattr(b.attn, m) for b in model.decoder.blocks for m in ("query", "key", "value", "out", "qkv_attention"))


class PagedText:
    """Pages for the text of ``n_streams`` rows of a decoder loop, one cache per layer.  Row i of a loop is sequence i: its
    pages are its own, in order."""

    def __init__(self, model, n_streams: int, dtype):
        dims = model.dims
        self.model, self.n_streams = model, int(n_streams)
        self.heads, self.width = dims.n_text_head, dims.n_text_state // dims.n_text_head
        self.pages = -(-dims.n_text_ctx // PAGE)
        shape = (2, self.n_streams * self.pages, self.heads, PAGE, self.width)
        self.caches = []
        for _ in model.decoder.blocks:
            k, v = torch.empty(shape, dtype=dtype, device=model.device)
            self.caches.append(PagedKVCache(k, v))
        self.table = torch.arange(self.n_streams * self.pages, dtype=torch.int32, device=model.device).reshape(self.n_streams, self.pages)
        self.past = 0
        self._step = None

    # --- one decoder call: positions of its rows, the same for every layer
    def _begin(self, batch, n_new):
        if batch > self.n_streams or self.past + n_new > self.pages * PAGE:
            raise WtError(f"paged text: {batch} rows of {self.past} + {n_new} tokens, room for {self.n_streams} of {self.pages * PAGE}")
        dev = self.table.device
        if n_new == 1 and self.past and self._step is not None and self._step[0].shape[0] == batch:
            positions, lengths, _ = self._step           # token by token: both one further
            positions += 1
            lengths += 1
        else:
            at = torch.arange(self.past, self.past + n_new, dtype=torch.int32, device=dev).repeat(batch)
            rows = None if n_new == 1 else torch.arange(batch, dtype=torch.int32, device=dev).repeat_interleave(n_new)
            self._step = (at, torch.full((batch,), self.past + n_new, dtype=torch.int32, device=dev), rows) if n_new == 1 else None
            if n_new > 1:
                return at, None, rows
        return self._step

    def _forward(self, layer, attn, original, x, xa=None, mask=None, kv_cache=None):
        if kv_cache is None or xa is not None:
            return original(x, xa, mask=mask, kv_cache=kv_cache)
        batch, n_new, state = x.shape
        if layer == 0:
            self._now = self._begin(batch, n_new)
        positions, lengths, rows = self._now
        q, k, v = attn.query(x), attn.key(x), attn.value(x)
        cache, table = self.caches[layer], self.table[:batch]
        shape = (batch * n_new, self.heads, self.width)
        cache.append(k.reshape(shape), v.reshape(shape), table, positions, sequences=rows)
        if n_new == 1:
            wv = cache.attend(q.reshape(shape), table, lengths).reshape(batch, 1, state)
        elif self.past == 0:
            wv = attn.qkv_attention(q, k, v, mask)[0]
        else:
            raise WtError(f"paged text: {n_new} tokens at once behind {self.past}: only a loop's first call holds several")
        if layer == 0:       # what the backend's decoder takes its offset from: the first entry's second dimension
            kv_cache[attn.key] = x.new_empty(1).expand(batch, self.past + n_new, state)
        if layer == len(self.caches) - 1:       # (behind the line above: the first layer may be the last)
            self.past += n_new
        return attn.out(wv), None

    def _install_kv_cache_hooks(self, original, cache=None):
        """The backend's own hooks, without those of the self-attention modules."""
        cache, hooks = original(cache)
        own = {id(m._forward_hooks) for b in self.model.decoder.blocks for m in (b.attn.key, b.attn.value)}
        kept = []
        for h in hooks:
            if id(h.hooks_dict_ref()) in own:
                h.remove()
            else:
                kept.append(h)
        self.past, self._step = 0, None
        return cache, kept

    @contextmanager
    def attached(self):
        """For one decoder loop."""
        m = self.model
        if _replaced(m):
            raise WtError("paged text: the model's attention or cache hooks are replaced already (attached twice?)")
        blocks = list(m.decoder.blocks)
        install = m.install_kv_cache_hooks
        m.install_kv_cache_hooks = lambda cache=None: self._install_kv_cache_hooks(install, cache)
        for i, b in enumerate(blocks):
            b.attn.forward = _bound(self, i, b.attn, b.attn.forward)
        try:
            yield self
        finally:
            del m.install_kv_cache_hooks
            for b in blocks:
                del b.attn.forward


def _bound(text, layer, attn, original):
    def forward(x, xa=None, mask=None, kv_cache=None):
        return text._forward(layer, attn, original, x, xa, mask=mask, kv_cache=kv_cache)
    return forward
