"""The decoder over paged caches (paged_decoder.py) on the CPU: the cache replaced by a plain one, the backend's own as the oracle."""
import pytest
import torch

import whisper_double as W
from whisper_double.model import ModelDimensions, Whisper


class PlainCache:
    """append and attend of one new token over pages on the CPU."""

    def __init__(self, k, v):
        self.k, self.v = k, v

    def append(self, k, v, table, positions, sequences=None):
        for r, p in enumerate(positions.tolist()):
            s = r if sequences is None else int(sequences[r])
            page, slot = int(table[s, p // self.k.shape[2]]), p % self.k.shape[2]
            self.k[page, :, slot], self.v[page, :, slot] = k[r], v[r]

    def attend(self, q, table, lengths):
        out = torch.empty_like(q)
        for s, n in enumerate(lengths.tolist()):
            k, v = (x[table[s].long()].transpose(1, 2).reshape(-1, *q.shape[1:])[:n] for x in (self.k, self.v))
            w = torch.softmax((q[s][None] * k).sum(-1) * q.shape[-1] ** -0.5, 0)
            out[s] = (w[..., None] * v).sum(0)
        return out


def small_model(layers, seed=0):
    W.install()
    torch.manual_seed(seed)
    m = Whisper(ModelDimensions(n_mels=80, n_audio_ctx=30, n_audio_state=64, n_audio_head=2, n_audio_layer=1, n_vocab=300, n_text_ctx=64,
                                n_text_state=64, n_text_head=2, n_text_layer=layers)).eval()
    torch.nn.init.normal_(m.decoder.positional_embedding)
    return m


def decoded(model, prompt, steps, feats):
    cache, hooks = model.install_kv_cache_hooks()
    try:
        with torch.no_grad():
            return torch.cat([model.decoder(prompt, feats, kv_cache=cache)[:, -1:]] +
                             [model.decoder(steps[:, i:i + 1], feats, kv_cache=cache) for i in range(steps.shape[1])], 1)
    finally:
        for h in hooks:
            h.remove()


@pytest.mark.parametrize("prompt_len", [1, 5])
@pytest.mark.parametrize("layers", [1, 2, 3])
def test_decoders_of_any_depth(layers, prompt_len, monkeypatch):
    """The backend takes a call's positions from what the first layer leaves in its cache: logits call by call, a loop after
    another, for every depth of the decoder (one layer is the first and the last)."""
    from whisper_timestamped import paged_decoder
    monkeypatch.setattr(paged_decoder, "PagedKVCache", PlainCache)
    model = small_model(layers)
    assert paged_decoder.supported(model, torch.float32)
    g = torch.Generator().manual_seed(1)
    feats = torch.randn((3, 30, 64), generator=g)
    prompt, steps = torch.randint(0, 300, (3, prompt_len), generator=g), torch.randint(0, 300, (3, 40), generator=g)
    want = decoded(model, prompt, steps, feats)
    text = paged_decoder.PagedText(model, 4, torch.float32)
    for _ in range(2):
        with text.attached():
            got = decoded(model, prompt, steps, feats)
        # two orders of the same 32-bit sums: a few hundred roundings of 2^-24 a layer, logits of about 10; a wrong position
        # is off by 10 and more
        assert float((got - want).abs().max()) <= 2.0 ** -24 * 512 * layers * float(want.abs().max())


def test_a_model_is_attached_once(monkeypatch):
    """A second block over the same model is refused, and the first one still leaves the model as it was."""
    from whisper_timestamped import paged_decoder
    from whisper_timestamped._lib import WtError
    monkeypatch.setattr(paged_decoder, "PagedKVCache", PlainCache)
    model = small_model(2)
    one, two = (paged_decoder.PagedText(model, 1, torch.float32) for _ in range(2))
    with one.attached():
        with pytest.raises(WtError, match="attached"), two.attached():
            pass
        assert not paged_decoder.supported(model, torch.float32)
    assert "install_kv_cache_hooks" not in vars(model) and not any("forward" in vars(b.attn) for b in model.decoder.blocks)
    with two.attached():
        pass
    assert paged_decoder.supported(model, torch.float32)
