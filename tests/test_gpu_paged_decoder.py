"""The decoder over paged caches on the GPU: what every layer of every call attends over and what comes out of it, in 64 bits."""
import pytest
import torch

import kv_oracle as O
import whisper_double as W
from test_paged_decoder import small_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("layers", [1, 4])
def test_every_layers_attention(layers, dtype):
    """Each new token's attention against the oracle over all keys and values that the layer has had, at the oracle's bound (32-bit sums
    and one rounding to the type), which a key of another position, stream or layer does not meet."""
    from whisper_double.model import build_model
    from whisper_timestamped.paged_decoder import PagedText, supported
    W.install()
    model = small_model(1).to("cuda:0") if layers == 1 else build_model("tiny", device="cuda:0")
    assert len(model.decoder.blocks) == layers and supported(model, dtype)
    state, heads = model.dims.n_text_state, model.dims.n_text_head
    g = torch.Generator().manual_seed(0)
    feats = torch.randn((3, model.dims.n_audio_ctx, state), generator=g).to(dtype).cuda()
    tokens = torch.randint(0, model.dims.n_vocab, (3, 7 + 40), generator=g).cuda()
    text = PagedText(model, 4, dtype)
    seen = [{"query": None, "key": [], "value": [], "out": None} for _ in range(layers)]
    hooks = []
    for s, b in zip(seen, model.decoder.blocks):
        hooks += [b.attn.query.register_forward_hook(lambda m, i, o, s=s: s.update(query=o)),
                  b.attn.key.register_forward_hook(lambda m, i, o, s=s: s["key"].append(o)),
                  b.attn.value.register_forward_hook(lambda m, i, o, s=s: s["value"].append(o)),
                  b.attn.out.register_forward_pre_hook(lambda m, i, s=s: s.update(out=i[0]))]
    positions = []
    hooks.append(model.decoder.blocks[0].attn_ln.register_forward_pre_hook(lambda m, i: positions.append(i[0])))
    try:
        with text.attached(), torch.no_grad():
            cache, own = model.install_kv_cache_hooks()
            for at, end in [(0, 7)] + [(t, t + 1) for t in range(7, 47)]:
                model.decoder(tokens[:, at:end], feats, kv_cache=cache)
                want = model.decoder.token_embedding(tokens[:, at:end]) + model.decoder.positional_embedding[at:end]
                assert torch.equal(positions[-1], want.to(dtype))
                if at == 0:
                    continue
                for layer, s in enumerate(seen):
                    split = lambda x: x.reshape(*x.shape[:2], heads, -1)  # noqa: E731
                    k, v = split(torch.cat(s["key"], 1)), split(torch.cat(s["value"], 1))
                    for b in range(3):
                        ref, _, bound, _ = O.attend(split(s["query"])[b, 0].double().cpu(), k[b].double().cpu(), v[b].double().cpu(), (state // heads) ** -0.5)
                        assert O.far(split(s["out"])[b, 0], ref, bound, dtype) <= 1.0, (layer, end, b)
            for h in own:
                h.remove()
    finally:
        for h in hooks:
            h.remove()
    for c in text.caches:
        c.check()
