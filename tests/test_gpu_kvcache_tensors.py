"""What the paged cache's calls write is known to autograd: a saved tensor that they overwrite is an error in its backward pass."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def setup(dtype=torch.float32):
    from whisper_timestamped import PagedKVCache
    cache = PagedKVCache.allocate(4, 2, 64, 8, dtype=dtype, device=DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    rows = torch.randn((3, 2, 64), device=DEV)
    pos = torch.arange(3, dtype=torch.int32, device=DEV)
    return cache, table, rows, pos, torch.zeros(3, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("written", ["k", "v", "k_exp", "v_exp", "gather0", "gather1", "attend"])
def test_overwritten_saved_tensors_are_noticed(written):
    eight = written.endswith("exp")
    cache, table, rows, pos, seq = setup(torch.float8_e4m3fn if eight else torch.float32)
    outs = torch.randn((3, 2, 64), device=DEV), torch.randn((3, 2, 64), device=DEV)
    res = torch.randn((1, 2, 64), device=DEV)
    saved = {"gather0": outs[0], "gather1": outs[1], "attend": res}.get(written)
    saved = getattr(cache, written) if saved is None else saved
    weight = torch.ones((), device=DEV, requires_grad=True)
    loss = None if eight else (weight * saved).sum()
    before = [t._version for t in (cache.k, cache.v, *outs, res)]
    cache.append(rows, rows, table, pos, sequences=seq)
    assert [cache.k._version, cache.v._version] == [n + 1 for n in before[:2]]
    if eight:
        assert cache.k_exp._version == 1 and cache.v_exp._version == 1
        return
    cache.gather(table, pos, sequences=seq, out=outs)
    cache.attend(rows[:1], table, pos[1:2], out=res)
    assert [t._version for t in (*outs, res)] == [n + 1 for n in before[2:]]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_made_in_inference_mode():
    """They have no version; calls take them as before."""
    with torch.inference_mode():
        cache, table, rows, pos, seq = setup()
        cache.append(rows, rows, table, pos, sequences=seq)
    cache.append(rows, rows, table, pos, sequences=seq)
    out = cache.attend(rows[:1], table, pos[1:2], out=torch.empty_like(rows[:1]))
    assert torch.allclose(out[0], rows[0], atol=1e-6)
