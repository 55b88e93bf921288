"""PagedCache under bf16 models and under every kind of RoPE that it takes."""
import numpy as np
import pytest
import torch

from oracle import kv4 as plain
from test_gpu_paged import VOCAB, _model
from test_paged import check_phases, rope_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["default", "linear", "llama3", "yarn"])
def test_phases_of_rope_kinds(cuda, kind):
    from shard_amd import PagedCache
    model = rope_model(kind).to(cuda)
    check_phases(PagedCache.from_model(model, n_pages=2, max_len=1000), model)


def _checked(cache, half):
    """cache, each attend() compared with float64 on the q, k and v that the layer handed over; `half` half a step of their type."""
    attend, kept, seen = cache.attend, {}, []

    def checked(layer, q, k, v, scale=None):
        out = attend(layer, q, k, v, scale)
        st, ph = cache._step, cache.phases.cpu().numpy()
        table, lens = st["table"].cpu().numpy(), st["lens"].tolist()
        cu = None if st["cu"] is None else st["cu"].tolist()
        G, D = k.shape[1:]
        K, V = kept.setdefault(layer, tuple(np.zeros((cache.pool.shape[1], 64, G, D)) for _ in "kv"))
        q, k, v = (t.double().cpu().numpy() for t in (q, k, v))
        qr = np.zeros(q.shape)
        for r, b, pos in plain.places(cu, lens, table.shape[1], len(lens)):
            at = table[b, pos // 64], pos % 64
            K[at] = plain.round4(plain.rotate(k[r], ph, pos).reshape(G, -1, 32)).reshape(G, D)
            V[at] = plain.round4(v[r].reshape(G, -1, 32)).reshape(G, D)
            qr[r] = plain.rotate(q[r], ph, pos)
        want, a, d = plain.attention(qr, K, V, table, lens, cu, D ** -0.5 if scale is None else scale)
        # scores: the rotated q is rounded to its type (half a step, and what its fp32 sum of two products is off by, of
        # numbers as large as the row's), bf16 queries are held to 2^-26 of their row's largest, D products are summed in
        # fp32; they move a weight by twice their size.  Weights fp16, their sums fp32; the output's own rounding last.
        size = np.sqrt(2) * d[..., None]
        weight = 2 * size * (half + 2.0 ** -22 + (D + 4) * 2.0 ** -24 + D * 2.0 ** -26) + 2.0 ** -11 \
            + max(lens) * 2.0 ** -36 + (max(lens) + 264) * 2.0 ** -24
        err = weight * 2 * a
        off = np.abs(out.double().cpu().numpy() - want)
        assert (off <= err + half * (np.abs(want) + err) + 2.0 ** -25).all(), (off.max(), (off / (err + half * np.abs(want))).max())
        seen.append(out.shape[0])
        return out
    cache.attend = checked
    return seen


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(8, 2, 128), (12, 4, 64)], ids=str)
def test_layers_of_uneven_steps(cuda, shape, dtype):
    """Prompts, single tokens and both in one step, every layer against float64."""
    from shard_amd import PagedCache, enable_llama_fused_attention
    model = _model(cuda, *shape, dtype=dtype)
    enable_llama_fused_attention(model)
    cache = PagedCache.from_model(model, n_pages=12, max_len=300)
    seen = _checked(cache, torch.finfo(dtype).eps / 2)
    g = torch.Generator().manual_seed(4)
    ids = lambda n: torch.randint(0, VOCAB, (n,), generator=g)
    a, b, c = cache.add(), cache.add(), cache.add()
    logits = cache.run(model, [a, b], [ids(90), ids(2)])
    assert logits.dtype == dtype
    cache.run(model, [b, a], logits.argmax(-1, keepdim=True).flip(0))
    cache.run(model, [a, c, b], [ids(1), ids(150), ids(3)])
    assert seen == [92, 92, 2, 2, 154, 154]


@pytest.mark.parametrize("how", ["sdpa", "eager"])
def test_padded_batches_are_refused(cuda, how):
    """A batch of rows of one length runs through the model as it is; one with padding does not, and its step is undone."""
    from shard_amd import PagedCache, enable_llama_fused_attention
    model = _model(cuda)
    model.set_attn_implementation(how)
    enable_llama_fused_attention(model)
    ids = torch.randint(0, VOCAB, (2, 20), generator=torch.Generator().manual_seed(1)).to(cuda)
    cache = PagedCache.from_model(model, n_pages=4, max_len=64)
    a, b, c, d = (cache.add() for _ in range(4))
    mask = torch.ones(2, 20, dtype=torch.int64, device=cuda)
    mask[0, :5] = 0
    with torch.no_grad():
        pos = cache.begin([a, b], [20, 20])
        with pytest.raises(ValueError, match="mask"):
            model(input_ids=ids, attention_mask=mask, position_ids=pos.view(2, 20), past_key_values=cache, use_cache=True)
        cache.cancel()
        assert cache.length(a) == 0 and cache.free_pages() == 4
        pos = cache.begin([a, b], [20, 20])
        got = model(input_ids=ids, attention_mask=torch.ones_like(mask), position_ids=pos.view(2, 20), past_key_values=cache,
                    use_cache=True).logits
    want = cache.run(model, [c, d], list(ids), last_only=False)
    assert torch.equal(got.view(40, -1), want)
