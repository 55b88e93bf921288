"""PagedCache under a random-init Llama: uneven sequences that join, grow and
leave, every layer's attention against the float64 restatement of the cache on
the q, k and v that the layer handed over.  And the log probabilities that a
captured decode step reports."""
import numpy as np
import pytest
import torch

from oracle import kv4 as plain

pytestmark = pytest.mark.gpu

VOCAB = 512


def _model(dev, n_q=8, n_kv=2, hd=128, dtype=torch.float16):
    from transformers import LlamaConfig, LlamaForCausalLM
    cfg = LlamaConfig(vocab_size=VOCAB, hidden_size=n_q * hd, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=n_q, num_key_value_heads=n_kv, head_dim=hd, max_position_embeddings=4096,
                      rope_theta=500000.0)
    torch.manual_seed(0)
    return LlamaForCausalLM(cfg).to(dev, dtype).eval()


def _checked(cls):
    class Checked(cls):
        """attend() as it is, its result compared with float64."""
        seen = 0

        def attend(self, layer, q, k, v, scale=None):
            out = super().attend(layer, q, k, v, scale)
            st = self._step
            kept = self.__dict__.setdefault("kept", {})
            ph, table, lens = self.phases.cpu().numpy(), st["table"].cpu().numpy(), st["lens"].tolist()
            cu = None if st["cu"] is None else st["cu"].tolist()
            G, D = k.shape[1:]
            K, V = kept.setdefault(layer, tuple(np.zeros((self.pool.shape[1], 64, G, D)) for _ in "kv"))
            qr = np.zeros(tuple(q.shape))
            for r, b, pos in plain.places(cu, lens, table.shape[1], len(lens)):
                page = table[b, pos // 64]
                K[page, pos % 64] = plain.round4(plain.rotate(k[r].cpu().numpy(), ph, pos).reshape(G, -1, 32)).reshape(G, D)
                V[page, pos % 64] = plain.round4(v[r].double().cpu().numpy().reshape(G, -1, 32)).reshape(G, D)
                qr[r] = plain.rotate(q[r].cpu().numpy(), ph, pos)
            s = D ** -0.5 if scale is None else scale
            want, a, d = plain.attention(qr, K, V, table, lens, cu, s)
            # q is rounded once more than in ops.kv4_attn's own bound: 2^-11 of each score's size
            weight = 2 * d[..., None] * (2.0 ** -11 + (D + 4) * 2.0 ** -24) + 2.0 ** -11 + (max(lens) + 64) * 2.0 ** -25 \
                + (max(lens) + 264) * 2.0 ** -24
            err = weight * 2 * a
            off = np.abs(out.double().cpu().numpy() - want)
            assert (off <= err + 2.0 ** -11 * (np.abs(want) + err) + 2.0 ** -25).all(), off.max()
            Checked.seen += out.shape[0]
            return out
    return Checked


@pytest.mark.parametrize("shape", [(8, 2, 128), (8, 2, 64), (12, 4, 64)], ids=str)
def test_uneven_sequences_join_grow_and_leave(cuda, shape):
    from shard_amd import PagedCache, enable_llama_fused_attention
    model = _model(cuda, *shape)
    assert enable_llama_fused_attention(model)
    cls = _checked(PagedCache)
    cache = cls.from_model(model, n_pages=12, max_len=300)
    g = torch.Generator().manual_seed(1)
    ids = lambda n: torch.randint(0, VOCAB, (n,), generator=g)
    a, b = cache.add(), cache.add()
    logits = cache.run(model, [a, b], [ids(70), ids(3)])
    assert logits.shape == (2, VOCAB)
    for _ in range(3):                                   # a step of one token each
        logits = cache.run(model, [b, a], logits.argmax(-1, keepdim=True).flip(0)).flip(0)
    c = cache.add()
    cache.run(model, [a, c, b], [ids(1), ids(130), ids(5)])   # a prompt beside decode steps
    assert [cache.length(s) for s in (a, b, c)] == [74, 11, 130] and cache.free_pages() == 12 - 2 - 1 - 3
    cache.drop(a)
    d = cache.add()
    every = cache.run(model, [d, c], [ids(64), ids(2)], last_only=False)   # in a's old pages
    assert every.shape == (66, VOCAB) and bool(every.isfinite().all())
    assert cls.seen == 2 * (73 + 6 + 136 + 66)


def test_steps_agree_with_one_prompt(cuda):
    """A text in pieces gives the logits of the text at once, up to fp16: a
    layer's input differs by roundings, which can move a 4-bit code."""
    from shard_amd import PagedCache, enable_llama_fused_attention, token_logprobs
    model = _model(cuda)
    enable_llama_fused_attention(model)
    ids = torch.randint(0, VOCAB, (150,), generator=torch.Generator().manual_seed(2)).to(cuda)
    cache = PagedCache.from_model(model, n_pages=8, max_len=256)
    a, b = cache.add(), cache.add()
    whole = cache.run(model, [a], [ids], last_only=False)
    parts, at = [], 0
    for n in (100, 1, 1, 30, 18):
        parts.append(cache.run(model, [b], [ids[at:at + n]], last_only=False))
        at += n
    parts = torch.cat(parts)
    cos = torch.nn.functional.cosine_similarity(whole.float(), parts.float(), dim=-1)
    assert float(cos.min()) > 0.999
    lp = token_logprobs(whole[:-1], ids[1:])[0]
    want = torch.log_softmax(whole[:-1].double(), -1).gather(1, ids[1:, None])[:, 0]
    # sums of 512 terms in fp32 and exponents of at most a few tens: far below 1e-5
    assert float((lp.double() - want).abs().max()) < 1e-5


def test_bfloat16_model(cuda):
    from shard_amd import PagedCache, enable_llama_fused_attention
    model = _model(cuda, dtype=torch.bfloat16)
    enable_llama_fused_attention(model)
    cache = PagedCache.from_model(model, n_pages=4, max_len=128)
    s = cache.add()
    logits = cache.run(model, [s], [torch.arange(90)])
    assert logits.dtype == torch.bfloat16 and bool(logits.isfinite().all())


def test_refusals(cuda):
    from shard_amd import PagedCache
    cache = PagedCache(3, 100, head_dim=64, num_layers=1, n_kv_heads=2, device=cuda)
    a, b = cache.add(), cache.add()
    with pytest.raises(ValueError):
        cache.begin([a], [101])
    with pytest.raises(ValueError):
        cache.begin([a, a], [1, 1])
    with pytest.raises(ValueError):
        cache.begin([a], [0])
    with pytest.raises(ValueError):
        cache.begin([], [])
    with pytest.raises(KeyError):
        cache.begin([7], [1])
    with pytest.raises(RuntimeError):
        cache.begin([a, b], [100, 100])
    assert cache.free_pages() == 3 and cache.length(a) == 0
    x = torch.zeros(5, 2, 64, dtype=torch.float16, device=cuda)
    with pytest.raises(ValueError):
        cache.attend(0, x, x, x)
    assert cache.begin([a, b], [4, 2]).tolist() == [[0, 1, 2, 3, 0, 1]]
    with pytest.raises(ValueError):
        cache.attend(0, x, x, x)
    with pytest.raises(RuntimeError):
        cache.update(x[None], x[None], 0)
    cache.cancel()
    assert cache.free_pages() == 3 and cache.length(a) == cache.length(b) == 0
    with pytest.raises(ValueError):
        cache.cancel()
    with pytest.raises(ValueError):
        cache.attend(0, x, x, x)


def test_a_failed_step_changes_nothing(cuda):
    """A model whose second layer fails: the step is undone, the next one is as if it had not been."""
    from shard_amd import PagedCache, enable_llama_fused_attention
    model = _model(cuda)
    enable_llama_fused_attention(model)
    ids = torch.arange(80) % VOCAB
    caches = [PagedCache.from_model(model, n_pages=4, max_len=128) for _ in range(2)]
    seqs = [c.add() for c in caches]
    for c, s in zip(caches, seqs):
        c.run(model, [s], [ids[:50]])

    def fail(*args):
        raise ArithmeticError
    hook = model.model.layers[1].register_forward_pre_hook(fail)
    with pytest.raises(ArithmeticError):
        caches[0].run(model, [seqs[0]], [ids[60:]])
    hook.remove()
    assert caches[0].length(seqs[0]) == 50 and caches[0].free_pages() == 3
    got, want = (c.run(model, [s], [ids[50:]]) for c, s in zip(caches, seqs))
    assert torch.equal(got, want)


def test_decode_graph_reports_log_probabilities(cuda):
    from shard_amd import Cache, enable_llama_fused_attention, token_logprobs
    from shard_amd.graph import DecodeGraph
    model = _model(cuda)
    enable_llama_fused_attention(model)
    g = torch.Generator().manual_seed(3)
    ids, first = torch.randint(0, VOCAB, (2, 300), generator=g).to(cuda), torch.randint(0, VOCAB, (2, 1), generator=g).to(cuda)

    def opened(**kw):
        cache = Cache.from_model(model)
        cache._streaming = True
        cache._basis_override = None
        with torch.no_grad():
            model(ids, past_key_values=cache, use_cache=True)
            model(first, past_key_values=cache, use_cache=True)
        return DecodeGraph(model, cache, first, 6, **kw)

    for bad in (-1, 65):
        with pytest.raises(ValueError):
            opened(top_logprobs=bad)
    dg, silent = opened(top_logprobs=4), opened()
    for _ in range(6):
        tok = dg.step()
        assert torch.equal(tok, silent.step()) and silent.logprob is None
        want = token_logprobs(dg.logits, tok, top=4)
        assert all(torch.equal(x, y) for x, y in zip((dg.logprob, dg.entropy, dg.top_logprobs, dg.top_ids), want))
        assert torch.equal(dg.logprob, dg.top_logprobs[:, 0])      # greedy: the most probable
    dg.close()
    silent.close()
