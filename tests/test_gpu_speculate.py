"""PagedCache.speculate under a random-init Llama: every layer's attention over trees against the float64
restatement, and the accepted tokens against the model's own logits."""
import numpy as np
import pytest
import torch

from oracle import drafts as plain
from oracle import kv4
from tests.test_gpu_drafts import random_parents
from tests.test_gpu_paged import VOCAB, _model

pytestmark = pytest.mark.gpu


def _checked(cls):
    class Checked(cls):
        """attend() as it is, its result on trees compared with float64 on what the cache holds."""
        seen = 0

        def attend(self, layer, q, k, v, scale=None):
            out = super().attend(layer, q, k, v, scale)
            st = self._step
            if st["tree"] is None:
                return out
            lens, cu, parents = st["lens"].tolist(), None if st["cu"] is None else st["cu"].tolist(), st["tree"][2].tolist()
            K, V = kv4.held(self.pool[layer].cpu().numpy())
            ph, D = self.phases.cpu().numpy(), q.shape[2]
            tree = plain.tree(parents, lens, cu, 16)
            qr = np.stack([kv4.rotate(x, ph, tree[r][1]) for r, x in enumerate(q.cpu().numpy())])
            s = D ** -0.5 if scale is None else scale
            want, a, d = plain.attention(qr, K, V, st["table"].cpu().numpy(), lens, cu, s, [tree[r][0] for r in range(len(parents))])
            # q is rounded once before the scores: 2^-11 of each score's size; the rest as in ops.kv4_tree_attn's own bound
            weight = 2 * d[..., None] * (2.0 ** -11 + (D + 4) * 2.0 ** -24) + 2.0 ** -11 + (max(lens) + 64) * 2.0 ** -25 \
                + (max(lens) + 264) * 2.0 ** -24
            err = weight * 2 * a
            off = np.abs(out.double().cpu().numpy() - want)
            assert (off <= err + 2.0 ** -11 * (np.abs(want) + err) + 2.0 ** -25).all(), off.max()
            Checked.seen += out.shape[0]
            return out
    return Checked


class Recorded:
    """A model that keeps its last logits."""

    def __init__(self, model):
        self.model = model

    def __call__(self, **kw):
        out = self.model(**kw)
        self.logits = out.logits[0]
        return out


@pytest.mark.parametrize("shape", [(8, 2, 128), (12, 4, 64)], ids=str)
def test_greedy_speculation(cuda, shape):
    """Drafts that hold the model's own next tokens: what is gained is the model's largest logit after each accepted row,
    and the cache goes on from there."""
    from shard_amd import PagedCache, enable_llama_fused_attention
    model = _model(cuda, *shape)
    enable_llama_fused_attention(model)
    cls = _checked(PagedCache)
    cache = cls.from_model(model, n_pages=16, max_len=300)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (61, 7)]
    a, b = cache.add(), cache.add()
    # the model's own continuation, token by token, in a cache of its own
    own = cls.from_model(model, n_pages=16, max_len=300)
    oa, ob = own.add(), own.add()
    last = own.run(model, [oa, ob], prompts).argmax(-1)
    texts = [[int(t)] for t in last]
    for _ in range(9):
        last = own.run(model, [oa, ob], last[:, None]).argmax(-1)
        for text, t in zip(texts, last.tolist()):
            text.append(t)
    first = cache.run(model, [a, b], prompts).argmax(-1).tolist()
    rec, total, accepted = Recorded(model), [61, 7], 0
    tokens = [[t] for t in first]
    for turn in range(3):
        drafts, parents = [], []
        for s in range(2):
            good = texts[s][len(tokens[s]):len(tokens[s]) + 3]
            # the last token, then its likely continuation with a wrong sibling before each
            row, up, at = [tokens[s][-1]], [-1], 0
            for t in good:
                row += [(t + 1) % VOCAB, t]
                up += [at, at]
                at = len(row) - 1
            drafts.append(row)
            parents.append(up)
        gained = cache.speculate(rec, [a, b], drafts, parents)
        top, at = rec.logits.float().cpu().numpy().argmax(-1).tolist(), 0
        for s in range(2):
            want, row = [], 0
            while True:
                want.append(top[at + row])
                row = next((i for i, p in enumerate(parents[s]) if p == row and drafts[s][i] == want[-1]), None)
                if row is None:
                    break
            assert gained[s] == want, (turn, s)
            tokens[s] += want
            total[s] += len(want)
            accepted += len(want) - 1
            at += len(drafts[s])
        assert [cache.length(x) for x in (a, b)] == total
        assert cache.free_pages() == 16 - sum((n + 63) // 64 for n in total)
    assert accepted > 0 and cls.seen > 0
    cache.drop(a)
    cache.drop(b)
    assert cache.free_pages() == 16


def test_branches_agree_with_plain_sequences(cuda):
    """The logits of every row of a tree are, up to fp16, those of its path as a plain sequence; sampling and bf16."""
    from shard_amd import PagedCache, enable_llama_fused_attention
    for dtype, cos_min in ((torch.float16, 0.999), (torch.bfloat16, 0.99)):
        model = _model(cuda, dtype=dtype)
        enable_llama_fused_attention(model)
        cache = PagedCache.from_model(model, n_pages=8, max_len=256)
        g = torch.Generator().manual_seed(2)
        prompt, ids = torch.randint(0, VOCAB, (100,), generator=g), torch.randint(0, VOCAB, (12,), generator=g)
        parents = random_parents([12], 4)
        a, b = cache.add(), cache.add()
        cache.run(model, [a, b], [prompt, prompt])
        rows = cache.run(model, [a], [ids], last_only=False, parents=[parents])
        cache.cancel()
        assert cache.length(a) == 100
        for r in (0, 3, 7, 11):
            path, at = [], r
            while at >= 0:
                path.insert(0, at)
                at = parents[at]
            want = cache.run(model, [b], [ids[path]])
            assert float(torch.nn.functional.cosine_similarity(rows[r].float(), want[0].float(), dim=0)) > cos_min
            cache.drop(b)
            b = cache.add()
            cache.run(model, [b], [prompt])
        probs = torch.full((12, VOCAB), 1.0 / VOCAB, device=cuda)
        for kw in (dict(temperature=0.8), dict(temperature=1.2, draft_probs=probs), dict(temperature=torch.tensor([0.5], device=cuda))):
            before = cache.length(a)
            gained = cache.speculate(model, [a], [ids], [parents], uniforms=torch.rand(12, 2, generator=g).to(cuda), **kw)
            assert cache.length(a) == before + len(gained[0]) and all(0 <= t < VOCAB for t in gained[0])
