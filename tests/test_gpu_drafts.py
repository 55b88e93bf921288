"""Trees of drafted tokens over the paged 4-bit cache on the GPU (ops.draft_tree,
kv4_append at positions, kv4_tree_attn, kv4_keep) against the float64 restatement
in oracle/drafts.py."""
import random

import numpy as np
import pytest
import torch

from oracle import drafts as plain
from oracle import kv4
from tests.test_gpu_kv4 import Batch

pytestmark = pytest.mark.gpu


def random_parents(new, seed=0, width=4):
    """A tree for each sequence; sizes of 1 and 0 too."""
    rng = random.Random(seed)
    out = []
    for n in new:
        t = []
        for i in range(n):
            t.append(rng.randrange(max(0, i - width), i) if i else -1)
        out += t
    return out


def bits(mask):
    """The rows that each row's mask (T, W) int64 names."""
    return [{64 * w + j for w, x in enumerate(row) for j in range(64) if x >> j & 1} for row in mask.tolist()]


class Trees(Batch):
    def __init__(self, total, new, *args, parents=None, **kw):
        super().__init__(total, new, *args, **kw)
        self.parents = torch.tensor(random_parents(new, sum(total)) if parents is None else parents, dtype=torch.int32)
        self.max_new = max(new)

    def plan(self):
        from shard_amd import ops
        self.mask, self.positions = ops.draft_tree(self.d_parents, self.d_lens, cu_seqlens=self.d_cu, max_new=self.max_new)
        return self.mask

    def tree_attn(self, mask=None, **kw):
        from shard_amd import ops
        mask = self.mask if mask is None else mask
        return ops.kv4_tree_attn(kw.pop("q", self.d_q), self.d_cache, self.d_table, self.d_lens, mask,
                                 cu_seqlens=kw.pop("cu_seqlens", self.d_cu), **kw)

    def check(self, out, scale=None, mask=None):
        scale = self.D ** -0.5 if scale is None else scale
        k, v = kv4.held(self.d_cache.cpu().numpy())
        want, a, d = plain.attention(self.q.double().numpy(), k, v, self.table.numpy(), self.lens.tolist(), self.cu.tolist(), scale,
                                     bits(self.mask if mask is None else mask))
        d, n = d[:, :, None], max(self.total) + 64
        # scores: D products of exact operands summed in fp32, one scaling, one subtraction of the maximum (2^-24 each of
        # at most d); bf16 queries are held to 2^-26 of their row's largest.  They move a weight by twice their size, relative.
        # weights: fp16, 2^-11 each and 2^-25 below fp16's normal range; exp2, their sums and the joins of waves and splits
        # in fp32 (n + 200 roundings at most).  The output's own rounding comes last.
        weight = 2 * (self.D + 4) * 2.0 ** -24 * d + (2 * self.D * 2.0 ** -26 * d if self.type == torch.bfloat16 else 0)
        weight = weight + 2.0 ** -11 + n * 2.0 ** -25 + (n + 200) * 2.0 ** -24
        err = weight * 2 * a
        tol = err + torch.finfo(self.type).eps / 2 * (np.abs(want) + err) + 2.0 ** -25
        off = np.abs(out.cpu().double().numpy() - want)
        assert (off <= tol).all(), (off.max(), (off / tol).max())


# ---------------------------------------------------------------------------
# the plan
# ---------------------------------------------------------------------------
PLANS = [([1], [1]), ([64], [64]), ([65, 3], [65, 2]), ([200, 131, 7, 40], [3, 131, 0, 33]), ([1024], [1024]), ([2000, 129], [300, 128])]


@pytest.mark.parametrize("total,new", PLANS, ids=str)
def test_plan(cuda, total, new):
    from shard_amd import ops
    parents = random_parents(new, len(total))
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    mask, positions = ops.draft_tree(dev(parents), dev(total), cu_seqlens=dev(cu.tolist()), max_new=max(new))
    assert mask.shape == (sum(new), (max(new) + 63) // 64)
    want = plain.tree(parents, total, cu.tolist(), mask.shape[1])
    for r, (seen, got, pos) in enumerate(zip(range(len(parents)), bits(mask), positions.tolist())):
        assert got == want[r][0] and pos == want[r][1], r


def test_plan_of_odd_parents(cuda):
    """A chain as long as a tree may be, parents that are none, rows behind the bound and behind the last sequence,
    lengths below the rows."""
    from shard_amd import ops
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    chain = list(range(-1, 1023))
    mask, positions = ops.draft_tree(dev(chain), dev([5000]), cu_seqlens=dev([0, 1024]))
    assert positions.tolist() == list(range(3976, 5000))
    assert bits(mask) == [set(range(i + 1)) for i in range(1024)]
    odd = [-1, 5, 1, -7, 3, 2 ** 31 - 1, -2 ** 31, 2] + [7] * 100 + [0, 0]
    lens, cu = [3, 200], [0, 8, 108]
    mask, positions = ops.draft_tree(dev(odd), dev(lens), cu_seqlens=dev(cu), max_new=64)
    want = plain.tree(odd, lens, cu, 1)
    for r in range(108):
        assert (bits(mask)[r], int(positions[r])) == want[r], r
    assert int(positions[8 + 64]) == -1 and int(mask[8 + 64, 0]) == 0
    # one row a sequence needs no cu_seqlens
    mask, positions = ops.draft_tree(dev([-1, 4]), dev([7, 0]))
    assert mask.tolist() == [[1], [1]] and positions.tolist() == [6, -1]


# ---------------------------------------------------------------------------
# append at positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("total,new,H,G,D", [([1], [1], 4, 1, 128), ([70, 131, 9], [5, 40, 0], 8, 2, 64), ([130], [33], 6, 2, 128)], ids=str)
def test_append_at_positions(cuda, total, new, H, G, D, type):
    b = Trees(total, new, H, G, D, type, seed=3)
    b.plan()
    q = b.append(q=b.d_q, positions=b.positions)
    before, after = kv4.held(b.cache.numpy()), kv4.held(b.d_cache.cpu().numpy())
    ph, pos = b.phases.numpy(), b.positions.tolist()
    touched = np.zeros(before[0].shape[:2], bool)
    for r, s, place in b.where():
        page = kv4.page_at(b.table.numpy(), b.n_pages, s, place)
        touched[page, place % 64] = True
        k = kv4.rotate(b.k[r].double().numpy(), ph, pos[r])
        assert np.array_equal(after[0][page, place % 64], kv4.round4(k.reshape(G, -1, 32)).reshape(G, D)), r
        assert np.array_equal(after[1][page, place % 64], kv4.round4(b.v[r].double().numpy().reshape(G, -1, 32)).reshape(G, D)), r
        want = kv4.rotate(b.q[r].double().numpy(), ph, pos[r])
        size = np.abs(b.q[r].double().numpy())
        size = np.concatenate([size[:, :D // 2] + size[:, D // 2:]] * 2, -1)
        # two products and their sum in fp32, one rounding to the type (and its smallest step below the normal range)
        tol = torch.finfo(b.type).eps / 2 * np.abs(want) + 2.0 ** -22 * size + 2.0 ** -25
        assert (np.abs(q[r].cpu().double().numpy() - want) <= tol).all()
    for x, y in zip(before, after):
        assert np.array_equal(x[~touched], y[~touched], equal_nan=True)


def test_append_at_own_positions_is_append(cuda):
    """Positions that are the rows' places give the bytes of a call without them, prompts of several groups too."""
    b = Trees([300, 64, 31], [290, 1, 30], 4, 2, 64, seed=14)
    q = b.append(q=b.d_q)
    want = b.d_cache.clone()
    b.d_cache = b.cache.to(cuda)
    places = torch.tensor([p for _, _, p in b.where()], dtype=torch.int32, device=cuda)
    assert torch.equal(b.append(q=b.d_q, positions=places), q) and torch.equal(b.d_cache, want)


def test_rows_without_a_position_are_left_out(cuda):
    """Neither K nor V of a row whose position is negative or past the phases; its rotated q is zeros."""
    b = Trees([75, 40], [20, 9], 4, 2, 128, seed=4)
    b.plan()
    end = b.phases.shape[0]
    out = [2, 3, 17, 22]
    b.positions[out] = torch.tensor([-1, end, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=cuda)
    q = b.append(q=b.d_q, positions=b.positions)
    before, after = kv4.held(b.cache.numpy()), kv4.held(b.d_cache.cpu().numpy())
    for r, s, place in b.where():
        at = kv4.page_at(b.table.numpy(), b.n_pages, s, place), place % 64
        for x, y in zip(before, after):
            assert np.array_equal(x[at], y[at], equal_nan=True) == (r in out), r
        assert bool(q[r].any()) == (r not in out)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
ATTN = [  # total, new, H, G, D: every kernel, trees across pages and words, prefixes of nothing
    ([1], [1], 4, 1, 128), ([2], [2], 4, 4, 64), ([64], [8], 8, 2, 128), ([65], [8], 8, 2, 64), ([67], [8], 8, 2, 128),
    ([1000], [7], 12, 4, 128), ([3000, 5, 64, 517], [4, 5, 3, 1], 8, 2, 64), ([300, 77], [13, 2], 40, 2, 128),
    ([130, 500, 9], [9, 4, 9], 8, 2, 64), ([257], [16], 64, 1, 64), ([700], [61], 8, 2, 128), ([333, 64, 200], [66, 1, 64], 8, 2, 64),
    ([640], [200], 4, 4, 128), ([400, 50, 129, 1], [0, 50, 128, 1], 6, 2, 128), ([900], [300], 2, 1, 64), ([100], [100], 8, 2, 128),
]


@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("total,new,H,G,D", ATTN, ids=str)
def test_tree_attention(cuda, total, new, H, G, D, type):
    b = Trees(total, new, H, G, D, type, seed=len(total) + H, wide=2).fill()
    b.plan()
    for kw in (dict(), dict(max_new=max(new), max_len=max(total)), dict(max_new=1, max_len=1)):
        b.check(b.tree_attn(**kw))


FOLDED = [([400, 321], [1, 1], 256, 256, 64), ([417, 330], [2, 1], 512, 256, 64), ([500, 3], [2, 3], 512, 256, 64),
          ([385, 200], [1, 1], 2048, 256, 64), ([390, 130], [4, 3], 256, 256, 64), ([2300], [3], 128, 64, 64), ([2305], [7], 64, 64, 64)]


@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("total,new,H,G,D", FOLDED, ids=str)
def test_tree_attention_few_rows_many_pages(cuda, total, new, H, G, D, type):
    b = Trees(total, new, H, G, D, type, seed=len(total) + H, wide=2).fill()
    b.plan()
    for kw in (dict(max_new=max(new)), dict(max_new=max(new), max_len=max(total))):
        b.check(b.tree_attn(**kw))


@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("B,most,G,H,D", [(130, 3, 8, 16, 64), (65, 9, 16, 32, 128)], ids=str)
def test_tree_attention_of_many_uneven_sequences(cuda, B, most, G, H, D, type):
    g = torch.Generator().manual_seed(B)
    total = [int(n) for n in torch.randint(0, 200, (B,), generator=g)]
    total[3:9] = [0, 1, 64, 64, 64, 350]
    new = [min(n, 1 + i % most) for i, n in enumerate(total)]
    b = Trees(total, new, H, G, D, type, seed=B, wide=1).fill()
    b.plan()
    for kw in (dict(max_new=most, max_len=max(total)), dict(max_new=1, max_len=30)):
        b.check(b.tree_attn(**kw))


@pytest.mark.parametrize("new", [5, 70])
def test_tree_attention_of_a_chain_is_causal(cuda, new):
    """A chain's rows see what kv4_attn shows them (its tiles and splits may be others: not its bits)."""
    b = Trees([390], [new], 8, 2, 128, seed=2, parents=list(range(-1, new - 1))).fill()
    b.plan()
    b.check(b.tree_attn())
    b.check(b.attn())


@pytest.mark.parametrize("new", [3, 70])
def test_masks_of_any_bits(cuda, new):
    """Rows that see no row of the step, themselves included; rows that see later ones; bits behind the rows; fewer
    words than the rows would need; a sequence of nothing but its rows, some of which then see nothing at all."""
    b = Trees([new + 130, new, 0], [new, new, 0], 8, 2, 64, seed=6).fill()
    g = torch.Generator().manual_seed(1)
    for words in (1, 2, 3):
        mask = torch.randint(-2 ** 62, 2 ** 62, (2 * new, words), generator=g) * 2 + 1
        mask[new - 1] = 0
        mask[new + 1] = 0
        out = b.tree_attn(mask=mask.to(cuda))
        assert not out[new + 1].any()
        b.check(out, mask=mask)


def test_tree_attention_rows_nobody_has(cuda):
    """Lengths below the rows, below zero, pages outside the cache, rows behind the last sequence."""
    b = Trees([130, 70, 190, 64], [10, 20, 20, 8], 4, 2, 128, seed=8).fill()
    b.lens = torch.tensor([130, 13, 190, -5], dtype=torch.int32)  # the second's first 7 rows stand before place 0
    b.table[0, 1] = b.n_pages
    b.cu = torch.tensor([0, 10, 30, 50, 54], dtype=torch.int32)
    b.plan()
    b.mask[54:] = -1
    out = torch.full_like(b.d_q, 7.0)
    b.tree_attn(out=out)
    assert bool((out[54:] == 7).all()) and not out[50:54].any()
    out[54:] = 0
    b.check(out)


def test_tree_attention_scales_and_specials(cuda):
    """A scale of 0, a large and a negative one; a query of NaN ruins its own row only."""
    b = Trees([200], [9], 8, 2, 128, seed=3).fill()
    b.plan()
    for scale in (0.0, 2.0, -0.1):
        b.check(b.tree_attn(scale=scale), scale=scale)
    want = b.tree_attn()
    q = b.d_q.clone()
    q[4, 1, 3] = float("nan")
    got = b.tree_attn(q=q)
    assert bool(got[4, 1].isnan().all())
    got[4, 1] = want[4, 1]
    assert torch.equal(got, want)


def test_tree_attention_far_pages_and_strides(cuda):
    """Pages past 4 GiB of a pool of layers; q as a slice of wider rows; another stream."""
    b = Trees([190, 130], [6, 70], 8, 2, 128, seed=9, spare=0).fill()
    b.plan()
    want = b.tree_attn()
    b.check(want)
    pool = torch.empty(140_000, 2, 2, 68 * 128, dtype=torch.uint8, device=cuda)
    far = torch.arange(pool.shape[0] - b.n_pages, pool.shape[0], device=cuda)
    pool[:, 1][far] = b.d_cache
    b.d_table = far[b.d_table.clamp(max=b.n_pages - 1).long()].int()
    b.d_cache = pool[:, 1]
    assert torch.equal(b.tree_attn(), want)
    wide = torch.cat([b.d_q.flatten(1), b.d_q.flatten(1)], 1)[:, :1024].unflatten(1, (8, 128))
    assert not wide.is_contiguous() and torch.equal(b.tree_attn(q=wide), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [b.tree_attn() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, want) for x in got)


# ---------------------------------------------------------------------------
# keep
# ---------------------------------------------------------------------------
KEEP = [  # total, new, paths
    ([70], [9], [[0, 2, 5, 8]]), ([64], [64], [[0, 63]]), ([130, 66, 20], [40, 6, 20], [[0, 30, 31, 32, 33, 39], [0, 1, 2, 3, 4, 5], [0, 19]]),
    ([200], [150], [list(range(0, 150, 2))]), ([300], [90], [[0] + list(range(4, 90))]), ([61, 3], [12, 1], [[0, 1, 5, 6, 11], [0]]),
    ([90], [20], [[]]), ([90, 7], [20, 0], [[3], []]),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("layers", [1, 3])
@pytest.mark.parametrize("total,new,paths", KEEP, ids=str)
def test_keep(cuda, total, new, paths, layers, D):
    from shard_amd import ops
    b = Trees(total, new, 10, 5, D, seed=len(total))
    pool = torch.randint(0, 256, (layers, *b.cache.shape), generator=torch.Generator().manual_seed(3), dtype=torch.uint8)
    P = max(len(p) for p in paths) + 2
    rows = torch.tensor([p + [-1] * (P - len(p)) for p in paths], dtype=torch.int32, device=cuda)
    counts = torch.tensor([len(p) for p in paths], dtype=torch.int32, device=cuda)
    got = pool.to(cuda)
    ops.kv4_keep(got if layers > 1 else got[0], b.d_table, b.d_lens, rows, counts, cu_seqlens=b.d_cu)
    for x, y in zip(pool.numpy(), got.cpu().numpy()):
        want = kv4.held(x)
        after = kv4.held(y)
        for w, a in zip(want, after):
            w, old = w.copy(), w
            for s, path in enumerate(paths):
                first = total[s] - new[s]
                for j, r in enumerate(path):
                    dst, src = ((kv4.page_at(b.table.numpy(), b.n_pages, s, t), t % 64) for t in (first + j, first + r))
                    w[dst] = old[src]
            assert np.array_equal(w, a, equal_nan=True)


def test_keep_of_nothing_and_odd_entries(cuda):
    """Counts of zero, below it and beyond the path's width; entries below their index, behind the rows or without a
    page; lengths below the rows: nothing else moves and nothing outside is written."""
    from shard_amd import ops
    b = Trees([130, 70, 190, 5, 40], [10, 20, 20, 8, 3], 4, 2, 64, seed=8)
    b.table[2, 2] = b.n_pages + 5                                 # tokens from 128 on
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    rows = dev([[0, 3, 1, 10, 9], [2, 2, 2, 19, 2 ** 31 - 1], [5, 6, 7, 8, 9], [1, 2, 3, 5, 6], [2, 2, 2, 2, 2]])
    counts = dev([5, 2 ** 31 - 1, 5, 5, -2 ** 31])
    b.d_lens = dev([130, 70, 190, 5, 40])
    before = kv4.held(b.cache.numpy())
    ops.kv4_keep(b.d_cache, b.d_table, b.d_lens, rows, counts, cu_seqlens=b.d_cu)
    after = kv4.held(b.d_cache.cpu().numpy())
    moves = [(0, 121, 123), (0, 124, 129), (1, 50, 52), (1, 51, 52), (1, 53, 69), (3, 0, 2), (3, 1, 3)]
    # sequence 3: rows 0 .. 2 stand at -3 .. -1, so entries 0 .. 2 have no place to go to
    for w, a in zip(before, after):
        w, old = w.copy(), w
        for s, dst, src in moves:
            d, f = ((kv4.page_at(b.table.numpy(), b.n_pages, s, t), t % 64) for t in (dst, src))
            w[d] = old[f]
        assert np.array_equal(w, a, equal_nan=True)


def test_keep_layers_page_by_page_and_far(cuda):
    """Layers that alternate page by page, and a pool past 4 GiB."""
    from shard_amd import ops
    b = Trees([190, 64], [50, 20], 4, 2, 128, seed=5)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    rows, counts = dev([[0, 7, 9, 49], [0, 1, 19, -1]]), dev([4, 3])
    two = torch.randint(0, 256, (2, *b.cache.shape), generator=torch.Generator().manual_seed(3), dtype=torch.uint8).to(cuda)
    want = two.clone()
    ops.kv4_keep(want, b.d_table, b.d_lens, rows, counts, cu_seqlens=b.d_cu)
    assert not torch.equal(want, two)
    woven = two.transpose(0, 1).contiguous().transpose(0, 1)
    ops.kv4_keep(woven, b.d_table, b.d_lens, rows, counts, cu_seqlens=b.d_cu)
    assert torch.equal(woven, want)
    pool = torch.zeros(2, 140_000, 2, 68 * 128, dtype=torch.uint8, device=cuda)
    far = torch.arange(pool.shape[1] - b.n_pages, pool.shape[1], device=cuda)
    pool[:, far] = two
    table = far[b.d_table.clamp(max=b.n_pages - 1).long()].int()
    ops.kv4_keep(pool, table, b.d_lens, rows, counts, cu_seqlens=b.d_cu)
    assert torch.equal(pool[:, far], want)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type,D", [("fp16", 128), ("bf16", 64)])
def test_a_tree_stored_attended_verified_and_kept(cuda, type, D):
    """Rounds of drafting over three sequences: the cache holds afterwards, bit for bit, what appending the accepted
    tokens one after the other gives, and every accepted row's attention is that of the plain sequence."""
    from shard_amd import ops
    H, G, V, rounds, start = 8, 2, 50, 6, [100, 1, 60]
    g = torch.Generator().manual_seed(D)
    caches, tables = [ops.kv4_cache(12, G, D) for _ in range(2)], torch.arange(12, dtype=torch.int32, device=cuda).view(3, 4)
    inv = 1.0 / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
    phases = ops.rope_phases(0, 256, inv.float().to(cuda))
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    rows = lambda n, heads: (torch.randn(n, heads, D, generator=g) * 2).to(cuda, torch.float16 if type == "fp16" else torch.bfloat16)
    cu = [0, 100, 101, 161]
    k, v = rows(161, G), rows(161, G)
    for c in caches:
        ops.kv4_append(k, v, c, tables, dev(start), phases, cu_seqlens=dev(cu))
    lens = list(start)
    for turn in range(rounds):
        new = [1 + (3 * turn + 5 * s) % 9 for s in range(3)]
        parents = random_parents(new, turn)
        cu = [0, new[0], new[0] + new[1], sum(new)]
        T, total = sum(new), [a + n for a, n in zip(lens, new)]
        q, k, v = rows(T, H), rows(T, G), rows(T, G)
        logits = (torch.randn(T, V, generator=g) * 3).to(cuda)
        tokens = torch.randint(0, V, (T,), generator=g).to(cuda)
        for s in range(3):                                        # a likely child, so that paths have some length
            for i in range(1, new[s]):
                logits[cu[s] + parents[cu[s] + i], tokens[cu[s] + i]] += 8
        uniforms = torch.rand(T, 2, generator=g).to(cuda)
        mask, positions = ops.draft_tree(dev(parents), dev(total), cu_seqlens=dev(cu), max_new=max(new))
        qr = ops.kv4_append(k, v, caches[0], tables, dev(total), phases, q=q, cu_seqlens=dev(cu), positions=positions)
        out = ops.kv4_tree_attn(qr, caches[0], tables, dev(total), mask, cu_seqlens=dev(cu), max_new=max(new))
        path, counts, following = ops.verify_drafts(logits, tokens, dev(parents), uniforms, cu_seqlens=dev(cu), max_new=max(new))
        ops.kv4_keep(caches[0], tables, dev(total), path, counts, cu_seqlens=dev(cu))
        want, margin = plain.verify(logits.cpu().numpy(), tokens.tolist(), parents, uniforms.cpu().numpy(), cu, None, [1.0] * 3)
        assert margin > V * 2.0 ** -50
        n = counts.tolist()
        for s in range(3):
            assert path[s, :n[s]].tolist() == want[s][0] and int(following[s]) == want[s][1]
        # the accepted rows alone, in order
        kept = [cu[s] + i for s in range(3) for i in want[s][0]]
        cu_kept = dev([0] + np.cumsum(n).tolist())
        lens = [a + c for a, c in zip(lens, n)]
        qr2 = ops.kv4_append(k[kept], v[kept], caches[1], tables, dev(lens), phases, q=q[kept], cu_seqlens=cu_kept)
        assert torch.equal(qr2, qr[kept])
        plain_out = ops.kv4_attn(qr2, caches[1], tables, dev(lens), cu_seqlens=cu_kept, max_new=max(new))
        every = dev([0] + np.cumsum(lens).tolist())
        held = [ops.kv4_read(c, tables, dev(lens), sum(lens), cu_seqlens=every) for c in caches]
        assert torch.equal(held[0][0], held[1][0]) and torch.equal(held[0][1], held[1][1])
        # each output is off by its weights' 2^-11 in sum and total, of the largest value at most, and its rounding;
        # scores of the same keys in 32 bits (a tenth of that)
        most = float(held[0][1].abs().max())
        tol = 2 * most * (2.2 * 2.0 ** -11 + torch.finfo(out.dtype).eps / 2)
        assert float((plain_out.float() - out[kept].float()).abs().max()) <= tol
    assert max(lens) < 256


def test_a_step_captured(cuda):
    """Plan, storing, attention, verification and keeping in one graph, replayed with other inputs in the same memory."""
    from shard_amd import ops
    H, G, D, V, new = 8, 2, 128, 1000, [6, 9]
    g = torch.Generator().manual_seed(2)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    cu, T = dev([0, 6, 15]), 15
    phases = ops.rope_phases(0, 512, (1.0 / 10000.0 ** (torch.arange(0, D, 2) / D)).to(cuda))
    table = torch.arange(16, dtype=torch.int32, device=cuda).view(2, 8)

    def inputs():
        x = lambda *s: torch.randn(*s, generator=g).to(cuda)
        return [x(T, H, D).half(), x(T, G, D).half(), x(T, G, D).half(), x(T, V) * 3, torch.randint(0, V, (T,), generator=g).to(cuda),
                torch.rand(T, 2, generator=g).to(cuda), dev(random_parents(new, int(torch.randint(0, 99, (1,), generator=g)))),
                dev([300 + int(torch.randint(0, 200, (1,), generator=g)), 15])]

    def step(cache, q, k, v, logits, tokens, uniforms, parents, lens):
        mask, positions = ops.draft_tree(parents, lens, cu_seqlens=cu, max_new=9)
        qr = ops.kv4_append(k, v, cache, table, lens, phases, q=q, cu_seqlens=cu, max_new=9, positions=positions)
        out = ops.kv4_tree_attn(qr, cache, table, lens, mask, cu_seqlens=cu, max_new=9)
        path, counts, following = ops.verify_drafts(logits, tokens, parents, uniforms, cu_seqlens=cu, max_new=9, temperature=0.9)
        probs = torch.softmax(logits, -1)
        again = ops.verify_drafts(logits, tokens, parents, uniforms, cu_seqlens=cu, max_new=9, draft_probs=probs)
        ops.kv4_keep(cache, table, lens, path, counts, cu_seqlens=cu)
        return [mask, positions, out, path, counts, following, *again]

    base = torch.randint(0, 100, (16, G, 68 * D), generator=g, dtype=torch.uint8).to(cuda)
    eager, captured = base.clone(), base.clone()
    held = inputs()
    step(base.clone(), *held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(captured, *held)
    captured.copy_(base)
    for _ in range(4):
        new_in = inputs()
        want = step(eager, *new_in)
        for dst, src in zip(held, new_in):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(captured, eager)
        assert bool(torch.randn(64, device=cuda).isfinite().all())


@pytest.mark.parametrize("type", ["fp16", "bf16"])
def test_compiled_and_plain_dispatch_agree(cuda, type, monkeypatch):
    """The compiled way and the one through Python give the same bits, and the compiled one takes plain calls."""
    from shard_amd import ops
    results = []
    for direct in (ops._bind_direct(), False):
        monkeypatch.setattr(ops, "_direct", direct)
        b = Trees([300, 64, 90], [20, 1, 33], 8, 2, 128, type, seed=16).fill()
        g = torch.Generator().manual_seed(1)
        logits, tokens = torch.randn(54, 500, generator=g).to(b.type).to(cuda) * 3, torch.randint(0, 500, (54,), generator=g).to(cuda)
        u, probs = torch.rand(54, 2, generator=g).to(cuda), torch.softmax(torch.randn(54, 600, generator=g), -1).to(cuda)[:, :500]
        temps = torch.tensor([0.0, 1.0, 0.6], device=cuda)
        verify = lambda **kw: ops.verify_drafts(logits, tokens, b.d_parents, u, cu_seqlens=b.d_cu, **kw)
        b.plan()
        q = b.append(q=b.d_q, positions=b.positions)
        res = [b.mask, b.positions, *ops.draft_tree(b.d_parents, b.d_lens, cu_seqlens=b.d_cu), q, b.d_cache.clone(), b.tree_attn(),
               b.tree_attn(scale=0.3, max_new=33), *verify(), *verify(temperature=temps, max_new=33), *verify(draft_probs=probs, max_depth=2)]
        path, counts, _ = verify(temperature=0.0, max_new=33)
        pool = torch.stack([b.d_cache, b.d_cache])
        ops.kv4_keep(pool, b.d_table, b.d_lens, path, counts, cu_seqlens=b.d_cu)
        ops.kv4_keep(b.d_cache, b.d_table, b.d_lens, path[:, :9], counts, cu_seqlens=b.d_cu)
        results.append(res + [path, counts, pool, b.d_cache])
        if direct:
            dev, none = torch.cuda.current_device(), None
            assert direct.kv4_tree_attn(b.d_q, b.d_cache, b.d_table, b.d_lens, b.d_cu, none, 33, 300, b.mask, dev, 0) is not None
            assert direct.draft_tree(b.d_parents, b.d_lens, b.d_cu, 33, dev, 0) is not None
            assert direct.verify_drafts(logits, tokens, b.d_parents, u, b.d_cu, none, 1.0, none, none, dev, 0) is not None
            assert direct.kv4_keep(pool, b.d_table, b.d_lens, path, counts * 0, b.d_cu, dev, 0) is not None
            torch.cuda.synchronize()
    for x, y in zip(*results):
        assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)


def test_refusals(cuda):
    from shard_amd import ops
    b = Trees([70, 40], [5, 4], 4, 2, 64, seed=1)
    b.plan()
    i32 = dict(dtype=torch.int32, device=cuda)
    for bad in (b.d_parents.long(), b.d_parents[::2], b.d_parents[None]):
        with pytest.raises((TypeError, ValueError)):
            ops.draft_tree(bad, b.d_lens, cu_seqlens=b.d_cu)
    with pytest.raises(ValueError):
        ops.draft_tree(b.d_parents, b.d_lens)
    with pytest.raises(ValueError):
        ops.draft_tree(torch.zeros(1100, **i32), b.d_lens, cu_seqlens=b.d_cu)
    with pytest.raises(TypeError):
        ops.draft_tree(b.d_parents, b.d_lens, cu_seqlens=b.d_cu[:2])
    for bad in (b.mask.int(), b.mask[:3], b.mask[:, :0], b.mask.expand(-1, 2), b.mask[:, 0]):
        with pytest.raises(TypeError):
            b.tree_attn(mask=bad)
    with pytest.raises(ops.ShardHipUnavailable):
        b.tree_attn(mask=b.mask.cpu())
    with pytest.raises(TypeError):
        b.append(positions=b.positions.long())
    with pytest.raises(TypeError):
        b.append(positions=b.positions[:4])
    with pytest.raises(ops.ShardHipUnavailable):
        b.append(positions=b.positions.cpu())
    rows, counts = torch.zeros(2, 3, **i32), torch.ones(2, **i32)
    for r, c in ((rows.long(), counts), (rows[:1], counts), (rows, counts[:1]), (rows, counts.long()), (rows.T, counts),
                 (rows[0], counts), (rows[:, :1].expand(2, 3), counts)):
        with pytest.raises(TypeError):
            ops.kv4_keep(b.d_cache, b.d_table, b.d_lens, r, c, cu_seqlens=b.d_cu)
    with pytest.raises(TypeError):
        ops.kv4_keep(b.d_cache.short(), b.d_table, b.d_lens, rows, counts, cu_seqlens=b.d_cu)
    with pytest.raises(ops.ShardHipUnavailable):
        ops.kv4_keep(b.d_cache, b.d_table, b.d_lens, rows.cpu(), counts, cu_seqlens=b.d_cu)
    same = b.d_cache.unsqueeze(0).expand(2, -1, -1, -1)            # layers on each other
    with pytest.raises(ops.ShardHipError):
        ops.kv4_keep(same, b.d_table, b.d_lens, rows, counts, cu_seqlens=b.d_cu)


@pytest.mark.parametrize("type", ["fp16", "bf16"])
def test_append_at_every_border(cuda, type):
    """Codes at the borders of every scale, and next to them: numbers of the type (V, and K at an angle of 0), and products that
    lie beside a border by a unit of 2^-23 or less (K at cosines next to 1)."""
    from shard_amd import ops
    D, dt = 64, {"fp16": torch.float16, "bf16": torch.bfloat16}[type]
    marks = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    rows = []
    for s in kv4.SCALES:
        x = torch.tensor(np.concatenate([marks * s, -marks * s])).to(dt)
        x = x.where(x.double().abs() <= 6.5 * s, 0)
        bits16 = x.view(torch.int16)
        near = [x] + [(bits16 + step).view(dt) for step in (-1, 1)]      # the next numbers of the type (of 0: NaN and subnormal)
        x = torch.cat([n.where(n.double().abs() <= 6.5 * s, 0) for n in near])
        x = torch.cat([x, x[:14]]).view(2, 31)
        top = torch.tensor([[6.25 * s], [-6.25 * s]]).to(dt)               # 4 significant bits: the block's scale is s
        rows.append(torch.cat([x, top], 1).reshape(1, D))
    rows = torch.stack(rows)
    n = len(rows)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    table = torch.arange((n + 63) // 64, dtype=torch.int32, device=cuda)[None]
    for cos in (1.0, 1 + 2.0 ** -23, 1 - 2.0 ** -24, -1.0, -1 - 2.0 ** -23):
        phases = torch.zeros(128, D // 2, 2)
        phases[..., 0] = cos
        cache = ops.kv4_cache(table.shape[1], 1, D, device=cuda)
        d = rows.to(cuda)
        ops.kv4_append(d, d, cache, table, lens, phases.to(cuda), cu_seqlens=torch.tensor([0, n], dtype=torch.int32, device=cuda))
        K, V = (t.reshape(-1, D)[:n] for t in kv4.held(cache.cpu().numpy()))
        x = rows[:, 0].double().numpy()
        assert np.array_equal(V, kv4.round4(x.reshape(n, 2, 32)).reshape(n, D))
        want = kv4.round4((x * np.float64(np.float32(cos))).reshape(n, 2, 32)).reshape(n, D)
        assert np.array_equal(K, want), (cos, np.argwhere(K != want)[:4])


# ---------------------------------------------------------------------------
# the plans that large calls get
# ---------------------------------------------------------------------------
def _plan(b):
    """(rows of a tile, row tiles, splits, longest first, tiles of the same pages side by side) of a call with its
    launch hints, restated; the splits are those that its workspace is for."""
    import ctypes
    from shard_amd import _lib
    B, T, most, length = len(b.total), sum(b.new), max(b.new), max(b.total)
    args = _lib.KV4Args(batch=B, n_tokens=T, n_q_heads=b.H, n_kv_heads=b.G, head_dim=b.D, dtype=0, n_pages=b.n_pages,
                        table_width=b.table.shape[1], cache=4096, page_stride=b.G * 68 * b.D, block_table=4096,
                        table_stride=b.table.shape[1], seq_lens=4096, cu_seqlens=4096, max_new=most, max_len=length)
    need = _lib.load().shard_kv4_tree_attn_workspace(ctypes.byref(args))
    splits, left = divmod(need, T * b.H * (b.D + 2) * 4)
    splits = max(splits, 1)
    assert left == 0
    up = lambda n, d: -(-n // d)
    rows, pages = most * (b.H // b.G), up(length, 64)
    whole = 400 * up(rows, 128) <= 115 * up(rows, 32) and B * b.G * up(rows, 128) * pages > 6500
    tile = 16 if rows <= 16 else 128 if whole else 32
    tiles = up(rows, tile)
    groups = B * b.G * tiles
    want = max(up(512, groups), up(pages, 32 if groups * up(pages, 32) <= 1152 else 64))
    want = min(want, up(pages, 4), 128)
    assert splits == max(2 ** k for k in range(8) if k == 0 or 2 ** (2 * k - 1) < want * want)
    return tile, tiles, splits, tile != 128 and B > 1 and groups * splits >= 1024, tiles > 1 and B * b.G * splits % 8 == 0


class Large(Trees):
    """Trees with the reference by matrix products."""

    def reference(self, scale, mask):
        k, v = kv4.held(self.d_cache.cpu().numpy())
        T, group = sum(self.new), self.H // self.G
        want, a, d = np.zeros((T, self.H, self.D)), np.zeros((T, self.H, self.D)), np.zeros((T, self.H))
        words = mask.cpu().numpy().view(np.uint64)
        for b, (n, m) in enumerate(zip(self.total, self.new)):
            r0, t = int(self.cu[b]), np.arange(n)
            page = self.table[b].numpy()[t // 64]
            K, V = k[page, t % 64], v[page, t % 64]
            bits = (words[r0:r0 + m, :, None] >> np.arange(64, dtype=np.uint64) & np.uint64(1)).reshape(m, 64 * words.shape[1]).astype(bool)
            bits = np.pad(bits, ((0, 0), (0, max(0, m - bits.shape[1]))))[:, :m]
            seen = np.concatenate([np.ones((m, n - m), bool), bits], 1)
            seen, some = np.repeat(seen, group, 0), np.repeat(seen.any(1), group)
            for g in range(self.G):
                q = self.q[r0:r0 + m, g * group:(g + 1) * group].double().numpy().reshape(m * group, self.D)[some]
                s = np.where(seen[some], q @ K[:, g].T * scale, -np.inf)
                w = np.exp(s - s.max(1, keepdims=True, initial=-1e300))
                w /= w.sum(1, keepdims=True)
                size = np.where(seen[some], np.abs(q) @ np.abs(K[:, g]).T * abs(scale), 0).max(1, initial=0)
                for out, x in ((want, w @ V[:, g]), (a, w @ np.abs(V[:, g])), (d[..., None], size[:, None])):
                    of = np.zeros((m * group, x.shape[1]))
                    of[some] = x
                    out[r0:r0 + m, g * group:(g + 1) * group] = of.reshape(m, group, x.shape[1])
        return want, a, d

    def check(self, out, mask=None):
        want, a, d = self.reference(self.D ** -0.5, self.mask if mask is None else mask)
        d, n = d[:, :, None], max(self.total) + 64
        # as Trees.check
        weight = 2 * (self.D + 4) * 2.0 ** -24 * d + (2 * self.D * 2.0 ** -26 * d if self.type == torch.bfloat16 else 0)
        weight = weight + 2.0 ** -11 + n * 2.0 ** -25 + (n + 200) * 2.0 ** -24
        err = weight * 2 * a
        tol = err + torch.finfo(self.type).eps / 2 * (np.abs(want) + err) + 2.0 ** -25
        off = np.abs(out.cpu().double().numpy() - want)
        assert (off <= tol).all(), (off.max(), (off / tol).max())

    def check_all(self):
        """Trees; any bits; fewer words than rows, of which most rows see none; the same bits again on another stream."""
        hints = dict(max_new=max(self.new), max_len=max(self.total))
        self.plan()
        out = self.tree_attn(**hints)
        self.check(out)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = self.tree_attn(**hints)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(again, out)
        g = torch.Generator().manual_seed(7)
        any_bits = lambda words: torch.randint(-2 ** 63, 2 ** 63 - 1, (sum(self.new), words), generator=g)
        for mask in (any_bits(self.mask.shape[1]), any_bits(1) & any_bits(1) & any_bits(1) & any_bits(1) & any_bits(1) & any_bits(1)):
            mask[::5] = 0
            mask[1::5, :-1] = 0                                   # of a tree without tokens before it: no key of the first page
            self.check(self.tree_attn(mask=mask.to("cuda"), **hints), mask=mask)


TILES = [  # total, new, H, G, splits
    ([26100], [256], 8, 2, 32), ([8800, 70, 170, 300], [170, 0, 170, 128], 9, 3, 8),
    ([900 - 7 * i for i in range(30)] + [128, 60], [128, 128, 77, 0, 1] * 6 + [128, 60], 16, 4, 1),
]


@pytest.mark.parametrize("type,D", [("fp16", 128), ("bf16", 64), ("fp16", 64), ("bf16", 128)])
@pytest.mark.parametrize("total,new,H,G,splits", TILES, ids=["one", "uneven", "whole"])
def test_tree_attention_by_tiles_of_128_rows(cuda, total, new, H, G, splits, type, D):
    b = Large(total, new, H, G, D, type, seed=len(total), wide=2)
    tile, _, n, *_ = _plan(b)
    assert (tile, n) == (128, splits)
    b.fill().check_all()


@pytest.mark.parametrize("type,D", [("fp16", 128), ("bf16", 64)])
@pytest.mark.parametrize("B,longest,most", [(32, 8300, 16), (70, 2000, 13)])
def test_tree_attention_longest_first_and_side_by_side(cuda, B, longest, most, type, D):
    rng = random.Random(B)
    total = [longest] + [min(longest - 1, int(40 * 1.2 ** rng.uniform(0, 20))) for _ in range(B - 1)]
    new = [most] + [rng.choice([0, 1, 5, most, most]) for _ in range(B - 1)]
    b = Large(total, new, 32, 8, D, type, seed=B, wide=1)
    tile, tiles, _, by_length, paired = _plan(b)
    assert tile == 32 and tiles == 2 and by_length and paired
    b.fill().check_all()
