"""The paged 4-bit cache on the GPU (ops.kv4_append, kv4_read, kv4_attn) against
the float64 restatement in oracle/kv4.py."""
import numpy as np
import pytest
import torch

from oracle import kv4 as plain

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _phases(n, D, theta=500000.0):
    inv = 1.0 / theta ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


class Batch:
    """A random batch: tokens of each sequence (`total`, the new ones among
    them), its new tokens, shuffled pages; `wide` more pages in every table row."""

    def __init__(self, total, new, H, G, D, type="fp16", seed=0, wide=0, spare=3, dev="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.total, self.new, self.H, self.G, self.D, self.type = total, new, H, G, D, TYPES[type]
        need = [max(1, (n + 63) // 64) for n in total]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g).int()
        self.table = torch.full((len(total), max(need) + wide), 1 << 30, dtype=torch.int32)  # no page
        at = 0
        for b, p in enumerate(need):
            self.table[b, :p] = order[at:at + p]
            at += p
        self.cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
        self.lens = torch.tensor(total, dtype=torch.int32)
        T = sum(new)
        x = lambda heads: torch.randn(T, heads, D, generator=g) * (1 + 4 * (torch.rand(heads, D, generator=g) < 0.05))
        self.q, self.k, self.v = x(H).to(self.type), x(G).to(self.type), x(G).to(self.type)
        self.phases = _phases(self.table.shape[1] * 64, D)
        # whatever bytes freed pages hold
        self.cache = torch.randint(0, 256, (self.n_pages, G, 68 * D), generator=g, dtype=torch.uint8)
        self.dev = dev

    def __getattr__(self, name):  # d_x: x on the device, once
        if name.startswith("d_"):
            t = getattr(self, name[2:]).to(self.dev)
            setattr(self, name, t)
            return t
        raise AttributeError(name)

    def fill(self, seed=1):
        """Valid random bytes (scales of ordinary size) for the sequences' tokens, garbage elsewhere."""
        g = torch.Generator().manual_seed(seed)
        D = self.D
        lens = {}
        for b, n in enumerate(self.total):
            for p in range(self.table.shape[1]):
                if self.table[b, p] < self.n_pages:
                    lens[int(self.table[b, p])] = max(0, min(64, n - 64 * p))
        for p, n in lens.items():
            ks = torch.randint(0x28, 0x38, (64, self.G, D // 32), generator=g, dtype=torch.uint8)
            vs = torch.randint(0x30, 0x3c, (64, self.G, D // 32), generator=g, dtype=torch.uint8)
            for t in range(n):
                blk = torch.arange(D // 32)
                self.cache[p][:, 32 * D + (blk * 16 + t % 16) * 4 + t // 16] = ks[t]
                e = t % 32 // 16 * 4 + t % 4
                self.cache[p][:, 66 * D + ((t // 4 % 4 * 2 + t // 32) * (D // 32) + blk) * 8 + e] = vs[t]
        return self

    def append(self, **kw):
        from shard_amd import ops
        return ops.kv4_append(kw.pop("k", self.d_k), kw.pop("v", self.d_v), self.d_cache, self.d_table, self.d_lens,
                              self.d_phases, cu_seqlens=kw.pop("cu_seqlens", self.d_cu), **kw)

    def read(self, n=None, **kw):
        from shard_amd import ops
        return ops.kv4_read(self.d_cache, self.d_table, kw.pop("lens", self.d_lens), self.k.shape[0] if n is None else n,
                            cu_seqlens=kw.pop("cu_seqlens", self.d_cu), **kw)

    def attn(self, **kw):
        from shard_amd import ops
        return ops.kv4_attn(kw.pop("q", self.d_q), self.d_cache, self.d_table, self.d_lens,
                            cu_seqlens=kw.pop("cu_seqlens", self.d_cu), **kw)

    def where(self):
        return list(plain.places(self.cu.tolist(), self.lens.tolist(), self.table.shape[1], len(self.total)))


SHAPES = [([1], [1], 4, 1, 128), ([64], [64], 8, 2, 128), ([65, 63, 1], [65, 63, 1], 8, 2, 64),
          ([200, 131, 7, 40], [3, 131, 0, 33], 6, 2, 128), ([97, 33, 320], [31, 33, 257], 8, 8, 64),
          ([500], [37], 4, 4, 128)]


@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("total,new,H,G,D", SHAPES, ids=str)
def test_append_and_read(cuda, total, new, H, G, D, type):
    b = Batch(total, new, H, G, D, type, seed=sum(total), wide=1)
    q = b.append(q=b.d_q)
    k, v = b.read(dtype=b.type)
    before_k, before_v = plain.held(b.cache.numpy())
    after_k, after_v = plain.held(b.d_cache.cpu().numpy())
    ph, table = b.phases.numpy(), b.table.numpy()
    touched = np.zeros(before_k.shape[:2], bool)
    for r, s, pos in b.where():
        page = plain.page_at(table, b.n_pages, s, pos)
        touched[page, pos % 64] = True
        for x, got, held in ((plain.rotate(b.k[r].double().numpy(), ph, pos), k, after_k), (b.v[r].double().numpy(), v, after_v)):
            want = plain.round4(x.reshape(G, -1, 32)).reshape(G, D)
            assert np.array_equal(held[page, pos % 64], want), (r, s, pos)
            assert np.array_equal(got[r].cpu().double().numpy(), want), (r, s, pos)
        want = plain.rotate(b.q[r].double().numpy(), ph, pos)
        size = np.abs(b.q[r].double().numpy())
        size = np.concatenate([size[:, :D // 2] + size[:, D // 2:]] * 2, -1)
        # two products and their sum in fp32 (2^-24 each of at most |x| + |y|), one rounding to the type
        # (and the type's smallest step below its normal range)
        tol = torch.finfo(b.type).eps / 2 * np.abs(want) + 2.0 ** -22 * size + 2.0 ** -25
        assert (np.abs(q[r].cpu().double().numpy() - want) <= tol).all()
    # tokens that were there before, and every page of nobody, as they were
    assert np.array_equal(before_k[~touched], after_k[~touched], equal_nan=True)
    assert np.array_equal(before_v[~touched], after_v[~touched], equal_nan=True)


@pytest.mark.parametrize("D", [64, 128])
def test_append_in_steps_gives_the_same_bytes(cuda, D):
    """Token by token (words of V codes shared with the token before), in
    uneven pieces, and at once."""
    from shard_amd import ops
    n = 75
    b = Batch([n], [n], 2, 2, D, seed=5)
    caches = []
    for step in (n, 1, 13):
        c = b.cache.to(cuda)
        for at in range(0, n, step):
            m = min(step, n - at)
            ops.kv4_append(b.d_k[at:at + m], b.d_v[at:at + m], c, b.d_table, torch.tensor([at + m], dtype=torch.int32, device=cuda),
                           b.d_phases, cu_seqlens=torch.tensor([0, m], dtype=torch.int32, device=cuda))
        caches.append(c.cpu())
    assert torch.equal(caches[0], caches[1]) and torch.equal(caches[0], caches[2])


@pytest.mark.parametrize("kw", [dict(max_new=1), dict(max_new=1000), dict()], ids=str)
def test_launch_hints_change_nothing(cuda, kw):
    """Whatever max_new says, all tokens are stored and read; block tables that are part of wider ones."""
    b = Batch([300, 64, 31], [290, 1, 30], 4, 2, 64, seed=14)
    want_q = b.append(q=b.d_q)
    want, (k, v) = b.d_cache.clone(), b.read()
    b.d_cache = b.cache.to(cuda)
    wide = torch.full((3, 40), 1 << 30, dtype=torch.int32, device=cuda)
    wide[:, 7:7 + b.table.shape[1]] = b.d_table
    b.d_table = wide[:, 7:7 + b.table.shape[1]]
    assert not b.d_table.is_contiguous()
    assert torch.equal(b.append(q=b.d_q, **kw), want_q) and torch.equal(b.d_cache, want)
    k2, v2 = b.read(**kw)
    assert torch.equal(k, k2) and torch.equal(v, v2)


def test_largest_launch_hints(cuda):
    """Hints far beyond what the call holds are only hints."""
    b = Batch([300, 64, 31], [290, 1, 30], 4, 2, 64, seed=15)
    want_q, want_out = b.append(q=b.d_q), b.attn()
    want, (k, v) = b.d_cache.clone(), b.read()
    b.d_cache = b.cache.to(cuda)
    hint = 2 ** 31 - 1
    assert torch.equal(b.append(q=b.d_q, max_new=hint), want_q) and torch.equal(b.d_cache, want)
    k2, v2 = b.read(max_new=hint)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    # the bits: old tokens are whatever random bytes say, NaN among them
    assert torch.equal(b.attn(max_new=hint, max_len=hint).view(torch.int16), want_out.view(torch.int16))


def test_append_strided_operands(cuda):
    """q, k and v as slices of one fused projection's rows, and rows at odd places."""
    b = Batch([70, 40], [50, 3], 4, 2, 128, seed=6)
    want_q = b.append(q=b.d_q)
    want = b.d_cache.clone()
    qkv = torch.cat([b.d_q.flatten(1), b.d_k.flatten(1), b.d_v.flatten(1)], 1)
    q, k, v = (x.unflatten(1, (-1, 128)) for x in qkv.split([512, 256, 256], 1))
    assert not k.is_contiguous()
    b.d_cache = b.cache.to(cuda)
    assert torch.equal(b.append(q=q, k=k, v=v), want_q) and torch.equal(b.d_cache, want)
    odd = torch.empty(b.k.numel() + 1, dtype=b.type, device=cuda)[1:].view(b.k.shape)
    odd.copy_(b.d_k)
    turned = b.d_v.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    b.d_cache = b.cache.to(cuda)
    b.append(k=odd, v=turned)
    assert torch.equal(b.d_cache, want)
    # one value a head, broadcast
    same = b.d_k[:, :1].expand(-1, 2, -1)
    b.append(k=same)
    again = b.d_cache.clone()
    b.append(k=same.contiguous())
    assert torch.equal(b.d_cache, again)


def test_append_specials(cuda):
    """NaN, infinities, zeros, subnormals and the largest numbers of the type."""
    for type in ("fp16", "bf16"):
        b = Batch([33], [33], 2, 1, 64, type, seed=7)
        big = torch.finfo(b.type).max
        vals = torch.tensor([np.nan, np.inf, -np.inf, 0.0, -0.0, big, -big, 1e-7, -6e-5, 1.0], dtype=torch.float64)
        g = torch.Generator().manual_seed(1)
        for t in (b.k, b.v):
            t[3:] = vals[torch.randint(0, len(vals), t[3:].shape, generator=g)].to(b.type)
        b.k[9], b.v[9] = 0, 0
        b.append()
        k, v = b.read(dtype=b.type)
        assert bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all())
        for r, s, pos in b.where():
            want_k = plain.round4(plain.rotate(b.k[r].double().numpy(), b.phases.numpy(), pos).reshape(1, 2, 32)).reshape(1, 64)
            want_v = plain.round4(b.v[r].double().numpy().reshape(1, 2, 32)).reshape(1, 64)
            assert np.array_equal(k[r].cpu().double().numpy(), want_k), (type, r)
            assert np.array_equal(v[r].cpu().double().numpy(), want_v), (type, r)


def test_tokens_without_a_place(cuda):
    """Lengths below the new tokens' number, below zero and past the table, pages
    outside the cache, rows past the last sequence: left out, nothing else touched."""
    b = Batch([130, 70, 190, 64], [10, 20, 20, 8], 4, 2, 128, seed=8).fill()
    b.lens = torch.tensor([130, 13, 201, -5], dtype=torch.int32)  # 7 tokens before 0; 9 past 3 pages of 64; none
    b.table[0, 2] = b.n_pages                                     # page of tokens 128, 129
    b.cu = torch.tensor([0, 10, 30, 50, 54], dtype=torch.int32)   # 58 rows, the last 4 nobody's
    before = plain.held(b.cache.numpy())
    q = b.append(q=b.d_q)
    after = plain.held(b.d_cache.cpu().numpy())
    k, v = b.read()
    ok = np.ones(before[0].shape[:2], bool)
    for r, s, pos in b.where():
        page = plain.page_at(b.table.numpy(), b.n_pages, s, pos)
        if page < 0:
            assert not k[r].any() and not v[r].any()
            if not 0 <= pos < 192:
                assert not q[r].any()
        else:
            ok[page, pos % 64] = False
            want = plain.round4(b.v[r].double().numpy().reshape(2, 4, 32)).reshape(2, 128)
            assert np.array_equal(after[1][page, pos % 64], want)
    assert (~ok).sum() == 8 + 13 + 11
    for x, y in zip(before, after):
        assert np.array_equal(x[ok], y[ok], equal_nan=True)
    out = torch.full_like(b.d_q, 7.0)
    b.attn(out=out)
    assert bool((out[54:] == 7).all()) and bool(torch.isfinite(out).all())
    assert not out[30 - 20:17].any() and not out[50:54].any()     # rows before position 0 and of no token
    _check_attention(b, out[:54], rows=54)


def _check_attention(b, out, rows=None, scale=None):
    scale = b.D ** -0.5 if scale is None else scale
    k, v = plain.held(b.d_cache.cpu().numpy())
    want, a, d = plain.attention(b.q.double().numpy(), k, v, b.table.numpy(), b.lens.tolist(), b.cu.tolist(), scale)
    want, a, d = want[:rows], a[:rows], d[:rows, :, None]
    n = max(b.total) + 64
    # scores: D products of exact operands summed in fp32, one scaling, one subtraction of the maximum (2^-24 each of
    # at most d); bf16 queries are held to 2^-26 of their row's largest.  They move a weight by twice their size, relative.
    # weights: fp16, 2^-11 each and 2^-25 below fp16's normal range; exp2, their sums and the joins of waves and splits
    # in fp32 (n + 200 roundings at most).  The output's own rounding comes last.
    weight = 2 * (b.D + 4) * 2.0 ** -24 * d + (2 * b.D * 2.0 ** -26 * d if b.type == torch.bfloat16 else 0)
    weight = weight + 2.0 ** -11 + n * 2.0 ** -25 + (n + 200) * 2.0 ** -24
    err = weight * 2 * a
    tol = err + torch.finfo(b.type).eps / 2 * (np.abs(want) + err) + 2.0 ** -25
    got = out.cpu().double().numpy()
    off = np.abs(got - want)
    assert (off <= tol).all(), (off.max(), (off / tol).max())
    print(f"attention: largest error {off.max():.2e}, {(off / tol).max():.2f} of the bound", flush=True)


ATTN = [  # total, new, H, G, D
    ([1], [1], 4, 1, 128), ([64], [1], 4, 4, 64), ([65], [1], 16, 1, 128), ([1000], [1], 12, 4, 128),
    ([3000, 1, 64, 517], [1, 1, 1, 1], 8, 2, 64), ([700, 90], [1, 1], 40, 2, 128),           # 20 query heads a kv head
    ([300, 77], [5, 2], 6, 2, 128), ([130, 500, 9], [9, 4, 9], 8, 2, 64), ([257], [8], 64, 1, 64),
    ([100], [100], 8, 2, 128), ([333, 64, 200], [333, 1, 130], 8, 2, 64), ([640], [200], 4, 4, 128),
    ([400, 50, 129, 1], [0, 50, 128, 1], 6, 2, 128), ([900], [513], 2, 1, 64),
]


@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("total,new,H,G,D", ATTN, ids=str)
def test_attention(cuda, total, new, H, G, D, type):
    b = Batch(total, new, H, G, D, type, seed=len(total) + H, wide=2).fill()
    one = set(new) == {1}
    for kw in (dict(), dict(max_new=max(new), max_len=max(total)), dict(max_new=1, max_len=1)):
        if one:
            kw["cu_seqlens"] = None
        _check_attention(b, b.attn(**kw))


FOLDED = [  # total, new, H, G, D: few rows a kv head and more than four pages a split
    ([400, 321], [1, 1], 256, 256, 64), ([417, 330], [2, 1], 512, 256, 64), ([500, 1], [1, 1], 1024, 256, 64),
    ([385, 200], [1, 1], 2048, 256, 64), ([400, 390], [2, 0], 768, 256, 64), ([338, 337], [3, 3], 256, 256, 64),
    ([2300], [1], 256, 64, 64), ([2300], [3], 128, 64, 64), ([700, 10, 64, 65, 330, 450, 129, 1], [1] * 8, 256, 64, 128),
    ([350, 10, 64, 65, 330, 450, 129, 1], [1] * 8, 448, 64, 128),
]


@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("total,new,H,G,D", FOLDED, ids=str)
def test_attention_few_rows_many_pages(cuda, total, new, H, G, D, type):
    """A column of the scores' tiles for every quarter of a page; hints below what the call holds too."""
    b = Batch(total, new, H, G, D, type, seed=len(total) + H, wide=2).fill()
    for kw in (dict(max_new=max(new)), dict(max_new=max(new), max_len=max(total)), dict(max_new=1)):
        if set(new) == {1}:
            kw["cu_seqlens"] = None
        _check_attention(b, b.attn(**kw))


@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("B,most,G,H,D", [(70, 1, 16, 64, 64), (130, 3, 8, 16, 64), (65, 9, 16, 32, 128), (64, 1, 32, 32, 64)], ids=str)
def test_attention_of_many_uneven_sequences(cuda, B, most, G, H, D, type):
    """Workgroups that take sequences by length: more than 64 of them, empty ones, equal lengths, hints too short."""
    g = torch.Generator().manual_seed(B)
    total = [int(n) for n in torch.randint(0, 200, (B,), generator=g)]
    total[3:9] = [0, 1, 64, 64, 64, 350]
    if most == 1:
        total = [max(n, 1) for n in total]
    new = [min(n, 1 + i % most) for i, n in enumerate(total)]
    b = Batch(total, new, H, G, D, type, seed=B, wide=1).fill()
    for kw in (dict(max_new=most, max_len=max(total)), dict(max_new=most), dict(max_new=1, max_len=30)):
        if most == 1:
            kw["cu_seqlens"] = None
        _check_attention(b, b.attn(**kw))


def test_attention_scale_and_large_scores(cuda):
    """Scores of hundreds: one key takes all; and a scale of 0: the mean."""
    b = Batch([200], [3], 8, 2, 128, seed=3).fill()
    _check_attention(b, b.attn(scale=0.0), scale=0.0)
    _check_attention(b, b.attn(scale=2.0), scale=2.0)
    _check_attention(b, b.attn(scale=-0.1), scale=-0.1)


@pytest.mark.parametrize("new", [3, 40])
def test_attention_scores_that_vanish(cuda, new):
    """bf16 queries of the smallest numbers and a scale that takes them below fp32's: all keys weigh the same."""
    b = Batch([100], [new], 8, 2, 64, "bf16", seed=15).fill()
    b.q *= 1e-39
    out = b.attn(scale=1e-20)
    assert bool(torch.isfinite(out).all())
    _check_attention(b, out, scale=1e-20)


def test_attention_specials(cuda):
    """A query row of NaN or infinity ruins its own row only; bf16 queries of any
    size are held; queries of zero attend evenly."""
    b = Batch([150], [20], 8, 2, 64, "bf16", seed=4).fill()
    b.q[0] = 0
    b.q[1] *= 1e-30
    b.q[2] *= 2.0 ** 20
    b.q[3, 0, 5], b.q[4, 1, 0] = float("nan"), float("inf")
    out = b.attn().cpu()
    assert bool(out[3, 0].isnan().all()) and bool(out[4, 1].isnan().all())
    keep = torch.ones(20, 8, dtype=torch.bool)
    keep[3, 0] = keep[4, 1] = False
    assert bool(torch.isfinite(out[keep]).all())
    b.q[3, 0], b.q[4, 1] = 0, 0
    again = b.attn(q=b.q.to(cuda)).cpu()
    assert torch.equal(again[keep], out[keep])
    out = again
    _check_attention(b, out)


def test_attention_pages_far_apart(cuda):
    """Pages past 4 GiB of the cache, pages shared by two sequences, and a cache
    whose pages are strided (one layer of a pool)."""
    from shard_amd import ops
    b = Batch([190, 130], [4, 1], 8, 2, 128, seed=9, spare=0).fill()
    b.table[1] = b.table[0]                                       # a shared prefix, both read only
    want = b.attn()
    _check_attention(b, want)
    pool = torch.empty(140_000, 2, 2, 68 * 128, dtype=torch.uint8, device=cuda)  # two layers: 4.9 GB
    assert (pool.shape[0] - 1) * pool.stride(0) > 1 << 32
    layer = pool[:, 1]
    far = torch.arange(pool.shape[0] - b.n_pages, pool.shape[0], device=cuda)
    layer[far] = b.d_cache
    table = far[b.d_table.clamp(max=b.n_pages - 1).long()].int()
    out = ops.kv4_attn(b.d_q, layer, table, b.d_lens, cu_seqlens=b.d_cu)
    assert torch.equal(out, want)
    # append there and read back, the other layer as it was
    mark = pool[far, 0].clone()
    new = Batch([190], [60], 8, 2, 128, seed=10)
    ops.kv4_append(new.d_k, new.d_v, layer, table[:1].contiguous(), new.d_lens, new.d_phases, cu_seqlens=new.d_cu)
    k, v = ops.kv4_read(layer, table[:1].contiguous(), new.d_lens, 60, cu_seqlens=new.d_cu)
    new.append()
    k2, v2 = new.read()
    assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(pool[far, 0], mark)


def test_attention_of_many_sequences_in_order_of_nothing(cuda):
    """A batch larger than the chip, every length from 0 on."""
    n = 300
    total = [(37 * i) % 211 for i in range(n)]
    b = Batch(total, [1] * n, 4, 2, 64, seed=11).fill()
    out = b.attn(cu_seqlens=None)
    assert not out[[i for i, t in enumerate(total) if t == 0]].any()
    _check_attention(b, out)


def test_streams_and_repeats(cuda):
    """The same bits every time, on another stream too."""
    b = Batch([2000, 700], [2, 2], 8, 2, 128, seed=12).fill()
    want = b.attn()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [b.attn() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)


def test_serving_loop_eager_and_captured(cuda):
    """A prompt appended and attended to, then decode steps: eager ones, and one
    step captured and replayed with the lengths in device memory; both give
    the same cache and outputs, those of the float64 restatement."""
    from shard_amd import ops
    H, G, D, steps, prompts = 8, 2, 128, 70, [100, 1, 63]
    full = Batch([p + steps for p in prompts], [p + steps for p in prompts], H, G, D, seed=13)
    B, dev = len(prompts), cuda
    rows = lambda x, lo, hi: torch.cat([x[int(full.cu[b]) + lo[b]:int(full.cu[b]) + hi[b]] for b in range(B)])
    step_in = [tuple(rows(x, [p + i for p in prompts], [p + i + 1 for p in prompts]) for x in (full.d_q, full.d_k, full.d_v))
               for i in range(steps)]

    def prefill(cache):
        q, k, v = (rows(x, [0] * B, prompts) for x in (full.d_q, full.d_k, full.d_v))
        cu = torch.tensor([0, 100, 101, 164], dtype=torch.int32, device=dev)
        lens = torch.tensor(prompts, dtype=torch.int32, device=dev)
        qr = ops.kv4_append(k, v, cache, full.d_table, lens, full.d_phases, q=q, cu_seqlens=cu)
        return ops.kv4_attn(qr, cache, full.d_table, lens, cu_seqlens=cu), lens

    def step(q, k, v, cache, lens):
        lens.add_(1)
        qr = ops.kv4_append(k, v, cache, full.d_table, lens, full.d_phases, q=q)
        return ops.kv4_attn(qr, cache, full.d_table, lens)

    eager, lens_e = torch.zeros_like(full.d_cache), None
    first, lens_e = prefill(eager)
    want = [step(*x, eager, lens_e) for x in step_in]

    captured = torch.zeros_like(full.d_cache)
    first2, lens_c = prefill(captured)
    assert torch.equal(first, first2)
    held_in = [t.clone() for t in step_in[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held_in, captured, lens_c)
    for i, x in enumerate(step_in):
        for dst, src in zip(held_in, x):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        assert bool(torch.randn(64, device=dev).isfinite().all())   # eager work between the replays
    assert torch.equal(captured, eager)
    # the whole against float64
    full.d_cache = eager
    every = torch.empty_like(full.q)
    for b in range(B):
        at = int(full.cu[b])
        s = sum(prompts[:b])
        every[at:at + prompts[b]] = first[s:s + prompts[b]].cpu()
        for i in range(steps):
            every[at + prompts[b] + i] = want[i][b].cpu()
    full.q = full.append(q=full.d_q).cpu()
    assert torch.equal(full.d_cache, captured)
    _check_attention(full, every)


def test_refusals(cuda):
    from shard_amd import ops
    b = Batch([70, 5], [2, 3], 4, 2, 128)
    c, t, n, ph = b.d_cache, b.d_table, b.d_lens, b.d_phases
    with pytest.raises(TypeError):
        b.append(k=b.d_k.float())
    with pytest.raises(TypeError):
        b.append(v=b.d_v.bfloat16())
    with pytest.raises(ValueError):
        b.append(k=b.d_k[:, :1])
    with pytest.raises(ValueError):
        b.append(v=b.d_v[:4])
    with pytest.raises(ValueError):
        b.append(cu_seqlens=None)                     # five tokens for two sequences
    with pytest.raises(TypeError):
        b.append(cu_seqlens=b.d_cu.long())
    with pytest.raises(TypeError):
        b.append(cu_seqlens=b.d_cu[:2])
    with pytest.raises(ValueError):
        ops.kv4_append(b.d_k, b.d_v, c, t, n, ph[:100], cu_seqlens=b.d_cu)
    with pytest.raises(TypeError):
        ops.kv4_append(b.d_k, b.d_v, c, t, n, ph.double(), cu_seqlens=b.d_cu)
    with pytest.raises(TypeError):
        b.attn(q=b.d_q.float())
    with pytest.raises(ValueError):
        b.attn(q=b.d_q[:, :3])                        # 3 query heads of 2 kv heads
    with pytest.raises(ValueError):
        b.attn(q=b.d_q[..., :64])
    with pytest.raises(TypeError):
        b.attn(out=b.d_q.new_empty(5, 4, 256)[..., ::2])
    with pytest.raises(TypeError):
        b.read(dtype=torch.float32)
    with pytest.raises(TypeError):
        ops.kv4_attn(b.d_q, c.view(torch.int8), t, n, cu_seqlens=b.d_cu)
    with pytest.raises(TypeError):
        ops.kv4_attn(b.d_q, c[..., :-1], t, n, cu_seqlens=b.d_cu)
    with pytest.raises(ValueError):
        ops.kv4_attn(b.d_q, c.transpose(0, 1).contiguous().transpose(0, 1), t, n, cu_seqlens=b.d_cu)
    with pytest.raises(TypeError):
        ops.kv4_attn(b.d_q, c, t.long(), n, cu_seqlens=b.d_cu)
    with pytest.raises(TypeError):
        ops.kv4_attn(b.d_q, c, t, n[:1], cu_seqlens=b.d_cu)
    with pytest.raises(ops.ShardHipUnavailable):
        ops.kv4_attn(b.d_q, c, b.table, n, cu_seqlens=b.d_cu)
    empty = b.d_q[:0]
    none = torch.zeros(3, dtype=torch.int32, device=cuda)
    assert b.attn(q=empty, cu_seqlens=none).shape == (0, 4, 128)
    assert b.append(k=b.d_k[:0], v=b.d_v[:0], q=empty, cu_seqlens=none).shape == (0, 4, 128)
    assert b.read(0, cu_seqlens=none)[0].shape == (0, 2, 128)


@pytest.mark.parametrize("type", ["fp16", "bf16"])
def test_compiled_and_plain_dispatch_agree(cuda, type, monkeypatch):
    """The compiled way and the one through Python give the same bits, and the
    compiled one takes plain calls."""
    from shard_amd import ops
    results = []
    for direct in (ops._bind_direct(), False):
        monkeypatch.setattr(ops, "_direct", direct)
        b = Batch([300, 64, 90], [20, 1, 90], 8, 2, 128, type, seed=16).fill()
        if direct:
            assert direct.kv4_attn(b.d_q, b.d_cache, b.d_table, b.d_lens, b.d_cu, None, 90, 300, 0, 0) is not None
        q = b.append(q=b.d_q)
        assert b.append() is None
        res = [q, b.d_cache, *b.read(dtype=b.type), *b.read(), b.attn(), b.attn(scale=0.3, max_new=90), b.attn(max_len=300)]
        x = torch.randn(3, 5000, generator=torch.Generator().manual_seed(1)).to(b.type).to(cuda)
        t = torch.tensor([1, 4999, 0], device=cuda)
        for y in (x, x[:, 3:], x[::2]):
            res += ops.token_logprobs(y, t[:y.shape[0]].clamp(max=4900), top=4)
            res += ops.token_logprobs(y, top=0)[1:]
        results.append(res)
    assert len(results[0]) == len(results[1])
    for x, y in zip(*results):
        assert x.dtype == y.dtype and x.shape == y.shape and x.device == y.device and torch.equal(x, y)


@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("n,new,H,G,D", [(8192, 1, 64, 64, 64), (8192, 1, 512, 64, 64), (8192, 3, 8, 1, 128), (8192, 4096, 32, 8, 64),
                                         (4096, 2048, 32, 8, 128)], ids=str)
@pytest.mark.parametrize("gap", [17.4, 22.7, 24.9, 27.0])
def test_attention_many_keys_far_below_one(cuda, n, new, H, G, D, type, gap):
    """One key has almost all of the weight and a value of zero (as models' first tokens have): the output is what
    thousands of keys, 2^-gap of its weight and less, add up to."""
    from shard_amd import ops
    g = torch.Generator().manual_seed(n + new)
    k, v = torch.zeros(n, D), torch.ones(n, D) * 0.5
    k[0, 0] = 6.0
    k[1:, 1] = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6])[torch.randint(0, 8, (n - 1,), generator=g)]
    v[1:, ::3] = torch.tensor([0.5, 1, 1.5, 2, 3])[torch.randint(0, 5, v[1:, ::3].shape, generator=g)]
    k[1:, 2], v[:, 31::32] = 6.0, 6.0                              # scale 1: every value is held as it is
    v[0] = 0
    q = torch.zeros(new, D)
    q[:, 0], q[:, 1] = 1, -1 / 64                                  # the other keys within 2^-(gap / 64) of each other
    dtype = TYPES[type]
    pages = n // 64
    cache = ops.kv4_cache(pages, G, D)
    table = torch.randperm(pages, generator=g).int()[None].to(cuda)
    lens, cu = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([n], [0, n]))
    still = torch.zeros(n, D // 2, 2, device=cuda)
    still[..., 0] = 1                                              # no rotation
    held = [x.to(cuda, dtype)[:, None].expand(n, G, D) for x in (k, v)]
    ops.kv4_append(*held, cache, table, lens, still, cu_seqlens=cu)
    assert all(torch.equal(a, b) for a, b in zip(ops.kv4_read(cache, table, lens, n, dtype=dtype, cu_seqlens=cu), held))
    scale = float(np.float32(gap * np.log(2) / 6))
    out = ops.kv4_attn(q.to(cuda, dtype)[:, None].expand(new, H, D), cache, table, lens, scale=scale, max_new=new, max_len=n,
                       cu_seqlens=torch.tensor([0, new], dtype=torch.int32, device=cuda))
    assert bool((out == out[:, :1]).all())                         # every head has the same
    rows = torch.arange(max(0, new - 64), new)
    s = q[rows].double() @ k.double().T * scale
    s = s.masked_fill(torch.arange(n) > (n - new + rows)[:, None], -np.inf)
    w = torch.softmax(s, -1)
    want = w @ v.double()
    # scores: the largest is gap ln 2 < 19, each off by (D + 4) 2^-24 of it.  Weights: fp16, 2^-11 each; below
    # 2^-25 of the largest 2^-36 of the largest, which is all but 1 of their sum.  Their sums as in _check_attention.
    rel = 2 * (D + 4) * 2.0 ** -24 * 19 + 2.0 ** -11 + (n + 200) * 2.0 ** -24
    err = 2 * rel * want + n * 2.0 ** -36 * float(v.max())
    off = (out[rows.to(cuda), 0].double().cpu() - want).abs()
    tol = err + torch.finfo(dtype).eps / 2 * (want + err) + 2.0 ** -25
    print(f"largest error {off.max():.2e}, {(off / tol).max():.2f} of the bound", flush=True)
    assert bool((off <= tol).all())


def test_scale_is_a_number(cuda):
    b = Batch([70], [3], 4, 2, 64).fill()
    for bad in (float("nan"), float("inf"), -float("inf"), 1e300):
        with pytest.raises(ValueError):
            b.attn(scale=bad)
        with pytest.raises(ValueError):
            b.attn(scale=bad, out=torch.empty_like(b.d_q))
    _check_attention(b, b.attn(scale=1), scale=1)


SLOW = r"""
#include <unistd.h>
#include "shard_hip.h"
extern "C" {
volatile int entered, go;
static int wait_for_go() {
  entered = 1;
  for (int i = 0; i < 3000 && !go; ++i) usleep(1000);
  return go ? 0 : -1;
}
uint64_t shard_kv4_args_layout(void) { return SHARD_KV4_ARGS_LAYOUT; }
int shard_kv4_append(const shard_kv4_args*, void*) { return wait_for_go(); }
int shard_kv4_read(const shard_kv4_args*, void*) { return wait_for_go(); }
size_t shard_kv4_attn_workspace(const shard_kv4_args*) { return 4096; }
int shard_kv4_attn(const shard_kv4_args*, void*, size_t, void*) { return wait_for_go(); }
size_t shard_token_logprobs_workspace(int64_t, int64_t, int32_t) { return 0; }
int shard_token_logprobs(const void*, int32_t, int64_t, int64_t, int64_t, const int64_t*, int32_t, float*, float*, float*, int64_t*,
                         void*, size_t, void*) { return wait_for_go(); }
}
"""


def test_other_threads_run_during_a_compiled_call(cuda, tmp_path):
    """A call that waits in the library (a full queue, say) leaves Python to the other threads.  The library is stood in
    for by one that launches nothing and waits, 3 s at most, for what only another thread can tell it."""
    import ctypes
    import os
    import subprocess
    import threading
    import time
    from conftest import ROOT
    from shard_amd import _lib, ops
    src, so = tmp_path / "slow.cpp", str(tmp_path / "slow.so")
    src.write_text(SLOW)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"), str(src), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    entered, go = (ctypes.c_int.in_dll(lib, name) for name in ("entered", "go"))
    b = Batch([70], [3], 4, 2, 64)
    d, st = ops._bind_direct(), torch.cuda.current_stream().cuda_stream
    x = torch.zeros(2, 50, device=cuda)
    args = b.d_cache, b.d_table, b.d_lens
    calls = [lambda: d.kv4_append(b.d_k, b.d_v, *args, b.d_phases, b.d_q, b.d_cu, None, 0, st),
             lambda: d.kv4_read(*args, 3, False, b.d_cu, None, 0, st),
             lambda: d.kv4_attn(b.d_q, *args, b.d_cu, None, None, None, 0, st),
             lambda: d.token_logprobs(x, None, 2, 0, st)]
    assert all(call() is not None for call in calls)    # with the library itself
    d.bind(so)
    try:
        for call in calls:
            entered.value = go.value = 0
            done = []
            t = threading.Thread(target=lambda: done.append(call()))
            t.start()
            while not entered.value and t.is_alive():
                time.sleep(0.001)
            go.value = 1
            t.join()
            assert done[0] is not None, "the call waited in vain"
    finally:
        d.bind(_lib.LIB_PATH)


def test_two_threads_at_once(cuda):
    """Each on its own stream and its own batch: the results of one after the other."""
    import threading
    from shard_amd import ops
    batches = [Batch([400, 77], [9, 2], 8, 2, 128, "fp16", seed=20).fill(), Batch([1000], [1], 8, 2, 64, "bf16", seed=21).fill()]
    x = [torch.randn(3, 9000, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2)]

    def work(i, n):
        b, out = batches[i], []
        for _ in range(n):
            q = b.append(q=b.d_q)
            out.append([q, b.attn(q=q), *b.read(dtype=b.type), *ops.token_logprobs(x[i], top=3)[1:]])
        return out
    for b in batches:
        b.append()
    want = [work(i, 1)[0] for i in range(2)]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got[i] = work(i, 50)
        s.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert all(torch.equal(a, b) for row in got[i] for a, b in zip(row, want[i]))


def _splits(b, **hints):
    """Splits that a call of the batch takes, from its workspace."""
    import ctypes
    from shard_amd import _lib
    a = _lib.KV4Args(batch=len(b.total), n_tokens=b.q.shape[0], n_q_heads=b.H, n_kv_heads=b.G, head_dim=b.D, n_pages=b.n_pages,
                     table_width=b.table.shape[1], cache=4096, page_stride=b.G * 68 * b.D, block_table=4096,
                     table_stride=b.table.shape[1], seq_lens=4096, cu_seqlens=4096, **hints)
    size = _lib.load().shard_kv4_attn_workspace(ctypes.byref(a))
    return size // (b.q.shape[0] * b.H * (b.D + 2) * 4)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("total,new,wide,splits,type", [
    ([8192], [1], 0, 32, "fp16"), ([16384], [1], 0, 64, "bf16"), ([32768], [1], 0, 128, "fp16"), ([24001], [2], 3, 128, "bf16"),
    ([300], [1], 507, 128, "fp16"), ([20000, 31000], [1, 3], 0, 128, "fp16")], ids=str)
def test_attention_joins_many_splits(cuda, total, new, wide, splits, type, D):
    """Up to 128 splits of a row, empty ones at the end; the heads' heaviest keys lie in splits of their own, at both
    sides of every 32: a split left out, or weighed as another, is off by most of the output."""
    H = 8
    b = Batch(total, new, H, 1, D, type, seed=splits + D, wide=wide, spare=1).fill()
    assert _splits(b) == splits
    K, _ = plain.held(b.cache.numpy())
    for r, s, pos in b.where():
        n = pos + 1
        per = max(4, -(-((total[s] + 63) // 64) // splits))               # pages of a split
        last = (n - 1) // (per * 64)
        for h, at in enumerate((0, 31, 32, 63, 64, 95, 96, last)):
            page = b.table[s, min(at, last) * per:][:per]
            keys = K[page[page < b.n_pages].long(), :, 0].reshape(-1, D)[:n - min(at, last) * per * 64]
            key = keys[(keys * keys).sum(-1).argmax()]
            # a score of 14, the others' a few either side of 0: a large part of the weight
            b.q[r, h] = torch.from_numpy(key * (14 / (key @ key) * D ** 0.5)).to(b.type)
    _check_attention(b, b.attn())
    _check_attention(b, b.attn(max_new=max(new), max_len=max(total)))


@pytest.mark.parametrize("type,size", [("fp16", 40.0), ("fp16", 3e3), ("fp16", 3e4), ("bf16", 3e4), ("bf16", 1e25)], ids=str)
@pytest.mark.parametrize("total,new,H,G,D", [([300, 90], [1, 1], 8, 2, 128), ([300], [20], 4, 1, 64), ([400, 200], [180, 200], 8, 4, 64),
                                             ([2300], [3], 128, 64, 64), ([300], [200], 4, 1, 128)], ids=str)
def test_attention_huge_scores(cuda, total, new, H, G, D, type, size):
    """Scores up to 1e9 and (bf16 queries) 1e30, far from each other: every row's weight is on its one best key, whatever
    fp32 leaves of the differences."""
    b = Batch(total, new, H, G, D, type, seed=17, wide=1)
    b.new = b.total                                                # every token is appended
    T = sum(total)
    cu = torch.tensor([sum(total[:i]) for i in range(len(total) + 1)], dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(3)
    k = (torch.sign(torch.randn(T, G, D, generator=g)) * min(size, 3e4)).to(b.type)
    v = torch.randn(T, G, D, generator=g).to(b.type)
    still = torch.zeros(b.table.shape[1] * 64, D // 2, 2, device=cuda)
    still[..., 0] = 1                                              # no rotation
    from shard_amd import ops
    ops.kv4_append(k.to(cuda), v.to(cuda), b.d_cache, b.d_table, b.d_lens, still, cu_seqlens=cu)
    want = torch.empty(b.q.shape, dtype=torch.float64)
    K, V = plain.held(b.d_cache.cpu().numpy())
    best = torch.randint(0, 1 << 30, (b.q.shape[0], H), generator=g)
    for r, s, pos in b.where():
        for h in range(H):
            t = int(best[r, h]) % (pos + 1)                        # its query: the key's own signs
            at = int(b.table[s, t // 64]), t % 64, h // (H // G)
            b.q[r, h] = torch.from_numpy(np.sign(K[at]) * size).to(b.type)
            want[r, h] = torch.from_numpy(V[at])
    # keys of random signs: the best key's score is D |q k| scale, any other's at least 8 |q k| scale less (4 signs apart;
    # 20 and more in fact), so that its weight is below e^-100 and the output the best key's value, times its weight in
    # fp16 over its weight in fp32 (2^-11), the division and one rounding to the type
    assert size * min(size, 3e4) * 8 * D ** -0.5 > 100
    out = b.attn().cpu()
    assert bool(out.isfinite().all())
    assert bool(((out.double() - want).abs() <= (2.0 ** -11 + torch.finfo(b.type).eps / 2 + 2.0 ** -21) * want.abs()).all())


@pytest.mark.parametrize("hint", [1 << 31, 1 << 40, 1 << 70, -1, -(1 << 40)])
def test_hints_of_any_size(cuda, hint):
    """Below zero is unknown, beyond 32 bits the largest: neither is an error, by either way through the calls."""
    b = Batch([130, 40], [30, 1], 4, 2, 64, seed=18).fill()
    want_q = b.append(q=b.d_q)
    want, read = b.attn(), b.read()
    assert torch.equal(b.append(q=b.d_q, max_new=hint), want_q)
    assert all(torch.equal(x, y) for x, y in zip(b.read(max_new=hint), read))
    assert torch.equal(b.attn(max_new=hint, max_len=hint), want)
