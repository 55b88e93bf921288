"""Operators of speculative decoding over a paged cache held in 4 bits.

A step of a sequence holds a tree of drafted tokens: its first row is the last
token that was decided on, every other row names its parent among the rows
before it.  Three kinds of case:

  attend  attention of the rows of such trees over the paged cache: a row sees
          the tokens before the tree, its ancestors and itself
          (ops.kv4_tree_attn).
  verify  the drafted tokens against the target model's logits, from given
          random numbers: the accepted path of each tree and the token that
          follows it (ops.verify_drafts).
  store   what surrounds the two in the cache: the tree's plan (ops.draft_tree),
          its keys and values rotated at the tree's positions and stored
          (ops.kv4_append), the accepted path moved to where the sequence goes
          on (ops.kv4_keep), in every layer, and what the cache then holds for
          it (ops.kv4_read).

The cache: pages of 64 tokens, (pages, kv heads, 68 * head_dim) bytes.  An
element is an E2M1 code (4 bits); 32 channels of a token share an E5M2 scale,
the smallest that is at least their largest magnitude / 6.5, from 2^-16 to
10240.  Codes go to the nearest value, ties to the even code, magnitudes above
6 scales saturate.  Within a page a kv head's bytes are K codes, K scales, V
codes, V scales, in the orders that _places() spells out.

Verification of a sequence starts at its first row.  p = softmax(logits /
temperature) of the row it is at; the row's children are tried in their order,
child c with token x and random number u = uniforms[c, 0]:

  drafted without probabilities   accepted where u * sum(s) < s[x], s = p at
                                  first; a rejected token's s becomes 0
  drafted from draft_probs[c] = q accepted where u * q[x] * sum(s) < s[x]; if
                                  not, s becomes max(s / sum(s) - q, 0) (unless
                                  that leaves nothing)

An accepted child is where it goes on.  Where none is accepted the answer is the
first token at which the cumulative sum of s exceeds uniforms[row, 1] * sum(s).
Temperature 0: p is 1 at the largest logit (the first of equal ones).

Inputs are seeded and made on the GPU; the trees' shapes and the sequences'
lengths go with the case.
"""
import functools
import math
import random

import torch

own = False

DEV = "cuda"
THETA = 500000.0
PAGE = 64
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    llama8b = dict(n_q=32, n_kv=8, hd=128)
    llama1b = dict(n_q=32, n_kv=8, hd=64)
    llama3b = dict(n_q=24, n_kv=8, hd=128)
    return [
        # one conversation with a small tree after a short prompt: latency
        dict(name="attend_1x2k_n8", kind="attend", batch=1, nodes=8, width=3, depth=4, spread=1, context=2048, type="fp16", **llama8b),
        # one conversation with the large tree that low load leaves room for
        dict(name="attend_1x8k_n61", kind="attend", batch=1, nodes=61, width=4, depth=7, spread=1, context=8192, type="fp16", **llama8b),
        # batch serving at the end-to-end run's sizes, small trees
        dict(name="attend_b16_16k_n16", kind="attend", batch=16, nodes=16, width=3, depth=5, spread=1, context=16384, type="bf16", **llama8b),
        # conversations of very uneven lengths and trees, head_dim 64
        dict(name="attend_b24_ragged", kind="attend", batch=24, nodes=33, width=4, depth=6, spread=16, context=8192, type="bf16", **llama1b),
        # trees of several mask words, 3 query heads per kv head
        dict(name="attend_n200_gqa3", kind="attend", batch=2, nodes=200, width=8, depth=9, spread=2, context=5003, type="fp16", **llama3b),
        # one conversation with a chain of four drafted tokens: latency
        dict(name="verify_chain5", kind="verify", batch=1, nodes=5, width=1, depth=4, spread=1, vocab=128256, probs=False, temperature=0.8, type="fp16"),
        # one conversation with a large tree
        dict(name="verify_tree61", kind="verify", batch=1, nodes=61, width=4, depth=7, spread=1, vocab=128256, probs=False, temperature=1.0, type="bf16"),
        # chains sampled from a draft model, whose probabilities count
        dict(name="verify_b32_probs", kind="verify", batch=32, nodes=6, width=1, depth=5, spread=1, vocab=128256, probs=True, temperature=0.7, type="bf16"),
        # a serving batch with small uneven trees, greedy and sampling sequences together
        dict(name="verify_b64_trees", kind="verify", batch=64, nodes=26, width=3, depth=6, spread=2, vocab=128256, probs=False, temperature="mixed", type="bf16"),
        # one conversation's small tree through one layer: latency
        dict(name="store_1_n8", kind="store", layers=1, batch=1, nodes=8, width=3, depth=4, spread=1, context=2048, type="fp16", **llama8b),
        # a serving batch's trees through all layers
        dict(name="store_b64_n26_l32", kind="store", layers=32, batch=64, nodes=26, width=3, depth=6, spread=2, context=500, type="bf16", **llama8b),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "verify", "verify", "store"])
    c = dict(kind=kind, width=rng.randint(2, 8), depth=rng.randint(1, 9), spread=rng.choice([1, 2, 16]))
    if kind == "verify":
        c["probs"] = rng.random() < 0.4
        c["width"] = rng.choice([1, 1, 2, 4]) if c["probs"] else rng.choice([1, 2, 4, 8])
        c["nodes"] = _log(rng, 1, 64)
        c["vocab"] = _log(rng, 500, 128256)
        c["type"] = rng.choice(["fp16", "bf16", "fp32"])
        most = 150_000_000 // (2 if c["type"] == "fp32" else 1) // (3 if c["probs"] else 1)
        c["batch"] = _log(rng, 1, max(1, min(64, most // (c["nodes"] * c["vocab"]))))
        c["temperature"] = rng.choice([0.0, "mixed", rng.uniform(0.3, 1.5), rng.uniform(0.3, 1.5)])
        return c
    c["n_q"], c["n_kv"], c["hd"] = rng.choice([(32, 8, 128), (32, 8, 128), (32, 8, 64), (24, 8, 128), (8, 2, 128), (32, 4, 64), (8, 8, 128)])
    c["type"] = rng.choice(["fp16", "bf16"])
    c["batch"] = _log(rng, 1, 32)
    c["nodes"] = _log(rng, 2, min(256, 2048 // c["batch"]))
    if kind == "store":
        c["layers"] = _log(rng, 1, max(1, min(32, 40_000 // (c["batch"] * c["nodes"]))))
        c["context"] = c["nodes"] + _log(rng, 1, 600)
    else:
        c["context"] = c["nodes"] + _log(rng, 1, min(16384, 4_000_000 // (c["batch"] * c["nodes"])))
    return c


def _lengths(case):
    """Tokens of each sequence, its tree's rows among them, and the rows:
    log-uniform between the case's sizes and their `spread`-th part."""
    rng = random.Random(case.get("context", 0) * 131 + case["batch"])
    least = lambda n: max(1, n // case["spread"])
    new = [case["nodes"]] + [_log(rng, least(case["nodes"]), case["nodes"]) for _ in range(case["batch"] - 1)]
    if "context" not in case:
        return new, new
    total = [case["context"]] + [_log(rng, least(case["context"]), case["context"]) for _ in range(case["batch"] - 1)]
    return [max(a, n) for a, n in zip(total, new)], new


def _trees(case):
    """The rows' parents of each sequence: at most `width` children a row, `depth` levels below the first row
    (as many as it takes to hold all rows)."""
    rng = random.Random(case["nodes"] * 977 + case["width"] * 31 + case["depth"])
    trees = []
    for n in _lengths(case)[1]:
        parents, depth, free, limit = [-1], [0], [case["width"]], case["depth"]
        while len(parents) < n:
            open_ = [i for i in range(len(parents)) if free[i] and depth[i] < limit]
            if not open_:
                limit += 1
                continue
            p = rng.choice(open_[-32:])
            free[p] -= 1
            parents.append(p)
            depth.append(depth[p] + 1)
            free.append(case["width"])
        trees.append(parents)
    return trees


def _paths(case):
    """Accepted rows of each tree, from its first row down."""
    rng = random.Random(case["nodes"] * 37 + case["batch"])
    paths = []
    for parents in _trees(case):
        path = [0]
        while rng.random() < 0.8:
            children = [i for i, p in enumerate(parents) if p == path[-1]]
            if not children:
                break
            path.append(rng.choice(children))
        paths.append(path)
    return paths


# ---------------------------------------------------------------------------
# the cache's bytes
# ---------------------------------------------------------------------------
def _places(t, hd):
    """Byte places within a kv head's part of a page for its tokens t (any
    shape): K codes (..., hd) [the low 4 bits are the even channel], K scales
    (..., hd / 32), V codes (..., hd) [the low 4 bits are the even token], V
    scales (..., hd / 32)."""
    t = t.unsqueeze(-1)
    c = torch.arange(hd, device=t.device)
    blk = torch.arange(hd // 32, device=t.device)
    sub, r = t // 16, t % 16
    lane = hd // 8                                   # bytes of a quarter of a token's channels
    kq, ki = c // (hd // 4), c % (hd // 4)
    per = 16 // lane                                 # 16-token groups side by side in 16 bytes
    k = (sub // per * 64 + kq * 16 + r) * 16 + sub % per * lane + ki // 2
    ks = 32 * hd + (blk * 16 + r) * 4 + sub
    s, u = t // 32, t % 32
    e, vq = u // 16 * 4 + u % 4, u // 4 % 4
    n, cc = c // 16, c % 16
    v = 34 * hd + (((s * (hd // 64) + n // 4) * 64 + vq * 16 + cc) * 4 + n % 4) * 4 + e // 2
    vs = 66 * hd + ((vq * 2 + s) * (hd // 32) + blk) * 8 + e
    return k, ks, v, vs


@functools.lru_cache(maxsize=None)
def _scales(device):
    """The 113 scales, 2^-16 .. 10240: value i - 1 belongs to byte i."""
    b = torch.arange(1, 114, device=device)
    return torch.where(b < 4, b * 2.0 ** -16, (4 + b % 4) * torch.exp2((b // 4 - 17).double()))


@functools.lru_cache(maxsize=None)
def _levels(device):
    m = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=device, dtype=torch.float64)
    return torch.cat([m, -m])


def _round4(x):
    """x (T, G, hd) in 64 bits -> codes (T, G, hd), scale bytes (T, G, hd / 32), values in 64 bits."""
    x = torch.nan_to_num(x, nan=0.0, posinf=1e30, neginf=-1e30).unflatten(-1, (-1, 32))
    a = x.abs()
    sc = _scales(x.device)
    at = torch.searchsorted(sc * 6.5, a.amax(-1)).clamp_(max=112)
    s = sc[at].unsqueeze(-1)
    m = ((a > 0.25 * s).byte() + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s) + (a > 2.5 * s) + (a >= 3.5 * s) + (a > 5 * s))
    codes = m | (x < 0).byte() << 3
    values = _levels(x.device)[codes.long()] * s
    return codes.flatten(-2), (at + 1).byte(), values.flatten(-2)


def _at(cache, page, slot, hd):
    """Places in the whole cache of tokens at page, slot (T): K codes, K scales, V codes, V scales, (T, G, ...) each."""
    g = torch.arange(cache.shape[1], device=cache.device)
    base = ((page[:, None] * cache.shape[1] + g) * cache.shape[2]).unsqueeze(-1)
    return [p.unsqueeze(1) + base for p in _places(slot, hd)]


def _write(cache, page, slot, kc, ks, vc, vs):
    """The codes and scales of tokens (T, G, ...) into their pages, those that share a byte one after the other."""
    flat = cache.view(-1)
    pk, pks, pv, pvs = _at(cache, page, slot, kc.shape[-1])
    flat[pk[..., 0::2]] = kc[..., 0::2] | kc[..., 1::2] << 4
    flat[pks] = ks
    flat[pvs] = vs
    even = (slot % 2 == 0).view(-1, 1, 1)
    spare = flat.numel() - 1                          # the spare page's last byte
    for_even, for_odd = pv.where(even, pv.new_tensor(spare)), pv.where(~even, pv.new_tensor(spare))
    flat[for_even] = flat[for_even] & 0xF0 | vc
    flat[for_odd] = flat[for_odd] & 0x0F | vc << 4


def _codes(cache, page, slot, hd):
    """What _write takes, of the tokens that the cache holds at page, slot (T)."""
    flat = cache.view(-1)
    pk, pks, pv, pvs = _at(cache, page, slot, hd)
    odd = (torch.arange(hd, device=cache.device) % 2 * 4).byte()
    return flat[pk] >> odd & 15, flat[pks], flat[pv] >> (slot % 2 * 4).byte()[:, None, None] & 15, flat[pvs]


def _values(cache, page, slot, hd):
    """K and V (T, G, hd) fp32 that the cache holds for tokens at page, slot (T)."""
    kc, ks, vc, vs = _codes(cache, page, slot, hd)
    level, scale = _levels(cache.device).float(), torch.cat([_scales(cache.device).new_zeros(1), _scales(cache.device)]).float()
    return tuple(level[c.int()] * scale[s.int()].repeat_interleave(32, -1) for c, s in ((kc, ks), (vc, vs)))


# ---------------------------------------------------------------------------
# inputs: made from the seed alone
# ---------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _tokens(g, n, heads, hd, type):
    """Rows with a few channels several times larger than the rest, as keys and queries have them."""
    size = 1 + 4 * (torch.rand(heads, hd, generator=g, device=DEV) < 0.05)
    return (_randn(g, n, heads, hd) * size).to(TYPES[type])


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _batch(case, g):
    """A batch of trees: where each sequence's rows begin, their parents, and their block table."""
    total, new = _lengths(case)
    trees = _trees(case)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    st = dict(case=case, cu=_int(cu), parents=_int([p for t in trees for p in t]), max_new=max(new), max_len=max(total))
    st["seq"] = torch.arange(case["batch"], device=DEV).repeat_interleave(torch.tensor(new, device=DEV))
    st["row"] = torch.arange(cu[-1], device=DEV) - st["cu"][st["seq"]]
    if case["kind"] == "verify":
        return st, trees
    width, each = (max(total) + PAGE - 1) // PAGE, [(n + PAGE - 1) // PAGE for n in total]
    pages = sum(each)
    order = torch.randperm(pages, generator=g, device=DEV)
    table = torch.zeros(case["batch"], width, dtype=torch.int32, device=DEV)
    at = 0
    for b, p in enumerate(each):
        table[b, :p] = order[at:at + p]
        at += p
    st["table"], st["lens"] = table, _int(total)
    st["first"] = st["lens"] - st["cu"].diff()             # where each sequence's rows begin in its cache
    # one page more than the sequences have
    st["cache"] = torch.zeros(case.get("layers", 1), pages + 1, case["n_kv"], 68 * case["hd"], dtype=torch.uint8, device=DEV)
    return st, trees


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + 7)
    st, trees = _batch(case, g)
    T = len(st["seq"])
    if case["kind"] == "verify":
        return _prepare_verify(case, st, trees, g)
    G, hd, type = case["n_kv"], case["hd"], case["type"]
    lens = st["lens"].long()
    if case["kind"] == "store":
        L, W = case["layers"], st["table"].shape[1]
        st["phases"] = _phases(W * PAGE, hd)
        # all layers' pages as one cache: a table row for every layer of every sequence
        per = st["cache"].shape[1]
        st["all_table"] = (st["table"] + torch.arange(L, device=DEV, dtype=torch.int32)[:, None, None] * per).flatten(0, 1)
        st["all_lens"] = st["lens"].repeat(L)
        layer = torch.arange(L, device=DEV, dtype=torch.int32)[:, None]
        last = lambda cu, n: torch.cat([(cu[:-1] + layer * n).flatten(), cu.new_tensor([L * n])])
        st["all_cu"] = last(st["cu"], T)
        paths = _paths(case)
        P = max(len(p) for p in paths)
        st["rows"], st["counts"] = _int([p + [-1] * (P - len(p)) for p in paths]), _int([len(p) for p in paths])
        kept = torch.cat([st["counts"].new_zeros(1), st["counts"].cumsum(0, dtype=torch.int32)])
        st["kept_rows"] = sum(len(p) for p in paths) * L
        st["kept_lens"], st["kept_cu"] = (st["first"] + st["counts"]).repeat(L), last(kept, sum(len(p) for p in paths))
        for name in "kv":
            st[name] = _tokens(g, L * T, G, hd, type)
        return st
    seq = torch.arange(case["batch"], device=DEV).repeat_interleave(lens)
    at = torch.arange(len(seq), device=DEV) - (lens.cumsum(0) - lens)[seq]
    for part in torch.arange(len(seq), device=DEV).split(65536):  # so that making it stays small
        kc, ks, _ = _round4(_tokens(g, len(part), G, hd, "fp32").double())
        vc, vs, _ = _round4(_randn(g, len(part), G, hd).double())
        _write(st["cache"][0], st["table"][seq[part], at[part] // PAGE].long(), at[part] % PAGE, kc, ks, vc, vs)
    st["q"] = _tokens(g, T, case["n_q"], hd, type)
    # each row's ancestors and itself as bits, 64 rows of its sequence a word: a step's plan, the same for every layer
    mask = []
    for parents in trees:
        bits = []
        for i, p in enumerate(parents):
            bits.append(1 << i | (bits[p] if p >= 0 else 0))
        mask += bits
    words = (st["max_new"] + 63) // 64
    signed = lambda x: x - (1 << 64) if x >> 63 else x
    st["mask"] = torch.tensor([[signed(m >> 64 * w & (1 << 64) - 1) for w in range(words)] for m in mask], device=DEV)
    return st


def _prepare_verify(case, st, trees, g):
    n, v, cu = len(st["seq"]), case["vocab"], st["cu"].tolist()
    x = _randn(g, n, v) * 2.5
    x.scatter_add_(1, torch.randint(0, v, (n, 1), generator=g, device=DEV), torch.rand(n, 1, generator=g, device=DEV) * 15)
    st["logits"] = x.to(TYPES[case["type"]])
    t = case["temperature"]
    if t == "mixed":
        t = torch.rand(case["batch"], generator=g, device=DEV) * 1.2 + 0.2
        t[::3] = 0.0
    st["temperature"] = t
    # each row's children, and its place among its parent's
    children, order, st["levels"] = [[] for _ in range(n)], [0] * n, 0
    for b, parents in enumerate(trees):
        depth = [0]
        for i, p in enumerate(parents[1:], 1):
            depth.append(depth[p] + 1)
            order[cu[b] + i] = len(children[cu[b] + p])
            children[cu[b] + p].append(cu[b] + i)
        st["levels"] = max([st["levels"]] + depth)
    most = max(1, max(len(c) for c in children))
    st["children"] = torch.tensor([c + [-1] * (most - len(c)) for c in children], device=DEV)
    parent = (st["cu"][st["seq"]] + st["parents"].clamp(min=0)).long()
    order = torch.tensor(order, device=DEV)
    draft = x
    draft += _randn(g, n, v) * (0.7 if case["probs"] else 1.5)  # what a draft model thinks after each row
    if case["probs"]:
        warm = t if isinstance(t, float) else 0.7
        q = torch.softmax(draft / (warm or 1.0), -1)
        noise = torch.rand(n, v, generator=g, device=DEV).clamp_(min=1e-30).log_().neg_().clamp_(min=1e-30)
        st["probs"] = q[parent]
        st["tokens"] = (st["probs"] / noise).argmax(-1)
    else:
        st["probs"] = None
        st["tokens"] = draft.topk(min(most, v), -1).indices[parent, order.clamp(max=v - 1)]
    st["uniforms"] = torch.rand(n, 2, generator=g, device=DEV)
    return st


@functools.lru_cache(maxsize=4)
def _phases(n, hd):
    """(n, hd / 2, 2) fp32: cosine and sine of each position's angles."""
    inv = 1.0 / THETA ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _ancestors(st):
    """(T, max_new) truth values: which rows of its sequence a row sees; (T) its depth."""
    T = len(st["seq"])
    parent = torch.where(st["parents"] >= 0, st["cu"][st["seq"]] + st["parents"], -1).long()
    seen = torch.zeros(T, st["max_new"], dtype=torch.bool, device=DEV)
    depth, at, all_rows = torch.full((T,), -1, device=DEV), torch.arange(T, device=DEV), torch.arange(T, device=DEV)
    for _ in range(st["max_new"]):
        on = at >= 0
        seen[all_rows, st["row"][at.clamp(min=0)]] |= on
        depth += on
        at = torch.where(on, parent[at.clamp(min=0)], -1)
    return seen, depth


def _plain_attend(st):
    q, lens = st["q"], st["lens"].long()
    T, H, hd = q.shape
    B, G = lens.numel(), st["cache"].shape[2]
    keys = torch.arange(st["max_len"], device=q.device)
    page = st["table"].long()[:, keys // PAGE]
    k, v = _values(st["cache"][0], page.flatten(), (keys % PAGE).repeat(B), hd)       # (B * keys, G, hd)
    k, v = (x.view(B, -1, G, hd).transpose(1, 2) for x in (k, v))
    k, v = k.transpose(2, 3).contiguous(), v.contiguous()
    rows = q.new_zeros(B, st["max_new"], H, hd, dtype=torch.float32)
    rows[st["seq"], st["row"]] = q.float()
    rows = rows.view(B, -1, G, H // G, hd).transpose(1, 2).reshape(B, G, -1, hd)
    s = (rows @ k).view(B, G, -1, H // G, st["max_len"]) / math.sqrt(hd)
    bits = st["mask"][:, torch.arange(st["max_new"], device=DEV) // 64] >> torch.arange(st["max_new"], device=DEV) % 64 & 1
    node = keys - st["first"][:, None]                                                # of each sequence's keys
    seen = torch.zeros(B, st["max_new"], st["max_len"], dtype=torch.bool, device=DEV)
    mine = bits.gather(1, node.clamp(0, st["max_new"] - 1)[st["seq"]]).bool() & (node < st["max_new"])[st["seq"]]
    seen[st["seq"], st["row"]] = ((node < 0)[st["seq"]] | mine) & (keys < lens[:, None])[st["seq"]]
    s.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    p = p / p.sum(-1, keepdim=True).clamp_(min=1e-30)
    o = (p.view(B, G, -1, st["max_len"]) @ v).view(B, G, -1, H // G, hd).transpose(1, 2).reshape(B, -1, H, hd)
    return o[st["seq"], st["row"]].to(q.dtype)


def _plain_verify(st):
    B, P = st["cu"].numel() - 1, st["max_new"]
    x, tokens, u, children = st["logits"].double(), st["tokens"], st["uniforms"].double(), st["children"]
    T, v = x.shape
    t = st["temperature"]
    t = (t.double() if isinstance(t, torch.Tensor) else torch.full((B,), t, dtype=torch.float64, device=DEV).float().double())[st["seq"], None]
    largest = x.amax(-1, keepdim=True)
    index = torch.arange(v, device=DEV)
    first = torch.where(x == largest, index, v).amin(-1, keepdim=True)
    w = torch.where(t > 0, ((x - largest) / torch.where(t > 0, t, 1.0)).exp(), (index == first).double())
    each, at = torch.arange(B, device=DEV), st["cu"][:-1].long()
    rows = torch.full((B, P), -1, dtype=torch.int32, device=DEV)
    rows[:, 0] = 0
    counts = torch.ones(B, dtype=torch.int32, device=DEV)
    s, going = w[at], torch.ones(B, dtype=torch.bool, device=DEV)
    for level in range(1, st["levels"] + 1):
        taken = torch.zeros_like(going)
        for c in range(children.shape[1]):
            child = children[at, c]
            trying = going & ~taken & (child >= 0)
            child = child.clamp(min=0)
            token, total = tokens[child], s.sum(-1)
            here = s[each, token]
            drafted = st["probs"][child].double() if st["probs"] is not None else None
            bar = u[child, 0] * total if drafted is None else u[child, 0] * drafted[each, token] * total
            yes = trying & (bar < here)
            no = trying & ~yes
            if drafted is None:
                s = torch.where(no[:, None] & (index == token[:, None]), 0.0, s)
            else:
                left = (s / total[:, None] - drafted).clamp(min=0)
                s = torch.where((no & (left.sum(-1) > 0))[:, None], left, s)
            taken |= yes
            chosen = torch.where(yes, child, at) if c == 0 else torch.where(yes, child, chosen)
        at = torch.where(taken, chosen, at)
        s = torch.where(taken[:, None], w[at], s)
        rows[:, level] = torch.where(taken, st["row"][at].int(), -1)
        counts += taken
        going = going & taken
    sums = s.cumsum(-1)
    return {"rows": rows, "counts": counts, "next": (sums <= u[at, 1:] * sums[:, -1:]).sum(-1)}


def _rotated(x, phases, pos):
    lo, hi = x.double().chunk(2, -1)
    c, s = phases[pos].double().unsqueeze(1).unbind(-1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def _plain_store(st):
    L, T, hd = st["case"]["layers"], len(st["seq"]), st["case"]["hd"]
    seen, depth = _ancestors(st)
    positions = st["first"][st["seq"]] + depth
    words = (st["max_new"] + 63) // 64
    mask = torch.zeros(T, words * 64, dtype=torch.int64, device=DEV)
    mask[:, :st["max_new"]] = seen
    mask = (mask.view(T, words, 64) << torch.arange(64, device=DEV)).sum(-1)
    flat = st["cache"].flatten(0, 1)
    layer = torch.arange(L, device=DEV)[:, None]
    of = lambda seq, pos: (st["all_table"].long()[(layer * (st["cu"].numel() - 1) + seq).flatten(), (pos // PAGE).repeat(L)], (pos % PAGE).repeat(L))
    page, slot = of(st["seq"], st["first"][st["seq"]] + st["row"])
    kc, ks, _ = _round4(_rotated(st["k"], st["phases"], positions.repeat(L)))
    vc, vs, _ = _round4(st["v"].double())
    _write(flat, page, slot, kc, ks, vc, vs)
    # the accepted rows, one after the other from the first row's place on
    seq, j = torch.nonzero(st["rows"] >= 0, as_tuple=True)
    held = _codes(flat, *of(seq, st["first"][seq] + st["rows"][seq, j]), hd)
    to = of(seq, st["first"][seq] + j)
    _write(flat, *to, *held)
    k, v = _values(flat, *to, hd)
    return {"mask": mask, "positions": positions.int(), "k": k.to(st["k"].dtype), "v": v.to(st["k"].dtype)}


def run(st):
    kind = st["case"]["kind"]
    if not own:
        return {"attend": _plain_attend, "verify": _plain_verify, "store": _plain_store}[kind](st)
    from shard_amd import ops
    if kind == "attend":
        return ops.kv4_tree_attn(st["q"], st["cache"][0], st["table"], st["lens"], st["mask"], cu_seqlens=st["cu"],
                                 max_new=st["max_new"], max_len=st["max_len"])
    if kind == "verify":
        rows, counts, tokens = ops.verify_drafts(st["logits"], st["tokens"], st["parents"], st["uniforms"], cu_seqlens=st["cu"],
                                                 draft_probs=st["probs"], temperature=st["temperature"], max_new=st["max_new"],
                                                 max_depth=st["levels"])
        return {"rows": rows, "counts": counts, "next": tokens}
    mask, positions = ops.draft_tree(st["parents"], st["lens"], cu_seqlens=st["cu"], max_new=st["max_new"])
    flat = st["cache"].flatten(0, 1)
    ops.kv4_append(st["k"], st["v"], flat, st["all_table"], st["all_lens"], st["phases"], cu_seqlens=st["all_cu"],
                   max_new=st["max_new"], positions=positions.repeat(st["case"]["layers"]))
    ops.kv4_keep(st["cache"], st["table"], st["lens"], st["rows"], st["counts"], cu_seqlens=st["cu"])
    k, v = ops.kv4_read(flat, st["all_table"], st["kept_lens"], st["kept_rows"], dtype=st["k"].dtype, cu_seqlens=st["kept_cu"],
                        max_new=st["rows"].shape[1])
    return {"mask": mask, "positions": positions, "k": k, "v": v}


def work(case):
    total, new = _lengths(case)
    if case["kind"] == "verify":
        n, v = sum(new), case["vocab"]
        size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["type"]]
        # of the draft's probabilities one row a sequence, of the token that is rejected
        return {"bytes": n * (v * size + 24) + case["batch"] * (v * 4 * case["probs"] + 12 + 4 * max(new)), "flops": 4 * n * v}
    H, G, hd = case["n_q"], case["n_kv"], case["hd"]
    held = G * hd * 68 // 64                                     # bytes of a token's K and V in the cache
    if case["kind"] == "store":
        n, kept, words = sum(new), sum(map(len, _paths(case))), (max(new) + 63) // 64
        moved = sum(i != j for path in _paths(case) for j, i in enumerate(path))
        return {"bytes": n * (4 + 8 * words + 4) + case["layers"] * (n * (4 * G * hd + held) + moved * 2 * held + kept * (held + 4 * G * hd)) + n * 4 * hd,
                "flops": case["layers"] * n * 2 * G * hd * 6}
    pairs = 0
    for t, parents in zip(total, _trees(case)):
        depth = []
        for p in parents:
            depth.append(depth[p] + 1 if p >= 0 else 1)
        pairs += len(parents) * (t - len(parents)) + sum(depth)
    return {"bytes": sum(total) * held + sum(new) * (2 * 2 * H * hd + 8 * ((max(new) + 63) // 64)), "flops": 4 * H * hd * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _nearest(x):
    """E2M1 times an E5M2 scale for every 32 channels, from the formats' exponents."""
    rows = x.reshape(-1, 32)
    most = rows.abs().amax(1, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2((most / 6.5).clamp(min=2.0 ** -40))).clamp(min=-14) - 2)  # the scale's last place
    s = unit * torch.ceil(most / 6.5 / unit)
    s = torch.where((s - unit) * 6.5 >= most, s - unit, torch.where(s * 6.5 < most, s + unit, s)).clamp(2.0 ** -16, 10240.0)
    a = rows.abs() / s
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return ((torch.round(a / step) * step).clamp(max=6.0) * s * rows.sign()).view(x.shape)


def _unpacked(pages, hd):
    """A kv head's pages (P, 68 hd) as K and V (P * 64, hd) in 64 bits, by taking the bytes' order apart."""
    P = pages.shape[0]
    nib = lambda b: torch.stack([b & 15, b >> 4], -1).flatten(-2)
    level = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=pages.device)
    e5m2 = lambda b: torch.where(b < 4, b.double() * 2.0 ** -16, (1 + (b & 3).double() / 4) * torch.exp2((b >> 2).double() - 15))
    kc, ks, vc, vs = (t.contiguous() for t in pages.split([32 * hd, 2 * hd, 32 * hd, 2 * hd], 1))
    per = 128 // hd                                    # groups of 16 tokens in a lane's 16 bytes
    k = nib(kc.view(P, 4 // per, 4, 16, per, hd // 8)).permute(0, 1, 4, 3, 2, 5).reshape(P, 64, hd)
    ks = e5m2(ks.view(P, hd // 32, 16, 4).permute(0, 3, 2, 1).reshape(P, 64, hd // 32))
    v = nib(vc.view(P, 2, hd // 64, 4, 16, 4, 4))      # step, 64 channels, 4 tokens of 16, channel, 16 channels, places
    v = v.view(P, 2, hd // 64, 4, 16, 4, 2, 4).permute(0, 1, 6, 3, 7, 2, 5, 4).reshape(P, 64, hd)
    vs = e5m2(vs.view(P, 4, 2, hd // 32, 2, 4).permute(0, 2, 4, 1, 5, 3).reshape(P, 64, hd // 32))
    k, v = (level[c.int()].view(P, 64, hd // 32, 32) * s.unsqueeze(-1) for c, s in ((k, ks), (v, vs)))
    return k.reshape(-1, hd), v.reshape(-1, hd)


def _exact_verify(case, st):
    cu, tokens, u = st["cu"].tolist(), st["tokens"].tolist(), st["uniforms"].double().cpu().tolist()
    t = st["temperature"]
    temps = t.tolist() if isinstance(t, torch.Tensor) else torch.full((case["batch"],), t).tolist()
    rows, counts, answers = [], [], []
    for b, parents in enumerate(_trees(case)):
        path, row = [], 0
        while row is not None:
            path.append(row)
            x = st["logits"][cu[b] + row].double()
            if temps[b] > 0:
                p = torch.softmax(x / temps[b], 0)
            else:
                p = torch.nn.functional.one_hot(torch.nonzero(x == x.max())[0, 0], len(x)).double()
            following = None
            for c in (i for i, parent in enumerate(parents) if parent == row and i):
                token = tokens[cu[b] + c]
                if case["probs"]:
                    q = st["probs"][cu[b] + c].double()
                    if u[cu[b] + c][0] * float(q[token]) < float(p[token]):
                        following = c
                        break
                    rest = torch.relu(p - q)
                    p = rest / rest.sum() if float(rest.sum()) > 0 else p
                else:
                    if u[cu[b] + c][0] < float(p[token]):
                        following = c
                        break
                    rest = p.clone()
                    rest[token] = 0
                    p = rest / rest.sum()
            if following is None:
                up_to = p.cumsum(0)
                answers.append(int(torch.searchsorted(up_to, u[cu[b] + row][1] * up_to[-1], right=True)))
            row = following
        counts.append(len(path))
        rows.append(path + [-1] * (st["max_new"] - len(path)))
    return {"rows": _int(rows), "counts": _int(counts), "next": torch.tensor(answers, device=DEV)}


def _exact_store(case, st):
    T, L = len(st["seq"]), case["layers"]
    mask, positions, kept = [], [], []
    words, first, cu = (st["max_new"] + 63) // 64, st["first"].tolist(), st["cu"].tolist()
    for b, (parents, path) in enumerate(zip(_trees(case), _paths(case))):
        for i in range(len(parents)):
            line = {i}
            while parents[min(line)] >= 0:
                line.add(parents[min(line)])
            mask.append([sum(1 << i % 64 for i in line if i // 64 == w) for w in range(words)])
            positions.append(first[b] + len(line) - 1)
        kept += [cu[b] + i for i in path]
    mask = torch.tensor([[m - (1 << 64) if m >> 63 else m for m in row] for row in mask], device=DEV)
    positions = _int(positions)
    kept = (torch.tensor(kept, device=DEV) + torch.arange(L, device=DEV)[:, None] * T).flatten()
    z = torch.view_as_complex(st["phases"].double())[positions[kept % T]].unsqueeze(1)
    half = case["hd"] // 2
    x = torch.complex(st["k"][kept][..., :half].double(), st["k"][kept][..., half:].double()) * z
    return {"mask": mask, "positions": positions, "k": _nearest(torch.cat([x.real, x.imag], -1)), "v": _nearest(st["v"][kept].double())}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(case, st)
    if case["kind"] == "store":
        return _exact_store(case, st)
    total, new = _lengths(case)
    hd, G = case["hd"], case["n_kv"]
    outs, at = [], 0
    for b, (n, parents) in enumerate(zip(total, _trees(case))):
        m = len(parents)
        pages = st["cache"][0][st["table"][b, :(n + PAGE - 1) // PAGE].long()]
        tree = torch.eye(m, dtype=torch.bool)
        for i, p in enumerate(parents):
            if p >= 0:
                tree[i] |= tree[p]
        seen = torch.cat([torch.ones(m, n - m, dtype=torch.bool), tree], 1).to(DEV)
        heads = []
        for h in range(G):
            k, v = _unpacked(pages[:, h], hd)
            q = st["q"][at:at + m].unflatten(1, (G, -1))[:, h].double()          # (m, group, hd)
            s = torch.einsum("mgd,td->mgt", q, k[:n]) * hd ** -0.5
            w = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
            heads.append(torch.einsum("mgt,td->mgd", w, v[:n]))
        outs.append(torch.cat(heads, 1))
        at += m
    return torch.cat(outs)
