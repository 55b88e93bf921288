"""Operators of a serving step over a paged cache held in 4 bits, and of its answer.

Three kinds of case:

  append    new tokens of a batch: q and k rotated at their positions, k and v
            rounded to 4 bits and written into the sequences' pages
            (ops.kv4_append), then those tokens' K and V as the cache now holds
            them (ops.kv4_read).
  attend    causal attention of a batch's newest tokens over their paged cache
            (ops.kv4_attn): one token a sequence, a few, or whole prompts.
  logprobs  log probabilities of given tokens, the entropy of each row and its
            most probable tokens, from a batch of logits (ops.token_logprobs).

The cache: pages of 64 tokens, (pages, kv heads, 68 * head_dim) bytes.  An
element is an E2M1 code (4 bits); 32 channels of a token share an E5M2 scale,
the smallest that is at least their largest magnitude / 6.5, from 2^-16 to
10240.  Codes go to the nearest value, ties to the even code, magnitudes above
6 scales saturate.  Within a page a kv head's bytes are K codes, K scales, V
codes, V scales, in the orders that _places() spells out.

Inputs are seeded and made on the GPU.
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
        # the new token of one interactive conversation
        dict(name="append_1", kind="append", batch=1, new=1, spread=1, context=8192, type="fp16", **llama8b),
        # one token for each of 64 conversations of uneven lengths, head_dim 64
        dict(name="append_b64_ragged", kind="append", batch=64, new=1, spread=1, context=5003, type="bf16", **llama1b),
        # four prompts of the prefill benchmark's length, the whole batch at once
        dict(name="append_b4_8k", kind="append", batch=4, new=8192, spread=1, context=8192, type="fp16", **llama8b),
        # one conversation after a short prompt: latency
        dict(name="attend_1x2k", kind="attend", batch=1, new=1, spread=1, context=2048, type="fp16", **llama8b),
        # one long conversation
        dict(name="attend_1x32k", kind="attend", batch=1, new=1, spread=1, context=32768, type="fp16", **llama8b),
        # batch serving at the end-to-end run's sizes
        dict(name="attend_b16_16k", kind="attend", batch=16, new=1, spread=1, context=16384, type="fp16", **llama8b),
        # many conversations of very uneven lengths, head_dim 64
        dict(name="attend_b64_ragged", kind="attend", batch=64, new=1, spread=64, context=8192, type="bf16", **llama1b),
        # four sequences whose five drafted tokens are verified, 3 query heads per kv head
        dict(name="attend_draft5_gqa3", kind="attend", batch=4, new=5, spread=2, context=5003, type="fp16", **llama3b),
        # one chunk of a long prompt's prefill
        dict(name="attend_chunk512_16k", kind="attend", batch=1, new=512, spread=1, context=16384, type="bf16", **llama8b),
        # a whole prompt
        dict(name="attend_prompt_8k", kind="attend", batch=1, new=8192, spread=1, context=8192, type="fp16", **llama8b),
        # the chosen token of one decode step with its five best alternatives
        dict(name="logprobs_1", kind="logprobs", rows=1, vocab=128256, top=5, masked=False, type="fp16"),
        # a 2048-token text scored (perplexity), with 20 alternatives a token
        dict(name="logprobs_2k", kind="logprobs", rows=2048, vocab=128256, top=20, masked=False, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "logprobs"])
    if kind == "logprobs":
        rows = _log(rng, 1, 2048)
        return dict(kind=kind, rows=rows, vocab=_log(rng, 500, 128256), top=rng.choice([0, 1, 5, 20]),
                    masked=rng.random() < 0.3, type=rng.choice(["fp16", "bf16", "fp32"]))
    n_q, n_kv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (32, 8, 64), (24, 8, 128), (8, 2, 128), (32, 4, 64), (8, 8, 128)])
    c = dict(kind=kind, n_q=n_q, n_kv=n_kv, hd=hd, type=rng.choice(["fp16", "bf16"]))
    if kind == "append":
        c["batch"] = _log(rng, 1, 64)
        c["new"] = rng.choice([1, _log(rng, 1, 16384 // c["batch"])])
        c["context"] = max(c["new"], _log(rng, 1, 16384))
        c["spread"] = rng.choice([1, 2, 16])
        return c
    how = rng.choice(["one", "few", "chunk"])
    if how == "one":
        c["batch"] = _log(rng, 1, 64)
        c["new"], c["context"] = 1, _log(rng, 1, min(32768, 196608 // c["batch"]))
    elif how == "few":
        c["batch"] = _log(rng, 1, 16)
        c["new"] = rng.randint(2, 12)
        c["context"] = c["new"] + _log(rng, 1, 8192)
    else:
        c["batch"] = rng.choice([1, 1, 2, 3])
        c["new"] = _log(rng, 13, 4096 // c["batch"])
        c["context"] = c["new"] + _log(rng, 1, 4096) - 1
    c["spread"] = rng.choice([1, 1, 2, 16])
    return c


def _lengths(case):
    """Tokens of each sequence, the new ones among them, and its new tokens:
    log-uniform between the case's sizes and their `spread`-th part."""
    rng = random.Random(case["context"] * 131 + case["batch"])
    least = lambda n: max(1, n // case["spread"])
    new = [case["new"]] + [_log(rng, least(case["new"]), case["new"]) for _ in range(case["batch"] - 1)]
    total = [case["context"]] + [_log(rng, least(case["context"]), case["context"]) for _ in range(case["batch"] - 1)]
    return [max(a, n) for a, n in zip(total, new)], new


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


def _write(cache, page, slot, kc, ks, vc, vs):
    """The codes and scales of tokens (T, G, ...) into their pages, those that share a byte one after the other."""
    hd = kc.shape[-1]
    flat, g = cache.view(-1), torch.arange(cache.shape[1], device=cache.device)[:, None]
    base = (page[:, None] * cache.shape[1] + g.T).unsqueeze(-1) * cache.shape[2]
    pk, pks, pv, pvs = (p.unsqueeze(1) + base for p in _places(slot, hd))
    flat[pk[..., 0::2]] = kc[..., 0::2] | kc[..., 1::2] << 4
    flat[pks] = ks
    flat[pvs] = vs
    even = (slot % 2 == 0).view(-1, 1, 1)
    spare = flat.numel() - 1                          # the spare page's last byte
    for_even, for_odd = pv.where(even, pv.new_tensor(spare)), pv.where(~even, pv.new_tensor(spare))
    flat[for_even] = flat[for_even] & 0xF0 | vc
    flat[for_odd] = flat[for_odd] & 0x0F | vc << 4


def _held(cache, page, slot, hd):
    """K and V (..., G, hd) fp32 that the cache holds for tokens at page, slot (...)."""
    flat, g = cache.view(-1), torch.arange(cache.shape[1], device=cache.device)
    base = (page.unsqueeze(-1) * cache.shape[1] + g).unsqueeze(-1) * cache.shape[2]
    pk, pks, pv, pvs = (p.unsqueeze(-2) + base for p in _places(slot, hd))
    odd = torch.arange(hd, device=cache.device) % 2 * 4
    level, scale = _levels(cache.device).float(), torch.cat([_scales(cache.device).new_zeros(1), _scales(cache.device)]).float()
    k = level[(flat[pk] >> odd & 15).int()] * scale[flat[pks].int()].repeat_interleave(32, -1)
    v = level[(flat[pv] >> (slot % 2 * 4)[..., None, None] & 15).int()] * scale[flat[pvs].int()].repeat_interleave(32, -1)
    return k, v


# ---------------------------------------------------------------------------
# inputs: made from the seed alone
# ---------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _tokens(g, n, heads, hd, type):
    """Rows with a few channels several times larger than the rest, as keys and queries have them."""
    size = 1 + 4 * (torch.rand(heads, hd, generator=g, device=DEV) < 0.05)
    return (_randn(g, n, heads, hd) * size).to(TYPES[type])


def _batch(case, g):
    """Pages of a batch of sequences: their block table, lengths and where each new token goes."""
    total, new = _lengths(case)
    width = (max(total) + PAGE - 1) // PAGE
    pages = sum((n + PAGE - 1) // PAGE for n in total)
    order = torch.randperm(pages, generator=g, device=DEV)
    table = torch.zeros(case["batch"], width, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(total):
        p = (n + PAGE - 1) // PAGE
        table[b, :p] = order[at:at + p]
        at += p
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    seq = torch.arange(case["batch"], device=DEV).repeat_interleave(torch.tensor(new, device=DEV))
    lens = torch.tensor(total, dtype=torch.int32, device=DEV)
    pos = torch.arange(len(seq), device=DEV) - cu[seq] + (lens - cu.diff())[seq]
    # one page more than the sequences have
    cache = torch.zeros(pages + 1, case["n_kv"], 68 * case["hd"], dtype=torch.uint8, device=DEV)
    return dict(case=case, table=table, lens=lens, cu=None if max(new) == 1 else cu, seq=seq, pos=pos, cache=cache,
                max_new=max(new), max_len=max(total))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + 5)
    if case["kind"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        x = _randn(g, n, v) * 2.5
        x.scatter_add_(1, torch.randint(0, v, (n, 1), generator=g, device=DEV), torch.rand(n, 1, generator=g, device=DEV) * 15)
        tokens = torch.where(torch.rand(n, generator=g, device=DEV) < 0.5, x.argmax(-1),
                             torch.randint(0, v, (n,), generator=g, device=DEV))
        if case["masked"]:  # tokens that a grammar excludes
            x.masked_fill_(torch.rand(n, v, generator=g, device=DEV) < 0.4, -math.inf)
            x[:, 0] = 0.0
        return dict(case=case, logits=x.to(TYPES[case["type"]]), tokens=tokens)
    st = _batch(case, g)
    G, hd, type = case["n_kv"], case["hd"], case["type"]
    if case["kind"] == "append":
        st["phases"] = _phases(st["table"].shape[1] * PAGE, hd)
        for name, heads in (("q", case["n_q"]), ("k", G), ("v", G)):
            st[name] = _tokens(g, len(st["seq"]), heads, hd, type)
        return st
    lens = st["lens"].long()
    seq = torch.arange(case["batch"], device=DEV).repeat_interleave(lens)
    at = torch.arange(len(seq), device=DEV) - (lens.cumsum(0) - lens)[seq]
    for part in torch.arange(len(seq), device=DEV).split(65536):  # so that making it stays small
        kc, ks, _ = _round4(_tokens(g, len(part), G, hd, "fp32").double())
        vc, vs, _ = _round4(_randn(g, len(part), G, hd).double())
        _write(st["cache"], st["table"][seq[part], at[part] // PAGE].long(), at[part] % PAGE, kc, ks, vc, vs)
    st["q"] = _tokens(g, len(st["seq"]), case["n_q"], hd, type)
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
def _rotated(x, phases, pos):
    lo, hi = x.double().chunk(2, -1)
    c, s = phases[pos].double().unsqueeze(1).unbind(-1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def _plain_append(st):
    k, v = st["k"], st["v"]
    page, slot = st["table"][st["seq"], st["pos"] // PAGE].long(), st["pos"] % PAGE
    kc, ks, kv = _round4(_rotated(k, st["phases"], st["pos"]))
    vc, vs, vv = _round4(v.double())
    _write(st["cache"], page, slot, kc, ks, vc, vs)
    return {"q": _rotated(st["q"], st["phases"], st["pos"]).to(st["q"].dtype), "k": kv.to(k.dtype), "v": vv.to(v.dtype)}


def _plain_attend(st):
    q, lens = st["q"], st["lens"].long()
    T, H, hd = q.shape
    B, G = lens.numel(), st["cache"].shape[1]
    keys = torch.arange(st["max_len"], device=q.device)
    page = st["table"].long()[:, keys // PAGE]
    k, v = _held(st["cache"], page, (keys % PAGE).expand(B, -1), hd)            # (B, keys, G, hd)
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    # the new tokens of each sequence in rows of one length, its last row its last token
    row = st["pos"] - lens[st["seq"]] + st["max_new"]
    rows = q.new_zeros(B, st["max_new"], H, hd, dtype=torch.float32)
    rows[st["seq"], row] = q.float()
    rows = rows.view(B, -1, G, H // G, hd).transpose(1, 2).reshape(B, G, -1, hd)
    s = (rows @ k).view(B, G, -1, H // G, st["max_len"]) / math.sqrt(hd)
    last = lens[:, None] - st["max_new"] + torch.arange(st["max_new"], device=q.device)
    s.masked_fill_((keys > last.unsqueeze(-1))[:, None, :, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(B, G, -1, st["max_len"]) @ v).view(B, G, -1, H // G, hd).transpose(1, 2).reshape(B, -1, H, hd)
    return o[st["seq"], row].to(q.dtype)


def _plain_logprobs(st):
    x, n = st["logits"].float(), st["case"]["top"]
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    lse = total.log()
    out = {"logprob": (d.gather(1, st["tokens"][:, None]) - lse)[:, 0],
           "entropy": lse[:, 0] - (e * d.clamp(min=-1e4)).sum(-1) / total[:, 0]}
    if n:  # by value, then by index: whole numbers that order the same way
        bits = st["logits"].float().view(torch.int32).long()
        bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        v = x.shape[1]
        ids = v - 1 - (bits * v + (v - 1 - torch.arange(v, device=x.device))).topk(n, -1).values % v
        out["top_ids"], out["top_logprobs"] = ids, d.gather(1, ids) - lse
    return out


def run(st):
    kind = st["case"]["kind"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[kind](st)
    from shard_amd import ops
    if kind == "append":
        q = ops.kv4_append(st["k"], st["v"], st["cache"], st["table"], st["lens"], st["phases"], q=st["q"],
                           cu_seqlens=st["cu"], max_new=st["max_new"])
        k, v = ops.kv4_read(st["cache"], st["table"], st["lens"], st["k"].shape[0], dtype=st["k"].dtype,
                            cu_seqlens=st["cu"], max_new=st["max_new"])
        return {"q": q, "k": k, "v": v}
    if kind == "attend":
        return ops.kv4_attn(st["q"], st["cache"], st["table"], st["lens"], cu_seqlens=st["cu"], max_new=st["max_new"],
                            max_len=st["max_len"])
    logprob, entropy, top_logprobs, top_ids = ops.token_logprobs(st["logits"], st["tokens"], top=st["case"]["top"])
    out = {"logprob": logprob, "entropy": entropy}
    if st["case"]["top"]:
        out["top_ids"], out["top_logprobs"] = top_ids, top_logprobs
    return out


def work(case):
    if case["kind"] == "logprobs":
        n, size = case["rows"], {"fp16": 2, "bf16": 2, "fp32": 4}[case["type"]]
        return {"bytes": n * (case["vocab"] * size + 16 + 12 * case["top"]), "flops": 5 * n * case["vocab"]}
    total, new = _lengths(case)
    H, G, hd = case["n_q"], case["n_kv"], case["hd"]
    held = G * hd * 68 // 64                                     # bytes of a token's K and V in the cache
    if case["kind"] == "append":
        n = sum(new)                                             # written and read back: the cache's bytes twice
        return {"bytes": n * (2 * (2 * H + 2 * G + 2 * G) * hd + 4 * hd + 2 * held), "flops": n * (H + 2 * G) * hd * 6}
    pairs = sum(n * t - n * (n - 1) // 2 for t, n in zip(total, new))
    return {"bytes": sum(total) * held + sum(new) * 2 * 2 * H * hd, "flops": 4 * H * hd * pairs}


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


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logprobs":
        out = {"logprob": [], "entropy": [], "top_ids": [], "top_logprobs": []}
        for x, tok in zip(st["logits"].split(256), st["tokens"].split(256)):
            x = x.double()
            lp = x - torch.logsumexp(x, -1, keepdim=True)
            out["logprob"].append(lp[torch.arange(len(tok), device=DEV), tok])
            out["entropy"].append(-torch.where(lp == -math.inf, 0.0, lp.exp() * lp).sum(-1))
            if case["top"]:
                _, ids = torch.sort(x, descending=True, stable=True)
                out["top_ids"].append(ids[:, :case["top"]].contiguous())
                out["top_logprobs"].append(lp.gather(1, out["top_ids"][-1]))
        return {name: torch.cat(parts) for name, parts in out.items() if parts}
    total, new = _lengths(case)
    hd, G = case["hd"], case["n_kv"]
    if case["kind"] == "append":
        z = torch.view_as_complex(st["phases"].double())[st["pos"]].unsqueeze(1)
        turned = {}
        for name in "qk":
            x = torch.complex(st[name][..., :hd // 2].double(), st[name][..., hd // 2:].double()) * z
            turned[name] = torch.cat([x.real, x.imag], -1)
        return {"q": turned["q"], "k": _nearest(turned["k"]), "v": _nearest(st["v"].double())}
    outs, at = [], 0
    for b, (n, m) in enumerate(zip(total, new)):
        pages = st["cache"][st["table"][b, :(n + PAGE - 1) // PAGE].long()]
        heads = []
        for h in range(G):
            k, v = _unpacked(pages[:, h], hd)
            q = st["q"][at:at + m].unflatten(1, (G, -1))[:, h].double()          # (m, group, hd)
            s = torch.einsum("mgd,td->mgt", q, k[:n]) * hd ** -0.5
            seen = torch.arange(n, device=DEV) <= torch.arange(n - m, n, device=DEV)[:, None]
            w = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
            heads.append(torch.einsum("mgt,td->mgd", w, v[:n]))
        outs.append(torch.cat(heads, 1))
        at += m
    return torch.cat(outs)
