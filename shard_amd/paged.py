"""A paged KV cache held in 4 bits that serves batches of uneven sequences.

`Cache` compresses once, after prompts of one length.  A `PagedCache` takes
tokens as they come: each sequence owns pages of 64 tokens (E2M1 codes with an
E5M2 scale for 32 channels, 4.25 bits an element), new ones join and finished
ones leave between steps, and a step may hold one token of some sequences and
whole prompts of others.  Per layer a step is two calls: ops.kv4_append (RoPE
of q and k, 4-bit rounding, writing) and ops.kv4_attn.

    enable_llama_fused_attention(model)
    cache = PagedCache.from_model(model, n_pages=4096, max_len=32768)
    a, b = cache.add(), cache.add()
    logits = cache.run(model, [a, b], [prompt_a, prompt_b])       # (2, vocab), of the last tokens
    logits = cache.run(model, [a, b], logits.argmax(-1, keepdim=True))
    cache.drop(a)

The tokens of a step are packed in rows, one sequence after the other; there is
no padding and no attention mask.  A step is open from begin() until every layer
has stored its tokens (run() does both); one that will not come to that is undone
by cancel(), as no other can begin over tokens that are not there.
"""
import torch
from transformers.cache_utils import Cache as HFCache, CacheLayerMixin

from . import host, ops
from .ops import KV4_PAGE


class PagedLayer(CacheLayerMixin):
    """Stands for a layer where transformers asks for one; the pages are the cache's."""

    is_sliding = False
    is_compileable = False

    def __init__(self, cache):
        self._cache = cache
        self.is_initialized = True

    def update(self, key_states, value_states, *args, **kwargs):
        raise RuntimeError("a PagedCache is read and written by the patched attention: "
                           "call enable_llama_fused_attention first")

    def get_seq_length(self):
        return 0

    def get_max_length(self):
        return -1

    def get_max_cache_shape(self):
        return None

    def get_mask_sizes(self, query_length, *args, **kwargs):
        return query_length, 0

    def lazy_initialization(self, *args, **kwargs):
        pass

    def _rows(self, *args, **kwargs):
        raise RuntimeError("a PagedCache has sequences, not rows of a batch: add(), drop() and run() by their numbers")

    reset = reorder_cache = crop = batch_repeat_interleave = batch_select_indices = _rows


class PagedCache(HFCache):
    def __init__(self, n_pages, max_len, head_dim=128, num_layers=32, n_kv_heads=8, device="cuda", rope_inv_freq=None,
                 rope_scale=1.0):
        """n_pages pages of every layer, shared by all sequences; a sequence holds
        at most max_len tokens.  rope_inv_freq (head_dim / 2,), rope_scale a
        factor of the rotation (1 for Llama)."""
        if max_len <= 0 or n_pages <= 0 or num_layers <= 0:
            raise ValueError("max_len, n_pages and num_layers must be positive")
        self.max_len = max_len
        self.pool = ops.kv4_cache(num_layers * n_pages, n_kv_heads, head_dim, device).unflatten(0, (num_layers, n_pages))
        width = (max_len + KV4_PAGE - 1) // KV4_PAGE
        inv = rope_inv_freq if rope_inv_freq is not None else 1.0 / 10000.0 ** (torch.arange(0, head_dim, 2) / head_dim)
        self.phases = ops.rope_phases(0, width * KV4_PAGE, inv.to(device, torch.float32))
        if rope_scale != 1.0:
            self.phases *= rope_scale
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages, self._lens, self._next = {}, {}, 0
        self._step = None
        super().__init__(layers=[PagedLayer(self) for _ in range(num_layers)])

    @classmethod
    def from_model(cls, model, n_pages, max_len):
        cfg = model.config
        rot = getattr(getattr(model, "model", None), "rotary_emb", None)
        kind = getattr(rot, "rope_type", "default")
        if kind not in ("default", "linear", "llama3", "yarn"):
            raise ValueError(f"rope type {kind!r} changes its frequencies with the length; the cache rotates once")
        hd = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
        return cls(n_pages, max_len, head_dim=hd, num_layers=cfg.num_hidden_layers,
                   n_kv_heads=getattr(cfg, "num_key_value_heads", cfg.num_attention_heads),
                   device=next(model.parameters()).device, rope_inv_freq=host.get_rope_inv_freq(model),
                   rope_scale=float(getattr(rot, "attention_scaling", 1.0)))

    # -- sequences ---------------------------------------------------------
    def add(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._lens[seq] = [], 0
        return seq

    def drop(self, seq):
        """Give a sequence's pages back.  A step that is open for it is undone, for
        all its sequences; one of other sequences stays open."""
        if seq not in self._pages:
            raise KeyError(seq)
        step = self._open()
        if step is not None and any(s == seq for s, _, _ in step["undo"]):
            self._undo()
        self._free += reversed(self._pages.pop(seq))
        del self._lens[seq]

    def length(self, seq) -> int:
        return self._lens[seq]

    def free_pages(self) -> int:
        return len(self._free)

    def device_bytes(self) -> int:
        return self.pool.numel() + self.phases.numel() * 4

    # -- a step ------------------------------------------------------------
    def _open(self):
        """The step that some layer has not stored yet, or None."""
        return self._step if self._step is not None and self._step["left"] else None

    def begin(self, seqs, new):
        """Open a step in which sequence seqs[i] gets new[i] tokens (0 allowed),
        packed in this order.  Pages are taken here: RuntimeError where too few are
        free; ValueError while another step is open; a call that fails, for
        whatever reason, changes nothing.  Returns the tokens' positions, (1, T)."""
        if self._open():
            raise ValueError("a step is open: run its layers or cancel() it")
        seqs, new = list(seqs), [int(n) for n in new]
        if len(seqs) != len(new) or not seqs or len(set(seqs)) != len(seqs) or min(new) < 0 or max(new) == 0:
            raise ValueError("a step needs distinct sequences and at least one new token")
        total = [self._lens[s] + n for s, n in zip(seqs, new)]
        if max(total) > self.max_len:
            raise ValueError(f"a sequence would hold {max(total)} tokens, max_len is {self.max_len}")
        want = [(t + KV4_PAGE - 1) // KV4_PAGE - len(self._pages[s]) for s, t in zip(seqs, total)]
        if sum(want) > len(self._free):
            raise RuntimeError(f"the step needs {sum(want)} more pages, {len(self._free)} are free")
        took = self._free[len(self._free) - sum(want):][::-1]
        pages, at = [], 0
        for s, n in zip(seqs, want):
            pages.append(self._pages[s] + took[at:at + n])
            at += n
        dev, width = self.pool.device, max(len(p) for p in pages)
        rows = [p + [0] * (width - len(p)) for p in pages]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        meta = torch.tensor([x for r in rows for x in r] + total + cu, dtype=torch.int32).to(dev)  # one copy
        B = len(seqs)
        table, lens, cu_dev = meta[:B * width].view(B, width), meta[B * width:B * width + B], meta[B * width + B:]
        pos = torch.cat([torch.arange(t - n, t) for n, t in zip(new, total)])[None].to(dev)
        # nothing has changed so far; nothing below fails
        del self._free[len(self._free) - sum(want):]
        for s, p, t in zip(seqs, pages, total):
            self._pages[s], self._lens[s] = p, t
        self._step = dict(table=table, lens=lens, cu=None if max(new) == min(new) == 1 else cu_dev, rows=cu[-1],
                          max_new=max(new), max_len=max(total), undo=list(zip(seqs, new, want)),
                          left=set(range(len(self.layers))))
        return pos

    def cancel(self):
        """Undo the open step: its tokens were not stored in every layer."""
        if not self._open():
            raise ValueError("no step is open")
        self._undo()

    def _undo(self):
        step, self._step = self._step, None
        for seq, n, pages in step["undo"]:
            self._lens[seq] -= n
            for _ in range(pages):
                self._free.append(self._pages[seq].pop())

    def attend(self, layer_idx, q, k, v, scale=None):
        """One layer of the open step: q (T, H, D), k and v (T, G, D) before RoPE,
        stored and attended to.  The step is closed with its last layer.  Returns
        (T, H, D)."""
        st = self._open()
        if st is None or k.shape[0] != st["rows"]:
            raise ValueError(f"{k.shape[0]} rows for a step of {None if st is None else st['rows']}: open it with begin()")
        pages = self.pool[layer_idx]
        q = ops.kv4_append(k, v, pages, st["table"], st["lens"], self.phases, q=q, cu_seqlens=st["cu"], max_new=st["max_new"])
        out = ops.kv4_attn(q, pages, st["table"], st["lens"], cu_seqlens=st["cu"], scale=scale, max_new=st["max_new"],
                           max_len=st["max_len"])
        st["left"].discard(layer_idx % len(self.layers))
        return out

    @torch.no_grad()
    def run(self, model, seqs, tokens, last_only=True):
        """A step of a patched Llama model: tokens[i], a 1-D sequence of token ids,
        go to sequence seqs[i].  Returns the logits of each sequence's last token
        (len(seqs), vocab), or of every token (T, vocab), rows packed."""
        dev = self.pool.device
        tokens = [torch.as_tensor(t).reshape(-1) for t in tokens]
        if min(len(t) for t in tokens) == 0:
            raise ValueError("every sequence of a step of the model needs a token")
        ids = torch.cat([t.to(dev) for t in tokens])[None]
        keep = 0
        if last_only:
            keep = torch.tensor([len(t) for t in tokens]).cumsum(0).to(dev) - 1
        pos = self.begin(seqs, [len(t) for t in tokens])
        step = self._step
        step["unmasked"] = True
        try:
            logits = model(input_ids=ids, position_ids=pos, past_key_values=self, use_cache=True, logits_to_keep=keep).logits[0]
        except BaseException:
            if self._step is step:
                self._undo()
            raise
        step["left"].clear()
        return logits


def _hides(mask) -> bool:
    """Whether an attention mask as transformers hands it to a layer keeps a token from one at or before its own place."""
    if mask.dim() == 2:
        return not bool(mask.bool().all())
    seen = mask if mask.dtype == torch.bool else mask == 0
    n, keys = mask.shape[-2:]
    return not bool((seen | torch.ones(n, keys, dtype=torch.bool, device=mask.device).triu(1 + keys - n)).all())


def paged_forward(attention, hidden_states, cache, attention_mask=None):
    """LlamaAttention.forward on an open step of a PagedCache.  A mask that hides
    tokens (a padded batch) is refused: there is none in a step, whose pages
    would keep the padding.  It is looked at once a step, and not in run()'s."""
    step = cache._open()
    if isinstance(attention_mask, torch.Tensor) and step is not None and not step.get("unmasked"):
        if _hides(attention_mask):
            raise ValueError("a PagedCache takes no padding and no attention mask: pack the sequences' tokens in one row (run() does)")
        step["unmasked"] = True
    shape = hidden_states.shape[:-1]
    x = hidden_states.reshape(-1, hidden_states.shape[-1])
    q, k, v = (proj(x).unflatten(-1, (-1, attention.head_dim)) for proj in (attention.q_proj, attention.k_proj, attention.v_proj))
    out = cache.attend(attention.layer_idx, q, k, v, scale=attention.scaling)
    return attention.o_proj(out.reshape(*shape, -1)), None
