"""Trees of drafted tokens on the CPU: the oracle's own definitions, every refusal of the C entry points
(placeholder pointers: nothing is launched) and PagedCache's bookkeeping with its operators stood in for."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import drafts as plain
from tests.test_kv4 import P, _args


def test_oracle_verifies_small_trees():
    """Walks whose answers can be read off: three tokens of probabilities 1/2, 1/4, 1/4."""
    x = np.log(np.array([[0.5, 0.25, 0.25]] * 4))
    run = lambda tokens, u, probs=None, t=1.0: plain.verify(x, tokens, [-1, 0, 0, 1], np.array(u), [0, 4], probs, [t])[0][0]
    # token 1 at 0.2 < 1/4: accepted; its child 0 at 0.6: not, which leaves 1/4, 1/4 for tokens 1 and 2
    assert run([9, 1, 2, 0], [[0, 0], [0.2, 0.51], [0, 0], [0.6, 0]]) == ([0, 1], 2)
    # token 1 at 0.3: rejected; token 2 at 0.32: of 1/2 + 1/4 it has a third
    assert run([9, 1, 2, 0], [[0, 0], [0.3, 0], [0.32, 0.4], [0, 0]]) == ([0, 2], 0)
    assert run([9, 1, 2, 0], [[0, 0.9], [0.3, 0], [0.34, 0], [0, 0]]) == ([0], 0)
    # drawn from q = 0, 1/2, 1/2: accepted below a half; two rejections leave token 0
    q = np.array([[0, 0.5, 0.5]] * 4)
    assert run([9, 1, 2, 0], [[0, 0], [0.49, 0.1], [0, 0], [0.9, 0]], q) == ([0, 1, 3], 0)
    assert run([9, 1, 2, 0], [[0, 0.99], [0.51, 0], [0.1, 0], [0, 0]], q) == ([0], 0)
    # greedy
    assert run([9, 1, 0, 0], [[0, 0]] * 4, t=0.0) == ([0, 2], 0)


def test_oracle_trees():
    assert plain.tree([-1, 0, 0, 2, 9], [20], [0, 5], 1) == {
        0: ({0}, 15), 1: ({0, 1}, 16), 2: ({0, 2}, 16), 3: ({0, 2, 3}, 17), 4: ({4}, 15)}


def test_refusals():
    from shard_amd import _lib
    lib = _lib.load()
    for kw, code in ((dict(cache=None), -1), (dict(head_dim=96), -2), (dict(n_tokens=3), -1), (dict(table_stride=3), -1)):
        assert lib.shard_kv4_append_at(_args(**kw), P, None) == code
        assert lib.shard_kv4_tree_attn(_args(**kw), P, 1, None, 0, None) == code
        assert lib.shard_kv4_keep(_args(**kw), 1, 0, P, 4, 4, P, None) == code
    for mask, words in ((None, 1), (P + 4, 1), (P, 0), (P, -1)):
        assert lib.shard_kv4_tree_attn(_args(), mask, words, None, 0, None) == -1
    for kw, code in ((dict(q=None), -1), (dict(n_q_heads=12), -2), (dict(scale=float("nan")), -1), (dict(out=P + 8), -1)):
        assert lib.shard_kv4_tree_attn(_args(**kw), P, 1, None, 0, None) == code
    wide = _args(table_width=512, table_stride=512)
    assert lib.shard_kv4_tree_attn(wide, P, 1, None, lib.shard_kv4_tree_attn_workspace(wide), None) == -4

    page = 8 * 68 * 128
    keep = lambda layers=1, stride=0, rows=P, rows_stride=4, width=4, counts=P, **kw: \
        lib.shard_kv4_keep(_args(**kw), layers, stride, rows, rows_stride, width, counts, None)
    for kw in (dict(layers=0), dict(rows=None), dict(counts=None), dict(width=-1), dict(rows_stride=3),
               dict(layers=2, stride=0), dict(layers=2, stride=-10 * page), dict(layers=2, stride=10 * page - 16),
               dict(layers=2, stride=10 * page + 8), dict(layers=3, stride=page, page_stride=2 * page), dict(layers=2, stride=page)):
        assert keep(**kw) == -1, kw
    assert keep(layers=70000, stride=10 * page) == -2
    assert keep(width=0) == 0 and keep(n_tokens=0, cu_seqlens=P) == 0

    tree = lambda parents=P, lens=P, cu=P, batch=2, T=5, words=1, mask=P, pos=P: \
        lib.shard_draft_tree(parents, lens, cu, batch, T, words, mask, pos, None)
    for kw in (dict(parents=None), dict(lens=None), dict(mask=None), dict(mask=P + 4), dict(pos=None), dict(batch=0), dict(T=-1),
               dict(words=0), dict(cu=None)):
        assert tree(**kw) == -1, kw
    assert tree(words=17) == -2 and tree(batch=70000) == -2 and tree(T=0) == 0


def test_verify_refusals():
    from shard_amd import _lib
    lib = _lib.load()

    def call(ws=P, n=None, **kw):
        a = _lib.VerifyArgs(batch=2, n_tokens=6, vocab=1000, logits=P, row_stride=1000, dtype=0, width=4, tokens=P, parents=P,
                            uniforms=P, cu_seqlens=P, temperature=1.0, max_depth=9, path=P, counts=P, next=P)
        for name, value in kw.items():
            setattr(a, name, value)
        a = ctypes.byref(a)
        need = lib.shard_verify_drafts_workspace(a)
        return lib.shard_verify_drafts(a, ws, need + n if n is not None else need, None), need
    for kw in (*({name: None} for name in ("logits", "tokens", "parents", "uniforms", "path", "counts", "next")), dict(batch=0),
               dict(n_tokens=-1), dict(vocab=0), dict(width=0), dict(max_depth=-1), dict(row_stride=-1), dict(cu_seqlens=None),
               dict(draft_probs=P, probs_stride=-1), dict(draft_probs=P + 2), dict(temperature=-0.5), dict(temperature=float("nan")),
               dict(temperature=float("inf")), dict(logits=P + 1), dict(logits=P + 2, dtype=2)):
        assert call(**kw)[0] == -1, kw
    for kw in (dict(width=1025), dict(vocab=2 ** 31 - 1), dict(dtype=3), dict(n_tokens=1 << 24), dict(batch=70000)):
        assert call(**kw)[0] == -2, kw
    assert lib.shard_verify_drafts(None, P, 1 << 20, None) == -1 and lib.shard_verify_drafts_workspace(None) == 0
    for kw in (dict(ws=None), dict(ws=P + 8), dict(n=-1)):
        code, need = call(**kw)
        assert code == -4 and need > 0 and str(need).encode() in lib.shard_last_error()
    assert call()[1] < call(draft_probs=P, n=-1)[1]


def test_cpu_tensors_are_refused():
    from shard_amd import ops
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    c = ops.kv4_cache(2, 2, 64, device="cpu")
    q = torch.zeros(1, 2, 64, dtype=torch.float16)
    for call in (lambda: ops.draft_tree(i32(1), i32(1)), lambda: ops.kv4_tree_attn(q, c, i32(1, 2), i32(1), torch.ones(1, 1, dtype=torch.int64)),
                 lambda: ops.kv4_keep(c, i32(1, 2), i32(1), i32(1, 3), i32(1)),
                 lambda: ops.kv4_append(q, q, c, i32(1, 2), i32(1), torch.zeros(128, 32, 2), positions=i32(1)),
                 lambda: ops.verify_drafts(torch.zeros(1, 5), torch.zeros(1, dtype=torch.int64), i32(1), torch.zeros(1, 2))):
        with pytest.raises(ops.ShardHipUnavailable):
            call()


def test_compiled_dispatch_leaves_odd_calls():
    """None (the way through ops.py) for operands that it does not take."""
    from shard_amd import _lib, ops
    _lib.load()
    d = ops._bind_direct()
    assert d
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    c, q = ops.kv4_cache(2, 2, 64, device="cpu"), torch.zeros(1, 2, 64, dtype=torch.float16)
    for bad in ((), (None,) * 11, (q, c, i32(1, 2), i32(1), None, None, None, None, torch.ones(1, 1, dtype=torch.int64), 0, 0)):
        assert d.kv4_tree_attn(*bad) is None
    assert d.kv4_append(q, q, c, i32(1, 2), i32(1), torch.zeros(128, 32, 2), None, None, None, i32(1), 0, 0) is None
    for bad in ((), (None,) * 6, (i32(1), i32(1), None, None, 0, 0)):
        assert d.draft_tree(*bad) is None
    for bad in ((), (None,) * 8, (c, i32(1, 2), i32(1), i32(1, 3), i32(1), None, 0, 0)):
        assert d.kv4_keep(*bad) is None
    for bad in ((), (None,) * 11, (torch.zeros(1, 5), torch.zeros(1, dtype=torch.int64), i32(1), torch.zeros(1, 2), None, None, 1.0, None, None, 0, 0)):
        assert d.verify_drafts(*bad) is None


# ---------------------------------------------------------------------------
# PagedCache
# ---------------------------------------------------------------------------
@pytest.fixture
def paged(monkeypatch):
    """A cache of two layers on the CPU; its operators return q as it is, kept rows are written down."""
    from shard_amd import PagedCache, ops

    def draft_tree(parents, lens, cu_seqlens, max_new):
        got = plain.tree(parents.tolist(), lens.tolist(), cu_seqlens.tolist(), (max_new + 63) // 64)
        return "mask", torch.tensor([got[r][1] for r in range(len(parents))], dtype=torch.int32)
    calls = []
    monkeypatch.setattr(ops, "rope_phases", lambda start, n, inv: torch.zeros(n, inv.numel(), 2))
    monkeypatch.setattr(ops, "draft_tree", draft_tree)
    monkeypatch.setattr(ops, "kv4_append", lambda k, v, *args, q=None, positions=None, **kw: calls.append(positions) or q)
    monkeypatch.setattr(ops, "kv4_attn", lambda q, *args, **kw: q)
    monkeypatch.setattr(ops, "kv4_tree_attn", lambda q, cache, table, lens, mask, **kw: calls.append(mask) or q)
    monkeypatch.setattr(ops, "kv4_keep", lambda cache, table, lens, rows, counts, cu_seqlens: calls.append((lens.tolist(), rows, counts)))
    cache = PagedCache(8, 300, head_dim=64, num_layers=2, n_kv_heads=2, device="cpu")
    cache.calls = calls
    return cache


def _store(cache, rows):
    x = torch.zeros(rows, 2, 64)
    for layer in range(2):
        cache.attend(layer, x, x, x)


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_a_tree_is_accepted(paged):
    a, b = paged.add(), paged.add()
    paged.begin([a, b], [62, 3])
    _store(paged, 65)
    assert paged.calls == [None, None]
    pos = paged.begin([b, a], [2, 5], parents=[[-1, 0], [-1, 0, 0, 2, 3]])
    assert pos.tolist() == [[3, 4, 62, 63, 63, 64, 65]] and pos.dtype == torch.int64
    assert paged.length(a) == 67 and paged.free_pages() == 8 - 3
    with pytest.raises(ValueError):                      # not stored yet
        paged.accept(_i32([0, 1], [0, 2]), _i32(2, 2))
    _store(paged, 7)
    assert [c if isinstance(c, str) else c.tolist() for c in paged.calls[2:]] == [pos[0].tolist(), "mask"] * 2
    with pytest.raises(ValueError, match="drafted"):     # stored, not settled
        paged.begin([a], [1])
    for counts in ((3, 1), (1, 6), (-1, 1), (1, 3)):     # more than its rows, or than the path has
        with pytest.raises(ValueError):
            paged.accept(_i32([0, 1], [0, 2]), _i32(*counts))
    with pytest.raises(ValueError):
        paged.accept(_i32([0, 1]), _i32(1))
    assert paged.accept(_i32([0, -1], [0, 2]), _i32(1, 2)) == [1, 2]
    assert paged.calls[-1][0] == [5, 67]
    # 64 tokens fit one page: the second page of a is free again, the next one taken
    assert paged.length(a) == 64 and paged.length(b) == 4 and paged.free_pages() == 8 - 2
    with pytest.raises(ValueError):
        paged.accept(_i32([0, -1], [0, 2]), _i32(1, 2))
    with pytest.raises(ValueError):
        paged.cancel()
    assert paged.begin([a, b], [1, 0]).tolist() == [[64]]


def test_a_tree_is_cancelled_or_its_sequence_dropped(paged):
    a, b = paged.add(), paged.add()
    paged.begin([a, b], [10, 3])
    _store(paged, 13)
    for stored in (False, True):
        paged.begin([a, b], [60, 1], parents=[[-1] + list(range(59)), [-1]])
        if stored:
            _store(paged, 61)
        assert paged.free_pages() == 8 - 3
        paged.cancel()
        assert (paged.length(a), paged.length(b), paged.free_pages()) == (10, 3, 6)
    paged.begin([a, b], [60, 1], parents=[[-1] + list(range(59)), [-1]])
    _store(paged, 61)
    paged.drop(paged.add())                              # not of the step
    assert paged._drafted()
    paged.drop(a)
    assert paged.length(b) == 3 and paged.free_pages() == 7 and not paged._drafted()
    assert paged.begin([b], [1]).tolist() == [[3]]


def test_trees_that_are_none(paged):
    a, b = paged.add(), paged.add()
    for new, parents in (([2], [[-1]]), ([2], [[-1, 1]]), ([2], [[0, 0]]), ([2], [[-1, -1]]), ([3], [[-1, 0, 2]]), ([1, 1], [[-1]]),
                         ([1025], [[-1] + [0] * 1024])):
        with pytest.raises(ValueError):
            paged.begin([a, b][:len(new)], new, parents=parents)
    assert paged.length(a) == 0 and paged.free_pages() == 8 and paged._step is None
    assert paged.begin([a, b], [0, 2], parents=[[], [-1, 0]]).tolist() == [[0, 1]]


def test_a_verification_that_fails_undoes_the_step(paged, monkeypatch):
    from shard_amd import ops
    a = paged.add()

    class Model:
        def __call__(self, input_ids, past_key_values, **kw):
            _store(past_key_values, input_ids.numel())
            return type("Output", (), dict(logits=torch.zeros(1, input_ids.numel(), 7)))

    def verify(logits, ids, parents, uniforms, cu_seqlens, draft_probs, temperature, max_new, max_depth):
        assert ids.tolist() == [5, 6, 1] and parents.tolist() == [-1, 0, 1] and max_new == 3 and max_depth == 2
        assert cu_seqlens.tolist() == [0, 3] and uniforms.shape == (3, 2) and temperature == 0.5
        return _i32([0, 1, -1]), _i32(2), torch.tensor([3])
    monkeypatch.setattr(ops, "verify_drafts", verify)
    assert paged.speculate(Model(), [a], [[5, 6, 1]], [[-1, 0, 1]], temperature=0.5) == [[6, 3]]
    assert paged.length(a) == 2
    for name in ("verify_drafts", "kv4_keep"):
        with monkeypatch.context() as m:
            def fail(*args, **kw):
                raise MemoryError
            m.setattr(ops, name, fail)
            with pytest.raises(MemoryError):
                paged.speculate(Model(), [a], [[5, 6, 1]], [[-1, 0, 1]], temperature=0.5)
        assert paged.length(a) == 2 and paged.free_pages() == 7 and not paged._drafted()
    assert paged.begin([a], [1]).tolist() == [[2]]


def test_errors_name_their_entry_point():
    from shard_amd import _lib
    lib = _lib.load()
    wide = _args(table_width=512, table_stride=512)
    for call, need, name in ((lambda a: lib.shard_kv4_tree_attn(a, P, 1, None, 0, None), lib.shard_kv4_tree_attn_workspace(wide), b"shard_kv4_tree_attn"),
                             (lambda a: lib.shard_kv4_attn(a, None, 0, None), lib.shard_kv4_attn_workspace(wide), b"shard_kv4_attn")):
        assert call(wide) == -4 and lib.shard_last_error().startswith(name + b" needs %d bytes" % need)


def test_rows_that_are_no_path_are_refused(paged):
    """accept() takes a path from row 0 down each row's child: other rows' keys are rotated at other positions, and ones
    out of order, of another sequence or -1 would leave the cache without the tokens that the lengths count."""
    a, b = paged.add(), paged.add()
    paged.begin([a, b], [5, 2], parents=[[-1, 0, 0, 2, 3], [-1, 0]])
    _store(paged, 7)
    for path in ([[0, 3, -1], [0, 1, -1]], [[0, 2, 2], [0, 1, -1]], [[2, 3, 4], [0, 1, -1]], [[0, 2, -1], [0, 1, -1]], [[0, 2, 5], [0, 1, -1]],
                 [[0, 2, 3], [1, 0, -1]], [[0, 2, 3], [0, 2, -1]], [[0, 1, 2], [0, 1, -1]], [[0, -2, -1], [0, 1, -1]]):
        with pytest.raises(ValueError, match="path"):
            paged.accept(_i32(*path), _i32(3, 2))
    assert paged._drafted() and paged.length(a) == 5 and not [c for c in paged.calls if isinstance(c, tuple)]
    assert paged.accept(_i32([0, 2, 3], [0, -1, 7]), _i32(3, 1)) == [3, 1]
    assert paged.length(a) == 3 and paged.length(b) == 1
