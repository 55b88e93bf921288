"""PagedCache's bookkeeping on the CPU: the operators are stood in for, sequences, pages and steps are the class's own."""
import pytest
import torch


@pytest.fixture
def paged(monkeypatch):
    """A cache of two layers on the CPU; its operators return q as it is."""
    from shard_amd import PagedCache, ops
    monkeypatch.setattr(ops, "rope_phases", lambda start, n, inv: torch.zeros(n, inv.numel(), 2))
    monkeypatch.setattr(ops, "kv4_append", lambda k, v, *args, q=None, **kw: q)
    monkeypatch.setattr(ops, "kv4_attn", lambda q, *args, **kw: q)
    return PagedCache(8, 300, head_dim=64, num_layers=2, n_kv_heads=2, device="cpu")


def _attend(cache, layer, rows):
    x = torch.zeros(rows, 2, 64)
    return cache.attend(layer, x, x, x)


def _state(cache):
    return {s: (cache.length(s), list(cache._pages[s])) for s in cache._pages}, list(cache._free)


def test_pages_and_positions(paged):
    a, b = paged.add(), paged.add()
    assert paged.begin([a, b], [70, 3]).tolist() == [[*range(70), *range(3)]]
    st = paged._step
    assert st["table"].tolist() == [[0, 1], [2, 0]] and st["lens"].tolist() == [70, 3] and st["cu"].tolist() == [0, 70, 73]
    for layer in range(2):
        _attend(paged, layer, 73)
    assert paged.begin([b, a], [62, 1]).tolist() == [[*range(3, 65), 70]]
    assert paged._step["table"].tolist() == [[2, 3], [0, 1]] and paged.free_pages() == 4
    paged.cancel()
    assert _state(paged) == ({a: (70, [0, 1]), b: (3, [2])}, [7, 6, 5, 4, 3])


@pytest.mark.parametrize("what", ["tensor", "arange", "cat"])
def test_a_begin_that_fails_changes_nothing(paged, monkeypatch, what):
    """Out of memory at any of begin()'s tensors: lengths, pages and the step as they were."""
    a, b = paged.add(), paged.add()
    paged.begin([a], [70])
    for layer in range(2):
        _attend(paged, layer, 70)
    before, step = _state(paged), paged._step

    def fail(*args, **kw):
        raise MemoryError
    with monkeypatch.context() as m:
        m.setattr(torch, what, fail)
        with pytest.raises(MemoryError):
            paged.begin([a, b], [100, 5])
    assert _state(paged) == before and paged._step is step
    assert paged.begin([a, b], [1, 5]).tolist() == [[70, *range(5)]]


def test_a_step_is_open_until_every_layer_has_stored_it(paged):
    a = paged.add()
    paged.begin([a], [5])
    with pytest.raises(ValueError):                      # nothing stored yet
        paged.begin([a], [1])
    _attend(paged, 0, 5)
    _attend(paged, 0, 5)                                 # a layer again, in the same step
    with pytest.raises(ValueError):                      # nor in the second layer
        paged.begin([a], [1])
    assert paged.length(a) == 5
    _attend(paged, -1, 5)
    before = _state(paged)
    with pytest.raises(ValueError):                      # stored: no step to undo, none to store over
        paged.cancel()
    with pytest.raises(ValueError):
        _attend(paged, 0, 5)
    assert _state(paged) == before
    assert paged.begin([a], [1]).tolist() == [[5]]
    _attend(paged, 0, 1)
    paged.cancel()
    assert _state(paged) == before
    assert paged.begin([a], [2]).tolist() == [[5, 6]]


class _Model:
    """Attends in `layers`, then fails where asked to."""

    def __init__(self, layers, fails=False):
        self.layers, self.fails = layers, fails

    def __call__(self, input_ids, past_key_values, **kw):
        for layer in self.layers:
            _attend(past_key_values, layer, input_ids.numel())
        if self.fails:
            raise ArithmeticError
        return type("Output", (), dict(logits=torch.zeros(1, 1, 7)))


def test_run_closes_its_step(paged):
    a, ids = paged.add(), torch.arange(70)
    paged.run(_Model([0, 1]), [a], [ids])
    before = _state(paged)
    with pytest.raises(ValueError):
        paged.cancel()
    for layers in ([], [0], [0, 1]):                     # before, between and after the layers
        with pytest.raises(ArithmeticError):
            paged.run(_Model(layers, fails=True), [a], [ids])
        assert _state(paged) == before
        with pytest.raises(ValueError):
            paged.cancel()
    paged.run(_Model([0]), [a], [ids])                   # a model without the cache's last layer
    paged.run(_Model([0, 1]), [a], [ids])
    assert paged.length(a) == 210 and paged.free_pages() == 8 - 4
    paged.begin([a], [3])
    step = _state(paged)
    with pytest.raises(ValueError):                      # somebody else's step stays open
        paged.run(_Model([0, 1]), [a], [ids])
    assert _state(paged) == step
    paged.cancel()
    assert paged.length(a) == 210


def test_a_sequence_dropped_from_an_open_step(paged):
    """The other sequences of the step hold what they held before it: nothing of it was stored in every layer."""
    a, b, c = paged.add(), paged.add(), paged.add()
    paged.run(_Model([0, 1]), [a, b], [torch.arange(60), torch.arange(10)])
    paged.begin([a, b], [100, 3])
    _attend(paged, 0, 103)
    paged.drop(a)
    assert paged.length(b) == 10 and len(paged._pages[b]) == 1 and paged.free_pages() == 7
    with pytest.raises(ValueError):
        paged.cancel()
    with pytest.raises(ValueError):
        _attend(paged, 1, 103)
    assert paged.begin([b], [2]).tolist() == [[10, 11]]
    paged.drop(c)                                        # not of this step: it stays open
    with pytest.raises(KeyError):
        paged.drop(c)
    for layer in range(2):
        _attend(paged, layer, 2)
    paged.drop(b)                                        # its step is closed
    assert _state(paged)[0] == {} and sorted(paged._free) == list(range(8))


@pytest.mark.parametrize("current,other", [(0, False), (1, True)])
def test_phases_are_made_on_their_own_device(monkeypatch, current, other):
    """A PagedCache on a device that is not the current one: the table's launch makes it the current one."""
    from types import SimpleNamespace
    from shard_amd import _lib, ops
    seen, made = [], []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            made.append(self.dev)

        def __exit__(self, *args):
            made.pop()
    freq = torch.ones(32)
    monkeypatch.setattr(ops, "_require_gpu", lambda *args: None)
    monkeypatch.setattr(ops, "_contig", lambda t, *args: SimpleNamespace(
        numel=t.numel, device=t.device, data_ptr=t.data_ptr, get_device=lambda: 0, is_cuda=True))
    monkeypatch.setattr(ops, "_current_device", lambda: current)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 70 + dev)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev: SimpleNamespace(cuda_stream=70 + dev))
    stub = SimpleNamespace(shard_rope_phases=lambda *args: seen.append((list(made), args[-1])) or 0)
    monkeypatch.setattr(_lib, "load", lambda: stub)
    assert ops.rope_phases(0, 64, freq).shape == (64, 32, 2)
    stream = getattr(seen[0][1], "value", seen[0][1])
    assert len(seen) == 1 and seen[0][0] == ([0] if other else []) and stream == 70


ROPES = {
    "default": dict(), "linear": dict(factor=4.0), "llama3": dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                                                   original_max_position_embeddings=512),
    "yarn": dict(factor=4.0, original_max_position_embeddings=512),
    "dynamic": dict(factor=2.0), "longrope": dict(short_factor=[1.0] * 32, long_factor=[2.0] * 32, factor=4.0,
                                                   original_max_position_embeddings=512),
}


def rope_model(kind, dtype=torch.float32):
    from transformers import LlamaConfig, LlamaForCausalLM
    cfg = LlamaConfig(vocab_size=32, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2,
                      num_key_value_heads=1, max_position_embeddings=2048,
                      rope_parameters=dict(rope_type=kind, rope_theta=500000.0, **ROPES[kind]))
    torch.manual_seed(0)
    return LlamaForCausalLM(cfg).to(dtype).eval()


def check_phases(cache, model):
    """The cache's table against the model's own cosines and sines, both fp32."""
    n = cache.phases.shape[0]
    x = torch.zeros(1, 1, 1, device=cache.phases.device)
    cos, sin = (t[0, :, :32].double().cpu() for t in model.model.rotary_emb(x, torch.arange(n, device=x.device)[None]))
    size = float(cos.abs().max())
    got = cache.phases.double().cpu()
    # the angle is one fp32 product on both sides; cosine and sine are off by 2 units each, their factor by one rounding
    assert float((got[..., 0] - cos).abs().max()) <= 6 * 2.0 ** -24 * size
    assert float((got[..., 1] - sin).abs().max()) <= 6 * 2.0 ** -24 * size


@pytest.mark.parametrize("kind", ROPES)
def test_rope_kinds(monkeypatch, kind):
    """A model's frequencies and their factor; kinds whose frequencies follow the length are refused."""
    from shard_amd import PagedCache, ops

    def phases(start, n, inv):
        angle = torch.arange(start, start + n, dtype=torch.float32)[:, None] * inv
        return torch.stack([angle.cos(), angle.sin()], -1)
    monkeypatch.setattr(ops, "rope_phases", phases)
    model = rope_model(kind)
    if kind in ("dynamic", "longrope"):
        with pytest.raises(ValueError, match=kind):
            PagedCache.from_model(model, n_pages=2, max_len=100)
        return
    cache = PagedCache.from_model(model, n_pages=2, max_len=1000)
    assert cache.phases.shape == (1024, 32, 2)
    check_phases(cache, model)
    assert (kind == "yarn") == (float(cache.phases.abs().max()) > 1.01)


def _masks(B, n, hidden):
    """What transformers hands to a layer for a batch whose first row begins with `hidden` pad tokens."""
    keep = torch.ones(B, n, dtype=torch.bool)
    keep[0, :hidden] = False
    both = torch.ones(n, n, dtype=torch.bool).tril() & keep[:, None, None]
    low = torch.finfo(torch.float16).min
    return [both, torch.zeros(both.shape, dtype=torch.float16).masked_fill(~both, low), keep, keep.long()]


@pytest.mark.parametrize("form", range(4), ids=["bool", "additive", "rows", "0 and 1"])
def test_a_padded_batch_is_refused(paged, form):
    """Before anything is stored; a mask that is only causal is none."""
    from types import SimpleNamespace
    from shard_amd.paged import paged_forward
    layer = SimpleNamespace(head_dim=64, layer_idx=0, scaling=0.125, o_proj=lambda x: x, **{
        name: (lambda x: x) for name in ("q_proj", "k_proj", "v_proj")})
    a, b = paged.add(), paged.add()
    x = torch.randn(2, 6, 128)
    paged.begin([a, b], [6, 6])
    with pytest.raises(ValueError, match="mask"):
        paged_forward(layer, x, paged, _masks(2, 6, 2)[form])
    assert paged._open()["left"] == {0, 1}
    out, weights = paged_forward(layer, x, paged, _masks(2, 6, 0)[form])
    assert torch.equal(out, x) and weights is None and paged._open()["left"] == {1}
    paged.cancel()
    paged.begin([a], [6])
    assert torch.equal(paged_forward(layer, x[:1], paged)[0], x[:1])


def test_calls_of_batched_caches_are_refused(paged):
    """transformers' own reorder_cache would do nothing, for a length of 0, and say nothing."""
    idx = torch.tensor([0])
    for call in (lambda: paged.reorder_cache(idx), paged.reset, lambda: paged.crop(1), lambda: paged.batch_repeat_interleave(2),
                 lambda: paged.batch_select_indices(idx)):
        with pytest.raises(RuntimeError, match="sequences"):
            call()
