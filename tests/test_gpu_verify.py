"""Verification of drafted tokens on the GPU (ops.verify_drafts) against the float64
restatement in oracle/drafts.py."""
import numpy as np
import pytest
import torch

from oracle import drafts as plain
from tests.test_gpu_drafts import random_parents

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


class Case:
    def __init__(self, new, V, type="fp16", probs=False, temperature=1.0, seed=0, width=4, close=6.0):
        g = torch.Generator().manual_seed(seed)
        T = sum(new)
        self.new, self.V, self.temperature = new, V, temperature
        self.parents = random_parents(new, seed, width)
        self.cu = [0] + np.cumsum(new).tolist()
        x = torch.randn(T, V, generator=g) * 2
        self.tokens = torch.randint(0, V, (T,), generator=g)
        first = [c for c, n in zip(self.cu, new) for _ in range(n)]
        at = torch.tensor([f + max(p, 0) for f, p in zip(first, self.parents)], dtype=torch.long)
        if close and T:   # drafted tokens are likely ones
            x.index_put_((at, self.tokens), torch.rand(T, generator=g) * close, accumulate=True)
        self.logits = x.to(TYPES[type])
        self.probs = torch.softmax(x[at] + torch.randn(T, V, generator=g) * 0.5, -1) if probs else None
        self.uniforms = torch.rand(T, 2, generator=g)

    def run(self, **kw):
        from shard_amd import ops
        d = lambda t: None if t is None else t.cuda()
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        t = self.temperature
        args = dict(cu_seqlens=i32(self.cu), draft_probs=d(self.probs), temperature=t if isinstance(t, float) else torch.tensor(t).cuda(),
                    max_new=max(self.new))
        args.update(kw)
        return ops.verify_drafts(d(self.logits), d(self.tokens), i32(self.parents), d(self.uniforms), **args)

    def check(self, max_depth=None, max_new=None):
        path, counts, following = self.run(max_depth=max_depth, max_new=max_new or max(self.new))
        temps = [self.temperature] * len(self.new) if isinstance(self.temperature, float) else self.temperature
        want, margin = plain.verify(self.logits.float().numpy(), self.tokens.tolist(), self.parents, self.uniforms.numpy(), self.cu,
                                    None if self.probs is None else self.probs.numpy(), temps, *(1 << 30 if x is None else x for x in (max_depth, max_new)))
        # sums of V numbers in 64 bits, each to 2^-48: the answers are determined where no number is nearer to its border
        assert margin > self.V * 2.0 ** -48, "the inputs decide nothing"
        for b, (rows, token) in enumerate(want):
            n = int(counts[b])
            assert path[b, :n].tolist() == rows and int(following[b]) == token, (b, path[b].tolist(), int(following[b]), want[b])
            assert (path[b, n:] == -1).all()
        return want


SIZES = [([1], 7), ([5], 1000), ([1, 4, 0, 9], 129), ([61], 5003), ([66, 3], 64), ([200], 999), ([3, 8], 32001), ([2], 128256)]


@pytest.mark.parametrize("probs", [False, True], ids=["chosen", "drawn"])
@pytest.mark.parametrize("type", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("new,V", SIZES, ids=str)
def test_trees(cuda, new, V, type, probs):
    for seed in range(3):
        Case(new, V, type, probs, temperature=[1.0, 0.6, 1.7][seed], seed=seed).check()


@pytest.mark.parametrize("probs", [False, True], ids=["chosen", "drawn"])
def test_chains(cuda, probs):
    for seed in range(4):
        Case([6] * 20, 500, "bf16", probs, seed=seed, width=1).check()


@pytest.mark.parametrize("probs", [False, True], ids=["chosen", "drawn"])
@pytest.mark.parametrize("width", [1, 3])
def test_long_paths(cuda, probs, width):
    """Drafts that the target likes: most are accepted, several of a path."""
    lengths = []
    for seed in range(20, 24):
        lengths += [len(p) for p, _ in Case([12] * 20, 500, "fp32", probs, seed=seed, width=width, close=30.0).check()]
    print("paths", np.bincount(lengths).tolist())


@pytest.mark.parametrize("probs", [False, True], ids=["chosen", "drawn"])
@pytest.mark.parametrize("rejected", ["all", "none"])
def test_all_or_none_accepted(cuda, probs, rejected):
    c = Case([40, 12], 300, "fp32", probs, seed=5, close=0.5)
    c.uniforms[:, 0] = 0.0 if rejected == "none" else 1 - 2.0 ** -24
    want = c.check()
    if rejected == "none" or not probs:   # drawn ones that the target likes better are accepted always
        assert all((len(p) > 1) == (rejected == "none") for p, _ in want)


def test_many_children(cuda):
    """A row with 900 children, several of one token; the walk tries them all."""
    c = Case([901], 4000, "fp32", seed=3, close=0)
    c.parents = [-1] + [0] * 900
    c.uniforms[:, 0] = 1 - 2.0 ** -24
    c.tokens[400:410] = 17
    c.check()
    c.uniforms[905 - 200:, 0] = 0.0
    c.check()
    c = Case([9], 300, "fp32", True, seed=4)
    c.parents = [-1] + [0] * 8
    c.uniforms[:, 0] = 1 - 2.0 ** -24
    c.check()


def test_extreme_temperatures(cuda):
    """Nearly greedy, nearly uniform, and an infinite one: every token that is not masked alike."""
    for probs in (False, True):
        for t in (1e-3, 1e-30, 1e6, 1e30):
            Case([6, 3], 200, "fp32", probs, t, seed=3).check()
    c = Case([5] * 8, 200, "fp32", temperature=[float("inf")] * 8, seed=4)
    c.logits[:, 50:] = -torch.inf
    path, counts, following = c.run()
    c.temperature, c.logits[:, :50] = [1.0] * 8, 0.0
    want = c.check()
    assert [(p[:n], t) for p, n, t in zip(path.tolist(), counts.tolist(), following.tolist())] == want


def test_temperatures_of_each_sequence(cuda):
    """Greedy and sampling sequences in one call, more than a wave's lanes of them, empty ones among them."""
    new = [(3 * i) % 5 for i in range(150)]
    temps = [[0.0, 0.5, 1.0, 2.5][i % 4] for i in range(150)]
    for probs in (False, True):
        Case(new, 257, "bf16", probs, temps, seed=1).check()


def test_greedy(cuda):
    """Ties go to the first; random numbers and draft_probs do not count; a greedy path follows the largest logits."""
    c = Case([8, 1], 1000, "fp16", temperature=0.0, seed=2)
    c.logits[:, 700] = c.logits[:, 300] = 50.0
    c.tokens[2:5] = 300
    c.parents[1:5] = [0, 0, 2, 3]
    c.uniforms[:] = 0.999
    want = c.check()
    assert want[0][0][:3] == [0, 2, 3] and want[1][1] == 300
    c.probs = torch.rand(9, 1000)
    assert c.check() == want
    c.logits[0, 10], c.logits[3, 5] = float("inf"), float("nan")
    want = c.check()
    assert want[0] == ([0], 10)


@pytest.mark.parametrize("probs", [False, True], ids=["chosen", "drawn"])
def test_masked_and_odd_rows(cuda, probs):
    """Rows masked by -inf and by the type's lowest value, a single possible token, rows without any, NaN and +inf."""
    c = Case([4] * 8, 300, "bf16", probs, seed=6, close=9.0)
    lowest = torch.finfo(torch.bfloat16).min
    c.logits[0:4, 50:] = -torch.inf
    c.logits[4:8, :250] = lowest
    c.logits[8:12] = -torch.inf
    c.logits[8:12, 77] = -3.0
    c.tokens[9] = 77
    c.logits[12] = -torch.inf
    c.logits[17, 3] = torch.nan
    c.logits[16, c.tokens[17]] = 30.0
    c.parents[16:20] = [-1, 0, 1, 2]
    c.uniforms[17, 0] = 0.1
    c.logits[20, 4] = torch.inf
    c.logits[24] = lowest
    c.logits[28:32] = 1000.0
    if probs:
        c.probs[17, c.tokens[17]] = 0.5
    want = c.check()
    assert want[2][1] == 77 and want[3] == ([0], -1) and want[4] == ([0, 1], -1) and want[5] == ([0], -1)


def test_tokens_outside_the_vocabulary(cuda):
    """Padding among the drafts is passed over, and so are parents that are none."""
    c = Case([6, 6], 100, "fp32", seed=8)
    c.parents[:6] = [-1, 0, 0, 0, 3, 9]
    c.tokens[1], c.tokens[2], c.tokens[7] = -1, 100, 2 ** 40
    c.uniforms[:, 0] = 0.0
    want = c.check()
    assert want[0][0] == [0, 3, 4]
    c.probs = torch.full((12, 100), 0.01)
    c.check()


@pytest.mark.parametrize("probs", [False, True], ids=["chosen", "drawn"])
def test_bounds(cuda, probs):
    """max_depth ends a walk before its children are tried; max_new hides rows."""
    c = Case([30, 4], 200, "fp32", probs, seed=9)
    c.uniforms[:, 0] = 0.0
    for depth in (0, 1, 3):
        assert max(len(p) for p, _ in c.check(max_depth=depth)) == depth + 1
    c.check(max_new=3)
    assert c.run(max_new=3)[0].shape == (2, 3)


@pytest.mark.parametrize("type", ["fp16", "bf16", "fp32"])
def test_a_launch_a_level(cuda, type):
    """Many rows, few of them on a path: the sizes that go level by level, with greedy and sampling sequences, empty
    ones, walks that end early, at max_depth, at odd rows, and those that go to the end."""
    for depth in (0, 2, 3):
        Case([90], 128257, type, seed=depth, close=25.0).check(max_depth=depth)
    new = [9, 0, 4, 1] * 20
    temps = [[1.0, 0.5, 0.0, 0.8, 2.0][i % 5] for i in range(80)]
    c = Case(new, 40009, type, temperature=temps, seed=7, close=25.0)
    c.logits[0, 11], c.logits[15, 20000], c.logits[c.cu[16]] = torch.nan, torch.inf, -torch.inf
    lengths = [len(p) for p, _ in c.check(max_depth=2)]
    c.uniforms[:, 0] = 0.0
    lengths += [len(p) for p, _ in c.check(max_depth=3)]
    assert {0, 1, 2, 3, 4} <= set(lengths)
    chain = Case([6] * 60, 40009, type, temperature=0.7, seed=8, width=1)
    chain.uniforms[:, 0] = 0.0
    assert max(len(p) for p, _ in chain.check(max_depth=3)) == 4


@pytest.mark.parametrize("what", ["rows", "levels", "probs"])
def test_captured(cuda, what):
    """All three ways, captured and replayed with other inputs in the same memory."""
    from shard_amd import ops
    V, new = (40009, [6] * 60) if what == "levels" else (3001, [9, 4, 0, 30])
    B, T = len(new), sum(new)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    cu, g = i32([0] + np.cumsum(new).tolist()), torch.Generator(device="cuda").manual_seed(1)

    def inputs(seed):
        x = torch.randn(T, V, generator=g, device=cuda) * 4
        return [x.bfloat16(), torch.randint(0, V, (T,), generator=g, device=cuda), i32(random_parents(new, seed)),
                torch.rand(T, 2, generator=g, device=cuda) * 0.3, torch.softmax(x * 1.1, -1), torch.rand(B, generator=g, device=cuda)]
    call = lambda x, tok, up, u, q, t: ops.verify_drafts(x, tok, up, u, cu_seqlens=cu, draft_probs=q if what == "probs" else None,
                                                         temperature=t, max_new=30, max_depth=3)
    held = inputs(0)
    call(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call(*held)
    for seed in range(1, 5):
        new_in = inputs(seed)
        want = call(*new_in)
        for dst, src in zip(held, new_in):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert bool(torch.randn(64, device=cuda).isfinite().all())


@pytest.mark.parametrize("probs", [False, True], ids=["chosen", "drawn"])
def test_the_answers_are_the_targets_own(cuda, probs):
    """The first token of 40,000 sequences is distributed as the target's, whatever is drafted, and so is the second
    after a given first: six standard deviations of every count."""
    V, B = 7, 40_000
    g = torch.Generator().manual_seed(11)
    target = torch.randn(2, V, generator=g) * 1.5                 # after the first row, after token 2
    draft = torch.softmax(torch.randn(V, generator=g), -1)
    n = 4                                                         # the row, two drafts of it, one below the first
    logits = torch.empty(B, n, V)
    logits[:, 0], logits[:, 1:] = target[0], target[1]
    tokens = torch.full((B, n), 2)
    if probs:
        tokens[:, 1] = torch.multinomial(draft, B, replacement=True, generator=g)
        tokens[:, 2] = torch.multinomial(draft, B, replacement=True, generator=g)
        tokens[:, 3] = torch.multinomial(draft, B, replacement=True, generator=g)
        logits[:, 1:3] = torch.where(tokens[:, 1:3, None] == 2, target[1], torch.zeros(V))
    else:
        tokens[:, 2], tokens[:, 3] = 5, 1
        logits[:, 2] = 0
    d = lambda t: t.reshape(B * n, *t.shape[2:]).cuda()
    uniforms = torch.rand(B * n, 2, generator=g).cuda()
    from shard_amd import ops
    path, counts, following = ops.verify_drafts(
        d(logits), d(tokens), torch.tensor([-1, 0, 0, 1] * B, dtype=torch.int32).cuda(), uniforms, max_new=n,
        cu_seqlens=torch.arange(0, B * n + 1, n, dtype=torch.int32).cuda(), draft_probs=draft.expand(B * n, V).cuda() if probs else None)
    path, counts, following = path.cpu(), counts.cpu(), following.cpu()
    all_tokens = torch.cat([tokens.gather(1, path.clamp(min=0).long()), following[:, None]], 1)
    all_tokens[torch.arange(B), counts.long()] = following
    first, second = all_tokens[:, 1], all_tokens[(counts >= 2) & (all_tokens[:, 1] == 2), 2]
    assert len(second) > 100                                      # the target likes token 2 in one of 70
    for got, p in ((first, torch.softmax(target[0].double(), -1)), (second, torch.softmax(target[1].double(), -1))):
        have = torch.bincount(got, minlength=V).double()
        dev = (len(got) * p * (1 - p)).sqrt()
        assert ((have - len(got) * p).abs() <= 6 * dev).all(), (have / len(got), p)


def test_drafts_equal_to_the_target(cuda):
    """q = p: what is drafted is accepted; a forced rejection that leaves nothing answers from p."""
    c = Case([3, 3], 64, "fp32", True, seed=12, close=0)
    c.parents = [-1, 0, 0] * 2
    q = torch.zeros(64)
    q[5] = 1.0
    c.probs[:] = q
    c.logits[0], c.logits[3] = -torch.inf, -torch.inf
    c.logits[0, 5] = 1.0                                          # p = q: one token, not the drafted one
    c.tokens[:3] = 9
    c.logits[3, 5], c.logits[3, 6] = 0.0, 0.0                     # the rest of p is token 6
    c.tokens[3:] = 9
    path, counts, following = c.run()
    assert counts.tolist() == [1, 1] and following.tolist() == [5, 6]


def test_strides_streams_and_repeats(cuda):
    """Rows of wider tensors at odd places, one row a sequence without cu_seqlens, another stream, the same every time."""
    from shard_amd import ops
    for type in TYPES:
        c = Case([7, 5], 1003, type, True, seed=13)
        want = c.run()
        wide = torch.zeros(12, 1101, dtype=TYPES[type], device=cuda)
        wide[:, 50:1053] = c.logits.to(cuda)
        deep = torch.zeros(12, 1024, device=cuda)
        deep[:, 21:] = c.probs.to(cuda)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        with torch.cuda.stream(side):
            for x, q in ((wide[:, 50:1053], deep[:, 21:]), (c.logits.to(cuda).T.contiguous().T, c.probs.to(cuda).T.contiguous().T)):
                got = ops.verify_drafts(x, c.tokens.to(cuda), i32(c.parents), torch.cat([c.uniforms] * 2, 1).to(cuda)[:, :2],
                                        cu_seqlens=i32(c.cu), draft_probs=q, max_new=7)
                side.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
    c = Case([1] * 70, 300, "fp16", seed=14)
    a, b = c.run(), c.run(cu_seqlens=None)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # rows behind the last sequence are nobody's
    c = Case([4, 4, 3], 300, "fp16", seed=15)
    c.cu, c.new = c.cu[:3], [4, 4]
    c.check()


def test_refusals(cuda):
    from shard_amd import ops
    x, tok, up, u = torch.zeros(4, 9, device=cuda), torch.zeros(4, dtype=torch.int64, device=cuda), \
        torch.zeros(4, dtype=torch.int32, device=cuda), torch.zeros(4, 2, device=cuda)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=cuda)
    call = lambda logits=x, tokens=tok, parents=up, uniforms=u, cu_seqlens=cu, **kw: \
        ops.verify_drafts(logits, tokens, parents, uniforms, cu_seqlens=cu_seqlens, **kw)
    call()
    for kw in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=x[:, :0]), dict(tokens=tok.int()), dict(tokens=tok[:3]),
               dict(parents=up.long()), dict(parents=up[:3]), dict(uniforms=u[:, :1]), dict(uniforms=u.half()), dict(cu_seqlens=cu.long()),
               dict(draft_probs=x.half()), dict(draft_probs=x[:, :5]), dict(temperature=torch.zeros(2, device=cuda)),
               dict(temperature=torch.zeros(1, device=cuda).double())):
        with pytest.raises(TypeError):
            call(**kw)
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(max_depth=-1),
               dict(max_new=-1), dict(cu_seqlens=cu[:1])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError):
        big = torch.zeros(1100, 4, device=cuda)
        call(logits=big, tokens=torch.zeros(1100, dtype=torch.int64, device=cuda), parents=torch.zeros(1100, dtype=torch.int32, device=cuda),
             uniforms=torch.zeros(1100, 2, device=cuda), cu_seqlens=torch.tensor([0, 1100], dtype=torch.int32, device=cuda))
    for kw in (dict(tokens=tok.cpu()), dict(parents=up.cpu()), dict(temperature=torch.zeros(1))):
        with pytest.raises(ops.ShardHipUnavailable):
            call(**kw)
    # no rows, no sequences
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    path, counts, following = call(x[:0], tok[:0], none, u[:0], torch.zeros(3, dtype=torch.int32, device=cuda))
    assert counts.tolist() == [0, 0] and following.tolist() == [-1, -1]


@pytest.mark.parametrize("probs", [False, True], ids=["chosen", "drawn"])
def test_operands_within_larger_ones(cuda, probs):
    """Uniforms, parents, offsets, tokens, temperatures and logits that begin at any element of a larger tensor."""
    from shard_amd import ops
    c = Case([6, 9], 777, "fp16", probs, temperature=[0.7, 1.3], seed=21)
    want = c.run()

    def within(t, dtype=None):
        t = torch.as_tensor(t, dtype=dtype)
        return torch.cat([torch.zeros(1, dtype=t.dtype), t.flatten()]).cuda()[1:].view(t.shape)
    got = ops.verify_drafts(within(c.logits), within(c.tokens), within(c.parents, torch.int32), within(c.uniforms),
                            cu_seqlens=within(c.cu, torch.int32), draft_probs=within(c.probs) if probs else None,
                            temperature=within([0.7, 1.3], torch.float32), max_new=9)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _plan_is_by_levels(rows, batch, V, type, width, max_depth):
    """Whether a call of these sizes goes a launch a level: its workspace holds two levels of every sequence then,
    instead of every row's parts (16 bytes each)."""
    import ctypes
    from shard_amd import _lib
    code, vec = {"fp16": (0, 8), "bf16": (1, 8), "fp32": (2, 4)}[type]
    args = _lib.VerifyArgs(batch=batch, n_tokens=rows, vocab=V, dtype=code, width=width, max_depth=max_depth)
    need = _lib.load().shard_verify_drafts_workspace(ctypes.byref(args))
    granules = (V + 2 * vec - 2) // vec
    parts = -(-granules // max(-(-granules // 64), 128))
    assert need in (rows * parts * 16, 2 * batch * (parts * 16 + 12))
    return need == 2 * batch * (parts * 16 + 12)


def _siblings(levels, kept, tokens, u, after, V=10007):
    """Sequences whose first row has logits at kept[b] ({token: logit}, -inf elsewhere) and children tokens[b] with
    random numbers u[b], the answer's after[b]; by levels there are many more rows, which no walk reaches."""
    B, n = len(kept), 40 if levels else 1 + max(map(len, tokens))
    logits = torch.full((B, n, V), -torch.inf)
    ids, uniforms, parents = torch.zeros(B, n, dtype=torch.int64), torch.zeros(B, n, 2), []
    for b in range(B):
        for t, x in kept[b].items():
            logits[b, 0, t] = x
        m = len(tokens[b])
        ids[b, 1:1 + m], uniforms[b, 1:1 + m, 0], uniforms[b, 0, 1] = torch.tensor(tokens[b]), torch.tensor(u[b]), after[b]
        parents += [-1] + [0] * m + [1] * (n - 1 - m)
    assert _plan_is_by_levels(B * n, B, V, "fp32", n, 1) == levels
    from shard_amd import ops
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    path, counts, following = ops.verify_drafts(logits.view(B * n, V).cuda(), ids.flatten().cuda(), i32(parents), uniforms.view(-1, 2).cuda(),
                                                cu_seqlens=i32(list(range(0, B * n + 1, n))), max_new=n, max_depth=1)
    return [path[b, :c].tolist() for b, c in enumerate(counts.tolist())], following.tolist()


@pytest.mark.parametrize("levels", [False, True], ids=["rows", "levels"])
def test_first_token_with_weight(cuda, levels):
    """A random number of 0 gives the first token that has any weight: none of a part whose tokens were all rejected
    (the rest masked, or too far below to have a weight), and a tiny one beside them where there is one."""
    g = torch.Generator().manual_seed(31)
    kept, tokens, u, want = [], [], [], []
    for b in range(24):
        x = (torch.randn(2, generator=g) * 2).tolist()
        kept.append({100: x[0], 611: x[1], 9000: max(x) + 4.0, 9001: 0.0})
        want.append(9000)
        if b % 3 == 1:
            kept[-1].update({7: -2000.0, 900: -1e30})              # exp(-2000) is 0 in 64 bits
        elif b % 3 == 2:
            kept[-1][300] = x[0] - 60.0
            want[-1] = 300
        tokens.append([100, 611])
        u.append([0.999, 0.999])
    paths, following = _siblings(levels, kept, tokens, u, [0.0] * 24)
    assert paths == [[0]] * 24 and following == want


@pytest.mark.parametrize("levels", [False, True], ids=["rows", "levels"])
def test_what_rejections_leave(cuda, levels):
    """After two rejected tokens of weights 1 and 2^-22 the third child, and the answer, are decided among weights of
    2^-45, within a millionth of each border: a sum that is what subtraction leaves of the first one knows none of that."""
    g = torch.Generator().manual_seed(32)
    kept, tokens, u, after, paths, answers = [], [], [], [], [], []
    for b in range(24):
        # the small ones beside the large ones, and in parts of their own
        ids = [40, 900, *torch.randperm(30 if b % 2 else 10007, generator=g)[:4].add(50).remainder(10007).tolist()]
        ids[2:] = [t + 5000 if t in (40, 900) else t for t in ids[2:]]
        x = [0.0, -22 * np.log(2.0), *(-45 * np.log(2.0) + torch.rand(4, generator=g).double().numpy())]
        x = [float(np.float32(v)) for v in x]
        w = np.exp(np.array(x))
        left = w[2:].sum()                                        # after the first two; child 3 is ids[2]
        accepted = b % 4 < 2
        third = w[2] / left * (1 + (-1e-6 if accepted else 1e-6))
        assert (1 - 2.0 ** -24) * w.sum() > w[0] and (1 - 2.0 ** -24) * w[1:].sum() > w[1]
        kept.append(dict(zip(ids, x)))
        tokens.append(ids[:3])
        u.append([1 - 2.0 ** -24, 1 - 2.0 ** -24, third])
        order = sorted(range(3, 6), key=lambda k: ids[k])         # where it is rejected: one of the other three
        ends = np.cumsum([w[k] for k in order]) / w[3:].sum()
        k = b // 4 % 2
        above = b // 8 % 2
        after.append(ends[k] * (1 + (1e-6 if above else -1e-6)))
        paths.append([0, 3] if accepted else [0])
        answers.append(-1 if accepted else ids[order[k + above]])
    got, following = _siblings(levels, kept, tokens, u, after)
    assert got == paths and following == answers


def test_offsets_that_do_not_ascend(cuda):
    """Sequences that share rows, with draft_probs: whatever is theirs, their answers are rows and tokens, and the other
    sequences' are right.  600 rejected rows of the first lie where the third keeps its own."""
    c = Case([600, 100], 200, "fp32", True, seed=41)
    c.parents = [-1] + [0] * 599 + random_parents([100], 3)
    c.uniforms[:, 0] = 1 - 2.0 ** -24
    c.uniforms[640:, 0] *= 0.3
    c.parents[640:] = random_parents([60], 4)
    path, counts, following = c.run(cu_seqlens=torch.tensor([0, 600, 590, 640, 700], dtype=torch.int32, device=cuda), max_new=600)
    n, path = counts.tolist(), path.tolist()
    assert n[1] == 0 and int(following[1]) == -1
    for b, rows in ((0, 600), (2, 50)):
        assert 1 <= n[b] <= rows and all(0 <= r < rows for r in path[b][:n[b]]) and -1 <= int(following[b]) < 200
    want, margin = plain.verify(c.logits[640:].numpy(), c.tokens[640:].tolist(), c.parents[640:], c.uniforms[640:].numpy(), [0, 60],
                                c.probs[640:].numpy(), [1.0])
    assert margin > 200 * 2.0 ** -48
    assert (path[3][:n[3]], int(following[3])) == want[0]


class ByLevels(Case):
    """A case whose sizes go a launch a level."""

    def check(self, max_depth):
        type = {v: k for k, v in TYPES.items()}[self.logits.dtype]
        assert _plan_is_by_levels(len(self.parents), len(self.new), self.V, type, max(self.new), max_depth)
        return super().check(max_depth=max_depth)


@pytest.mark.parametrize("type", ["fp16", "bf16", "fp32"])
def test_levels_of_uneven_trees(cuda, type):
    """By levels: sequences of their own temperatures, greedy ones among them, empty ones, rows of NaN, +inf and nothing,
    walks that end at every level from the first to the last and at max_depth."""
    new = [33, 0, 9, 1, 20, 40] * 7
    temps = [[1.0, 0.5, 0.0, 0.8, 2.0][i % 5] for i in range(len(new))]
    c = ByLevels(new, 28001, type, temperature=temps, seed=17, close=25.0)
    first = c.cu
    c.logits[first[0], 11], c.logits[first[6], 20000], c.logits[first[12]] = torch.nan, torch.inf, -torch.inf
    lengths = [len(p) for p, _ in c.check(max_depth=5)]
    c.uniforms[:, 0] = 0.0
    lengths += [len(p) for p, _ in c.check(max_depth=4)]
    assert {0, 1, 2, 3, 4, 5} <= set(lengths)
    chain = ByLevels([10] * 45, 40009, type, temperature=0.7, seed=18, width=1, close=25.0)
    lengths = {len(p) for p, _ in chain.check(max_depth=4)}
    chain.uniforms[:, 0] = 0.0
    lengths |= {len(p) for p, _ in chain.check(max_depth=3)}
    assert {1, 2, 4} <= lengths


def test_levels_to_the_last_row(cuda):
    """By levels where max_depth is the most that a tree of so many rows can have: the walk ends as no row is left."""
    c = ByLevels([5] * 90, 70001, "fp16", temperature=0.9, seed=19, width=1, close=30.0)
    for u in (None, 0.0):
        if u is not None:
            c.uniforms[:, 0] = u
        lengths = [len(p) for p, _ in c.check(max_depth=4)]
    assert max(lengths) == 5


def test_levels_captured(cuda):
    """By levels in a graph, replayed with other inputs in the same memory and eager work between."""
    from shard_amd import ops
    V, new = 40009, [20] * 20
    B, T = len(new), sum(new)
    assert _plan_is_by_levels(T, B, V, "bf16", 20, 3)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    cu, g = i32([0] + np.cumsum(new).tolist()), torch.Generator(device="cuda").manual_seed(1)

    def inputs(seed):
        tokens, parents = torch.randint(0, V, (T,), generator=g, device=cuda), i32(random_parents(new, seed))
        x = torch.randn(T, V, generator=g, device=cuda) * 2
        at = (torch.arange(T, device=cuda) // 20 * 20 + parents.clamp(min=0)).long()
        x.index_put_((at, tokens), torch.rand(T, generator=g, device=cuda) * 20, accumulate=True)
        return [x.bfloat16(), tokens, parents, torch.rand(T, 2, generator=g, device=cuda), torch.rand(B, generator=g, device=cuda) - 0.2]
    call = lambda x, tok, up, u, t: ops.verify_drafts(x, tok, up, u, cu_seqlens=cu, temperature=t, max_new=20, max_depth=3)
    held = inputs(0)
    call(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call(*held)
    seen = set()
    for seed in range(1, 5):
        new_in = inputs(seed)
        want = call(*new_in)
        for dst, src in zip(held, new_in):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        seen |= set(want[1].tolist())
        temps = new_in[4].tolist()
        answers, margin = plain.verify(new_in[0].float().cpu().numpy(), new_in[1].tolist(), new_in[2].tolist(), new_in[3].cpu().numpy(),
                                       cu.tolist(), None, temps, 3, 20)
        assert margin > V * 2.0 ** -48
        assert [(p[:n], t) for p, n, t in zip(want[0].tolist(), want[1].tolist(), want[2].tolist())] == answers
        assert bool(torch.randn(64, device=cuda).isfinite().all())
    assert {1, 2, 3, 4} <= seen
