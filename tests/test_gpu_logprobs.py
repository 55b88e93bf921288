"""ops.token_logprobs against float64."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _plain(x, tokens, top):
    """float64 on the CPU: logprob, entropy, top ids (value, then index), their log probabilities."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    lse = (x - m).exp().sum(-1, keepdim=True).log()
    lp = x - m - lse
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top]
    chosen = torch.where(tokens < 0, 0.0, lp.gather(-1, tokens.clamp(min=0)[..., None])[..., 0])
    return chosen, entropy, lp.gather(-1, order), order, lp, p


def _check(x, tokens, top):
    from shard_amd import ops
    got = [t.cpu() for t in ops.token_logprobs(x, tokens, top=top)]
    xc, tc = x.cpu(), tokens.cpu()
    chosen, entropy, top_lp, ids, lp, p = _plain(xc, tc, top)
    V = x.shape[-1]
    # a sum of V positive terms in 256 threads and their joins: V / 256 + 80 roundings of 2^-24 (a granule's 8 terms
    # one after the other); a term's exponent d = (x - max) log2 e is off by 2 roundings of |d| (one for the
    # difference, one for the product) and exp2 by 2 units; ln and the final differences a rounding of the result each
    d = (xc.double() - xc.double().amax(-1, keepdim=True)).clamp(min=-200)
    ed, ed2 = -(p * d).sum(-1), (p * d * d).sum(-1)
    u = 2.0 ** -24
    ln = lambda: (V / 256 + 84) * u + 3 * u * ed
    tol = ln()
    near = lambda got, want, tol: bool(((got.double() - want).abs() <= tol + 4 * u * want.abs()).all())
    fin = torch.isfinite(chosen)
    assert torch.equal(got[0].double()[~fin], chosen[~fin])
    assert near(got[0][fin], chosen[fin], (tol + 2 * u * (d.abs().amax(-1)))[fin])
    # entropy = ln l - E[d]: the same sums, weighted with |d|
    assert near(got[1], entropy, tol + (V / 256 + 90) * u * ed + 3 * u * ed2 + 4 * u * (ed + math.log(V)))
    assert torch.equal(got[3], ids)
    fin = torch.isfinite(top_lp)
    assert torch.equal(got[2].double()[~fin], top_lp[~fin])
    assert near(torch.where(fin, got[2], 0), torch.where(fin, top_lp, 0), (tol + 2 * u * d.abs().amax(-1))[..., None])


def _logits(rows, V, type, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, V, generator=g) * scale
    return x.to(TYPES[type]).cuda(), torch.randint(0, V, (rows,), generator=g).cuda()


@pytest.mark.parametrize("type", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("V,top", [(1, 1), (2, 0), (7, 7), (8, 3), (9, 5), (255, 64), (500, 20), (2049, 1), (32001, 5), (128256, 20)])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_rows(cuda, rows, V, top, type):
    """bf16 and fp16 logits have many equal values: the lower index comes first."""
    x, t = _logits(rows, V, type, rows * V + top)
    _check(x, t, top)


@pytest.mark.parametrize("rows", [2, 1100])
@pytest.mark.parametrize("type", ["fp16", "fp32"])
def test_strided_rows(cuda, rows, type):
    """Rows that begin at any element, rows of a wider tensor, three dimensions."""
    wide, t = _logits(rows, 1200, type, 5)
    for lo, hi in ((0, 1001), (3, 1000), (1, 1200), (5, 9)):
        x = wide[:, lo:hi]
        _check(x, t.clamp(max=x.shape[1] - 1), 3)
    flat = wide.flatten()
    odd = flat[1:1 + (rows - 1) * 1199].view(rows - 1, 1199)
    _check(odd, t[1:].clamp(max=1198), 3)
    _check(wide.unflatten(0, (2, -1)), t.unflatten(0, (2, -1)), 2)
    _check(wide[0], t[0], 2)


def test_equal_logits(cuda):
    """More equal logits than the kernel's list holds: all the same, and few values."""
    for rows in (1, 1300):
        for V in (300, 5000, 20011):
            x = torch.full((rows, V), -3.25, dtype=torch.float16, device=cuda)
            _check(x, torch.full((rows,), V - 1, device=cuda), 20)
            _check(x, torch.full((rows,), V // 2, device=cuda), 64)
            g = torch.Generator().manual_seed(V)
            x = torch.randint(0, 3, (rows, V), generator=g).to(torch.bfloat16).to(cuda)
            x[:, 5] = -0.0
            _check(x, torch.zeros(rows, dtype=torch.int64, device=cuda), 30)
    # the best of every thread in one place, and in descending order of index
    x = torch.arange(60000, dtype=torch.float32).flip(0)[None].cuda() / 100
    _check(x, torch.tensor([3], device=cuda), 64)
    _check(x.flip(1).contiguous(), torch.tensor([3], device=cuda), 64)
    x = torch.zeros(1200, 40000, device=cuda)
    for i in range(64):
        x[:, i * 2048 // 4 % 40000] = 5 + i       # granules of one thread
    _check(x, torch.zeros(1200, dtype=torch.int64, device=cuda), 64)


def test_excluded_tokens(cuda):
    """-inf and each type's lowest value; all tokens but a few; rows far from 0."""
    for type in TYPES:
        for rows in (1, 40):
            x, t = _logits(rows, 4000, type, 9)
            mask = torch.rand(rows, 4000, generator=torch.Generator().manual_seed(1)).cuda()
            low = torch.finfo(TYPES[type]).min
            _check(x.masked_fill(mask < 0.5, -math.inf), t, 20)
            _check(x.masked_fill(mask < 0.5, low), t, 20)
            few = x.masked_fill(mask < 0.999, -math.inf)
            few[:, 77] = 1.0
            _check(few, t, 20)                     # fewer finite logits than alternatives
            one = torch.full_like(x, -math.inf)
            one[:, 1234] = -7.0
            _check(one, t, 3)
            _check(torch.full_like(x, low), t, 3)
            _check((x.float() + 20000).to(x.dtype), t, 3)


def test_no_token_given(cuda):
    from shard_amd import ops
    x, t = _logits(6, 999, "fp16", 3)
    t[1], t[2] = -100, -1
    _check(x, t, 4)
    t[3], t[4] = 999, 1 << 40
    lp = ops.token_logprobs(x, t)[0].cpu()
    assert lp[1] == 0 and lp[2] == 0 and lp[3].isnan() and lp[4].isnan() and not lp[0].isnan()
    none, ent, tl, ti = ops.token_logprobs(x)
    assert none is None and tl.shape == (6, 0) and ti.shape == (6, 0) and bool(ent.isfinite().all())


@pytest.mark.parametrize("rows", [1, 1100])
def test_rows_without_a_distribution(cuda, rows):
    from shard_amd import ops
    for V in (50, 3000):
        for bad in (math.inf, math.nan, -math.inf):
            x, t = _logits(rows, V, "fp32", 4)
            last = rows - 1
            if bad == -math.inf:
                x[last] = bad
            else:
                x[last, V // 2] = bad
            lp, ent, tl, ti = (a.cpu() for a in ops.token_logprobs(x, t, top=3))
            assert lp[last].isnan() and ent[last].isnan() and bool(tl[last].isnan().all())
            assert bool(((ti >= 0) & (ti < V)).all())
            assert bool(lp[:last].isfinite().all())
            if bad == math.inf:
                assert ti[last, 0] == V // 2
            if bad != bad:
                assert V // 2 not in ti[last].tolist()
        x = torch.full((rows, V), math.nan, device=cuda)
        x[:, 1] = 2.0
        lp, ent, tl, ti = (a.cpu() for a in ops.token_logprobs(x, top=3, tokens=torch.zeros(rows, dtype=torch.int64, device=cuda)))
        assert ti.tolist() == [[1, -1, -1]] * rows and bool(tl.isnan().all())


def test_captured(cuda):
    """A captured call's replays read the logits of the moment; two graphs at once."""
    from shard_amd import ops
    x, t = _logits(2, 30000, "fp16", 1)
    ops.token_logprobs(x, t, top=5)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.token_logprobs(x, t, top=5)
        graphs.append((g, out))
    for i in range(4):
        x.copy_(_logits(2, 30000, "fp16", 10 + i)[0])
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = ops.token_logprobs(x, t, top=5)
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(cuda):
    from shard_amd import ops
    x, t = _logits(3, 100, "fp16", 1)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.double(), t)
    with pytest.raises(TypeError):
        ops.token_logprobs(x, t.int())
    with pytest.raises(TypeError):
        ops.token_logprobs(x, t[:2])
    with pytest.raises(ops.ShardHipUnavailable):
        ops.token_logprobs(x, t.cpu())
    for top in (-1, 65, 101):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, t, top=top)
    with pytest.raises(ValueError):
        ops.token_logprobs(x[:, :0], t)
    assert ops.token_logprobs(x[:0], t[:0], top=2)[2].shape == (0, 2)
    assert np.isfinite(ops.token_logprobs(x, t)[0].cpu().numpy()).all()


@pytest.mark.parametrize("type", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,at", [(1, 20000), (1200, 8192), (1200, 39999), (3000, 3073)])
def test_one_logit_above_a_thread_s_first(cuda, rows, at, type):
    """A token nearly certain, found by a thread after a lesser one: errors of a few 2^-24, signs as they must be."""
    from shard_amd import ops
    V, u = 40000, 2.0 ** -24
    x = torch.full((rows, V), -90.0, dtype=TYPES[type], device=cuda)
    x[:, at % 2048 if type != "fp32" else at % 1024] = 0            # in the same thread's first granule where a workgroup has a row
    tok = torch.full((rows,), at, device=cuda)
    for i in range(8, 129):
        d = i / 16
        x[:, at] = d
        lp, entropy, top_lp, ids = (t.cpu() for t in ops.token_logprobs(x, tok, top=1))
        tail = math.exp(-d)
        want, want_e = -math.log1p(tail), math.log1p(tail) + d * tail / (1 + tail)
        assert bool((ids == at).all()) and torch.equal(lp, top_lp[:, 0])
        assert bool((lp <= 0).all()) and bool((entropy >= 0).all())
        # the sum 1 + tail rounds once (2^-24); the tail's exponent is off by 2 roundings of it and exp2 by 2 units of
        # its result; ln by 2 units, the last differences a rounding of the result each
        tail_off = tail * (2 * d + 8)
        assert float((lp.double() - want).abs().max()) <= u * (1 + tail_off + 6 * -want), d
        # E[d] = d tail / (1 + tail): its own three roundings and the sum's
        assert float((entropy.double() - want_e).abs().max()) <= u * (1 + tail_off + 6 * want_e + d * tail * (2 * d + 12)), d
