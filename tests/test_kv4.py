"""The paged 4-bit cache and the log probabilities on the CPU: the oracle
against the formats' definitions, argument blocks, and every refusal of the C
entry points (placeholder pointers: nothing is launched)."""
import ctypes

import numpy as np
import pytest

from oracle import kv4 as plain

P = 4096  # a placeholder address, 16-byte aligned


def test_formats():
    assert plain.SCALES[0] == 2.0 ** -16 and plain.SCALES[-1] == 10240.0 and len(plain.SCALES) == 113
    assert (np.diff(plain.SCALES) > 0).all()
    # every value fits fp16
    v = np.outer(plain.SCALES, plain.LEVELS)
    assert (v.astype(np.float16).astype(np.float64) == v).all()


def test_round4_ties_saturation_and_specials():
    row = np.zeros(32)
    row[:8] = [6.5, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]          # scale 1, every border
    assert plain.round4(row)[:8].tolist() == [6, 0, 1, 1, 2, 2, 4, 4]
    assert plain.round4(-row)[:8].tolist() == [-6, 0, -1, -1, -2, -2, -4, -4]
    row[:] = 0
    row[:3] = [np.nan, np.inf, 1e6]
    assert plain.round4(row)[:3].tolist() == [0, 61440, 61440]
    assert (plain.round4(np.full(32, 1e-9)) == 0).all()


def _args(**kw):
    from shard_amd import _lib
    a = _lib.KV4Args()
    base = dict(batch=2, n_tokens=2, n_q_heads=32, n_kv_heads=8, head_dim=128, dtype=0, n_pages=10, table_width=4,
                cache=P, page_stride=8 * 68 * 128, block_table=P, table_stride=4, seq_lens=P,
                q=P, q_stride=4096, q_head_stride=128, k=P, k_stride=1024, k_head_stride=128,
                v=P, v_stride=1024, v_head_stride=128, phases=P, n_phases=256, scale=1.0,
                q_out=P, k_out=P, v_out=P, out=P)
    base.update(kw)
    for name, value in base.items():
        setattr(a, name, value)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,code", [
    (dict(cache=None), -1), (dict(block_table=None), -1), (dict(seq_lens=None), -1), (dict(batch=0), -1),
    (dict(n_tokens=-1), -1), (dict(n_tokens=3), -1), (dict(n_pages=0), -1), (dict(table_width=0), -1),
    (dict(head_dim=96), -2), (dict(head_dim=256), -2), (dict(dtype=2), -2), (dict(dtype=-1), -2),
    (dict(batch=70000, n_tokens=70000), -2), (dict(table_width=1 << 26, table_stride=1 << 26), -2),
    (dict(page_stride=8 * 68 * 128 - 16), -1), (dict(page_stride=8 * 68 * 128 + 8), -1), (dict(table_stride=3), -1),
    (dict(cache=P + 8), -1),
], ids=str)
def test_batch_refusals(kw, code):
    from shard_amd import _lib
    lib = _lib.load()
    assert lib.shard_kv4_append(_args(**kw), None) == code
    assert lib.shard_kv4_read(_args(**kw), None) == code
    assert lib.shard_kv4_attn(_args(**kw), None, 0, None) == code
    assert lib.shard_kv4_attn_workspace(_args(**kw)) == 0


def test_operand_refusals():
    from shard_amd import _lib
    lib = _lib.load()
    for fn in (lib.shard_kv4_append, lib.shard_kv4_read):
        assert fn(None, None) == -1
    assert lib.shard_kv4_attn(None, None, 0, None) == -1
    for kw in (dict(k=None), dict(v=None), dict(k=P + 2), dict(k_stride=4), dict(v_head_stride=-8), dict(phases=None),
               dict(phases=P + 8), dict(n_phases=0), dict(q_out=None), dict(q=P + 4), dict(n_q_heads=0), dict(q_out=P + 2)):
        assert lib.shard_kv4_append(_args(**kw), None) == -1, kw
    for kw in (dict(k_out=None), dict(v_out=None), dict(k_out=P + 8)):
        assert lib.shard_kv4_read(_args(**kw), None) == -1, kw
    for kw, code in ((dict(q=None), -1), (dict(out=None), -1), (dict(out=P + 8), -1), (dict(q_stride=3), -1),
                     (dict(n_q_heads=12), -2), (dict(n_q_heads=0), -2)):
        assert lib.shard_kv4_attn(_args(**kw), None, 0, None) == code, kw
    # nothing to do is no error
    assert lib.shard_kv4_append(_args(n_tokens=0, cu_seqlens=P), None) == 0
    assert lib.shard_kv4_attn(_args(n_tokens=0, cu_seqlens=P), None, 0, None) == 0


def test_workspace_is_checked_before_any_launch():
    from shard_amd import _lib
    lib = _lib.load()
    a = _args(table_width=512, table_stride=512)
    need = lib.shard_kv4_attn_workspace(a)
    assert need > 0 and need % (130 * 4) == 0
    assert lib.shard_kv4_attn(a, None, need, None) == -4
    assert lib.shard_kv4_attn(a, P, need - 1, None) == -4
    assert str(need).encode() in lib.shard_last_error()
    assert lib.shard_kv4_attn(a, P + 4, need, None) == -4
    assert lib.shard_kv4_attn_workspace(_args(max_len=64)) == 0   # one split


def test_page_bytes():
    from shard_amd import _lib
    lib = _lib.load()
    assert lib.shard_kv4_page_bytes(8, 128) == 8 * (64 * 128 + 64 * 8)   # 4 bits an element, a byte for 32
    assert lib.shard_kv4_page_bytes(8, 64) == 8 * (64 * 64 + 64 * 4)
    assert lib.shard_kv4_page_bytes(8, 96) == 0 and lib.shard_kv4_page_bytes(0, 128) == 0


def test_cpu_tensors_are_refused():
    import torch
    from shard_amd import ops
    c = ops.kv4_cache(2, 2, 64, device="cpu")
    assert c.shape == (2, 2, 68 * 64)
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    k = torch.zeros(1, 2, 64, dtype=torch.float16)
    with pytest.raises(ops.ShardHipUnavailable):
        ops.kv4_append(k, k, c, t, n, torch.zeros(128, 32, 2))
    with pytest.raises(ops.ShardHipUnavailable):
        ops.kv4_read(c, t, n, 1)
    with pytest.raises(ops.ShardHipUnavailable):
        ops.kv4_attn(k, c, t, n)
    with pytest.raises(ops.ShardHipUnavailable):
        ops.token_logprobs(torch.zeros(2, 5))
    for bad in ((0, 2, 64), (2, 0, 64), (2, 2, 96)):
        with pytest.raises(ValueError):
            ops.kv4_cache(*bad, device="cpu")


def test_logprobs_refusals():
    from shard_amd import _lib
    lib = _lib.load()
    call = lambda logits=P, dtype=0, rows=4, vocab=1000, stride=1000, tokens=P, top=5, lp=P, ent=P, tl=P, ti=P, ws=P, n=1 << 30: \
        lib.shard_token_logprobs(logits, dtype, rows, vocab, stride, tokens, top, lp, ent, tl, ti, ws, n, None)
    for kw in (dict(logits=None), dict(ent=None), dict(lp=None), dict(tl=None), dict(ti=None), dict(rows=-1), dict(vocab=0),
               dict(top=-1), dict(stride=-1), dict(logits=P + 1), dict(dtype=2, logits=P + 2)):
        assert call(**kw) == -1, kw
    for kw in (dict(top=65), dict(top=5, vocab=4), dict(vocab=1 << 31), dict(dtype=3)):
        assert call(**kw) == -2, kw
    assert call(rows=0) == 0
    need = lib.shard_token_logprobs_workspace(4, 128256, 5)
    assert need > 0
    big = dict(vocab=128256, stride=128256)
    assert call(**big, ws=None) == -4 and call(**big, n=need - 1) == -4 and call(**big, ws=P + 8) == -4
    assert str(need).encode() in lib.shard_last_error()
    assert lib.shard_token_logprobs_workspace(4096, 128256, 5) == 0    # a workgroup a row
    assert lib.shard_token_logprobs_workspace(4, 128256, 65) == 0


def test_compiled_dispatch_is_built_and_leaves_odd_calls():
    """_dispatch.so loads, binds the library, and returns None (the way through
    ops.py) for operands it does not take."""
    import torch
    from shard_amd import _lib, ops
    _lib.load()
    d = ops._bind_direct()
    assert d, "shard_amd/_dispatch.so is not built"
    c = ops.kv4_cache(2, 2, 64, device="cpu")
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    k = torch.zeros(1, 2, 64, dtype=torch.float16)
    assert d.kv4_attn(k, c, t, n, None, None, None, None, 0, 0) is None
    assert d.kv4_append(k, k, c, t, n, torch.zeros(128, 32, 2), None, None, None, 0, 0) is None
    assert d.kv4_read(c, t, n, 1, False, None, None, 0, 0) is None
    assert d.token_logprobs(torch.zeros(2, 5), None, 1, 0, 0) is None
    for bad in ((), (None,) * 10, ("q", c, t, n, None, None, None, None, 0, 0), (k, c, t, n, None, None, 1 << 70, None, 0, 0)):
        assert d.kv4_attn(*bad) is None
    with pytest.raises(ImportError):
        d.bind("/nowhere/lib.so")


def test_rows_beyond_a_launch():
    """A launch has at most 2^32 - 1 threads: rows of logits are refused there, attention does without splits."""
    from shard_amd import _lib
    lib = _lib.load()
    rows = lambda n: lib.shard_token_logprobs(P, 0, n, 100, 100, None, 0, None, P, None, None, P, 1 << 40, None)
    assert rows(1 << 24) == -2 and rows(1 << 31) == -2
    wide = dict(n_q_heads=1024, n_kv_heads=1024, page_stride=1024 * 68 * 128, table_width=1 << 16, table_stride=1 << 16)
    fits, over = (1 << 14) - 1, 1 << 14   # tokens of 1,024 heads: below 2^24 rows, and 2^24
    assert lib.shard_kv4_attn_workspace(_args(**wide, batch=fits, n_tokens=fits)) == fits * 1024 * 128 * 130 * 4
    assert lib.shard_kv4_attn_workspace(_args(**wide, batch=over, n_tokens=over)) == 0


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38, -3e38])
def test_scale_is_a_number(scale):
    """No answer for a scale that leaves no scores; refused before the workspace is looked at, with tokens or without."""
    from shard_amd import _lib
    lib = _lib.load()
    assert lib.shard_kv4_attn(_args(scale=scale), None, 0, None) == -1
    assert lib.shard_kv4_attn(_args(scale=scale, n_tokens=0, cu_seqlens=P), None, 0, None) == -1
    assert lib.shard_kv4_attn(_args(scale=2e38, n_tokens=0, cu_seqlens=P), None, 0, None) == 0


STUB = r"""
#include "shard_hip.h"
extern "C" {
LAYOUT
int shard_kv4_append(const shard_kv4_args*, void*) { return 0; }
int shard_kv4_read(const shard_kv4_args*, void*) { return 0; }
size_t shard_kv4_attn_workspace(const shard_kv4_args*) { return 0; }
ATTN
size_t shard_token_logprobs_workspace(int64_t, int64_t, int32_t) { return 0; }
int shard_token_logprobs(const void*, int32_t, int64_t, int64_t, int64_t, const int64_t*, int32_t, float*, float*, float*, int64_t*,
                         void*, size_t, void*) { return 0; }
}
"""
LAYOUT = "uint64_t shard_kv4_args_layout(void) { return SHARD_KV4_ARGS_LAYOUT%s; }"
ATTN = "int shard_kv4_attn(const shard_kv4_args*, void*, size_t, void*) { return 0; }"


@pytest.mark.parametrize("layout,attn,fits", [(LAYOUT % "", ATTN, True), (LAYOUT % " + 8", ATTN, False), ("", ATTN, False),
                                              (LAYOUT % "", "", False)], ids=["fits", "other", "none", "misses"])
def test_compiled_dispatch_binds_no_other_argument_block(tmp_path, layout, attn, fits):
    """A library from before a change of shard_kv4_args, or from after it, is not called with this one's."""
    import os
    import subprocess
    from conftest import ROOT
    from shard_amd import _lib, ops
    src, so = tmp_path / "stub.cpp", str(tmp_path / "stub.so")
    src.write_text(STUB.replace("LAYOUT\n", layout + "\n", 1).replace("ATTN\n", attn + "\n", 1))
    subprocess.run(["g++", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"), str(src), "-o", so], check=True)
    _lib.load()
    d = ops._bind_direct()
    assert d
    if fits:
        d.bind(so)
    else:
        with pytest.raises(ImportError):
            d.bind(so)
    d.bind(_lib.LIB_PATH)


def test_argument_block_layout():
    """The binding's block is the header's, and no two equally large fields could change places unseen."""
    from shard_amd import _lib
    assert _lib.load().shard_kv4_args_layout() == _lib.KV4_LAYOUT
    fields = _lib.KV4Args._fields_
    for i in range(len(fields)):
        for j in range(i):
            moved = list(fields)
            moved[i], moved[j] = moved[j], moved[i]
            other = type("Other", (ctypes.Structure,), {"_fields_": moved})
            total = (ctypes.sizeof(other) << 32) + sum((2 * n + 1) * getattr(other, f).offset for n, (f, _) in enumerate(fields))
            assert total != _lib.KV4_LAYOUT, (fields[i], fields[j])
