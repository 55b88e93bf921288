"""The paged 4-bit cache and its attention restated from their definition, one
token at a time, in float64 on the CPU (test infrastructure only).

A cache here is the value that every slot holds, (pages, 64, heads, D); the
bytes of a device cache are read by `held`, from each element's own place."""
import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
SCALES = np.array([float(np.uint16(b << 8).view(np.float16)) for b in range(1, 114)])  # E5M2, 2^-16 .. 10240


def round4(x):
    """Rows of 32 values -> the values their codes and scale stand for."""
    x = np.nan_to_num(np.asarray(x, np.float64), nan=0.0, posinf=1e30, neginf=-1e30)
    out = np.empty_like(x)
    for row in np.ndindex(x.shape[:-1]):
        amax = np.abs(x[row]).max()
        fits = SCALES * 6.5 >= amax
        s = SCALES[np.argmax(fits)] if fits.any() else SCALES[-1]
        off = np.abs(np.minimum(np.abs(x[row]), 6 * s)[:, None] - LEVELS * s)
        near = off == off.min(-1, keepdims=True)
        code = np.argmax(near, -1)                       # the lower of two equally near codes
        tie = near.sum(-1) == 2
        code = np.where(tie & (code % 2 == 1), code + 1, code)
        out[row] = np.sign(x[row]) * LEVELS[code] * s
    return out


def rotate(x, phases, pos):
    """x (heads, D) at position pos."""
    h = x.shape[-1] // 2
    c, s = phases[pos, :, 0].astype(np.float64), phases[pos, :, 1].astype(np.float64)
    lo, hi = x[:, :h].astype(np.float64), x[:, h:].astype(np.float64)
    with np.errstate(invalid="ignore"):
        return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)


def places(cu, seq_lens, width, batch):
    """(row, sequence, position) of every new token; positions may be outside."""
    for b in range(batch):
        r0, r1 = (b, b + 1) if cu is None else (cu[b], cu[b + 1])
        for i in range(r1 - r0):
            yield r0 + i, b, max(seq_lens[b], 0) - (r1 - r0) + i


def page_at(table, n_pages, b, pos):
    if not 0 <= pos < table.shape[1] * 64:
        return -1
    p = table[b, pos // 64]
    return p if 0 <= p < n_pages else -1


@np.errstate(invalid="ignore")  # scale bytes of unwritten slots may be anything
def held(cache):
    """Values of a device cache's bytes: (K, V), (pages, 64, heads, D) each."""
    P, G, width = cache.shape
    D = width // 68
    k, v = np.empty((P, 64, G, D)), np.empty((P, 64, G, D))
    e5m2 = lambda b: (b.astype(np.uint16) << 8).view(np.float16).astype(np.float64)
    value = lambda nib: np.where(nib & 8, -1.0, 1.0) * LEVELS[nib & 7]
    for t in range(64):
        sub, r, s, kq, e = t // 16, t % 16, t // 32, t // 4 % 4, t % 32 // 16 * 4 + t % 4
        for c in range(D):
            lane, i = c // (D // 4), c % (D // 4)
            if D == 128:
                at = (sub * 64 + lane * 16 + r) * 16 + i // 2
            else:
                at = (sub // 2 * 64 + lane * 16 + r) * 16 + sub % 2 * 8 + i // 2
            k[:, t, :, c] = value(cache[..., at] >> 4 * (i % 2) & 15) * e5m2(cache[..., 32 * D + (c // 32 * 16 + r) * 4 + sub])
            n = c // 16
            at = 34 * D + (((s * (D // 64) + n // 4) * 64 + kq * 16 + c % 16) * 4 + n % 4) * 4 + e // 2
            scale = cache[..., 66 * D + ((kq * 2 + s) * (D // 32) + c // 32) * 8 + e]
            v[:, t, :, c] = value(cache[..., at] >> 4 * (e % 2) & 15) * e5m2(scale)
    return k, v


def attention(q, k, v, table, seq_lens, cu, scale):
    """q (T, H, D); k, v as `held` gives them.  Returns (out, a, d): out (T, H, D) and, for error bounds, the
    weighted mean of |v| (T, H, D) and the largest sum of |q k| scale over a row's keys (T, H)."""
    T, H, D = q.shape
    G = k.shape[2]
    out, a, d = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H))
    for r, b, pos in places(cu, seq_lens, table.shape[1], len(seq_lens)):
        toks = [(page_at(table, k.shape[0], b, t), t % 64) for t in range(min(pos + 1, table.shape[1] * 64))]
        toks = [x for x in toks if x[0] >= 0]
        if not toks:
            continue
        p, sl = np.array(toks).T
        for g in range(G):
            kk, vv = k[p, sl, g], v[p, sl, g]
            hs = slice(g * (H // G), (g + 1) * (H // G))
            qq = q[r, hs].astype(np.float64)
            s = qq @ kk.T * scale
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            out[r, hs], a[r, hs] = w @ vv, w @ np.abs(vv)
            d[r, hs] = (np.abs(qq) @ np.abs(kk).T * abs(scale)).max(-1)
    return out, a, d
