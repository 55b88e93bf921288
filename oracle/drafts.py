"""Trees of drafted tokens and their verification restated from their definitions
in float64 on the CPU (test infrastructure only)."""
import numpy as np

from . import kv4


def rows_of(cu, batch, n_rows):
    for b in range(batch):
        r0, r1 = (b, b + 1) if cu is None else (cu[b], cu[b + 1])
        yield b, range(min(max(r0, 0), n_rows), min(max(r1, 0), n_rows))


def parent_of(parents, i):
    return parents[i] if 0 <= parents[i] < i else -1


def tree(parents, seq_lens, cu, words):
    """{row: (the rows of its sequence that it sees, its position)}, no rows and -1 behind the bound."""
    out = {}
    for b, rows in rows_of(cu, len(seq_lens), len(parents)):
        up = [parents[r] for r in rows]
        for i, r in enumerate(rows):
            seen, at = set(), i
            while at >= 0:
                seen.add(at)
                at = parent_of(up, at)
            out[r] = (seen, max(seq_lens[b], 0) - len(up) + len(seen) - 1) if i < 64 * words else (set(), -1)
    return out


def attention(q, k, v, table, seq_lens, cu, scale, seen):
    """kv4.attention where row r sees the tokens before its sequence's rows and the rows in seen[r]."""
    T, H, D = q.shape
    G = k.shape[2]
    out, a, d = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H))
    for b, rows in rows_of(cu, len(seq_lens), T):
        first = max(seq_lens[b], 0) - len(rows)
        for r in rows:
            toks = list(range(first)) + [first + i for i in sorted(seen[r]) if i < len(rows)]
            toks = [(kv4.page_at(table, k.shape[0], b, t), t % 64) for t in toks]
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


def verify(logits, tokens, parents, uniforms, cu, probs, temperatures, max_depth=1 << 30, most=1 << 30):
    """[(path, next token)] of each sequence, and the smallest distance of a number from the border that it was
    compared with, in units of the error that both carry where every weight and every sum has a relative error of one.
    A weight's error stays as large when another number is taken from it, and what is clearly below zero is exactly 0
    (an error of 2^-48 V, V numbers summed)."""
    answers, margin = [], np.inf
    V = logits.shape[1]
    for b, rows in rows_of(cu, len(temperatures), len(parents)):
        rows = list(rows)[:most]
        if not rows:
            answers.append(([], -1))
            continue
        up, path, cold = [parents[r] for r in rows], [0], not temperatures[b] > 0
        while True:
            x = logits[rows[path[-1]]].astype(np.float64)
            if np.isnan(x).any() or x.max() == -np.inf or (x.max() == np.inf and not cold):
                answers.append((path, -1))
                break
            if cold:
                s = np.zeros(V)
                s[np.argmax(x)] = 1
            else:
                s = np.exp((x - x.max()) / np.float64(np.float32(temperatures[b])))
            following, off, off_sum = None, s.copy(), s.sum()   # errors of s and of its sum, of a relative one
            if len(path) <= max_depth:
                for c in range(path[-1] + 1, len(rows)):
                    t = tokens[rows[c]]
                    if parent_of(up, c) != path[-1] or not 0 <= t < V:
                        continue
                    if cold:
                        if s[t] == 1:
                            following = c
                            break
                        continue
                    u, total = np.float64(uniforms[rows[c], 0]), s.sum()
                    bar = u * total * (1 if probs is None else np.float64(probs[rows[c], t]))
                    if s[t] or bar:
                        margin = min(margin, abs(bar - s[t]) / (off[t] + bar / total * off_sum))
                    if bar < s[t]:
                        following = c
                        break
                    if probs is None:
                        s[t] = off[t] = 0
                    else:
                        left = np.maximum(s / total - probs[rows[c]].astype(np.float64), 0)
                        if left.sum() > 0:
                            off = off / total + s / total * (off_sum / total)
                            off[s / total - probs[rows[c]] < -V * 2.0 ** -48 * off] = 0
                            s, off_sum = left, off.sum() + left.sum()
            if following is not None:
                path.append(following)
                continue
            run = np.cumsum(s)
            target = np.float64(uniforms[rows[path[-1]], 1]) * run[-1]
            if not cold:
                margin = min(margin, np.abs(run - target)[s > 0].min() / (2 * off_sum) if target > 0 else np.inf)
            answers.append((path, int(np.argmax(run > target))))
            break
    return answers, margin
