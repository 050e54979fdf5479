"""The operators of zklm_compile_b200.serving from their definition, in numpy's 64-bit integers (a product of two field elements is
below 2^62; sums of reduced products stay far below 2^63)."""
import numpy as np

P = (1 << 31) - 1


def centred(x):
    x = np.asarray(x).astype(np.int64)
    return np.where(x > P // 2, x - P, x)


def halved(x, shift):
    """x / 2^shift, to the nearest integer, halves away from zero; Python integers, so nothing can overflow."""
    def one(v):
        v = int(v)
        m = (abs(v) + ((1 << shift) >> 1)) >> shift
        return -m if v < 0 else m
    return np.array([one(v) for v in np.asarray(x, dtype=object).reshape(-1)], dtype=object).reshape(np.shape(x))


def rotate(x, cs, shift, pairs):
    """x: one head's d elements; cs: (rot / 2, 2)."""
    v = [int(a) for a in centred(x)]
    half = len(cs)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + half)
        c, s = int(cs[i][0]), int(cs[i][1])
        v[a], v[b] = int(halved(np.array([v[a] * c - v[b] * s], dtype=object), shift)[0]), int(halved(np.array([v[a] * s + v[b] * c], dtype=object), shift)[0])
    return np.array([a % P for a in v], dtype=np.int64)


def append(k_pages, v_pages, k, v, table, row_start, start, cs=None, shift=14, pairs=False, q=None, q_out=None, small=False):
    """k_pages, v_pages: (pages, kv, page, d); they and q_out are changed in place.  Status words are returned."""
    page = k_pages.shape[2]
    status = np.zeros(len(start), np.int64)
    for s in range(len(start)):
        for t in range(max(0, row_start[s]), min(row_start[s + 1], len(k))):
            pos = int(start[s]) + t - row_start[s]
            place = int(table[s][pos // page]) if 0 <= pos < table.shape[1] * page else -1
            if not 0 <= place < len(k_pages):
                status[s] = max(status[s], 1)
                continue
            if cs is not None and cs.shape[1] and pos >= len(cs):
                status[s] = max(status[s], 2)
                continue
            turn = (lambda x: rotate(x, cs[pos], shift, pairs)) if cs is not None else (lambda x: x.astype(np.int64))
            for h in range(k.shape[1]):
                for pages, x in ((k_pages, turn(k[t, h])), (v_pages, v[t, h].astype(np.int64))):
                    if small:
                        x = centred(x)
                        if (x < -32768).any() or (x > 32767).any():
                            status[s] = max(status[s], 3)
                    pages[place, h, pos % page] = x.astype(pages.dtype)
            if q is not None:
                for h in range(q.shape[1]):
                    q_out[t, h] = turn(q[t, h])
    return status


def attend(k_pages, v_pages, q, table, lens, exp_table, shift):
    """q: (seqs, heads, d) -> (out, status)."""
    seqs, heads, d = q.shape
    kv, page = k_pages.shape[1:3]
    n_table, limit = len(exp_table), table.shape[1] * page
    out, status = np.zeros((seqs, heads, d), np.int64), np.zeros(seqs, np.int64)
    for s in range(seqs):
        n = int(lens[s])
        if not 0 <= n <= limit:
            status[s] = max(status[s], 1)
            continue
        pos = np.arange(n)
        place = table[s][pos // page] if n else np.zeros(0, np.int64)
        if ((place < 0) | (place >= len(k_pages))).any():
            status[s] = max(status[s], 1)
            continue
        for h in range(heads):
            k = np.mod(k_pages[place, h // (heads // kv), pos % page].astype(np.int64), P)
            v = np.mod(v_pages[place, h // (heads // kv), pos % page].astype(np.int64), P)
            score = centred((k * q[s, h].astype(np.int64) % P).sum(1) % P)
            score = halved(score, shift).astype(np.int64)
            if ((score < -(n_table // 2)) | (score >= n_table // 2)).any():
                status[s] = max(status[s], 4)
                continue
            e = exp_table[np.mod(score, n_table)].astype(np.int64)
            total = int(e.sum()) % P
            if n and total == 0:
                status[s] = max(status[s], 5)
                continue
            out[s, h] = (e[:, None] * v % P).sum(0) % P * pow(total, P - 2, P) % P
    return out, status


def linear(x, w, bias=None, a=None, b=None, of=None):
    x, w = x.astype(np.int64), w.astype(np.int64)
    y = np.zeros((len(x), len(w)), np.int64)
    for t in range(len(x)):
        y[t] = (w * x[t] % P).sum(1) + (0 if bias is None else bias.astype(np.int64))
        if a is not None and 0 <= of[t] < len(a):
            u = (a[of[t]].astype(np.int64) * x[t] % P).sum(1) % P
            y[t] += (b[of[t]].astype(np.int64) * u % P).sum(1)
    return y % P


def linear_wide(x, w):
    """The same product by halves of 16 bits, whose sums of products are exact in 64-bit floats (below 2^53 for less than 2^20 columns)."""
    x0, x1, w0, w1 = ((v & 0xffff).astype(np.float64) if low else (v >> 16).astype(np.float64) for v in (x, w) for low in (True, False))
    part = lambda a, b: (a @ b.T).astype(np.int64) % P
    return (part(x0, w0) + (part(x0, w1) + part(x1, w0)) * 65536 + part(x1, w1) * 2) % P
