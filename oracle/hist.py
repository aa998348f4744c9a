"""User histories: a paged cache of keys and values and the attention over it, restated in numpy.

TEST INFRASTRUCTURE ONLY - nothing under recommendation_amd/ may import this.

The reference holds no histories (its nearest analogue is the six-id bag it pools with equal weights,
recommendation/code/r_model.py:68-80); this restates the definitions that the device path follows, position by position
and in 64 bits.  Parity against the reference itself is unpinned: there is nothing to compare with.

Layout: kv [n_pages][heads][2][page_size][dim] (0 keys, 1 values) as float64 VALUES; an 8-bit cache is held as the values
its codes stand for.
"""
import numpy as np

E4M3_MAX = 448.0
MIN_EXPONENT = -126


def e4m3_round(y):
    """Nearest e4m3 value (ties to even) of |y| <= 448; steps of 2^-9 below 2^-6."""
    y = np.asarray(y, np.float64)
    _, e = np.frexp(np.where(y == 0, 1.0, y))                  # |y| in [2^(e-1), 2^e)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.round(y / step) * step                           # np.round: ties to even


def row_exponent(x):
    """The smallest e >= -126 for which max finite |x| * 2^-e <= 448, per row of the last axis."""
    x = np.asarray(x, np.float64)
    top = np.where(np.isfinite(x), np.abs(x), 0.0).max(-1)
    m, e = np.frexp(top)                                        # top = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875)
    return np.where(top == 0, MIN_EXPONENT, np.maximum(e, MIN_EXPONENT)).astype(np.int64)


def quantise(x):
    """Values that rows x stand for in an 8-bit cache (+-inf and NaN: NaN), and their exponents."""
    x = np.asarray(x, np.float64)
    e = row_exponent(x)
    fine = np.isfinite(x)
    y = e4m3_round(np.ldexp(np.where(fine, x, 0.0), -e[..., None]))
    return np.where(fine, np.ldexp(y, e[..., None]), np.nan), e


def places(n_rows, offsets, n_seqs, table, page_size, n_pages, lengths):
    """Per row: (page, slot), None if it has no place, or 'none' if no sequence owns it.  Second result: whether a
    page id or length was out of range."""
    table, lengths = np.asarray(table), np.asarray(lengths)
    out, bad = ['none'] * n_rows, False
    for b in range(n_seqs):
        lo, hi = (offsets[b], offsets[b + 1]) if offsets is not None else (b * (n_rows // n_seqs), (b + 1) * (n_rows // n_seqs))
        for i in range(lo, min(hi, n_rows)):
            pos = int(lengths[b]) - (hi - i)
            out[i] = None
            if pos < 0:
                continue
            if pos // page_size >= table.shape[1] or not 0 <= table[b, pos // page_size] < n_pages:
                bad = True
                continue
            out[i] = (int(table[b, pos // page_size]), pos % page_size)
    return out, bad


def write(kv, k, v, where):
    for i, w in enumerate(where):
        if isinstance(w, tuple):
            kv[w[0], :, 0, w[1]], kv[w[0], :, 1, w[1]] = k[i], v[i]


def read(kv, where, k, v):
    for i, w in enumerate(where):
        if w != 'none':
            k[i], v[i] = (kv[w[0], :, 0, w[1]], kv[w[0], :, 1, w[1]]) if w is not None else (0.0, 0.0)


def attention(kv, q, table, lengths, scale, page_size):
    """out [sequences, tokens, heads, dim]; beside it what error bounds need: sum_j p_j |v_j| (same shape) and
    max_j sum_d |q_d k_jd| * scale per row."""
    q = np.asarray(q, np.float64)
    n, T, Hq, D = q.shape
    H = kv.shape[1]
    out, absv, size = np.zeros_like(q), np.zeros_like(q), np.zeros((n, T, Hq))
    room = table.shape[1] * page_size
    for b in range(n):
        L = min(int(lengths[b]), room)
        pos = np.arange(max(L, 0))
        pages = np.asarray(table)[b, pos // page_size]
        ok = (pages >= 0) & (pages < kv.shape[0])
        pos, pages = pos[ok], pages[ok]
        if not len(pos):
            continue
        for h in range(Hq):
            k, v = kv[pages, h // (Hq // H), 0, pos % page_size], kv[pages, h // (Hq // H), 1, pos % page_size]
            s = (q[b, :, h] @ k.T) * scale
            top = s.max(-1, keepdims=True)
            with np.errstate(invalid='ignore'):
                p = np.exp(s - np.where(top == -np.inf, 0.0, top))
            total = p.sum(-1, keepdims=True)
            p = p / np.where(total == 0, 1.0, total)
            out[b, :, h], absv[b, :, h] = p @ v, p @ np.abs(v)
            size[b, :, h] = (np.abs(q[b, :, h]) @ np.abs(k).T).max(-1) * abs(scale)
    return out, absv, size
