"""Plain 64-bit forms of the paged 8-bit KV cache's operators (numpy), and the
inputs that its tests share."""
import numpy as np


def plan(cached, new, tables, free, n_free, page, rows):
    """(tables, kv_lens, cu, slots, n_free, missing) of a step."""
    tables, n_pages, width = tables.copy(), len(free), tables.shape[1]
    kv, cu, slots, missing, top = [], [0], [-1] * rows, 0, n_free
    for s, (c, n) in enumerate(zip(cached, new)):
        c, n = max(int(c), 0), max(int(n), 0)
        for j in range(min(-(-c // page), width), min(-(-(c + n) // page), width)):
            top -= 1
            tables[s, j] = free[top] if top >= 0 else -1
        for i in range(n):
            r, pos = cu[-1] + i, c + i
            p = tables[s, pos // page] if pos // page < width else -1
            ok = 0 <= p < n_pages
            if r < rows:
                slots[r] = p * page + pos % page if ok else -1
                missing += not ok
        kv.append(c + n)
        cu.append(cu[-1] + n)
    return tables, kv, cu, slots, max(top, 0), missing + max(cu[-1] - rows, 0)


def release(done, kv, tables, free, n_free, page):
    kv, tables, free = list(kv), tables.copy(), free.copy()
    for s, d in enumerate(done):
        if not d:
            continue
        for j in range(min(-(-max(kv[s], 0) // page), tables.shape[1])):
            if 0 <= tables[s, j] < len(free) and n_free < len(free):
                free[n_free] = tables[s, j]
                n_free += 1
        tables[s] = -1
        kv[s] = 0
    return kv, tables, free, n_free


def rows_of_v(vq):
    """[n_pages, n_kv, P/32, hd, 32] -> [n_pages, n_kv, P, hd]"""
    n, h, _, hd, _ = vq.shape
    return np.ascontiguousarray(vq.transpose(0, 1, 2, 4, 3)).reshape(n, h, -1, hd)


def v_of_rows(q):
    n, h, p, hd = q.shape
    return np.ascontiguousarray(q.reshape(n, h, p // 32, 32, hd).transpose(0, 1, 2, 4, 3))


def append(q, d, x, slots):
    """Rows x [n, n_kv, hd] into quants q [n_pages, n_kv, P, hd] with scales d
    (fp32), in place."""
    page, n_pages = q.shape[2], q.shape[0]
    ok = [0 <= s < n_pages * page for s in slots]
    i = 0
    while i < len(slots):
        if not ok[i]:
            i += 1
            continue
        p, e = slots[i] // page, i
        while e < len(slots) and ok[e] and slots[e] // page == p:
            e += 1
        offs = [s % page for s in slots[i:e]]
        for h in range(q.shape[1]):
            r = x[i:e, h].astype(np.float64)
            with np.errstate(all="ignore"):
                need = np.float32(np.abs(r).max() / 127.0) if np.isfinite(r).all() else np.float32(np.nan)
                old = d[p, h]
                if 0 in offs:
                    scale = need
                elif np.isnan(need) or np.isnan(old):
                    scale = np.float32(np.nan)
                else:
                    scale = max(old, need)
                    if need > old:
                        q[p, h] = np.rint(q[p, h].astype(np.float64) * float(old) / float(need))
                d[p, h] = scale
                v = np.rint(r / float(scale)) if scale > 0 else np.zeros_like(r)
            for o, row in zip(offs, v):
                q[p, h, o] = np.clip(row, -127, 127)
        i = e


def attention(q, kq, ks, vq_rows, vs, tables, kv_lens, cu, window, scale, max_new=None):
    """fp64 outputs [rows, n_q, hd] of the batch, NaN where no row is, with what
    its error bounds are made of: (out, Σ p|v| per value, the largest
    scale·Σ|q||k| and |score| per row, 127·keys·max(p·vs) per row)."""
    rows, n_q, hd = q.shape
    n_kv, page, n_pages = kq.shape[1], kq.shape[2], kq.shape[0]
    g = n_q // n_kv
    out = np.full((rows, n_q, hd), np.nan)
    mag = np.zeros((rows, n_q, hd))
    cond = np.zeros((rows, n_q, 1))
    peak = np.zeros((rows, n_q, 1))
    qd = q.astype(np.float64)
    for s in range(len(kv_lens)):
        a, b, kv = cu[s], cu[s + 1], kv_lens[s]
        j = np.arange(min(max(kv, 0), tables.shape[1] * page))
        p = tables[s, j // page] if len(j) else j
        real = (p >= 0) & (p < n_pages)
        j, p = j[real], p[real]
        for h in range(n_kv):
            kh = kq[p, h, j % page].astype(np.float64) * ks[p, h].astype(np.float64)[:, None]
            vh = vq_rows[p, h, j % page].astype(np.float64) * vs[p, h].astype(np.float64)[:, None]
            for i in range(min(b - a, max_new or b - a)):
                pos = kv - (b - a) + i
                m = (j <= pos) & ((j > pos - window) if window else True)
                for y in range(h * g, (h + 1) * g):
                    if not m.any():
                        out[a + i, y] = 0
                        continue
                    t = kh[m] @ qd[a + i, y] * scale
                    w = np.exp(t - t.max())
                    w /= w.sum()
                    out[a + i, y] = w @ vh[m]
                    mag[a + i, y] = w @ np.abs(vh[m])
                    peak[a + i, y] = 127 * m.sum() * (w * vs[p, h][m]).max()
                    cond[a + i, y] = max((np.abs(kh[m]) @ np.abs(qd[a + i, y])).max() * abs(scale),
                                         np.abs(t).max())
    return out, mag, cond, peak


def attention_bound(out, mag, cond, peak, hd, keys, f16):
    """|got - out| at most.  A relative error e of every weight moves the output
    by at most 2·e·Σp|v|.  e: the score's rounding - q's 22 bits (2^-22) and hd
    fp32 sums (2^-24 each) of scale·Σ|q||k|, four roundings of log2-scaled
    scores and their references (2^-21·|score|, which cond covers too) -, two
    exp2 and reciprocals (2^-21), the weight's 22 bits (2^-22), `keys` fp32 sums.
    f16 rows: each weight rounded once to f16 (2^-11, in the numerator only),
    and the output once (2^-11); fp32 outputs round by 2^-24.
    Weights are f16 numbers (fp32 rows: sums of two) in which the row's largest
    p·vs is 2^6 or more, so each is also off by half of f16's smallest step,
    2^-25: 2^-31 of the largest, against quants of up to 127."""
    e = cond * (2.0 ** -22 + hd * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -21 + 2.0 ** -22 + keys * 2.0 ** -24
    floor = peak * 2.0 ** -31
    if f16:
        return floor + mag * (2 * e + 2.0 ** -11) + np.abs(out) * 2.0 ** -11 + 2.0 ** -25
    return floor + mag * 2 * e + np.abs(out) * 2.0 ** -24
