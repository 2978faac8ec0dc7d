"""The paged 8-bit KV cache of a batch of requests: block tables and slot maps
(sgq_kv_pages_plan / _release), append and read-back (sgq_kv_append_paged_q8 /
_gather_), attention (sgq_attn_paged_q8), against plain forms in 64 bits
(tests/_paged.py).  Tables, quants and scales are compared exactly; attention
to the bound of _paged.attention_bound.  The refusals run on the CPU: a
validation error comes before any launch."""
import ctypes as C

import numpy as np
import pytest
import torch

import _paged as ref

gpu = pytest.mark.gpu


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def pool(rng, n_pages, n_kv, page, hd):
    """Random quants and scales on the host: (kq, vq as rows, ks, vs)."""
    q = [np.clip(np.rint(rng.standard_normal((n_pages, n_kv, page, hd)) * 36), -127, 127).astype(np.int8)
         for _ in range(2)]
    d = [(0.02 + 0.02 * rng.random((n_pages, n_kv))).astype(np.float32) for _ in range(2)]
    return q[0], q[1], d[0], d[1]


def to_pages(kq, vq, ks, vs):
    import sgq
    return sgq.KvPages(*(torch.from_numpy(np.ascontiguousarray(t)).cuda()
                         for t in (kq, ref.v_of_rows(vq), ks, vs)))


def from_pages(pages):
    kq, vq, ks, vs = (t.cpu().numpy() for t in pages.tensors)
    return kq, ref.rows_of_v(vq), ks, vs


# ---- block tables ---------------------------------------------------------------

PLANS = [  # cached, new, page, width, spare pages, capacity of the slot map
    ([0], [1], 32, 4, 5, 1),
    ([31, 32, 33, 0, 64], [1, 1, 1, 0, 0], 32, 4, 9, 8),
    ([0, 5, 127, 128, 40], [300, 1, 2, 129, 0], 64, 8, 40, 512),
    ([10, 20, 30], [500, 1, 1], 128, 3, 20, 600),        # a table row too narrow
    ([10, 31, 30, 32], [200, 3, 1, 1], 32, 16, 4, 256),  # the pool runs out
    ([10, 31, 30, 32], [200, 3, 1, 1], 32, 16, 0, 100),  # no page at all, rows past the map
    ([-3, 7, 64], [2, -1, 1], 32, 4, 8, 3),              # negative lengths count as 0
]


def plan_inputs(cached, new, page, width, spare, seed=0):
    rng = np.random.default_rng(seed)
    need = [min(max(-(-c // page), 0), width) for c in cached]
    n_pages = sum(need) + spare + 2
    perm = rng.permutation(n_pages).astype(np.int32)
    tables = np.full((len(cached), width), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = perm[at:at + n]
        at += n
    free = np.zeros(n_pages, np.int32)
    free[:spare] = perm[at:at + spare]
    return tables, free


def run_plan(ctx, cached, new, tables, free, n_free, page, rows, alias=False):
    n = len(cached)
    a = dict(cached=i32(cached), new=i32(new), tables=i32(tables), free=i32(free), nf=i32([n_free]),
             cu=i32([-7] * (n + 1)), slots=i32([-9] * rows), missing=i32([-5]))
    a["kv"] = a["cached"] if alias else i32([-7] * n)
    a["nf_out"] = a["nf"] if alias else i32([-7])
    ctx.kv_pages_plan(a["cached"], a["new"], a["tables"], a["free"], a["nf"], a["nf_out"], a["kv"],
                      a["cu"], a["slots"], a["missing"], page)
    return a


@gpu
@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("case", range(len(PLANS)))
def test_plan_matches_plain(ctx, case, alias):
    cached, new, page, width, spare, rows = PLANS[case]
    tables, free = plan_inputs(cached, new, page, width, spare)
    a = run_plan(ctx, cached, new, tables, free, spare, page, rows, alias)
    want = ref.plan(cached, new, tables, free, spare, page, rows)
    for name, w in zip(("tables", "kv", "cu", "slots", "nf_out", "missing"), want):
        assert np.array_equal(a[name].cpu().numpy().reshape(-1), np.asarray(w, np.int32).reshape(-1)), name
    assert np.array_equal(a["free"].cpu().numpy(), free)


@gpu
@pytest.mark.parametrize("n", [63, 1024, 1025, 4096])
def test_plan_and_release_of_large_batches(ctx, n):
    rng = np.random.default_rng(n)
    page, width = 32, 12
    cached = rng.integers(0, page * width - 40, n)
    new = np.where(rng.random(n) < 0.1, rng.integers(0, 40, n), 1)
    spare = int(sum(-(-(c + m) // page) for c, m in zip(cached, new)))
    tables, free = plan_inputs(cached, new, page, width, spare, n)
    rows = int(new.sum()) + 13
    a = run_plan(ctx, cached, new, tables, free, spare, page, rows)
    want = ref.plan(cached, new, tables, free, spare, page, rows)
    for name, w in zip(("tables", "kv", "cu", "slots", "nf_out", "missing"), want):
        assert np.array_equal(a[name].cpu().numpy().reshape(-1), np.asarray(w, np.int32).reshape(-1)), name
    done = (rng.random(n) < 0.3).astype(np.int32)
    ctx.kv_pages_release(i32(done), a["kv"], a["tables"], a["free"], a["nf_out"], page)
    kv, tb, fr, nf = ref.release(done, want[1], want[0], free, want[4], page)
    assert np.array_equal(a["kv"].cpu().numpy(), kv)
    assert np.array_equal(a["tables"].cpu().numpy(), tb)
    assert a["nf_out"].item() == nf
    assert np.array_equal(a["free"].cpu().numpy()[:nf], fr[:nf])


@gpu
def test_release_leaves_out_missing_pages_and_keeps_the_stack_in_bounds(ctx):
    page = 32
    tables = np.array([[4, -1, 2, 9], [1, 0, -1, -1], [3, 5, -1, -1]], np.int32)  # 9: outside the pool
    kv, free, n_free = [128, 40, 64], np.array([6, 0, 0, 0, 0, 0, 0], np.int32), 1
    for done in ([1, 0, 1], [0, 0, 0], [1, 1, 1]):
        t = [i32(done), i32(kv), i32(tables), i32(free), i32([n_free])]
        ctx.kv_pages_release(*t, page)
        want = ref.release(done, kv, tables, free, n_free, page)
        for got, w in zip(t[1:], want):
            assert np.array_equal(got.cpu().numpy().reshape(-1), np.asarray(w, np.int32).reshape(-1)), done
    # a stack that says it is full takes nothing more
    t = [i32([1, 1, 1]), i32(kv), i32(tables), i32(free), i32([7])]
    ctx.kv_pages_release(*t, page)
    assert t[4].item() == 7 and np.array_equal(t[3].cpu().numpy(), free)


@gpu
@pytest.mark.parametrize("n,width", [(400, 90), (3, 20011), (4096, 30)])
def test_release_of_many_pages(ctx, n, width):
    """More pages than one round of the workgroup takes, some of them missing or
    outside the pool, by requests with none, few and more than their table holds."""
    rng = np.random.default_rng(n)
    page, n_pages = 64, n * width
    kv = rng.integers(0, page * (width + 5), n)
    kv[rng.random(n) < 0.2] = 0
    kv[0] = page * width
    tables = rng.permutation(n_pages).reshape(n, width).astype(np.int32)
    tables[rng.random((n, width)) < 0.03] = -1
    tables[rng.random((n, width)) < 0.01] = n_pages
    done = (rng.random(n) < 0.8).astype(np.int32)
    done[0] = 1
    free, n_free = np.full(n_pages, -7, np.int32), 5
    t = [i32(done), i32(kv), i32(tables), i32(free), i32([n_free])]
    ctx.kv_pages_release(*t, page)
    want = ref.release(done, kv, tables, free, n_free, page)
    for got, w in zip(t[1:], want):
        assert np.array_equal(got.cpu().numpy().reshape(-1), np.asarray(w, np.int32).reshape(-1))


# ---- append and read-back -----------------------------------------------------------

def run_append(ctx, host, x, slots, fused=False, skip=True):
    """The pages after an append of k = x[0], v = x[1] on the device, with the
    plain form's."""
    pages = to_pages(*host)
    if fused:  # K and V as slices of wider rows
        n, n_kv, hd = x[0].shape
        buf = torch.zeros((n, 3, n_kv, hd), dtype=torch.from_numpy(x[0]).dtype, device="cuda")
        buf[:, 1] = torch.from_numpy(x[0]).cuda()
        buf[:, 2] = torch.from_numpy(x[1]).cuda()
        k, v = buf[:, 1], buf[:, 2]
    else:
        k, v = (torch.from_numpy(t).cuda() for t in x)
    ctx.kv_append_paged_q8(pages, k, v, i32(slots))
    want = [t.copy() for t in host]
    ref.append(want[0], want[2], x[0], slots)
    ref.append(want[1], want[3], x[1], slots)
    return pages, want


def assert_pages(pages, want):
    for name, g, w in zip(("k quants", "v quants", "k scales", "v scales"), from_pages(pages), want):
        assert np.array_equal(g, w, equal_nan=g.dtype == np.float32), (
            name, int((g != w).sum()), np.argwhere(g != w)[:4].tolist())


@gpu
@pytest.mark.parametrize("hd,n_kv", [(128, 16), (128, 3), (256, 2), (512, 4)])
@pytest.mark.parametrize("page", [32, 64, 128])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_append_matches_plain(ctx, hd, n_kv, page, dtype):
    """Runs of one row, whole pages, pages begun and ended inside; blocks that
    grow and blocks that do not; rows without a slot."""
    rng = np.random.default_rng(hd + page)
    host = pool(rng, 12, n_kv, page, hd)
    slots = []
    for p, a, b in ((3, 5, 6), (0, 0, page), (7, 0, 1), (5, page - 2, page), (9, 0, 11), (11, 1, 30),
                    (1, 31, 32)):
        slots += list(range(p * page + a, p * page + b))
        if p in (7, 11):
            slots += [-1, 12 * page, 2 ** 31 - 1]
    x = [rng.standard_normal((len(slots), n_kv, hd)) for _ in range(2)]
    x[0][0] *= 3  # page 3 grows
    x[1][-1] *= 0.1  # page 1's V does not
    x = [t.astype(dtype) for t in x]
    pages, want = run_append(ctx, host, x, slots, fused=page == 64)
    assert_pages(pages, want)


@gpu
@pytest.mark.parametrize("n", [1, 1023, 1025, 2311])
def test_append_of_long_runs(ctx, n):
    """A prompt that begins inside a page and ends inside another."""
    rng = np.random.default_rng(n)
    page, hd, n_kv = 32, 128, 2
    n_pages = n // page + 3
    host = pool(rng, n_pages, n_kv, page, hd)
    order = rng.permutation(n_pages)
    slots = [int(order[(i + 19) // page]) * page + (i + 19) % page for i in range(n)]
    x = [rng.standard_normal((n, n_kv, hd)).astype(np.float32) * s for s in (1.0, 40.0)]
    pages, want = run_append(ctx, host, x, slots)
    assert_pages(pages, want)


@gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n", [130, 900, 2100, 4300])
def test_append_of_mixed_runs(ctx, n, dtype):
    """Runs of all lengths, in and out of order, with slots named twice and rows
    without one between them: many runs begin in a workgroup's window."""
    rng = np.random.default_rng(n)
    page, hd, n_kv = 64, 128, 2
    slots, p = [], 0
    while len(slots) < n:
        m = int(rng.choice([1, 1, 1, 2, 17, 40, 64]))
        a = int(rng.integers(0, page - m + 1))
        run = [p * page + a + i for i in range(m)]
        kind = rng.integers(0, 4)
        if kind == 1:
            run = run[::-1]
        elif kind == 2:
            run = [run[i] for i in rng.integers(0, m, m)]
        slots += run + ([-1] * int(rng.integers(1, 4)) if rng.random() < 0.2 else [])
        p += 1
    host = pool(rng, p + 1, n_kv, page, hd)
    x = [(rng.standard_normal((len(slots), n_kv, hd)) * s).astype(dtype) for s in (1.0, 3.0)]
    pages, want = run_append(ctx, host, x, slots)
    assert_pages(pages, want)


@gpu
def test_append_special_values(ctx):
    """All-zero rows, subnormal and huge ones, ties, infinities and NaN; a block
    with a NaN scale stays so until it begins anew; a slot named twice takes the
    later row; slots in no order."""
    rng = np.random.default_rng(5)
    page, hd, n_kv = 32, 128, 3
    host = pool(rng, 10, n_kv, page, hd)
    host[2][8] = np.nan
    x = rng.standard_normal((22, n_kv, hd)).astype(np.float32)
    slots = [0, 1, 1 * page, 2 * page, 3 * page, 4 * page, 5 * page + 3, 6 * page + 1, 8 * page + 4,
             9 * page + 7, 9 * page + 2, 9 * page + 7, 9 * page + 30, -1, 7 * page, 7 * page + 1]
    slots += [-1] * (len(x) - len(slots))
    x[0:2] = 0
    x[2] *= 1e-42
    x[3] *= 1e37
    x[4] = np.rint(rng.uniform(-254, 254, (n_kv, hd))) / 2  # scale 1: halves are ties
    x[4, :, 0] = 127
    x[5, 1, 7] = np.inf
    x[6, 0, 0] = np.nan
    x[7] = 0  # a zero row into a block that has a scale
    x[14] = x[15] = 3e-39
    pages, want = run_append(ctx, host, [x, x[:, ::-1].copy()], slots)
    assert_pages(pages, want)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd,page,n", [(128, 32, 1), (128, 64, 77), (256, 128, 200), (512, 32, 33)])
def test_gather_matches_plain(ctx, hd, page, n, dtype):
    rng = np.random.default_rng(n)
    n_kv = 4
    host = pool(rng, 9, n_kv, page, hd)
    slots = rng.integers(0, 9 * page, n)
    if n > 8:
        slots[3], slots[5] = -1, 9 * page
        slots[8:40] = np.arange(2 * page, 2 * page + 32)[:n - 8]
    pages = to_pages(*host)
    k = torch.full((n, 2, n_kv, hd), 7.0, dtype=dtype, device="cuda")
    ctx.kv_gather_paged_q8(pages, i32(slots), k[:, 0], k[:, 1])
    got = k.cpu().numpy()
    for i, s in enumerate(slots):
        for w, (q, d) in enumerate(((host[0], host[2]), (host[1], host[3]))):
            if 0 <= s < 9 * page:
                want = q[s // page, :, s % page].astype(np.float32) * d[s // page][:, None]
                assert np.array_equal(got[i, w], want.astype(got.dtype)), (i, s, w)
            else:
                assert (got[i, w] == 7.0).all()


# ---- attention ------------------------------------------------------------------------

def batch(rng, kv, new, page, n_kv, hd, spare=3):
    """Pages and block tables of requests with kv tokens each."""
    need = [-(-max(n, 0) // page) for n in kv]
    n_pages = sum(need) + spare
    host = pool(rng, n_pages, n_kv, page, hd)
    perm = rng.permutation(n_pages)
    tables = np.full((len(kv), max(need + [1]) + 1), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = perm[at:at + n]
        at += n
    return host, tables, np.concatenate([[0], np.cumsum(new)]).astype(np.int64)


def attend(ctx, pages, q, tables, kv, cu, n_q, **kw):
    """The device's outputs in a buffer that held 7 before."""
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    kw.setdefault("max_new", int(max(np.diff(cu))))
    if kw.pop("split", True):
        kw["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    ctx.attn_paged_q8(pages, q, i32(tables), i32(kv), i32(cu), out, **kw)
    return out.double().cpu().numpy()


def check_attention(ctx, seed, kv, new, page, n_q, n_kv, hd, f16, window=0, rows=None, scale=None,
                    gain=1.5, split=True, max_kv=None):
    rng = np.random.default_rng(seed)
    host, tables, cu = batch(rng, kv, new, page, n_kv, hd)
    rows = cu[-1] if rows is None else rows
    q = (rng.standard_normal((rows, n_q, hd)) * gain).astype(np.float16 if f16 else np.float32)
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q, window=window,
                 scale=scale, split=split, max_kv=max_kv)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, window,
                                    hd ** -0.5 if scale is None else scale)
    live = ~np.isnan(want)
    assert (got[~live] == 7.0).all(), "rows behind the last request"
    bound = ref.attention_bound(want, mag, cond, peak, hd, max(list(kv) + [1]), f16)
    off = np.abs(got - want)
    bad = live & ~(off <= bound)
    assert not bad.any(), (np.argwhere(bad)[:4].tolist(), off[bad][:4], bound[bad][:4])


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,n_q,n_kv", [(128, 32, 16), (128, 4, 4), (256, 32, 16), (512, 32, 4)])
@pytest.mark.parametrize("page", [32, 64, 128])
def test_attention_of_single_tokens(ctx, f16, hd, n_q, n_kv, page):
    """One new token a request, from the first token on; a request without any."""
    kv = [1, 2, 31, 32, 33, 0, 64, 65, 257, 700]
    new = [1, 1, 1, 1, 1, 0, 1, 1, 1, 1]
    check_attention(ctx, hd + page, kv, new, page, n_q, n_kv, hd, f16)


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,n_q,n_kv", [(128, 8, 4), (128, 6, 2), (128, 12, 1), (256, 4, 2), (512, 8, 1)])
@pytest.mark.parametrize("window", [0, 1, 33, 100])
def test_attention_of_ragged_chunks(ctx, f16, hd, n_q, n_kv, window):
    """Prompts from their first token, later chunks, single tokens and requests
    without new ones in one batch; rows behind the last request."""
    kv = [70, 1, 150, 17, 129, 5, 64]
    new = [70, 1, 33, 0, 1, 5, 16]
    check_attention(ctx, hd + window, kv, new, 32 if window % 2 else 64, n_q, n_kv, hd, f16, window,
                    rows=sum(new) + 5)


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n", [127, 128, 129, 400])
def test_attention_of_whole_prompts(ctx, f16, n):
    check_attention(ctx, n, [n, n + 77], [n, n], 64, 4, 2, 128, f16)


@gpu
@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("kv,window", [(4097, 0), (9000, 0), (9000, 1500)])
def test_attention_of_long_requests(ctx, kv, window, split):
    check_attention(ctx, kv, [kv, 40], [1, 1], 32, 4, 2, 128, False, window, split=split)
    check_attention(ctx, kv, [kv, 40], [9, 1], 64, 8, 1, 128, True, window, split=split, max_kv=100)
    check_attention(ctx, kv, [kv, 300], [41, 270], 128, 4, 2, 256, True, window, split=split)


@gpu
@pytest.mark.parametrize("f16", [True, False])
def test_attention_scales_and_magnitudes(ctx, f16):
    """Sharp softmaxes, a zero and a negative scale, rows of tiny and large q."""
    kv, new = [300, 90], [1, 20]
    for i, (scale, gain) in enumerate([(0.5, 3.0), (0.0, 1.0), (-0.1, 1.0), (1e3, 1e-4), (1e-5, 1e3)]):
        check_attention(ctx, i, kv, new, 32, 4, 2, 128, f16, scale=scale, gain=gain)


@gpu
@pytest.mark.parametrize("f16", [True, False])
def test_attention_over_blocks_of_very_different_scales(ctx, f16):
    """V blocks from zero to large beside each other, K blocks of zero: what
    a block weighs in the output and in the denominator are kept apart."""
    rng = np.random.default_rng(9)
    page, n_q, n_kv, hd = 32, 4, 2, 128
    kv, new = [200, 129], [1, 40]
    host, tables, cu = batch(rng, kv, new, page, n_kv, hd)
    host[3][:] = np.exp(rng.uniform(-30, 6, host[3].shape)).astype(np.float32)
    for s in range(2):  # all-zero blocks: scale 0, quants 0
        p = tables[s, 1]
        host[3][p] = 0
        host[1][p] = 0
        host[2][tables[s, 2]] = 0
    q = (rng.standard_normal((cu[-1], n_q, hd))).astype(np.float16 if f16 else np.float32)
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, 0, hd ** -0.5)
    bound = ref.attention_bound(want, mag, cond, peak, hd, max(kv), f16)
    # log2 of a V scale (|log2| <= 44) is rounded to 2^-19 at most, as a factor 2^-19
    assert (np.abs(got - want) <= bound + mag * 2.0 ** -18).all()
    # every V block zero: the output is zero
    host[3][:] = 0
    host[1][:] = 0
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q)
    assert (got == 0).all()


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_rows_that_attend_nothing_and_pages_that_are_not_there(ctx, f16, new):
    """Positions before the first token (kv_len < rows), requests whose pages are
    missing in part or altogether, tables too short for kv_len: rows without a
    key are 0, the others attend what is there."""
    rng = np.random.default_rng(new)
    page, n_q, n_kv, hd = 32, 4, 2, 128
    kv, cnt = [0, new - 1, 150, 100, 200, 2 ** 31 - 1], [new] * 6
    host, tables, cu = batch(rng, [0, new, 150, 100, 200, 200], cnt, page, n_kv, hd)
    n_pages = len(host[0])
    tables[2, 1] = -1
    tables[2, 3] = n_pages
    tables[3, :] = [-5, 2 ** 31 - 1, -2 ** 31, n_pages + 7] + [-1] * (tables.shape[1] - 4)
    q = rng.standard_normal((cu[-1], n_q, hd)).astype(np.float16 if f16 else np.float32)
    # kv_lens a little past the table for the fifth: its keys end with the table
    kv[4] = tables.shape[1] * page + 9
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, 0, hd ** -0.5)
    bound = ref.attention_bound(want, mag, cond, peak, hd, 300, f16)
    assert (np.abs(got - want) <= bound).all()
    assert (want[cu[3]:cu[4]] == 0).all() and (got[cu[3]:cu[4]] == 0).all()


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_keeps_nan_to_the_rows_that_see_it(ctx, f16, new):
    """NaN scales in pages outside a request, behind its end and before its
    window leave no trace; a row that attends a NaN block is NaN, a NaN or
    infinite q touches its own row and head only."""
    rng = np.random.default_rng(new)
    page, n_q, n_kv, hd, window = 32, 4, 2, 128, 70
    kv, cnt = [200, 300], [new, new]
    host, tables, cu = batch(rng, kv, cnt, page, n_kv, hd, spare=6)
    used = set(tables[tables >= 0].tolist())
    for p in range(len(host[0])):
        if p not in used:
            host[2][p] = host[3][p] = np.nan
    first = (kv[1] - new - window + 1) // page  # pages before this one are outside the window
    for j in range(first):
        host[2][tables[1, j]] = host[3][tables[1, j]] = np.nan
    q = rng.standard_normal((cu[-1], n_q, hd)).astype(np.float16 if f16 else np.float32)
    args = (torch.from_numpy(q).cuda(), tables, kv, cu, n_q)
    got = attend(ctx, to_pages(*host), *args, window=window)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, window, hd ** -0.5)
    assert np.isfinite(want).all()
    assert (np.abs(got - want) <= ref.attention_bound(want, mag, cond, peak, hd, 300, f16)).all()
    # the block of the last token: only the rows that reach it
    p = tables[0, (kv[0] - 1) // page]
    for d in (host[2], host[3]):
        keep = d[p, 1]
        d[p, 1] = np.nan
        bad = attend(ctx, to_pages(*host), *args, window=window)
        d[p, 1] = keep
        reach = np.zeros(bad.shape[:2], bool)
        for i in range(new):
            reach[i, 2:] = kv[0] - new + i >= (kv[0] - 1) // page * page
        assert np.isnan(bad[reach]).all()
        assert np.array_equal(bad[~reach], got[~reach])
    q[cu[-1] - 1, 1, 5] = np.nan
    q[0, 2, 0] = np.inf
    bad = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), *args[1:], window=window)
    hit = np.zeros(bad.shape[:2], bool)
    hit[cu[-1] - 1, 1] = hit[0, 2] = True
    assert np.isnan(bad[hit]).all() and np.array_equal(bad[~hit], got[~hit])


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("max_new,rows", [(3, 58), (24, 58), (48, 53)])
def test_attention_of_requests_with_more_rows_than_announced(ctx, f16, max_new, rows):
    """Rows past max_new or past the buffers are left out; the others keep their positions."""
    rng = np.random.default_rng(17)
    page, n_q, n_kv, hd = 32, 4, 2, 128
    kv, new = [91, 300, 48], [10, 40, 8]
    host, tables, cu = batch(rng, kv, new, page, n_kv, hd)
    q = rng.standard_normal((cu[-1], n_q, hd)).astype(np.float16 if f16 else np.float32)
    got = attend(ctx, to_pages(*host), torch.from_numpy(q[:rows]).cuda(), tables, kv, cu, n_q, max_new=max_new)
    want, mag, cond, peak = (x[:rows] for x in ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu,
                                                             0, hd ** -0.5, max_new=max_new))
    live = ~np.isnan(want)
    assert live.any() and (got[~live] == 7.0).all()
    bound = ref.attention_bound(want, mag, cond, peak, hd, max(kv), f16)
    assert (np.abs(got - want) <= bound)[live].all()


@gpu
def test_attention_of_strided_rows_and_a_small_workspace(ctx):
    """q and out as slices of wider rows; a workspace for fewer splits than wanted."""
    rng = np.random.default_rng(3)
    page, n_q, n_kv, hd = 64, 8, 2, 128
    kv, new = [2500, 1300, 3], [1, 1, 1]
    host, tables, cu = batch(rng, kv, new, page, n_kv, hd)
    q = rng.standard_normal((3, n_q, hd)).astype(np.float16)
    wide = torch.full((3, n_q + 4, hd), 7.0, dtype=torch.float16, device="cuda")
    wide[:, :n_q] = torch.from_numpy(q).cuda()
    out = torch.full((3, 3 * n_q, hd), 7.0, dtype=torch.float16, device="cuda")
    pages = to_pages(*host)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, 0, hd ** -0.5)
    bound = ref.attention_bound(want, mag, cond, peak, hd, max(kv), True)
    full = ctx.attn_paged_workspace(pages, 3, 3, n_q, 1, max(kv))
    row = 3 * n_q * (hd + 2) * 4
    assert full >= 2 * row and full % row == 0
    for size in (full, full - 16, 3 * row, 2 * row - 16, 0):
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")[:size] if size else None
        ctx.attn_paged_q8(pages, wide[:, :n_q], i32(tables), i32(kv), i32(cu), out[:, n_q:2 * n_q],
                          max_new=1, max_kv=max(kv), workspace=ws)
        got = out.double().cpu().numpy()
        assert (np.abs(got[:, n_q:2 * n_q] - want) <= bound).all(), size
        assert (got[:, :n_q] == 7.0).all() and (got[:, 2 * n_q:] == 7.0).all()


@gpu
def test_pools_past_four_gigabytes(ctx):
    """Pages whose bytes lie behind 2^32: append, read-back and attention."""
    import sgq
    page, n_kv, hd, n_q = 128, 4, 512, 8
    n_pages = (1 << 32) // (page * n_kv * hd) + 40
    pages = sgq.KvPages.empty(n_pages, page, n_kv, hd)
    rng = np.random.default_rng(1)
    ids = np.array([n_pages - 1, 3, n_pages - 30], np.int32)
    n = 2 * page + 21
    slots = [int(ids[i // page]) * page + i % page for i in range(n)]
    x = [rng.standard_normal((n, n_kv, hd)).astype(np.float32) for _ in range(2)]
    ctx.kv_append_paged_q8(pages, *(torch.from_numpy(t).cuda() for t in x), i32(slots))
    kq, vq = np.zeros((3, n_kv, page, hd), np.int8), np.zeros((3, n_kv, page, hd), np.int8)
    ks, vs = np.zeros((3, n_kv), np.float32), np.zeros((3, n_kv), np.float32)
    ref.append(kq, ks, x[0], list(range(n)))
    ref.append(vq, vs, x[1], list(range(n)))
    back = torch.empty((2, n, n_kv, hd), device="cuda")
    ctx.kv_gather_paged_q8(pages, i32(slots), back[0], back[1])
    for b, qn, d in zip(back.cpu().numpy(), (kq, vq), (ks, vs)):
        want = qn[np.arange(n) // page, :, np.arange(n) % page] * d[np.arange(n) // page][..., None]
        assert np.array_equal(b, want)
    q = rng.standard_normal((2, n_q, hd)).astype(np.float32)
    got = attend(ctx, pages, torch.from_numpy(q).cuda(), ids[None], [n], [0, 2], n_q)
    want, mag, cond, peak = ref.attention(q, kq, ks, vq, vs, np.arange(3)[None], [n], [0, 2], 0, hd ** -0.5)
    assert (np.abs(got - want) <= ref.attention_bound(want, mag, cond, peak, hd, n, False)).all()


# ---- together ------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("f16", [True, False])
def test_steps_of_a_server(ctx, f16):
    """Requests come with prompts, decode, finish and give their pages to new
    ones: plan, append and attention of every step against the plain forms."""
    import sgq
    rng = np.random.default_rng(17)
    page, n_q, n_kv, hd, n, width, n_pages = 32, 8, 4, 128, 5, 6, 16
    typ = np.float16 if f16 else np.float32
    pages = sgq.KvPages.empty(n_pages, page, n_kv, hd)
    host = [np.zeros((n_pages, n_kv, page, hd), np.int8), np.zeros((n_pages, n_kv, page, hd), np.int8),
            np.zeros((n_pages, n_kv), np.float32), np.zeros((n_pages, n_kv), np.float32)]
    lens, tables, free, n_free = [0] * n, np.full((n, width), -1, np.int32), np.arange(n_pages, dtype=np.int32), n_pages
    d_lens, d_tables, d_free, d_nf = i32(lens), i32(tables), i32(free), i32([n_free])
    cu, slots, missing, cap = i32([0] * (n + 1)), i32([0] * 160), i32([0]), 160
    ws = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")
    steps = [([40, 0, 33, 1, 0], None), ([1, 70, 1, 1, 0], None), ([1, 1, 30, 1, 5], None),
             ([50, 1, 0, 1, 1], [1, 0, 1, 0, 0]), ([1, 1, 90, 1, 1], None), ([1, 1, 1, 0, 1], [0, 0, 0, 1, 0])]
    for new, done in steps:
        if done:
            ctx.kv_pages_release(i32(done), d_lens, d_tables, d_free, d_nf, page)
            lens, tables, free, n_free = ref.release(done, lens, tables, free, n_free, page)
        ctx.kv_pages_plan(d_lens, i32(new), d_tables, d_free, d_nf, d_nf, d_lens, cu, slots, missing, page)
        tables, lens, h_cu, h_slots, n_free, miss = ref.plan(lens, new, tables, free, n_free, page, cap)
        assert np.array_equal(slots.cpu().numpy(), h_slots) and missing.item() == miss
        x = [rng.standard_normal((cap, n_kv, hd)).astype(typ) for _ in range(2)]
        ctx.kv_append_paged_q8(pages, *(torch.from_numpy(t).cuda() for t in x), slots)
        ref.append(host[0], host[2], x[0], h_slots)
        ref.append(host[1], host[3], x[1], h_slots)
        q = rng.standard_normal((cap, n_q, hd)).astype(typ)
        out = torch.full(q.shape, 7.0, dtype=torch.from_numpy(q).dtype, device="cuda")
        ctx.attn_paged_q8(pages, torch.from_numpy(q).cuda(), d_tables, d_lens, cu, out,
                          max_new=max(new), workspace=ws)
        got = out.double().cpu().numpy()
        assert np.array_equal(d_tables.cpu().numpy(), tables) and d_lens.tolist() == lens
        assert_pages(pages, host)
        want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, lens, h_cu, 0, hd ** -0.5)
        live = ~np.isnan(want)
        bound = ref.attention_bound(want, mag, cond, peak, hd, 200, f16)
        assert (np.abs(got - want) <= bound)[live].all()
        assert (got[~live] == 7.0).all()


@gpu
def test_a_captured_decode_step_replays_with_growing_lengths():
    """plan, append and attention of one token a request recorded once: each
    replay advances lengths, tables and the free stack by itself and equals the
    eager calls, with eager work between the replays."""
    import sgq
    page, n_q, n_kv, hd, n, width, n_pages = 32, 8, 4, 128, 3, 40, 90
    rng = np.random.default_rng(23)
    start = [30, 1000, 63]
    side = torch.cuda.Stream()
    gctx = sgq.GpuContext(0)

    def fresh():
        g = np.random.default_rng(1)
        host = pool(g, n_pages, n_kv, page, hd)
        need = [-(-s // page) for s in start]
        tables = np.full((n, width), -1, np.int32)
        at = 0
        for s, m in enumerate(need):
            tables[s, :m] = np.arange(at, at + m)
            at += m
        free = np.concatenate([np.arange(n_pages - 1, at - 1, -1), np.zeros(at, np.int64)])
        return dict(pages=to_pages(*host), lens=i32(start), new=i32([1] * n), tables=i32(tables),
                    free=i32(free), nf=i32([n_pages - at]), cu=i32([0] * (n + 1)), slots=i32([0] * n),
                    missing=i32([0]), k=torch.zeros((n, n_kv, hd), device="cuda"),
                    v=torch.zeros((n, n_kv, hd), device="cuda"), q=torch.zeros((n, n_q, hd), device="cuda"),
                    out=torch.zeros((n, n_q, hd), device="cuda"),
                    ws=torch.empty(8 << 20, dtype=torch.uint8, device="cuda"))

    def step(c, s):
        c.kv_pages_plan(s["lens"], s["new"], s["tables"], s["free"], s["nf"], s["nf"], s["lens"], s["cu"],
                        s["slots"], s["missing"], page)
        c.kv_append_paged_q8(s["pages"], s["k"], s["v"], s["slots"])
        c.attn_paged_q8(s["pages"], s["q"], s["tables"], s["lens"], s["cu"], s["out"], max_new=1,
                        max_kv=width * page, workspace=s["ws"])

    a, b = fresh(), fresh()
    ectx = sgq.GpuContext(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        gctx.set_stream(side)
        with sgq.GraphRecorder(gctx) as rec:
            step(gctx, a)
    for i in range(5):
        x = [torch.from_numpy(rng.standard_normal(a[m].shape).astype(np.float32)) for m in "kvq"]
        for s in (a, b):
            for m, t in zip("kvq", x):
                s[m].copy_(t)
        torch.cuda.synchronize()
        rec.graph.submit()
        side.synchronize()
        torch.ones(1 << 20, device="cuda").sum().item()  # eager work between the replays
        step(ectx, b)
        torch.cuda.synchronize()
        for m in ("out", "lens", "tables", "slots", "nf", "cu"):
            assert torch.equal(a[m], b[m]), (i, m)
        assert a["lens"].tolist() == [s + i + 1 for s in start] and a["missing"].item() == 0
    del rec


@gpu
@pytest.mark.parametrize("f16", [True, False])
def test_a_very_long_prompt(ctx, f16):
    """70001 tokens of one request planned, appended and attended in one step; rows from
    its start to its end are checked."""
    page, n_q, n_kv, hd, n, width = 128, 2, 1, 128, 70001, 600
    import sgq
    rng = np.random.default_rng(77)
    dt = np.float16 if f16 else np.float32
    q, k, v = (rng.standard_normal((n, h, hd)).astype(dt) for h in (n_q, n_kv, n_kv))
    pages = sgq.KvPages.empty(width, page, n_kv, hd)
    lens, tables, cu, slots, missing = i32([0]), i32(np.full((1, width), -1)), i32([0, 0]), i32([0] * n), i32([9])
    nf = i32([width])
    ctx.kv_pages_plan(lens, i32([n]), tables, i32(rng.permutation(width)), nf, nf, lens, cu, slots, missing, page)
    qd, kd, vd = (torch.from_numpy(x).cuda() for x in (q, k, v))
    ctx.kv_append_paged_q8(pages, kd, vd, slots)
    got = attend(ctx, pages, qd, tables.cpu().numpy(), [n], np.array([0, n]), n_q)
    assert missing.item() == 0 and lens.item() == n and nf.item() == width - -(-n // page)
    table = tables.cpu().numpy()
    kq, vq, ks, vs = from_pages(pages)
    for x, quants, d in ((k, kq, ks), (v, vq, vs)):  # runs of whole pages: half a step of the block's scale
        for row in rng.integers(0, n, 300):
            p, o = table[0, row // page], row % page
            run = x[row // page * page:row // page * page + page].astype(np.float64)
            assert d[p, 0] == np.float32(np.abs(run).max().astype(np.float32) / np.float32(127))
            assert (quants[p, 0, o] == np.rint(x[row, 0].astype(np.float64) / np.float64(d[p, 0]))).all()
    for row in (0, 1, 127, 128, 4095, 35000, 69888, n - 1):
        want, mag, cond, peak = ref.attention(q[row:row + 1], kq, ks, vq, vs, table, [row + 1], np.array([0, 1]), 0,
                                              hd ** -0.5)
        bound = ref.attention_bound(want, mag, cond, peak, hd, row + 1, f16)
        assert (np.abs(got[row:row + 1] - want) <= bound).all(), row


@gpu
@pytest.mark.parametrize("new", [1, 20])
def test_attention_of_many_heads(ctx, new):
    """1024 kv heads: more units than a round of the GPU has workgroups."""
    check_attention(ctx, 3, [41], [new], 32, 1024, 1024, 128, True)


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n", [255, 300, 700])
def test_attention_of_many_requests(ctx, f16, n):
    """Single tokens, chunks and empty requests in batches past one scan of the
    lengths; a few requests are long enough to be cut."""
    rng = np.random.default_rng(n)
    new = rng.choice([0, 1, 1, 1, 2, 20, 41], n)
    kv = new + rng.integers(0, 70, n)
    for s in (0, n // 2, n - 1):
        new[s], kv[s] = (1, 45, 150)[s * 2 // n], 700
    check_attention(ctx, n, list(kv), list(new), 32, 2, 1, 128, f16, rows=int(new.sum()) + 3)


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,n_q,n_kv,new", [
    (128, 6, 3, [130]), (128, 10, 5, [9, 1, 1]), (128, 64, 1, [1, 3]), (256, 12, 6, [40, 1]), (512, 7, 7, [33, 2])])
@pytest.mark.parametrize("room", [0, 200_000, 3_000_000, 64 << 20])
def test_attention_of_chunks_over_long_caches(ctx, f16, hd, n_q, n_kv, new, room):
    """Row tiles cut into parts, with heads that do not divide the GPU and
    workspaces for none, few and all of the parts."""
    rng = np.random.default_rng(hd + n_kv)
    page, kv = 64, [2000 + 700 * i for i in range(len(new))]
    host, tables, cu = batch(rng, kv, new, page, n_kv, hd)
    q = rng.standard_normal((cu[-1], n_q, hd)).astype(np.float16 if f16 else np.float32)
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q, split=False,
                 workspace=torch.empty(room, dtype=torch.uint8, device="cuda") if room else None)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, 0, hd ** -0.5)
    bound = ref.attention_bound(want, mag, cond, peak, hd, max(kv), f16)
    assert (np.abs(got - want) <= bound).all()


@gpu
def test_a_captured_mixed_step_follows_its_lengths():
    """One recording serves steps of different chunks: requests grow from nothing to
    many rows and back to single tokens between the replays."""
    import sgq
    page, n_q, n_kv, hd, n, width, n_pages, rows = 32, 4, 2, 128, 4, 64, 200, 200
    rng = np.random.default_rng(5)
    side, gctx, ectx = torch.cuda.Stream(), sgq.GpuContext(0), sgq.GpuContext(0)

    def fresh():
        host = pool(np.random.default_rng(1), n_pages, n_kv, page, hd)
        return dict(pages=to_pages(*host), lens=i32([0] * n), new=i32([0] * n), done=i32([0] * n),
                    tables=i32(np.full((n, width), -1)), free=i32(np.arange(n_pages)), nf=i32([n_pages]),
                    cu=i32([0] * (n + 1)), slots=i32([0] * rows), missing=i32([0]),
                    k=torch.zeros((rows, n_kv, hd), device="cuda"), v=torch.zeros((rows, n_kv, hd), device="cuda"),
                    q=torch.zeros((rows, n_q, hd), device="cuda"), out=torch.zeros((rows, n_q, hd), device="cuda"),
                    ws=torch.empty(32 << 20, dtype=torch.uint8, device="cuda"))

    def step(c, s):
        c.kv_pages_release(s["done"], s["lens"], s["tables"], s["free"], s["nf"], page)
        c.kv_pages_plan(s["lens"], s["new"], s["tables"], s["free"], s["nf"], s["nf"], s["lens"], s["cu"],
                        s["slots"], s["missing"], page)
        c.kv_append_paged_q8(s["pages"], s["k"], s["v"], s["slots"])
        c.attn_paged_q8(s["pages"], s["q"], s["tables"], s["lens"], s["cu"], s["out"], max_new=rows,
                        max_kv=width * page, workspace=s["ws"])

    a, b = fresh(), fresh()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        gctx.set_stream(side)
        with sgq.GraphRecorder(gctx) as rec:
            step(gctx, a)
    lens = np.zeros(n, int)
    for i, (new, done) in enumerate([([150, 0, 1, 20], [0, 0, 0, 0]), ([1, 190, 1, 1], [0, 0, 0, 0]),
                                     ([1, 1, 150, 40], [1, 0, 0, 0]), ([0, 0, 0, 0], [0, 0, 0, 1]),
                                     ([1, 1, 1, 100], [0, 0, 0, 0])]):
        x = [torch.from_numpy(rng.standard_normal(a[m].shape).astype(np.float32)) for m in "kvq"]
        for s in (a, b):
            for m, t in zip("kvq", x):
                s[m].copy_(t)
            s["new"].copy_(i32(new))
            s["done"].copy_(i32(done))
            s["out"].fill_(7.0)
        torch.cuda.synchronize()
        rec.graph.submit()
        side.synchronize()
        torch.ones(1 << 20, device="cuda").sum().item()  # eager work between the replays
        step(ectx, b)
        torch.cuda.synchronize()
        lens = np.where(done, 0, lens) + new
        for m in ("out", "lens", "tables", "slots", "nf", "cu"):
            assert torch.equal(a[m], b[m]), (i, m)
        assert a["lens"].tolist() == list(lens) and a["missing"].item() == 0
        assert (a["out"][sum(new):] == 7.0).all() and not (a["out"][:sum(new)] == 7.0).all(-1).any()
    del rec


@gpu
def test_two_streams_at_once(ctx):
    """Two contexts on two streams, each with its own cache and workspace."""
    import sgq
    kv, page, n_q, n_kv, hd = [5000, 1200], 32, 8, 4, 128
    runs = []
    for i in range(2):
        rng = np.random.default_rng(i)
        host, tables, cu = batch(rng, kv, [1, 1], page, n_kv, hd)
        q = torch.from_numpy(rng.standard_normal((2, n_q, hd)).astype(np.float16)).cuda()
        runs.append(dict(pages=to_pages(*host), q=q, tables=i32(tables), kv=i32(kv), cu=i32(cu),
                         out=torch.zeros_like(q), ws=torch.empty(8 << 20, dtype=torch.uint8, device="cuda"),
                         ctx=sgq.GpuContext(0), stream=torch.cuda.Stream()))

    def call(c, r):
        c.attn_paged_q8(r["pages"], r["q"], r["tables"], r["kv"], r["cu"], r["out"], max_new=1,
                        max_kv=5000, workspace=r["ws"])

    want = []
    for r in runs:
        call(ctx, r)
        want.append(r["out"].clone())
        r["out"].zero_()
    torch.cuda.synchronize()
    for r in runs:
        r["ctx"].set_stream(r["stream"])
    for _ in range(20):
        for r in runs:
            call(r["ctx"], r)
    torch.cuda.synchronize()
    for r, w in zip(runs, want):
        assert torch.equal(r["out"], w)


# ---- refusals (no launch, so no device is needed) ---------------------------------------------

def _pages_struct(**kw):
    import sgq
    v = dict(k=0x10000, v=0x20000, ks=0x30000, vs=0x40000, n_pages=8, page=32, n_kv=4, hd=128) | kw
    return sgq._KvPages(v["k"], v["v"], v["ks"], v["vs"], v["n_pages"], v["page"], v["n_kv"], v["hd"])


FAKE = C.c_void_p(0x50000)  # never dereferenced: every call here is refused before it


def refused(rc, text):
    import sgq
    msg = sgq.lib().sgq_last_error().decode()
    assert rc == 6 and text in msg, (rc, msg)


@pytest.mark.parametrize("change,text", [
    (dict(page=16), "page_size"), (dict(page=0), "page_size"), (dict(page=96), "page_size"),
    (dict(hd=64), "head_dim"), (dict(hd=192), "head_dim"), (dict(n_kv=0), "n_kv_heads"),
    (dict(n_kv=1025), "n_kv_heads"), (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 27), "n_pages"),
    (dict(k=0), "NULL"), (dict(vs=0), "NULL"), (dict(k=0x10008), "misaligned"), (dict(ks=0x30002), "misaligned"),
])
def test_bad_pages_are_refused(change, text):
    import sgq
    L, p = sgq.lib(), _pages_struct(**change)
    pp = C.byref(p)
    pp = C.cast(pp, C.c_void_p)
    refused(L.sgq_kv_append_paged_q8(FAKE, pp, FAKE, 512, FAKE, 512, 0, FAKE, 3), text)
    refused(L.sgq_kv_gather_paged_q8(FAKE, pp, FAKE, 3, 0, FAKE, 512, FAKE, 512), text)
    refused(L.sgq_attn_paged_q8(FAKE, pp, FAKE, 1024, 0, FAKE, 4, FAKE, FAKE, 2, 2, 8, 1, 99, 0, 0.1, FAKE,
                                1024, None, 0), text)
    assert L.sgq_attn_paged_workspace(pp, 2, 2, 8, 1, 99) == 0


def test_bad_arguments_are_refused():
    import sgq
    L = sgq.lib()
    p = _pages_struct()
    pp = C.cast(C.byref(p), C.c_void_p)
    odd = C.c_void_p(0x50008)

    def app(ctx=FAKE, pages=pp, k=FAKE, ks=512, v=FAKE, vs=512, act=0, slots=FAKE, n=3):
        return L.sgq_kv_append_paged_q8(ctx, pages, k, ks, v, vs, act, slots, n)

    for kw, text in [(dict(ctx=None), "NULL"), (dict(k=None), "NULL"), (dict(slots=None), "NULL"),
                     (dict(pages=None), "NULL"), (dict(act=2), "activation type"), (dict(act=-1), "activation type"),
                     (dict(ks=511), "stride"), (dict(vs=514), "aligned"), (dict(act=1, ks=516), "aligned"),
                     (dict(k=odd), "aligned"), (dict(n=(1 << 22) + 1), "n_tokens")]:
        refused(app(**kw), text)

    def att(ctx=FAKE, pages=pp, q=FAKE, qs=1024, act=0, tables=FAKE, width=4, kv=FAKE, cu=FAKE, n=2, rows=2,
            n_q=8, max_new=1, max_kv=99, window=0, scale=0.1, out=FAKE, os_=1024, ws=None, wb=0):
        return L.sgq_attn_paged_q8(ctx, pages, q, qs, act, tables, width, kv, cu, n, rows, n_q, max_new, max_kv,
                                   window, scale, out, os_, ws, wb)

    for kw, text in [(dict(ctx=None), "NULL"), (dict(q=None), "NULL"), (dict(cu=None), "NULL"),
                     (dict(tables=None), "NULL"), (dict(act=3), "activation type"), (dict(n_q=6), "query heads"),
                     (dict(n_q=0), "query heads"), (dict(n_q=4 * 65, qs=40000, os_=40000), "query heads"),
                     (dict(n=0), "n_seqs"), (dict(n=4097), "n_seqs"), (dict(width=0), "max_pages"),
                     (dict(width=1 << 26), "max_pages"), (dict(window=1 << 31), "window"),
                     (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
                     (dict(qs=1000), "stride"), (dict(os_=1026), "aligned"), (dict(out=odd), "aligned"),
                     (dict(ws=odd, wb=1 << 20), "workspace"), (dict(rows=(1 << 22) + 1), "n_tokens")]:
        refused(att(**kw), text)

    def plan(ctx=FAKE, cached=FAKE, new=C.c_void_p(0x60000), n=2, page=32, tables=FAKE, width=4,
             free=C.c_void_p(0x70000), pages=9, nf=FAKE, nfo=FAKE, kv=FAKE, cu=FAKE, slots=FAKE, rows=4, miss=FAKE):
        return L.sgq_kv_pages_plan(ctx, cached, new, n, page, tables, width, free, pages, nf, nfo, kv, cu, slots,
                                   rows, miss)

    for kw, text in [(dict(ctx=None), "NULL"), (dict(new=None), "NULL"), (dict(slots=None), "NULL"),
                     (dict(miss=None), "NULL"), (dict(n=0), "n_seqs"), (dict(n=5000), "n_seqs"),
                     (dict(page=48), "page_size"), (dict(width=0), "max_pages"), (dict(pages=0), "n_pages"),
                     (dict(rows=1 << 23), "n_tokens"), (dict(new=FAKE), "overlapping"), (dict(free=FAKE), "overlapping")]:
        refused(plan(**kw), text)
    for kw, text in [(dict(done=None), "NULL"), (dict(n=0), "n_seqs"), (dict(page=7), "page_size"),
                     (dict(kv=C.c_void_p(0x60000)), "overlapping")]:
        v = dict(done=C.c_void_p(0x60000), n=2, page=32, kv=FAKE) | kw
        refused(L.sgq_kv_pages_release(FAKE, v["done"], v["n"], v["page"], v["kv"], FAKE, 4, C.c_void_p(0x70000), 9,
                                       FAKE), text)


def test_steps_too_large_for_a_launch_are_refused():
    """Up to 2^26 (row, head) pairs: below it every grid has fewer than 2^32 threads."""
    import sgq
    L = sgq.lib()
    p = _pages_struct(n_kv=64)
    pp = C.cast(C.byref(p), C.c_void_p)
    w, rows = 64 * 128, (1 << 20) + 1
    refused(L.sgq_kv_append_paged_q8(FAKE, pp, FAKE, w, FAKE, w, 0, FAKE, rows), "heads")
    refused(L.sgq_kv_gather_paged_q8(FAKE, pp, FAKE, rows, 0, FAKE, w, FAKE, w), "heads")
    refused(L.sgq_attn_paged_q8(FAKE, pp, FAKE, w, 0, FAKE, 4, FAKE, FAKE, 2, rows, 64, 1, 99, 0, 0.1, FAKE, w,
                                None, 0), "heads")
    assert L.sgq_attn_paged_workspace(pp, 2, rows, 64, 1, 99) == 0
    # the most that is taken, of many requests: no split makes more workgroups than a launch takes
    for n_kv, n_q, seqs, rows in [(1, 1, 4096, 4096), (100, 100, 4096, 1), (128, 8192, 4096, 4096)]:
        p = _pages_struct(n_kv=n_kv, n_pages=1 << 20)
        pp = C.cast(C.byref(p), C.c_void_p)
        hd_row = (128 + 2) * 4
        for max_new in (1, 17, 1 << 22):
            got = L.sgq_attn_paged_workspace(pp, seqs, rows, n_q, max_new, 1 << 25)
            assert got % hd_row == 0 and got // hd_row < 1 << 31


def test_workspace_follows_the_shape():
    """What the splits need: nothing where the rows fill the GPU or the requests
    are short, whole split rows otherwise."""
    import sgq
    L = sgq.lib()
    pp = C.cast(C.byref(_pages_struct(n_kv=16, n_pages=4096)), C.c_void_p)
    row = 32 * (128 + 2) * 4
    long1 = L.sgq_attn_paged_workspace(pp, 1, 1, 32, 1, 32768)
    assert long1 >= 2 * row and long1 % row == 0
    assert L.sgq_attn_paged_workspace(pp, 1, 1, 32, 1, 40) == 0
    assert L.sgq_attn_paged_workspace(pp, 1, 0, 32, 1, 40) == 0
    assert L.sgq_attn_paged_workspace(pp, 1, 1, 31, 1, 4000) == 0


def test_tensors_are_checked_before_the_call():
    """The Python mirror's own checks (types, shapes, strides, devices)."""
    import sgq
    z = torch.zeros
    good = (z((4, 2, 32, 128), dtype=torch.int8), z((4, 2, 1, 128, 32), dtype=torch.int8), z((4, 2)), z((4, 2)))
    for i, bad in [(0, z((4, 2, 32), dtype=torch.int8)), (0, z((4, 2, 48, 128), dtype=torch.int8)),
                   (1, z((4, 2, 32, 128), dtype=torch.int8)), (2, z((4, 3))), (3, z((4, 2), dtype=torch.float16)),
                   (0, z((4, 2, 32, 128)))]:
        with pytest.raises(sgq.ValidationError):
            sgq.KvPages(*[bad if i == j else t for j, t in enumerate(good)])
    with pytest.raises(sgq.ValidationError):  # host tensors
        sgq.KvPages(*good)
    dev = torch.device("cpu")
    rows = z((3, 2, 128))
    assert sgq._rows(rows, 2, 128, dev, "x") == (rows.data_ptr(), 256, 3)
    assert sgq._rows(z((3, 5, 128))[:, 1:3], 2, 128, dev, "x")[1] == 640
    assert sgq._rows(z((1, 5, 128)).expand(1, 5, 128)[:, :2], 2, 128, dev, "x")[1] == 256
    for bad in (z((3, 2, 64)), z((3, 256)), z((3, 2, 128), dtype=torch.float64), z((3, 128, 2)).transpose(1, 2),
                z((1, 2, 128)).expand(3, 2, 128), z((3, 2, 256))[..., ::2]):
        with pytest.raises(sgq.ValidationError):
            sgq._rows(bad, 2, 128, dev, "x")
    with pytest.raises(sgq.ValidationError):
        sgq._i32(z(4), 4, dev, "x")
    with pytest.raises(sgq.ValidationError):
        sgq._i32(z(4, dtype=torch.int32), 5, dev, "x")
    with pytest.raises(sgq.ValidationError):
        sgq._i32(z((4, 2), dtype=torch.int32)[:, 0], 4, dev, "x")
