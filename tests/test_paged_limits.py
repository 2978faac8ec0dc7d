"""The paged 8-bit KV cache at the ends of what its entry points accept: scores of
any finite size, K and V blocks far apart, many query heads a kv head, blocks that
grow again and again, pools that run out.  Plain forms are those of
tests/_paged.py."""
import ctypes as C

import numpy as np
import pytest
import torch

import _paged as ref
from test_paged import FAKE, _pages_struct, attend, batch, from_pages, i32, pool, refused, to_pages

gpu = pytest.mark.gpu


# ---- attention ----------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("k_scale", [1e4, 1e7, 1e12, 1e28, 1e33])
def test_attention_of_scores_of_any_size(ctx, f16, new, sign, k_scale):
    """Scores of 10^6 to 10^36, all of one sign: one key is at least a quarter ahead of
    all others, so the output is its value.  Its weight is a power of two and the others'
    are 0; what is left are the roundings of 1/vs, of the sum, its reciprocal and the
    product (2^-24 each) and the output's."""
    rng = np.random.default_rng(int(np.log10(k_scale)) + new)
    page, n_q, n_kv, hd, kv = 32, 4, 2, 128, [900, 130]
    host, tables, cu = batch(rng, kv, [new, new], page, n_kv, hd)
    host[2][:] = k_scale
    host[0][:] = rng.integers(50, 81, host[0].shape)
    best = [int(rng.integers(0, n - new)) for n in kv]
    for s, j in enumerate(best):
        host[0][tables[s, j // page], :, j % page] = 120 if sign > 0 else 30
    q = (sign * (0.5 + rng.random((cu[-1], n_q, hd)))).astype(np.float16 if f16 else np.float32)
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q)
    for s, j in enumerate(best):
        p = tables[s, j // page]
        want = host[1][p, :, j % page].astype(np.float64) * host[3][p].astype(np.float64)[:, None]
        want = np.repeat(want, n_q // n_kv, 0)[None]
        bound = np.abs(want) * (2.0 ** -22 + (2.0 ** -11 if f16 else 2.0 ** -24))
        assert (np.abs(got[cu[s]:cu[s + 1]] - want) <= bound).all(), s


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("k_scale", [1e20, 1e33, 1e35])
def test_attention_of_queries_without_a_sum_over_large_k_scales(ctx, f16, new, k_scale):
    """q of zeros weighs all keys alike; q of pairs that cancel prefers the key whose
    quants differ most."""
    rng = np.random.default_rng(new)
    page, n_q, n_kv, hd, kv = 32, 4, 2, 128, [330, 130]
    host, tables, cu = batch(rng, kv, [new, new], page, n_kv, hd)
    host[2][:] = k_scale
    host[0][:, :, :, ::2] = rng.integers(50, 60, host[0][:, :, :, ::2].shape)
    host[0][:, :, :, 1::2] = rng.integers(40, 50, host[0][:, :, :, ::2].shape)
    for s in range(2):
        host[0][tables[s, 1], :, 7, ::2], host[0][tables[s, 1], :, 7, 1::2] = 110, 10
    q = np.zeros((cu[-1], n_q, hd), np.float16 if f16 else np.float32)
    q[:, 1::2, ::2], q[:, 1::2, 1::2] = 1, -1  # heads 1 and 3
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q)
    small = [t.copy() for t in host]
    small[2][:] = 1  # the same softmax, to less than fp64 tells
    want, mag, cond, peak = ref.attention(q, small[0], small[2], host[1], host[3], tables, kv, cu, 0, hd ** -0.5)
    # exact scores (0, or apart by 10^20 and more): the weights' and sums' roundings only
    bound = ref.attention_bound(want, mag, 0 * cond, peak, hd, max(kv), f16)
    rows = np.concatenate([np.arange(kv[s] - new, kv[s]) for s in range(2)]) >= 39
    assert rows.any()
    assert (np.abs(got - want) <= bound)[:, ::2].all()
    assert (np.abs(got - want) <= bound)[rows].all()

@gpu
@pytest.mark.parametrize("hd,n_q,n_kv", [(128, 4, 2), (256, 8, 2), (512, 8, 1)])
@pytest.mark.parametrize("new", [1, 2, 9])
@pytest.mark.parametrize("every", [1, 3])
def test_attention_of_offset_queries_over_blocks_with_an_outlier(ctx, hd, n_q, n_kv, new, every):
    """f16 rows of q around 40 over blocks whose quants are 0 and a few +-1 beside an
    outlier of 127 in a dim that q does not have: 128·Σq is two hundred and more times
    the score.  `every`: other blocks between them use their whole range."""
    rng = np.random.default_rng(hd + new)
    page, kv = 32, [300, 41, 2500]
    host, tables, cu = batch(rng, kv, [new] * 3, page, n_kv, hd)
    for s in range(3):
        for p in tables[s, ::every]:
            if p >= 0:
                k = np.zeros((n_kv, page, hd), np.int8)
                at = rng.integers(1, hd, (n_kv, page, 4))
                np.put_along_axis(k, at, rng.choice([-1, 1], at.shape).astype(np.int8), 2)
                k[:, :, 0] = 127
                host[0][p] = k
                host[2][p] = 1.0
            if every > 1:  # the others: scores of a like size
                for o in tables[s, 1::every]:
                    host[2][o] = 2e-3
    q = 40 + rng.standard_normal((cu[-1], n_q, hd))
    q[:, :, 0] = 0
    q = q.astype(np.float16)
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q, scale=1 / 32)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, 0, 1 / 32)
    bound = ref.attention_bound(want, mag, cond, peak, hd, max(kv), True)
    worst = (np.abs(got - want) / bound).max()
    assert worst <= 1


@gpu
@pytest.mark.parametrize("hd,n_q,n_kv", [(128, 4, 2), (512, 8, 1)])
@pytest.mark.parametrize("first", [0, 9000, 17900])
def test_attention_of_offset_queries_over_a_long_request(ctx, hd, n_q, n_kv, first):
    """The same in an uncut request of more pages than a wave looks up at a time, of which
    only those of tokens first .. first + 100 have an outlier."""
    rng = np.random.default_rng(hd + first)
    page, kv = 32, [18000]
    host, tables, cu = batch(rng, kv, [1], page, n_kv, hd)
    host[2][:] = 1e-4
    for p in tables[0, first // page:(first + 100) // page]:
        k = np.zeros((n_kv, page, hd), np.int8)
        at = rng.integers(1, hd, (n_kv, page, 8))
        np.put_along_axis(k, at, 1, 2)
        k[:, :, 0] = 127
        host[0][p], host[2][p] = k, 1.0
    q = 40 + rng.standard_normal((1, n_q, hd))
    q[:, :, 0] = 0
    q = q.astype(np.float16)
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q, scale=1 / 16, split=False)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, 0, 1 / 16)
    bound = ref.attention_bound(want, mag, cond, peak, hd, kv[0], True)
    worst = (np.abs(got - want) / bound).max()
    assert worst <= 1

@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("tokens", [300, 160_000])
def test_attention_over_a_long_run_of_zero_blocks(ctx, f16, new, tokens):
    """V blocks of zeros (scale 0) with scores 7.9 (log2) above the first keys', where
    the running maximum need not move, and a last page that is not zero: the sum of
    weights over scales stays finite."""
    rng = np.random.default_rng(tokens + new)
    page, n_q, n_kv, hd = 128, 2, 1, 128
    host, tables, cu = batch(rng, [tokens], [new], page, n_kv, hd)
    last = tables[0, (tokens - 1 - new) // page:]
    rest = np.setdiff1d(tables[0][tables[0] >= 0], last)
    host[1][rest], host[3][rest] = 0, 0
    host[0][:], host[2][:] = 0, 1 / 64
    host[0][:, :, :, 0] = 64  # scores of 7.9
    host[0][tables[0, 0], :, :, 0] = 0
    q = np.zeros((new, n_q, hd), np.float16 if f16 else np.float32)
    scale = 7.9 * np.log(2)
    q[:, :, 0] = 1
    for split in (True, False):
        got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, [tokens], cu, n_q, scale=scale,
                     split=split)
        want, mag, cond, peak = ref.attention(q[-1:], host[0], host[2], host[1], host[3], tables, [tokens],
                                              np.array([0, 1]), 0, scale)
        assert np.abs(want).max() > 1e-6
        bound = ref.attention_bound(want, mag, cond, peak, hd, tokens, f16)
        assert (np.abs(got[-1:] - want) <= bound).all(), split


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [1, 20])
def test_attention_over_v_scales_to_the_smallest(ctx, f16, new):
    """V scales from the smallest subnormal on beside ordinary ones and in requests of
    their own, to 127*2^-80 more than the bound."""
    rng = np.random.default_rng(new)
    page, n_q, n_kv, hd, kv = 32, 4, 2, 128, [200, 130, 70]
    host, tables, cu = batch(rng, kv, [new] * 3, page, n_kv, hd)
    small = (2.0 ** rng.uniform(-149, -70, host[3].shape)).astype(np.float32)
    for s in range(3):  # every other page, all pages, all pages at 1e-35
        for j, p in enumerate(tables[s]):
            if p >= 0 and (s or j % 2):
                host[3][p] = small[p] if s < 2 else 1e-35
    q = rng.standard_normal((cu[-1], n_q, hd)).astype(np.float16 if f16 else np.float32)
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, 0, hd ** -0.5)
    bound = ref.attention_bound(want, mag, cond, peak, hd, max(kv), f16) + 127 * 2.0 ** -80
    # log2 of a V scale (|log2| <= 80) is rounded to 2^-18 at most, as a factor 2^-18
    assert (np.abs(got - want) <= bound + mag * 2.0 ** -17).all()


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,n_q,n_kv", [(128, 64, 1), (128, 34, 2), (256, 20, 1), (512, 32, 1)])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [1, 0, 2, 9]])
@pytest.mark.parametrize("room", [0, 400_000, 64 << 20])
def test_attention_of_more_than_16_query_heads_a_kv_head(ctx, f16, hd, n_q, n_kv, new, room):
    """A single token has more rows than the kernel of few rows takes: every request goes
    to the other one, and the whole workspace with it."""
    rng = np.random.default_rng(hd + n_q)
    page, kv = 64, [2100, 3, 900, 3000]
    kv = [max(k, n) for k, n in zip(kv, new)]
    host, tables, cu = batch(rng, kv, new, page, n_kv, hd)
    q = rng.standard_normal((cu[-1] + 2, n_q, hd)).astype(np.float16 if f16 else np.float32)
    got = attend(ctx, to_pages(*host), torch.from_numpy(q).cuda(), tables, kv, cu, n_q, split=False,
                 workspace=torch.empty(room, dtype=torch.uint8, device="cuda") if room else None)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, 0, hd ** -0.5)
    live = ~np.isnan(want)
    assert (got[~live] == 7.0).all()
    bound = ref.attention_bound(want, mag, cond, peak, hd, max(kv), f16)
    assert (np.abs(got - want) <= bound)[live].all()


def test_workspace_of_more_than_16_query_heads_a_kv_head():
    """No part of it is for requests of few rows, which cannot occur: at most two rounds
    of 256 parts of 256 rows."""
    import sgq
    L = sgq.lib()
    p = _pages_struct(n_kv=1, n_pages=4096)
    pp = C.cast(C.byref(p), C.c_void_p)
    row = (128 + 2) * 4
    for n_q, few in ((16, True), (17, False), (32, False), (64, False)):
        got = L.sgq_attn_paged_workspace(pp, 64, 64, n_q, 40, 32768)
        assert got and got % row == 0
        assert (got // row > 512 * 256) == few, n_q


@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,n_q,n_kv", [(128, 8, 4), (256, 8, 2), (512, 8, 1)])
def test_attention_of_drafts_beside_a_nan_block_a_missing_page_and_a_zero_one(ctx, f16, hd, n_q, n_kv):
    """Two tokens of which the second begins a page: a NaN scale there is the second row's
    alone, and a page that is missing or zero weighs as it should, at every head_dim."""
    rng = np.random.default_rng(hd)
    page, kv = 32, [129, 97, 65]
    host, tables, cu = batch(rng, kv, [2, 2, 2], page, n_kv, hd)
    tables[1, 1] = -1
    host[1][tables[2, 0]], host[3][tables[2, 0]] = 0, 0
    q = rng.standard_normal((cu[-1], n_q, hd)).astype(np.float16 if f16 else np.float32)
    args = (torch.from_numpy(q).cuda(), tables, kv, cu, n_q)
    got = attend(ctx, to_pages(*host), *args)
    want, mag, cond, peak = ref.attention(q, host[0], host[2], host[1], host[3], tables, kv, cu, 0, hd ** -0.5)
    assert (np.abs(got - want) <= ref.attention_bound(want, mag, cond, peak, hd, max(kv), f16)).all()
    for d in (host[2], host[3]):
        keep = d.copy()
        for s in range(3):
            d[tables[s, (kv[s] - 1) // page]] = np.nan
        bad = attend(ctx, to_pages(*host), *args)
        d[:] = keep
        assert np.isnan(bad[1::2]).all() and np.array_equal(bad[::2], got[::2])

# ---- pools that run out -------------------------------------------------------------------

def all_pages(tables, lens, free, n_free, page):
    """The pages in use and on the stack, each once if none is lost."""
    used = [p for row, n in zip(tables, lens) for p in row[:min(-(-n // page), len(row))] if p >= 0]
    return sorted([int(p) for p in used] + [int(p) for p in free[:n_free]])


class Server:
    """Five requests over 16 pages of 32 tokens, on the device or as the plain form."""
    page, n, width, pool = 32, 5, 8, 16

    def __init__(self, ctx=None):
        self.ctx = ctx
        self.lens, self.tables = [0] * self.n, np.full((self.n, self.width), -1, np.int32)
        self.free, self.n_free = np.arange(self.pool, dtype=np.int32), self.pool
        self.slots = None

    def plan(self, new, rows=400):
        if self.ctx is None:
            self.tables, self.lens, _, self.slots, self.n_free, missing = ref.plan(
                self.lens, new, self.tables, self.free, self.n_free, self.page, rows)
            return missing
        d = [i32(x) for x in (self.lens, new, self.tables, self.free, [self.n_free])]
        out = [i32([0]), i32([0] * self.n), i32([0] * (self.n + 1)), i32([0] * rows), i32([0])]
        self.ctx.kv_pages_plan(*d, *out, self.page)
        self.tables, self.lens, self.n_free = d[2].cpu().numpy(), out[1].tolist(), out[0].item()
        self.slots = out[3].tolist()
        assert np.array_equal(d[3].cpu().numpy(), self.free)  # popping leaves the entries
        return out[4].item()

    def release(self, done):
        if self.ctx is None:
            self.lens, self.tables, self.free, self.n_free = ref.release(
                done, self.lens, self.tables, self.free, self.n_free, self.page)
            return
        d = [i32(x) for x in (done, self.lens, self.tables, self.free, [self.n_free])]
        self.ctx.kv_pages_release(*d, self.page)
        self.lens, self.tables, self.free, self.n_free = (d[1].tolist(), d[2].cpu().numpy(), d[3].cpu().numpy(),
                                                          d[4].item())

    def whole(self):
        return all_pages(self.tables, self.lens, self.free, self.n_free, self.page) == list(range(self.pool))


def run_out_and_go_on(ctx):
    for undo in (True, False):
        s = Server(ctx)
        assert s.plan([100, 30, 64, 1, 20]) == 0 and s.whole()  # 4 + 1 + 2 + 1 + 1 of 16
        lens, n_free = list(s.lens), s.n_free
        assert s.plan([1, 120, 1, 40, 90]) > 0 and s.n_free == 0  # 4 + 1 + 1 + 3, of 7
        short = [i for i in range(s.n) if (s.tables[i, :-(-s.lens[i] // s.page)] < 0).any()]
        assert short == [4] and (s.tables[4] >= 0).sum() == 2  # one of the three it needs
        if undo:
            s.lens, s.n_free = lens, n_free
            assert s.whole()
            s.release([0, 0, 1, 0, 0])
            assert s.whole()
            assert s.plan([1, 120, 0, 40, 90]) == 0 and s.whole()
            assert s.lens == [101, 150, 0, 41, 110]
        else:
            assert s.whole()  # with the advanced lengths the tables hold what was popped
            s.release([int(i in short) for i in range(s.n)])
            assert s.whole() and s.lens[4] == 0
            assert s.plan([1, 1, 1, 1, 33]) == 0 and s.whole()
        live = [x for x in s.slots if x >= 0]
        assert len(set(live)) == len(live)  # no slot of two tokens


def test_a_pool_that_runs_out_loses_no_page_plain():
    run_out_and_go_on(None)


@gpu
def test_a_pool_that_runs_out_loses_no_page(ctx):
    """missing > 0, then either the step undone (lengths and count of free pages), others
    released and the step planned again, or the short request released as it is."""
    run_out_and_go_on(ctx)


# ---- blocks that grow again and again ---------------------------------------------------

def append_rows(q, d, x, slots, growth):
    """One append of rows of one page, as the header has it."""
    page = q.shape[2]
    p, offs = slots[0] // page, [s % page for s in slots]
    assert all(s // page == p for s in slots)
    r = x.astype(np.float64)
    for h in range(q.shape[1]):
        need, old = np.float32(np.abs(r[:, h]).max() / 127.0), d[p, h]
        if 0 in offs:
            d[p, h] = need
        elif need > old:
            d[p, h] = max(need, old * np.float32(growth))
            q[p, h] = np.rint(q[p, h].astype(np.float64) * float(old) / float(d[p, h]))
        q[p, h, offs] = np.rint(r[:, h] / float(d[p, h]))


def rising_rows(rng, page, n_kv, hd, rise):
    """A page's rows, each `rise` times the size of the one before it."""
    x = rng.uniform(-1, 1, (page, n_kv, hd)) * 0.9
    x[:, :, 0] = 1
    return (x * rise ** np.arange(page)[:, None, None]).astype(np.float32)


def one_by_one(x, growth):
    """Quants, scales and the largest |value - row| in steps after a page's rows were
    appended one call each."""
    page = len(x)
    q, d = np.zeros((1, x.shape[1], page, x.shape[2]), np.int8), np.zeros((1, x.shape[1]), np.float32)
    for i in range(page):
        append_rows(q, d, x[i:i + 1], [i], growth)
    back = q[0].transpose(1, 0, 2).astype(np.float64) * d[0].astype(np.float64)[None, :, None]
    return q, d, (np.abs(back - x) / d[0][None, :, None]).max()


def steps_lost(page):
    """growth/(2·(growth-1)) at 1.25, and that each grown scale is an fp32 number."""
    return 2.5 * (1 + page * 2.0 ** -23)


@pytest.mark.parametrize("rise", [1.005, 1.02, 1.3, 1.9])
@pytest.mark.parametrize("page", [32, 128])
def test_headroom_bounds_what_rounding_again_loses(page, rise):
    """The definition itself; growing as far as needed alone loses tens of steps."""
    x = rising_rows(np.random.default_rng(page), page, 1, 128, rise)
    assert one_by_one(x, 1.25)[2] <= steps_lost(page)
    q, d, plain = one_by_one(x, 1.0)
    assert plain <= page / 2
    if rise == 1.005 and page == 128:
        assert plain > 20
    q1, d1 = np.zeros_like(q), np.zeros_like(d)  # without headroom: the shared plain form's rule
    for i in range(page):
        ref.append(q1, d1, x[i:i + 1], [i])
    assert np.array_equal(q, q1) and np.array_equal(d, d1)


@gpu
@pytest.mark.parametrize("headroom", [False, True])
@pytest.mark.parametrize("page,hd,f16", [(32, 128, False), (64, 256, True), (128, 512, False)])
def test_rows_appended_one_by_one_stay_within_the_bound(ctx, headroom, page, hd, f16):
    """Rising rows one call each, K and V: equal to the definition, and with headroom read
    back within the bound of the rows that went in."""
    import sgq
    n_kv = 2
    rng = np.random.default_rng(page)
    dt = np.float16 if f16 else np.float32
    x = [rising_rows(rng, page, n_kv, hd, r).astype(dt) for r in (1.005, 1.03)]
    pages = sgq.KvPages.empty(3, page, n_kv, hd)
    slots = i32(np.arange(page) + page)
    dev = [torch.from_numpy(t).cuda() for t in x]
    for i in range(page):
        ctx.kv_append_paged_q8(pages, dev[0][i:i + 1], dev[1][i:i + 1], slots[i:i + 1], headroom=headroom)
    back = torch.empty((2, page, n_kv, hd), device="cuda")
    ctx.kv_gather_paged_q8(pages, slots, back[0], back[1])
    kq, vq, ks, vs = from_pages(pages)
    for got, quants, scales, rows in zip(back.double().cpu().numpy(), (kq, vq), (ks, vs), x):
        q, d, _ = one_by_one(rows, 1.25 if headroom else 1.0)
        assert np.array_equal(quants[1], q[0]) and np.array_equal(scales[1], d[0])
        assert (quants[[0, 2]] == 0).all() and (scales[[0, 2]] == 0).all()
        if headroom:  # the value is rounded once more, by 2^-24 of 127 steps
            steps = steps_lost(page) + 127 * 2.0 ** -24
            assert (np.abs(got - rows.astype(np.float64)) <= steps * scales[1][None, :, None]).all()


@gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_headroom_of_runs(ctx, dtype):
    """Runs of several rows with headroom: blocks that begin anew, that stay, that grow by
    less and by more than a quarter, of subnormal scales, of scale 0 and NaN."""
    rng = np.random.default_rng(4)
    page, n_kv, hd = 32, 2, 128
    host = pool(rng, 9, n_kv, page, hd)
    size = [1.0, 0.5, 1.1, 3.0, 1.0, 1.0, 1.0, 0.0]
    for d in (host[2], host[3]):
        d[:] = 1 / 127
        d[4], d[5], d[6] = 1e-41, 0, np.nan
    host[0][5] = host[1][5] = 0
    x, slots = [], []
    for p, s in enumerate(size):
        first = 0 if p == 0 else 3
        slots.append(list(range(p * page + first, p * page + first + 5)))
        r = rng.uniform(-1, 1, (5, n_kv, hd))
        r[1, :, 7] = 1
        x.append((r * s).astype(dtype))
    pages = to_pages(*host)
    k = torch.from_numpy(np.concatenate(x)).cuda()
    ctx.kv_append_paged_q8(pages, k, k, i32(sum(slots, [])), headroom=True)
    for quants, scales, q, d in zip(from_pages(pages)[:2], from_pages(pages)[2:], host[:2], host[2:]):
        for r, s in zip(x, slots):
            if np.isnan(d[s[0] // page]).all():
                q[6][:, 3:8] = 0
                continue
            append_rows(q, d, r, s, 1.25)
        assert np.array_equal(scales, d, equal_nan=True) and np.array_equal(quants, q)


@pytest.mark.parametrize("act", [0x102, 0x200, 0x301, -0x100, -1])
def test_bad_append_flags_are_refused(act):
    import sgq
    L = sgq.lib()
    p = _pages_struct()
    pp = C.cast(C.byref(p), C.c_void_p)
    refused(L.sgq_kv_append_paged_q8(FAKE, pp, FAKE, 512, FAKE, 512, act, FAKE, 3), "activation type")
    # headroom is the append's alone
    refused(L.sgq_kv_gather_paged_q8(FAKE, pp, FAKE, 3, 0x100, FAKE, 512, FAKE, 512), "activation type")
    refused(L.sgq_attn_paged_q8(FAKE, pp, FAKE, 1024, 0x101, FAKE, 4, FAKE, FAKE, 2, 2, 8, 1, 99, 0, 0.1, FAKE,
                                1024, None, 0), "activation type")
