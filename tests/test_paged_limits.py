"""The paged 8-bit KV cache at the ends of what its entry points accept: scores of
any finite size, K and V blocks far apart, many query heads a kv head, blocks that
grow again and again, pools that run out.  Plain forms are those of
tests/_paged.py."""
import ctypes as C

import numpy as np
import pytest
import torch

import _paged as ref
from test_paged import FAKE, _pages_struct, attend, batch, from_pages, i32, refused, to_pages

gpu = pytest.mark.gpu


# ---- attention ----------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("k_scale", [1e4, 1e7, 1e12, 1e28])
def test_attention_of_scores_of_any_size(ctx, f16, new, sign, k_scale):
    """Scores of 10^6 to 10^31, all of one sign: one key is at least a quarter ahead of
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
