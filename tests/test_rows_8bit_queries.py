"""attend_8bit of queries that are not finite: the score of every row is then an
infinity or NaN, and a softmax over such scores NaN, also where all of them
are minus infinity. A head whose list holds no row yields zeros all the same."""

import math

import pytest
import torch

from nano_hisparse import row_kernels as rk
from test_rows_8bit import attend_case, attend_oracle, bf16, check, e4m3, f16, f32, i8


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("heads, kv, dim", [(8, 2, 128), (4, 2, 64), (4, 2, 32), (4, 1, 256), (6, 2, 80), (6, 2, 72), (2, 1, 300)])
def test_queries_with_infinities(gpu, heads, kv, dim, dtype, code):
    """One dimension of every key is negative, and the query +inf there, so
    that every score is minus infinity; other heads hold the other sign, NaN,
    both signs, or are finite."""
    gen = torch.Generator().manual_seed(dim)
    for N in (1, 33, 300, 1030):
        form, pool, rows, q = attend_case(gen, gpu, heads, kv, dim, code, dtype, 3, N)
        form.codes(pool)[:, 0, ..., 5] = torch.full((), -3.0, device=gpu).to(code)
        q[:, 0, 5] = math.inf
        q[0, 1, 5] = -math.inf
        q[1, 1, 7] = math.nan
        q[2, 1, 5], q[2, 1, 9] = math.inf, -math.inf
        rows[2, ::2] = -1
        got = rk.attend_8bit(q, pool, form, rows)
        empty = not (rows[2] >= 0).any()
        for b in range(3):
            for h in (0, 1):
                assert bool(got[b, h].isnan().all()) if not (b == 2 and empty) else not got[b, h].any(), (N, b, h)
        if heads > 2:
            check(got[:, 2:], *(t[:, 2:] for t in attend_oracle(form, torch.where(q.isfinite(), q, 0.0), pool, rows)))
        rows[1] = -1
        assert not rk.attend_8bit(q, pool, form, rows)[1].any()
