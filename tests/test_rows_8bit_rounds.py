"""attend_8bit where a wave takes four tiles of rows in its only round: a split
of 513 to 1024 rows (768 or 1024 in whole steps of eight waves), heads of 32,
64 or 128 dims, 16-bit queries, or fp32 ones of less than 128 dims. Oracle and
tolerances are those of test_rows_8bit."""

import pytest
import torch

from nano_hisparse import row_kernels as rk
from test_rows_8bit import attend_case, attend_oracle, bf16, check, e4m3, f16, f32, i8

# 256 (request, KV head) pairs leave a list whole; the last ones are split: in two, and in 27 parts of 768 rows
SHAPES = [(8, 8, 128, 32, 513), (8, 8, 128, 32, 545), (8, 8, 128, 32, 769), (8, 8, 128, 32, 1000), (8, 8, 128, 32, 1024),
          (8, 8, 64, 33, 545), (8, 8, 64, 33, 1024), (8, 8, 32, 32, 513), (8, 8, 32, 32, 1000), (28, 4, 128, 64, 1024),
          (32, 8, 128, 16, 2048), (32, 8, 128, 16, 1500), (16, 8, 128, 1, 20000)]
KINDS = [(*shape, dtype, code) for shape in SHAPES for dtype, code in ((bf16, e4m3), (f16, i8))] \
    + [(*shape, f32, i8) for shape in SHAPES if shape[2] < 128]


def mask_some(rows, total, gen):
    """Requests with every row, some masked, none, the last one only, the second half only, some outside the pool."""
    N = rows.shape[-1]
    gone = torch.rand(rows.shape, generator=gen).to(rows.device)
    for b in range(len(rows)):
        kind = b % 6
        if kind == 1:
            rows[b] = torch.where(gone[b] < 0.3, -1, rows[b])
        elif kind == 2:
            rows[b] = -1
        elif kind == 3:
            rows[b, ..., : N - 1] = -1
        elif kind == 4:
            rows[b, ..., : N // 2] = -1
        elif kind == 5:
            rows[b] = torch.where(gone[b] < 0.5, total + b, rows[b])
    return rows


def hide(pool, rows, form):
    """NaN codes and scales in every row that no list names."""
    total = pool.shape[0] * pool.shape[2]
    named = torch.zeros(total, dtype=torch.bool, device=pool.device)
    named[rows[(rows >= 0) & (rows < total)]] = True
    dead = (~named).view(pool.shape[0], -1).nonzero()
    pool[dead[:, 0], :, dead[:, 1]] = 0xFF


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv, dim, B, N, dtype, code", KINDS)
def test_attend_four_tiles(gpu, heads, kv, dim, B, N, dtype, code):
    gen = torch.Generator().manual_seed(B + N)
    form, pool, rows, q = attend_case(gen, gpu, heads, kv, dim, code, dtype, B, N, 64)
    if B > 1:
        rows = mask_some(rows, pool.shape[0] * 64, gen)
    else:
        rows[0, torch.rand(N, generator=gen) < 0.3] = -1
    hide(pool, rows, form)
    got = rk.attend_8bit(q, pool, form, rows)
    some = list(range(min(B, 6))) + [B - 1]
    check(got[some], *attend_oracle(form, q[some], pool, rows[some]))
    if B > 2:
        assert not got[2].any()
    for _ in range(3):
        assert torch.equal(rk.attend_8bit(q, pool, form, rows), got)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv, dim, dtype, code", [(8, 4, 64, bf16, i8), (8, 2, 128, f16, e4m3), (8, 8, 32, f32, i8)])
def test_attend_four_tiles_of_a_list_per_head(gpu, heads, kv, dim, dtype, code):
    gen = torch.Generator().manual_seed(dim)
    B, N = 22, 900
    form, pool, rows, q = attend_case(gen, gpu, heads, kv, dim, code, dtype, B, N, 64)
    lists = torch.stack([rows[:, torch.randperm(N, generator=gen).to(gpu)] for _ in range(heads)], 1)
    lists[torch.rand(lists.shape, generator=gen).to(gpu) < 0.2] = -1
    lists = mask_some(lists, pool.shape[0] * 64, gen)
    hide(pool, lists, form)
    got = rk.attend_8bit(q, pool, form, lists)
    check(got[:6], *attend_oracle(form, q[:6], pool, lists[:6]))
    assert not got[2].any()
