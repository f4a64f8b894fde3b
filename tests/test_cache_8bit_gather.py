"""SparseDecodeBatch(form=): the rows that a step has to fetch from a host store
in 8 bits, counted and moved."""

import pytest
import torch

from nano_hisparse import row_kernels as rk
from nano_hisparse.batch_step import BatchTables, SparseDecodeBatch
from test_rows_8bit import attend_oracle, check, keys, quantised


@pytest.mark.gpu
@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("chunks", [1, 2])
def test_missed_rows_are_fetched(gpu, code, chunks):
    """A pool of which all but the resident pages holds NaN and no hot row yet:
    the first step misses every selected row that is not resident, a second
    one of the same queries none, and the output is the attention over the
    host's rows."""
    gen = torch.Generator().manual_seed(4)
    B, Hq, Hkv, D, P, n_pages, top, H = 3, 8, 2, 64, 16, 24, 4, 64
    form = rk.Rows8(code, Hkv, D)
    host = torch.zeros(B * n_pages, 2, P, form.row_bytes, dtype=torch.uint8)
    k = keys(gen, B * n_pages, P, Hkv, D)
    for plane, x in enumerate((k, keys(gen, B * n_pages, P, Hkv, D))):
        codes, scale = quantised(x, code)
        form.codes(host)[:, plane] = codes.to(code)
        form.scales(host)[:, plane] = scale
    host = host.pin_memory()
    blocks, held = H // P + 3, (0, n_pages - 2, n_pages - 1)
    pool = torch.full((B * blocks, 2, P, form.row_bytes), 0xFF, dtype=torch.uint8)
    resident = torch.full((B, n_pages), -1, dtype=torch.int32)
    hot = torch.empty(B, H // P, dtype=torch.int32)
    for b in range(B):
        base = b * blocks
        hot[b] = torch.arange(base, base + H // P, dtype=torch.int32)
        for i, page in enumerate(held):
            resident[b, page] = base + H // P + i
            pool[base + H // P + i] = host[b * n_pages + page]
    pool = pool.to(gpu)
    low, high = (t.view(B, n_pages, Hkv, D).to(torch.bfloat16).to(gpu) for t in (k.amin(1), k.amax(1)))
    tables = BatchTables(
        source=torch.arange(B * n_pages, dtype=torch.int32).view(B, n_pages).to(gpu), resident=resident.to(gpu),
        hot=hot.to(gpu), tags=torch.full((B, H), -1, dtype=torch.int32, device=gpu),
        lru=torch.arange(H, device=gpu).repeat(B, 1).contiguous(), minimum=low, maximum=high,
        lengths=torch.full((B,), n_pages * P, device=gpu))
    step = SparseDecodeBatch(pool, host, tables, P, top, chunks=chunks, form=form)
    q = torch.randn(B, Hq, D, generator=gen).to(torch.bfloat16)
    for again in (False, True):
        out, result = step.step(q.to(gpu))
        torch.cuda.synchronize()
        rows, at = result.positions.cpu().long(), result.physical.cpu()
        selected = rows >= 0
        missed = selected & ~torch.isin(rows // P, torch.tensor(held))
        assert bool(missed.any(1).all()) and bool(((at >= 0) == selected).all())
        counts = result.counts.cpu()
        assert torch.equal(counts[:, 0], (selected & ~missed).sum(1))
        assert torch.equal(counts[:, 1 if again else 2], missed.sum(1)) and not counts[:, 2 if again else 1].any()
        flat = torch.where(selected, rows + torch.arange(B)[:, None] * n_pages * P, -1)
        assert torch.equal(pool.cpu()[at[selected] // P, :, at[selected] % P],
                           host[flat[selected] // P, :, flat[selected] % P])
        check(out, *attend_oracle(form, q, host, flat))
