"""SparseDecodeBatch(form=) refuses pools and host stores that are not of the
form, and page sizes that are not theirs: the gather would move bytes between
other places than the attention reads."""

import pytest
import torch

from nano_hisparse import row_kernels as rk
from nano_hisparse.batch_step import BatchTables, SparseDecodeBatch


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_a_step_refuses_other_forms(device):
    form, P = rk.Rows8(torch.int8, 2, 64), 16
    pool = torch.zeros(6, 2, P, form.row_bytes, dtype=torch.uint8, device=device)
    host = torch.zeros(4, 2, P, form.row_bytes, dtype=torch.uint8)
    tables = BatchTables(*(torch.zeros(1, 4, device=device) for _ in BatchTables.__dataclass_fields__))

    def refused(match="8 bits|pool", pool=pool, host=host, page_size=P, form=form):
        with pytest.raises(ValueError, match=match):
            SparseDecodeBatch(pool, host, tables, page_size, 2, form=form)

    refused(page_size=32)
    refused(host=host[:, :, :8])
    refused(host=host[:, :, ::2])
    refused(host=torch.zeros(4, 2, 8, 2 * form.row_bytes, dtype=torch.uint8))
    refused(host=host.view(torch.int8))
    refused(pool=pool[..., : form.row_bytes - 16])
    refused(pool=pool.view(torch.int8))
    refused(pool=torch.zeros(6, 2, P, 2, 64, device=device))
    refused(form=rk.Rows8(torch.int8, 4, 64))
    refused(form=rk.Rows8(torch.uint8, 2, 64))
    refused(form=None)  # rows in 8 bits without their form
    if device == "cpu":
        refused("runs on a GPU")
    else:
        SparseDecodeBatch(pool, host.pin_memory(), tables, P, 2, form=form)
