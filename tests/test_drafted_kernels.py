"""The drafted-token operators where their tests at small sizes do not reach:
outputs that a call must not take."""

import pytest
import torch

from nano_hisparse import row_kernels as rk
from test_drafted_tokens import check_tree, f16, f32, norm_case, run_tree, tree_case


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_outputs_that_hold_an_element_twice_are_refused(gpu, native, monkeypatch):
    """Rows or heads that overlap would be written by several workgroups in any order."""
    if not native:
        class PythonOnly:
            def __getattr__(self, name):
                return lambda *a: None

        monkeypatch.setattr(rk, "_launch", PythonOnly())
    B, T, H, D = 2, 3, 4, 64
    c = tree_case(gpu, f16, B, T, H, 2, D, 16, 20)
    memory = torch.zeros(B * T * H * D * 2, dtype=f16, device=gpu)
    for strides in ((0, H * D, D, 1), (T * H * D, H * D - 1, D, 1), (T * H * D, H * D, D - 1, 1), (1, H * D, D, 1),
                    (T * H * D, D, D, 1), (2 * H * D, H * D, D, 1), (T * H * D, H * D, D // 2, 1)):
        with pytest.raises(ValueError, match="distinct"):
            run_tree(c, out=memory.as_strided((B, T, H, D), strides))
    with pytest.raises(ValueError, match="contiguous"):
        run_tree(c, out=memory.as_strided((B, T, H, D), (2 * T * H * D, 2 * H * D, 2 * D, 2)))
    for strides in ((T * H * D, H * D, D, 1), (D, B * D, T * B * D, 1), (T * H * D + 5, H * D + 1, D, 1),
                    (H * D, B * H * D, D, 1), (D, H * B * D, B * D, 1)):
        out = memory.as_strided((B, T, H, D), strides)
        assert run_tree(c, out=out) is out
        check_tree(c, out)
    n = norm_case(gpu, f32, 5, 2, 2, 32, f32, 9)
    args = n["q"], n["k"], n["qw"], n["kw"], 1e-6, n["cos"], n["sin"], n["at"]
    x, y = torch.zeros(5, 2, 32, device=gpu), torch.zeros(5, 2, 32, device=gpu)
    for bad in ((x, x), (x.as_strided((5, 2, 32), (32, 32, 1)), y), (x, y.as_strided((5, 2, 32), (64, 16, 1)))):
        with pytest.raises(ValueError, match="distinct"):
            rk.qk_norm_rope(*args, out=bad)
    both = torch.zeros(5, 4, 32, device=gpu)
    got, expected = rk.qk_norm_rope(*args, out=(both[:, ::2], both[:, 1::2])), rk.qk_norm_rope(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, expected))
