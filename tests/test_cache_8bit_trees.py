"""Drafted tokens over a cache held in 8 bits (HybridKVCache.tree_attention):
what a node sees is what the token sees when it is decoded alone, the values
code * scale in fp32, in models of every type. On the CPU the kernels are
computed in 64 bits, on a GPU by libnhs_hip.so. Tolerances are those of
test_rows_8bit, whose sums the fp32 tree attention's are: products and weights
in fp32 (it loses no 2^-17 of a weight), the output rounded once."""

import pytest
import torch

from nano_hisparse import row_kernels as rk
from nano_hisparse.hybrid import HotConfig
from nano_hisparse.selection import Selection
from test_cache_8bit import Provider8, cache_for, e4m3, f16, f32, i8, bf16
from test_cache_8bit import where  # noqa: F401
from test_rows_8bit import attend_oracle, check, keys, quantised

TREES = [[-1], [-1, 0, 0, 1, 1, 2, 5]]


def ancestors(parents, t):
    path = []
    while t >= 0:
        path.append(t)
        t = parents[t]
    return path[::-1]


@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("heads, kv, dim, P", [(4, 2, 8, 4), (8, 2, 64, 16), (4, 1, 128, 16)])
@pytest.mark.parametrize("pages", [0, 5])
def test_a_node_sees_what_its_token_sees_alone(where, dtype, heads, kv, dim, P, code, pages):  # noqa: F811
    """Every node of a tree, and its first token appended and decoded, against
    64-bit attention over one rounded history: few rows, whose values partly
    cancel, and many."""
    gen = torch.Generator().manual_seed(heads * dim + pages)
    n = pages * P + 2
    for parents in TREES:
        T = len(parents)
        cache = cache_for(where, 16, HotConfig(8 * P, 8 * P), code, dtype, P, kv, dim)
        cache.reserve("a", n + T, 1)
        k, v = keys(gen, n + T, kv, dim, dtype=dtype), keys(gen, n + T, kv, dim, dtype=dtype)
        q = (torch.randn(T, heads, dim, generator=gen) * 0.5).to(dtype)
        cache.write("a", 0, k[:n].to(where), v[:n].to(where))
        form = cache.storage.rows8
        history = torch.zeros(1, 2, n + T, form.row_bytes, dtype=torch.uint8)
        for plane, x in enumerate((k, v)):
            codes, scale = quantised(x, code)
            form.codes(history)[0, plane] = codes.to(code)
            form.scales(history)[0, plane] = scale
        paths = [ancestors(parents, t) for t in range(T)]
        mask = torch.tensor([sum(1 << j for j in path) for path in paths])
        selection = Selection.from_pages(list(range(-(-n // P))), n, P, heads)
        got = cache.tree_attention(q.to(where), k[n:].to(where), v[n:].to(where), mask.to(where), "a", 0, selection)
        assert got.dtype == dtype
        for t, path in enumerate(paths):
            rows = torch.tensor([list(range(n)) + [n + j for j in path]])
            check(got[t:t + 1], *attend_oracle(form, q[t:t + 1], history, rows))
        cache.write("a", 0, k[n:n + 1].to(where), v[n:n + 1].to(where))
        alone = cache.attention(q[0].to(where), "a", 0, Selection.from_pages(list(range(-(-(n + 1) // P))), n + 1, P, heads))
        check(alone[None], *attend_oracle(form, q[:1], history, torch.arange(n + 1)[None]))


def test_a_tree_has_the_cache_s_type(where):  # noqa: F811
    """As over rows that are not in 8 bits."""
    cache = cache_for(where, 16, HotConfig(32, 32), i8, bf16)
    cache.reserve("a", 8, 1)
    k = torch.ones(4, 2, 8, dtype=bf16, device=where)
    cache.write("a", 0, k, k)
    q, mask = torch.ones(4, 4, 8, dtype=bf16, device=where), torch.tensor([1, 3, 7, 15], device=where)
    selection = Selection.from_pages([0], 4, 4, 4)
    cache.tree_attention(q, k, k, mask, "a", 0, selection)
    for change in ((q.float(), k, k), (q, k.float(), k.float()), (q, k, k.half()), (q.float(), k.float(), k.float()),
                   (q.double(), k, k)):
        with pytest.raises(ValueError):
            cache.tree_attention(*change, mask, "a", 0, selection)
    cache.assert_invariants()
