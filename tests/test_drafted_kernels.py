"""The drafted-token operators where their tests at small sizes do not reach:
outputs that a call must not take, histories of many rounds and stages of the
attention's row loop, prompts of many rows. Tolerances are those of
test_drafted_tokens.py, evaluated on the GPU in 64 bits."""

import math

import pytest
import torch

from nano_hisparse import _hip
from nano_hisparse import row_kernels as rk
from test_drafted_tokens import (HALF, U, bf16, check, check_norm, check_tree, f16, f32, norm_case, plan_oracle,
                                 random_parents, run_tree, seen_nodes, tree_case, tree_oracle)


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


# ---- long histories ------------------------------------------------------------------------------

ROUND, STAGE = 128, 2048  # most keys of a round of the row loop, and rows whose addresses it has at a time


def rows_of_a_split(B, T, N, Hq, Hkv, D):
    """At least so many rows has some split: the workspace holds D + 2 numbers per split and output row, for the most
    splits that any kernel makes of the shape."""
    need = _hip.load().nhs_tree_attention_workspace_bytes(B, T, N, Hq, Hkv, D)
    return N / max(need // (B * T * Hq * (D + 2) * 4), 1)


def long_case(gpu, dtype, B, T, Hq, Hkv, D, N, seed):
    """Requests over one pool whose keys grow with their position: row lists
    in random order, with masked stretches, with one row left, rising (the
    largest scores come last) and falling."""
    P = 16
    g = torch.Generator(device=gpu).manual_seed(seed)
    blocks = N // P + 5
    pool = rk.padded_pool(blocks, P, Hkv, D, dtype, gpu)
    pool.copy_(torch.randn(pool.shape, generator=g, device=gpu))
    grown = 0.2 + 2.8 * torch.arange(blocks * P, device=gpu).view(blocks, P, 1, 1) / (blocks * P)
    pool[:, 0] = (pool[:, 0].float() * grown).to(dtype)
    rows = torch.rand(B, blocks * P, generator=g, device=gpu).argsort(1)[:, :N].clone()
    rows[3], rows[4] = rows[3].sort().values, rows[4].sort(descending=True).values
    rows[torch.rand(B, N, generator=g, device=gpu) < 0.1] = -1
    rows[1, 100:700] = -1
    rows[2, : N - 1] = -1
    x = torch.randn(B, T, (Hq + 2 * Hkv) * D, generator=g, device=gpu).to(dtype)
    q, k, v = x.split([Hq * D, Hkv * D, Hkv * D], 2)
    mask, _ = plan_oracle(random_parents(B, T, torch.Generator().manual_seed(seed)), torch.zeros(B, dtype=torch.int64))
    return dict(q=q.view(B, T, Hq, D), pool=pool, rows=rows, k=k.view(B, T, Hkv, D), v=v.view(B, T, Hkv, D),
                mask=mask.to(gpu), page=P)


def check_requests(c, got, requests):
    q, pool, P = c["q"], c["pool"], c["page"]
    _, T, Hq, D = q.shape
    Hkv, half = pool.shape[3], HALF[q.dtype]
    g = Hq // Hkv
    for b in requests:
        at = c["rows"][b][c["rows"][b] >= 0]
        keys, values = (torch.cat((pool[at // P, i, at % P], c[n][b])).double() for i, n in ((0, "k"), (1, "v")))
        words = c["mask"][b].cpu()
        seen = (seen_nodes(words) & (words != 0)).to(q.device)
        seen = torch.cat((torch.ones(T, len(at), dtype=torch.bool, device=q.device), seen), 1).repeat_interleave(g, 0)
        out = torch.empty(T, Hq, D, dtype=torch.float64, device=q.device)
        tol = torch.empty_like(out)
        for kv in range(Hkv):
            heads = slice(kv * g, (kv + 1) * g)
            qh, kh, vh = q[b, :, heads].reshape(T * g, D).double(), keys[:, kv], values[:, kv].contiguous()
            s = torch.mm(qh, kh.t().contiguous()) / math.sqrt(D)
            size = torch.mm(qh.abs(), kh.abs().t().contiguous()) / math.sqrt(D)
            w = s.masked_fill(~seen, -math.inf).softmax(1)
            o = torch.mm(w, vh)
            s_err = 2 * (D + 4) * U * (size * seen).amax(1) + 2 * U * (s.abs() * seen).amax(1)
            w_err = 2 * s_err + 2.0 ** -22 + (half if q.dtype != f32 else 0.0)
            rel = 2 * w_err + 2 * (seen.sum(1) + 64) * U
            bound = rel[:, None] * torch.mm(w, vh.abs()) + half * o.abs() + 1e-30 + (2.0 ** -25 if q.dtype == f16 else 0)
            out[:, heads], tol[:, heads] = o.view(T, g, D), bound.view(T, g, D)
        absent = (words == 0).to(q.device)
        out[absent] = 0.0
        check(got[b], out.cpu(), tol.cpu())


KERNELS = [  # dtype, D, nodes, query heads per KV head: every size of workgroup, of each row length
    (bf16, 64, 8, 4), (f16, 32, 5, 4), (f32, 32, 3, 2),  # up to 32 query rows of up to 128 bytes
    (bf16, 128, 8, 4), (f16, 64, 16, 4), (bf16, 256, 7, 2), (f16, 256, 33, 4), (f32, 64, 9, 4), (f32, 128, 3, 4),
    (bf16, 128, 20, 4), (f32, 128, 30, 4), (f16, 64, 64, 4), (f32, 32, 40, 2), (bf16, 32, 64, 2),
    (bf16, 128, 64, 4), (f16, 128, 33, 7),  # blocks of 256 query rows
    (bf16, 128, 1, 1), (f32, 64, 1, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,T,g", KERNELS)
@pytest.mark.parametrize("N", [300, 640, 2049, 4500])
def test_tree_attention_of_many_rounds(gpu, dtype, D, T, g, N):
    """Enough requests that a workgroup has whole histories: three rounds and more, and more than one stage of rows."""
    print("case:", dict(dtype=dtype, D=D, T=T, g=g, N=N), flush=True)
    B, Hkv = 32, 8
    rows = rows_of_a_split(B, T, N, g * Hkv, Hkv, D)
    assert rows > ROUND and (N < 4500 or rows > STAGE)
    c = long_case(gpu, dtype, B, T, g * Hkv, Hkv, D, N, seed=N + D + T)
    check_requests(c, run_tree(c), (0, 1, 2, 3, 4, B - 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,T,g", [(bf16, 128, 8, 4), (f16, 64, 3, 2), (f32, 32, 40, 2), (bf16, 128, 64, 2),
                                         (f16, 256, 5, 4), (f32, 128, 2, 1)])
def test_tree_attention_of_splits_of_several_stages(gpu, dtype, D, T, g):
    print("case:", dict(dtype=dtype, D=D, T=T, g=g), flush=True)
    B, Hkv, N = 8, 8, 24001
    rows = rows_of_a_split(B, T, N, g * Hkv, Hkv, D)
    assert STAGE < rows <= N / 2
    c = long_case(gpu, dtype, B, T, g * Hkv, Hkv, D, N, seed=D + T)
    check_requests(c, run_tree(c), (0, 1, 2, 3, 4, B - 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,T,g", [(bf16, 128, 8, 4), (f16, 64, 7, 4), (bf16, 32, 30, 2), (f16, 128, 33, 7),
                                         (bf16, 256, 5, 2), (f16, 64, 64, 4), (bf16, 128, 20, 4)])
def test_weights_of_sixteen_bit_heads_keep_their_rests(gpu, dtype, D, T, g):
    """Outputs are the exact ones, rounded once. The exact values' neighbours
    would be taken for a third of them if the weights were rounded to the type
    (each off by up to 2^-9 relative in bf16 and independent of the others, so
    an output by about as much, where its steps are 2^-8 to 2^-7 of it; fp16
    likewise); with the rests of that rounding, rounded themselves, an output
    is off by some 2^-17 (2^-20 in fp16, whose scores and sums are what is
    left), which takes the neighbour for less than one in a hundred."""
    print("case:", dict(dtype=dtype, D=D, T=T, g=g), flush=True)
    B, Hkv, N, P = 4, 4, 1500, 16
    c = tree_case(gpu, dtype, B, T, g * Hkv, Hkv, D, P, N, seed=D + T, spread=0.5)
    got = run_tree(c)
    differ = total = 0
    for b in range(B):
        at = c["rows"][b][c["rows"][b] >= 0]
        for t in range(T):
            word = int(c["mask"][b, t])
            nodes = [j for j in range(T) if word >> j & 1]
            keys, values = (torch.cat((c["pool"][at // P, i, at % P], c[n][b, nodes])).double().repeat_interleave(g, 1)
                            for i, n in ((0, "k"), (1, "v")))
            w = ((c["q"][b, t].double() * keys).sum(-1) / math.sqrt(D)).softmax(0)
            exact = (w[..., None] * values).sum(0) if word else torch.zeros_like(got[b, t])
            differ += (got[b, t] != exact.to(dtype)).sum().item()
            total += exact.numel()
    assert differ <= 0.02 * total, f"{differ} of {total}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(f16, 32), (f16, 64), (f16, 128), (f16, 256), (bf16, 128), (f32, 64), (f16, 48)])
@pytest.mark.parametrize("power", [18, 21])
@pytest.mark.parametrize("B,N", [(1, 8000), (40, 1200)])
def test_many_small_weights_add_up(gpu, dtype, D, power, B, N):
    """One key with all but a little of the weight, thousands with exp(-18) or
    exp(-21) of it each (below fp16's numbers) and the only values that are not
    0. fp16 weights are multiples of 2^-39 of the largest, half of which per key
    comes to the tolerance."""
    print("case:", dict(dtype=dtype, D=D, power=power, B=B, N=N), flush=True)
    c = tree_case(gpu, dtype, B, 2, 4, 2, D, 16, N, seed=D, fused=False)
    for x in (c["q"], c["k"], c["pool"]):
        x.zero_()
    c["q"][..., 0] = 8.0
    c["k"][:, 0, :, 0] = round(power * math.sqrt(D)) / 8
    c["v"].zero_()
    c["pool"][:, 1] = 1024.0
    c["pool"][:, 1, :, :, 1::2] = -512.0
    c["mask"].copy_(torch.tensor([[1, 3]], device=gpu).expand(B, 2))
    some = dict(c, **{n: c[n][-1:] for n in ("q", "rows", "k", "v", "mask")})
    expected, tol = tree_oracle(*(some[n] for n in ("q", "pool", "rows", "k", "v", "mask", "page")), False)
    assert expected.abs().min() > 2.0 ** -13  # (a number in every type)
    if dtype == f16:
        tol += 2.0 ** -40 * N * 1024.0
    check(run_tree(c)[-1:], expected, tol)


# ---- long prompts --------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,table", [(bf16, bf16), (f16, f32), (f32, f32)])
@pytest.mark.parametrize("n,Hq,Hkv,D", [(41001, 2, 1, 16), (13700, 60, 10, 32), (41000, 14, 2, 64), (8200, 32, 8, 128),
                                        (8300, 15, 2, 256), (1500, 30, 1, 1024)])
def test_qk_norm_rope_of_long_prompts(gpu, dtype, table, n, Hq, Hkv, D):
    """From 40960 rounds of heads on, a wave takes two: the same as the call
    over parts of the rows, and right at the ends and some rows between."""
    print("case:", dict(dtype=dtype, table=table, n=n, Hq=Hq, Hkv=Hkv, D=D), flush=True)
    groups = 64 // max(D // 16, 1)
    rounds = -(-(Hq + Hkv) // groups)
    assert n * rounds >= 40960 and D // 16 <= 64
    c = norm_case(gpu, dtype, n, Hq, Hkv, D, table, 4000, seed=n)
    q, k, args = c["q"], c["k"], (c["qw"], c["kw"], 1e-6, c["cos"], c["sin"])
    got = rk.qk_norm_rope(q, k, *args, c["at"])
    step = 40959 // rounds
    for at in range(0, n, step):
        some = slice(at, at + step)
        for a, b in zip(got, rk.qk_norm_rope(q[some], k[some], *args, c["at"][some])):
            assert torch.equal(a[some], b)
    rows = torch.cat((torch.arange(3), torch.randperm(n)[:200], torch.arange(n - 3, n))).to(gpu)
    few = dict(c, q=q[rows], k=k[rows])
    check_norm(few, [x[rows] for x in got], c["at"][rows])
    done = rk.qk_norm_rope(q, k, *args, c["at"], out=(q, k))  # in place, in one projection's rows
    assert done[0].data_ptr() == q.data_ptr() and all(torch.equal(a, b) for a, b in zip(done, got))
