"""The operators that verify drafted tokens (tree_plan, tree_attention,
qk_norm_rope, token_logprobs) against their formulas in 64 bits, at the sizes
and masks where they can go wrong.

Tolerances, with u = 2^-24 (half a step of fp32) and r = half a step of the
output's type relative to the value:

- attention: a score is a sum of D products, off by 2 (D + 4) u sum|q k| D^-1/2
  at most (twice u: a matrix core need not round to nearest); a weight's
  relative error is that of its score and of its maximum's, plus 2^-22 for
  exp2 and the rounding of its argument (2 u |score|), and r once more where
  the weights are rounded to the type for the matrix cores; numerator and
  denominator take N + T terms, u each. Both enter the output times
  sum w |V|, and its own rounding is r |out|.
- log probabilities: x - m is rounded once (u |x - m|), a term of S by
  2^-22 + 2 u |x - m| relative, S over at most V / 64 + 64 additions in a
  row; ln adds 2 u |ln S|.
- norm and rotation: the mean over D / 2 + 8 roundings, the products three
  more; a rotated element has the error of both its terms.
"""

import math

import pytest
import torch

from nano_hisparse import _hip
from nano_hisparse import row_kernels as rk

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (bf16, f16, f32)}


# ---- oracles -------------------------------------------------------------------------------


def plan_oracle(parents, lengths):
    masks, positions = [], []
    for tree, length in zip(parents.tolist(), lengths.tolist()):
        paths = []
        for t, p in enumerate(tree):
            if p == -1:
                paths.append([t])
            elif 0 <= p < t and paths[p]:
                paths.append(paths[p] + [t])
            else:
                paths.append([])
        words = [sum(1 << j for j in path) for path in paths]
        masks.append([w - (1 << 64) if w >> 63 else w for w in words])
        positions.append([length + len(path) - 1 if path else 0 for path in paths])
    return torch.tensor(masks), torch.tensor(positions)


def seen_nodes(mask):
    """bool [..., T]: the bits of the words."""
    return ((mask[..., None] >> torch.arange(mask.shape[-1])) & 1).bool()


def tree_oracle(q, pool, rows, k, v, mask, page, rounded):
    """(out, tolerance) in float64 on the CPU; `rounded`: the weights' own
    rounding is allowed for."""
    dtype = q.dtype
    q, k, v, mask, rows = (t.cpu() for t in (q, k, v, mask, rows))
    B, T, Hq, D = q.shape
    Hkv = pool.shape[3]
    g = Hq // Hkv
    total = pool.shape[0] * page
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        r = rows[b][(rows[b] >= 0) & (rows[b] < total)]
        at = r.to(pool.device)
        past_k, past_v = (pool[at // page, i, at % page].cpu().double() for i in (0, 1))
        for t in range(T):
            if mask[b, t] == 0:
                continue
            seen = seen_nodes(mask[b])[t] & (mask[b] != 0)  # an absent node is no one's ancestor
            keys = torch.cat((past_k, k[b, seen].double()))
            values = torch.cat((past_v, v[b, seen].double()))
            keys, values = (x.repeat_interleave(g, 1) for x in (keys, values))
            qt = q[b, t].double()
            s = (qt * keys).sum(-1) / math.sqrt(D)  # [n, Hq]
            w = torch.softmax(s, 0)
            out[b, t] = (w[..., None] * values).sum(0)
            s_err = 2 * (D + 4) * U * ((qt * keys).abs().sum(-1) / math.sqrt(D)).amax(0) + 2 * U * s.abs().amax(0)
            w_err = 2 * s_err + 2.0 ** -22 + (HALF[dtype] if rounded else 0.0)
            rel = 2 * w_err + 2 * (len(keys) + 64) * U
            tol[b, t] = rel[:, None] * (w[..., None] * values.abs()).sum(0) + HALF[dtype] * out[b, t].abs() + 1e-30
    if dtype == f16:
        tol += 2.0 ** -25  # half a step of the subnormals
    return out, tol


def check(got, expected, tol):
    got = got.detach().cpu().double()
    assert got.shape == expected.shape
    same = (got == expected) | (got.isnan() & expected.isnan())
    worst = torch.where(same, 0.0, (got - expected).abs() / tol)
    assert not worst.isnan().any(), "a NaN on one side only"
    assert worst.max().item() <= 1.0 if worst.numel() else True, f"{worst.max().item():.3g} times the tolerance"


def norm_oracle(q, k, qw, kw, eps, cos, sin, positions):
    at = torch.arange(len(q)) if positions is None else positions.cpu().clamp(0, len(cos) - 1)
    c, s = cos.cpu().double()[at][:, None], sin.cpu().double()[at][:, None]
    results = []
    for x, w in ((q, qw), (k, kw)):
        x, w, D = x.cpu().double(), w.cpu().double(), x.shape[-1]
        y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
        lo, hi = y[..., : D // 2], y[..., D // 2:]
        out = torch.cat((lo * c - hi * s, hi * c + lo * s), -1)
        size = torch.cat((lo.abs() * c.abs() + hi.abs() * s.abs(), hi.abs() * c.abs() + lo.abs() * s.abs()), -1)
        tol = (D / 2 + 16) * U * size + HALF[q.dtype] * out.abs() + 1e-30
        results.append((out, tol + 2.0 ** -25 if q.dtype == f16 else tol))
    return results


def logprob_oracle(logits, tokens, top):
    x = logits.cpu().double()
    R, V = x.shape
    m = x.amax(1, keepdim=True)
    log_s = (x - m).exp().sum(1, keepdim=True).log()
    logs = ((x - m) - log_s).float().double()  # differences beyond fp32's range are -inf
    p = logs.exp()
    entropy = -torch.where(p > 0, p * logs, 0.0).sum(1)
    none = torch.isnan(m) | torch.isinf(m)
    logs, entropy = torch.where(none, math.nan, logs), torch.where(none[:, 0], math.nan, entropy)
    tol = U * (4 * (x - m).abs().clamp(max=1e39) + 4 * log_s.abs() + V / 64 + 64)
    tok = tokens.cpu().view(R, -1)
    known = (tok >= 0) & (tok < V)
    at = tok.clamp(0, V - 1)
    chosen = torch.where(known, logs.gather(1, at), torch.where(none, math.nan, -math.inf))
    # a NaN above every number (as torch sorts), equal logits by index, -0 equal to +0
    ids = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    return {"logprobs": (chosen.view(tokens.shape), tol.gather(1, at).view(tokens.shape)),
            "entropy": (entropy, U * (V / 64 + 64) * (4 + 2 * entropy.nan_to_num())), "ids": ids,
            "values": (logs.gather(1, ids), tol.gather(1, ids))}


# ---- inputs --------------------------------------------------------------------------------


def random_parents(B, T, gen, absent=True):
    parents = torch.full((B, T), -1, dtype=torch.int32)
    for t in range(1, T):
        parents[:, t] = torch.randint(-1, t, (B,), generator=gen).int()
    if absent:
        for b in range(1, B):
            parents[b, T - (b * T) // (2 * B):] = -2
    return parents


def tree_case(gpu, dtype, B, T, Hq, Hkv, D, P, N, seed=0, spread=1.0, fused=True, blocks=None):
    g = torch.Generator().manual_seed(seed)
    blocks = blocks or (N // P + 3) * 2
    pool = rk.padded_pool(blocks, P, Hkv, D, dtype, gpu)
    pool.copy_(torch.randn(pool.shape, generator=g) * spread)
    rows = torch.stack([torch.randperm(blocks * P, generator=g)[:N] for _ in range(B)]).view(B, N)
    rows[torch.rand(B, N, generator=g) < 0.1] = -1
    x = (torch.randn(B, T, (Hq + 2 * Hkv) * D, generator=g) * spread).to(dtype).to(gpu)
    q, k, v = x.split([Hq * D, Hkv * D, Hkv * D], 2)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    mask, _ = plan_oracle(random_parents(B, T, g), torch.zeros(B, dtype=torch.int64))
    return dict(q=q.view(B, T, Hq, D), pool=pool, rows=rows.to(gpu), k=k.view(B, T, Hkv, D), v=v.view(B, T, Hkv, D),
                mask=mask.to(gpu), page=P)


def run_tree(c, **kw):
    return rk.tree_attention(c["q"], c["pool"], c["rows"], c["k"], c["v"], c["mask"], c["page"], **kw)


def check_tree(c, got):
    out, tol = tree_oracle(c["q"], c["pool"], c["rows"], c["k"], c["v"], c["mask"], c["page"], c["q"].dtype != f32)
    check(got, out, tol)


# ---- refusals (no GPU) -------------------------------------------------------------------------


def test_cpu_tensors_are_refused():
    z = torch.zeros
    with pytest.raises(ValueError, match="must be on a GPU"):
        rk.tree_plan(z(1, 2, dtype=torch.int32), z(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="must be on a GPU"):
        rk.tree_attention(z(1, 1, 2, 8), z(2, 2, 4, 1, 8), z(1, 3, dtype=torch.int64), z(1, 1, 1, 8), z(1, 1, 1, 8),
                          z(1, 1, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="must be on a GPU"):
        rk.qk_norm_rope(z(1, 2, 8), z(1, 1, 8), z(8), z(8), 1e-6, z(1, 4), z(1, 4))
    with pytest.raises(ValueError, match="must be on a GPU"):
        rk.token_logprobs(z(1, 8), z(1, dtype=torch.int64))


@pytest.fixture(scope="module")
def lib(native_launchers):
    return _hip.load()


def attention_status(lib, **change):
    """nhs_tree_attention's status for a call that never reaches a launch."""
    a = dict(q=256, k=256, v=256, mask=256, dtype=1, pool=256, pool_rows=64, block=0, rows=256, batch=1, nodes=4,
             n_rows=8, q_heads=4, kv_heads=2, head_dim=64, page=16, out=256, ws=0, ws_bytes=0)
    a.update(change)
    return lib.nhs_tree_attention(
        a["q"], 0, 0, 0, a["k"], 0, 0, 0, a["v"], 0, 0, 0, a["mask"], 0, a["dtype"], a["pool"], a["pool_rows"],
        a["block"], a["rows"], 0, 1, a["batch"], a["nodes"], a["n_rows"], a["q_heads"], a["kv_heads"], a["head_dim"],
        a["page"], a["out"], 0, 0, 0, a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("change,status", [
    (dict(nodes=65), -1), (dict(nodes=0), -1), (dict(batch=-1), -1), (dict(n_rows=-1), -1), (dict(kv_heads=3), -1),
    (dict(n_rows=(1 << 30) + 1), -1), (dict(head_dim=0), -1), (dict(page=0), -1), (dict(dtype=3), -1), (dict(q=0), -1), (dict(k=0), -1), (dict(v=0), -1),
    (dict(mask=0), -1), (dict(out=0), -1), (dict(pool=0), -1), (dict(rows=0), -1), (dict(q=257), -1),
    (dict(mask=260), -1), (dict(pool_rows=-1), -1), (dict(block=16), -1), (dict(head_dim=258), -2),
    (dict(pool_rows=1 << 31), -2), (dict(n_rows=100000), -3), (dict(n_rows=100000, ws=256, ws_bytes=64), -3),
    (dict(batch=0), 0),
])
def test_tree_attention_refuses(lib, change, status):
    assert attention_status(lib, **change) == status


@pytest.mark.parametrize("args,status", [
    ((0, 4, 256, 4, 256, 256, 256, None), 0), ((1, 0, 256, 4, 256, 256, 256, None), -1),
    ((-1, 4, 256, 4, 256, 256, 256, None), -1), ((1, 65, 256, 65, 256, 256, 256, None), -2),
    ((1, 4, None, 4, 256, 256, 256, None), -1), ((1, 4, 256, 4, 256, None, 256, None), -1),
    ((1 << 26, 4, 256, 4, 256, 256, 256, None), -2),
])
def test_tree_plan_refuses(lib, args, status):
    assert lib.nhs_tree_plan(*args) == status


def test_qk_norm_rope_refuses(lib):
    def status(rows=2, q_heads=4, k_heads=2, dim=64, dtype=1, q=256, w=256, cos=256, table=1, table_rows=2,
               positions=None, out=256):
        return lib.nhs_qk_norm_rope(rows, q_heads, k_heads, dim, dtype, q, 0, 0, 256, 0, 0, w, 256, 1e-6, cos, 256,
                                    table, table_rows, positions, out, 0, 0, 256, 0, 0, None)

    assert status(rows=0) == 0
    for bad in (dict(rows=-1), dict(q_heads=0), dict(k_heads=0), dict(dim=63), dict(dim=0), dict(dtype=5),
                dict(table=2), dict(q=None), dict(w=None), dict(cos=None), dict(out=None), dict(table_rows=1),
                dict(table_rows=0, positions=256), dict(q=257), dict(positions=260)):
        assert status(**bad) == -1, bad
    for dim in (64, 66):  # more heads than a launch has waves
        assert status(rows=1 << 26, positions=256, dim=dim, q_heads=62) == -2


def test_token_logprobs_refuses(lib):
    def status(logits=256, dtype=0, rows=2, vocab=100, tokens=256, per_row=1, top=5, ids=256, entropy=256):
        return lib.nhs_token_logprobs(logits, vocab, dtype, rows, vocab, tokens, per_row, per_row, top, 256, entropy,
                                      ids, 256, 256, 1 << 30, None)

    assert status(rows=0) == 0
    assert status(top=65) == -2 and status(vocab=(1 << 30) + 1) == -2 and status(rows=1 << 24) == -2
    for bad in (dict(rows=-1), dict(vocab=0, top=0), dict(top=-1), dict(top=6, vocab=5), dict(dtype=4),
                dict(logits=None), dict(tokens=None), dict(ids=None), dict(entropy=None), dict(logits=258),
                dict(tokens=260), dict(per_row=-1)):
        assert status(**bad) == -1, bad


@pytest.mark.gpu
def test_bad_arguments_raise(gpu):
    c = tree_case(gpu, f16, 2, 3, 4, 2, 64, 16, 20)

    def call(**kw):
        d = dict(c, **kw)
        return rk.tree_attention(d["q"], d["pool"], d["rows"], d["k"], d["v"], d["mask"], d["page"], d.get("out"))

    for bad in (dict(q=c["q"][0]), dict(q=c["q"].float()), dict(k=c["k"][:1]), dict(v=c["v"].float()),
                dict(rows=c["rows"].int()), dict(rows=c["rows"][:1]), dict(mask=c["mask"].int()),
                dict(mask=c["mask"][:, :2]), dict(page=8), dict(q=c["q"][:, :, :3]), dict(k=c["k"].cpu()),
                dict(out=torch.empty_like(c["k"])), dict(out=c["q"][:, :1].expand_as(c["q"])),
                dict(q=c["q"].transpose(2, 3).contiguous().transpose(2, 3)),
                dict(pool=c["pool"][:, :, ::2])):
        with pytest.raises(ValueError):
            call(**bad)
    wide = tree_case(gpu, f16, 1, 2, 2, 1, 258, 4, 4)
    with pytest.raises(ValueError, match="at most 64 nodes and heads of 256"):
        run_tree(wide)
    p, n = torch.zeros(2, 3, dtype=torch.int32, device=gpu), torch.zeros(2, dtype=torch.int64, device=gpu)
    for bad in ((p.long(), n), (p, n.int()), (p, n[:1]), (p[0], n), (p.expand(2, 3).new_zeros(2, 65), n)):
        with pytest.raises(ValueError):
            rk.tree_plan(*bad)
    with pytest.raises(ValueError, match="sizes"):
        rk.tree_plan(p[:1].expand(2**31, 3), n[:1].expand(2**31))
    x, t = torch.zeros(2, 10, device=gpu), torch.zeros(2, dtype=torch.int64, device=gpu)
    with pytest.raises(ValueError, match="sizes"):
        rk.token_logprobs(x[:1].expand(2**31, 10), t[:1].expand(2**31))
    for bad in ((x.double(), t), (x, t.int()), (x, t[:1]), (x[0], t), (x, t, 11), (x, t, -1),
                (x.new_zeros(2, 100), t, 65), (x.t().contiguous().t(), t), (x[:, :0], t)):
        with pytest.raises(ValueError):
            rk.token_logprobs(*bad)
    q, k, w = torch.zeros(3, 4, 8, device=gpu), torch.zeros(3, 2, 8, device=gpu), torch.ones(8, device=gpu)
    cos = torch.zeros(3, 4, device=gpu)
    at = torch.zeros(3, dtype=torch.int64, device=gpu)
    for bad in ((q, k.half(), w, w, 1e-6, cos, cos), (q, k, w.half(), w, 1e-6, cos, cos),
                (q, k, w, w[:4], 1e-6, cos, cos), (q, k, w, w, 1e-6, cos[:2], cos[:2]),
                (q, k, w, w, 1e-6, cos, cos[:2]), (q, k, w, w, 1e-6, cos.half(), cos.half()),
                (q, k, w, w, 1e-6, cos, cos, at.int()), (q, k, w, w, 1e-6, cos, cos, at[:2]),
                (q[..., :7], k[..., :7], w[:7], w[:7], 1e-6, cos, cos), (q[:2], k, w, w, 1e-6, cos, cos),
                (q, k, w, w, 1e-6, cos, cos, at, (q,)), (q, k, w, w, 1e-6, cos, cos, at, (k, k)),
                (q, k, w, w, 1e-6, cos[:0], cos[:0], at), (q.cpu(), k, w, w, 1e-6, cos, cos)):
        with pytest.raises(ValueError):
            rk.qk_norm_rope(*bad)
    with pytest.raises(ValueError, match="sizes"):
        rk.qk_norm_rope(q[:1].expand(2**31, 4, 8), k[:1].expand(2**31, 2, 8), w, w, 1e-6, cos, cos, at[:1].expand(2**31))


# ---- tree_plan ---------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("B,T", [(1, 1), (3, 2), (5, 17), (64, 63), (7, 64)])
def test_tree_plan(gpu, B, T):
    print("case:", dict(B=B, T=T), flush=True)
    g = torch.Generator().manual_seed(B * 100 + T)
    lengths = torch.randint(0, 1 << 40, (B,), generator=g)
    chain = (torch.arange(T) - 1).int().repeat(B, 1)
    wild = torch.randint(-3, T + 2, (B, T), generator=g).int()  # parents out of order and out of range
    wild[0] = 2**31 - 1
    for parents in (random_parents(B, T, g), chain, torch.full((B, T), -1).int(), torch.full((B, T), -2).int(), wild):
        expected = plan_oracle(parents, lengths)
        wide = torch.full((B, T + 3), 5, dtype=torch.int32)
        wide[:, 1: T + 1] = parents
        for p in (parents.to(gpu), wide.to(gpu)[:, 1: T + 1], parents.t().contiguous().to(gpu).t()):
            got = rk.tree_plan(p, lengths.to(gpu))
            assert all(torch.equal(a.cpu(), e) for a, e in zip(got, expected))
    assert [tuple(t.shape) for t in rk.tree_plan(chain[:0].to(gpu), lengths[:0].to(gpu))] == [(0, T), (0, T)]


# ---- tree_attention ------------------------------------------------------------------------------

SHAPES = [  # B, T, Hq, Hkv, D, P, N
    (1, 1, 4, 2, 64, 16, 0), (1, 1, 4, 2, 64, 16, 1), (2, 8, 4, 2, 64, 16, 123), (3, 5, 28, 4, 128, 32, 200),
    (2, 64, 8, 2, 128, 64, 1111), (1, 33, 14, 2, 64, 8, 700), (2, 7, 8, 8, 128, 5, 65), (1, 16, 32, 8, 128, 64, 2048),
    (1, 3, 16, 1, 128, 16, 300), (1, 64, 32, 1, 64, 16, 129), (5, 2, 4, 2, 32, 3, 40), (2, 9, 6, 3, 80, 7, 91),
    (1, 12, 4, 2, 256, 16, 150), (1, 4, 2, 1, 2, 4, 30), (2, 3, 3, 3, 17, 4, 33), (2, 2, 4, 2, 64, 16, 31),
    (1, 20, 16, 4, 128, 16, 6000), (2, 64, 4, 2, 256, 16, 400), (3, 40, 8, 2, 32, 16, 1300), (1, 17, 4, 2, 256, 8, 77),
    (2, 30, 4, 1, 32, 32, 129), (1, 50, 7, 1, 64, 64, 3000),
    (32, 33, 32, 4, 128, 16, 100),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("shape", SHAPES)
def test_tree_attention(gpu, dtype, shape):
    print("case:", dict(dtype=dtype, shape=shape), flush=True)
    c = tree_case(gpu, dtype, *shape, seed=sum(shape))
    check_tree(c, run_tree(c))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 32)])
@pytest.mark.parametrize("B,T", [(1, 16), (5, 64)])
@pytest.mark.parametrize("N", [1, 127, 128, 129, 256, 257, 384, 500, 512, 513, 640, 2049])
def test_tree_attention_around_the_borders_of_splits(gpu, dtype, D, B, T, N):
    """Whole, split, and with splits that have the draft alone."""
    print("case:", dict(dtype=dtype, D=D, B=B, T=T, N=N), flush=True)
    c = tree_case(gpu, dtype, B, T, 4, 2, D, 16, N, seed=N + B)
    check_tree(c, run_tree(c))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f16, 64), (f32, 32), (bf16, 80)])
def test_tree_attention_peaky_scores(gpu, dtype, D):
    c = tree_case(gpu, dtype, 2, 16, 8, 2, D, 16, 500, seed=5, spread=3.0)
    check_tree(c, run_tree(c))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f16, 64), (f32, 32), (bf16, 80)])
@pytest.mark.parametrize("N", [40, 1500])
def test_scores_of_billions(gpu, dtype, D, N):
    """Keys of one number each, queries of another: the scores are exact in
    fp32 and thousands of powers of two apart, so the output is the mean of the
    values whose keys are the largest."""
    print("case:", dict(dtype=dtype, D=D, N=N), flush=True)
    c = tree_case(gpu, dtype, 2, 5, 4, 2, D, 16, N, seed=N + D, fused=False)
    blocks, total = len(c["pool"]), c["pool"].shape[0] * 16
    c["pool"][:, 0] = 128.0 * (torch.arange(total, device=gpu) % 150).view(blocks, 16, 1, 1).to(dtype)
    c["q"].fill_(2.0 ** (14 if dtype == f16 else 17))
    c["k"].copy_(128.0 * torch.arange(130, 150, 2, device=gpu).view(2, 5, 1, 1).expand(c["k"].shape))
    expected, _ = tree_oracle(*(c[n] for n in ("q", "pool", "rows", "k", "v", "mask", "page")), False)
    # weights of 1 or 0; up to 64 equal keys added and divided
    check(run_tree(c), expected, HALF[dtype] * expected.abs() + 2.0 ** -25 + 66 * U * 6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f16, 64), (f32, 32), (bf16, 80)])
@pytest.mark.parametrize("N", [0, 40, 1500])
def test_a_query_that_is_not_a_number_has_no_answer(gpu, dtype, D, N):
    print("case:", dict(dtype=dtype, D=D, N=N), flush=True)
    c = tree_case(gpu, dtype, 2, 7, 8, 2, D, 16, N, seed=N + D, fused=False)
    c["mask"][1, 3] = 0
    expected, tol = tree_oracle(*(c[n] for n in ("q", "pool", "rows", "k", "v", "mask", "page")), dtype != f32)
    for b, t, h in ((0, 2, 5), (1, 0, 0), (1, 3, 1)):  # (the last node is absent: zeros)
        c["q"][b, t, h, D - 1] = float("nan")
        if (b, t) != (1, 3):
            expected[b, t, h] = float("nan")
    check(run_tree(c), expected, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f16, 64), (f32, 48), (bf16, 24)])
@pytest.mark.parametrize("N", [0, 100, 1500])
def test_masked_places_may_hold_anything(gpu, dtype, D, N):
    """NaN and infinities where a mask hides them, no rows at all, rows
    outside the pool, the same row twice, whole requests absent."""
    print("case:", dict(dtype=dtype, D=D, N=N), flush=True)
    B, T, Hq, Hkv, P = 4, 37, 8, 2, 16
    c = tree_case(gpu, dtype, B, T, Hq, Hkv, D, P, N, seed=N + D, fused=False)
    total = c["pool"].shape[0] * P
    if N:
        c["rows"][0] = -1  # nothing but the draft
        c["rows"][1, ::3] = c["rows"][1, 0]  # rows that repeat
        c["rows"][2, ::2] = torch.tensor([total, -2, 2**62, -2**62, 2**32], device=gpu).repeat(N)[: len(range(0, N, 2))]
        # no selected row lies in the last block: it may hold anything
        inside = c["rows"] < total - P
        c["rows"] = torch.where(inside | (c["rows"] >= total), c["rows"], -1)
        c["pool"][-1] = float("nan")
    c["mask"][3] = 0
    absent = c["mask"] == 0
    c["k"][absent] = float("nan")
    c["v"][absent] = float("inf")
    c["q"][absent] = float("nan")
    c["k"][3], c["v"][3] = float("-inf"), float("nan")
    check_tree(c, run_tree(c))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f16, 64), (f32, 48)])
def test_a_draft_s_infinities_reach_its_descendants_only(gpu, dtype, D):
    c = tree_case(gpu, dtype, 1, 40, 8, 2, D, 16, 200, seed=3, fused=False)
    parents = torch.tensor([[-1] + [(t - 1) // 2 for t in range(1, 40)]], dtype=torch.int32)
    c["mask"] = plan_oracle(parents, torch.zeros(1).long())[0].to(gpu)
    c["v"][0, 5, 0, 3] = float("inf")
    c["v"][0, 11, 0, 3] = float("-inf")  # below node 5: inf - inf
    c["v"][0, 36, 1, D - 1] = float("nan")
    c["v"][0, 2, 1, 7] = float("-inf")
    out = run_tree(c)
    seen = seen_nodes(c["mask"].cpu())[0]
    for t in range(40):
        nan_3 = bool(seen[t, 5] and seen[t, 11])
        assert bool(out[0, t, 0, 3].isnan()) == nan_3
        assert bool(out[0, t, 0, 3] == float("inf")) == bool(seen[t, 5] and not nan_3)
        assert bool(out[0, t, 7, D - 1].isnan()) == bool(seen[t, 36])
        assert bool(out[0, t, 4, 7] == float("-inf")) == bool(seen[t, 2])
    finite = dict(c, v=c["v"].nan_to_num(0.0, 0.0, 0.0))
    expected, tol = tree_oracle(*(finite[n] for n in ("q", "pool", "rows", "k", "v", "mask", "page")), dtype != f32)
    clean = out.cpu().double().isfinite()
    assert clean.sum() > 0.95 * clean.numel()
    check(torch.where(clean, out.cpu().double(), expected), expected, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,T", [(bf16, 128, 9), (f16, 64, 3), (bf16, 128, 20), (f16, 128, 33), (f32, 32, 9)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_the_last_node_s_value_reaches_no_other(gpu, dtype, D, T, value):
    """Nor its key: tiles hold more keys than the tree has nodes."""
    print("case:", dict(dtype=dtype, D=D, T=T, value=value), flush=True)
    c = tree_case(gpu, dtype, 2, T, 8, 2, D, 16, 70, seed=T, fused=False)
    c["mask"] = plan_oracle(torch.tensor([[-1] + [0] * (T - 1)] * 2, dtype=torch.int32), torch.zeros(2).long())[0].to(gpu)
    expected, tol = tree_oracle(*(c[n] for n in ("q", "pool", "rows", "k", "v", "mask", "page")), dtype != f32)
    c["v"][:, T - 1], c["k"][:, T - 1] = value, value
    got = run_tree(c)
    check(got[:, : T - 1], expected[:, : T - 1], tol[:, : T - 1])
    assert not got[:, T - 1].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [bf16, f32])
def test_infinite_keys_of_the_past(gpu, dtype):
    """A key of -inf against a positive query scores -inf (weight 0); NaN keys make their readers NaN, no one else."""
    c = tree_case(gpu, dtype, 2, 4, 4, 2, 128, 16, 300, seed=1, fused=False)
    c["q"].abs_()
    row = int(c["rows"][0][c["rows"][0] >= 0][0])
    c["rows"][1][c["rows"][1] == row] = -1
    c["pool"][row // 16, 0, row % 16, 0] = float("-inf")
    expected, tol = tree_oracle(*(c[n] for n in ("q", "pool", "rows", "k", "v", "mask", "page")), dtype != f32)
    without = dict(c, rows=torch.where(c["rows"] == row, -1, c["rows"]))
    expected_0, tol_0 = tree_oracle(*(without[n] for n in ("q", "pool", "rows", "k", "v", "mask", "page")),
                                    dtype != f32)
    got = run_tree(c)
    check(got[:, :, :2], expected_0[:, :, :2], tol_0[:, :, :2])
    check(got[:, :, 2:], expected[:, :, 2:], tol[:, :, 2:])
    c["pool"][row // 16, 0, row % 16, 0] = float("nan")
    got = run_tree(c)
    live = (c["mask"][0] != 0).cpu()
    assert got[0, live][:, :2].isnan().all() and not got[0, :, 2:].isnan().any() and not got[1].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f16, 64), (f32, 32)])
def test_tree_attention_layouts(gpu, dtype, D):
    """Strides of their own for every operand, an output inside a larger
    buffer (the rest stays), another stream, and the Python launcher."""
    B, T, Hq, Hkv, P, N = 2, 6, 8, 2, 16, 150
    c = tree_case(gpu, dtype, B, T, Hq, Hkv, D, P, N, seed=8)
    expected = run_tree(c)
    check_tree(c, expected)
    order = dict(c)
    order["q"] = c["q"].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    order["k"] = c["k"].permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)
    order["v"] = c["v"].permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)
    order["rows"] = c["rows"].t().contiguous().t()
    order["mask"] = c["mask"].t().contiguous().t()
    order["pool"] = c["pool"].contiguous()
    assert torch.equal(run_tree(order), expected)
    wide = torch.full((B, T + 2, Hq + 3, D + 16), 7.0, dtype=dtype, device=gpu)
    out = wide[:, 1: T + 1, 2: Hq + 2, 8: D + 8]
    assert run_tree(c, out=out) is not None
    assert torch.equal(out, expected)
    wide[:, 1: T + 1, 2: Hq + 2, 8: D + 8] = 7.0
    assert (wide == 7.0).all()
    # heads whose addresses are multiples of their element size only
    off = torch.zeros(B * T * (Hq + 1) * (D + 1) + 1, dtype=dtype, device=gpu)[1:].view(B, T, Hq + 1, D + 1)
    off = off[:, :, :Hq, :D].copy_(c["q"])
    check_tree(c, run_tree(dict(c, q=off)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run_tree(c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, expected)


@pytest.mark.gpu
def test_tree_attention_rows_beyond_four_gigabytes(gpu):
    """Pool offsets that pass 32 bits."""
    P, Hkv, D = 64, 8, 128
    blocks = (5 << 30) // (2 * P * Hkv * D * 2)
    pool = rk.padded_pool(blocks, P, Hkv, D, bf16, gpu)
    pool.zero_()
    c = tree_case(gpu, bf16, 1, 5, 8, Hkv, D, P, 64)
    pool[blocks - 2:] = c["pool"][:2]
    rows = torch.where(c["rows"] >= 0, c["rows"] % (2 * P), -1)
    small = run_tree(dict(c, rows=rows))
    assert torch.equal(run_tree(dict(c, pool=pool, rows=torch.where(rows >= 0, rows + (blocks - 2) * P, -1))), small)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,N", [(bf16, 128, 1500), (f16, 64, 40), (f32, 32, 300)])
def test_tree_attention_graphs(gpu, dtype, D, N):
    """Two captured calls replayed in turn and at once, eager calls between:
    each keeps its own result."""
    cases = [tree_case(gpu, dtype, 2, 9, 8, 2, D, 16, N, seed=s, fused=False) for s in (0, 1)]
    run_tree(cases[0])
    torch.cuda.synchronize()
    graphs = []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run_tree(c)
        graphs.append((graph, out))
    side = torch.cuda.Stream()
    for i in range(3):
        for c in cases:
            c["q"].copy_(c["q"].roll(1, 0))
            c["v"].mul_(-1)
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for c, (_, out) in zip(cases, graphs):
            assert torch.equal(out, run_tree(c)), i


@pytest.mark.gpu
def test_reruns_are_bit_identical(gpu):
    c = tree_case(gpu, bf16, 2, 16, 28, 4, 128, 32, 3000)
    first = run_tree(c)
    assert all(torch.equal(run_tree(c), first) for _ in range(5))
    x = torch.randn(3, 50000, device=gpu)
    t = torch.tensor([1, 2, 3], device=gpu)
    first = rk.token_logprobs(x, t, 20)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(rk.token_logprobs(x, t, 20), first))


# ---- qk_norm_rope --------------------------------------------------------------------------------


def norm_case(gpu, dtype, n, Hq, Hkv, D, table, rows, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, (Hq + 2 * Hkv) * D, generator=g) * scale).to(dtype).to(gpu)
    angle = torch.rand(rows, D // 2, generator=g) * 6.3
    return dict(q=x[:, : Hq * D].view(n, Hq, D), k=x[:, Hq * D: (Hq + Hkv) * D].view(n, Hkv, D),
                qw=(1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(gpu),
                kw=(1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(gpu),
                cos=angle.cos().to(table).to(gpu), sin=angle.sin().to(table).to(gpu),
                at=torch.randint(0, rows, (n,), generator=g).to(gpu))


def check_norm(c, got, positions, eps=1e-6):
    for x, (out, tol) in zip(got, norm_oracle(c["q"], c["k"], c["qw"], c["kw"], eps, c["cos"], c["sin"], positions)):
        check(x, out, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,table", [(bf16, bf16), (bf16, f32), (f16, f16), (f16, f32), (f32, f32)])
@pytest.mark.parametrize("n,Hq,Hkv,D", [(1, 1, 1, 2), (3, 4, 2, 64), (1, 32, 8, 128), (17, 28, 4, 128), (5, 14, 2, 64),
                                        (4, 3, 1, 96), (2, 5, 5, 30), (2, 8, 2, 256), (300, 4, 2, 32), (2, 2, 2, 1024),
                                        (1, 2, 1, 2050)])
def test_qk_norm_rope(gpu, dtype, table, n, Hq, Hkv, D):
    print("case:", dict(dtype=dtype, table=table, n=n, Hq=Hq, Hkv=Hkv, D=D), flush=True)
    c = norm_case(gpu, dtype, n, Hq, Hkv, D, table, n + 9, seed=n + D)
    args = c["q"], c["k"], c["qw"], c["kw"], 1e-6, c["cos"], c["sin"]
    check_norm(c, rk.qk_norm_rope(*args, c["at"]), c["at"])
    check_norm(c, rk.qk_norm_rope(*args), None)
    wild = c["at"].clone()
    wild[0] = -5
    wild[-1] = 2**40
    check_norm(c, rk.qk_norm_rope(*args, wild), wild)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
def test_qk_norm_rope_in_place_and_layouts(gpu, dtype):
    c = norm_case(gpu, dtype, 13, 6, 2, 64, dtype, 40, seed=2)
    args = c["qw"], c["kw"], 1e-5, c["cos"], c["sin"], c["at"]
    expected = rk.qk_norm_rope(c["q"], c["k"], *args)
    check_norm(c, expected, c["at"], 1e-5)
    same = rk.qk_norm_rope(c["q"].clone().transpose(0, 1).contiguous().transpose(0, 1), c["k"].contiguous(), *args)
    assert all(torch.equal(a, b) for a, b in zip(same, expected))
    # heads at any element: another order of the squares' sum, within the bound that holds for every order
    off = torch.zeros(13 * 7 * 67 + 1, dtype=dtype, device=gpu)[1:].view(13, 7, 67)[:, :6, :64].copy_(c["q"])
    check_norm(c, rk.qk_norm_rope(off, c["k"], *args), c["at"], 1e-5)
    wide = torch.full((15, 10, 80), 3.0, dtype=dtype, device=gpu)
    outs = wide[1:14, 1:7, 8:72], wide[1:14, 7:9, 8:72]
    rk.qk_norm_rope(c["q"], c["k"], *args, out=outs)
    assert torch.equal(outs[0], expected[0]) and torch.equal(outs[1], expected[1])
    wide[1:14, 1:9, 8:72] = 3.0
    assert (wide == 3.0).all()
    q, k = c["q"], c["k"]  # views of one projection
    done = rk.qk_norm_rope(q, k, *args, out=(q, k))
    assert done[0].data_ptr() == q.data_ptr()
    assert torch.equal(q, expected[0]) and torch.equal(k, expected[1])
    empty = rk.qk_norm_rope(q[:0], k[:0], c["qw"], c["kw"], 1e-6, c["cos"], c["sin"], c["at"][:0])
    assert empty[0].shape == (0, 6, 64)


@pytest.mark.gpu
def test_qk_norm_rope_extremes(gpu):
    """Zero heads (eps alone), the largest squares that fp32 holds, NaN in one head only."""
    c = norm_case(gpu, bf16, 3, 4, 2, 128, bf16, 8, seed=4)
    c["q"][0, 1] = 0
    c["q"][1] *= 2.0 ** 55
    c["k"][2, 0] = 2.0 ** -60
    args = c["qw"], c["kw"], 1e-6, c["cos"], c["sin"], c["at"]
    check_norm(c, rk.qk_norm_rope(c["q"], c["k"], *args), c["at"])
    c["q"][2, 3, 5] = float("nan")
    got, _ = rk.qk_norm_rope(c["q"], c["k"], *args)
    assert got[2, 3].isnan().all() and got.isnan().sum() == 128


# ---- token_logprobs --------------------------------------------------------------------------------


def check_logprobs(logits, tokens, top):
    got, e = rk.token_logprobs(logits, tokens, top), logprob_oracle(logits, tokens, top)
    assert torch.equal(got.top_ids.cpu(), e["ids"])
    check(got.logprobs, *e["logprobs"])
    check(got.entropy, *e["entropy"])
    check(got.top_logprobs, *e["values"])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (2, 2, 0), (3, 7, 7), (5, 256, 64), (1, 128256, 5), (9, 32001, 20),
                                     (300, 1000, 3), (2, 65, 64), (1, 152064, 64), (700, 4099, 1), (33, 20000, 0)])
def test_token_logprobs(gpu, dtype, R, V, top):
    print("case:", dict(dtype=dtype, R=R, V=V, top=top), flush=True)
    g = torch.Generator().manual_seed(R + V)
    logits = (torch.randn(R, V, generator=g) * 3).to(dtype).to(gpu)
    check_logprobs(logits, torch.randint(0, V, (R,), generator=g).to(gpu), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("V", [130, 5000, 40001])
def test_token_logprobs_masks_and_ties(gpu, dtype, V):
    """Grammars that leave 0, 1, 3 or 1000 tokens (-inf or the type's lowest
    value elsewhere), rows of one value, few distinct values, zeros of both
    signs, ascending, descending and clustered logits, NaN and +inf."""
    print("case:", dict(dtype=dtype, V=V), flush=True)
    g = torch.Generator().manual_seed(V)
    low = torch.finfo(dtype).min
    base = torch.randn(V, generator=g)
    rows = []
    for fill in (-math.inf, low):
        for keep in (0, 1, 3, 1000):
            row = torch.full((V,), fill)
            at = torch.randperm(V, generator=g)[:keep]
            row[at] = base[at]
            rows.append(row)
    ramp = torch.linspace(-10, 10, V)
    cluster = base.clone()
    cluster[V // 2: V // 2 + 100] += 20
    cluster_high = torch.full((V,), -5.0)
    cluster_high[-70:] = torch.arange(70).float() / 8
    rows += [torch.zeros(V), torch.where(base > 0, 0.0, -0.0), (base * 2).round(), ramp, ramp.flip(0), cluster,
             cluster_high, torch.full((V,), -3.0), torch.full((V,), torch.finfo(dtype).max),
             torch.where(torch.arange(V) % 3 == 0, torch.finfo(dtype).max, low), base.clone(), base.clone(),
             base.clone(), base.clone(), torch.full((V,), math.inf)]
    rows[-5][V // 3] = math.nan
    rows[-4][V // 2] = math.inf
    rows[-3][::2] = math.nan
    rows[-2][V - 1], rows[-2][0] = math.inf, math.nan
    logits = torch.stack(rows).to(dtype).to(gpu)
    tokens = torch.randint(0, V, (len(rows),), generator=g).to(gpu)
    for top in (0, 1, 5, 64):
        check_logprobs(logits, tokens, top)
    for i in range(0, len(rows), 3):  # the same rows one at a time: other splits
        check_logprobs(logits[i: i + 1], tokens[i: i + 1], 5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
def test_token_logprobs_layouts(gpu, dtype):
    """Rows at any element offset and stride, several tokens per row, tokens
    outside the vocabulary, strided tokens, no rows."""
    g = torch.Generator().manual_seed(1)
    V = 3001
    flat = (torch.randn(7 * 3017 + 9, generator=g) * 2).to(dtype).to(gpu)
    for offset in range(9):
        logits = flat[offset: offset + 7 * 3017].view(7, 3017)[:, :V]
        tokens = torch.randint(-2, V + 2, (7, 4), generator=g)
        tokens[0] = torch.tensor([-1, V, 2**40, -2**40])
        tokens = tokens.to(gpu)
        check_logprobs(logits, tokens, 6)
    check_logprobs(logits, tokens.t().contiguous().t(), 2)
    check_logprobs(logits, tokens[:, 1], 2)
    check_logprobs(logits.expand(7, V)[::2], tokens[::2, 0], 1)
    check_logprobs(flat[:V].expand(5, V), tokens[:5, 0], 4)
    none = rk.token_logprobs(logits, tokens[:, :0], 3)
    assert none.logprobs.shape == (7, 0)
    assert torch.equal(none.top_ids, rk.token_logprobs(logits, tokens, 3).top_ids)
    empty = rk.token_logprobs(logits[:0], tokens[:0], 3)
    assert empty.logprobs.shape == (0, 4) and empty.top_ids.shape == (0, 3) and empty.entropy.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
def test_certain_tokens(gpu, dtype):
    """One token alone, or far above the others: no rounding puts its log probability above 0 or the entropy below."""
    V = 5001
    logits = torch.full((40, V), -math.inf)
    logits[20:] = -60000.0
    at = torch.randint(0, V, (40,), generator=torch.Generator().manual_seed(0))
    logits[torch.arange(40), at] = torch.linspace(-700, 900, 40)
    got = check_logprobs(logits.to(dtype).to(gpu), at.to(gpu), 3)
    assert (got.logprobs <= 0).all() and (got.entropy >= 0).all() and (got.top_logprobs <= 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [bf16, f32])
def test_a_whole_verification_in_one_graph(gpu, dtype):
    """Plan, norm + rotation, attention and log probabilities one after the
    other, captured and replayed with other inputs, against the eager calls."""
    B, T, Hq, Hkv, D, P, N, V = 2, 12, 8, 2, 64, 16, 400, 3000
    g = torch.Generator().manual_seed(0)
    c = tree_case(gpu, dtype, B, T, Hq, Hkv, D, P, N)
    parents = random_parents(B, T, g).to(gpu)
    lengths = torch.tensor([400, 380], device=gpu)
    table = torch.rand(512, D // 2, generator=g).to(gpu)
    weights = [torch.rand(D, generator=g).to(dtype).to(gpu) for _ in range(2)]
    head = (torch.randn(Hq * D, V, generator=g) * 0.1).to(dtype).to(gpu)
    tokens = torch.randint(0, V, (B * T,), generator=g).to(gpu)

    def verify():
        mask, positions = rk.tree_plan(parents, lengths)
        q, k = rk.qk_norm_rope(c["q"].reshape(B * T, Hq, D), c["k"].reshape(B * T, Hkv, D), *weights, 1e-6, table.cos(),
                               table.sin(), positions.view(-1))
        out = rk.tree_attention(q.view(B, T, Hq, D), c["pool"], c["rows"], k.view(B, T, Hkv, D), c["v"], mask, P)
        return (mask, positions, q, k, out) + tuple(rk.token_logprobs(out.view(B * T, -1) @ head, tokens, 4))

    verify()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = verify()
    for i in range(3):
        parents.copy_(random_parents(B, T, g))
        lengths += 7
        c["q"].mul_(-1)
        c["rows"].copy_(c["rows"].roll(3, 1))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, verify())), i


@pytest.mark.gpu
def test_token_logprobs_beyond_four_gigabytes(gpu):
    """Row offsets that pass 32 bits."""
    R, V = 9, 256
    logits = torch.empty_strided((R, V), (300_000_000, 1), dtype=bf16, device=gpu)
    for r in range(R):
        logits[r] = torch.randn(V, generator=torch.Generator().manual_seed(r)).to(bf16)
    check_logprobs(logits, torch.arange(R, device=gpu), 3)


@pytest.mark.gpu
def test_token_logprobs_graphs(gpu):
    """Two captured calls of one shape, replayed with eager calls between."""
    inputs = [torch.randn(3, 50001, device=gpu) for _ in range(2)]
    tokens = torch.tensor([5, 50000, 7], device=gpu)
    rk.token_logprobs(inputs[0], tokens, 8)
    torch.cuda.synchronize()
    graphs = []
    for x in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = rk.token_logprobs(x, tokens, 8)
        graphs.append((graph, out))
    side = torch.cuda.Stream()
    for _ in range(3):
        for x in inputs:
            x.copy_(x.roll(17, 1))
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for x, (_, out) in zip(inputs, graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, rk.token_logprobs(x, tokens, 8)))


# ---- launchers -------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_native_and_python_launchers_agree(gpu, monkeypatch):
    class PythonOnly:
        def __getattr__(self, name):
            return lambda *a: None

    c = tree_case(gpu, bf16, 2, 9, 8, 2, 128, 16, 700)
    n = norm_case(gpu, f16, 5, 4, 2, 64, f32, 20)
    x, t = torch.randn(4, 9001, device=gpu), torch.tensor([[1, 2], [3, 4], [5, -6], [7, 8]], device=gpu)
    parents = random_parents(3, 20, torch.Generator().manual_seed(0)).to(gpu)
    lengths = torch.tensor([5, 6, 7], device=gpu)
    out = torch.empty_like(c["q"])
    pair = torch.empty_like(n["q"]), torch.empty_like(n["k"])
    calls = [lambda: (run_tree(c),), lambda: (run_tree(c, out=out).clone(),), lambda: rk.tree_plan(parents, lengths),
             lambda: rk.token_logprobs(x, t, 9), lambda: rk.token_logprobs(x, t[:, 0].contiguous(), 0),
             lambda: rk.qk_norm_rope(n["q"], n["k"], n["qw"], n["kw"], 1e-6, n["cos"], n["sin"], n["at"]),
             lambda: rk.qk_norm_rope(n["q"], n["k"], n["qw"], n["kw"], 1e-6, n["cos"], n["sin"], out=pair)]
    module = rk._load_launch()
    taken = []

    class Counting:
        def __getattr__(self, name):
            def call(*a):
                done = getattr(module, name)(*a)
                taken.append(done is not None)
                return done
            return call

    monkeypatch.setattr(rk, "_launch", Counting())
    native = [[r.clone() for r in call()] for call in calls]
    assert all(taken) and len(taken) == len(calls)
    monkeypatch.setattr(rk, "_launch", PythonOnly())
    for a, b in zip(native, [call() for call in calls]):
        assert all(torch.equal(x, y) and x.dtype == y.dtype and x.shape == y.shape for x, y in zip(a, b))
