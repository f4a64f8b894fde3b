"""Rows held in 8 bits (append_page_8bit, PageAppender(form=), append_items_8bit,
read_rows_8bit, attend_8bit) against their definitions in 64 bits, at the sizes
and values where they can go wrong.

Codes, scales and values read back are exact: the scale is the fp32 number
nearest to max|x| / Q, the code the one nearest to the exact quotient by it,
the value their product rounded to fp32 and then to the type asked for. Bounds
are exact. Tolerances of the others, with u = 2^-24 (half a step of fp32) and
r = half a step of the output's type relative to the value:

- page means of the products code * scale: one rounding to fp32 (u), behind
  sums in 64 bits;
- attention: a score is a sum of D products of a query with whole codes, off by
  2 (D + 4) u sum|q code| scale D^-1/2 at most (twice u: a matrix core need not
  round to nearest) and 4 u of itself for the two factors behind it; a weight's
  relative error is that of its score and of its maximum's, 2^-22 for exp2 and
  the rounding of its argument (2 u |score|), u for the values' scale, and
  2^-17 where it goes to the matrix cores as two 8-bit parts; numerator and
  denominator take N terms, 2 u each. Both enter the output times sum w |V|,
  and its own rounding is r |out|.
"""

import ctypes
import math

import pytest
import torch

from nano_hisparse import _hip
from nano_hisparse import row_kernels as rk

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
i8, e4m3 = torch.int8, torch.float8_e4m3fn
U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (bf16, f16, f32)}
LARGEST = {i8: 127.0, e4m3: 448.0}

# ---- oracles -------------------------------------------------------------------------------

E4M3 = torch.tensor([m * 2.0 ** -9 for m in range(8)]
                    + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119], dtype=torch.float64)


def quantised(x, code):
    """(codes as numbers, scales) of x [..., D] in float64: the nearest code
    by search, ties to the even one."""
    x = x.double()
    odd = ~torch.isfinite(x).all(-1, keepdim=True)
    largest = x.abs().nan_to_num(nan=0.0, posinf=0.0).amax(-1, keepdim=True)
    scale = (largest / LARGEST[code]).float().clamp(min=2.0 ** -80).double()
    size = torch.where(odd, 0.0, x.abs() / scale)
    table = torch.arange(128, dtype=torch.float64) if code == i8 else E4M3
    above = torch.searchsorted(table, size.contiguous()).clamp(1, len(table) - 1)
    low, high = table[above - 1], table[above]
    down = (size - low < high - size) | ((size - low == high - size) & (above % 2 == 1))
    codes = torch.where(down, low, high) * torch.sign(x).nan_to_num()
    return torch.where(odd, 0.0, codes), torch.where(odd, math.nan, scale)[..., 0]


def values(form, rows, exact=False):
    """The fp32 values [..., Hkv, D] of rows [..., row_bytes] on the CPU, from
    the bytes (exact: in float64, their product not rounded)."""
    rows = rows.cpu().contiguous()
    n = form.kv_heads * form.head_dim
    byte = rows[..., :n].long().unflatten(-1, (form.kv_heads, form.head_dim))
    if form.code == i8:
        codes = (byte - 256 * (byte > 127)).float()
    else:
        size = torch.cat((E4M3, torch.tensor([math.nan], dtype=torch.float64))).float()[byte & 127]
        codes = torch.where(byte > 127, -size, size)
    scales = rows[..., form.scales_at:form.scales_at + 4 * form.kv_heads].contiguous().view(torch.float32)
    return codes.double() * scales.double()[..., None] if exact else codes * scales[..., None]


def held(form, pool, rows):
    """K and V [n, Hkv, D] (fp32, CPU) of pool rows, which are all in the pool."""
    P = pool.shape[2]
    at = rows.to(pool.device)
    return [values(form, pool[at // P, plane, at % P]) for plane in (0, 1)]


def attend_oracle(form, q, pool, rows):
    """(out, tolerance) in float64 on the CPU."""
    B, Hq, D = q.shape
    g, total, dtype = Hq // form.kv_heads, pool.shape[0] * pool.shape[2], q.dtype
    q, lists = q.cpu().double(), rows.cpu()
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        for h in range(Hq) if rows.ndim == 3 else [slice(0, Hq)]:
            one = lists[b] if rows.ndim == 2 else lists[b, h]
            one = one[(one >= 0) & (one < total)]
            if not len(one):
                continue
            hs = list(range(Hq))[h] if isinstance(h, slice) else [h]
            kv = torch.tensor(hs) // g
            keys, vals = (x.double()[:, kv] for x in held(form, pool, one))
            qt = q[b, hs]
            s = (qt * keys).sum(-1) / math.sqrt(D)
            w = torch.softmax(s, 0)
            o = (w[..., None] * vals).sum(0)
            size = (w[..., None] * vals.abs()).sum(0)
            s_err = 2 * (D + 4) * U * ((qt * keys).abs().sum(-1) / math.sqrt(D)).amax(0) + 6 * U * s.abs().amax(0)
            w_err = 2 * s_err + 2.0 ** -22 + 2.0 ** -17 * (dtype != f32) + 2 * U
            rel = 2 * w_err + 2 * (len(one) + 64) * U
            out[b, hs], tol[b, hs] = o, rel[:, None] * size + HALF[dtype] * o.abs() + 1e-30
    return out, tol + 2.0 ** -25 if dtype == f16 else tol


def check(got, expected, tol):
    got = got.detach().cpu().double()
    assert got.shape == expected.shape
    same = (got == expected) | (got.isnan() & expected.isnan())
    worst = torch.where(same, 0.0, (got - expected).abs() / tol)
    assert not worst.isnan().any(), "a NaN on one side only"
    assert worst.max().item() <= 1.0 if worst.numel() else True, f"{worst.max().item():.3g} times the tolerance"


# ---- inputs ----------------------------------------------------------------------------------


def keys(gen, *shape, dtype=f32):
    size = torch.exp(torch.randn(*shape[-2:], generator=gen) * 0.5)
    return (torch.randn(*shape, generator=gen) * size).to(dtype)


def make_pool(form, blocks, P, gen, device, gap=0):
    """A pool of random codes and scales (every finite code occurs); `gap`
    bytes follow each block."""
    R = form.row_bytes
    flat = torch.zeros(blocks * (2 * P * R + gap), dtype=torch.uint8)
    pool = flat.as_strided((blocks, 2, P, R), (2 * P * R + gap, P * R, R, 1))
    n = form.kv_heads * form.head_dim
    codes = torch.randint(0, 256, (blocks, 2, P, n), generator=gen)
    codes = torch.where((codes & 127) == 127, codes - 1, codes)  # e4m3's NaN
    pool[..., :n] = codes.to(torch.uint8)
    scales = torch.exp(torch.randn(blocks, 2, P, form.kv_heads, generator=gen)) / LARGEST[form.code]
    form.scales(pool).copy_(scales)
    moved = flat.to(device)
    return moved.as_strided(pool.shape, pool.stride())


def empty_page(form, dtype, device):
    shape = (form.kv_heads, form.head_dim)
    return (torch.zeros(shape, device=device), torch.full(shape, math.inf, dtype=dtype, device=device),
            torch.full(shape, -math.inf, dtype=dtype, device=device))


def check_page(form, pool, block, earlier, k, v, within, summary, low, high, low0, high0):
    """The page's rows, bounds and mean after k and v were appended at `within`
    to `earlier` (the earlier keys' exact values, CPU)."""
    n = len(k)
    for plane, x in enumerate((k, v)):
        rows = pool[block, plane, within:within + n].cpu()
        codes, scale = quantised(x.cpu(), form.code)
        got = form.scales(rows.contiguous())
        assert torch.equal(got.nan_to_num(nan=-1.0), scale.float().nan_to_num(nan=-1.0))
        assert torch.equal(form.codes(rows.contiguous()).float().double(), codes)
    kd = k.cpu().float()
    assert torch.equal(low.cpu().float().nan_to_num(nan=7e7), torch.minimum(low0.float(), kd.amin(0)).nan_to_num(nan=7e7))
    assert torch.equal(high.cpu().float().nan_to_num(nan=7e7),
                       torch.maximum(high0.float(), kd.amax(0)).nan_to_num(nan=7e7))
    codes, scale = quantised(k.cpu(), form.code)
    total = torch.cat((earlier.double(), codes * scale[..., None]))
    mean = total.mean(0)
    check(summary, mean, U * mean.abs() + 2.0 ** -50 * total.abs().mean(0) + 2.0 ** -149)


# ---- the form, the tables of arguments, refusals (CPU) -----------------------------------------


@pytest.mark.parametrize("heads, dim, scales_at, row", [(8, 128, 1024, 1056), (2, 64, 128, 144), (1, 1, 4, 16),
                                                       (3, 5, 16, 32), (4, 128, 512, 528), (1, 1024, 1024, 1040)])
def test_row_form(heads, dim, scales_at, row):
    form = rk.Rows8(i8, heads, dim)
    assert (form.scales_at, form.row_bytes) == (scales_at, row)
    assert _hip.load(check_runtime=False).nhs_row8_bytes(heads, dim) == row
    pool = rk.pool_8bit(3, 4, form, "cpu")
    assert pool.shape == (3, 2, 4, row) and rk.pool_block_stride(pool) == 8 * row
    form.codes(pool).zero_()
    form.scales(pool).fill_(1.0)
    assert form.codes(pool).shape == (3, 2, 4, heads, dim) and form.scales(pool).shape == (3, 2, 4, heads)


def test_refused_forms():
    for form in (rk.Rows8(torch.uint8, 2, 8), rk.Rows8(i8, 0, 8), rk.Rows8(e4m3, 2, 1025), rk.Rows8(i8, 2, 0)):
        with pytest.raises(ValueError):
            rk.pool_8bit(2, 4, form, "cpu")


def test_cpu_tensors_are_refused():
    form = rk.Rows8(i8, 2, 16)
    pool = rk.pool_8bit(2, 4, form, "cpu")
    rows = torch.zeros(1, 3, dtype=torch.int64)
    k = torch.zeros(2, 2, 16)
    summary, low, high = empty_page(form, f32, "cpu")
    with pytest.raises(ValueError, match="GPU"):
        rk.attend_8bit(torch.zeros(1, 2, 16), pool, form, rows)
    with pytest.raises(ValueError, match="GPU"):
        rk.read_rows_8bit(pool, form, rows[0], f32)
    with pytest.raises(ValueError, match="GPU"):
        rk.append_page_8bit(k, k, pool, form, 0, 0, None, 0, summary, low, high)
    with pytest.raises(ValueError, match="GPU"):
        rk.PageAppender(k, k, pool, None, summary, low, high, form)
    with pytest.raises(ValueError, match="GPU"):
        rk.append_items_8bit(k, k, pool, form, None, torch.zeros(2, 9, dtype=torch.int64), rows[0, :2])


def call(name, **changed):
    """A library call with well-formed arguments at addresses that nothing may
    read (every call here is refused before it launches), but for `changed`."""
    at = 1 << 20
    args = {
        "nhs_append_page8": dict(k=at, v=at, token_stride=32, dtype=0, code=0, kv=2, dim=16, page=4, pool=at, stride=0,
                                 block=0, within=0, count=1, host=at, host_page=0, summary=at, low=at, high=at,
                                 stream=0),
        "nhs_append_items8": dict(batch=1, k=at, v=at, token_stride=32, dtype=0, code=0, kv=2, dim=16, page=4, pool=at,
                                  stride=0, host=at, items=at, lengths=at, stream=0),
        "nhs_read_rows8": dict(pool=at, pool_rows=8, stride=0, code=0, kv=2, dim=16, page=4, rows=at, rows_stride=1, n=2,
                               dtype=0, k=at, k_stride=32, v=at, v_stride=32, stream=0),
        "nhs_attend_rows8": dict(q=at, dtype=0, q_b=32, q_h=16, pool=at, pool_rows=8, stride=0, code=0, rows=at, r_b=3,
                                 r_h=0, r_c=1, batch=1, n=3, heads=2, kv=2, dim=16, page=4, out=at, o_b=32, o_h=16,
                                 ws=at, ws_bytes=1 << 30, stream=0),
    }[name]
    assert not changed.keys() - args.keys()
    args.update(changed)
    lib = _hip.load(check_runtime=False)
    types = _hip.SIGNATURES[name][0]
    return getattr(lib, name)(*(ctypes.c_void_p(v) if t is ctypes.c_void_p else v for v, t in zip(args.values(), types)))


BAD = {
    "nhs_append_page8": [dict(k=0), dict(v=0), dict(pool=0), dict(summary=0), dict(low=0), dict(high=0), dict(dtype=3),
                         dict(dtype=-1), dict(code=2), dict(kv=0), dict(dim=0), dict(dim=1025), dict(page=0),
                         dict(pool=(1 << 20) + 8), dict(host=(1 << 20) + 4), dict(stride=24), dict(stride=300),
                         dict(block=-1), dict(within=-1), dict(within=4), dict(count=0), dict(count=5),
                         dict(within=2, count=3), dict(within=2 ** 31 - 1, count=4), dict(token_stride=31),
                         dict(host_page=-1), dict(kv=(1 << 20) + 1, token_stride=1 << 25)],
    "nhs_append_items8": [dict(batch=-1), dict(batch=65536), dict(k=0), dict(v=0), dict(pool=0), dict(items=0),
                          dict(lengths=0), dict(dtype=7), dict(code=-1), dict(token_stride=0), dict(page=-4),
                          dict(stride=16), dict(host=(1 << 20) + 8), dict(dim=2000, token_stride=4000)],
    "nhs_read_rows8": [dict(pool=0), dict(rows=0), dict(k=0), dict(v=0), dict(code=5), dict(dtype=9), dict(n=-1),
                       dict(pool_rows=-1), dict(pool_rows=1 << 31), dict(k_stride=31), dict(v_stride=0), dict(kv=-2),
                       dict(dim=1 << 20), dict(page=0), dict(stride=100), dict(pool=(1 << 20) + 4), dict(n=1 << 33)],
    "nhs_attend_rows8": [dict(q=0), dict(pool=0), dict(rows=0), dict(out=0), dict(dtype=4), dict(code=2), dict(batch=0),
                         dict(n=0), dict(heads=0), dict(kv=0), dict(dim=0), dict(page=0), dict(heads=3),
                         dict(dim=1025), dict(n=(1 << 30) + 1), dict(pool_rows=-1), dict(pool_rows=1 << 31),
                         dict(stride=8), dict(pool=(1 << 20) + 2), dict(n=4096, ws=0), dict(n=4096, ws_bytes=16),
                         dict(n=4096, ws=(1 << 20) + 4)],
}


@pytest.mark.parametrize("name", BAD)
def test_the_library_refuses(name):
    for changed in BAD[name]:
        assert call(name, **changed) < 0, changed
        assert name.encode() in _hip.load(check_runtime=False).nhs_last_error()


def test_a_planted_mistake_is_seen():
    """check() on the oracle's own output with one code off by a step."""
    gen = torch.Generator().manual_seed(1)
    form = rk.Rows8(i8, 2, 16)
    pool = make_pool(form, 2, 4, gen, "cpu")
    q, rows = torch.randn(1, 4, 16, generator=gen), torch.tensor([[0, 5, 2]])
    out, tol = attend_oracle(form, q, pool, rows)
    check(out.float(), out, tol)
    # each code of row 5 in turn moves by one, the largest of its own kind
    form.codes(pool)[1, 1, 1] += torch.where(form.codes(pool)[1, 1, 1] > 0, -1, 1).to(i8)
    moved, _ = attend_oracle(form, q, pool, rows)
    with pytest.raises(AssertionError):
        check(moved.float(), out, tol)


# ---- appends (GPU) -----------------------------------------------------------------------------

SHAPES = [(8, 128), (4, 128), (2, 64), (2, 32), (1, 256), (3, 80), (5, 16), (1, 1), (3, 5), (2, 130), (1, 1024), (2, 300),
          (12, 48), (2, 96), (9, 112), (3, 192), (1, 240), (70, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("heads, dim", SHAPES)
def test_append_page(gpu, heads, dim, dtype, code):
    gen = torch.Generator().manual_seed(heads * dim)
    form = rk.Rows8(code, heads, dim)
    for P, parts in ((64, [64]), (32, [1, 8, 9, 10, 4]), (16, [15, 1]), (1, [1]), (100, [70, 29])):
        pool = torch.full((3, 2, P, form.row_bytes), 0xA5, dtype=torch.uint8, device=gpu)
        host = torch.full((2, 2, P, form.row_bytes), 0xA5, dtype=torch.uint8).pin_memory()
        alias = rk.MappedHost(host)
        summary, low, high = empty_page(form, dtype, gpu)
        at = 0
        for n in parts:
            wide = keys(gen, n, 3 * heads, dim, dtype=dtype).to(gpu)  # k and v as views of one projection
            k, v = wide[:, :heads], wide[:, heads:2 * heads]
            earlier = values(form, pool[1, 0, :at], exact=True).view(at, heads, dim)
            low0, high0 = low.cpu(), high.cpu()
            rk.append_page_8bit(k, v, pool, form, 1, at, alias, 1, summary, low, high)
            torch.cuda.synchronize()
            check_page(form, pool, 1, earlier, k, v, at, summary, low, high, low0, high0)
            at += n
        assert torch.equal(pool[1].cpu(), host[1])
        untouched = torch.ones_like(host[1], dtype=torch.bool)
        for span in (slice(0, heads * dim), slice(form.scales_at, form.scales_at + 4 * heads)):
            untouched[:, :at, span] = False
        assert bool((pool[1].cpu()[untouched] == 0xA5).all())
        assert bool((pool[[0, 2]] == 0xA5).all()) and bool((host[0] == 0xA5).all())


SPECIAL = [0.0, -0.0, 1e-30, -1e-40, 2.0 ** -126, 2.0 ** -80, 3e-24, 1.0, 126.5, 127.0, 0.5, 1.5, 2.5, -3.5, 447.9, 448.0,
           2.0 ** -10, 2.0 ** -9, 3 * 2.0 ** -10, 0.0078125, 17.0, 18.0, 19.0, 240.0, 3e38, -1e37]


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("count", [3, 40])
def test_append_special_values(gpu, dtype, code, count):
    """Zeros, subnormals, quotients on the borders of two codes (scale 1 or a
    power of two), the largest numbers, NaN and infinities (a slice of them
    reads as NaN, and its neighbours as if nothing were)."""
    gen = torch.Generator().manual_seed(3)
    form = rk.Rows8(code, 4, 64)
    top = LARGEST[code]
    x = torch.zeros(count, 4, 64)
    for t in range(count):
        scale = 2.0 ** ((t % 7) - 3)
        x[t, 0] = torch.tensor(SPECIAL)[torch.randint(0, len(SPECIAL) - 2, (64,), generator=gen)].clamp(-top, top) * scale
        x[t, 0, 5] = top * scale  # the scale is a power of two, so ties are ties
        x[t, 1] = torch.tensor(SPECIAL)[torch.randint(0, len(SPECIAL), (64,), generator=gen)]
        x[t, 2] = torch.randn(64, generator=gen) * 10.0 ** (t % 60 - 30) if t % 3 else 0.0
        x[t, 3] = torch.randn(64, generator=gen)
        if t % 2:
            x[t, 3, t % 64] = (math.nan, math.inf, -math.inf)[t % 3]
    if dtype == f16:
        x = torch.where(torch.isfinite(x), x.clamp(-65504, 65504), x)
    k, v = x.to(dtype).to(gpu), x.flip(0).to(dtype).to(gpu)
    pool = torch.zeros(1, 2, 64, form.row_bytes, dtype=torch.uint8, device=gpu)
    summary, low, high = empty_page(form, dtype, gpu)
    rk.append_page_8bit(k, v, pool, form, 0, 2, None, 0, summary, low, high)
    torch.cuda.synchronize()
    inf = torch.full((4, 64), math.inf)
    # -0 and subnormals in the bounds stay as given; the two earlier rows hold zeros
    kk = torch.where(k == 0, 0.0, k)
    check_page(form, pool, 0, torch.zeros(2, 4, 64), kk, v, 2, summary, low, high, inf, -inf)
    got = rk.read_rows_8bit(pool, form, torch.arange(2, 2 + count, device=gpu), f32)[0]
    odd = ~torch.isfinite(k).all(-1)
    assert torch.equal(got.isnan(), odd[..., None].expand_as(got).to(gpu))


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
def test_append_quotients_near_borders(gpu, code):
    """fp32 elements a step or two from the borders of neighbouring codes,
    for scales that are no powers of two: a quotient rounded to fp32 first
    would often fall on the border."""
    gen = torch.Generator().manual_seed(11)
    form = rk.Rows8(code, 16, 128)
    table = torch.arange(128, dtype=torch.float64) if code == i8 else E4M3
    middle = (table[1:] + table[:-1]) / 2
    top = torch.exp(torch.randn(64, 16, 1, generator=gen)).float()
    scale = (top.double() / LARGEST[code]).float().double()
    x = (middle[torch.randint(0, len(middle), (64, 16, 128), generator=gen)] * scale).float()
    x = (x.view(torch.int32) + torch.randint(-2, 3, x.shape, generator=gen, dtype=torch.int32)).view(torch.float32)
    x[..., 7] = top[..., 0]
    x = torch.where(x > top, top, x) * torch.where(torch.rand(x.shape, generator=gen) < 0.5, -1.0, 1.0)
    k = x.to(gpu)
    for count in (64, 4):
        pool = torch.zeros(1, 2, 64, form.row_bytes, dtype=torch.uint8, device=gpu)
        summary, low, high = empty_page(form, f32, gpu)
        rk.append_page_8bit(k[:count], k[:count], pool, form, 0, 0, None, 0, summary, low, high)
        torch.cuda.synchronize()
        inf = torch.full((16, 128), math.inf)
        check_page(form, pool, 0, torch.zeros(0, 16, 128), k[:count], k[:count], 0, summary, low, high, inf, -inf)


@pytest.mark.gpu
def test_page_appender(gpu):
    """A write over several pages as a cache makes it: the same pages as one
    append_page_8bit each."""
    gen = torch.Generator().manual_seed(5)
    form = rk.Rows8(e4m3, 4, 64)
    P, n = 16, 53
    k, v = keys(gen, n, 4, 64, dtype=bf16).to(gpu), keys(gen, n, 4, 64, dtype=bf16).to(gpu)
    pages, blocks = 4, [3, 0, 5, 1]
    got, want = [], []
    for out, several in ((got, True), (want, False)):
        pool = torch.zeros(6, 2, P, form.row_bytes, dtype=torch.uint8, device=gpu)
        host = torch.zeros(4, 2, P, form.row_bytes, dtype=torch.uint8).pin_memory()
        summary, low, high = (torch.stack([t] * 8).view(2, 4, 4, 64).contiguous() for t in empty_page(form, bf16, gpu))
        alias = rk.MappedHost(host)
        appender = rk.PageAppender(k, v, pool, alias, summary, low, high, form) if several else None
        for page in range(pages):
            first, count = page * P, min(P, n - page * P)
            if several:
                appender(first, count, blocks[page], 0, page, 4 + page)
            else:
                rk.append_page_8bit(k[first:first + count], v[first:first + count], pool, form, blocks[page], 0, alias,
                                    page, summary[1, page], low[1, page], high[1, page])
        torch.cuda.synchronize()
        out += [pool.cpu(), host, summary.cpu(), low.cpu(), high.cpu()]
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with pytest.raises(ValueError):
        appender = rk.PageAppender(k, v, pool, alias, summary, low, high, form)
        appender(0, 16, 6, 0, 0, 0)
    for bad in ((0, 16, -1, 0, 0, 0), (0, 16, 0, 0, 4, 0), (0, 16, 0, 0, 0, 8), (50, 4, 0, 0, 0, 0)):
        with pytest.raises(ValueError):
            appender(*bad)
    with pytest.raises(RuntimeError):
        appender(0, 16, 0, 1, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("heads, dim, P", [(8, 128, 64), (4, 128, 32), (2, 64, 16), (3, 80, 16), (2, 5, 4), (1, 1024, 8)])
def test_append_items(gpu, heads, dim, P, dtype, code):
    gen = torch.Generator().manual_seed(heads + dim)
    form = rk.Rows8(code, heads, dim)
    B, pages = 7, 3
    pool0 = make_pool(form, B * pages + 2, P, gen, "cpu")
    pool = pool0.to(gpu)
    host = torch.zeros(B * pages, 2, P, form.row_bytes, dtype=torch.uint8).pin_memory()
    blocks = torch.randperm(B * pages + 2, generator=gen)[:B * pages].view(B, pages).int()
    source = torch.randperm(B * pages, generator=gen).view(B, pages).int()
    lengths = torch.tensor([0, P, P - 1, 2 * P + P // 2, 3 * P - 1, 3 * P, 1])  # the sixth is beyond its tables
    blocks[6, 0] = -1  # a page that is not bound
    source[2, 0] = -1  # one without a host page
    summary, low, high = (torch.stack([t] * (B * pages)).view(B, pages, heads, dim) for t in empty_page(form, dtype, gpu))
    dev_blocks, dev_source, unused = blocks.to(gpu), source.to(gpu), torch.zeros(4, dtype=torch.int64, device=gpu)
    table = rk.layer_items([[dict(source=dev_source[b], resident=dev_blocks[b], hot=dev_blocks[b], tags=dev_blocks[b],
                                  lru=unused, minimum=low[b], maximum=high[b], summaries=summary[b], n_pages=pages)
                             for b in range(B)]], gpu)
    fused = keys(gen, B, 3 * heads, dim, dtype=dtype).to(gpu)
    k, v = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    rk.append_items_8bit(k, v, pool, form, rk.MappedHost(host), table[0], lengths.to(gpu))
    torch.cuda.synchronize()
    untouched = torch.ones(pool0.shape, dtype=torch.bool)
    inf = torch.full((heads, dim), math.inf)
    for b, length in enumerate(lengths.tolist()):
        page, within = divmod(length, P)
        if page >= pages or blocks[b, page] < 0:
            assert bool((summary[b] == 0).all()) and bool((low[b] == math.inf).all())
            continue
        block = int(blocks[b, page])
        earlier = values(form, pool0[block, 0, :within], exact=True)
        check_page(form, pool, block, earlier, k[b:b + 1], v[b:b + 1], within, summary[b, page], low[b, page],
                   high[b, page], inf, -inf)
        untouched[block, :, within] = False
        mirror = pool[block, :, within].cpu() if source[b, page] >= 0 else None
        if mirror is not None:
            wrote = torch.cat((mirror[:, :heads * dim], mirror[:, form.scales_at:form.scales_at + 4 * heads]), 1)
            got = host[int(source[b, page]), :, within]
            assert torch.equal(torch.cat((got[:, :heads * dim], got[:, form.scales_at:form.scales_at + 4 * heads]), 1),
                               wrote)
    assert torch.equal(pool.cpu()[untouched], pool0[untouched])


@pytest.mark.gpu
def test_append_refusals(gpu):
    form = rk.Rows8(i8, 2, 16)
    pool = torch.zeros(2, 2, 8, form.row_bytes, dtype=torch.uint8, device=gpu)
    k = torch.zeros(4, 2, 16, device=gpu)
    summary, low, high = empty_page(form, f32, gpu)
    host = rk.MappedHost(torch.zeros(2, 2, 8, form.row_bytes, dtype=torch.uint8).pin_memory())
    good = dict(k=k, v=k, pool=pool, form=form, block=0, within=0, host=host, host_page=0, summary=summary, minimum=low,
                maximum=high)
    rk.append_page_8bit(**good)
    other = rk.MappedHost(torch.zeros(2, 2, 8, 2 * form.row_bytes, dtype=torch.uint8).pin_memory())
    for change in (dict(k=k[:, :1]), dict(v=k[:2]), dict(k=k.half()), dict(minimum=low.half()), dict(summary=low.double()),
                   dict(block=2), dict(block=-1), dict(within=5), dict(within=-1), dict(host_page=2), dict(host_page=-1),
                   dict(host=other), dict(form=rk.Rows8(i8, 2, 32)), dict(form=rk.Rows8(torch.uint8, 2, 16)),
                   dict(pool=pool.view(torch.int8)), dict(pool=pool[:, :, ::2]), dict(k=k[:0], v=k[:0]),
                   dict(k=k.transpose(1, 2).contiguous().transpose(1, 2)), dict(k=k[:1].expand(4, 2, 16)),
                   dict(maximum=high[:1]), dict(k=k.double(), v=k.double()), dict(k=k.cpu())):
        with pytest.raises(ValueError):
            rk.append_page_8bit(**{**good, **change})
    items, lengths = torch.zeros(4, 9, dtype=torch.int64, device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu)
    for args in ((k, k, pool, form, None, items[:3], lengths), (k, k, pool, form, None, items, lengths.int()),
                 (k, k, pool, form, None, items[:, :8], lengths), (k, k[:3], pool, form, None, items, lengths),
                 (k, k, pool, form, other, items, lengths), (k, k, pool, form, None, items, lengths.cpu())):
        with pytest.raises(ValueError):
            rk.append_items_8bit(*args)
    rk.append_items_8bit(k[:0], k[:0], pool, form, None, items[:0], lengths[:0])  # nothing to do
    one = k[:1].as_strided((1, 2, 16), (1, 16, 1))  # the stride of a single token does not count
    rk.append_page_8bit(**{**good, "k": one, "v": one})


# ---- read back (GPU) -----------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("heads, dim", SHAPES)
def test_read_rows(gpu, heads, dim, dtype, code):
    gen = torch.Generator().manual_seed(heads + dim)
    form = rk.Rows8(code, heads, dim)
    for P, blocks, n, gap in ((16, 5, 1, 0), (64, 3, 200, 0), (7, 9, 63, 48), (1, 20, 37, 16), (32, 40, 1111, 0)):
        pool = make_pool(form, blocks, P, gen, gpu, gap)
        rows = torch.randint(-2, blocks * P + 2, (n,), generator=gen)
        k, v = rk.read_rows_8bit(pool, form, rows.to(gpu), dtype)
        inside = (rows >= 0) & (rows < blocks * P)
        for got, want in zip((k, v), held(form, pool, rows.clamp(0, blocks * P - 1))):
            want = torch.where(inside[:, None, None], want, 0.0).to(dtype)
            assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype, n", [(bf16, 24577), (f16, 26001), (f32, 12700)])
def test_read_rows_into_large_outputs(gpu, dtype, n, code):
    """Outputs above 96 MB, which are stored past the caches: the values of reads in parts, and read by the next kernel
    on the stream."""
    gen = torch.Generator().manual_seed(9)
    form, P = rk.Rows8(code, 8, 128), 16
    pool = make_pool(form, 9, P, gen, gpu)
    rows = torch.randint(-1, 9 * P + 1, (n,), generator=gen).to(gpu)
    for got, parts in zip(rk.read_rows_8bit(pool, form, rows, dtype),
                          zip(*(rk.read_rows_8bit(pool, form, x, dtype) for x in rows.split(5000)))):
        assert torch.equal(got, torch.cat(parts))


@pytest.mark.gpu
def test_read_rows_outputs_strides_and_refusals(gpu):
    gen = torch.Generator().manual_seed(2)
    form = rk.Rows8(e4m3, 4, 64)
    pool = make_pool(form, 4, 16, gen, gpu)
    rows = torch.randint(0, 64, (30,), generator=gen).to(gpu)
    want = rk.read_rows_8bit(pool, form, rows, bf16)
    apart = rows.repeat_interleave(2).view(30, 2)[:, 0]  # a stride of two
    assert all(torch.equal(a, b) for a, b in zip(rk.read_rows_8bit(pool, form, apart, bf16), want))
    assert all(torch.equal(a, b) for a, b in zip(rk.read_rows_8bit(pool, form, rows[:1].expand(5), bf16),
                                                 [x[:1].expand(5, 4, 64) for x in want]))
    both = torch.zeros(31, 2, 4, 64, dtype=bf16, device=gpu)
    got = rk.read_rows_8bit(pool, form, rows, bf16, out=(both[:30, 0], both[:30, 1]))
    assert got[0].data_ptr() == both.data_ptr()
    assert torch.equal(both[:30, 0], want[0]) and torch.equal(both[:30, 1], want[1]) and not both[30].any()
    odd = torch.zeros(30 * 257 + 1, dtype=bf16, device=gpu)[1:].as_strided((30, 4, 64), (257, 64, 1))  # no alignment
    rk.read_rows_8bit(pool, form, rows, bf16, out=(odd, both[:30, 1]))
    assert torch.equal(odd, want[0])
    k, v = rk.read_rows_8bit(pool, form, rows[:0], bf16)
    assert k.shape == v.shape == (0, 4, 64)
    k, v = rk.read_rows_8bit(pool[:0], form, rows, bf16)
    assert not k.any() and not v.any()
    a, b = want
    for args, kw in (((pool, form, rows.int(), bf16), {}), ((pool, form, rows[None], bf16), {}),
                     ((pool, form, rows, torch.float64), {}), ((pool, form, rows.cpu(), bf16), {}),
                     ((pool, rk.Rows8(e4m3, 4, 32), rows, bf16), {}), ((pool[:, :1], form, rows, bf16), {}),
                     ((pool, form, rows, bf16), dict(out=(a, a))), ((pool, form, rows, bf16), dict(out=(a,))),
                     ((pool, form, rows, bf16), dict(out=(a.half(), b))), ((pool, form, rows, bf16), dict(out=(a[:9], b))),
                     ((pool, form, rows, bf16), dict(out=(a.transpose(1, 2).contiguous().transpose(1, 2), b))),
                     ((pool, form, rows, bf16), dict(out=(torch.zeros(30, 8, 64, dtype=bf16, device=gpu)[:, ::2], b))),
                     ((pool, form, rows, bf16), dict(out=(a[:1].expand(30, 4, 64), b)))):
        with pytest.raises(ValueError):
            rk.read_rows_8bit(*args, **kw)


# ---- attention (GPU) -----------------------------------------------------------------------------

HEADS = [(32, 8, 128), (28, 4, 128), (16, 16, 128), (4, 2, 64), (14, 2, 64), (4, 2, 32), (8, 2, 256), (6, 2, 80),
         (5, 1, 8), (3, 3, 2), (2, 1, 1024), (40, 2, 128), (4, 4, 130), (1, 1, 128), (17, 1, 64), (6, 3, 1),
         (8, 4, 96), (6, 2, 112), (3, 1, 192), (4, 2, 240), (5, 5, 16), (6, 3, 48)]


def attend_case(gen, device, heads, kv, dim, code, dtype, B, N, P=16, scale=1.0, gap=0):
    form = rk.Rows8(code, kv, dim)
    blocks = -(-B * N // P) + 2
    pool = make_pool(form, blocks, P, gen, device, gap)
    rows = torch.randperm(blocks * P, generator=gen)[:B * N].view(B, N)
    q = (torch.randn(B, heads, dim, generator=gen) * scale).to(dtype).to(device)
    return form, pool, rows.to(device), q


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("heads, kv, dim", HEADS)
def test_attend(gpu, heads, kv, dim, dtype, code):
    gen = torch.Generator().manual_seed(heads * dim)
    for B, N, P in ((1, 1, 16), (2, 15, 16), (1, 33, 1), (3, 64, 64), (1, 65, 32), (2, 130, 7), (1, 700, 16), (5, 257, 64)):
        form, pool, rows, q = attend_case(gen, gpu, heads, kv, dim, code, dtype, B, N, P)
        got = rk.attend_8bit(q, pool, form, rows)
        assert got.dtype == dtype
        check(got, *attend_oracle(form, q, pool, rows))
        again = rk.attend_8bit(q, pool, form, rows)
        assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("heads, kv, dim", [(32, 8, 128), (14, 2, 64), (8, 2, 256), (4, 2, 32), (6, 2, 80), (6, 2, 40)])
@pytest.mark.parametrize("dtype", [bf16, f32])
def test_attend_masks(gpu, heads, kv, dim, dtype, code):
    """Masked rows anywhere, lists without a row, rows outside the pool, and
    NaN codes and scales in every row that no list names."""
    gen = torch.Generator().manual_seed(heads)
    for N in (5, 64, 96, 300, 1025):
        form, pool, rows, q = attend_case(gen, gpu, heads, kv, dim, code, dtype, 6, N)
        named = torch.zeros(pool.shape[0] * 16, dtype=torch.bool, device=gpu)
        gone = torch.rand(rows.shape, generator=gen).to(gpu)
        rows[0] = torch.where(gone[0] < 0.5, -1, rows[0])
        rows[1] = -1
        rows[2, 1:] = -7
        rows[3, :-1] = pool.shape[0] * 16  # just behind the pool
        rows[4] = torch.where(gone[4] < 0.9, 2 ** 40, rows[4])
        rows[5, N // 2:] = -1
        inside = rows[(rows >= 0) & (rows < len(named))]
        named[inside] = True
        view = pool.view(-1, 2, 16, form.row_bytes)
        dead = (~named).view(-1, 16).nonzero()
        view[dead[:, 0], :, dead[:, 1]] = 0xFF
        got = rk.attend_8bit(q, pool, form, rows)
        check(got, *attend_oracle(form, q, pool, rows))
        assert not got[1].any()
        per_head = rows[:, None].expand(-1, heads, -1).clone()
        per_head[0, 0] = -1
        per_head[2, :, 0] = inside[torch.randint(0, len(inside), (heads,), generator=gen).to(gpu)]
        check(rk.attend_8bit(q, pool, form, per_head), *attend_oracle(form, q, pool, per_head))


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("heads, kv, dim", [(32, 8, 128), (28, 4, 128), (4, 2, 64), (2, 1, 40)])
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
def test_attend_long_lists_and_sharp_scores(gpu, heads, kv, dim, dtype, code):
    gen = torch.Generator().manual_seed(9)
    for B, N, scale in ((1, 9000, 1.0), (2, 2048, 8.0), (16, 511, 0.0), (3, 1999, 3.0)):
        form, pool, rows, q = attend_case(gen, gpu, heads, kv, dim, code, dtype, B, N, 64, scale)
        check(rk.attend_8bit(q, pool, form, rows), *attend_oracle(form, q, pool, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("heads, kv, dim, B, N", [(16, 8, 64, 33, 1300), (8, 8, 128, 32, 1025), (8, 8, 32, 40, 2049),
                                                 (4, 4, 256, 66, 600), (8, 8, 96, 34, 1200), (4, 4, 160, 70, 520)])
def test_attend_large_batches(gpu, heads, kv, dim, B, N, dtype, code):
    """Enough (request, KV head) pairs that no list is split: waves go over
    several rounds of rows. Every fifth request has a shorter list, one none."""
    gen = torch.Generator().manual_seed(B)
    form, pool, rows, q = attend_case(gen, gpu, heads, kv, dim, code, dtype, B, N, 64)
    for b in range(0, B, 5):
        rows[b, N * b // B:] = -1
    check(rk.attend_8bit(q, pool, form, rows), *attend_oracle(form, q, pool, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv, dim", [(8, 2, 128), (4, 2, 64), (6, 2, 80), (6, 2, 72)])
def test_attend_strides_and_outputs(gpu, heads, kv, dim):
    gen = torch.Generator().manual_seed(4)
    form, pool, rows, q = attend_case(gen, gpu, heads, kv, dim, e4m3, bf16, 3, 150, 16, gap=32)
    want = rk.attend_8bit(q, pool, form, rows)
    check(want, *attend_oracle(form, q, pool, rows))
    wide = torch.zeros(3, heads, 2 * dim + 2, dtype=bf16, device=gpu)
    odd = wide[:, :, 1:dim + 1]  # rows that begin at odd elements
    odd.copy_(q)
    assert torch.equal(rk.attend_8bit(odd, pool, form, rows), want)
    apart = rows.repeat_interleave(3, 1)[:, ::3]
    assert apart.stride(1) == 3 and torch.equal(rk.attend_8bit(q, pool, form, apart), want)
    shared = rows[:1].expand(3, -1)
    assert torch.equal(rk.attend_8bit(q, pool, form, shared), rk.attend_8bit(q, pool, form, shared.contiguous()))
    out = torch.full((3, heads, 2 * dim + 2), 7.0, dtype=bf16, device=gpu)
    got = rk.attend_8bit(q, pool, form, rows, out=out[:, :, 1:dim + 1])
    assert got.data_ptr() == out[:, :, 1:].data_ptr() and torch.equal(got, want)
    assert bool((out[:, :, 0] == 7).all()) and bool((out[:, :, dim + 1:] == 7).all())
    assert not rk.attend_8bit(q, pool, form, rows[:, :0]).any()
    assert not rk.attend_8bit(q, pool[:0], form, rows).any()
    assert rk.attend_8bit(q[:0], pool, form, rows[:0]).shape == (0, heads, dim)
    backwards = pool.flip(0)
    assert torch.equal(rk.attend_8bit(q, backwards, form, (len(pool) - 1 - rows // 16) * 16 + rows % 16), want)


@pytest.mark.gpu
def test_attend_refusals(gpu):
    gen = torch.Generator().manual_seed(4)
    form, pool, rows, q = attend_case(gen, gpu, 8, 2, 64, i8, bf16, 2, 40)
    rk.attend_8bit(q, pool, form, rows)
    for args in ((q[0], pool, form, rows), (q, pool, form, rows[0]), (q, pool, form, rows.int()),
                 (q, pool, form, rows[:1]), (q, pool, form, rows[:, None].expand(2, 3, 40)), (q[:, :7], pool, form, rows),
                 (q[..., :32], pool, form, rows), (q, pool.view(torch.int8), form, rows), (q, pool[:, :, :-1], form, rows),
                 (q, pool, rk.Rows8(i8, 4, 64), rows), (q, pool, rk.Rows8(torch.uint8, 2, 64), rows),
                 (q.double(), pool, form, rows), (q, pool, form, rows.cpu()), (q.cpu(), pool, form, rows),
                 (q.transpose(1, 2).contiguous().transpose(1, 2), pool, form, rows),
                 (q, pool, form, rows, q[:1]), (q, pool, form, rows, q.half()), (q, pool, form, rows, q[:1].expand(2, 8, 64))):
        with pytest.raises(ValueError):
            rk.attend_8bit(*args)


@pytest.mark.gpu
def test_rows_beyond_four_gigabytes(gpu):
    """Offsets that pass 32 bits: the last blocks of a pool of 5 GB."""
    gen = torch.Generator().manual_seed(8)
    form, P = rk.Rows8(e4m3, 8, 128), 64
    blocks = (5 << 30) // (2 * P * form.row_bytes)
    pool = rk.pool_8bit(blocks, P, form, gpu)
    few = make_pool(form, 4, P, gen, gpu)
    pool[-4:] = few
    rows = torch.randperm(4 * P, generator=gen)[:200].to(gpu)
    far = rows + (blocks - 4) * P
    q = torch.randn(1, 32, 128, generator=gen).to(bf16).to(gpu)
    assert torch.equal(rk.attend_8bit(q, pool, form, far[None]), rk.attend_8bit(q, few, form, rows[None]))
    for a, b in zip(rk.read_rows_8bit(pool, form, far, bf16), rk.read_rows_8bit(few, form, rows, bf16)):
        assert torch.equal(a, b)
    k = keys(gen, 20, 8, 128, dtype=bf16).to(gpu)
    for target, block in ((pool, blocks - 1), (few, 3)):
        rk.append_page_8bit(k, k, target, form, block, 3, None, 0, *empty_page(form, bf16, gpu))
    assert torch.equal(pool[-1], few[3])


@pytest.mark.gpu
def test_streams_and_graphs(gpu):
    """The write, read and attention of one step: on another stream, from two
    graphs that are replayed on two streams at once, and replayed with new
    inputs, eager work between the replays."""
    gen = torch.Generator().manual_seed(6)
    form, P = rk.Rows8(i8, 4, 64), 16

    def make(seed):
        g = torch.Generator().manual_seed(seed)
        form_, pool, rows, q = attend_case(g, gpu, 16, 4, 64, i8, bf16, 3, 700, P)
        k = keys(g, P, 4, 64, dtype=bf16).to(gpu)
        return {"pool": pool, "rows": rows, "q": q, "k": k, "bounds": empty_page(form, bf16, gpu)}

    def step(s):
        rk.append_page_8bit(s["k"], s["k"], s["pool"], form, 1, 0, None, 0, *s["bounds"])
        out = rk.attend_8bit(s["q"], s["pool"], form, s["rows"])
        return (out, *rk.read_rows_8bit(s["pool"], form, s["rows"][0], bf16), *s["bounds"])

    states = [make(1), make(2)]
    expected = [[x.clone() for x in step(s)] for s in states]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(states[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, expected[0]))
    graphs, outs = [], []
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(s))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round_ in range(4):
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, expected):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        for i, s in enumerate(states):  # new inputs in the same buffers, the eager result beside them
            s["q"].copy_(torch.randn(s["q"].shape, generator=gen).to(bf16))
            s["k"].copy_(torch.randn(s["k"].shape, generator=gen).to(bf16))
            expected[i] = [x.clone() for x in step(s)]
