"""A cache whose rows are held in 8 bits (CacheConfig(storage_dtype=)): appends,
mirrors and residency, attention through the cache, batched and captured
decode, drafted tokens and the engine. On the CPU the kernels are computed in
64 bits from the bytes (test_rows_8bit's oracles), on a GPU by libnhs_hip.so.
Attention tolerances are those of test_rows_8bit."""

import math

import pytest
import torch

from nano_hisparse import row_kernels as rk
from nano_hisparse.batch_step import BatchTables, SparseDecodeBatch
from nano_hisparse.config import CacheConfig
from nano_hisparse.engine import Engine
from nano_hisparse.hybrid import HotConfig, HybridKVCache
from nano_hisparse.model import Model, ModelConfig
from nano_hisparse.selection import Selection, quest_selection
from test_rows_8bit import attend_oracle, check, held, keys, quantised, values
from test_tree_decode import TreeProvider

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
i8, e4m3 = torch.int8, torch.float8_e4m3fn
TINY = dict(hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
            vocab_size=64)


class Provider8(TreeProvider):
    def attend_8bit(self, query, pool, form, rows):
        return attend_oracle(form, query, pool, rows)[0].to(query.dtype)

    def read_rows_8bit(self, pool, form, rows, dtype, out):
        for got, want in zip(out, held(form, pool, rows.clamp(min=0))):
            got.copy_(torch.where(rows[:, None, None] >= 0, want, 0.0))

    def round_8bit(self, k, v, form):
        def rounded(x):
            codes, scale = quantised(x, form.code)
            return (codes.float() * scale.float()[..., None]).to(x.dtype)

        return rounded(k), rounded(v)


@pytest.fixture(params=["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def where(request):
    torch.set_num_threads(1)
    if request.param == "cpu":
        rk.set_cpu_provider(Provider8())
        yield "cpu"
        rk.set_cpu_provider(None)
        return
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield request.param


def cache_for(device, gpu_pages, hot, code, dtype=f32, page_size=4, heads=2, dim=8, host_pages=96):
    cfg = CacheConfig(gpu_pages=gpu_pages, host_pages=host_pages, page_size=page_size, kv_heads=heads, head_dim=dim,
                      dtype=dtype, device=device, storage_dtype=code)
    return HybridKVCache(cfg, hot)


def rounded(x, code):
    """(rows as the cache reads them in fp32) of x, by the oracle."""
    codes, scale = quantised(x.cpu(), code)
    return codes.float() * scale.float()[..., None]


def test_config():
    cfg = CacheConfig(kv_heads=8, head_dim=128, dtype=bf16, storage_dtype=e4m3)
    assert cfg.row_bytes == 2 * 1056 and cfg.rows8 == rk.Rows8(e4m3, 8, 128)
    assert CacheConfig(kv_heads=8, head_dim=128, dtype=bf16).rows8 is None
    for bad in (dict(storage_dtype=torch.uint8), dict(storage_dtype=bf16), dict(storage_dtype=i8, head_dim=2048),
                dict(storage_dtype=i8, dtype=torch.float64)):
        with pytest.raises(ValueError):
            CacheConfig(**bad)


@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_a_cache_keeps_rounded_rows(where, dtype, code):
    """Rows written by a prompt and one by one, in pages that move to the host
    and back: host rows, bounds and means, and the capacity accounts."""
    gen = torch.Generator().manual_seed(1)
    cache = cache_for(where, 14, HotConfig(8, 8, resident_window_pages=3), code, dtype, heads=2, dim=16)
    cache.reserve("a", 60, 2)
    k, v = keys(gen, 45, 2, 16, dtype=dtype), keys(gen, 45, 2, 16, dtype=dtype)
    k[20, 1, 3] = math.nan
    for layer in (0, 1):
        cache.write("a", layer, k[:30].to(where), v[:30].to(where))
        for t in range(30, 45):
            cache.write("a", layer, k[t:t + 1].to(where), v[t:t + 1].to(where))
    store = cache.storage
    store.synchronize()
    for layer in (0, 1):
        for got, x in zip(store.host_kv("a", layer), (k, v)):
            assert torch.equal(got.cpu().nan_to_num(nan=9e9), rounded(x, code).to(dtype).nan_to_num(nan=9e9))
        request = store.requests["a"]
        for page in range(12):
            rows = slice(4 * page, min(4 * page + 4, 45))
            for bound, how in ((request.minimum, "amin"), (request.maximum, "amax")):
                want = getattr(k[rows].float(), how)(0)
                assert torch.equal(bound[layer, page].cpu().float().nan_to_num(nan=9e9), want.nan_to_num(nan=9e9))
            codes, scale = quantised(k[rows], code)
            exact = (codes * scale[..., None]).mean(0)
            size = (codes * scale[..., None]).abs().mean(0)
            check(request.summaries[layer, page], exact, 2.0 ** -24 * exact.abs() + 2.0 ** -50 * size + 2.0 ** -149)
    cache.update_residency()
    cache.assert_invariants()
    row = 2 * rk.Rows8(code, 2, 16).row_bytes
    assert store.page_bytes == 4 * row and store.stats["d2h_bytes"] == 2 * 45 * row
    cache.release_request("a")
    cache.assert_invariants()


@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("dtype, heads, kv, dim, P", [(f32, 4, 2, 8, 4), (bf16, 8, 2, 64, 16), (f16, 7, 1, 128, 16),
                                                     (bf16, 4, 4, 80, 8)])
def test_attention_through_the_cache(where, dtype, heads, kv, dim, P, code):
    """Every step appends a token, selects and attends, with rows resident,
    hot and missed: against 64-bit attention over the rounded history."""
    gen = torch.Generator().manual_seed(7)
    cache = cache_for(where, 9, HotConfig(3 * P, 4 * P, resident_window_pages=4), code, dtype, P, kv, dim)
    cache.reserve("a", 10 * P + 16, 1)
    n = 10 * P + 3
    k, v = keys(gen, n + 10, kv, dim, dtype=dtype), keys(gen, n + 10, kv, dim, dtype=dtype)
    cache.write("a", 0, k[:n].to(where), v[:n].to(where))
    form = cache.storage.rows8
    history = torch.zeros(1, 2, n + 10, form.row_bytes, dtype=torch.uint8)
    for plane, x in enumerate((k, v)):
        codes, scale = quantised(x, code)
        form.codes(history)[0, plane] = codes.to(code)
        form.scales(history)[0, plane] = scale
    for t in range(n, n + 10):
        cache.write("a", 0, k[t:t + 1].to(where), v[t:t + 1].to(where))
        q = torch.randn(heads, dim, generator=gen).to(dtype)
        request = cache.storage.requests["a"]
        selection = quest_selection(q.to(where), request.minimum[0], request.maximum[0], t + 1, P, 3)
        if t % 3 == 0:  # a list per head
            pages = torch.randperm(t // P, generator=gen)[:2].tolist()
            lists = [[p * P + i for p in pages[h % 2:] for i in range(P - h % 3)] for h in range(heads)]
            selection = Selection.from_tokens(lists, t + 1, P, heads)
        got = cache.attention(q.to(where), "a", 0, selection)
        once = torch.full((heads, 3 * P), -1)
        for h, row in enumerate(selection.positions):
            once[h, :len(row)] = torch.tensor(row)
        check(got[None], *attend_oracle(form, q[None], history, once[None]))
    stats = cache.snapshot()["row_stats"]
    assert stats["misses"] > 0 and stats["hot_hits"] > 0 and stats["resident_hits"] > 0
    assert stats["h2d_bytes"] == stats["misses"] * 2 * form.row_bytes
    cache.assert_invariants()


@pytest.mark.parametrize("code", [i8, e4m3])
@pytest.mark.parametrize("top_k", [None, 2])
def test_generation_does_not_depend_on_what_is_resident(where, top_k, code):
    torch.manual_seed(31)
    model = Model(ModelConfig(**TINY)).eval().to(where)
    union = 28 if top_k is None else 8
    hot = HotConfig(union, union)
    results = []
    for budget in (64, hot.admission_blocks(4, 2)):
        engine = Engine(model, cache_for(where, budget, hot, code), top_k=top_k)
        engine.add_request("a", list(range(1, 18)), 8)
        engine.add_request("b", list(range(8, 30)), 6)
        results.append(engine.run())
    assert results[0] == results[1]
    other = Model(ModelConfig(**TINY)).eval().to(where, torch.float16 if where != "cpu" else torch.bfloat16)
    with pytest.raises(ValueError, match="dtype"):
        Engine(other, cache_for(where, 64, hot, code))


@pytest.mark.parametrize("code", [i8, e4m3])
def test_drafts_change_no_token(where, code):
    """Right and wrong drafts, accepted nodes appended: the tokens of plain
    decoding over the same cache."""
    torch.manual_seed(5)
    model = Model(ModelConfig(**TINY)).eval().to(where)
    hot = HotConfig(48, 48)

    def run(draft):
        engine = Engine(model, cache_for(where, 80, hot, code), draft=draft)
        engine.add_request("a", list(range(3, 20)), 20)
        return engine.run(), engine.requests["a"]

    plain, _ = run(None)
    tokens = list(plain["a"])

    def right(r):
        rest = tokens[len(r.generated):][:5]
        return rest, list(range(-1, len(rest) - 1))

    def mixed(r):
        rest = tokens[len(r.generated):][:3]
        wrong = [(t + 1) % 64 for t in rest]
        return rest + wrong, list(range(-1, len(rest) - 1)) + [-1] * len(wrong)

    for draft in (right, mixed):
        out, request = run(draft)
        assert out == plain
        assert request.accepted_count > 0


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
def test_batched_engine_steps(gpu, code):
    torch.manual_seed(9)
    model = Model(ModelConfig(**TINY)).eval().to(gpu)
    results = []
    for options in (dict(), dict(batch_decode=True), dict(batch_decode=True, graph=True),
                    dict(batch_decode=True, micro_batches=2)):
        engine = Engine(model, cache_for(gpu, 40, HotConfig(8, 16, resident_window_pages=4), code), top_k=2, **options)
        for i in range(3):
            engine.add_request(f"r{i}", list(range(1 + i, 15 + 3 * i)), 9)
        results.append(engine.run())
    assert all(r == results[0] for r in results)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
def test_graph_steps_are_the_eager_ones(gpu, code):
    """decode_batch(graph=True) replayed over steps that open pages and miss
    rows, eager work between them: bit-identical to eager steps on a twin."""
    torch.manual_seed(2)
    cfg = ModelConfig(hidden_size=512, intermediate_size=256, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=2, vocab_size=128)
    model = Model(cfg).eval().to(gpu, bf16)
    caches = [cache_for(gpu, 70, HotConfig(48, 64, resident_window_pages=3), code, bf16, 16, 2, 64) for _ in range(2)]
    ids = ["a", "b", "c"]
    for cache in caches:
        for i, name in enumerate(ids):
            cache.reserve(name, 150, 2)
            model.prefill([(7 * t + i) % 128 for t in range(90 + 13 * i)], cache, name)
    for step in range(20):
        tokens = [(step * 5 + i) % 128 for i in range(3)]
        eager = model.decode_batch(tokens, ids, caches[0], 3)
        replayed = model.decode_batch(tokens, ids, caches[1], 3, graph=True)
        assert torch.equal(eager, replayed)
    for cache in caches:
        cache.storage.synchronize()
        assert cache.snapshot()["row_stats"]["misses"] > 0
    # the bytes of a page's rows, not of the pad behind them
    for a, b in zip(caches[0].storage.host_kv("c", 1), caches[1].storage.host_kv("c", 1)):
        assert torch.equal(a, b)
    model.clear_decode_graphs()


@pytest.mark.gpu
@pytest.mark.parametrize("code", [i8, e4m3])
def test_sparse_step_over_rows_in_8_bits(gpu, code):
    """SparseDecodeBatch(form=): the gathered rows are the host's and the
    output is the attention over them."""
    gen = torch.Generator().manual_seed(4)
    B, Hq, Hkv, D, P, n_pages, top, H = 3, 8, 2, 64, 16, 24, 4, 64
    form = rk.Rows8(code, Hkv, D)
    hot_blocks = H // P
    host = torch.zeros(B * n_pages, 2, P, form.row_bytes, dtype=torch.uint8)
    k = keys(gen, B * n_pages, P, Hkv, D)
    for plane, x in enumerate((k, keys(gen, B * n_pages, P, Hkv, D))):
        codes, scale = quantised(x, code)
        form.codes(host)[:, plane] = codes.to(code)
        form.scales(host)[:, plane] = scale
    host = host.pin_memory()
    pool = torch.zeros(B * (hot_blocks + 3), 2, P, form.row_bytes, dtype=torch.uint8)
    resident = torch.full((B, n_pages), -1, dtype=torch.int32)
    hot = torch.empty(B, hot_blocks, dtype=torch.int32)
    for b in range(B):
        base = b * (hot_blocks + 3)
        hot[b] = torch.arange(base, base + hot_blocks, dtype=torch.int32)
        for i, page in enumerate((0, n_pages - 2, n_pages - 1)):
            resident[b, page] = base + hot_blocks + i
            pool[base + hot_blocks + i] = host[b * n_pages + page]
    pool = pool.to(gpu)
    tables = BatchTables(
        source=torch.arange(B * n_pages, dtype=torch.int32).view(B, n_pages).to(gpu), resident=resident.to(gpu),
        hot=hot.to(gpu), tags=torch.full((B, H), -1, dtype=torch.int32, device=gpu),
        lru=torch.arange(H, device=gpu).repeat(B, 1).contiguous(),
        minimum=k.amin(1).view(B, n_pages, Hkv, D).to(bf16).to(gpu), maximum=k.amax(1).view(B, n_pages, Hkv, D).to(bf16).to(gpu),
        lengths=torch.full((B,), n_pages * P, device=gpu))
    step = SparseDecodeBatch(pool, host, tables, P, top, form=form)
    for _ in range(3):
        q = torch.randn(B, Hq, D, generator=gen).to(bf16)
        out, result = step.step(q.to(gpu))
        torch.cuda.synchronize()
        rows = result.positions.cpu().long()
        flat = torch.where(rows >= 0, rows + torch.arange(B)[:, None] * n_pages * P, -1)
        check(out, *attend_oracle(form, q, host, flat))
        at = result.physical.cpu()
        assert bool(((at >= 0) == (rows >= 0)).all())
        there = at >= 0
        assert torch.equal(pool.cpu()[at[there] // P, :, at[there] % P], host[flat[there] // P, :, flat[there] % P])
    assert int(result.counts[:, 2].sum()) >= 0


@pytest.mark.gpu
def test_round_8bit(gpu):
    gen = torch.Generator().manual_seed(3)
    for code in (i8, e4m3):
        for heads, dim in ((2, 64), (3, 20)):
            form = rk.Rows8(code, heads, dim)
            k, v = keys(gen, 13, heads, dim, dtype=bf16), keys(gen, 13, heads, dim, dtype=bf16)
            for got, x in zip(rk.round_8bit(k.to(gpu), v.to(gpu), form), (k, v)):
                assert torch.equal(got.cpu(), rounded(x, code).to(bf16))
            assert rk.round_8bit(k[:0].to(gpu), v[:0].to(gpu), form)[0].shape == (0, heads, dim)
