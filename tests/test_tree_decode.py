"""Drafted tokens through the model and the engine: a tree's logits against
decoding each of its paths token by token, commits, greedy generation with
drafts of every quality, log probabilities of answers and texts, and models
with per-head norms. On the CPU the kernels are computed by plain expressions
in 64 bits (and the oracle), on a GPU by libnhs_hip.so."""

import pytest
import torch

import cpu_provider
from nano_hisparse import row_kernels as rk
from nano_hisparse.config import CacheConfig
from nano_hisparse.engine import Engine
from nano_hisparse.hybrid import HotConfig, HybridKVCache
from nano_hisparse.model import Model, ModelConfig
from nano_hisparse.selection import Selection

TINY = dict(hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=4,
            num_key_value_heads=2, vocab_size=64)
# the fp32 model's logits, from attention whose sums are ordered differently: 2^-24 * (about 50 sums and products of
# values up to 1 on the way through two layers)
ATOL = 3e-6


class TreeProvider(cpu_provider.OracleProvider):
    def tree_plan(self, parents, lengths):
        masks, positions = [], []
        for tree, length in zip(parents.tolist(), lengths.tolist()):
            paths = []
            for t, p in enumerate(tree):
                paths.append((paths[p] if p >= 0 else []) + [t])
            words = [sum(1 << j for j in path) for path in paths]
            masks.append([w - (1 << 64) if w >> 63 else w for w in words])
            positions.append([length + len(path) - 1 for path in paths])
        return torch.tensor(masks), torch.tensor(positions)

    def tree_attention(self, query, pool, rows, k, v, mask, page_size):
        g = query.shape[2] // pool.shape[3]
        out = torch.zeros_like(query)
        for b in range(len(query)):
            at = rows[b][rows[b] >= 0]
            past = [pool[at // page_size, i, at % page_size] for i in (0, 1)]
            for t in range(query.shape[1]):
                seen = ((mask[b, t] >> torch.arange(query.shape[1])) & 1).bool()
                keys, values = (torch.cat((p, d[b, seen])).double().repeat_interleave(g, 1)
                                for p, d in zip(past, (k, v)))
                w = ((query[b, t].double() * keys).sum(-1) / query.shape[-1] ** 0.5).softmax(0)
                out[b, t] = (w[..., None] * values).sum(0)
        return out

    def token_logprobs(self, logits, tokens, top):
        logs = logits.double().log_softmax(1)
        ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
        return rk.TokenLogprobs(logs.gather(1, tokens.view(len(logits), -1)).view(tokens.shape).float(),
                                -(logs.exp() * logs).sum(1).float(), ids, logs.gather(1, ids).float())


@pytest.fixture(params=["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def where(request):
    torch.set_num_threads(1)
    if request.param == "cpu":
        rk.set_cpu_provider(TreeProvider())
        yield "cpu"
        rk.set_cpu_provider(None)
        return
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield request.param


def tiny(where, seed=0, **change):
    torch.manual_seed(seed)
    model = Model(ModelConfig(**{**TINY, **change})).eval()
    for name, p in model.named_parameters():
        if "_norm" in name:  # weights that are not all one
            torch.nn.init.normal_(p, 1.0, 0.3)
    return model.to(where)


def cache_for(model, gpu_pages=64, hot=64, page=4, host_pages=128):
    cfg = CacheConfig(gpu_pages=gpu_pages, host_pages=host_pages, page_size=page, dtype=model.dtype,
                      kv_heads=model.config.num_key_value_heads, head_dim=model.config.head_dim,
                      device=str(model.device))
    return HybridKVCache(cfg, HotConfig(hot, hot))


def started(model, prompt, name="r", room=16, **kw):
    cache = cache_for(model, **kw)
    cache.reserve(name, len(prompt) + room, model.config.num_hidden_layers)
    logits = model.prefill(prompt, cache, name)
    return cache, logits


def paths_of(parents):
    paths = []
    for t, p in enumerate(parents):
        paths.append((paths[p] if p >= 0 else []) + [t])
    return paths


TREES = [([5], [-1]), ([5, 6, 7, 8], [-1, 0, 1, 2]), ([5, 6, 7, 8, 9, 6, 3], [-1, 0, 0, 1, 1, 2, 5]),
         ([5, 6, 7], [-1, -1, 0])]


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("tokens,parents", TREES)
@pytest.mark.parametrize("top_k", [None, 2])
def test_a_tree_s_logits_are_those_of_its_paths(where, tokens, parents, top_k, qk_norm):
    model = tiny(where, qk_norm=qk_norm)
    # 17 tokens: pages of 4 whose last one has room for the paths' first tokens, so that Quest ranks the same pages
    prompt = [(7 * i + 3) % 64 for i in range(17)]
    cache, _ = started(model, prompt)
    step = model.decode_tree(tokens, parents, "r", cache, top_k)
    assert step.logits.shape == (len(tokens), 64) and step.logits.dtype == torch.float32
    for node, path in enumerate(paths_of(parents)):
        if top_k is not None and len(path) > 1:
            continue  # deeper nodes choose pages by the first node's query
        one, _ = started(model, prompt)
        for t in path:
            logits = model.decode(tokens[t], "r", one, top_k)
        assert (step.logits[node] - logits).abs().max().item() <= ATOL
    assert cache.storage.requests["r"].lengths == [17, 17]  # nothing was written
    cache.assert_invariants()


@pytest.mark.parametrize("nodes", [[0], [0, 1, 3], [0, 2, 5, 6], []])
def test_a_committed_path_is_the_history_that_decoding_leaves(where, nodes):
    tokens, parents = TREES[2]
    model = tiny(where)
    prompt = list(range(10, 29))
    cache, _ = started(model, prompt)
    model.decode_tree(tokens, parents, "r", cache).commit(nodes)
    one, _ = started(model, prompt)
    for t in nodes:
        model.decode(tokens[t], "r", one)
    assert cache.storage.requests["r"].lengths == one.storage.requests["r"].lengths
    assert (model.decode(1, "r", cache) - model.decode(1, "r", one)).abs().max().item() <= ATOL
    assert (model.decode(2, "r", cache, 2) - model.decode(2, "r", one, 2)).abs().max().item() <= ATOL
    cache.assert_invariants()


def test_trees_and_commits_that_cannot_be(where):
    model = tiny(where)
    cache, _ = started(model, [1, 2, 3], room=2)
    for tokens, parents in (([], []), ([1], []), ([1, 2], [-1, 1]), ([1, 2], [-1, -2]), ([1], [0]),
                            ([1] * 65, [-1] + list(range(64)))):
        with pytest.raises(ValueError):
            model.decode_tree(tokens, parents, "r", cache)
    for bad in (64, -1):
        with pytest.raises(IndexError, match="vocabulary"):
            model.decode_tree([1, bad], [-1, 0], "r", cache)
    with pytest.raises(ValueError, match="selector"):
        model.decode_tree([1], [-1], "r", cache, selector="best")
    empty = cache_for(model)
    empty.reserve("r", 4, 2)
    with pytest.raises(ValueError, match="nonempty history"):
        model.decode_tree([1], [-1], "r", empty)
    step = model.decode_tree([1, 2, 3, 4], [-1, 0, 1, 0], "r", cache)
    for nodes in ([1], [0, 2], [0, 1, 3], [4], [-1], [0, 0], [0, 3, 1]):
        with pytest.raises(ValueError, match="a path"):
            step.commit(nodes)
    with pytest.raises(ValueError, match="reserved tokens"):
        step.commit([0, 1, 2])
    step.commit([0, 3])
    with pytest.raises(ValueError, match="has changed"):
        step.commit([0])
    cache.assert_invariants()


def test_tree_attention_of_the_cache_checks_its_arguments(where):
    model = tiny(where)
    cache, _ = started(model, list(range(9)))
    q, kv = torch.zeros(2, 4, 8, device=where), torch.zeros(2, 2, 8, device=where)
    mask = torch.tensor([1, 3], device=where)
    whole = Selection.from_pages([0, 1, 2], 9, 4, 4)
    assert cache.tree_attention(q, kv, kv, mask, "r", 0, whole).shape == (2, 4, 8)
    for bad in (dict(selection=Selection.from_pages([0], 4, 4, 4)), dict(selection=Selection.from_pages([0, 1, 2], 9, 4, 2)),
                dict(q=q[0]), dict(q=q[..., :4]), dict(k=kv[:1]), dict(v=kv[..., :4]), dict(backend="cutlass")):
        a = dict(dict(q=q, k=kv, v=kv, selection=whole, backend="auto"), **bad)
        with pytest.raises(ValueError):
            cache.tree_attention(a["q"], a["k"], a["v"], mask, "r", 0, a["selection"], a["backend"])
    cache.assert_invariants()


# ---- the engine --------------------------------------------------------------------------------


def generate(model, prompts, top_k=None, draft=None, limit=12, eos=None, logprobs=None, **kw):
    engine = Engine(model, cache_for(model, **kw), top_k=top_k, draft=draft, eos_token_id=eos, logprobs=logprobs)
    for name, prompt in prompts.items():
        engine.add_request(name, prompt, limit)
    engine.run()
    assert not engine.cache.storage.requests
    engine.cache.assert_invariants()
    return engine


PROMPTS = {"a": [(5 * i + 1) % 64 for i in range(15)], "b": [3] * 7}


@pytest.mark.parametrize("kind", ["right", "wrong", "tree", "late", "long", "none", "sometimes"])
def test_drafts_change_how_many_passes_are_made_and_no_token(where, kind):
    model = tiny(where, seed=2)
    plain = generate(model, PROMPTS)
    expected = {name: r.generated for name, r in plain.requests.items()}

    def draft(request):
        following = expected[request.request_id][len(request.generated):]
        if kind == "right":
            return following[:3], [-1, 0, 1][: len(following[:3])]
        if kind == "wrong":
            return [(following[0] + 1) % 64, 5], [-1, 0]
        if kind == "tree":  # two wrong branches beside the right one
            right = following[:4]
            return ([(following[0] + 9) % 64, *right, 7],
                    [-1, *[-1, 1, 2, 3][: len(right)], 0])
        if kind == "late":  # right, then wrong, then what would be right after it
            return [following[0], (following[min(1, len(following) - 1)] + 1) % 64, following[-1]], [-1, 0, 1]
        if kind == "long":  # beyond the request's length, and 63 tokens
            return (following + [1] * 63)[:63], list(range(-1, 62))
        if kind == "sometimes":
            return None if len(request.generated) % 2 else (following[:2], [-1, 0][: len(following[:2])])
        return [], []

    engine = generate(model, PROMPTS, draft=draft)
    for name, r in engine.requests.items():
        assert r.generated == expected[name]
        passes = {"right": 3, "wrong": 11, "tree": 3, "late": 6, "long": 1, "none": 11}.get(kind)
        if passes is not None:
            assert r.decode_count == passes
        assert r.decode_count + r.accepted_count == 11  # the first token is the prompt's
    assert all(r.drafted_count == 0 for r in plain.requests.values())


def test_the_end_of_a_text_inside_a_draft_ends_it(where):
    model = tiny(where, seed=3)
    expected = generate(model, PROMPTS).requests["a"].generated
    end = expected[4]
    cut = expected[: expected.index(end) + 1]

    def draft(request):
        return expected[len(request.generated): len(request.generated) + 6], list(range(-1, 5))

    engine = generate(model, {"a": PROMPTS["a"]}, draft=draft, eos=end)
    assert engine.requests["a"].generated == cut


def test_generation_with_drafts_under_pressure_of_the_pool(where):
    """Rows that were evicted to the host come back for a tree as they do for a token."""
    model = tiny(where, seed=5)
    prompts = {"a": [(11 * i + 2) % 64 for i in range(40)], "b": [(3 * i) % 64 for i in range(33)]}
    hot = HotConfig(64, 64)
    expected = generate(model, prompts).requests
    budget = hot.admission_blocks(4, 2)

    def draft(request):
        following = expected[request.request_id].generated[len(request.generated):][:2]
        return [1] + following, [-1, -1, 1][: 1 + len(following)]

    engine = generate(model, prompts, draft=draft, gpu_pages=budget)
    assert {n: r.generated for n, r in engine.requests.items()} == {n: r.generated for n, r in expected.items()}
    assert engine.cache.snapshot()["row_stats"]["misses"] > 0


def test_bad_proposals_leave_the_request_running(where):
    model = tiny(where)
    proposals = [([1], []), ([1], [0]), ([1], [-2]), ([99], [-1]), ([1] * 64, [-1] * 64)]

    def draft(request):
        return proposals.pop(0) if proposals else None

    engine = Engine(model, cache_for(model), draft=draft)
    engine.add_request("a", [1, 2, 3], 4)
    for _ in range(len(proposals)):
        with pytest.raises((ValueError, IndexError)):
            engine.step()
    assert engine.run() == {"a": generate(model, {"a": [1, 2, 3]}, limit=4).requests["a"].generated}


def test_what_followed_the_same_tokens_before_as_a_draft(where):
    """The loops that small random models fall into are found by looking them up."""

    def draft(request):
        text = request.prompt + request.generated
        for at in range(len(text) - 3, 0, -1):
            if text[at - 1: at + 1] == text[-2:]:
                tokens = text[at + 1: at + 6]
                return tokens, list(range(-1, len(tokens) - 1))

    model = tiny(where, seed=4)
    prompts = {"a": [7, 3, 9, 4] * 4, "b": [1, 2, 3]}
    plain = generate(model, prompts, limit=40)
    engine = generate(model, prompts, limit=40, draft=draft)
    for name, r in engine.requests.items():
        assert r.generated == plain.requests[name].generated
        assert r.decode_count + r.accepted_count == 39
    assert sum(r.drafted_count for r in engine.requests.values()) > 0


def test_drafts_may_cancel_requests(where):
    """Their own one and others, before and after them in the turn."""
    model = tiny(where, seed=2)
    prompts = {"a": [1, 2, 3], "b": [4, 5], "c": [6], "d": [7, 8]}
    expected = {n: r.generated for n, r in generate(model, prompts).requests.items()}
    plan = {("b", 2): ["b"], ("c", 3): ["a", "c"]}  # by whose draft, with how many tokens: who is cancelled

    def draft(request):
        for name in plan.pop((request.request_id, len(request.generated)), []):
            engine.cancel(name)
        return None

    engine = Engine(model, cache_for(model, gpu_pages=512, host_pages=512), draft=draft)
    for name, prompt in prompts.items():
        engine.add_request(name, prompt, 12)
    out = engine.run()
    assert not plan and out["d"] == expected["d"]
    assert len(out["b"]) == 2 and len(out["c"]) == 3 and len(out["a"]) < 12
    assert all(out[n] == expected[n][: len(out[n])] for n in prompts)
    assert not engine.cache.storage.requests


def test_a_commit_needs_the_request_that_the_step_was_of(where):
    model = tiny(where)
    cache, _ = started(model, [1, 2, 3])
    step = model.decode_tree([4], [-1], "r", cache)
    cache.release_request("r")
    cache.reserve("r", 19, model.config.num_hidden_layers)
    model.prefill([5, 6, 7], cache, "r")
    with pytest.raises(ValueError, match="history"):
        step.commit([0])


def test_engine_options_are_checked(where):
    model = tiny(where)
    for bad in (dict(logprobs=-1), dict(logprobs=65)):
        with pytest.raises(ValueError, match="logprobs"):
            Engine(model, cache_for(model), **bad)
    if where != "cpu":
        with pytest.raises(ValueError, match="request by request"):
            Engine(model, cache_for(model), top_k=2, batch_decode=True, draft=lambda r: None)


@pytest.mark.parametrize("drafts,qk_norm", [(False, False), (True, False), (True, True)])
def test_log_probabilities_of_the_generated_tokens(where, drafts, qk_norm):
    model = tiny(where, seed=7, qk_norm=qk_norm)
    expected = generate(model, PROMPTS).requests

    def draft(request):
        following = expected[request.request_id].generated[len(request.generated):][:3]
        return following, list(range(-1, len(following) - 1))

    engine = generate(model, PROMPTS, logprobs=4, draft=draft if drafts else None)
    for name, r in engine.requests.items():
        assert r.generated == expected[name].generated and len(r.logprobs) == len(r.generated)
        history = list(PROMPTS[name])
        for info, token in zip(r.logprobs, r.generated):
            logs = model.prefill(history).double().log_softmax(0).cpu()
            assert info.token == token and info.top[0][0] == token and len(info.top) == 4
            assert abs(info.logprob - logs[token].item()) <= 2 * ATOL and info.top[0][1] == info.logprob
            assert abs(info.entropy + (logs.exp() * logs).sum().item()) <= 5 * ATOL
            for (i, p), best in zip(info.top, logs.topk(4).values):
                assert abs(p - best.item()) <= 2 * ATOL and abs(p - logs[i].item()) <= 2 * ATOL
            history.append(token)
    assert all(not r.logprobs for r in expected.values())


@pytest.mark.parametrize("n", [2, 3, 40])
def test_score_is_the_log_probability_of_every_token(where, n, monkeypatch):
    from nano_hisparse import model as model_module

    model = tiny(where, seed=8, qk_norm=n == 40)
    text = [(13 * i + 5) % 64 for i in range(n)]
    got = model.score(text, top=3)
    assert got.logprobs.shape == (n - 1,) and got.top_ids.shape == (n - 1, 3)
    for i in range(1, n):
        logs = model.prefill(text[:i]).double().log_softmax(0)
        assert abs(got.logprobs[i - 1].item() - logs[text[i]].item()) <= 3 * ATOL
        assert abs(got.entropy[i - 1].item() + (logs.exp() * logs).sum().item()) <= 10 * ATOL
        assert (got.top_logprobs[i - 1].double() - logs.topk(3).values).abs().max().item() <= 3 * ATOL
    monkeypatch.setattr(model_module, "SCORE_ROWS", 7)
    again = model.score(text, top=3)
    assert all((a - b).abs().max().item() <= 3 * ATOL for a, b in zip(got, again))
    for bad in ([], [1]):
        with pytest.raises(ValueError):
            model.score(bad)
    with pytest.raises(IndexError):
        model.score([1, 64])


# ---- per-head norms ------------------------------------------------------------------------------


def test_a_model_with_per_head_norms_decodes_as_it_reads(where):
    model = tiny(where, seed=9, qk_norm=True)
    prompt = [(9 * i + 4) % 64 for i in range(12)]
    cache, logits = started(model, prompt)
    for token in (3, 60, 17):
        prompt.append(token)
        logits = model.decode(token, "r", cache)
        assert (logits - model.prefill(prompt)).abs().max().item() <= ATOL
    assert any("q_norm" in k for k in model.state_dict()) and not any("q_norm" in k for k in tiny(where).state_dict())
    other = tiny(where, seed=9)  # the seeded draws of the other parameters are the same
    for name, p in other.named_parameters():
        if "_norm" not in name:
            assert torch.equal(p, dict(model.named_parameters())[name])


def test_a_layer_normalises_every_head_and_then_rotates_it():
    model = tiny("cpu", seed=10, qk_norm=True)
    x = torch.randn(5, 32)
    layer = model.model.layers[0]
    q, k, v = model._project(layer, x, 7)
    h = layer.input_layernorm(x)
    for got, proj, norm, heads in ((q, "q_proj", "q_norm", 4), (k, "k_proj", "k_norm", 2)):
        y = getattr(layer.self_attn, proj)(h).view(5, heads, 8).double()
        y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * getattr(layer.self_attn, norm).weight.double()
        angle = torch.arange(7, 12).double()[:, None] * 10000.0 ** (-torch.arange(0, 8, 2).double() / 8)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        lo, hi = y.chunk(2, -1)
        assert (torch.cat((lo * c - hi * s, hi * c + lo * s), -1) - got.double()).abs().max() <= 1e-5


BIG = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
           vocab_size=512)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("qk_norm,hooked", [(False, False), (True, False), (True, True)])
def test_sixteen_bit_models_agree_over_their_paths(gpu, dtype, qk_norm, hooked):
    """Prompt pass, single tokens, trees, batches and graphs of one 16-bit
    model against the same model in fp32: each is within a few roundings of
    the logits (their size is about 1; 2^-8 of it a rounding in bf16, some
    twenty of them on the way, and two layers' amplification)."""
    model = tiny(gpu, seed=11, **BIG, qk_norm=qk_norm)
    exact = tiny(gpu, seed=11, **BIG, qk_norm=qk_norm)
    model = model.to(dtype)
    exact.load_state_dict({k: v.float() for k, v in model.state_dict().items()})
    if hooked:
        for layer in model.model.layers:
            if qk_norm:
                layer.self_attn.q_norm.register_forward_hook(lambda m, i, o: o)
    tol = 40 * torch.finfo(dtype).eps / 2
    prompt = [(31 * i + 3) % 512 for i in range(45)]
    cache, logits = started(model, prompt, page=16)
    reference, expected = started(exact, prompt, page=16)
    assert (logits - expected).abs().max().item() <= tol
    tokens, parents = [9, 200, 311, 7, 45], [-1, 0, 0, 1, 3]
    got = model.decode_tree(tokens, parents, "r", cache)
    want = exact.decode_tree(tokens, parents, "r", reference)
    assert (got.logits - want.logits).abs().max().item() <= tol
    got.commit([0, 1, 3])
    want.commit([0, 1, 3])
    assert (model.decode(77, "r", cache) - exact.decode(77, "r", reference)).abs().max().item() <= tol
    for graph in (False, True, True):
        a = model.decode_batch([5], ["r"], cache, 3, graph=graph)
        b = exact.decode(5, "r", reference, 3)
        assert (a[0] - b).abs().max().item() <= tol
    scored, wanted = model.score(prompt, 5), exact.score(prompt, 5)
    assert (scored.logprobs - wanted.logprobs).abs().max().item() <= 2 * tol
    cache.assert_invariants()
    model.clear_decode_graphs()


@pytest.mark.gpu
def test_batched_answers_carry_log_probabilities(gpu):
    model = tiny(gpu, seed=12, **BIG).to(torch.bfloat16)
    requests = {}
    for batched in (False, True):
        engine = Engine(model, cache_for(model, page=16), top_k=3, logprobs=2, batch_decode=batched, graph=batched)
        for name in ("a", "b", "c"):
            engine.add_request(name, [ord(name) + i for i in range(30)], 6)
        engine.run()
        for r in engine.requests.values():
            assert len(r.logprobs) == 6 and [i.token for i in r.logprobs] == r.generated
            assert all(i.top[0] == (i.token, i.logprob) and i.entropy > 0 for i in r.logprobs)
        requests[batched] = engine.requests
    for name, r in requests[True].items():
        assert r.generated[0] == requests[False][name].generated[0]
        assert abs(r.logprobs[0].logprob - requests[False][name].logprobs[0].logprob) <= 0.05
