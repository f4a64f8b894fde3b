"""Turns of the engine with drafts that do not go as planned: appends that
are refused. The text has to be that of plain decoding."""

import pytest
import torch

from nano_hisparse.engine import Engine
from nano_hisparse.selection import draft_selection
from nano_hisparse.storage import PageLease
from test_tree_decode import ATOL, PROMPTS, cache_for, generate, started, tiny, where  # noqa: F401 (where is a fixture)


def texts(engine):
    return {name: r.generated for name, r in engine.requests.items()}


def chain(tokens):
    """A draft of tokens that follow one another."""
    return list(tokens), list(range(-1, len(tokens) - 1))


def lease_of(engine, name, layers):
    store = engine.cache.storage
    return PageLease(store, [p for key, p in store.pages.items() if key[0] == name and key[1] in layers])


# ---- appends that are refused ------------------------------------------------------------------


@pytest.mark.parametrize("layers", [(0,), (1,), (0, 1)])
@pytest.mark.parametrize("drafted", [1, 3])
def test_a_turn_whose_append_is_refused_emits_nothing_and_is_made_again(where, layers, drafted):  # noqa: F811
    """The store refuses to append to a layer that a reader holds."""
    model = tiny(where, seed=2)
    expected = texts(generate(model, PROMPTS))["a"]
    engine = Engine(model, cache_for(model),
                    draft=lambda r: chain(expected[len(r.generated):][:drafted]))
    request = engine.add_request("a", PROMPTS["a"], 12)
    engine.step()
    while not request.finished:
        before = list(request.generated)
        if len(before) + drafted + 1 < 12:  # (a turn that ends the request appends nothing)
            lease = lease_of(engine, "a", layers)
            with pytest.raises(RuntimeError, match="lease"):
                engine.step()
            lease.release()
            assert request.generated == before and not request.logprobs
            lengths = engine.cache.storage.requests["a"].lengths
            assert lengths == [len(PROMPTS["a"]) + len(before) - 1] * 2
        engine.step()
        assert len(request.generated) > len(before)
    assert request.generated == expected
    engine.cache.collect(wait=True)
    assert not engine.cache.storage.requests
    engine.cache.assert_invariants()


def test_a_refused_commit_may_be_repeated(where):  # noqa: F811
    model = tiny(where)
    engine = Engine(model, cache_for(model))
    engine.add_request("r", [1, 2, 3], 12)
    engine.step()
    step = model.decode_tree([4, 5], [-1, 0], "r", engine.cache)
    lengths = list(engine.cache.storage.requests["r"].lengths)
    for layers in ((0,), (1,)):
        lease = lease_of(engine, "r", layers)
        with pytest.raises(RuntimeError, match="lease"):
            step.commit([0, 1])
        lease.release()
        assert engine.cache.storage.requests["r"].lengths == lengths
    step.commit([0, 1])
    assert engine.cache.storage.requests["r"].lengths == [n + 2 for n in lengths]
    with pytest.raises(ValueError, match="has changed"):
        step.commit([0])
    engine.cache.assert_invariants()


# ---- turns that raise ----------------------------------------------------------------------------


def failing(model, monkeypatch, name, times=None, after=False):
    """Makes the decode turns of one request raise (its first `times` ones),
    before they compute anything or after."""
    left = [times]
    for method in ("decode", "decode_tree"):
        real = getattr(model, method)

        def call(tokens, *a, real=real, tree=method == "decode_tree", **kw):
            of = a[1] if tree else a[0]
            fails = of == name and left[0] != 0
            if fails and left[0] is not None:
                left[0] -= 1
            if fails and not after:
                raise RuntimeError("planned")
            result = real(tokens, *a, **kw)
            if fails:
                raise RuntimeError("planned")
            return result

        monkeypatch.setattr(model, method, call)


@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("bad", ["a", "b", "c"])
def test_a_request_whose_turns_raise_holds_up_no_other(where, monkeypatch, bad, drafts):  # noqa: F811
    model = tiny(where, seed=2)
    prompts = {"a": [1, 2, 3], "b": [4, 5], "c": [6, 7, 8, 9]}
    expected = texts(generate(model, prompts, gpu_pages=512, host_pages=512))
    draft = (lambda r: chain(expected[r.request_id][len(r.generated):][:2])) if drafts else None
    engine = Engine(model, cache_for(model, gpu_pages=512, host_pages=512), draft=draft)
    for name, prompt in prompts.items():
        engine.add_request(name, prompt, 12)
    for _ in range(3):
        engine.step()  # every prompt is in
    at = len(engine.requests[bad].generated)
    failing(model, monkeypatch, bad)
    raised = 0
    for _ in range(25):
        try:
            engine.step()
        except RuntimeError as e:
            assert str(e) == "planned"
            raised += 1
    assert raised >= 5  # it is tried again and again
    for name in prompts:
        assert engine.requests[name].generated == (expected[name] if name != bad else expected[name][:at])
    monkeypatch.undo()
    assert engine.run() == expected
    engine.cache.assert_invariants()


def test_a_request_that_ends_while_it_is_read_takes_no_more_turns(where):  # noqa: F811
    """Its blocks cannot be released then; it is done all the same."""
    model = tiny(where, seed=2)
    expected = texts(generate(model, PROMPTS))
    engine = Engine(model, cache_for(model), draft=lambda r: chain(expected[r.request_id][len(r.generated):])
                    if r.request_id == "a" or len(r.generated) > 1 else None)
    for name, prompt in PROMPTS.items():
        engine.add_request(name, prompt, 12)
    engine.step()
    engine.step()
    assert engine.requests["a"].finished and not engine.requests["b"].finished
    lease = lease_of(engine, "b", (0,))
    with pytest.raises(RuntimeError, match="lease"):
        engine.step()
    assert engine.step() == [("b", token) for token in expected["b"][2:]]
    assert engine.step() == []
    assert texts(engine) == expected and not engine.running
    lease.release()
    engine.cache.release_request("b")
    engine.cache.assert_invariants()


@pytest.mark.parametrize("drafts", [False, True])
def test_a_turn_that_raises_after_it_has_appended_is_not_made_again(where, monkeypatch, drafts):  # noqa: F811
    """The last token's keys would be in the history twice. (A tree appends nothing before its commit.)"""
    model = tiny(where, seed=2)
    expected = texts(generate(model, PROMPTS))
    draft = (lambda r: chain(expected[r.request_id][len(r.generated):][:2])) if drafts else None
    engine = Engine(model, cache_for(model, gpu_pages=512, host_pages=512), draft=draft)
    for name, prompt in PROMPTS.items():
        engine.add_request(name, prompt, 12)
    for _ in range(2):
        engine.step()
    failing(model, monkeypatch, "a", times=1, after=True)
    with pytest.raises(RuntimeError, match="planned"):
        engine.step()
    at = len(engine.requests["a"].generated)
    out = engine.run()
    assert out["b"] == expected["b"]
    assert out["a"] == (expected["a"] if drafts else expected["a"][:at])
    if not drafts:
        engine.cancel("a")
    engine.cache.collect(wait=True)
    assert not engine.cache.storage.requests
    engine.cache.assert_invariants()


def test_a_cancelled_request_may_have_left(where, monkeypatch):  # noqa: F811
    """A layer of it written and the next one refused: the request waits for its cancellation."""
    model = tiny(where, seed=2)
    engine = Engine(model, cache_for(model))
    engine.add_request("a", PROMPTS["a"], 12)
    engine.step()
    lease = lease_of(engine, "a", (1,))
    with pytest.raises(RuntimeError, match="lease"):
        engine.step()
    lease.release()
    assert not engine.running and not engine.requests["a"].finished and engine.step() == []
    engine.cancel("a")
    assert engine.requests["a"].cancelled and not engine.cache.storage.requests
    engine.cache.assert_invariants()


def steps_until_done(engine, limit=200):
    """Every event that step() returns, whatever it raises in between."""
    events = []
    for _ in range(limit):
        if not engine.waiting and not engine.running:
            return events
        try:
            events += engine.step()
        except (RuntimeError, ValueError):
            pass
    raise AssertionError("not done")


@pytest.mark.parametrize("bad", ["a", "b", "c"])
def test_steps_that_raise_lose_no_events(where, bad):  # noqa: F811
    """Proposals that are refused now and then: what step() returns is still every token in order."""
    model = tiny(where, seed=2)
    prompts = {"a": [1, 2, 3], "b": [4, 5], "c": [6, 7, 8, 9]}
    expected = texts(generate(model, prompts, gpu_pages=512, host_pages=512))
    calls = dict.fromkeys(prompts, 0)

    def draft(r):
        calls[r.request_id] += 1
        if r.request_id == bad and calls[bad] % 3:
            return [1], [0]
        return chain(expected[r.request_id][len(r.generated):][: calls[r.request_id] % 3])

    engine = Engine(model, cache_for(model, gpu_pages=512, host_pages=512), draft=draft)
    for name, prompt in prompts.items():
        engine.add_request(name, prompt, 12)
    events = steps_until_done(engine)
    assert texts(engine) == expected
    for name in prompts:
        assert [token for of, token in events if of == name] == expected[name]


def test_events_are_returned_while_requests_fail(where, monkeypatch):  # noqa: F811
    """Two of three fail for good: the third one's tokens come out, its last ones too."""
    model = tiny(where, seed=2)
    prompts = {"a": [1, 2, 3], "b": [4, 5], "c": [6, 7, 8, 9]}
    expected = texts(generate(model, prompts, gpu_pages=512, host_pages=512))
    engine = Engine(model, cache_for(model, gpu_pages=512, host_pages=512))
    for name, prompt in prompts.items():
        engine.add_request(name, prompt, 12)
    failing(model, monkeypatch, "a")
    failing(model, monkeypatch, "c")
    events = []
    for _ in range(40):
        try:
            events += engine.step()
        except RuntimeError:
            pass
    assert [token for of, token in events if of == "b"] == expected["b"]
    assert [token for of, token in events if of != "b"] == [expected["a"][0], expected["c"][0]]


# ---- trees with the same text twice ----------------------------------------------------------------


@pytest.mark.parametrize("first", [0, 1, 2])
def test_candidates_that_begin_alike_are_all_followed(where, first):  # noqa: F811
    """Several chains under one root, the right one among them: as many tokens are accepted wherever it stands."""
    model = tiny(where, seed=2)
    expected = texts(generate(model, PROMPTS))

    def draft(r):
        right = expected[r.request_id][len(r.generated):][:4]
        wrong = [[*right[:1], (right[-1] + 1) % 64], [*right[:2], (right[-1] + 3) % 64, 5]]
        chains = [*wrong[:first], right, *wrong[first:]]
        tokens, parents = [], []
        for c in chains:
            for i, token in enumerate(c):
                parents.append(len(tokens) - 1 if i else -1)
                tokens.append(token)
        return tokens, parents

    engine = generate(model, PROMPTS, draft=draft)
    assert texts(engine) == expected
    for r in engine.requests.values():
        assert r.decode_count == 3 and r.accepted_count == 8  # 11 tokens after the prompt's, in turns of up to 5


def test_every_mix_of_equal_nodes_accepts_the_longest_way():
    """The walk alone, against every path of random trees of few tokens."""
    import random

    rng = random.Random(0)
    engine = Engine.__new__(Engine)
    for _ in range(500):
        n = rng.randrange(1, 16)
        engine.eos_token_id = rng.choice([None, 2])
        tree = [rng.randrange(3) for _ in range(n)]
        above = [-1] + [rng.randrange(t) for t in range(1, n)]
        choices = [(rng.randrange(3), None) for _ in range(n)]
        room = rng.randrange(1, 6)
        good = []
        for t in range(n):
            path = [t]
            while above[path[0]] >= 0:
                path.insert(0, above[path[0]])
            steps = list(zip(path, path[1:]))
            if len(path) <= room and all(tree[b] == choices[a][0] != engine.eos_token_id for a, b in steps):
                good.append(path)
        got = engine._accepted(tree, above, choices, room)
        assert got in good and len(got) == max(map(len, good))


# ---- page budgets ----------------------------------------------------------------------------------


@pytest.mark.parametrize("selector", ["quest", "mean"])
@pytest.mark.parametrize("top_k", [1, 2, 3, 4, 5, 6, 9])
@pytest.mark.parametrize("length", [1, 3, 4, 5, 8, 15, 16, 17, 18, 19, 20, 21, 24])
def test_the_first_node_reads_the_pages_that_decoding_would(where, length, top_k, selector):  # noqa: F811
    """On both sides of the pages' borders (4 tokens each), budgets below, at and above the pages there are."""
    model = tiny(where, seed=6)
    prompt = [(7 * i + 3) % 64 for i in range(length)]
    cache, _ = started(model, prompt)
    step = model.decode_tree([5, 9], [-1, 0], "r", cache, top_k, selector=selector)
    logits = model.decode(5, "r", cache, top_k, selector=selector)
    assert (step.logits[0] - logits).abs().max().item() <= ATOL
    cache.assert_invariants()


@pytest.mark.parametrize("selector", ["quest", "mean"])
@pytest.mark.parametrize("length", [15, 16, 17])
def test_a_history_that_fills_its_reservation_can_be_drafted_upon(where, length, selector):  # noqa: F811
    """No page, and no bounds, are reserved for the tree's first token. (Up to a border, decoding's logits come from a
    cache with room.)"""
    model = tiny(where, seed=6)
    prompt = [(7 * i + 3) % 64 for i in range(length)]
    for top_k in (1, 2, 3, 4, 5, 6):
        full, _ = started(model, prompt, room=0)
        roomy, _ = started(model, prompt)
        step = model.decode_tree([5], [-1], "r", full, top_k, selector=selector)
        logits = model.decode(5, "r", roomy, top_k, selector=selector)
        assert (step.logits[0] - logits).abs().max().item() <= ATOL
        with pytest.raises(ValueError, match="reserved tokens"):
            step.commit([0])


@pytest.mark.parametrize("selector", ["quest", "mean"])
@pytest.mark.parametrize("top_k", [1, 2, 3])
def test_drafts_that_are_never_accepted_change_no_token(where, top_k, selector):  # noqa: F811
    model = tiny(where, seed=2)
    for start in range(4):
        prompts = {"a": [(5 * i + 1 + start) % 64 for i in range(17 + start)]}

        def engine(draft):
            e = Engine(model, cache_for(model), top_k=top_k, draft=draft, selector=selector)
            for name, prompt in prompts.items():
                e.add_request(name, prompt, 14)
            e.run()
            return e

        expected = texts(engine(None))

        def wrong(r):
            following = expected[r.request_id][len(r.generated)]
            return [(following + 1) % 64, 5, (following + 2) % 64], [-1, 0, -1]

        drafted = engine(wrong)
        assert texts(drafted) == expected
        assert all(r.accepted_count == 0 and r.decode_count == 13 for r in drafted.requests.values())


def test_selections_for_a_token_that_is_not_there_yet(where):  # noqa: F811
    """Positions: those of the history in the pages that are kept, the token's own page among them while it is empty."""
    model = tiny(where, seed=6)
    q = torch.randn(4, 8, device=where)
    for length in (15, 16):
        cache, _ = started(model, list(range(length)))
        for selector in ("quest", "mean"):
            for top_k in (1, 2, 3, 4, 5, 6, None):
                s = draft_selection(cache, "r", 0, q, top_k, selector)
                assert s.length == length and s.heads == 4 and s.page_size == 4
                kept = 4 if top_k is None else min(top_k - (length == 16), 4)
                assert len(s.pages) == kept and len(s.positions[0]) == 4 * kept - (kept > 0 and length == 15)
                assert not kept or top_k == 1 or s.pages[0] == 0
                assert length == 16 or s.pages[-1] == 3
        for bad in (dict(top_k=0), dict(top_k=2, selector="best")):
            with pytest.raises(ValueError):
                draft_selection(cache, "r", 0, q, **bad)
