"""The operators that verify drafted tokens, as cases that can be timed and compared.

A draft model (or a lookup in the text so far) proposes a tree of next tokens
per request; one pass of the model then checks all of them:

- plan: ancestor masks and positions of a batch of token trees
  (row_kernels.tree_plan);
- norm: per-head RMSNorm of queries and keys and their rotation by cos/sin
  rows looked up at each token's position (row_kernels.qk_norm_rope);
- tree: attention of every node over its request's selected pool rows and the
  node's own ancestors (row_kernels.tree_attention);
- logprobs: log probabilities of given tokens, the entropy and the most
  likely alternatives of every row of logits (row_kernels.token_logprobs).

With `own` false, run() computes the operators from elementary torch
operations in 32 bits; with it true, it makes the framework's calls. Head
shapes, vocabularies, page sizes and budgets are those of bench.py, tests/
and perf/cases.py.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS, THETA = 1e-6, 10000.0
NODES = 64  # most nodes of a tree


def listed():
    return [
        # one request's small draft over a short history of a small model: the smallest call
        _tree("tree-one", 1, 8, 4, 2, 64, 16, 8, 5, "fp16"),
        # eight requests' drafts over 32 selected pages of 64, as a serving step has them
        _tree("tree-b8", 8, 16, 32, 8, 128, 64, 32, 9, "bf16"),
        # one request's draft over a long history that is wholly selected
        _tree("tree-long", 1, 32, 32, 8, 128, 64, 512, 31, "bf16"),
        # the widest trees, group of seven, sixteen requests: matrix work counts beside the stream
        _tree("tree-wide", 16, 64, 28, 4, 128, 32, 128, 0, "bf16"),
        # an fp32 model with heads of 32 and an odd number of nodes
        _tree("tree-fp32", 2, 13, 4, 2, 32, 16, 33, 7, "fp32"),
        # one small tree: a launch
        _plan("plan-one", 1, 8),
        # the largest batch of the widest trees
        _plan("plan-b64", 64, NODES),
        # one request's next-token distribution, fp32 logits, as a serving step returns it
        _logprobs("logprobs-one", 1, 128256, 5, "fp32"),
        # the verified nodes of a batch, odd vocabulary, many alternatives
        _logprobs("logprobs-b128", 128, 32001, 20, "bf16"),
        # a prompt of 4000 tokens scored
        _logprobs("logprobs-prompt", 4000, 128256, 1, "bf16"),
        # the nodes of a small batch: a launch
        _norm("norm-nodes", 24, 28, 4, 128, "fp16"),
        # a long prompt's queries and keys
        _norm("norm-prompt", 16001, 32, 8, 128, "bf16"),
    ]


def draw(rng):
    """One more case of the ranges the listed ones stand for."""

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["tree"] * 5 + ["logprobs"] * 4 + ["norm"] * 2 + ["plan"])
    heads, kv, dim = rng.choice([(32, 8, 128), (28, 4, 128), (16, 4, 128), (4, 2, 64), (14, 2, 64), (4, 2, 32)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "tree":
        batch, page = size(1, 16), rng.choice([16, 32, 64])
        most = (65536 if dtype != "fp32" else 16384) // page
        pages = size(1, max(1, min(32768 // page, most // batch)))
        return _tree(None, batch, size(1, NODES), heads, kv, dim, page, pages, rng.randrange(page), dtype)
    if kind == "logprobs":
        vocab = size(256, 152064)
        return _logprobs(None, size(1, min(4000, 4000 * 128256 // (vocab * SIZE[dtype]))), vocab,
                         rng.choice([0, 1, 5, 20, 64]), dtype)
    if kind == "norm":
        return _norm(None, size(1, 16001 * 2 // SIZE[dtype]), heads, kv, dim, dtype)
    return _plan(None, size(1, 64), size(1, NODES))


def _case(name, **values):
    return dict(values, name=name) if name else values


def _tree(name, batch, nodes, heads, kv, dim, page, pages, pad, dtype):
    # pages * page selected rows per request, the last `pad` of them past the request's end (-1)
    return _case(name, kind="tree", batch=batch, nodes=nodes, heads=heads, kv=kv, dim=dim, page=page, pages=pages,
                 pad=pad, dtype=dtype)


def _plan(name, batch, nodes):
    return _case(name, kind="plan", batch=batch, nodes=nodes)


def _logprobs(name, rows, vocab, top, dtype):
    return _case(name, kind="logprobs", rows=rows, vocab=vocab, top=top, dtype=dtype)


def _norm(name, rows, heads, kv, dim, dtype):
    return _case(name, kind="norm", rows=rows, heads=heads, kv=kv, dim=dim, dtype=dtype)


# ---- inputs ---------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return _PREPARE[case["kind"]](case, gen)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _parents(batch, nodes, gen):
    """Random trees, int32 [batch, nodes]: node 0 follows the history (parent
    -1), every other node one of the nodes before it; where there are several
    trees, each of the others leaves up to a quarter of its last nodes absent
    (-2)."""
    index = torch.arange(nodes, device="cuda")
    at = (torch.rand(batch, nodes, generator=gen, device="cuda") * index).long()
    parents = torch.minimum(at, (index - 1).clamp(min=0))
    parents[:, 0] = -1
    kept = nodes - (torch.rand(batch, 1, generator=gen, device="cuda") * (nodes // 4 + 1)).long()
    kept[0] = nodes
    return torch.where(index < kept, parents, -2).int()


def _masks(parents):
    """Ancestor masks (int64, a bit per node, itself included; 0 where the
    node is absent) and depths of trees whose parents precede their nodes."""
    batch, nodes = parents.shape
    mask = torch.zeros(batch, nodes, dtype=torch.int64, device=parents.device)
    depth = torch.zeros_like(mask)
    for t in range(nodes):
        p = parents[:, t].long()
        above = p.clamp(0, max(t - 1, 0))[:, None]
        m, d = mask.gather(1, above)[:, 0], depth.gather(1, above)[:, 0]
        bit = torch.full_like(m, 1 << t if t < 63 else -(1 << 63))
        root, below = p == -1, (p >= 0) & (p < t) & (m != 0)
        mask[:, t] = torch.where(root, bit, torch.where(below, m | bit, 0))
        depth[:, t] = torch.where(below, d + 1, 0)
    return mask, depth


def _prepare_plan(c, gen):
    lengths = torch.randint(1, 131072 - NODES, (c["batch"],), generator=gen, device="cuda")
    return {"kind": "plan", "parents": _parents(c["batch"], c["nodes"], gen), "lengths": lengths}


def _prepare_tree(c, gen):
    t, B, P, n, T = DTYPES[c["dtype"]], c["batch"], c["page"], c["pages"], c["nodes"]
    Hq, Hkv, D = c["heads"], c["kv"], c["dim"]
    blocks = B * n + 3
    # the layout of a GPU cache's pool: three head slots between blocks
    block, pad = 2 * P * Hkv * D, 3 * D
    pool = torch.empty(blocks * (block + pad), dtype=t, device="cuda").as_strided(
        (blocks, 2, P, Hkv, D), (block + pad, P * Hkv * D, Hkv * D, D, 1))
    for at in range(0, blocks, 512):
        part = pool[at:at + 512]
        part.copy_(_randn(gen, *part.shape))
    order = torch.randperm(blocks, generator=gen, device="cuda")[: B * n].view(B, n, 1)
    rows = (order * P + torch.arange(P, device="cuda")).view(B, n * P)
    if c["pad"]:
        rows[:, n * P - c["pad"]:] = -1
    # q, k and v are views of one projection's rows
    fused = _randn(gen, B, T, (Hq + 2 * Hkv) * D, dtype=t)
    q, k, v = fused.split([Hq * D, Hkv * D, Hkv * D], 2)
    mask, _ = _masks(_parents(B, T, gen))
    return {"kind": "tree", "q": q.view(B, T, Hq, D), "k": k.view(B, T, Hkv, D), "v": v.view(B, T, Hkv, D),
            "pool": pool, "rows": rows, "mask": mask, "page": P}


def _prepare_logprobs(c, gen):
    t, R, V = DTYPES[c["dtype"]], c["rows"], c["vocab"]
    logits = torch.empty(R, V, dtype=t, device="cuda")
    step = max(1, (1 << 26) // V)
    for at in range(0, R, step):
        part = logits[at:at + step]
        # a language model's logits: a wide bulk and a few tokens far above it; every eighth row answers
        # within a grammar that forbids half of the vocabulary
        x = _randn(gen, *part.shape, scale=2.5)
        x += (torch.rand(part.shape, generator=gen, device="cuda") < 8 / V) * 10.0
        if at % 8 == 0:
            x[::8, V // 2:] = float("-inf")
        part.copy_(x)
    tokens = torch.randint(0, V // 2, (R,), generator=gen, device="cuda")
    return {"kind": "logprobs", "logits": logits, "tokens": tokens, "top": c["top"]}


def _prepare_norm(c, gen):
    t, n, Hq, Hkv, D = DTYPES[c["dtype"]], c["rows"], c["heads"], c["kv"], c["dim"]
    fused = _randn(gen, n, (Hq + 2 * Hkv) * D, dtype=t, scale=1.5)
    q, k, _ = fused.split([Hq * D, Hkv * D, Hkv * D], 1)
    table = torch.arange(32768, device="cuda").double()[:, None] * _inv_freq(D)
    return {"kind": "norm", "q": q.view(n, Hq, D), "k": k.view(n, Hkv, D),
            "q_weight": 1 + _randn(gen, D, scale=0.2).to(t), "k_weight": 1 + _randn(gen, D, scale=0.2).to(t),
            "cos": table.cos().to(t), "sin": table.sin().to(t),
            "positions": torch.randint(0, 32768, (n,), generator=gen, device="cuda")}


def _inv_freq(dim):
    return THETA ** (-torch.arange(0, dim, 2, device="cuda").double() / dim)


_PREPARE = {"tree": _prepare_tree, "plan": _prepare_plan, "logprobs": _prepare_logprobs, "norm": _prepare_norm}


# ---- one pass -------------------------------------------------------------------------------


def run(s):
    return (_OWN if own else _PLAIN)[s["kind"]](s)


_kernels = None


def _rk():
    global _kernels
    if _kernels is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "nano-hisparse_amd"))
        from nano_hisparse import row_kernels

        _kernels = row_kernels
    return _kernels


def _own_tree(s):
    return _rk().tree_attention(s["q"], s["pool"], s["rows"], s["k"], s["v"], s["mask"], s["page"])


def _own_plan(s):
    return _rk().tree_plan(s["parents"], s["lengths"])


def _own_logprobs(s):
    r = _rk().token_logprobs(s["logits"], s["tokens"], s["top"])
    return {"logprobs": r.logprobs, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}


def _own_norm(s):
    return _rk().qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], EPS, s["cos"], s["sin"], s["positions"])


_OWN = {"tree": _own_tree, "plan": _own_plan, "logprobs": _own_logprobs, "norm": _own_norm}


# ---- the plain forms: elementary operations, 32 bits, one rounding at the end -------------------


def _bits(mask, nodes):
    """bool [..., nodes]: the bits of int64 words."""
    return ((mask[..., None] >> torch.arange(nodes, device=mask.device)) & 1).bool()


def _plain_tree(s):
    q, pool, rows, mask, P = s["q"], s["pool"], s["rows"], s["mask"], s["page"]
    B, T, Hq, D = q.shape
    Hkv = pool.shape[3]
    g = Hq // Hkv
    outs = []
    for b in range(B):
        r = rows[b]
        at = r.clamp(min=0)
        keys = torch.cat((pool[at // P, 0, at % P], s["k"][b])).float()  # [N + T, Hkv, D]
        values = torch.cat((pool[at // P, 1, at % P], s["v"][b])).float()
        seen = torch.cat(((r >= 0).expand(T, -1), _bits(mask[b], T)), 1) & (mask[b] != 0)[:, None]  # [T, N + T]
        kh = keys.permute(1, 2, 0).contiguous()  # [Hkv, D, N + T]
        vh = values.permute(1, 0, 2).contiguous()
        qh = q[b].float().view(T, Hkv, g, D).permute(1, 0, 2, 3).reshape(Hkv, T * g, D)
        scores = torch.matmul(qh, kh).view(Hkv, T, g, -1) * D ** -0.5
        scores = scores.masked_fill(~seen[None, :, None, :], float("-inf"))
        top = scores.amax(-1, keepdim=True)
        w = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
        total = w.sum(-1, keepdim=True)
        w = (w / torch.where(total > 0, total, 1.0)).view(Hkv, T * g, -1)
        out = torch.matmul(w, vh).view(Hkv, T, g, D).permute(1, 0, 2, 3).reshape(T, Hq, D)
        outs.append(out.to(q.dtype))
    return torch.stack(outs)


def _plain_plan(s):
    mask, depth = _masks(s["parents"])
    return mask, torch.where(mask != 0, s["lengths"][:, None] + depth, 0)


def _plain_logprobs(s):
    logits, tokens, top = s["logits"], s["tokens"], s["top"]
    R, V = logits.shape
    parts = []
    step = max(1, (1 << 26) // V)
    for at in range(0, R, step):
        x = logits[at:at + step].float()
        m = x.amax(1, keepdim=True)
        e = torch.exp(x - m)
        total = e.sum(1, keepdim=True)
        log_total = torch.log(total)
        shifted = x - m
        entropy = log_total[:, 0] - (e * torch.where(e > 0, shifted, 0.0)).sum(1) / total[:, 0]
        chosen = shifted.gather(1, tokens[at:at + step, None])[:, 0] - log_total[:, 0]
        if top:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        else:
            order = tokens.new_empty(len(x), 0)
        parts.append((chosen, entropy, order, shifted.gather(1, order) - log_total))
    chosen, entropy, ids, values = (torch.cat(p) for p in zip(*parts))
    return {"logprobs": chosen, "entropy": entropy, "top_ids": ids, "top_logprobs": values}


def _plain_norm(s):
    cos, sin = (s[name][s["positions"]].float()[:, None, :] for name in ("cos", "sin"))

    def one(x, weight):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        lo, hi = x.chunk(2, -1)
        return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)

    return (one(s["q"], s["q_weight"]).to(s["q"].dtype), one(s["k"], s["k_weight"]).to(s["k"].dtype))


_PLAIN = {"tree": _plain_tree, "plan": _plain_plan, "logprobs": _plain_logprobs, "norm": _plain_norm}


# ---- the least that a pass has to move and compute ----------------------------------------------


def work(case):
    c = case
    if c["kind"] == "plan":
        return {"bytes": c["batch"] * (c["nodes"] * (4 + 8 + 8) + 8), "flops": c["batch"] * c["nodes"] * 6}
    if c["kind"] == "tree":
        e, B, T = SIZE[c["dtype"]], c["batch"], c["nodes"]
        n = c["pages"] * c["page"]
        valid = n - c["pad"]
        moved = B * (valid * 2 * c["kv"] * c["dim"] * e + 8 * n + T * (2 * c["heads"] + 2 * c["kv"]) * c["dim"] * e
                     + 8 * T)
        return {"bytes": moved, "flops": 4 * B * T * c["heads"] * c["dim"] * (valid + T // 2)}
    if c["kind"] == "logprobs":
        R, V = c["rows"], c["vocab"]
        return {"bytes": R * (V * SIZE[c["dtype"]] + 8 + 4 + 4 + 12 * c["top"]), "flops": 5 * R * V}
    e, n, heads = SIZE[c["dtype"]], c["rows"], c["heads"] + c["kv"]
    # q and k in and out; each token's cos and sin rows; its position
    return {"bytes": n * (2 * heads * c["dim"] * e + c["dim"] * e + 8), "flops": 9 * n * heads * c["dim"]}


# ---- the operators' definitions in 64 bits --------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](case, s)


def _exact_plan(c, s):
    parents, lengths = s["parents"].tolist(), s["lengths"].tolist()
    masks, positions = [], []
    for tree, length in zip(parents, lengths):
        words, places = [], []
        for t in range(len(tree)):
            path, at = [], t
            while at >= 0:
                path.append(at)
                up = tree[at]
                at = up if -1 <= up < at else -2
            word = sum(1 << j for j in path) if at == -1 else 0
            words.append(word - (1 << 64) if word >> 63 else word)
            places.append(length + len(path) - 1 if word else 0)
        masks.append(words)
        positions.append(places)
    return torch.tensor(masks, device="cuda"), torch.tensor(positions, device="cuda")


def _exact_tree(c, s):
    q = s["q"].double()
    B, T, Hq, D = q.shape
    group = Hq // c["kv"]
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device="cuda")
    flat_k, flat_v = s["pool"][:, 0], s["pool"][:, 1]
    for b in range(B):
        rows = s["rows"][b]
        rows = rows[rows >= 0]
        block, inside = rows // c["page"], rows % c["page"]
        words = s["mask"][b].tolist()
        for kv in range(c["kv"]):
            key = flat_k[block, inside, kv].double()
            value = flat_v[block, inside, kv].double()
            heads = slice(kv * group, (kv + 1) * group)
            past = torch.mm(q[b, :, heads].reshape(T * group, D), key.t().contiguous()) / math.sqrt(D)
            own_k, own_v = s["k"][b, :, kv].double(), s["v"][b, :, kv].double()
            drafted = torch.mm(q[b, :, heads].reshape(T * group, D), own_k.t().contiguous()) / math.sqrt(D)
            allowed = torch.tensor([[bool(w >> j & 1) for j in range(T)] for w in words], device="cuda")
            drafted.masked_fill_(~allowed.repeat_interleave(group, 0), -math.inf)
            weights = torch.softmax(torch.cat((past, drafted), 1), 1)
            mixed = torch.mm(weights, torch.cat((value, own_v)))
            out[b, :, heads] = mixed.view(T, group, D)
        absent = [t for t, w in enumerate(words) if w == 0]
        out[b, absent] = 0.0
    return out


def _exact_logprobs(c, s):
    chosen, entropy, ids, values = [], [], [], []
    for row, token in zip(s["logits"].split(max(1, (1 << 25) // c["vocab"])),
                          s["tokens"].split(max(1, (1 << 25) // c["vocab"]))):
        x = row.double()
        logs = x - torch.logsumexp(x, 1, keepdim=True)
        p = logs.exp()
        entropy.append(-(p * logs.clamp(min=-1e6)).sum(1))
        chosen.append(logs.gather(1, token[:, None])[:, 0])
        left, index = x.clone(), torch.arange(c["vocab"], device="cuda")
        found = []
        gone = torch.zeros_like(x, dtype=torch.bool)
        for _ in range(c["top"]):
            best = left.amax(1, keepdim=True)
            at = torch.where((left == best) & ~gone, index, c["vocab"]).amin(1, keepdim=True)
            found.append(at)
            left.scatter_(1, at, -math.inf)
            gone.scatter_(1, at, True)
        at = torch.cat(found, 1) if found else torch.empty(len(x), 0, dtype=torch.int64, device="cuda")
        ids.append(at)
        values.append(logs.gather(1, at))
    return {"logprobs": torch.cat(chosen), "entropy": torch.cat(entropy), "top_ids": torch.cat(ids),
            "top_logprobs": torch.cat(values)}


def _exact_norm(c, s):
    half = c["dim"] // 2
    cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
    outs = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        y = y / (y.pow(2).sum(-1, keepdim=True) / c["dim"] + EPS).sqrt() * w.double()
        z = torch.complex(y[..., :half], y[..., half:]) * torch.complex(cos, sin)[:, None, :]
        outs.append(torch.cat((z.real, z.imag), -1))
    return tuple(outs)


_EXACT = {"tree": _exact_tree, "plan": _exact_plan, "logprobs": _exact_logprobs, "norm": _exact_norm}
