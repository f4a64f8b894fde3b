"""Attention over selected physical rows (reference nano_hisparse/attention.py:6-35).

The row lease resolves the selection and gathers the missed rows; the
attention itself is libnhs_hip.so's split-K GQA row kernel on the compute
stream. `backend` keeps the reference's argument (`auto|torch|triton`,
reference attention.py:8-9, cli.py:48, engine.py:30) plus "hip": on a GPU
cache every one of them runs the HIP kernel, so a caller that asks for the
reference's torch path or its Triton kernels gets the same masked softmax
over the same rows from the one GPU implementation (no second code path).
CPU caches compute only through a CPU kernel provider that a test harness
installs.
"""

import torch

BACKENDS = ("auto", "hip", "torch", "triton")


@torch.inference_mode()
def row_attention(query, cache, request_id, layer, topk, backend="auto"):
    if backend not in BACKENDS:
        raise ValueError("invalid attention backend")
    if query.ndim != 2 or query.shape[1] != cache.config.head_dim:
        raise ValueError("invalid query shape")
    if query.shape[0] % cache.config.kv_heads or query.device != cache.pool.device:
        raise ValueError("query GQA/device mismatch")
    if topk.head_columns is not None and topk.head_columns.shape[0] != query.shape[0]:
        raise ValueError("selection must have one row per query head")
    if backend == "triton" and not cache.storage.cuda:
        raise ValueError("Triton requires CUDA")
    with cache.resolve(request_id, layer, topk) as lease:
        rows = lease.plan.physical_rows
        if rows.ndim == 1:
            rows = rows[None, :].expand(query.shape[0], -1)
        if cache.storage.cuda:
            from . import row_kernels as kernels
        else:
            from .row_kernels import cpu_provider

            kernels = cpu_provider("row_attention")
        form = cache.storage.rows8
        if form is not None:
            shared = rows.stride(0) == 0  # a stride-0 expansion of one list
            return kernels.attend_8bit(query[None], cache.pool, form, (rows[0] if shared else rows)[None])[0]
        return kernels.attend_rows(query, cache.pool, rows, cache.config)


@torch.inference_mode()
def tree_row_attention(query, k, v, mask, cache, request_id, layer, topk, backend="auto"):
    """row_attention for the drafted nodes of a request (query [nodes,
    q_heads, head_dim]) over the rows of one selection that all nodes share
    and over the drafted keys and values k, v [nodes, kv_heads, head_dim]
    that mask [nodes] (int64, see row_kernels.tree_plan) lets each node see."""
    if backend not in BACKENDS:
        raise ValueError("invalid attention backend")
    cfg = cache.config
    if query.ndim != 3 or query.shape[2] != cfg.head_dim:
        raise ValueError("invalid query shape")
    if query.shape[1] % cfg.kv_heads or query.device != cache.pool.device:
        raise ValueError("query GQA/device mismatch")
    if k.shape != (len(query), cfg.kv_heads, cfg.head_dim) or v.shape != k.shape:
        raise ValueError("expected one K/V row per node")
    if topk.head_columns is not None:
        raise ValueError("a tree's nodes and heads share one selection")
    if backend == "triton" and not cache.storage.cuda:
        raise ValueError("Triton requires CUDA")
    if cache.storage.rows8 is not None and not query.dtype == k.dtype == v.dtype == cfg.dtype:
        raise ValueError("query, K and V dtype must match the cache")
    with cache.resolve(request_id, layer, topk) as lease:
        rows = lease.plan.physical_rows
        if cache.storage.cuda:
            from . import row_kernels as kernels
        else:
            from .row_kernels import cpu_provider

            kernels = cpu_provider("tree_row_attention")
        pool, page_size, dtype = cache.pool, cfg.page_size, query.dtype
        if cache.storage.rows8 is not None:
            pool, rows, page_size, query, k, v = _read_for_tree(kernels, cache, rows, query, k, v)
        out = kernels.tree_attention(query[None], pool, rows[None], k[None], v[None], mask[None], page_size)[0]
        return out.to(dtype)  # (over rows in 8 bits the output's one rounding)


def _read_for_tree(kernels, cache, rows, query, k, v):
    """What tree_attention takes of a cache whose rows are in 8 bits: the
    selected rows read back as a pool of one page, and the drafted keys and
    values rounded as the cache will round them when they are appended. All of
    it in fp32, where code * scale is what attend_8bit multiplies with: a
    token accepted from a draft then sees what it would have seen alone, in a
    16-bit model too (whose type would round every value once more, by up to
    half a step of its own)."""
    form, n = cache.storage.rows8, rows.numel()
    pool = torch.empty(1, 2, n, form.kv_heads, form.head_dim, dtype=torch.float32, device=k.device)
    kernels.read_rows_8bit(cache.pool, form, rows, torch.float32, out=(pool[0, 0], pool[0, 1]))
    own = torch.where(rows >= 0, torch.arange(n, device=rows.device), -1)
    return pool, own, n, query.float(), *kernels.round_8bit(k.float(), v.float(), form)
