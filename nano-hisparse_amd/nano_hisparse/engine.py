"""Round-robin decode scheduler with host, index and device admission.

Reference: nano_hisparse/engine.py:12-143. Each step admits at most one
waiting prompt (prefill) and gives every running request one greedy decode
turn; requests are released when they finish or are cancelled.
"""

from __future__ import annotations

from collections import deque
from dataclasses import dataclass, field

from . import row_kernels as rk
from .config import CapacityError
from .model import Model


@dataclass
class TokenInfo:
    """A generated token's log probability, the entropy of the distribution
    that it was chosen from and the most likely tokens, (id, log probability)."""

    token: int
    logprob: float
    entropy: float
    top: list


@dataclass
class Request:
    request_id: str
    prompt: list
    max_new_tokens: int
    generated: list = field(default_factory=list)
    prefill_count: int = 0
    decode_count: int = 0
    finished: bool = False
    cancelled: bool = False
    logprobs: list = field(default_factory=list)  # a TokenInfo per generated token (Engine(logprobs=...))
    drafted_count: int = 0  # tokens that a draft proposed, and how many of them were accepted
    accepted_count: int = 0


class Engine:
    def __init__(self, model: Model, cache, top_k=None, backend="auto", eos_token_id=None, selector="quest",
                 batch_decode=False, micro_batches=1, graph=False, draft=None, logprobs=None):
        """batch_decode=True gives all running requests their decode turn in
        one Model.decode_batch call (GPU cache, Quest top_k; micro_batches=2
        pipelines two halves of the batch; graph=True replays each batch
        composition's step from a captured HIP graph); emission order and
        admission are unchanged.

        draft(request) may propose what follows a running request: (tokens,
        parents), a tree of up to 63 tokens whose parents are earlier tokens
        of the tree, or -1 for one that follows the request's last token. The
        request's decode turn then verifies the whole tree in one pass
        (Model.decode_tree) and emits every token of the path that greedy
        decoding takes, and the one after it; without a proposal (None or no
        tokens) it is an ordinary turn. With a top_k, a verified turn selects
        pages once, as an ordinary turn of the request's last token does; the
        tokens accepted after it may have read other pages than turns of
        their own would have selected.

        logprobs=n records a TokenInfo with the n most likely tokens for
        every generated token in its request's `logprobs`."""
        cfg, kv = model.config, cache.config
        if (cfg.num_key_value_heads, cfg.head_dim) != (kv.kv_heads, kv.head_dim):
            raise ValueError("model/cache head dimensions differ")
        if model.device != cache.pool.device or model.dtype != cache.pool.dtype:
            raise ValueError("model/cache dtype or device differ")
        if top_k is not None and top_k < 1:
            raise ValueError("top_k must be positive or None")
        self.model, self.cache, self.top_k, self.backend = model, cache, top_k, backend
        self.eos_token_id = eos_token_id
        self.selector = selector
        if batch_decode and (top_k is None or selector != "quest" or not cache.storage.cuda):
            raise ValueError("batched decode needs a GPU cache and the Quest selector with a top_k")
        self.batch_decode = batch_decode
        self.micro_batches = micro_batches
        self.graph = graph
        if graph and not batch_decode:
            raise ValueError("graph replay needs batch_decode")
        if draft is not None and batch_decode:
            raise ValueError("drafts are verified request by request, not with batch_decode")
        if logprobs is not None and not 0 <= logprobs <= min(rk.MAX_TOP_LOGPROBS, cfg.vocab_size):
            raise ValueError(f"logprobs must be None or 0 to {rk.MAX_TOP_LOGPROBS}, at most the vocabulary")
        self.draft = draft
        self.logprobs = logprobs
        self.requests: dict = {}
        self.waiting: deque = deque()
        self.running: deque = deque()
        self._events: list = []  # emitted in this step, or in steps that raised
        self._failed: set = set()  # requests whose turns raised since a step returned

    def add_request(self, request_id, prompt, max_new_tokens=16):
        if request_id in self.requests or not prompt or max_new_tokens < 1:
            raise ValueError("need a unique ID, nonempty prompt, and positive output length")
        if any(t < 0 or t >= self.model.config.vocab_size for t in prompt):
            raise ValueError("token outside model vocabulary")
        layers = self.model.config.num_hidden_layers
        total = len(prompt) + max_new_tokens
        pages = -(-total // self.cache.config.page_size)
        if pages * layers > self.cache.config.host_pages:
            raise CapacityError("request cannot fit even in an empty host pool")
        if self.cache.admission_blocks(layers) > self.cache.budget:
            raise CapacityError("request hot-region + tail footprint cannot fit the device pool")
        if self.cache.index_reservation_bytes(total, layers) > self.cache.config.index_budget_bytes:
            raise CapacityError("request index cannot fit even in an empty index budget")
        request = Request(request_id, list(prompt), max_new_tokens)
        self.requests[request_id] = request
        self.waiting.append(request)
        return request

    def _choose(self, logits):
        """(token, TokenInfo or None) for every row of logits [rows, vocab]."""
        chosen = logits.argmax(-1)
        if self.logprobs is None:
            return [(token, None) for token in chosen.tolist()]
        kernels = rk if logits.is_cuda else rk.cpu_provider("logprobs")
        info = kernels.token_logprobs(logits, chosen, self.logprobs)
        columns = (chosen, *info)
        return [(token, TokenInfo(token, logprob, entropy, list(zip(ids, values))))
                for token, logprob, entropy, ids, values in zip(*(c.tolist() for c in columns))]

    def _emit(self, request, choice):
        token, info = choice
        request.generated.append(token)
        self._events.append((request.request_id, token))
        if info is not None:
            request.logprobs.append(info)
        if token == self.eos_token_id or len(request.generated) >= request.max_new_tokens:
            request.finished = True
            self.cache.release_request(request.request_id, wait=False)

    def _decode(self, request):
        """One decode turn of a request."""
        proposal = self.draft(request) if self.draft is not None else None
        if request.finished:  # cancelled meanwhile
            return
        tokens, parents = proposal if proposal is not None else ((), ())
        if len(tokens) != len(parents):
            raise ValueError("a draft is a token list and a parent for each token")
        if not len(tokens):
            logits = self.model.decode(
                request.generated[-1], request.request_id, self.cache, self.top_k, self.backend,
                selector=self.selector,
            )
            request.decode_count += 1
            return self._emit(request, self._choose(logits[None])[0])
        tree = [request.generated[-1], *tokens]
        above = [-1, *(p + 1 for p in parents)]
        if min(above[1:]) < 0:
            raise ValueError("a drafted token's parent is -1 or a token before it")
        step = self.model.decode_tree(
            tree, above, request.request_id, self.cache, self.top_k, self.backend, selector=self.selector,
        )
        choices = self._choose(step.logits)
        room = request.max_new_tokens - len(request.generated)
        path = self._accepted(tree, above, choices, room)
        if len(path) < room and choices[path[-1]][0] != self.eos_token_id:  # the request goes on
            step.commit(path)  # before anything is emitted: an append may be refused
        request.decode_count += 1
        request.drafted_count += len(tokens)
        request.accepted_count += len(path) - 1
        for node in path:
            self._emit(request, choices[node])

    def _accepted(self, tree, above, choices, room):
        """The path of a verified tree that greedy decoding takes, of at most
        `room` nodes, up to the one after which the text ends. Among nodes
        that stand for the same text it is the one with the longest way on."""
        paths = [[0]]
        for t in range(1, len(tree)):
            way = paths[above[t]]
            taken = way and tree[t] == choices[above[t]][0] != self.eos_token_id and len(way) < room
            paths.append([*way, t] if taken else None)
        return max(filter(None, paths), key=len)

    def _admit(self, request):
        layers = self.model.config.num_hidden_layers
        total = len(request.prompt) + request.max_new_tokens
        try:
            self.cache.reserve(request.request_id, total, layers)
            return True
        except CapacityError:
            if self.running:
                return False  # retry after running requests progress
            if not self.cache.storage.retired:
                raise
            self.cache.collect(wait=True)  # idle: wait for retirements
            self.cache.reserve(request.request_id, total, layers)
            return True

    def step(self):
        """Admit at most one prompt, then one decode turn per running request
        (several tokens where a draft's were accepted). A request whose turn
        raises stays, behind the others, whose turns come first in the next
        step. If the turn had appended keys and values it cannot be made again
        and the request takes no more turns (cancel() releases it).

        Returns [(request_id, token)] in emission order, those of steps that
        raised before it among them; so that they are not kept for long, the
        step after one that raised leaves out the requests whose turns did.
        """
        self._turns()
        events, self._events = self._events, []
        self._failed = set()
        return events

    def _turns(self):
        self.cache.collect()
        if self.waiting and self._admit(self.waiting[0]):
            request = self.waiting.popleft()
            logits = self.model.prefill(request.prompt, self.cache, request.request_id)
            request.prefill_count += 1
            self._emit(request, self._choose(logits[None])[0])
            if not request.finished:
                self.running.append(request)
        if self.batch_decode and self.running:
            batch = list(self.running)
            self.running.clear()
            logits = self.model.decode_batch(
                [r.generated[-1] for r in batch], [r.request_id for r in batch], self.cache, self.top_k,
                micro_batches=self.micro_batches, graph=self.graph,
            )
            for request, choice in zip(batch, self._choose(logits)):
                request.decode_count += 1
                self._emit(request, choice)
                if not request.finished:
                    self.running.append(request)
            return
        others = {r.request_id for r in self.running} | {name for name, _ in self._events}
        left_out = self._failed if self._events and len(others) > 1 else ()
        for request in list(self.running):
            if request.finished:  # cancelled while another one's draft was made
                continue
            try:
                if request.request_id not in left_out:
                    self._decode(request)
            except BaseException:
                self._failed = self._failed | {request.request_id}
                raise
            finally:  # (a request whose turn raises goes behind the others too)
                if not request.cancelled:
                    self.running.popleft()
                if not request.finished and self._whole(request):
                    self.running.append(request)

    def _whole(self, request):
        """Whether a request's history is that of its tokens: every one but
        the last in every layer."""
        tokens = len(request.prompt) + len(request.generated) - 1
        stored = self.cache.storage.requests.get(request.request_id)
        return stored is not None and all(n == tokens for n in stored.lengths)

    def run(self):
        while self.waiting or self.running:
            self.step()
        self.cache.collect(wait=True)
        return {name: request.generated for name, request in self.requests.items()}

    def cancel(self, request_id):
        request = self.requests[request_id]
        if request.finished:
            return
        if request in self.waiting:
            self.waiting.remove(request)
        else:
            if request in self.running:
                self.running.remove(request)
            self.cache.release_request(request_id, wait=False)
        request.finished = request.cancelled = True
