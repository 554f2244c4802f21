"""A small continuous-batching server on the paged operators.

:class:`Sequences` is the host side: which tokens the next step takes in and where their keys and
values go. Every step it gives each running sequence one token and, in what is left of the step's
rows, one chunk of the oldest unfinished prompt. :class:`PagedServer` runs such a step through the
model: the projections of the batched ABI, and per layer ``paged_rope_append`` and
``paged_attention`` with the step's one plan; then ``logits_process`` and the argmax.

    server = PagedServer(DeviceWeights.load(model_dir), n_pages=4096)
    a = server.add(prompt, repetition=1.1)
    while server.running():
        for seq, token in server.step().items():
            ...  # server.remove(seq) once it has said what it had to
    server.remove(a)

A sequence runs until its page table (or the whole pool) is full; it then keeps its tokens, gives its pages back and
gets no more tokens. A step in which only prompts are taken in returns no tokens. When no sequence finds a page for its next
token, the youngest give theirs back, and are taken in again later, prompt and tokens.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np

from ._lib import call
from .paged import PagedPlan, logits_process, paged_attention, paged_rope_append, rope_inv_freq


@dataclass
class Sequence:
    prompt: list[int]
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: dict[int, float] = field(default_factory=dict)
    mask: np.ndarray | None = None  # int32 words, one bit per allowed token
    generated: list[int] = field(default_factory=list)
    cached: int = 0                 # positions whose keys and values are in the cache
    pages: list[int] = field(default_factory=list)

    def pending(self) -> int:
        return len(self.prompt) + len(self.generated) - self.cached

    def token(self, i: int) -> int:
        return self.prompt[i] if i < len(self.prompt) else self.generated[i - len(self.prompt)]


@dataclass
class Step:
    """One step's batch: sequence ids, their new tokens back to back, and the rows whose logits count."""
    ids: list[int]
    counts: list[int]
    tokens: list[int]
    outputs: list[tuple[int, int]]  # (row, id)


class Sequences:
    """Page accounting and the choice of each step's tokens; no device."""

    def __init__(self, n_pages: int, page_size: int, max_seqs: int, max_pages: int, chunk: int):
        self.page_size, self.max_seqs, self.max_pages, self.chunk = page_size, max_seqs, max_pages, chunk
        self.most = min(max_pages, n_pages) * page_size  # positions that one sequence can have
        self.free = list(range(n_pages - 1, -1, -1))
        self.live: dict[int, Sequence] = {}
        self._next = 0

    def add(self, seq: Sequence) -> int:
        if not seq.prompt:
            raise ValueError("an empty prompt")
        if len(self.live) == self.max_seqs:
            raise RuntimeError("every sequence slot is taken")
        if len(seq.prompt) > self.most:
            raise ValueError("the prompt is longer than a page table or the pool")
        self._next += 1
        self.live[self._next] = seq
        return self._next

    def _release(self, seq: Sequence) -> None:
        self.free += reversed(seq.pages)
        seq.pages = []

    def remove(self, i: int) -> None:
        self._release(self.live.pop(i))

    def running(self) -> list[int]:
        """The sequences that will still get tokens: those whose next position has a place."""
        return [i for i, seq in self.live.items() if seq.cached < self.most]

    def _grow(self, seq: Sequence, positions: int) -> bool:
        """Pages for this many positions, or no change and False."""
        need = -(-positions // self.page_size) - len(seq.pages)
        if need > len(self.free) or need + len(seq.pages) > self.max_pages:
            return False
        for _ in range(need):
            seq.pages.append(self.free.pop())
        return True

    def step(self) -> Step:
        """The next batch, not empty while a sequence is running. A sequence that finds no page sits the step out; if all
        would, the youngest lose theirs. The oldest alone always finds some, so that it comes to its end."""
        while True:
            out = self._choose()
            if out.ids or not self._preempt():
                return out

    def _preempt(self) -> bool:
        """Takes the pages of the youngest running sequence that has any, the oldest aside."""
        for i in reversed(self.running()[1:]):
            if self.live[i].pages:
                self._release(self.live[i])
                self.live[i].cached = 0
                return True
        return False

    def _choose(self) -> Step:
        out = Step([], [], [], [])

        def take(i, n):
            seq = self.live[i]
            if n <= 0 or not self._grow(seq, seq.cached + n):
                return False
            out.ids.append(i)
            out.counts.append(n)
            out.tokens += [seq.token(seq.cached + k) for k in range(n)]
            if seq.pending() == n:
                out.outputs.append((len(out.tokens) - 1, i))
            return True

        running = [(i, self.live[i]) for i in self.running()]
        for i, seq in running:
            if seq.pending() == 1:
                take(i, 1)
        for i, seq in running:
            if seq.pending() > 1 and take(i, min(seq.pending(), self.chunk)):
                break
        return out

    def commit(self, step: Step, tokens: list[int]) -> dict[int, int]:
        for i, n in zip(step.ids, step.counts):
            seq = self.live[i]
            seq.cached += n
            if seq.cached == self.most:  # at its end
                self._release(seq)
        done = {}
        for (_, i), t in zip(step.outputs, tokens):
            self.live[i].generated.append(t)
            done[i] = t
        return done


class PagedServer:
    """Greedy decoding of up to `max_seqs` sequences over a pool of `n_pages` pages per layer."""

    def __init__(self, weights, n_pages: int, page_size: int = 64, max_seqs: int = 32, max_positions: int | None = None,
                 chunk: int = 256, rope_kind: str = "plain", **rope):
        import torch
        self.torch, self.w, s = torch, weights, weights.shape
        self.shape = s
        max_pages = -(-(max_positions or s.max_position_embeddings) // page_size)
        self.seqs = Sequences(n_pages, page_size, max_seqs, max_pages, chunk)
        pool = (s.num_hidden_layers, n_pages, s.num_key_value_heads, page_size, s.head_dim)
        self.key_pages = torch.zeros(pool, dtype=torch.bfloat16, device="cuda")
        self.value_pages = torch.zeros_like(self.key_pages)
        freq, self.amplitude = rope_inv_freq(s.head_dim, s.rope_theta, rope_kind, **rope)
        self.inv_freq = torch.from_numpy(freq).cuda()
        heads = (s.num_attention_heads, s.num_key_value_heads, s.head_dim, page_size, n_pages, max_pages)
        # a step of decodes alone, and one with a chunk of a prompt: fixed numbers of rows, the last ones unused
        self.plans = {rows: PagedPlan(max_seqs, rows, q, *heads) for rows, q in ((max_seqs, 1), (max_seqs + chunk, chunk))}
        rows = max_seqs + chunk

        def rows_of(n, count=rows):
            return torch.zeros(count, n, dtype=torch.bfloat16, device="cuda")

        self.x, self.xb, self.act = rows_of(s.hidden_size), rows_of(s.hidden_size), rows_of(s.intermediate_size)
        self.q, self.att = rows_of(s.q_dim), rows_of(s.q_dim)
        self.k, self.v = rows_of(s.kv_dim), rows_of(s.kv_dim)
        self.last = rows_of(s.hidden_size, max_seqs)
        self.logits = rows_of(s.vocab_size, max_seqs)
        self.out = torch.zeros(max_seqs, dtype=torch.int32, device="cuda")

    def add(self, prompt, **sampling) -> int:
        """Takes a prompt in; sampling holds repetition, frequency, presence, bias and mask."""
        prompt = [int(t) for t in prompt]
        if any(t < 0 or t >= self.shape.vocab_size for t in prompt):
            raise ValueError("a token id outside the vocabulary")
        mask, words = sampling.get("mask"), (self.shape.vocab_size + 31) // 32
        if mask is not None:
            mask = np.asarray(mask)
            if mask.ndim != 1 or len(mask) < words or mask.dtype.kind not in "iu":
                raise ValueError(f"the mask must be {words} words of 32 bits")
            sampling["mask"] = mask[:words].astype(np.uint32).view(np.int32)
        return self.seqs.add(Sequence(prompt, **sampling))

    def remove(self, i: int) -> None:
        self.seqs.remove(i)

    def running(self) -> list[int]:
        """The sequences that will still get tokens."""
        return self.seqs.running()

    def step(self) -> dict[int, int]:
        """Runs one step; the next token of every sequence that got one."""
        step = self.seqs.step()
        if not step.ids:
            return {}
        self.forward(step)
        n = len(step.outputs)
        if n:
            self._pick([self.seqs.live[i] for _, i in step.outputs])
        return self.seqs.commit(step, self.out[:n].tolist())

    def _device(self, values, dtype="int32"):
        return self.torch.from_numpy(np.asarray(values, dtype)).cuda(non_blocking=True)

    def forward(self, step: Step) -> None:
        """The model over one step; leaves the logits of step.outputs in self.logits."""
        t, s, w, seqs = self.torch, self.shape, self.w, self.seqs
        rows = seqs.max_seqs if max(step.counts) == 1 else seqs.max_seqs + seqs.chunk
        plan = self.plans[rows]
        starts = np.cumsum([0] + step.counts)
        q_start = np.full(seqs.max_seqs + 1, starts[-1], np.int32)
        q_start[:len(starts)] = starts
        kv_len = np.zeros(seqs.max_seqs, np.int32)
        table = np.zeros((seqs.max_seqs, seqs.max_pages), np.int32)
        for b, (i, n) in enumerate(zip(step.ids, step.counts)):
            seq = seqs.live[i]
            kv_len[b] = seq.cached + n
            table[b, :len(seq.pages)] = seq.pages
        plan.update(self._device(q_start), self._device(kv_len), self._device(table))
        stream = t.cuda.current_stream().cuda_stream
        H, I, qd, kd, eps = s.hidden_size, s.intermediate_size, s.q_dim, s.kv_dim, s.rms_norm_eps
        x, xb, q, k, v, att, act = (b[:rows] for b in (self.x, self.xb, self.q, self.k, self.v, self.att, self.act))
        px, pxb, pq, pk, pv, pa, pact = (b.data_ptr() for b in (x, xb, q, k, v, att, act))
        tokens = self._device(step.tokens + [0] * (rows - len(step.tokens)))
        call("q3_embedding_batched", px, w.ptr["model.embed_tokens.weight"], tokens.data_ptr(), rows, H, s.vocab_size, stream)
        for l in range(s.num_hidden_layers):
            p = {n: w.ptr[f"model.layers.{l}.{n}.weight"] for n in (
                "input_layernorm", "self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj",
                "post_attention_layernorm", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")}
            norms = [w.tensor(f"model.layers.{l}.self_attn.{n}.weight") for n in ("q_norm", "k_norm")]
            call("q3_rmsnorm_forward", pxb, px, p["input_layernorm"], rows, H, eps, stream)
            call("q3_qkv_batched", pq, pk, pv, p["self_attn.q_proj"], p["self_attn.k_proj"], p["self_attn.v_proj"], pxb,
                 rows, qd, kd, H, stream)
            paged_rope_append(q, q, k, v, self.key_pages[l], self.value_pages[l], plan, self.inv_freq, norms[0], norms[1],
                              eps, amplitude=self.amplitude)
            paged_attention(att, q, self.key_pages[l], self.value_pages[l], plan)
            call("q3_gemv_residual_batched", px, p["self_attn.o_proj"], pa, rows, H, qd, None, stream)
            call("q3_rmsnorm_forward", pxb, px, p["post_attention_layernorm"], rows, H, eps, stream)
            call("q3_gate_up_batched", pact, p["mlp.gate_proj"], p["mlp.up_proj"], pxb, rows, I, H, None, None, stream)
            call("q3_gemv_residual_batched", px, p["mlp.down_proj"], pact, rows, H, I, None, stream)
        n = len(step.outputs)
        if n:
            picked = self._device([row for row, _ in step.outputs])
            last = self.last.data_ptr()
            call("q3_embedding_batched", last, px, picked.data_ptr(), n, H, rows, stream)  # the rows that count
            call("q3_rmsnorm_forward", last, last, w.ptr["model.norm.weight"], n, H, eps, stream)
            lm = w.ptr["model.embed_tokens.weight" if s.tie_word_embeddings else "lm_head.weight"]
            call("q3_gemv_batched", self.logits.data_ptr(), lm, last, n, s.vocab_size, H, stream)

    def _pick(self, seqs: list[Sequence]) -> None:
        """Penalties, biases and masks on the logits, then the largest of each row into self.out."""
        n, words = len(seqs), (self.shape.vocab_size + 31) // 32
        start, split, ids, bias_start, bias_ids, bias = [0], [], [], [0], [], []
        for q in seqs:
            split.append(start[-1] + len(q.prompt))
            ids += q.prompt + q.generated
            start.append(len(ids))
            bias_ids += list(q.bias)
            bias += list(q.bias.values())
            bias_start.append(len(bias))
        kw = {}
        if any((q.repetition, q.frequency, q.presence) != (1.0, 0.0, 0.0) for q in seqs):
            kw.update(hist_start=self._device(start), hist_split=self._device(split), hist_ids=self._device(ids),
                      repetition=self._device([q.repetition for q in seqs], "float32"),
                      frequency=self._device([q.frequency for q in seqs], "float32"),
                      presence=self._device([q.presence for q in seqs], "float32"))
        if bias:
            kw.update(bias_start=self._device(bias_start), bias_ids=self._device(bias_ids), bias=self._device(bias, "float32"))
        if any(q.mask is not None for q in seqs):
            free = np.full(words, -1, np.int32)
            kw["mask"] = self._device(np.stack([free if q.mask is None else q.mask for q in seqs]))
        rows = self.logits[:n]
        if kw:
            logits_process(rows, rows, **kw)
        call("q3_argmax_batched", self.out.data_ptr(), rows.data_ptr(), n, self.shape.vocab_size,
             self.torch.cuda.current_stream().cuda_stream)
