"""A small continuous-batching server on the paged operators.

:class:`Sequences` is the host side: which tokens the next step takes in and where their keys and
values go. Every step it gives each running sequence one token and, in what is left of the step's
rows, one chunk of the oldest unfinished prompt. :class:`PagedServer` runs such a step through the
model: the projections of the batched ABI, and per layer ``paged_rope_append`` and
``paged_attention`` with the step's one plan, and ``lora_add`` and ``lora_gate_up`` beside the projections of sequences with an
adapter; then ``logits_process`` and the argmax, or ``sample_logits`` where a sequence has a temperature.

    server = PagedServer(DeviceWeights.load(model_dir), n_pages=4096)
    a = server.add(prompt, repetition=1.1, temperature=0.6, top_k=20, top_p=0.95, seed=7)
    while server.running():
        for seq, token in server.step().items():
            ...  # server.remove(seq) once it has said what it had to
    server.remove(a)

A sequence runs until its page table (or the whole pool) is full; it then keeps its tokens, gives its pages back and
gets no more tokens. A step in which only prompts are taken in returns no tokens. When no sequence finds a page for its next
token, the youngest give theirs back, and are taken in again later, prompt and tokens.
"""
from __future__ import annotations

import operator
from dataclasses import dataclass, field

import numpy as np

from ._lib import call
from .lora import LoraPlan, lora_add, lora_gate_up
from .paged import PagedPlan, logits_process, paged_attention, paged_rope_append, rope_inv_freq, sample_logits


@dataclass
class Sequence:
    prompt: list[int]
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: dict[int, float] = field(default_factory=dict)
    mask: np.ndarray | None = None  # int32 words, one bit per allowed token
    temperature: float = 0.0        # 0: the largest logit
    top_k: int = 0                  # 0: all
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int | None = None         # of its random numbers; None: any
    adapter: int = -1               # -1: none
    random: np.random.Generator | None = field(default=None, repr=False)
    generated: list[int] = field(default_factory=list)
    cached: int = 0                 # positions whose keys and values are in the cache
    pages: list[int] = field(default_factory=list)

    def draw(self) -> float:
        """The next of its random numbers in [0, 1), an fp32 value."""
        if self.random is None:
            self.random = np.random.default_rng(self.seed)
        return self.random.random(dtype=np.float32)

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
    """Decoding of up to `max_seqs` sequences, greedy or sampled, each with one of the `adapters` (:class:`AdapterSet`) or none, over
    a pool of `n_pages` pages per layer."""

    def __init__(self, weights, n_pages: int, page_size: int = 64, max_seqs: int = 32, max_positions: int | None = None,
                 chunk: int = 256, rope_kind: str = "plain", adapters=None, **rope):
        import torch
        if adapters is not None and adapters.shape != weights.shape:
            raise ValueError("the adapters are for another model shape")
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
        self.adapters = adapters
        if adapters is not None:
            # of all rows with an adapter, and of those whose adapter has gate or up: the others' keep their activation to the bit
            self.lora_plans = {n: [LoraPlan(n, adapters.n_adapters) for _ in range(2)] for n in self.plans}

        def rows_of(n, count=rows):
            return torch.zeros(count, n, dtype=torch.bfloat16, device="cuda")

        self.x, self.xb, self.act = rows_of(s.hidden_size), rows_of(s.hidden_size), rows_of(s.intermediate_size)
        self.q, self.att = rows_of(s.q_dim), rows_of(s.q_dim)
        self.k, self.v = rows_of(s.kv_dim), rows_of(s.kv_dim)
        if adapters is not None:  # the feed-forward's taps, which the adapters change before the activation
            self.gate, self.up = rows_of(s.intermediate_size), rows_of(s.intermediate_size)
        self.last = rows_of(s.hidden_size, max_seqs)
        self.logits = rows_of(s.vocab_size, max_seqs)
        self.out = torch.zeros(max_seqs, dtype=torch.int32, device="cuda")

    def add(self, prompt, **sampling) -> int:
        """Takes a prompt in; sampling holds repetition, frequency, presence, bias and mask, temperature (0: the largest logit),
        top_k, top_p, min_p and seed, and adapter."""
        prompt = [int(t) for t in prompt]
        if any(t < 0 or t >= self.shape.vocab_size for t in prompt):
            raise ValueError("a token id outside the vocabulary")
        mask, words = sampling.get("mask"), (self.shape.vocab_size + 31) // 32
        if mask is not None:
            mask = np.asarray(mask)
            if mask.ndim != 1 or len(mask) < words or mask.dtype.kind not in "iu":
                raise ValueError(f"the mask must be {words} words of 32 bits")
            sampling["mask"] = mask[:words].astype(np.uint32).view(np.int32)
        seq = Sequence(prompt, **sampling)
        try:  # here, since an error in a step would stop all sequences
            for name in ("repetition", "frequency", "presence", "temperature", "top_p", "min_p"):
                setattr(seq, name, float(getattr(seq, name)))
            seq.bias = {int(t): float(v) for t, v in seq.bias.items()}
        except (AttributeError, OverflowError, TypeError, ValueError) as e:
            raise ValueError(f"penalties, the temperature, top_p and min_p must be numbers, biases numbers of token ids: {e}") from None
        if any(not -2 ** 31 <= t < 2 ** 31 for t in seq.bias):
            raise ValueError("a bias for no token id")
        if not 0.0 <= seq.temperature < float("inf"):
            raise ValueError("the temperature must be a finite number from 0 on")
        try:
            seq.top_k = operator.index(seq.top_k)
            if seq.random is None:
                seq.random = np.random.default_rng(seq.seed)
        except (TypeError, ValueError) as e:
            raise ValueError(f"top_k must be an int and the seed one from 0 on, or None: {e}") from None
        if not 0 <= seq.top_k < 2 ** 31 or not 0.0 <= seq.top_p <= 1.0 or not 0.0 <= seq.min_p <= 1.0:
            raise ValueError("top_k must be an int from 0 on, top_p and min_p within [0, 1]")
        if seq.adapter != -1 and (self.adapters is None or seq.adapter not in self.adapters.loaded):
            raise ValueError(f"there is no adapter {seq.adapter}")
        return self.seqs.add(seq)

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
        # where a mask leaves nothing the argmax takes token 0, and so does sampling
        return self.seqs.commit(step, [max(t, 0) for t in self.out[:n].tolist()])

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
        chosen = [seqs.live[i].adapter for i in step.ids]
        has, lora, planned = set(chosen) - {-1}, None, None
        if has:
            (lora, some), stacks = self.lora_plans[rows], self.adapters.stacks
            index = np.full(rows, -1, np.int32)
            index[:starts[-1]] = np.repeat(chosen, step.counts)
            lora.update(self._device(index))
            gate, up = self.gate[:rows], self.up[:rows]
        call("q3_embedding_batched", px, w.ptr["model.embed_tokens.weight"], tokens.data_ptr(), rows, H, s.vocab_size, stream)
        for l in range(s.num_hidden_layers):
            p = {n: w.ptr[f"model.layers.{l}.{n}.weight"] for n in (
                "input_layernorm", "self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj",
                "post_attention_layernorm", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")}
            norms = [w.tensor(f"model.layers.{l}.self_attn.{n}.weight") for n in ("q_norm", "k_norm")]
            call("q3_rmsnorm_forward", pxb, px, p["input_layernorm"], rows, H, eps, stream)
            call("q3_qkv_batched", pq, pk, pv, p["self_attn.q_proj"], p["self_attn.k_proj"], p["self_attn.v_proj"], pxb,
                 rows, qd, kd, H, stream)
            if lora:
                lora_add([q, k, v], [q, k, v], xb, stacks["qkv"][l], lora)
            paged_rope_append(q, q, k, v, self.key_pages[l], self.value_pages[l], plan, self.inv_freq, norms[0], norms[1],
                              eps, amplitude=self.amplitude)
            paged_attention(att, q, self.key_pages[l], self.value_pages[l], plan)
            call("q3_gemv_residual_batched", px, p["self_attn.o_proj"], pa, rows, H, qd, None, stream)
            if lora:
                lora_add(x, x, att, stacks["o"][l], lora)
            call("q3_rmsnorm_forward", pxb, px, p["post_attention_layernorm"], rows, H, eps, stream)
            changed = has & self.adapters.with_gate_up[l] if lora else None
            if changed and changed not in (has, planned):
                some.update(self._device(np.where(np.isin(index, list(changed)), index, -1)))
                planned = changed
            taps = (gate.data_ptr(), up.data_ptr()) if changed else (None, None)
            call("q3_gate_up_batched", pact, p["mlp.gate_proj"], p["mlp.up_proj"], pxb, rows, I, H, *taps, stream)
            if changed:
                lora_gate_up(act, gate, up, xb, stacks["gate_up"][l], lora if changed == has else some)
            call("q3_gemv_residual_batched", px, p["mlp.down_proj"], pact, rows, H, I, None, stream)
            if lora:
                lora_add(x, x, act, stacks["down"][l], lora)
        n = len(step.outputs)
        if n:
            picked = self._device([row for row, _ in step.outputs])
            last = self.last.data_ptr()
            call("q3_embedding_batched", last, px, picked.data_ptr(), n, H, rows, stream)  # the rows that count
            call("q3_rmsnorm_forward", last, last, w.ptr["model.norm.weight"], n, H, eps, stream)
            lm = w.ptr["model.embed_tokens.weight" if s.tie_word_embeddings else "lm_head.weight"]
            call("q3_gemv_batched", self.logits.data_ptr(), lm, last, n, s.vocab_size, H, stream)

    def _pick(self, seqs: list[Sequence]) -> None:
        """Penalties, biases and masks on the logits, then each row's token into self.out."""
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
        if any(q.temperature > 0.0 for q in seqs):
            f32 = [self._device([getattr(q, name) for q in seqs], "float32") for name in ("temperature", "top_p", "min_p")]
            u = self._device([q.draw() if q.temperature > 0.0 else 0.0 for q in seqs], "float32")
            sample_logits(self.out[:n], rows, u, f32[0], self._device([q.top_k for q in seqs]), f32[1], f32[2])
        else:
            call("q3_argmax_batched", self.out.data_ptr(), rows.data_ptr(), n, self.shape.vocab_size,
                 self.torch.cuda.current_stream().cuda_stream)
