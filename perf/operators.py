"""The paged serving operators at the sizes a server meets, in plain form and as the library's kernels.

  append   q/k norms, rotary positions and the write into a paged cache (paged_rope_append)
  attend   attention of each sequence's new tokens over its pages (paged_attention)
  logits   penalties, biases and grammar masks on a step's logits (logits_process)

`own` picks the side: False computes the definition with elementary torch operations in fp32,
rounded once at the end; True makes the calls a user of the library makes.
"""
from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

BF16 = torch.bfloat16


def _package():
    name = "llm_inference_b200"
    if name not in sys.modules:
        pkg = Path(__file__).resolve().parents[1] / "llm-inference_b200"
        spec = importlib.util.spec_from_file_location(name, pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ---------------------------------------------------------------- cases
# A batch is `seqs` sequences with `q` new tokens each and lengths (new tokens included) drawn between
# kv_lo and kv_hi by the generator `lens` seeds, then, if chunk > 0, one more sequence with `chunk` new
# tokens after chunk_ctx earlier ones. Sizes depend on the case alone; values depend on the seed too.

def listed():
    attend = dict(op="attend", heads=32, kv_heads=8, dim=128, chunk=0, chunk_ctx=0, q=1)
    append = dict(op="append", heads=32, kv_heads=8, dim=128, chunk=0, chunk_ctx=0, norm=True, rope_dim=128,
                  interleaved=False, scaled=False)
    return [
        # one user's next token early in a conversation: latency
        dict(attend, name="attend_one", seqs=1, kv_lo=256, kv_hi=256, page=16, slots_first=False, lens=1),
        # the decode benchmark's batch: 32 sequences around 4096 positions
        dict(attend, name="attend_32x4096", seqs=32, kv_lo=3900, kv_hi=4200, page=64, slots_first=False, lens=2),
        # a busy server: 64 sequences from just begun to 8192, small pages, heads interleaved within a slot
        dict(attend, name="attend_64_ragged", seqs=64, heads=16, kv_lo=1, kv_hi=8192, page=16, slots_first=True,
             lens=3),
        # draft tokens being verified: five rows a sequence, small heads, eight query heads a kv head
        dict(attend, name="attend_verify", seqs=16, q=5, heads=32, kv_heads=4, dim=64, kv_lo=200, kv_hi=6000, page=32,
             slots_first=False, lens=4),
        # a long prompt's last chunk
        dict(attend, name="attend_chunk_2048", seqs=0, kv_lo=1, kv_hi=1, chunk=2048, chunk_ctx=8192, page=64,
             slots_first=False, lens=5),
        # a step that decodes 31 sequences and takes in a chunk of a new prompt
        dict(attend, name="attend_mixed", seqs=31, kv_lo=100, kv_hi=6000, chunk=333, chunk_ctx=1500, page=16,
             slots_first=False, lens=6),
        # one user's next token
        dict(append, name="append_one", seqs=1, q=1, kv_lo=256, kv_hi=256, page=16, slots_first=False, lens=7),
        # a batch of few new tokens: interleaved pairs, half of the head, frequencies scaled for long contexts
        dict(append, name="append_partial", seqs=48, q=3, heads=16, kv_lo=3, kv_hi=20000, page=32, slots_first=True,
             norm=False, rope_dim=64, interleaved=True, scaled=True, lens=8),
        # four prompts of 2048 tokens
        dict(append, name="append_4x2048", seqs=4, q=2048, kv_lo=2048, kv_hi=6000, page=64, slots_first=False, lens=9),
        # one user's logits with a short history
        dict(op="logits", name="logits_one", rows=1, vocab=151936, f32=False, hist_lo=200, hist_hi=200, biases=0,
             mask=False, lens=10),
        # the decode benchmark's batch with everything on
        dict(op="logits", name="logits_32", rows=32, vocab=151936, f32=False, hist_lo=1, hist_hi=4096, biases=64,
             mask=True, lens=11),
        # fp32 logits of an odd vocabulary, long histories
        dict(op="logits", name="logits_f32", rows=100, vocab=32003, f32=True, hist_lo=0, hist_hi=16384, biases=300,
             mask=False, lens=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {"attend": work(listed()[4])["flops"], "append": work(listed()[8])["bytes"]}
    while True:
        op = rng.choice(["attend", "attend", "attend", "append", "logits"])
        lens = rng.randrange(1 << 30)
        if op == "logits":
            f32 = rng.random() < 0.4
            rows, vocab = _log_int(rng, 1, 100), _log_int(rng, 1000, 151936)
            if rows * vocab * (2 if f32 else 1) > 32 * 151936:
                continue
            hi = _log_int(rng, 1, 16384)
            return dict(op=op, rows=rows, vocab=vocab, f32=f32, hist_lo=rng.choice([0, hi // 2]), hist_hi=hi,
                        biases=rng.choice([0, 5, 300]), mask=rng.random() < 0.5, lens=lens)
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (16, 8, 128), (8, 8, 128), (64, 8, 128), (32, 4, 64), (4, 2, 64),
                                           (12, 2, 96)])
        page = rng.choice([8, 16, 32, 48, 64, 128, 256])
        case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=page, slots_first=rng.random() < 0.5, lens=lens)
        if op == "attend":
            kind = rng.choice(["decode", "verify", "chunk", "mixed"])
            seqs = 0 if kind == "chunk" else _log_int(rng, 1, 64)
            q = rng.randint(2, 16) if kind == "verify" else 1
            hi = _log_int(rng, 16, 8192)
            chunk = _log_int(rng, 2, 2048) if kind in ("chunk", "mixed") else 0
            case.update(seqs=seqs, q=q, kv_lo=rng.choice([q, max(q, hi // 2)]), kv_hi=max(q, hi), chunk=chunk,
                        chunk_ctx=_log_int(rng, 1, 8192) if chunk else 0)
            w = work(case)
            if w["flops"] > most[op] or w["bytes"] > 1.1e9:
                continue
        else:
            seqs = _log_int(rng, 1, 64)
            q = _log_int(rng, 1, 2048)
            lo = rng.choice([q, q + 1000])
            case.update(seqs=seqs, q=q, kv_lo=lo, kv_hi=lo + _log_int(rng, 1, 2000), chunk=0, chunk_ctx=0,
                        norm=rng.random() < 0.6, rope_dim=rng.choice([dim, dim, dim // 2]),
                        interleaved=rng.random() < 0.4, scaled=rng.random() < 0.4)
            if work(case)["bytes"] > most[op]:
                continue
        return case


def _lengths(case):
    """(new tokens, positions once they are in) of every sequence."""
    r = random.Random(case["lens"])
    out = [(case["q"], r.randint(case["kv_lo"], case["kv_hi"])) for _ in range(case["seqs"])]
    if case["chunk"]:
        out.append((case["chunk"], case["chunk_ctx"] + case["chunk"]))
    return out


def _history(case):
    """(prompt tokens, output tokens) of every row."""
    r = random.Random(case["lens"])
    out = []
    for _ in range(case["rows"]):
        n = r.randint(case["hist_lo"], case["hist_hi"])
        p = r.randint(0, n)
        out.append((p, n - p))
    return out


def work(case):
    if case["op"] == "logits":
        n, hist = case["rows"] * case["vocab"], sum(p + o for p, o in _history(case))
        return {"bytes": n * (8 if case["f32"] else 4) + (n // 8 if case["mask"] else 0) + 4 * hist
                + 8 * case["rows"] * case["biases"], "flops": 4 * n}
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    lens = _lengths(case)
    tokens = sum(q for q, _ in lens)
    if case["op"] == "append":
        return {"bytes": tokens * (2 * h + 4 * kvh) * d * 2, "flops": tokens * (h + kvh) * d * 8}
    rows = sum(q * (kv - q) + q * (q + 1) // 2 for q, kv in lens)
    return {"bytes": 2 * sum(kv for _, kv in lens) * kvh * d * 2 + 2 * tokens * h * d * 2, "flops": 4 * h * d * rows}


# ---------------------------------------------------------------- inputs

def _frequencies(case):
    """fp32 rotation frequencies: theta 1e6, and where scaled, the slow ones stretched eightfold with a
    smooth passage between wavelengths of 2048 and 8192 positions."""
    n = case["rope_dim"] // 2
    out = []
    for j in range(n):
        f = 1e6 ** (-2.0 * j / case["rope_dim"])
        if case["scaled"]:
            wave = 2 * math.pi / f
            t = min(1.0, max(0.0, (8192 / wave - 1.0) / (4.0 - 1.0)))
            f = t * f + (1 - t) * f / 8
        out.append(f)
    return torch.tensor(out, dtype=torch.float32)


def _normal(g, *shape, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(BF16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "logits":
        return _prepare_logits(case, g)
    h, kvh, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case)
    tokens = sum(q for q, _ in lens)
    max_pages = max(-(-kv // page) for _, kv in lens)
    n_pages = sum(-(-kv // page) for _, kv in lens) + 3
    shape = (n_pages, page, kvh, d) if case["slots_first"] else (n_pages, kvh, page, d)
    kp, vp = _normal(g, *shape), _normal(g, *shape)
    if case["slots_first"]:  # [page, head, slot, dim] views of either layout
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).tolist()
    table, starts, used = [], [0], 0
    for q, kv in lens:
        n = -(-kv // page)
        table.append(order[used:used + n] + [0] * (max_pages - n))
        used += n
        starts.append(starts[-1] + q)
    s = {"case": case, "lens": lens, "starts": starts, "key_pages": kp, "value_pages": vp,
         "table": torch.tensor(table, dtype=torch.int32, device="cuda"),
         "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
         "kv_len": torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda"),
         "q": _normal(g, tokens, h, d, std=1.5 if case["op"] == "attend" else 1.0)}
    s["out"] = torch.empty_like(s["q"])
    if case["op"] == "append":
        s["k"], s["v"] = _normal(g, tokens, kvh, d), _normal(g, tokens, kvh, d)
        s["inv_freq"] = _frequencies(case).cuda()
        s["q_norm"] = _normal(g, d, std=0.2, mean=1.0) if case["norm"] else None
        s["k_norm"] = _normal(g, d, std=0.2, mean=1.0) if case["norm"] else None
        # row r of the batch goes to this page and slot: what the plain form indexes with
        pos = [kv - q + i for q, kv in lens for i in range(q)]
        row = [b for b, (q, _) in enumerate(lens) for _ in range(q)]
        s["pos"] = torch.tensor(pos, device="cuda")
        s["row_page"] = s["table"].long()[torch.tensor(row, device="cuda"), s["pos"] // page]
    if own:
        q3 = _package()
        s["plan"] = q3.PagedPlan(len(lens), tokens, max(q for q, _ in lens), h, kvh, d, page, n_pages, max_pages)
        s["plan"].update(s["q_start"], s["kv_len"], s["table"])
    return s


def _prepare_logits(case, g):
    rows, vocab = case["rows"], case["vocab"]
    hist = _history(case)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
    n = sum(p + o for p, o in hist)
    # a few tokens make up most of a text
    ids = (torch.rand(n, generator=g, device="cuda") ** 4 * vocab).to(torch.int32).clamp_(max=vocab - 1)
    start, split = [0], []
    for p, o in hist:
        split.append(start[-1] + p)
        start.append(start[-1] + p + o)
    def param(lo, hi):
        return torch.rand(rows, generator=g, device="cuda") * (hi - lo) + lo
    s = {"case": case, "hist": hist, "logits": x if case["f32"] else x.to(BF16), "ids": ids,
         "start": torch.tensor(start, dtype=torch.int32, device="cuda"),
         "split": torch.tensor(split, dtype=torch.int32, device="cuda"),
         "repetition": param(1.0, 1.4), "frequency": param(0.0, 0.7), "presence": param(0.0, 0.7),
         "bias_start": None, "bias_ids": None, "bias": None, "mask": None}
    s["out"] = torch.empty_like(s["logits"])
    nb = min(case["biases"], vocab)
    if nb:
        picks = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:nb] for _ in range(rows)])
        s["bias_start"] = torch.arange(0, rows * nb + 1, nb, dtype=torch.int32, device="cuda")
        s["bias_ids"] = picks.to(torch.int32).flatten()
        s["bias"] = torch.randn(rows * nb, generator=g, device="cuda") * 3
    if case["mask"]:  # a grammar leaves some rows free and most others a small part of the vocabulary
        keep = torch.rand(rows, 1, generator=g, device="cuda") ** 3
        keep[0] = 1.0
        words = (vocab + 31) // 32
        bits = torch.rand(rows, words * 32, generator=g, device="cuda") < keep
        weights = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
        s["mask"] = (bits.view(rows, words, 32).long() * weights).sum(-1).to(torch.int32)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "logits": _own_logits}[op](state)
    return {"append": _plain_append, "attend": _plain_attend, "logits": _plain_logits}[op](state)


def _own_append(s):
    c = s["case"]
    _package().paged_rope_append(s["out"], s["q"], s["k"], s["v"], s["key_pages"], s["value_pages"], s["plan"],
                                 s["inv_freq"], q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], eps=1e-6,
                                 interleaved=c["interleaved"])
    return [s["out"], s["key_pages"], s["value_pages"]]


def _own_attend(s):
    _package().paged_attention(s["out"], s["q"], s["key_pages"], s["value_pages"], s["plan"],
                               scale=1.0 / math.sqrt(s["case"]["dim"]))
    return s["out"]


def _own_logits(s):
    _package().logits_process(s["out"], s["logits"], s["start"], s["split"], s["ids"], s["repetition"],
                              s["frequency"], s["presence"], bias_start=s["bias_start"], bias_ids=s["bias_ids"],
                              bias=s["bias"], mask=s["mask"])
    return s["out"]


def _plain_append(s):
    c = s["case"]
    half = c["rope_dim"] // 2
    angle = s["pos"].float()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        if c["interleaved"]:
            a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half:2 * half]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([r, x[..., 2 * half:]], -1)

    s["out"].copy_(turn(s["q"], s["q_norm"]))
    slot = s["pos"] % c["page"]
    s["key_pages"][s["row_page"], :, slot] = turn(s["k"], s["k_norm"]).to(BF16)
    s["value_pages"][s["row_page"], :, slot] = s["v"]
    return [s["out"], s["key_pages"], s["value_pages"]]


def _plain_attend(s):
    c = s["case"]
    kvh, d = c["kv_heads"], c["dim"]
    rep = c["heads"] // kvh
    scale = 1.0 / math.sqrt(d)
    for b, (q, kv) in enumerate(s["lens"]):
        pages = s["table"][b, :-(-kv // c["page"])].long()
        first = s["starts"][b]
        x = s["q"][first:first + q].float().view(q, kvh, rep, d)
        seen = torch.arange(kv, device="cuda") <= torch.arange(kv - q, kv, device="cuda")[:, None]
        k = s["key_pages"][pages].float().transpose(1, 2).reshape(-1, kvh, d)[:kv].permute(1, 2, 0)
        v = s["value_pages"][pages].float().transpose(1, 2).reshape(-1, kvh, d)[:kv].transpose(0, 1)
        rows = max(1, (1 << 29) // (kv * c["heads"]))  # query tokens at a time: at most 2 GB of scores
        for i in range(0, q, rows):
            y = x[i:i + rows].transpose(0, 1)
            p = torch.matmul(y.reshape(kvh, -1, d), k).view(kvh, -1, rep, kv) * scale
            p = p.masked_fill(~seen[i:i + rows, None, :], float("-inf"))
            p = torch.exp(p - p.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(kvh, -1, kv), v).view(kvh, -1, rep, d)
            s["out"][first + i:first + i + o.shape[1]] = o.transpose(0, 1).reshape(-1, c["heads"], d).to(BF16)
    return s["out"]


def _plain_logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    x = s["logits"].float()
    n = torch.zeros(rows, vocab, device="cuda")
    seen = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda")
    at = torch.arange(len(s["ids"]), device="cuda")
    row = torch.searchsorted(s["start"][1:].long(), at, right=True)
    ids = s["ids"].long()
    seen[row, ids] = True
    n.index_put_((row, ids), (at >= s["split"].long()[row]).float(), accumulate=True)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * n - s["presence"][:, None] * (n > 0)
    if s["bias"] is not None:
        add = torch.zeros(rows, vocab, device="cuda")
        per = s["bias_ids"].view(rows, -1).long()
        add.scatter_(1, per, s["bias"].view(rows, -1))
        x = x + add
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = x.masked_fill(bits.view(rows, -1)[:, :vocab] == 0, float("-inf"))
    s["out"].copy_(x)
    return s["out"]


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logits": _exact_logits}[case["op"]](s)


def _exact_append(s):
    c, f64 = s["case"], torch.float64
    d, r = c["dim"], c["rope_dim"]
    phase = torch.outer(s["pos"].to(f64), s["inv_freq"].to(f64))
    spin = torch.polar(torch.ones_like(phase), phase)[:, None, :]

    def rotated(x, w):
        y = x.to(f64)
        if w is not None:
            y = y / torch.sqrt(torch.einsum("thd,thd->th", y, y) / d + 1e-6)[..., None] * w.to(f64)
        y = y.clone()
        first = torch.arange(0, r, 2, device="cuda") if c["interleaved"] else torch.arange(r // 2, device="cuda")
        second = first + (1 if c["interleaved"] else r // 2)
        z = torch.complex(y[..., first], y[..., second]) * spin
        y[..., first], y[..., second] = z.real, z.imag
        return y

    kp, vp = s["key_pages"].to(f64), s["value_pages"].to(f64)
    slot = torch.remainder(s["pos"], c["page"])
    k, v = rotated(s["k"], s["k_norm"]), s["v"].to(f64)
    for h in range(c["kv_heads"]):
        kp[s["row_page"], h, slot] = k[:, h]
        vp[s["row_page"], h, slot] = v[:, h]
    return [rotated(s["q"], s["q_norm"]), kp, vp]


def _exact_attend(s):
    c, f64 = s["case"], torch.float64
    out = torch.empty(s["q"].shape, dtype=f64, device="cuda")
    rep = c["heads"] // c["kv_heads"]
    for b, (q, kv) in enumerate(s["lens"]):
        where = torch.arange(kv, device="cuda")
        page, slot = s["table"][b].long()[where // c["page"]], where % c["page"]
        mine = slice(s["starts"][b], s["starts"][b + 1])
        late = torch.triu(torch.ones(q, kv, dtype=torch.bool, device="cuda"), kv - q + 1)
        for head in range(c["heads"]):
            k = s["key_pages"][page, head // rep, slot].to(f64)
            v = s["value_pages"][page, head // rep, slot].to(f64)
            logit = torch.einsum("qd,td->qt", s["q"][mine, head].to(f64), k) / math.sqrt(c["dim"])
            logit[late] = float("-inf")
            out[mine, head] = torch.exp(logit - torch.logsumexp(logit, 1, keepdim=True)) @ v
    return out


def _exact_logits(s):
    c, f64 = s["case"], torch.float64
    rows, vocab = c["rows"], c["vocab"]
    out = s["logits"].to(f64).clone()
    start, split = s["start"].tolist(), s["split"].tolist()
    for r in range(rows):
        x = out[r]
        told, said = s["ids"][start[r]:split[r]].long(), s["ids"][split[r]:start[r + 1]].long()
        any_ = torch.unique(torch.cat([told, said]))
        rep = s["repetition"][r].to(f64)
        x[any_] = torch.where(x[any_] > 0, x[any_] / rep, x[any_] * rep)
        times = torch.bincount(said, minlength=vocab).to(f64)
        x -= times * s["frequency"][r].to(f64) + times.clamp(max=1) * s["presence"][r].to(f64)
        if s["bias"] is not None:
            b0, b1 = s["bias_start"][r].item(), s["bias_start"][r + 1].item()
            x[s["bias_ids"][b0:b1].long()] += s["bias"][b0:b1].to(f64)
        if s["mask"] is not None:
            tok = torch.arange(vocab, device="cuda")
            x[(s["mask"][r][tok // 32].long() >> (tok % 32)) & 1 == 0] = float("-inf")
    return out
