"""What a server's requests choose for themselves, in plain form and as the library's kernels.

  sample    the next token of each row from given random numbers: temperature, top-k, top-p, min-p, and a draft
            token that is kept with the probability the row gives it (sample_logits)
  add       low-rank adapters of many requests beside a shared projection, or three of one input (lora_add)
  gate_up   the same for the gated feed-forward, through its activation (lora_gate_up)

`own` picks the side: False computes the definition with elementary torch operations, sampling in fp64 (a border between
two tokens is a small difference of long sums), adapters in fp32, rounded once at the end; True makes the calls a user
of the library makes.
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
# Sampling: `kind` says how each row's temperature, top-k, top-p and min-p are drawn, by the generator `pick` seeds.
# Adapters: `seqs` sequences of one token and `chunk` tokens of one more; each sequence has one of `adapters` adapters,
# or none with probability `bare`; `ragged` gives the adapters ranks of their own up to `rank`. Sizes depend on
# the case alone; values depend on the seed too.

def listed():
    s = dict(op="sample", vocab=151936, f32=False, masked=False, draft=False)
    a = dict(op="add", k=2560, ns="4096,1024,1024", seqs=0, chunk=0, adapters=8, rank=16, bare=0.0, ragged=False)
    g = dict(a, op="gate_up", ns="9728")
    return [
        # one user's next token with a chat model's usual settings: latency
        dict(s, name="sample_one", rows=1, kind="chat", pick=1),
        # the decode benchmark's batch, each request with settings of its own, some under a grammar
        dict(s, name="sample_32_mixed", rows=32, kind="mixed", masked=True, pick=2),
        # fp32 logits of an odd vocabulary, top-p alone
        dict(s, name="sample_f32_100", rows=100, vocab=32003, f32=True, kind="nucleus", pick=3),
        # five rows of each of 16 sequences whose draft tokens are being verified
        dict(s, name="sample_verify", rows=80, kind="nucleus", draft=True, pick=4),
        # many rollouts of a policy: the whole distribution, nothing cut off
        dict(s, name="sample_256_free", rows=256, kind="free", pick=5),
        # one user's token through q, k and v
        dict(a, name="add_one", seqs=1, pick=6),
        # the decode benchmark's batch over 16 adapters of unequal rank, a few requests with none
        dict(a, name="add_32", seqs=32, adapters=16, rank=32, bare=0.1, ragged=True, pick=7),
        # the down projection of a batch in which nearly every request has an adapter of its own
        dict(a, name="add_down_64", k=9728, ns="2560", seqs=64, adapters=64, pick=8),
        # a chunk of a prompt beside 31 decodes, adapters of rank 64
        dict(a, name="add_chunk_2048", seqs=31, chunk=2048, rank=64, pick=9),
        # the decode benchmark's batch through gate and up
        dict(g, name="gate_up_32", seqs=32, bare=0.1, pick=10),
        # a smaller model, an odd chunk
        dict(g, name="gate_up_333", k=2048, ns="6144", seqs=14, chunk=333, adapters=5, rank=24, pick=11),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {c["op"]: work(c)["bytes"] for c in listed() if c["name"] in ("sample_256_free", "add_chunk_2048", "gate_up_333")}
    while True:
        op = rng.choice(["sample", "sample", "add", "add", "gate_up"])
        pick = rng.randrange(1 << 30)
        if op == "sample":
            case = dict(op=op, rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 1000, 151936), f32=rng.random() < 0.4,
                        masked=rng.random() < 0.3, draft=rng.random() < 0.3,
                        kind=rng.choice(["chat", "nucleus", "free", "floor", "mixed"]), pick=pick)
        else:
            k, qkv, inter = rng.choice([(1024, "2048,1024,1024", 4864), (2048, "2048,1024,1024", 6144), (2560, "4096,1024,1024", 9728),
                                        (1000, "1016,264,264", 2008)])
            if op == "gate_up":
                ns = str(inter)
            else:
                k, ns = rng.choice([(k, qkv), (k, qkv), (int(qkv.split(",")[0]), str(k)), (inter, str(k))])
            chunk = rng.choice([0, _log_int(rng, 2, 2048)])
            case = dict(op=op, k=k, ns=ns, seqs=_log_int(rng, 1, 100) if chunk == 0 or rng.random() < 0.5 else 0, chunk=chunk,
                        adapters=_log_int(rng, 1, 64), rank=rng.choice([8, 16, 16, 24, 32, 64, 128]),
                        bare=rng.choice([0.0, 0.3]), ragged=rng.random() < 0.5, pick=pick)
        if work(case)["bytes"] <= most[op]:
            return case


def _settings(case):
    """(temperature, top-k, top-p, min-p) of every row; temperature 0: the largest logit."""
    r = random.Random(case["pick"])
    out = []
    for i in range(case["rows"]):
        kind = case["kind"]
        if kind == "mixed":
            kind = ["chat", "nucleus", "free", "floor", "greedy", "many"][i % 6]
        out.append({"chat": lambda: (0.6, 20, 0.95, 0.0),
                    "nucleus": lambda: (r.uniform(0.5, 1.2), 0, r.uniform(0.7, 0.99), 0.0),
                    "free": lambda: (r.uniform(0.7, 1.3), 0, 1.0, 0.0),
                    "floor": lambda: (r.uniform(0.7, 2.0), 0, 1.0, r.uniform(0.01, 0.2)),
                    "greedy": lambda: (0.0, 0, 1.0, 0.0),
                    "many": lambda: (r.uniform(0.7, 1.3), r.randint(100, 2000), r.uniform(0.9, 1.0), 0.001)}[kind]())
    return out


def _layout(case):
    """Each row's adapter (-1: none) and each adapter's rank."""
    r = random.Random(case["pick"])
    def one():
        return -1 if r.random() < case["bare"] else r.randrange(case["adapters"])
    index = [one() for _ in range(case["seqs"])]
    if case["chunk"]:
        index += [r.randrange(case["adapters"])] * case["chunk"]
    ranks = [r.randint(1, case["rank"]) if case["ragged"] else case["rank"] for _ in range(case["adapters"])]
    return index, ranks


def _widths(case):
    ns = [int(n) for n in case["ns"].split(",")]
    return ns * 2 if case["op"] == "gate_up" else ns


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["f32"] else 2) + 32 * case["rows"], "flops": 4 * n}
    index, ranks = _layout(case)
    ns, k = _widths(case), case["k"]
    used = [i for i in index if i >= 0]
    rows = len(used) if case["op"] == "gate_up" else len(index)
    per_row = (3 * ns[0] if case["op"] == "gate_up" else 2 * sum(ns)) * 2
    return {"bytes": len(used) * k * 2 + rows * per_row + sum(2 * ranks[i] * (len(ns) * k + sum(ns)) for i in set(used)),
            "flops": sum(2 * ranks[i] * (len(ns) * k + sum(ns)) for i in used)}


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_sample(case, g) if case["op"] == "sample" else _prepare_lora(case, g)


def _prepare_sample(case, g):
    rows, vocab = case["rows"], case["vocab"]
    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")
    # a broad floor, and some tokens that the context asks for, more or less clearly
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.0
    likely = ((rand(rows, 1) * vocab).long() + torch.arange(64, device="cuda") * (vocab // 64)) % vocab
    lift = (13.0 - 2.0 * torch.log1p(torch.arange(64, device="cuda"))) * (0.4 + 0.8 * rand(rows, 1))
    x.scatter_add_(1, likely, lift)
    if case["masked"]:  # a grammar leaves a part of the vocabulary to every other row
        keep = rand(rows, 1) ** 3
        keep[::2] = 2.0
        drop = rand(rows, vocab) > keep
        drop.scatter_(1, likely[:, 5:6], False)  # never all of it
        x.masked_fill_(drop, float("-inf"))
    settings = _settings(case)
    def column(i, dtype):
        return torch.tensor([s[i] for s in settings], dtype=dtype, device="cuda")
    s = {"case": case, "logits": x if case["f32"] else x.to(BF16), "u": rand(rows), "temperature": column(0, torch.float32),
         "top_k": column(1, torch.int32), "top_p": column(2, torch.float32), "min_p": column(3, torch.float32),
         "draft": None, "out": torch.empty(rows, dtype=torch.int32, device="cuda"), "prob": torch.empty(rows, device="cuda")}
    if case["draft"]:  # good guesses, poor ones, and in every fifth row none
        s["draft"] = likely.gather(1, (rand(rows, 1) ** 3 * 64).long().clamp_(max=63))[:, 0].to(torch.int32)
        s["draft"][4::5] = -1
    return s


def _prepare_lora(case, g):
    index, ranks = _layout(case)
    ns, k, n, rank = _widths(case), case["k"], case["adapters"], case["rank"]
    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF16)
    rows = len(index)
    s = {"case": case, "index": index, "ranks": ranks, "x": normal(rows, k),
         "a": [normal(n, rank, k, std=k ** -0.5) for _ in ns], "b": [normal(n, w, rank, std=0.5 * rank ** -0.5) for w in ns],
         "scale": torch.rand(n, generator=g, device="cuda") * 1.5 + 0.5, "base": [normal(rows, w) for w in ns],
         "ranks_d": torch.tensor(ranks, dtype=torch.int32, device="cuda")}
    # rows of each adapter, and those of none: what the plain form goes by
    s["rows"] = {i: torch.tensor([r for r, a in enumerate(index) if a == i], device="cuda") for i in set(index)}
    if case["op"] == "gate_up":  # what the shared projection left, right for the rows without an adapter
        gate, up = (t.float() for t in s["base"])
        s["out"] = [(gate * torch.sigmoid(gate) * up).to(BF16)]
    else:
        s["out"] = [torch.empty_like(t) for t in s["base"]]
    if own:
        q3 = _package()
        s["stack"] = q3.LoraStack(s["a"], s["b"], s["scale"], s["ranks_d"])
        s["plan"] = q3.LoraPlan(rows, n)
        s["plan"].update(torch.tensor(index, dtype=torch.int32, device="cuda"))
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"sample": _own_sample, "add": _own_add, "gate_up": _own_gate_up}[op](state)
    return {"sample": _plain_sample, "add": _plain_add, "gate_up": _plain_gate_up}[op](state)


def _own_sample(s):
    _package().sample_logits(s["out"], s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                             draft=s["draft"], prob=s["prob"])
    return [s["out"], s["prob"]]


def _own_add(s):
    _package().lora_add(s["out"], s["base"], s["x"], s["stack"], s["plan"])
    return s["out"]


def _own_gate_up(s):
    _package().lora_gate_up(s["out"][0], s["base"][0], s["base"][1], s["x"], s["stack"], s["plan"])
    return s["out"]


def _plain_sample(s):
    x, vocab = s["logits"].double(), s["case"]["vocab"]
    t = s["temperature"].double()[:, None]
    x, token = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest index first
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    place = torch.arange(vocab, device="cuda")
    k = s["top_k"].long()[:, None]
    w = torch.where((t > 0) | (place == 0), w, 0.0)
    w = torch.where((k <= 0) | (place < k), w, 0.0)
    ends = torch.cumsum(w, 1)
    p = s["top_p"].double()[:, None]
    keep = (ends - w < p * ends[:, -1:]) | (p >= 1) | (place == 0)
    keep &= w >= s["min_p"].double()[:, None]
    w = torch.where(keep, w, 0.0)
    ends = torch.cumsum(w, 1)
    total = ends[:, -1:].clone()
    target = s["u"].double()[:, None] * total
    if s["draft"] is not None:  # the draft comes first, the others follow in their order
        first = token == s["draft"].long()[:, None]
        wd = torch.where(first, w, 0.0).sum(1, keepdim=True)
        before = torch.where(first, ends - w, 0.0).sum(1, keepdim=True)
        where = first.to(torch.int32).argmax(1, keepdim=True)
        hit = target < wd
        target = torch.where(target - wd < before, target - wd, target)
    at = (ends > target).to(torch.int32).argmax(1, keepdim=True)
    if s["draft"] is not None:
        at = torch.where(hit, where, at)
    s["out"].copy_(token.gather(1, at)[:, 0])
    s["prob"].copy_((w.gather(1, at) / total)[:, 0])
    return [s["out"], s["prob"]]


def _delta(s, i):
    """The adapters' part of projection i, fp32, zero in rows without one."""
    x = s["x"]
    d = torch.zeros(x.shape[0], s["b"][i].shape[1], device="cuda")
    for adapter, rows in s["rows"].items():
        if adapter >= 0:
            r = s["ranks"][adapter]
            h = torch.matmul(x[rows].float(), s["a"][i][adapter, :r].float().T)
            d[rows] = torch.matmul(h, s["b"][i][adapter, :, :r].float().T) * s["scale"][adapter]
    return d


def _plain_add(s):
    for i, out in enumerate(s["out"]):
        out.copy_(s["base"][i].float() + _delta(s, i))
    return s["out"]


def _plain_gate_up(s):
    gate, up = (s["base"][i].float() + _delta(s, i) for i in range(2))
    act = (gate * torch.sigmoid(gate) * up).to(BF16)
    for adapter, rows in s["rows"].items():
        if adapter >= 0:
            s["out"][0][rows] = act[rows]
    return s["out"]


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_sample(s) if case["op"] == "sample" else _exact_lora(s)


def _exact_sample(s):
    """Row by row: log probabilities, the kept tokens' probabilities renormalised, and the first whose sum passes u."""
    tokens, probs = [], []
    settings = list(zip(*(s[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p", "u"))))
    drafts = s["draft"].tolist() if s["draft"] is not None else [-1] * len(settings)
    for row, (t, k, p, floor, u), d in zip(s["logits"].to(torch.float64), settings, drafts):
        order = torch.argsort(row, descending=True, stable=True)
        if t <= 0:
            tokens.append(order[0].item())
            probs.append(1.0)
            continue
        order = order[:k] if k > 0 else order
        z = row[order] / t
        lp = z - torch.logsumexp(z, 0)
        n = len(order)
        if p < 1:
            mass = torch.cumsum(lp.exp(), 0)
            n = int((mass < p).sum().item()) + 1
        if floor > 0:
            n = min(n, int((lp - lp[0] >= math.log(floor)).sum().item()))
        n = max(1, min(n, len(order)))
        order, q = order[:n], torch.softmax(z[:n], 0)
        where = (order == d).nonzero()
        if len(where):  # the draft goes to the front
            j = where[0, 0].item()
            front = torch.cat([torch.tensor([j], device=q.device), torch.arange(j, device=q.device),
                               torch.arange(j + 1, n, device=q.device)])
            order, q = order[front], q[front]
        j = min(n - 1, int((torch.cumsum(q, 0) <= u).sum().item()))
        tokens.append(order[j].item())
        probs.append(q[j].item())
    return [torch.tensor(tokens, dtype=torch.int32, device="cuda"), torch.tensor(probs, dtype=torch.float64, device="cuda")]


def _exact_lora(s):
    f64 = torch.float64
    x = s["x"].to(f64)
    full = []
    for base, a, b in zip(s["base"], s["a"], s["b"]):
        y = base.to(f64)
        for adapter in set(s["index"]) - {-1}:
            mine = torch.tensor([i == adapter for i in s["index"]], device="cuda")
            w = torch.einsum("nr,rk->nk", b[adapter, :, :s["ranks"][adapter]].to(f64), a[adapter, :s["ranks"][adapter]].to(f64))
            y[mine] += s["scale"][adapter].to(f64) * (x[mine] @ w.T)
        full.append(y)
    if s["case"]["op"] == "add":
        return full
    gate, up = full
    act = gate / (1 + torch.exp(-gate)) * up
    bare = torch.tensor([i < 0 for i in s["index"]], device="cuda")
    act[bare] = s["out"][0][bare].to(f64)
    return [act]
