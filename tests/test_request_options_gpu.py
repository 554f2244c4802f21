"""The server with sampled sequences and adapters on a B200, teacher-forced with its own tokens.

Bars: with an adapter merged into fp32 weights, the logits' relative RMS difference from a plain fp32 forward pass stays below 2e-2, as
without one (the adapters' parts are held in more bits than the bf16 activations around them). A sampled token is the one that the
definition takes from the server's own logits and the sequence's random numbers.
"""
import sys
from pathlib import Path

import numpy as np
import pytest

HERE = Path(__file__).resolve().parent
sys.path.insert(0, str(HERE))
import conftest  # noqa: E402,F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llm_inference_b200 as q3  # noqa: E402
from llm_inference_b200 import checkpoint  # noqa: E402
from llm_inference_b200.adapters import AdapterSet, projection_sizes  # noqa: E402
from llm_inference_b200.engine import DeviceWeights  # noqa: E402
from llm_inference_b200.serving import PagedServer  # noqa: E402
from test_request_options import write_adapter  # noqa: E402
from test_sample_gpu import exact_row  # noqa: E402
from test_serving_gpu import SHAPES, plain_logits  # noqa: E402


class Merged:
    """Weights with an adapter's part added, as plain_logits reads them."""

    def __init__(self, w, tensors, scale):
        self.shape, self._w, self._tensors, self._scale = w.shape, w, tensors, scale

    def tensor(self, name):
        t = self._w.tensor(name)
        parts = name.split(".")
        if parts[1] == "layers":
            key = int(parts[2]), ".".join(parts[3:5])
            if key in self._tensors:
                a, b = (x.to(torch.bfloat16).float().cuda() for x in self._tensors[key])
                t = t.float() + self._scale * (b @ a)
        return t


def random_adapter(shape, seed, r, projections=None):
    g = torch.Generator().manual_seed(seed)
    return {(layer, p): (torch.randn(r, k, generator=g) * k ** -0.5, torch.randn(n, r, generator=g) * 0.1)
            for layer in range(shape.num_hidden_layers) for p, (k, n) in projection_sizes(shape).items() if projections is None or p in projections}


def run(server, steps):
    """(id, tokens before, logits) of every token."""
    seen = []
    for _ in range(steps):
        step = server.seqs.step()
        if not step.ids:
            break
        server.forward(step)
        n = len(step.outputs)
        rows = [server.logits[r].clone() for r in range(n)]
        if n:
            server._pick([server.seqs.live[i] for _, i in step.outputs])
        for (_, i), logits in zip(step.outputs, rows):
            q = server.seqs.live[i]
            seen.append((i, q.prompt + q.generated, logits))
        server.seqs.commit(step, [max(t, 0) for t in server.out[:n].tolist()])
    return seen


@pytest.mark.parametrize("name", list(SHAPES))
def test_adapters_follow_merged_weights(name, tmp_path):
    shape = SHAPES[name]
    w = DeviceWeights.random(shape, seed=4)
    some = ("self_attn.q_proj", "self_attn.v_proj", "mlp.down_proj")
    loaded = {0: (random_adapter(shape, 1, 16), 1.5), 2: (random_adapter(shape, 2, 3, some), -0.7)}
    adapters = AdapterSet(shape, 4, rank=16)
    for i, (tensors, scale) in loaded.items():
        adapters.set(i, tensors, scale)
    loaded[3] = write_adapter(tmp_path / "a", shape, r=8, alpha=12, projections=("self_attn.k_proj", "mlp.up_proj")), 1.5
    adapters.load(3, tmp_path / "a")
    server = PagedServer(w, n_pages=64, page_size=16, max_seqs=6, max_positions=300, chunk=40, adapters=adapters)
    rng = np.random.default_rng(1)
    ids = {}
    for n, adapter in ((1, 0), (90, 2), (23, -1), (60, 0), (7, 3)):
        ids[server.add(rng.integers(0, shape.vocab_size, n).tolist(), adapter=adapter)] = adapter
    seen = run(server, 14)
    assert q3.device_error() == 0
    assert {i for i, _, _ in seen} == set(ids)
    for i, before, logits in seen:
        ref = plain_logits(Merged(w, *loaded[ids[i]]) if ids[i] >= 0 else w, before)[-1]
        rel = ((logits.float() - ref).square().mean() / ref.square().mean()).sqrt().item()
        assert rel < 2e-2, (i, ids[i], len(before), rel)
        if ids[i] >= 0:  # the adapter changes more than that
            bare = plain_logits(w, before)[-1]
            assert ((ref - bare).square().mean() / ref.square().mean()).sqrt().item() > 4e-2


def test_sequences_without_an_adapter_stay_as_they_were():
    shape = SHAPES["tiny"]
    w = DeviceWeights.random(shape, seed=4)
    prompts = [list(range(5, 5 + n)) for n in (3, 30, 11)]

    def say(adapters, others):
        server = PagedServer(w, n_pages=64, page_size=8, max_seqs=6, max_positions=120, chunk=16, adapters=adapters)
        ids = [server.add(p) for p in prompts]
        for a in others:
            server.add([9, 8, 7], adapter=a)
        said = {i: [] for i in ids}
        for _ in range(30):
            for i, t in server.step().items():
                said.get(i, []).append(t)
        return [said[i][:20] for i in ids]

    adapters = AdapterSet(shape, 2, rank=8)
    adapters.set(0, random_adapter(shape, 1, 8), 2.0)
    want = say(None, [])
    assert say(adapters, []) == want and say(adapters, [0, 0]) == want


def test_sampled_tokens_are_the_definitions():
    shape = SHAPES["hd128"]
    server = PagedServer(DeviceWeights.random(shape, seed=4), n_pages=64, page_size=16, max_seqs=5, max_positions=200, chunk=32)
    kinds = [dict(temperature=0.7, seed=1), dict(temperature=1.3, top_k=20, top_p=0.9, seed=2), dict(temperature=1.0, min_p=0.2, seed=3),
             dict(), dict(temperature=2.0, top_k=500, seed=4)]
    ids = {server.add(list(range(3, 10 + 7 * j)), **kw): kw for j, kw in enumerate(kinds)}
    seen = run(server, 20)
    draws = {i: np.random.default_rng(kw.get("seed")) for i, kw in ids.items()}
    random_ones = 0
    for i, before, logits in seen:
        kw, q = ids[i], server.seqs.live[i]
        token = (q.prompt + q.generated)[len(before)]
        x = logits.double().cpu().numpy()
        if not kw:
            assert token == int(np.argmax(x))
            continue
        u = float(draws[i].random(dtype=np.float32))
        order, w, total, target = exact_row(x, u, kw["temperature"], kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))
        at = order.tolist().index(token)
        room = 1e-9 * total
        assert w[:at].sum() - room <= target <= w[:at + 1].sum() + room
        random_ones += token != int(np.argmax(x))
    assert random_ones > 10


def test_a_seed_repeats_and_masks_hold():
    shape = SHAPES["tiny"]
    w = DeviceWeights.random(shape, seed=4)
    only = np.zeros(shape.vocab_size // 32, np.int32)
    only[3] = 0b1010  # tokens 97 and 99

    def say():
        server = PagedServer(w, n_pages=32, page_size=8, max_seqs=4, max_positions=64, chunk=8)
        a = server.add([1, 2, 3], temperature=1.0, seed=11)
        b = server.add([4, 5], temperature=5.0, seed=12, mask=only)
        c = server.add([6], temperature=1.0, seed=13, mask=np.zeros_like(only))  # nothing is allowed
        out = {a: [], b: [], c: []}
        for _ in range(12):
            for i, t in server.step().items():
                out[i].append(t)
        return [out[i] for i in (a, b, c)]

    first = say()
    assert first == say()
    assert set(first[1]) == {97, 99} and len(set(first[0])) > 3 and set(first[2]) == {0}


def test_adapters_can_be_replaced():
    shape = SHAPES["tiny"]
    adapters = AdapterSet(shape, 1, rank=16)
    t1, t2 = random_adapter(shape, 1, 16), random_adapter(shape, 2, 5, ("self_attn.o_proj",))
    adapters.set(0, t1, 1.0)
    adapters.set(0, t2, 0.5)
    w = DeviceWeights.random(shape, seed=4)
    server = PagedServer(w, n_pages=32, page_size=8, max_seqs=2, max_positions=64, chunk=16, adapters=adapters)
    server.add(list(range(20)), adapter=0)
    for _, before, logits in run(server, 4):
        ref = plain_logits(Merged(w, t2, 0.5), before)[-1]
        assert ((logits.float() - ref).square().mean() / ref.square().mean()).sqrt().item() < 2e-2
    with pytest.raises(ValueError):
        adapters.set(1, t1, 1.0)
    with pytest.raises(ValueError):
        adapters.set(0, {(0, "self_attn.q_proj"): (torch.zeros(17, 256), torch.zeros(256, 17))}, 1.0)
    with pytest.raises(ValueError):
        adapters.set(0, {(0, "self_attn.q_proj"): (torch.zeros(4, 100), torch.zeros(256, 4))}, 1.0)
    with pytest.raises(ValueError):
        adapters.set(0, {(9, "self_attn.q_proj"): t2[0, "self_attn.o_proj"]}, 1.0)
    with pytest.raises(ValueError):
        PagedServer(DeviceWeights.random(SHAPES["hd128"], seed=1), n_pages=4, adapters=adapters)


def test_an_adapter_leaves_the_projections_that_it_does_not_have():
    # of zeros for q alone, beside one of everything, one with gate and up in the last layer only, and a sequence without: its logits
    # are those of a server without adapters, to the bit
    shape = SHAPES["tiny"]
    w, last = DeviceWeights.random(shape, seed=4), shape.num_hidden_layers - 1
    k, n = projection_sizes(shape)["self_attn.q_proj"]
    adapters = AdapterSet(shape, 3, rank=8)
    adapters.set(0, random_adapter(shape, 3, 8), 1.0)  # replaced
    adapters.set(0, {(layer, "self_attn.q_proj"): (torch.ones(2, k), torch.zeros(n, 2)) for layer in range(last + 1)}, 1.0)
    full, late = random_adapter(shape, 1, 8), random_adapter(shape, 2, 8)
    late = {key: t for key, t in late.items() if key[0] == last or key[1] not in ("mlp.gate_proj", "mlp.up_proj")}
    adapters.set(1, full, 1.5)
    adapters.set(2, late, -0.7)
    prompts = [list(range(5, 5 + n)) for n in (3, 40, 11, 7)]

    def say(adapters, chosen, steps):
        server = PagedServer(w, n_pages=64, page_size=8, max_seqs=6, max_positions=120, chunk=16, adapters=adapters)
        ids = [server.add(p, adapter=a) for p, a in zip(prompts, chosen)]
        return ids, run(server, steps)

    ids, bare = say(None, [-1] * 4, 12)
    for chosen in ([0, 0, -1, 0], [0, 0, 1, -1], [0, 0, 2, 1], [0, 0, 2, -1]):
        same, seen = say(adapters, chosen, 12)
        assert same == ids
        for i, a in zip(ids, chosen):
            got, want = ([s for s in x if s[0] == i] for x in (seen, bare))
            if a <= 0:
                assert len(got) == len(want) and all(x[1] == y[1] and torch.equal(x[2], y[2]) for x, y in zip(got, want)), (chosen, i)
            else:
                for _, before, logits in got:
                    ref = plain_logits(Merged(w, *((full, 1.5) if a == 1 else (late, -0.7))), before)[-1]
                    assert ((logits.float() - ref).square().mean() / ref.square().mean()).sqrt().item() < 2e-2
