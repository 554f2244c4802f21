"""What requests choose, without a GPU: refusals of the C entries, the server's checks, adapter directories."""
import ctypes
import json
import sys
from pathlib import Path

import numpy as np
import pytest

HERE = Path(__file__).resolve().parent
sys.path.insert(0, str(HERE))
import conftest  # noqa: E402,F401
import llm_inference_b200 as q3  # noqa: E402
from llm_inference_b200 import _lib, adapters, build, checkpoint, lora  # noqa: E402
from llm_inference_b200.serving import PagedServer, Sequence, Sequences  # noqa: E402

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()
    return _lib.load()


FAKE = 1 << 16  # never dereferenced: refused before any launch


def sample(lib, out=FAKE, prob=None, logits=FAKE, dtype=0, rows=2, vocab=64, stride=64, u=FAKE):
    return lib.q3_sample_logits(out, prob, logits, dtype, rows, vocab, stride, u, None, None, None, None, None, None)


def test_sample_logits_refuses(lib):
    assert sample(lib, dtype=2) == 5 and sample(lib, dtype=-1) == 5
    assert sample(lib, rows=-1) == 1 and sample(lib, rows=(1 << 24) + 1) == 1
    assert sample(lib, vocab=0) == 1 and sample(lib, vocab=(1 << 20) + 1, stride=1 << 21) == 1
    assert sample(lib, stride=63) == 1
    assert sample(lib, out=None) == 5 and sample(lib, logits=None) == 5 and sample(lib, u=None) == 5
    assert sample(lib, logits=FAKE + 1) == 2 and sample(lib, logits=FAKE + 2, dtype=1) == 2
    assert sample(lib, rows=0, out=None, logits=None, u=None) == 0  # nothing to do


def test_lora_plans_refuse(lib):
    assert lib.q3_lora_plan_bytes(4, 3) > 0 and lib.q3_lora_plan_bytes(65536, 8192) > 0 and lib.q3_lora_plan_bytes(0, 1) > 0
    for rows, n in ((-1, 3), (65537, 3), (4, 0), (4, 8193)):
        assert lib.q3_lora_plan_bytes(rows, n) == 0
        assert lib.q3_lora_plan(FAKE, rows, n, FAKE, None) == 1
    assert lib.q3_lora_plan(None, 4, 3, FAKE, None) == 5 and lib.q3_lora_plan(FAKE, 4, 3, None, None) == 5
    assert lib.q3_lora_plan(FAKE + 8, 4, 3, FAKE, None) == 2
    assert lib.q3_lora_plan(None, 0, 3, None, None) == 0


def add(lib, n_slices=2, gate_up=False, act=16 << 20, act_stride=64, slice1=None, **kw):
    """A call on addresses a megabyte apart: x, outs, bases."""
    slices = (lora.Q3LoraSlice * 3)()
    for i in range(3):
        slices[i] = lora.Q3LoraSlice((2 + i) << 20, (6 + i) << 20, 64, 64, FAKE, FAKE, 64)
    for key, v in (slice1 or {}).items():
        setattr(slices[1], key, v)
    args = lora.Q3Lora(**dict(dict(x=1 << 20, x_stride=128, k=128, rank=16, n_rows=4, n_adapters=3, ranks=None, scale=None, plan=FAKE), **kw))
    if gate_up:
        return lib.q3_lora_gate_up(act, act_stride, ctypes.byref(slices), ctypes.byref(args), None)
    return lib.q3_lora_add(ctypes.byref(slices), n_slices, ctypes.byref(args), None)


def test_lora_calls_refuse(lib):
    for status, kw in [
        (1, dict(n_slices=0)), (1, dict(n_slices=4)), (1, dict(k=0)), (1, dict(k=12)), (1, dict(rank=0)), (1, dict(rank=12)),
        (1, dict(rank=136)), (1, dict(n_rows=-1)), (1, dict(n_adapters=0)), (1, dict(x_stride=120)), (1, dict(x_stride=132)),
        (1, dict(slice1=dict(n=0))), (1, dict(slice1=dict(n=12))), (1, dict(slice1=dict(n=72))), (1, dict(slice1=dict(out_stride=68))),
        (1, dict(slice1=dict(base_stride=56))), (5, dict(x=None)), (5, dict(plan=None)), (5, dict(slice1=dict(a=None))),
        (5, dict(slice1=dict(b=None))), (5, dict(slice1=dict(out=None))), (5, dict(slice1=dict(base=None))),
        (2, dict(x=(1 << 20) + 8)), (2, dict(slice1=dict(b=FAKE + 8))), (2, dict(slice1=dict(out=(3 << 20) + 8))),
        (5, dict(slice1=dict(out=1 << 20))), (5, dict(slice1=dict(out=2 << 20))), (5, dict(slice1=dict(out=6 << 20))),
        (5, dict(slice1=dict(out=(7 << 20) + 128))),  # its own base, a row on
        (1, dict(gate_up=True, slice1=dict(n=32))), (1, dict(gate_up=True, act_stride=56)), (5, dict(gate_up=True, act=None)),
        (5, dict(gate_up=True, act=1 << 20)), (2, dict(gate_up=True, act=(16 << 20) + 8)),
    ]:
        assert add(lib, **kw) == status, kw
    assert add(lib, n_rows=0, x=None) == 0 and add(lib, n_rows=0, gate_up=True) == 0
    assert lib.q3_lora_add(None, 1, ctypes.byref(lora.Q3Lora()), None) == 5
    # column slices of one buffer are no overlap: these calls get as far as the device
    side = dict(out=(2 << 20) + 128, out_stride=128, base=(6 << 20) + 128, base_stride=128)
    assert add(lib, slice1=dict(side, out_stride=64)) == 5  # the same places with another stride are
    assert add(lib, slice1=dict(out=7 << 20)) not in (1, 2, 5)  # in place


def test_python_refuses_what_is_not_on_the_device():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(q3.Q3Error):
        q3.sample_logits(torch.zeros(2, dtype=torch.int32), x, torch.zeros(2))
    with pytest.raises(q3.Q3Error):
        q3.LoraStack([torch.zeros(2, 8, 16, dtype=torch.bfloat16)], [torch.zeros(2, 16, 8, dtype=torch.bfloat16)])
    with pytest.raises(q3.Q3Error):
        q3.LoraPlan(70000, 2, device="cpu")
    plan = q3.LoraPlan(2, 2, device="cpu")
    with pytest.raises(q3.Q3Error):
        plan.update(torch.zeros(2, dtype=torch.int32))


def server():
    """A server without its device side."""
    s = PagedServer.__new__(PagedServer)
    s.shape, s.adapters = checkpoint.PRESETS["tiny"], None
    s.seqs = Sequences(n_pages=8, page_size=8, max_seqs=4, max_pages=8, chunk=16)
    return s


def test_the_server_checks_what_a_request_chooses():
    s = server()
    a = s.add([1], temperature=0.6, top_k=20, top_p=0.95, min_p=0.01, seed=3)
    assert s.seqs.live[a].temperature == 0.6 and s.seqs.live[a].adapter == -1
    for bad in (dict(temperature=-0.1), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_k=2 ** 31),
                dict(top_p=1.5), dict(top_p=-0.1), dict(top_p=float("nan")), dict(min_p=1.1), dict(min_p=-1.0), dict(adapter=0), dict(adapter=-2)):
        with pytest.raises(ValueError):
            s.add([1], **bad)
    assert list(s.seqs.live) == [a]

    class Loaded:
        loaded = {1}
    s.adapters = Loaded
    assert s.seqs.live[s.add([1], adapter=1)].adapter == 1
    with pytest.raises(ValueError, match="adapter 0"):
        s.add([1], adapter=0)


def test_a_seed_gives_the_same_numbers():
    a, b, c = Sequence([1], seed=5), Sequence([2], seed=5), Sequence([3])
    one = [a.draw() for _ in range(100)]
    assert one == [b.draw() for _ in range(100)] and one != [c.draw() for _ in range(100)]
    assert all(np.float32(u) == u and 0.0 <= u < 1.0 for u in one) and len(set(one)) > 90


def write_adapter(path, shape, r=4, alpha=8, projections=("self_attn.q_proj", "mlp.down_proj"), dtype=torch.float32, seed=0, **cfg):
    """An adapter's directory, and its tensors."""
    g = torch.Generator().manual_seed(seed)
    sizes, tensors, header, blob = adapters.projection_sizes(shape), {}, {}, b""
    for layer in range(shape.num_hidden_layers):
        for p in projections:
            k, n = sizes[p]
            a, b = ((torch.randn(*s, generator=g) * 0.1).to(dtype) for s in ((r, k), (n, r)))
            tensors[layer, p] = a, b
            for which, t in (("lora_A", a), ("lora_B", b)):
                raw = t.view(torch.uint8).numpy().tobytes()
                header[f"base_model.model.model.layers.{layer}.{p}.{which}.weight"] = {
                    "dtype": {torch.float32: "F32", torch.bfloat16: "BF16", torch.float16: "F16"}[dtype], "shape": list(t.shape),
                    "data_offsets": [len(blob), len(blob) + len(raw)]}
                blob += raw
    path.mkdir(exist_ok=True)
    head = json.dumps(header).encode()
    (path / "adapter_model.safetensors").write_bytes(len(head).to_bytes(8, "little") + head + blob)
    (path / "adapter_config.json").write_text(json.dumps(dict(dict(peft_type="LORA", r=r, lora_alpha=alpha, bias="none"), **cfg)))
    return tensors


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_adapter_directories_are_read(tmp_path, dtype):
    shape = checkpoint.PRESETS["tiny"]
    want = write_adapter(tmp_path / "a", shape, dtype=dtype)
    got, scale = adapters.read_adapter(tmp_path / "a", shape)
    assert scale == 2.0 and got.keys() == want.keys()
    assert all(torch.equal(x, y) for key in want for x, y in zip(got[key], want[key]))
    write_adapter(tmp_path / "a", shape, use_rslora=True)
    assert adapters.read_adapter(tmp_path / "a", shape)[1] == 4.0


def test_adapter_directories_are_checked(tmp_path):
    shape, d = checkpoint.PRESETS["tiny"], tmp_path / "a"
    for cfg in (dict(peft_type="IA3"), dict(use_dora=True), dict(bias="all"), dict(rank_pattern={"q": 2}), dict(modules_to_save=["lm_head"]),
                dict(r=8), dict(r="4"), dict(lora_alpha=None)):
        write_adapter(d, shape, **{k: v for k, v in cfg.items() if k not in ("r", "lora_alpha")})
        if "r" in cfg or "lora_alpha" in cfg:  # the file's tensors are of rank 4
            (d / "adapter_config.json").write_text(json.dumps(dict(dict(r=4, lora_alpha=8), **cfg)))
        with pytest.raises(checkpoint.CheckpointError):
            adapters.read_adapter(d, shape)
    write_adapter(d, shape)
    raw = (d / "adapter_model.safetensors").read_bytes()
    n = int.from_bytes(raw[:8], "little")
    name = b"base_model.model.model.layers.0.self_attn.q_proj.lora_A.weight"
    for broken in (raw[:4], raw[:-8], (1 << 40).to_bytes(8, "little") + raw[8:], raw.replace(name, name.replace(b"layers.0", b"layers.9")),
                   raw.replace(name, name.replace(b"q_proj", b"x_proj")), raw.replace(name, name.replace(b"lora_A", b"lora_C")),
                   raw[:8] + raw[8:8 + n].replace(b'"F32"', b'"F64"') + raw[8 + n:]):
        (d / "adapter_model.safetensors").write_bytes(broken)
        with pytest.raises(checkpoint.CheckpointError):
            adapters.read_adapter(d, shape)


def test_the_server_checks_seeds_and_top_k():
    # an error in a step would stop every sequence
    s = server()
    a = s.add([1], temperature=1.0, seed=5, top_k=np.int64(20))
    for bad in (dict(seed=-1), dict(seed="a"), dict(seed=1.5), dict(top_k=0.5), dict(top_k=1.9), dict(top_k="20"), dict(top_k=None)):
        with pytest.raises(ValueError):
            s.add([1], temperature=1.0, **bad)
    assert list(s.seqs.live) == [a] and s.seqs.live[a].top_k == 20
    b = s.add([1], temperature=1.0, seed=5)
    want = Sequence([1], seed=5)
    want = [want.draw() for _ in range(3)]
    assert [s.seqs.live[a].draw() for _ in want] == want and s.seqs.live[b].draw() == want[0]


def test_adapters_of_another_base_or_kind_are_refused(tmp_path):
    shape, d = checkpoint.PRESETS["tiny"], tmp_path / "a"
    for cfg in ([dict(init_lora_weights=v) for v in ("pissa", "pissa_niter_16", "olora", "corda", "loftq", "lora_ga", {}, 2)] +
                [dict(alora_invocation_tokens=[5, 6]), dict(use_qalora=True), dict(arrow_config={"top_k": 3})]):
        write_adapter(d, shape, **cfg)
        with pytest.raises(checkpoint.CheckpointError):
            adapters.read_adapter(d, shape)
    for cfg in ([dict(init_lora_weights=v) for v in (None, True, False, "gaussian", "eva", "orthogonal")] +
                [dict(alora_invocation_tokens=None, use_qalora=False, arrow_config=None)]):
        write_adapter(d, shape, **cfg)
        assert adapters.read_adapter(d, shape)[1] == 2.0


def test_the_server_checks_penalties_and_biases():
    s = server()
    a = s.add([1], repetition=np.float32(1.5), frequency=1, presence=0.5, bias={np.int64(3): 1, -1: -2.0, 10 ** 6: 0.5})
    q = s.seqs.live[a]
    assert (q.repetition, q.frequency, q.presence, q.bias) == (1.5, 1.0, 0.5, {3: 1.0, -1: -2.0, 10 ** 6: 0.5})
    for bad in (dict(repetition="much"), dict(repetition=None), dict(frequency=[1.0, 2.0]), dict(presence={}), dict(bias={2 ** 31: 1.0}),
                dict(bias={"the": 1.0}), dict(bias={3: "a"}), dict(bias={3: None}), dict(bias=[3]), dict(bias=None), dict(temperature="hot"),
                dict(top_p=None), dict(min_p=1j)):
        with pytest.raises(ValueError):
            s.add([1], **bad)
    assert list(s.seqs.live) == [a]
