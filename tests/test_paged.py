"""Paged serving without a GPU: rotary frequencies, shape support and refusals of the C entries."""
import ctypes
import math
import sys
from pathlib import Path

import numpy as np
import pytest

HERE = Path(__file__).resolve().parent
sys.path.insert(0, str(HERE))
import conftest  # noqa: E402,F401
import llm_inference_b200 as q3  # noqa: E402
from llm_inference_b200 import _lib, build, paged  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()
    return _lib.load()


def plain(d, theta):
    return theta ** (-np.arange(0, d, 2, dtype=np.float64) / d)


def close(got, want):  # one fp32 rounding of a double
    assert got.dtype == np.float32
    assert np.all(np.abs(got - want) <= 2.0 ** -23 * np.abs(want))


@pytest.mark.parametrize("d", [2, 20, 64, 128])
@pytest.mark.parametrize("theta", [1e4, 1e6])
def test_plain_and_linear_frequencies(d, theta):
    f, a = q3.rope_inv_freq(d, theta)
    close(f, plain(d, theta))
    assert a == 1.0
    f, a = q3.rope_inv_freq(d, theta, "linear", factor=4.0)
    close(f, plain(d, theta) / 4)
    assert a == 1.0


def test_frequencies_by_parts():
    f, a = q3.rope_inv_freq(128, 5e5, "by_parts", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                            original_max=8192)
    want = []
    for w in plain(128, 5e5):
        wave = 2 * math.pi / w
        if wave < 8192 / 4:
            want.append(w)
        elif wave > 8192:
            want.append(w / 8)
        else:
            t = (8192 / wave - 1) / 3
            want.append((1 - t) * w / 8 + t * w)
    close(f, np.array(want))
    assert a == 1.0 and want[0] == 1.0 and want[-1] < plain(128, 5e5)[-1]


def test_yarn_frequencies():
    d, theta, factor, orig = 128, 1e6, 4.0, 32768
    f, a = q3.rope_inv_freq(d, theta, "yarn", factor=factor, beta_fast=32.0, beta_slow=1.0, original_max=orig)
    w = plain(d, theta)
    turns = orig * w / (2 * math.pi)
    # pairs that turn more than beta_fast times keep their frequency, those below beta_slow are divided
    low = math.floor(d * math.log(orig / (32 * 2 * math.pi)) / (2 * math.log(theta)))
    high = math.ceil(d * math.log(orig / (2 * math.pi)) / (2 * math.log(theta)))
    ramp = np.clip((np.arange(64) - low) / (high - low), 0, 1)
    close(f, w * (1 - ramp) + w / factor * ramp)
    assert turns[low] >= 32 and turns[min(high, 63)] <= 1
    assert abs(a - (0.1 * math.log(factor) + 1)) < 1e-6
    assert q3.rope_inv_freq(d, theta, "yarn", factor=factor, beta_fast=32.0, beta_slow=1.0, original_max=orig,
                            attention_factor=1.25)[1] == 1.25


@pytest.mark.parametrize("kw", [
    dict(rope_dim=0), dict(rope_dim=7), dict(theta=1.0), dict(theta=float("nan")), dict(kind="linear", factor=0.5),
    dict(kind="linear", factor=float("inf")), dict(kind="by_parts", factor=2.0, low_freq_factor=4.0, high_freq_factor=1.0,
                                                   original_max=10),
    dict(kind="yarn", factor=2.0, beta_fast=1.0, beta_slow=2.0, original_max=10),
    dict(kind="yarn", factor=2.0, beta_fast=32.0, beta_slow=1.0, original_max=0)])
def test_frequencies_refuse(kw):
    kw = dict(dict(rope_dim=64, theta=1e4), **kw)
    with pytest.raises(q3.Q3Error) as e:
        q3.rope_inv_freq(kw.pop("rope_dim"), kw.pop("theta"), **kw)
    assert e.value.status == 1
    with pytest.raises(q3.Q3Error):
        q3.rope_inv_freq(64, 1e4, "unknown")


GOOD = dict(n_seqs=4, n_tokens=9, max_q_len=3, n_heads=32, n_kv_heads=8, head_dim=128, page_size=16, n_pages=100,
            max_pages=20)


@pytest.mark.parametrize("bad", [
    dict(head_dim=136), dict(head_dim=100), dict(head_dim=0), dict(n_kv_heads=5), dict(n_kv_heads=0), dict(n_heads=0),
    dict(n_heads=129, n_kv_heads=1), dict(page_size=12), dict(page_size=0), dict(n_pages=0), dict(max_pages=0),
    dict(n_seqs=-1), dict(n_seqs=4097), dict(n_tokens=-1), dict(max_q_len=-1), dict(max_pages=1 << 28)])
def test_unsupported_shapes(lib, bad):
    good = paged.Q3PagedShape(**GOOD)
    assert lib.q3_paged_plan_bytes(ctypes.byref(good)) > 0
    assert lib.q3_paged_attention_scratch_bytes(ctypes.byref(good)) > 0
    s = paged.Q3PagedShape(**dict(GOOD, **bad))
    assert lib.q3_paged_plan_bytes(ctypes.byref(s)) == 0
    assert lib.q3_paged_attention_scratch_bytes(ctypes.byref(s)) == 0
    fake = 4096  # never dereferenced: refused before any launch
    assert lib.q3_paged_plan(fake, ctypes.byref(s), fake, fake, fake, None) == 1
    c = paged.Q3PagedCache(fake, fake, 16 * 8 * 128, 16 * 128, 128)
    assert lib.q3_paged_attention(fake, 1 << 20, fake, 1 << 20, ctypes.byref(c), 0.1, ctypes.byref(s), fake, fake, None) == 1


def attention(lib, **kw):
    fake = 4096
    a = dict(out=fake, out_stride=4096, q=fake, q_stride=4096, kp=fake, vp=fake, page=16 * 8 * 128, head=16 * 128,
             pos=128, plan=fake, scratch=fake)
    a.update(kw)
    c = paged.Q3PagedCache(a["kp"], a["vp"], a["page"], a["head"], a["pos"])
    s = paged.Q3PagedShape(**GOOD)
    return lib.q3_paged_attention(a["out"], a["out_stride"], a["q"], a["q_stride"], ctypes.byref(c), 0.1,
                                  ctypes.byref(s), a["plan"], a["scratch"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(out=None), 5), (dict(q=None), 5), (dict(kp=None), 5), (dict(vp=None), 5), (dict(plan=None), 5),
    (dict(scratch=None), 5), (dict(q_stride=4088), 1), (dict(out_stride=0), 1), (dict(page=0), 1), (dict(pos=-128), 1),
    (dict(q=4098), 2), (dict(kp=4104), 2), (dict(head=4), 2), (dict(out_stride=4100), 2), (dict(plan=4097), 2)])
def test_attention_refuses(lib, kw, status):
    assert attention(lib, **kw) == status


def append(lib, **kw):
    fake = 4096
    a = dict(q_out=8192, q_out_stride=4096, q=fake, q_stride=4096, k=fake, k_stride=1024, v=fake, v_stride=1024, qw=fake,
             kw=fake, f=fake, rope=128, pos=128, plan=fake)
    a.update(kw)
    c = paged.Q3PagedCache(fake, fake, 16 * 8 * 128, 16 * 128, a["pos"])
    s = paged.Q3PagedShape(**GOOD)
    return lib.q3_paged_rope_append(a["q_out"], a["q_out_stride"], a["q"], a["q_stride"], a["k"], a["k_stride"], a["v"],
                                    a["v_stride"], a["qw"], a["kw"], 1e-6, a["f"], a["rope"], 0, 1.0, ctypes.byref(c),
                                    ctypes.byref(s), a["plan"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(q_out=None), 5), (dict(k=None), 5), (dict(v=None), 5), (dict(plan=None), 5), (dict(f=None), 5),
    (dict(rope=130), 1), (dict(rope=-2), 1), (dict(rope=63), 1), (dict(k_stride=1016), 1), (dict(pos=0), 1),
    (dict(q_out=4096, q_out_stride=8192), 1), (dict(qw=4100), 2), (dict(k_stride=1028), 2), (dict(v=4100), 2)])
def test_append_refuses(lib, kw, status):
    assert append(lib, **kw) == status


def logits(lib, **kw):
    fake = 4096
    a = dict(out=fake, x=fake, dtype=0, rows=2, vocab=1000, out_stride=1000, stride=1000, hs=fake, hp=fake, hi=fake,
             bs=fake, bi=fake, b=fake, mask=fake, ms=32)
    a.update(kw)
    return lib.q3_logits_process(a["out"], a["x"], a["dtype"], a["rows"], a["vocab"], a["out_stride"], a["stride"],
                                 a["hs"], a["hp"], a["hi"], fake, fake, fake, a["bs"], a["bi"], a["b"], a["mask"],
                                 a["ms"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(out=None), 5), (dict(x=None), 5), (dict(dtype=2), 5), (dict(hp=None), 5), (dict(hi=None), 5), (dict(bi=None), 5),
    (dict(b=None), 5), (dict(rows=-1), 1), (dict(rows=65536), 1), (dict(vocab=0), 1), (dict(stride=999), 1),
    (dict(out_stride=999), 1), (dict(out_stride=1001), 1), (dict(ms=31), 1), (dict(out=4097), 2),
    (dict(x=4098, dtype=1, out=8192), 2)])
def test_logits_refuse(lib, kw, status):
    assert logits(lib, **kw) == status


def test_a_plan_is_refused_before_its_first_update():
    plan = q3.PagedPlan(*GOOD.values(), device="cpu")
    assert not plan.plan.any()
    for call in (lambda: q3.paged_attention(None, None, None, None, plan),
                 lambda: q3.paged_rope_append(None, None, None, None, None, None, plan)):
        with pytest.raises(q3.Q3Error, match="has not been updated") as e:
            call()
        assert e.value.status == 5


@pytest.mark.parametrize("n_hist,n_bias,status", [(-1, 5, 1), (5, -1, 1), (-1, -1, 1)])
def test_logits_refuse_negative_lengths(lib, n_hist, n_bias, status):
    fake = 4096
    assert lib.q3_logits_process_bounded(fake, fake, 0, 2, 1000, 1000, 1000, fake, fake, fake, n_hist, fake, fake, fake, fake,
                                         fake, fake, n_bias, None, 0, None) == status


class Elsewhere:
    """As much of a tensor as the checks look at; on GPU `device`, and without any memory."""

    def __init__(self, shape, dtype, device):
        self.shape, self.dtype, self.device, self.is_cuda = shape, dtype, device, True

    def get_device(self):
        return self.device

    def numel(self):
        return math.prod(self.shape)

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def stride(self, i=None):
        steps = tuple(math.prod(self.shape[j + 1:]) for j in range(len(self.shape)))
        return steps if i is None else steps[i]

    def data_ptr(self):
        return 4096  # never dereferenced: refused before any launch


def test_tensors_of_another_device_are_refused(monkeypatch):
    import torch
    paged._t()
    monkeypatch.setattr(paged, "_device", lambda: 0)
    monkeypatch.setattr(paged, "_raw_stream", lambda device: 0)
    bf, i32, f32 = torch.bfloat16, torch.int32, torch.float32
    plan = q3.PagedPlan(*GOOD.values(), device="cpu")
    plan._on, plan._updated = 0, True
    launched = []
    monkeypatch.setattr(paged, "call", lambda *a: launched.append(a[0]))

    class Lib:
        def __getattr__(self, name):
            return lambda *a: launched.append(name)

    monkeypatch.setattr(paged, "load", Lib)

    def tensors(which, away):
        return {k: Elsewhere(shape, dtype, 1 if k == away else 0) for k, (shape, dtype) in which.items()}

    pages, q, kv = ((100, 8, 16, 128), bf), ((9, 4096), bf), ((9, 1024), bf)
    calls = [
        (lambda t: plan.update(*t.values()), dict(q_start=((5,), i32), kv_len=((4,), i32), table=((4, 20), i32))),
        (lambda t: q3.paged_attention(*t.values(), plan), dict(out=q, q=q, key_pages=pages, value_pages=pages)),
        (lambda t: q3.paged_rope_append(*[t[k] for k in ("q_out", "q", "k", "v", "key_pages", "value_pages")], plan, t["inv_freq"],
                                        t["q_norm_w"], t["k_norm_w"]),
         dict(q_out=q, q=q, k=kv, v=kv, key_pages=pages, value_pages=pages, inv_freq=((64,), f32), q_norm_w=((128,), bf),
              k_norm_w=((128,), bf))),
        (lambda t: q3.logits_process(**t),
         dict(out=((3, 64), f32), logits=((3, 64), f32), hist_start=((4,), i32), hist_split=((3,), i32), hist_ids=((9,), i32),
              repetition=((3,), f32), frequency=((3,), f32), presence=((3,), f32), bias_start=((4,), i32), bias_ids=((5,), i32),
              bias=((5,), f32), mask=((3, 2), i32)))]
    for go, which in calls:
        launched.clear()
        go(tensors(which, None))
        assert len(launched) == 1
        for away in which:
            with pytest.raises(q3.Q3Error) as e:
                go(tensors(which, away))
            assert e.value.status == 5, away
        assert len(launched) == 1
    plan._on = 1
    for go, which in calls[:3]:
        with pytest.raises(q3.Q3Error, match="another device") as e:
            go(tensors(which, None))
        assert e.value.status == 5


# tensors of no elements have no address
def test_calls_without_rows_do_nothing(lib):
    fake = 4096
    c = paged.Q3PagedCache(fake, fake, 16 * 8 * 128, 16 * 128, 128)
    s = paged.Q3PagedShape(**dict(GOOD, n_tokens=0))
    assert lib.q3_paged_attention(None, 4096, None, 4096, ctypes.byref(c), 0.1, ctypes.byref(s), fake, fake, None) == 0
    assert lib.q3_paged_rope_append(None, 4096, None, 4096, None, 1024, None, 1024, None, None, 1e-6, fake, 128, 0, 1.0,
                                    ctypes.byref(c), ctypes.byref(s), fake, None) == 0
    assert logits(lib, rows=0, out=None, x=None) == 0
    # without sequences, a plan is not refused for its null lengths and page table (but for its alignment), and still is
    # for a null start
    none = paged.Q3PagedShape(**dict(GOOD, n_seqs=0, n_tokens=0))
    assert lib.q3_paged_plan(4097, ctypes.byref(none), fake, None, None, None) == 2
    assert lib.q3_paged_plan(fake, ctypes.byref(none), None, None, None, None) == 5
    assert lib.q3_paged_plan(fake, ctypes.byref(s), fake, None, fake, None) == 5
