"""Logits processing on a B200 against its definition in 64 bits.

Tolerance: fp32 operations in the stated order, at most six of them, each off by 2^-24 of its result,
whose magnitude the sum of the terms' magnitudes bounds: 6 * 2^-24 of that sum (2^-21 leaves room), and for
bf16 logits the one rounding at the end, 2^-9 of the result.
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

INF = float("inf")


def exact(x, hists, rep, freq, pres, biases, mask):
    """Row by row over python lists; hists [(prompt ids, generated ids)], biases [{id: value}]."""
    y = x.double().cpu().numpy().copy()
    mag = np.abs(y)
    rows, vocab = y.shape
    for r in range(rows):
        told, said = hists[r] if hists else ([], [])
        times = {}
        for t in said:
            times[t] = times.get(t, 0) + 1
        for t in set(told) | set(said):
            if not 0 <= t < vocab:
                continue
            if rep is not None:
                y[r, t] = y[r, t] / rep[r] if y[r, t] > 0 else y[r, t] * rep[r]
            mag[r, t] = max(mag[r, t], abs(y[r, t]))
            if t in times:
                y[r, t] -= (freq[r] * times[t] if freq is not None else 0.0) + (pres[r] if pres is not None else 0.0)
                mag[r, t] += abs(freq[r] * times[t] if freq is not None else 0.0) + abs(pres[r] if pres is not None else 0.0)
        for t, v in (biases[r] if biases else {}).items():
            if 0 <= t < vocab:
                y[r, t] += v
                mag[r, t] += abs(v)
        if mask is not None:
            for t in range(vocab):
                if not int(mask[r][t // 32]) >> (t % 32) & 1:
                    y[r, t] = -INF
    return y, mag


def check(got, y, mag, what):
    bf = got.dtype == torch.bfloat16
    g = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(g), np.isnan(y)), f"{what}: NaN pattern"
    inf = np.isinf(y)
    assert np.array_equal(g[inf], y[inf]), f"{what}: infinities"
    ok = np.isfinite(y)
    bound = 2.0 ** -21 * mag[ok] + (2.0 ** -8 * np.abs(y[ok]) if bf else 0) + 1e-37
    worst = (np.abs(g - np.where(ok, y, 0))[ok] / bound).max(initial=0.0)
    assert worst <= 1.0, f"{what}: error is {worst:.3f} of the bound"


def make(rows, vocab, dtype, seed, hist=40, n_bias=5, mask=True, stray=True):
    g = np.random.default_rng(seed)
    x = torch.from_numpy(g.normal(0, 3, (rows, vocab)).astype(np.float32)).cuda().to(dtype)
    hists, start, split, ids = [], [0], [], []
    for r in range(rows):
        n = int(g.integers(0, hist + 1)) if r != 1 else 0  # the second row has no history
        both = [int(v) for v in g.integers(-2 if stray else 0, vocab + (2 if stray else 0), n)]
        both += both[:n // 2]
        cut = int(g.integers(0, len(both) + 1))
        hists.append((both[:cut], both[cut:]))
        ids += both
        split.append(start[-1] + cut)
        start.append(start[-1] + len(both))
    bs, bi, bv, biases = [0], [], [], []
    for r in range(rows):
        n = int(g.integers(0, n_bias + 1))
        t = [int(v) for v in g.integers(-1, vocab + 1, n)]
        t += t[:1]  # a repeated id: the last entry counts
        v = [float(np.float32(w)) for w in g.normal(0, 4, len(t))]
        bi += t
        bv += v
        bs.append(len(bi))
        biases.append(dict(zip(t, v)))
    f32 = [g.uniform(0.5, 2, rows).astype(np.float32), g.uniform(-0.5, 1, rows).astype(np.float32),
           g.uniform(-0.5, 1, rows).astype(np.float32)]
    words = (vocab + 31) // 32
    m = g.integers(0, 2 ** 32, (rows, words), dtype=np.uint64).astype(np.uint32) if mask else None

    def i32(a):
        return torch.tensor(a, dtype=torch.int32, device="cuda")

    dev = dict(hist_start=i32(start), hist_split=i32(split), hist_ids=i32(ids),
               repetition=torch.from_numpy(f32[0]).cuda(), frequency=torch.from_numpy(f32[1]).cuda(),
               presence=torch.from_numpy(f32[2]).cuda(), bias_start=i32(bs), bias_ids=i32(bi),
               bias=torch.tensor(bv, dtype=torch.float32, device="cuda"),
               mask=torch.from_numpy(m.view(np.int32)).cuda() if mask else None)
    return x, dev, (hists, *[a.astype(np.float64) for a in f32], biases, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (2, 33), (3, 1000), (5, 8191), (2, 8192), (2, 16385), (3, 20011)])
def test_matches_definition(rows, vocab, dtype):
    x, dev, host = make(rows, vocab, dtype, rows * 7 + vocab)
    out = torch.empty_like(x)
    q3.logits_process(out, x, **dev)
    check(out, *exact(x, *host), f"{rows}x{vocab} {dtype}")
    q3.logits_process(x, x, **dev)  # in place
    assert torch.equal(x.view(torch.uint8), out.view(torch.uint8))
    assert q3.device_error() == 0


@pytest.mark.parametrize("leave_out", ["hist", "repetition", "frequency", "presence", "penalties", "bias", "mask", "all"])
def test_parts_can_be_left_out(leave_out):
    x, dev, (hists, rep, freq, pres, biases, m) = make(3, 5003, torch.bfloat16, 5)
    gone = {"hist": ["hist_start", "hist_split", "hist_ids"], "penalties": ["repetition", "frequency", "presence"],
            "bias": ["bias_start", "bias_ids", "bias"], "all": list(dev)}.get(leave_out, [leave_out])
    dev = {k: None if k in gone else v for k, v in dev.items()}
    out = torch.empty_like(x)
    q3.logits_process(out, x, **dev)
    y, mag = exact(x, hists if dev["hist_start"] is not None else None, rep if dev["repetition"] is not None else None,
                   freq if dev["frequency"] is not None else None, pres if dev["presence"] is not None else None,
                   biases if dev["bias"] is not None else None, m if dev["mask"] is not None else None)
    check(out, y, mag, f"without {leave_out}")
    if leave_out == "all":
        assert torch.equal(out, x)


def test_long_histories_and_counts():
    vocab, rows = 12345, 4
    x, dev, _ = make(rows, vocab, torch.float32, 3, mask=False)
    g = np.random.default_rng(1)
    hists, start, split, ids = [], [0], [], []
    for n in (0, 50000, 70000, 3):
        t = [int(v) for v in g.integers(0, 7, n)] if n != 70000 else [42] * n  # one token 70000 times
        cut = n // 3
        hists.append((t[:cut], t[cut:]))
        ids += t
        split.append(start[-1] + cut)
        start.append(len(ids))
    for k, v in (("hist_start", start), ("hist_split", split), ("hist_ids", ids)):
        dev[k] = torch.tensor(v, dtype=torch.int32, device="cuda")
    for k in ("bias_start", "bias_ids", "bias"):
        dev[k] = None
    out = torch.empty_like(x)
    q3.logits_process(out, x, **dev)
    host = [dev[k].double().cpu().numpy() for k in ("repetition", "frequency", "presence")]
    check(out, *exact(x, hists, *host, None, None), "long histories")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_unaligned_rows(dtype):
    x, dev, host = make(3, 9001, dtype, 8)
    wide = torch.zeros(3, 9001 + 13, dtype=dtype, device="cuda")
    wide[:, 3:9004] = x
    out = torch.full((3, 9500), 5.0, dtype=dtype, device="cuda")
    mask = torch.zeros(3, 300, dtype=torch.int32, device="cuda")
    mask[:, :dev["mask"].shape[1]] = dev["mask"]
    dev["mask"] = mask[:, :290]
    q3.logits_process(out[:, 1:9002], wide[:, 3:9004], **dev)
    check(out[:, 1:9002], *exact(x, *host), "strided")
    assert (out[:, 0] == 5.0).all() and (out[:, 9002:] == 5.0).all()


def test_special_values_and_full_masks():
    vocab = 100
    x = torch.randn(4, vocab, device="cuda")
    x[0, 0], x[0, 1], x[0, 2], x[0, 3], x[0, 4] = INF, -INF, float("nan"), 0.0, -0.0
    mask = torch.full((4, 4), -1, dtype=torch.int32, device="cuda")
    mask[1] = 0  # nothing allowed
    mask[2] = 0
    mask[2, 3] = 1 << 3  # only the last token, 99
    mask[0, 0] = ~(1 << 2)  # the NaN is masked
    i32 = dict(dtype=torch.int32, device="cuda")
    kw = dict(hist_start=torch.tensor([0, 5, 5, 5, 5], **i32), hist_split=torch.tensor([5, 5, 5, 5], **i32),
              hist_ids=torch.tensor([0, 1, 2, 3, 4], **i32), repetition=torch.full((4,), 2.0, device="cuda"))
    out = torch.empty_like(x)
    q3.logits_process(out, x, mask=mask, **kw)
    assert out[0, 0] == INF and out[0, 1] == -INF and out[0, 2] == -INF and out[0, 3] == 0 and out[0, 4] == 0
    assert (out[1] == -INF).all()
    assert (out[2, :99] == -INF).all() and out[2, 99] == x[2, 99]
    assert torch.equal(out[3], x[3])
    q3.logits_process(out, x, **kw)
    assert torch.isnan(out[0, 2])


def test_bad_ranges_are_flagged():
    i32 = dict(dtype=torch.int32, device="cuda")
    x = torch.randn(3, 64, device="cuda")
    out = torch.empty_like(x)
    ids = torch.tensor([1, 2, 3, 4], **i32)
    two = torch.full((3,), 2.0, device="cuda")
    start = torch.tensor([0, 3, 2, 4], **i32)  # the second row's history ends before it starts
    q3.logits_process(out, x, start, torch.tensor([0, 3, 9], **i32), ids, frequency=two)  # the third's split is outside
    assert q3.device_error() == 4
    want = x.clone()
    want[0, 1:4] -= 2.0
    assert torch.equal(out, want)
    q3.logits_process(out, x, bias_start=start, bias_ids=ids, bias=torch.ones(4, device="cuda"))
    assert q3.device_error() == 4


def test_refusals():
    x = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)

    def refuses(status, *a, **kw):
        with pytest.raises(q3.Q3Error) as e:
            q3.logits_process(*a, **kw)
        assert e.value.status == status, e.value

    refuses(1, x, x[:1])
    refuses(5, x.half(), x.half())
    refuses(5, x.float(), x)
    refuses(5, x.t(), x.t())
    refuses(1, x, x, mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    refuses(5, x, x, mask=torch.zeros(2, 2, dtype=torch.int64, device="cuda"))
    refuses(5, x, x, hist_start=torch.zeros(3, dtype=torch.int32, device="cuda"), repetition=torch.ones(2, device="cuda"))
    refuses(1, x, x, hist_start=torch.zeros(2, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("vocab", [64, 5001])
@pytest.mark.parametrize("have,hist,bias", [(4, 5, 3), (4, 2 ** 31 - 1, 4), (4, 4, 5), (4, 3, 2 ** 31 - 1), (0, 1, 0), (0, 0, 1)])
def test_ranges_past_their_arrays_are_flagged(vocab, have, hist, bias):
    # the second row's history or biases end past the arrays: it has none then, the first row has what it says
    i32 = dict(dtype=torch.int32, device="cuda")
    x = torch.randn(2, vocab, device="cuda")
    ids = torch.tensor([1, 2, 3, 4], **i32)[:have]
    own = min(have, 2)
    out = torch.empty_like(x)
    q3.logits_process(out, x, torch.tensor([0, own, hist], **i32), torch.tensor([0, own], **i32), ids,
                      frequency=torch.full((2,), 2.0, device="cuda"), bias_start=torch.tensor([0, own, bias], **i32), bias_ids=ids,
                      bias=torch.full((have,), 8.0, device="cuda"))
    assert q3.device_error() == 4
    want = x.clone()
    for row, (h, b) in enumerate([(own, own), (hist, bias)]):
        lo = [0, own][row]
        if h <= have:
            want[row, ids[lo:h].long()] -= 2.0
        if b <= have:
            want[row, ids[lo:b].long()] += 8.0
    assert torch.equal(out, want)


def test_empty_histories_and_biases():
    i32 = dict(dtype=torch.int32, device="cuda")
    x = torch.randn(3, 100, device="cuda")
    out, zero = torch.empty_like(x), torch.zeros(4, **i32)
    none, two = torch.zeros(0, **i32), torch.full((3,), 2.0, device="cuda")
    q3.logits_process(out, x, zero, zero[:3], none, repetition=two, bias_start=zero, bias_ids=none)
    assert torch.equal(out, x) and q3.device_error() == 0
