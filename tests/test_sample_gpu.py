"""Sampling from given random numbers on a B200 against its definition in 64 bits.

A token has to be the one whose interval of the running mass holds u M. Weights are off by 2^-42 of the largest at most
(and 3e-13 of themselves), so borders of the running mass by vocab * 2^-42 + 3e-13 M: a target closer than that to a border may fall
on either side of it. Probabilities: one fp32 rounding, 2^-24, and the weights' errors.
"""
import sys
from decimal import Decimal, getcontext
from pathlib import Path

import numpy as np
import pytest

HERE = Path(__file__).resolve().parent
sys.path.insert(0, str(HERE))
import conftest  # noqa: E402,F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llm_inference_b200 as q3  # noqa: E402

INF, NAN = float("inf"), float("nan")


def exact_row(x, u, t=1.0, k=0, p=1.0, floor=0.0, draft=-1):
    """(tokens in order, kept weights in order, their sum, target) or None for a row without tokens; x float64."""
    x = np.where(np.isnan(x), -INF, x)
    order = np.argsort(-x, kind="stable")
    if x[order[0]] == -INF:
        return None
    if not t > 0:
        return order[:1], np.ones(1), 1.0, 0.0
    order = order[x[order] > -INF]
    z = x[order]
    with np.errstate(invalid="ignore"):
        w = np.where(z == z[0], 1.0, np.exp((z - z[0]) / t))
    w = np.where(np.isnan(w), 0.0, w)  # beside an infinite logit, at an infinite temperature, too
    n = len(order) if k <= 0 else min(k, len(order))
    if p < 1:
        ends = np.cumsum(w[:n])
        n = 1 + int(np.sum(ends < max(p, 0.0) * ends[-1]))
    if floor > 0:
        n = min(n, max(1, int(np.sum(w >= min(floor, 1.0)))))
    order, w = order[:n], w[:n]
    if draft in order.tolist():
        j = order.tolist().index(draft)
        order, w = (np.concatenate([a[j:j + 1], a[:j], a[j + 1:]]) for a in (order, w))
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    return order, w, w.sum(), u * w.sum()


def check(x, out, prob, u, t=None, k=None, p=None, floor=None, draft=None):
    x64, vocab = x.double().cpu().numpy(), x.shape[1]

    def host(a, default):
        return [default] * x.shape[0] if a is None else a.tolist()

    columns = zip(host(t, 1.0), host(k, 0), host(p, 1.0), host(floor, 0.0), host(draft, -1))
    for r, (tt, kk, pp, ff, dd) in enumerate(columns):
        token, got = out[r].item(), prob[r].item()
        want = exact_row(x64[r], u[r].item(), tt, kk, pp, ff, dd)
        if want is None:
            assert token == -1 and got == 0.0
            continue
        order, w, total, target = want
        assert token in order, f"row {r}: token {token} is cut off"
        at = order.tolist().index(token)
        before, room = w[:at].sum(), vocab * 2.0 ** -42 + 3e-13 * total
        assert before - room <= target <= before + w[at] + room, f"row {r}: token {token} has {before}, {w[at]} and u M is {target}"
        share = w[at] / total
        assert abs(got - share) <= 2.0 ** -24 * share + 2 * room / total, f"row {r}: probability {got}, not {share}"


def run(x, u, t=None, k=None, p=None, floor=None, draft=None):
    out = torch.full((x.shape[0],), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((x.shape[0],), -7.0, device="cuda")
    q3.sample_logits(out, x, u, t, k, p, floor, draft=draft, prob=prob)
    check(x, out, prob, u, t, k, p, floor, draft)
    return out, prob


def f32(*v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def settings(rows, vocab, g):
    """Rows of every kind: none, each limit alone, all of them, greedy."""
    t = g.uniform(0.3, 2.0, rows)
    k = np.where(g.random(rows) < 0.5, g.integers(1, max(2, vocab), rows), 0)
    p = np.where(g.random(rows) < 0.5, g.uniform(0, 1, rows), 1.0)
    m = np.where(g.random(rows) < 0.4, g.uniform(0, 0.3, rows), 0.0)
    t[::7] = 0.0
    d = np.where(g.random(rows) < 0.5, g.integers(0, vocab, rows), -1)
    return f32(*t), i32(*k), f32(*p), f32(*m), i32(*d)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (70, 7), (64, 33), (33, 1000), (9, 5003), (21, 32003), (5, 70001), (1, 151936),
                                        (19, 151936), (150, 4099)])
def test_matches_definition(rows, vocab, dtype):
    g = np.random.default_rng(rows * 1000 + vocab)
    x = torch.from_numpy(g.normal(0, 2.5, (rows, vocab)).astype(np.float32)).cuda().to(dtype)
    t, k, p, m, d = settings(rows, vocab, g)
    likely = x.argmax(1).to(torch.int32)
    d[1::3] = likely[1::3]
    u = f32(*g.random(rows))
    run(x, u)
    run(x, u, t, k, p, m)
    run(x, u, t, k, p, m, d)
    run(x, u, draft=d)
    for part in ("t", "k", "p", "floor"):
        run(x, u, **{part: {"t": t, "k": k, "p": p, "floor": m}[part]})


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [513, 4000, 40000])
def test_many_equal_logits(vocab, dtype):
    # whole rows of one value, of two, of a few, and a plateau under a peak: told apart by index
    g = np.random.default_rng(vocab)
    rows = 8
    x = torch.zeros(rows, vocab, device="cuda")
    x[1] = -3.5
    x[2] = torch.from_numpy(g.integers(0, 2, vocab).astype(np.float32))
    x[3] = torch.from_numpy(g.integers(-2, 2, vocab) * 0.25)
    x[4, vocab // 2] = 4.0
    x[5, ::2] = -0.0  # equal to 0
    x[6] = torch.from_numpy(np.float32(1) + g.integers(0, 3, vocab) * np.float32(2.0 ** -7))
    x[7] = -INF
    x[7, 3::5] = 1.25
    x = x.to(dtype)
    for u in (0.0, 0.37, 0.93, 1 - 2.0 ** -24):
        uu = torch.full((rows,), u, device="cuda")
        run(x, uu)
        run(x, uu, k=i32(*g.integers(1, vocab, rows)))
        run(x, uu, p=f32(*g.uniform(0.01, 0.99, rows)))
        run(x, uu, k=i32(*g.integers(1, vocab, rows)), p=f32(*g.uniform(0.01, 0.99, rows)), draft=i32(*g.integers(0, vocab, rows)))
    out, _ = run(x, torch.zeros(rows, device="cuda"))
    assert out.tolist() == [0, 0, *(int(x[r].float().argmax()) for r in (2, 3, 4)), 0, int(x[6].float().argmax()), 3]


def test_close_logits_far_below_their_range():
    # nearly all tokens within 2^-20 of one another, one far above and one far below: the first bins cannot part them
    vocab = 30000
    g = np.random.default_rng(3)
    base = (np.float32(1.0) + g.integers(0, 40, (4, vocab)).astype(np.float32) * np.float32(2.0 ** -23)).astype(np.float32)
    base[1, 5], base[2, 5], base[3, 7] = 9.0, -60.0, 11.0
    base[3, 9] = -100.0
    x = torch.from_numpy(base).cuda()
    for u in (0.02, 0.5, 0.98):
        run(x, torch.full((4,), u, device="cuda"), p=f32(0.9, 0.9999, 0.8, 0.99))
        run(x, torch.full((4,), u, device="cuda"), t=f32(1e6, 1e6, INF, INF))
        run(x, torch.full((4,), u, device="cuda"), t=f32(1e-6, 1e-7, 1e-30, 1e-38), k=i32(0, 100, 5, 0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_and_nan(dtype):
    vocab = 3001
    x = torch.randn(8, vocab, device="cuda")
    x[0] = -INF
    x[1] = NAN
    x[2] = -INF
    x[2, 77] = -5.0
    x[3, 5:2000] = NAN
    x[4, [9, 800, 2900]] = INF
    x[5, 100:] = -INF
    x[6, 0], x[6, 1] = NAN, 50.0
    x[7] = torch.finfo(dtype).min  # the lowest value stands for a mask in many programs
    x[7, 40] = 0.0
    x = x.to(dtype)
    for u in (0.0, 0.4, 0.999):
        uu = torch.full((8,), u, device="cuda")
        out, prob = run(x, uu)
        assert out[:3].tolist() == [-1, -1, 77] and out[7] == 40 and prob[7] == 1.0
        assert out[4].item() == {0.0: 9, 0.4: 800, 0.999: 2900}[u]
        run(x, uu, t=f32(*[0.0] * 8))
        run(x, uu, t=f32(*[INF] * 8))
        run(x, uu, k=i32(*[2] * 8), p=f32(*[0.9] * 8), draft=i32(3, 3, 3, 5, 9, 200, 0, 40))


def test_settings_outside_their_ranges():
    vocab = 500
    x = torch.randn(6, vocab, device="cuda") * 3
    u = f32(0.5, -1.0, NAN, 1.0, INF, 0.5)
    top = x.argmax(1).tolist()
    out, prob = run(x, u)
    assert out[1:3].tolist() == top[1:3]
    out, prob = run(x, u, t=f32(-1.0, NAN, -INF, 0.0, -0.0, -1e-30))
    assert out.tolist() == top and (prob == 1).all()
    out, _ = run(x, u, p=f32(0.0, -1.0, 0.0, -INF, 1e-30, 0.0))
    assert out.tolist() == top
    out, _ = run(x, u, floor=f32(*[2.0] * 6))
    assert out.tolist() == top
    free, _ = run(x, u)
    same, _ = run(x, u, k=i32(0, -3, vocab, vocab + 5, 2 ** 31 - 1, -2 ** 31), p=f32(1.0, 2.0, INF, 1.0, 1.0, 1.0),
                  floor=f32(0.0, -1.0, -INF, 0.0, 0.0, 0.0), draft=i32(-1, vocab, 2 ** 31 - 1, -2 ** 31, -5, vocab + 1))
    assert torch.equal(free, same)
    out, _ = run(x, u, p=torch.full((6,), NAN, device="cuda"), floor=torch.full((6,), NAN, device="cuda"))
    assert torch.equal(free, out)


def test_drafts_keep_the_distribution():
    # a grid of u: each token comes out as often as its probability says, with a draft and without, to one grid point a border
    vocab, n = 12, 4096
    x = torch.linspace(-1, 2, vocab, device="cuda")[torch.randperm(vocab, generator=torch.Generator().manual_seed(1)).cuda()]
    u = (torch.arange(n, device="cuda") + 0.5) / n
    rows = x.expand(n, vocab).contiguous()
    p = torch.softmax(x.double(), 0)
    for d in (-1, 0, 5, 11):
        out, _ = run(rows, u, draft=torch.full((n,), d, dtype=torch.int32, device="cuda"))
        share = torch.bincount(out.long(), minlength=vocab).double() / n
        assert (share - p).abs().max() <= 2 / n
        if d >= 0:  # the draft is accepted for the first values of u
            assert torch.equal(out == d, u.double() < p[d])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_unaligned_rows(dtype):
    g = np.random.default_rng(5)
    x = torch.from_numpy(g.normal(0, 3, (5, 9001)).astype(np.float32)).cuda().to(dtype)
    t, k, p, m, d = settings(5, 9001, g)
    u = f32(*g.random(5))
    want, prob = run(x, u, t, k, p, m, d)
    for lead in range(1, 8):
        wide = torch.full((5, 9001 + 13), 99.0, dtype=dtype, device="cuda")  # what is beside a row is larger than all of it
        wide[:, lead:9001 + lead] = x
        got, pr = run(wide[:, lead:9001 + lead], u, t, k, p, m, d)
        assert torch.equal(got, want) and torch.equal(pr, prob)


def test_rows_do_not_depend_on_their_neighbours():
    # a row alone, in a batch and in a larger one is cut among other numbers of CTAs
    g = np.random.default_rng(6)
    x = torch.from_numpy(g.normal(0, 2, (200, 20001)).astype(np.float32)).cuda()
    t, k, p, m, d = settings(200, 20001, g)
    u = f32(*g.random(200))
    all_, prob = torch.empty(200, dtype=torch.int32, device="cuda"), torch.empty(200, device="cuda")
    q3.sample_logits(all_, x, u, t, k, p, m, draft=d, prob=prob)
    for n in (1, 30, 60):
        out, pr = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda")
        q3.sample_logits(out, x[:n], u[:n], t[:n], k[:n], p[:n], m[:n], draft=d[:n], prob=pr)
        assert torch.equal(out, all_[:n]) and torch.equal(pr, prob[:n])


def test_captured_with_logits_process_and_on_another_stream():
    g = np.random.default_rng(7)
    x = torch.from_numpy(g.normal(0, 2, (4, 30011)).astype(np.float32)).cuda().to(torch.bfloat16)
    u, t = f32(*g.random(4)), f32(0.7, 1.0, 0.0, 1.3)
    bias_start, bias_ids = i32(0, 1, 2, 3, 4), i32(5, 6, 7, 8)
    bias, y = f32(1.0, 2.0, 3.0, 4.0), torch.empty_like(x)
    out, prob = torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, device="cuda")

    def step():
        q3.logits_process(y, x, bias_start=bias_start, bias_ids=bias_ids, bias=bias)
        q3.sample_logits(out, y, u, t, prob=prob)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    check(y, out, prob, u, t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        u.copy_(f32(*g.random(4)))
        bias.copy_(f32(*g.normal(0, 10, 4)))
        graph.replay()
        check(y, out, prob, u, t)


def test_refusals():
    x, u = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(2, device="cuda")
    out = torch.zeros(2, dtype=torch.int32, device="cuda")

    def refuses(status, *a, **kw):
        with pytest.raises(q3.Q3Error) as e:
            q3.sample_logits(*a, **kw)
        assert e.value.status == status, e.value

    refuses(5, out, x.half(), u)
    refuses(5, out, torch.zeros(64, 2, device="cuda", dtype=torch.bfloat16).t(), u)
    refuses(1, out, x[:1].expand(2, 64), u)
    refuses(1, out, x[0], u)
    refuses(5, out.long(), x, u)
    refuses(1, out[:1], x, u)
    refuses(5, out, x, u.double())
    refuses(1, out, x, u[:1])
    refuses(5, out, x, u, u.double())
    refuses(5, out, x, u, None, u)
    refuses(1, out, x, u, draft=out[:1])
    refuses(1, out, x, u, prob=u[:1])
    refuses(1, out, torch.zeros(2, 1048577, device="cuda", dtype=torch.bfloat16), u)
    refuses(1, out, torch.zeros(2, 1048577, device="cuda"), u)
    refuses(5, out, x.cpu(), u)
    refuses(5, out, x, u.cpu())
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    q3.sample_logits(none, x[:0], u[:0], u[:0])  # no rows: nothing to do


def test_the_largest_vocabularies():
    for vocab, dtype in ((1048576, torch.bfloat16), (1048576, torch.float32)):
        g = np.random.default_rng(vocab)
        x = torch.from_numpy(g.normal(0, 2, (2, vocab)).astype(np.float32)).cuda().to(dtype)
        run(x, f32(0.3, 0.9))
        run(x, f32(0.3, 0.9), k=i32(1000, 0), p=f32(0.5, 0.9))


@pytest.mark.parametrize("scale,shift,t", [(200.0, 0.0, 40.0), (3.0, 500.0, 1.0), (3.0, -500.0, 0.8), (1e-11, 0.0, 1e-11), (1e-11, 3.0, 1.0),
                                           (1e30, 0.0, 3e29), (1e-38, 0.0, 1e-38), (3.0, 0.0, 1.0)])
def test_bf16_rows_of_any_magnitude(scale, shift, t):
    # most rows' logits lie where bf16 values are counted one by one; these are beside it, around it and across its borders
    g = np.random.default_rng(8)
    vocab = 6007
    x = torch.from_numpy((g.normal(0, 1, (12, vocab)) * scale + shift).astype(np.float32)).cuda()
    x[1::3, ::7] = -3e38
    x[2::3, ::5] = 0.0
    x[3::4, 11] = 2.0 ** -32 * 0.75
    x = x.to(torch.bfloat16)
    _, k, p, m, d = settings(12, vocab, g)
    for u in (f32(*g.random(12)), f32(*[0.0] * 12)):
        run(x, u, f32(*[t] * 12))
        run(x, u, f32(*[t] * 12), k, p, m, d)
        run(x, u, f32(*[0.0] * 12))


def test_two_calls_at_once():
    g = np.random.default_rng(9)
    x = torch.from_numpy(g.normal(0, 2, (6, 50021)).astype(np.float32)).cuda()
    t, k, p, m, d = settings(6, 50021, g)
    u = f32(*g.random(6))
    want, _ = run(x, u, t, k, p, m, d)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [[torch.empty(6, dtype=torch.int32, device="cuda") for _ in range(8)] for _ in streams]
    torch.cuda.synchronize()
    for n in range(8):
        for s, out in zip(streams, outs):
            with torch.cuda.stream(s):
                q3.sample_logits(out[n], x, u, t, k, p, m, draft=d)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for out in outs for o in out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 40000, 151936])
def test_greedy_rows_take_the_first_of_the_largest(vocab, dtype):
    # wherever its equals lie among the parts of a row; rows of one sign of zero and the other; beside NaN and -infinity
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(8, vocab, generator=g).clamp(max=3.0)
    want = torch.randint(0, vocab, (8,), generator=g)
    for r in range(8):
        x[r, want[r]:][torch.rand(vocab - want[r], generator=g) < 0.3] = 3.5
        x[r, want[r]] = 3.5
    x[5] = NAN
    x[5, want[5]:] = -INF
    x[5, want[5]] = -1e30
    x[6] = -INF
    x[6, want[6]:] = 0.0
    x[6, want[6]] = -0.0
    x[7] = -1000.0
    want[7] = 0
    x = x.cuda().to(dtype)
    out, prob = run(x, f32(*[0.999] * 8), t=f32(*[0.0] * 8), k=i32(*[3] * 8), draft=i32(*[vocab - 1] * 8))
    assert out.tolist() == want.tolist() and prob.tolist() == [1.0] * 8


@pytest.mark.parametrize("unit", [1, 3, 4096])
def test_zeros_above_subnormal_logits(unit):
    # more tokens than are ranked directly share a bin with exact zeros and lie below them: cut by the bits of their keys, the bins'
    # ends meet at the key of -0, which no logit has. Shuffled, and with top-k and top-p ends among them.
    tiny = 2.0 ** -149
    row = np.concatenate([[1.0, -1.0, 0x1fffff * tiny], np.zeros(50), -np.arange(1, 301) * tiny * unit, [-0x1fffff * tiny]]).astype(np.float32)
    row[3::7][:5] = -0.0
    g, n = np.random.default_rng(unit), 400
    x = torch.from_numpy(np.stack([row, *(g.permutation(row) for _ in range(n - 1))])).cuda()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    run(x, u)
    run(x, u, k=i32(*g.integers(2, 360, n)), p=f32(*g.uniform(0.2, 1.0, n)))
    run(x, u, t=f32(*g.uniform(0.5, 2.0, n)), draft=i32(*g.integers(0, 354, n)))


def test_weights_hold_their_bound():
    # rows of the logits 0 and x: top-p keeps the second one if its weight passes 1 / p - 1, from which it is more than 2^-42 away in
    # each of these; u takes the last one kept
    getcontext().prec = 50
    rows = [[float.fromhex(v) for v in row] for row in (
        ("-0x1.4c8994p-1", "0x1.fb79dep+0", "0x1.29910ap-1"), ("-0x1.4f4aap-1", "0x1.f332c8p+0", "0x1.2a9634p-1"),
        ("-0x1.d8946ap-2", "0x1.57d3ecp+0", "0x1.2b8e22p-1"), ("-0x1.ba55fcp-2", "0x1.448a1cp+0", "0x1.2b329ep-1"),
        ("-0x1.f8b25ep-2", "0x1.70bf7ep+0", "0x1.2b6012p-1"), ("-0x1.8639f6p-2", "0x1.1f39c4p+0", "0x1.2b0fecp-1"),
        ("-0x1.da3664p-3", "0x1.66f1acp-1", "0x1.29e564p-1"), ("-0x1.e66682p-3", "0x1.6164ccp-1", "0x1.2b9d46p-1"),
        ("-0x1.473e14p-1", "0x1.ee64e4p+0", "0x1.29fac2p-1"), ("-0x1.2c5ea4p-1", "0x1.cd0d14p+0", "0x1.29549ap-1"))]
    rows += [[x, t, p + 2.0 ** -24] for x, t, p in rows]  # and on the border's other side
    want = []
    for x, t, p in rows:
        past = (Decimal(x) / Decimal(t)).exp() - (1 / Decimal(p) - 1)
        assert abs(past) * 2 ** 42 > Decimal("1.05")
        want.append(int(past > 0))
    x = torch.tensor([[0.0, r[0]] for r in rows], dtype=torch.float32, device="cuda")
    assert want == [0] * 10 + [1] * 10
    out = torch.empty(len(rows), dtype=torch.int32, device="cuda")
    q3.sample_logits(out, x, f32(*[1 - 2.0 ** -24] * len(rows)), f32(*(r[1] for r in rows)), top_p=f32(*(r[2] for r in rows)))
    assert out.tolist() == want
