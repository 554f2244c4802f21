"""Adapters of many requests on a B200 against their definition in 64 bits.

Tolerance of out = base + s B (A x). The output's rounding is at most 2^-9 of it. A x is a sum of k products in fp32, off by at most
(k + 8) 2^-24 of sum |a x| (8: sums of partial sums), its two bf16 parts hold it to 2^-17 (each rounds to half a step of
8 bits), and the second sum of rank products in two parts, with the base, is off by at most (2 rank + 8) 2^-24 of its terms'
magnitudes. With D = |s| sum_r |b_r| sum_k |a_rk x_k|, which bounds all of these terms:
    2^-8 |out| (twice the half step) + ((k + 2 rank + 16) 2^-24 + 2^-16) D + 2^-23 |base|.
For act = silu(g) u both factors carry such errors e_g, e_u (without the output's rounding), |silu'| is at most 1.1, and its
evaluation is off by 2^-20 of it: 2^-8 |act| + 1.1 e_g |u| + |silu(g)| e_u + 1.1 e_g e_u + 2^-18 |act|.
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

BF16, NAN = torch.bfloat16, float("nan")


def normal(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(BF16).cuda()


class Case:
    """Adapters and rows; ranks: of each adapter, what is past them in a and b is NaN."""

    def __init__(self, rows, k, ns, rank, n_adapters, index, seed=0, ranks=None, scale=True):
        g = torch.Generator().manual_seed(seed)
        self.k, self.ns, self.rank, self.n_adapters, self.index = k, ns, rank, n_adapters, list(index)
        self.x = normal(g, rows, k)
        self.a = [normal(g, n_adapters, rank, k, std=k ** -0.5) for _ in ns]
        self.b = [normal(g, n_adapters, n, rank, std=rank ** -0.5) for n in ns]
        self.base = [normal(g, rows, n) for n in ns]
        self.scale = (torch.rand(n_adapters, generator=g) * 3 - 1).cuda() if scale else None
        self.ranks = ranks
        if ranks is not None:
            for i, r in enumerate(ranks):
                for t in self.a:
                    t[i, max(r, 0):] = NAN
                for t in self.b:
                    t[i, :, max(r, 0):] = NAN
        self.index_d = torch.tensor(self.index, dtype=torch.int32, device="cuda")
        self.ranks_d = None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device="cuda")
        self.stack = q3.LoraStack(self.a, self.b, self.scale, self.ranks_d)
        self.plan = q3.LoraPlan(rows, n_adapters)
        self.plan.update(self.index_d)

    def exact(self, j):
        """(base + delta, bound of the error before the output's rounding) of projection j."""
        base = self.base[j].double()
        y, mag = base.clone(), torch.zeros_like(base)
        for i in set(self.index):
            if not 0 <= i < self.n_adapters:
                continue
            r = self.rank if self.ranks is None else min(max(self.ranks[i], 0), self.rank)
            at = torch.tensor([n for n, v in enumerate(self.index) if v == i], device="cuda")
            s = 1.0 if self.scale is None else self.scale[i].double()
            a, b, x = self.a[j][i, :r].double(), self.b[j][i, :, :r].double(), self.x[at].double()
            y[at] += s * (x @ a.T) @ b.T
            mag[at] = abs(s) * (x.abs() @ a.abs().T) @ b.abs().T
        return y, ((self.k + 2 * self.rank + 16) * 2.0 ** -24 + 2.0 ** -16) * mag + 2.0 ** -23 * base.abs()

    def check_add(self, outs):
        for j, out in enumerate(outs):
            y, bound = self.exact(j)
            err = (out.double() - y).abs()
            bad = err > bound + 2.0 ** -8 * y.abs() + 1e-37
            assert not bad.any(), f"projection {j}: {bad.sum().item()} of {bad.numel()}, worst {(err / (bound + 2.0 ** -8 * y.abs())).max().item():.2f}"
            bare = torch.tensor([not 0 <= i < self.n_adapters for i in self.index], device="cuda")
            assert torch.equal(out[bare], self.base[j][bare])

    def check_gate_up(self, act, before):
        (g, eg), (u, eu) = self.exact(0), self.exact(1)
        silu = g / (1 + torch.exp(-g))
        y = silu * u
        bound = (2.0 ** -8 + 2.0 ** -18) * y.abs() + 1.1 * eg * u.abs() + silu.abs() * eu + 1.1 * eg * eu + 1e-37
        bare = torch.tensor([not 0 <= i < self.n_adapters for i in self.index], device="cuda")
        err = (act.double() - y).abs()
        assert (err <= bound)[~bare].all(), (err / bound)[~bare].max().item()
        assert torch.equal(act[bare], before[bare])

    def add(self):
        outs = [torch.full_like(t, NAN) for t in self.base]
        q3.lora_add(outs, self.base, self.x, self.stack, self.plan)
        self.check_add(outs)
        return outs

    def gate_up(self):
        before = normal(torch.Generator().manual_seed(9), *self.base[0].shape)
        act = before.clone()
        q3.lora_gate_up(act, self.base[0], self.base[1], self.x, self.stack, self.plan)
        self.check_gate_up(act, before)
        return act


def some(rows, n, seed=0, bare=0.2):
    g = np.random.default_rng(seed)
    return [-1 if g.random() < bare else int(g.integers(0, n)) for _ in range(rows)]


@pytest.mark.parametrize("rows,k,ns,rank,n", [
    (1, 8, [8], 8, 1), (1, 2560, [4096, 1024, 1024], 16, 4), (2, 40, [24, 8], 16, 2), (7, 72, [104], 24, 3), (16, 256, [256], 32, 1),
    (17, 264, [40, 48, 56], 40, 5), (33, 1000, [1016], 64, 9), (100, 512, [512, 256], 128, 30), (128, 136, [72], 8, 128),
    (129, 320, [96, 32], 16, 3), (200, 520, [264], 48, 7), (333, 256, [128, 128, 128], 128, 4), (700, 2048, [512], 64, 2),
    (64, 9728, [2560], 16, 64)])
def test_add_matches_definition(rows, k, ns, rank, n):
    c = Case(rows, k, ns, rank, n, some(rows, n, rows), seed=rows)
    c.add()
    assert q3.device_error() == 0


@pytest.mark.parametrize("rows,k,n_out,rank,n", [(1, 2560, 9728, 16, 2), (5, 72, 40, 8, 3), (32, 512, 264, 24, 8), (31, 256, 1000, 128, 4),
                                                 (130, 264, 96, 16, 5), (347, 1024, 512, 64, 3)])
def test_gate_up_matches_definition(rows, k, n_out, rank, n):
    Case(rows, k, [n_out, n_out], rank, n, some(rows, n, rows), seed=rows).gate_up()
    assert q3.device_error() == 0


@pytest.mark.parametrize("rows", [20, 150])
@pytest.mark.parametrize("rank", [8, 16, 40, 128])
def test_adapters_of_unequal_rank(rows, rank):
    # NaN past each adapter's rank must not get into its rows
    ranks = [0, 1, 2, 3, 4, 5, 7, rank - 1, rank, rank + 5, -3]
    c = Case(rows, 264, [72, 104], rank, len(ranks), some(rows, len(ranks), 3, 0.0), ranks=[min(r, rank + 5) for r in ranks])
    c.add()
    c2 = Case(rows, 264, [72, 72], rank, len(ranks), some(rows, len(ranks), 3, 0.0), ranks=ranks)
    c2.gate_up()


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 64, 128, 129, 191, 192, 193, 1025])
def test_all_rows_of_one_kind(rows):
    for index in ([-1] * rows, [2] * rows, [i % 3 for i in range(rows)], [0] * (rows - 1) + [-1]):
        c = Case(rows, 64, [32], 16, 3, index)
        c.add()


def test_many_adapters():
    # more adapters than a block has threads; each of its rows finds its own
    c = Case(300, 16, [8], 8, 3000, [int(v) for v in np.random.default_rng(1).integers(0, 3000, 300)])
    c.add()
    Case(40, 16, [8], 8, 8192, [8191 - 7 * i for i in range(40)]).add()


def test_in_place_and_strided():
    c = Case(50, 136, [64, 40, 24], 16, 4, some(50, 4))
    want = c.add()
    own = [t.clone() for t in c.base]
    q3.lora_add(own, own, c.x, c.stack, c.plan)
    assert all(torch.equal(a, b) for a, b in zip(own, want))
    # q, k and v side by side in one buffer, x in a wider one
    buf = torch.full((50, 160), 7.0, dtype=BF16, device="cuda")
    views = [buf[:, 8:72], buf[:, 80:120], buf[:, 128:152]]
    for v, t in zip(views, c.base):
        v.copy_(t)
    wide = torch.full((50, 200), NAN, dtype=BF16, device="cuda")
    wide[:, 16:152] = c.x
    q3.lora_add(views, views, wide[:, 16:152], c.stack, c.plan)
    assert all(torch.equal(a, b) for a, b in zip(views, want))
    rest = torch.ones(160, dtype=torch.bool)
    for lo, hi in ((8, 72), (80, 120), (128, 152)):
        rest[lo:hi] = False
    assert (buf[:, rest.cuda()] == 7.0).all()
    g = Case(50, 136, [64, 64], 16, 4, some(50, 4))
    act = g.gate_up()
    gate = g.base[0].clone()
    q3.lora_gate_up(gate, gate, g.base[1], g.x, g.stack, g.plan)  # over its own base
    has = torch.tensor([i >= 0 for i in g.index], device="cuda")
    assert torch.equal(gate[has], act[has]) and torch.equal(gate[~has], g.base[0][~has])


def test_rows_do_not_depend_on_their_neighbours():
    # with so few adapters the calls have clusters of one size, so a row's sums are cut alike, whatever shares its tile
    c = Case(100, 1024, [256], 32, 5, some(100, 5))
    want = c.add()[0]
    for at in ([3], [7, 50, 51, 99], list(range(0, 100, 3))):
        p = q3.LoraPlan(len(at), 5)
        p.update(c.index_d[at].contiguous())
        out = torch.empty(len(at), 256, dtype=BF16, device="cuda")
        q3.lora_add(out, c.base[0][at].contiguous(), c.x[at].contiguous(), c.stack, p)
        assert torch.equal(out, want[at])


def test_values_that_are_not_finite_stay_in_their_rows():
    c = Case(40, 64, [32], 16, 4, [i % 4 for i in range(40)])
    want = c.add()[0]
    c.x[5] = NAN
    c.x[12, 3] = float("inf")
    c.base[0][9, 4] = float("inf")
    out = torch.empty_like(want)
    q3.lora_add(out, c.base[0], c.x, c.stack, c.plan)
    ok = torch.ones(40, dtype=torch.bool)
    ok[[5, 12, 9]] = False
    assert torch.equal(out[ok.cuda()], want[ok.cuda()])
    assert torch.isnan(out[5]).all() and not torch.isfinite(out[12]).any()
    assert torch.isinf(out[9, 4]) and torch.equal(out[9, 5:], want[9, 5:])
    # an adapter of NaN spoils its own rows only
    c.a[0][2] = NAN
    q3.lora_add(out, c.base[0], c.x, c.stack, c.plan)
    mine = torch.tensor([i == 2 for i in c.index]) | ~ok
    assert torch.equal(out[~mine.cuda()], want[~mine.cuda()])


def test_bad_indices_are_flagged():
    c = Case(6, 16, [8], 8, 3, [0, 3, 2, 2 ** 31 - 1, -2 ** 31, 1])
    assert q3.device_error() == 4
    c.add()
    assert q3.device_error() == 0


def test_captured_with_a_changing_index():
    c = Case(70, 256, [128, 64], 16, 6, some(70, 6))
    outs = [torch.empty_like(t) for t in c.base]
    plan, index = q3.LoraPlan(70, 6), c.index_d.clone()

    def step():
        plan.update(index)
        q3.lora_add(outs, c.base, c.x, c.stack, plan)
        q3.lora_add(outs, outs, c.x, c.stack, plan)  # a second layer's call on the same plan

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        c.index = some(70, 6, seed)
        index.copy_(torch.tensor(c.index, dtype=torch.int32))
        graph.replay()
        once = [torch.empty_like(t) for t in c.base]
        c.plan.update(index)
        q3.lora_add(once, c.base, c.x, c.stack, c.plan)
        c.check_add(once)
        q3.lora_add(once, once, c.x, c.stack, c.plan)
        assert all(torch.equal(a, b) for a, b in zip(outs, once))


def test_a_captured_first_update_describes_nothing_yet():
    c = Case(5, 16, [8], 8, 2, [0, 1, -1, 0, 1])
    plan, graph = q3.LoraPlan(5, 2), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan.update(c.index_d)
    out = torch.full_like(c.base[0], 3.0)
    q3.lora_add(out, c.base[0], c.x, c.stack, plan)
    assert (out == 3.0).all()
    graph.replay()
    q3.lora_add(out, c.base[0], c.x, c.stack, plan)
    c.check_add([out])


def test_refusals():
    c = Case(4, 32, [16, 8], 8, 3, [0, 1, 2, -1])
    outs = [torch.empty_like(t) for t in c.base]

    def refuses(status, f, *a, **kw):
        with pytest.raises(q3.Q3Error) as e:
            f(*a, **kw)
        assert e.value.status == status, e.value

    def add(outs=outs, bases=c.base, x=c.x, stack=c.stack, plan=c.plan):
        q3.lora_add(outs, bases, x, stack, plan)

    add()
    refuses(5, add, plan=q3.LoraPlan(4, 3))  # never updated
    other = q3.LoraPlan(4, 5)
    other.update(c.index_d)
    refuses(1, add, plan=other)
    refuses(1, add, x=c.x[:3])
    refuses(5, add, x=c.x.float())
    refuses(5, add, x=c.x.cpu())
    refuses(1, add, outs=outs[:1])
    refuses(1, add, bases=[c.base[0], c.base[0]])
    refuses(5, add, outs=[outs[0].t().contiguous().t(), outs[1]])
    # an output that is x, another output or another projection's base
    sq = Case(4, 16, [16, 16], 8, 3, [0, 1, 2, -1])
    o = [torch.empty_like(t) for t in sq.base]
    refuses(5, q3.lora_add, [sq.x, o[1]], sq.base, sq.x, sq.stack, sq.plan)
    refuses(5, q3.lora_add, [o[0], o[0]], sq.base, sq.x, sq.stack, sq.plan)
    refuses(5, q3.lora_add, [sq.base[1], o[1]], sq.base, sq.x, sq.stack, sq.plan)
    refuses(5, q3.lora_gate_up, sq.x, sq.base[0], sq.base[1], sq.x, sq.stack, sq.plan)
    refuses(1, q3.lora_gate_up, outs[0], c.base[0], c.base[1], c.x, c.stack, c.plan)  # widths differ
    buf = torch.zeros(5, 16, dtype=BF16, device="cuda")
    refuses(5, q3.lora_add, [buf[1:], o[1]], [buf[:4], sq.base[1]], sq.x, sq.stack, sq.plan)  # shifted by a row
    odd = torch.zeros(4, 20, dtype=BF16, device="cuda")
    refuses(1, q3.lora_add, [odd[:, :16], o[1]], sq.base, sq.x, sq.stack, sq.plan)  # stride not a multiple of 8
    line = torch.zeros(4, 24, dtype=BF16, device="cuda")
    refuses(2, q3.lora_add, [line[:, 4:20], o[1]], sq.base, sq.x, sq.stack, sq.plan)  # not on 16 bytes
    # stacks
    refuses(1, q3.LoraStack, [], [])
    refuses(1, q3.LoraStack, c.a, c.b[:1])
    refuses(1, q3.LoraStack, [c.a[0][0]], [c.b[0]])
    refuses(1, q3.LoraStack, [c.a[0]], [c.b[0][:2]])
    refuses(1, q3.LoraStack, [torch.zeros(2, 12, 16, dtype=BF16, device="cuda")], [torch.zeros(2, 16, 12, dtype=BF16, device="cuda")])
    refuses(1, q3.LoraStack, [torch.zeros(2, 136, 16, dtype=BF16, device="cuda")], [torch.zeros(2, 16, 136, dtype=BF16, device="cuda")])
    refuses(5, q3.LoraStack, [c.a[0].float()], [c.b[0]])
    refuses(5, q3.LoraStack, [c.a[0].cpu()], [c.b[0]])
    refuses(1, q3.LoraStack, [c.a[0]], [c.b[0]], scale=torch.ones(2, device="cuda"))
    refuses(5, q3.LoraStack, [c.a[0]], [c.b[0]], ranks=torch.ones(3, device="cuda"))
    # plans
    refuses(1, q3.LoraPlan, 70000, 3)
    refuses(1, q3.LoraPlan, 4, 0)
    refuses(1, q3.LoraPlan, 4, 9000)
    refuses(1, c.plan.update, c.index_d[:3])
    refuses(5, c.plan.update, c.index_d.long())


def test_no_rows():
    c = Case(1, 16, [8], 8, 2, [0])
    plan = q3.LoraPlan(0, 2)
    plan.update(torch.zeros(0, dtype=torch.int32, device="cuda"))
    none = torch.zeros(0, 8, dtype=BF16, device="cuda")
    q3.lora_add(none, none, c.x[:0], c.stack, plan)


def test_two_calls_at_once():
    c = Case(150, 512, [256, 128], 16, 6, some(150, 6))
    want = c.add()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [[[torch.empty_like(t) for t in c.base] for _ in range(6)] for _ in streams]
    torch.cuda.synchronize()
    for n in range(6):
        for s, out in zip(streams, outs):  # one plan and one stack, read by all
            with torch.cuda.stream(s):
                q3.lora_add(out[n], c.base, c.x, c.stack, c.plan)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in outs for o in out for a, b in zip(o, want))


@pytest.mark.parametrize("rows", [5, 300])
def test_rows_far_apart(rows):
    # offsets past 32 bits: x and out are rows of a wide buffer
    stride = (1 << 31) // rows // 8 * 8 + 64
    c = Case(rows, 64, [32], 16, 3, some(rows, 3))
    want = c.add()[0]
    buf = torch.empty(rows * stride, dtype=BF16, device="cuda")
    x = buf.as_strided((rows, 64), (stride, 1))
    out = buf.as_strided((rows, 32), (stride, 1), 64)
    x.copy_(c.x)
    q3.lora_add(out, c.base[0], x, c.stack, c.plan)
    assert torch.equal(out, want)


def test_long_steps():
    c = Case(65536, 16, [8], 8, 100, [int(v) for v in np.random.default_rng(2).integers(-1, 100, 65536)])
    c.add()
    one = Case(5000, 64, [72], 128, 2, [1] * 5000)
    one.add()


@pytest.mark.parametrize("rows,n", [(33, 8192), (64, 4095), (129, 1), (2079, 1000), (4097, 5000), (65536, 3), (65536, 8192)])
def test_plans_of_any_size(rows, n):
    # every part of the rows, and every number of counters around those that a block has without asking
    g = torch.Generator().manual_seed(rows)
    index = torch.randint(-1, n, (rows,), generator=g, dtype=torch.int32).cuda()
    x, base = normal(g, rows, 8), normal(g, rows, 8)
    a, b = normal(g, n, 8, 8, std=0.3), normal(g, n, 8, 8, std=0.3)
    plan, out = q3.LoraPlan(rows, n), torch.full_like(base, NAN)
    for chosen in (index, index.flip(0)):
        plan.update(chosen)
        q3.lora_add(out, base, x, q3.LoraStack([a], [b]), plan)
        at, has = chosen.long().clamp(min=0), (chosen >= 0).double()[:, None]
        h = torch.einsum("nrk,nk->nr", a[at].double(), x.double())
        y = base.double() + has * torch.einsum("nor,nr->no", b[at].double(), h)
        mag = torch.einsum("nrk,nk->nr", a[at].double().abs(), x.double().abs())
        bound = (40 * 2.0 ** -24 + 2.0 ** -16) * has * torch.einsum("nor,nr->no", b[at].double().abs(), mag) + 2.0 ** -23 * base.double().abs()
        assert ((out.double() - y).abs() <= bound + 2.0 ** -8 * y.abs() + 1e-37).all()
        assert torch.equal(out[chosen < 0], base[chosen < 0])
    assert q3.device_error() == 0


@pytest.mark.parametrize("rows,k,rank,n", [(1, 8, 128, 1), (5, 264, 128, 3), (16, 1000, 72, 2), (31, 2560, 128, 40), (128, 2064, 128, 4), (128, 72, 40, 900)])
def test_wide_short_steps(rows, k, rank, n):
    # up to 384 columns of A x: as many as a pass holds, and two of them; clusters of each size
    Case(rows, k, [136, 40, 8], rank, n, some(rows, n, rank), seed=k).add()
    ranks = [(7 * i + rows) % (rank + 2) for i in range(n)]
    Case(rows, k, [72, 72], rank, n, some(rows, n, rank + 1), seed=k, ranks=ranks).gate_up()
    assert q3.device_error() == 0


@pytest.mark.parametrize("rows,rank", [(5, 8), (20, 40), (150, 16)])
def test_infinite_and_overflowing_weights(rows, rank):
    # A x = -3.01171875, whose two bf16 parts have opposite signs, for rank 0, and 2, 4, ... for the others; B inf, huge, or huge of both signs.
    # The second product's terms are of one sign or too far apart to depend on their order, so fp32 says the same in any.
    inf, n, k = float("inf"), 64, 32
    index = [i % 3 for i in range(rows)]
    c = Case(rows, k, [n, n], rank, 3, index, scale=False)
    c.x.zero_()
    c.x[:, 0] = 1.0
    c.x[:, 1] = 0.01171875
    for a in c.a:
        a.zero_()
        a[:, :, 0] = 2.0 * torch.arange(rank, device="cuda")
        a[:, 0, 0], a[:, 0, 1] = -3.0, -1.0
    h = torch.cat([torch.tensor([-3.01171875]), 2.0 * torch.arange(1, rank)]).cuda()
    for j, b in enumerate(c.b):
        b.zero_()
        b[:, :, 1] = 1.0
        b[:, 1, 0] = inf       # -inf
        b[:, 2, 0] = -inf      # inf
        b[:, 3, 0] = 3e38      # overflows to -inf
        b[:, 4, 0] = -3e38
        b[:, 5, 2] = inf       # inf, of a value without a second part
        b[:, 6, 0] = NAN
        b[:, 7, 0], b[:, 7, 2] = inf, inf  # of both signs: NaN
        b[1, 8 + 5 * j, 0] = inf           # one adapter's only
    y = [torch.einsum("bnr,r->bn", b.float(), h)[torch.tensor(index, device="cuda")] + base.float() for b, base in zip(c.b, c.base)]
    assert [torch.isfinite(v[0]).sum().item() for v in y] == [n - 7, n - 7]

    def same(got, want):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        some, fine = torch.isinf(want), torch.isfinite(want)
        assert torch.equal(got[some].float(), want[some])
        assert ((got - want)[fine].abs() <= 2.0 ** -8 * want[fine].abs() + 2.0 ** -20).all()  # the terms are exact, their sums below 16

    outs = [torch.full_like(t, 5.0) for t in c.base]
    q3.lora_add(outs, c.base, c.x, c.stack, c.plan)
    for out, want in zip(outs, y):
        same(out, want)
    own = [t.clone() for t in c.base]
    q3.lora_add(own, own, c.x, c.stack, c.plan)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(own, outs))
    act = torch.full_like(c.base[0], 5.0)
    q3.lora_gate_up(act, c.base[0], c.base[1], c.x, c.stack, c.plan)
    g, u = y
    want = g / (1 + torch.exp(-g)) * u
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(act), torch.isnan(want)) and torch.equal(act[torch.isinf(want)].float(), want[torch.isinf(want)])
    assert ((act - want)[fine].abs() <= 2.0 ** -8 * want[fine].abs() + 2.0 ** -10).all()


@pytest.mark.parametrize("rows", [3, 140])
def test_values_next_to_the_largest(rows):
    # A x above the largest bf16 number but not above fp32's: its first part must not round to infinity
    c = Case(rows, 8, [32], 8, 1, [0] * rows)
    top = 3.3895313892515355e38  # bf16's largest
    c.scale.fill_(1.0)
    c.x.fill_(1.0)
    c.a[0].zero_()
    c.a[0][0, 0, 0] = top
    c.a[0][0, 0, 1] = 1.2e36  # 0.9 of a step
    c.b[0].zero_()
    c.b[0][0, :, 0] = 0.5
    h = torch.tensor(top, dtype=torch.float32) + c.a[0][0, 0, 1].float().cpu()
    assert torch.isfinite(h) and torch.isinf(h.to(BF16))
    c.base[0].zero_()
    out = torch.empty_like(c.base[0])
    q3.lora_add(out, c.base[0], c.x, c.stack, c.plan)
    assert ((out.double() - 0.5 * h.double()).abs() <= 2.0 ** -8 * h.double()).all()


@pytest.mark.parametrize("rows", [40, 300])
def test_rows_beside_one_that_is_not_finite(rows):
    # their tiles' other rows are the same to the bit; the row's own columns stay within the bound
    c = Case(rows, 256, [2048, 40], 24, 3, [i % 3 for i in range(rows)])
    want = c.add()
    c.base[0][9, 5], c.base[0][9, 1030], c.base[1][17, 3], c.base[0][20, 2047] = float("inf"), NAN, float("-inf"), NAN
    c.x[33] = NAN
    outs = [torch.full_like(t, NAN) for t in c.base]
    q3.lora_add(outs, c.base, c.x, c.stack, c.plan)
    for j, (out, before) in enumerate(zip(outs, want)):
        others = torch.ones(rows, dtype=torch.bool, device="cuda")
        others[[9, 20, 33] if j == 0 else [17, 33]] = False
        assert torch.equal(out[others], before[others]) and torch.isnan(out[33]).all()
        y, bound = c.exact(j)
        odd = ~torch.isfinite(c.base[j])
        odd[33] = True
        assert ((out.double() - y).abs() <= bound + 2.0 ** -8 * y.abs())[~odd].all()
        assert torch.equal(torch.isnan(out[:33][odd[:33]]), torch.isnan(c.base[j][:33][odd[:33]]))
    own = [t.clone() for t in c.base]
    q3.lora_add(own, own, c.x, c.stack, c.plan)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(own, outs))


@pytest.mark.parametrize("rows", [5, 140])
def test_gates_far_below_zero(rows):
    # 1 + e^-g passes 2^126 there, silu(g) is a number like others: the output's rounding, 2^-8 (twice the half step), and the
    # exponential, which is off by 2 + 1.2 |g| steps of 2^-23 and, below the smallest normal number, by 2^-17 more: 2^-15
    c = Case(rows, 16, [64, 64], 8, 2, [i % 2 for i in range(rows)])
    c.x.zero_()
    c.base[0].copy_(torch.linspace(-90, -80, rows * 64, device="cuda").view(rows, 64))
    c.base[1].fill_(2.0)
    act = torch.zeros_like(c.base[0])
    q3.lora_gate_up(act, c.base[0], c.base[1], c.x, c.stack, c.plan)
    g = c.base[0].double()
    want = 2 * g * torch.exp(g) / (1 + torch.exp(g))
    assert want.abs().min() > 2.0 ** -126
    assert ((act.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -15) * want.abs()).all()
