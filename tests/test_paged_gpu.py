"""Paged append and attention on a B200 against the definitions in 64 bits.

Tolerances, from the kernels' arithmetic:
  - append: fp32 throughout, rounded to bf16 once. The rounding (8 significant bits, to nearest) is at most
    2^-8 of the result; the fp32 part (norm: a sum of head_dim squares, rsqrt, two products; rotation: sincospif of an angle reduced in
    fp64, two products, a sum) stays below 2^-18 of the two rotated terms' magnitudes.
  - attention: the output's rounding is 2^-8 of it; each probability enters the second product rounded to
    bf16, 2^-8 of itself; scores, exponentials and fp32 sums together stay below 2^-12 of the absolute
    terms: |o - exact| <= 2^-8 |exact| + (2^-8 + 2^-12) sum_t p_t |v_t|.
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

BF, F64 = torch.bfloat16, torch.float64
NAN = float("nan")


def rn(g, *shape, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(BF)


class Batch:
    """A ragged batch over a shuffled page pool. `lens` is [(new tokens, positions with them)]."""

    def __init__(self, lens, heads, kv_heads, dim, page, seed=0, slots_first=False, extra_rows=0, max_q=None,
                 fill=None, spare_pages=2):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.heads, self.kvh, self.dim, self.page = lens, heads, kv_heads, dim, page
        need = [-(-max(kv, 0) // page) for _, kv in lens]
        self.n_pages, self.max_pages = sum(need) + spare_pages, max(max(need, default=1), 1)
        shape = (self.n_pages, page, kv_heads, dim) if slots_first else (self.n_pages, kv_heads, page, dim)
        self.kp, self.vp = rn(g, *shape), rn(g, *shape)
        if slots_first:
            self.kp, self.vp = self.kp.transpose(1, 2), self.vp.transpose(1, 2)
        order = torch.randperm(self.n_pages, generator=g, device="cuda").tolist()
        self.table = torch.full((len(lens), self.max_pages), 2 ** 30, dtype=torch.int32)  # unused: out of range
        used = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(order[used:used + n], dtype=torch.int32)
            used += n
        self.starts = [0]
        for q, _ in lens:
            self.starts.append(self.starts[-1] + q)
        self.tokens = self.starts[-1] + extra_rows
        self.max_q = max_q if max_q is not None else max((q for q, _ in lens), default=1)
        self.table = self.table.cuda()
        self.q_start = torch.tensor(self.starts, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
        self.plan = q3.PagedPlan(len(lens), self.tokens, self.max_q, heads, kv_heads, dim, page, self.n_pages,
                                 self.max_pages)
        if fill is not None:  # every slot no position uses
            free = torch.ones(self.n_pages, page, dtype=torch.bool, device="cuda")
            for b, (_, kv) in enumerate(lens):
                t = torch.arange(kv, device="cuda")
                free[self.table[b].long()[t // page], t % page] = False
            self.kp.masked_fill_(free[:, None, :, None], fill)
            self.vp.masked_fill_(free[:, None, :, None], fill)

    def update(self):
        self.plan.update(self.q_start, self.kv_len, self.table)

    def rows(self, b):
        return slice(self.starts[b], self.starts[b + 1])

    def cached(self, pages, b):
        t = torch.arange(self.lens[b][1], device="cuda")
        return pages[self.table[b].long()[t // self.page], :, t % self.page]  # [kv, kvh, dim]

    def attention_exact(self, q, scale):
        """(exact output, sum of absolute terms), zero rows for padding."""
        rep = self.heads // self.kvh
        out = torch.zeros(self.tokens, self.heads, self.dim, dtype=F64, device="cuda")
        mag = torch.zeros_like(out)
        for b, (n, kv) in enumerate(self.lens):
            if n == 0 or kv == 0:
                continue
            k, v = self.cached(self.kp, b).to(F64), self.cached(self.vp, b).to(F64)
            for i in range(n):
                p = kv - n + i
                if p < 0:
                    continue
                x = q[self.starts[b] + i].to(F64).view(self.kvh, rep, self.dim)
                s = torch.einsum("grd,tgd->grt", x, k[:p + 1]) * scale
                w = torch.softmax(s, -1)
                o = torch.einsum("grt,tgd->grd", w, v[:p + 1])
                out[self.starts[b] + i] = o.reshape(self.heads, self.dim)
                mag[self.starts[b] + i] = torch.einsum("grt,tgd->grd", w, v[:p + 1].abs()).reshape(self.heads, self.dim)
        return out, mag


def check_attention(got, exact, mag, what):
    got = got.to(F64).view(exact.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(exact)), f"{what}: NaN pattern"
    inf = torch.isinf(exact)
    assert torch.equal(got[inf], exact[inf]), f"{what}: infinities"
    ok = torch.isfinite(exact)
    err = (got - exact).abs()[ok]
    bound = (2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2.0 ** -12) * mag)[ok]
    worst = (err / bound.clamp(min=1e-30)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: error is {worst:.3f} of the bound"


def attend(b, q, scale=None, **kw):
    out = torch.full((b.tokens, b.heads, b.dim), 7.0, dtype=BF, device="cuda")
    b.update()
    q3.paged_attention(out, q, b.kp, b.vp, b.plan, scale=scale, **kw)
    torch.cuda.synchronize()
    return out


SHAPES = [(32, 8, 128), (16, 8, 128), (4, 2, 64), (8, 8, 128), (64, 8, 128), (12, 2, 96), (6, 2, 40), (40, 2, 64)]


@pytest.mark.parametrize("heads,kvh,dim", SHAPES)
@pytest.mark.parametrize("page,slots_first", [(16, False), (48, True), (128, False)])
def test_decode_matches_definition(heads, kvh, dim, page, slots_first):
    lens = [(1, n) for n in (1, 2, 15, 16, 17, 127, 128, 129, 300, 1025)]
    b = Batch(lens, heads, kvh, dim, page, seed=heads + page, slots_first=slots_first, fill=NAN)
    q = rn(b.g, b.tokens, heads, dim, std=1.5)
    out = attend(b, q)
    check_attention(out, *b.attention_exact(q, dim ** -0.5), f"decode {heads}/{kvh}x{dim} page {page}")
    assert q3.device_error() == 0


@pytest.mark.parametrize("heads,kvh,dim", SHAPES)
@pytest.mark.parametrize("page", [8, 64])
def test_ragged_chunks_match_definition(heads, kvh, dim, page):
    lens = [(5, 5), (1, 77), (0, 30), (33, 200), (130, 130), (2, 641), (64, 64), (17, 1000), (1, 1)]
    b = Batch(lens, heads, kvh, dim, page, seed=heads * 3 + page, fill=NAN)
    q = rn(b.g, b.tokens, heads, dim, std=1.5)
    out = attend(b, q)
    check_attention(out, *b.attention_exact(q, dim ** -0.5), f"chunks {heads}/{kvh}x{dim} page {page}")
    assert q3.device_error() == 0


@pytest.mark.parametrize("page", [8, 80, 256])
@pytest.mark.parametrize("n,kv", [(300, 300), (257, 1500), (70, 5000), (20, 9000)])
def test_one_long_chunk(n, kv, page):
    b = Batch([(n, kv)], 8, 2, 128, page, seed=n, fill=NAN)
    q = rn(b.g, b.tokens, 8, 128, std=2.0)
    out = attend(b, q, scale=0.11)
    check_attention(out, *b.attention_exact(q, 0.11), f"chunk of {n} at {kv}")


@pytest.mark.parametrize("kv", [1, 4096, 30001])
def test_one_long_decode(kv):
    b = Batch([(1, kv)], 32, 8, 128, 32, seed=kv, fill=NAN)
    q = rn(b.g, 1, 32, 128, std=2.0)
    check_attention(attend(b, q), *b.attention_exact(q, 128 ** -0.5), f"decode at {kv}")


def test_many_sequences_of_all_lengths():
    g = np.random.default_rng(3)
    lens = [(1, int(n)) for n in g.integers(1, 700, 300)]
    b = Batch(lens, 16, 8, 128, 16, seed=5, fill=NAN)
    q = rn(b.g, b.tokens, 16, 128)
    check_attention(attend(b, q), *b.attention_exact(q, 128 ** -0.5), "300 sequences")


# rows without any position: padding, an empty sequence, a sequence that brings no tokens
@pytest.mark.parametrize("big", [False, True])
def test_empty_rows_are_zero_and_rows_outside_stay(big):
    lens = [(4, 2), (3, 0), (0, 0), (1, 40), (0, 9), (1, 0)] + ([(40, 13), (35, 36)] if big else [])
    b = Batch(lens, 8, 2, 64, 8, seed=11, extra_rows=3, fill=NAN)
    q = rn(b.g, b.tokens, 8, 64)
    q[0:2] = NAN  # padding rows of q may hold anything
    out = attend(b, q)
    exact, mag = b.attention_exact(q, 0.125)
    n = b.starts[-1]
    check_attention(out[:n], exact[:n], mag[:n], "padded batch")
    assert not out[0:2].any() and not out[4:7].any()
    assert (out[n:] == 7.0).all(), "rows outside every sequence were written"
    assert q3.device_error() == 0


# a NaN or infinity in the cache reaches exactly the rows that attend to its position
@pytest.mark.parametrize("heads,kvh", [(4, 2), (32, 8), (8, 8)])
@pytest.mark.parametrize("n,kv", [(6, 50), (200, 200), (200, 333)])
def test_bad_values_stay_behind_the_mask(n, kv, heads, kvh):
    for value in (NAN, float("inf"), -float("inf")):
        b = Batch([(n, kv), (1, 30)], heads, kvh, 128, 16, seed=n + kv, fill=NAN)
        q = rn(b.g, b.tokens, heads, 128)
        where = kv - n + n // 2  # a position some of the rows see
        page, slot = b.table[0, where // 16].item(), where % 16
        b.vp[page, 0, slot, 5] = value
        b.vp[page, 1, slot, 100] = -value
        exact, mag = b.attention_exact(q, 128 ** -0.5)
        check_attention(attend(b, q), exact, mag, f"value {value} at {where}")
        b.kp[page, 0, slot, 3] = NAN  # its score is NaN: so is every row of the head that sees it
        exact, mag = b.attention_exact(q, 128 ** -0.5)
        check_attention(attend(b, q), exact, mag, f"key NaN at {where}")


def test_extreme_scores():
    b = Batch([(1, 500), (40, 300)], 4, 2, 64, 16, seed=4)
    q = rn(b.g, b.tokens, 4, 64, std=20.0)  # few positions take all the weight
    check_attention(attend(b, q, scale=1.0), *b.attention_exact(q, 1.0), "large scores")
    check_attention(attend(b, q, scale=0.0), *b.attention_exact(q, 0.0), "scale 0")
    check_attention(attend(b, q, scale=-0.2), *b.attention_exact(q, -0.2), "negative scale")


def test_strided_rows_and_shared_pages():
    heads, kvh, dim = 8, 2, 128
    b = Batch([(3, 100), (1, 90), (40, 120)], heads, kvh, dim, 16, seed=8)
    b.table[1, :5] = b.table[0, :5]  # a common prefix of 80 positions
    wide = rn(b.g, b.tokens, (heads + 2 * kvh) * dim)
    q = wide[:, :heads * dim]  # rows of a fused qkv projection
    out = torch.zeros(b.tokens, 2 * heads * dim, dtype=BF, device="cuda")
    b.update()
    q3.paged_attention(out[:, heads * dim:], q, b.kp, b.vp, b.plan)
    check_attention(out[:, heads * dim:].reshape(b.tokens, heads, dim), *b.attention_exact(q, dim ** -0.5), "strided")
    assert not out[:, :heads * dim].any()


def test_offsets_past_32_bits():
    # a pool of more than 2^32 bytes per tensor whose last pages are in use
    kvh, dim, page = 8, 128, 64
    n_pages = (1 << 31) // (kvh * dim * page) + 8
    kp = torch.empty(n_pages, kvh, page, dim, dtype=BF, device="cuda")
    vp = torch.empty_like(kp)
    b = Batch([(1, 200), (70, 130)], 32, kvh, dim, page, seed=21)
    far = n_pages - b.n_pages
    kp[far:], vp[far:] = b.kp, b.vp
    b.kp, b.vp, b.n_pages = kp, vp, n_pages
    b.table = torch.where(b.table < 2 ** 30, b.table + far, b.table)
    b.plan = q3.PagedPlan(2, b.tokens, b.max_q, 32, kvh, dim, page, n_pages, b.max_pages)
    q = rn(b.g, b.tokens, 32, dim)
    check_attention(attend(b, q), *b.attention_exact(q, dim ** -0.5), "far pages")
    k, v = rn(b.g, b.tokens, kvh, dim), rn(b.g, b.tokens, kvh, dim)
    q3.paged_rope_append(torch.empty_like(q), q, k, v, kp, vp, b.plan)
    assert torch.equal(b.cached(kp, 0)[199], k[0]) and torch.equal(b.cached(vp, 1)[60:], v[1:])
    assert q3.device_error() == 0


def test_repeat_is_identical_and_follows_other_streams():
    b = Batch([(1, 4000), (1, 37), (90, 700), (5, 2000)], 32, 8, 128, 16, seed=2)
    q = rn(b.g, b.tokens, 32, 128)
    first = attend(b, q)
    side = torch.cuda.Stream()
    for _ in range(3):
        out = torch.empty_like(first)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            q3.paged_attention(out, q, b.kp, b.vp, b.plan)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, first)


def test_a_captured_step_follows_the_lengths():
    b = Batch([(1, 600), (1, 640), (1, 640)], 16, 8, 128, 16, seed=6)
    q = rn(b.g, 3, 16, 128)
    out = torch.empty_like(q)
    b.update()
    q3.paged_attention(out, q, b.kp, b.vp, b.plan)  # kernel attributes are set before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.update()
        q3.paged_attention(out, q, b.kp, b.vp, b.plan)
    for lens in ([600, 1, 640], [17, 128, 0]):
        b.lens = [(1, n) for n in lens]
        b.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check_attention(out, *b.attention_exact(q, 128 ** -0.5), f"replay at {lens}")


def test_bad_descriptions_are_flagged_and_read_nothing():
    def batch():
        return Batch([(1, 30), (2, 40), (20, 60)], 8, 2, 64, 16, seed=1, max_q=20)

    def go(b):
        q = rn(b.g, b.tokens, 8, 64)
        out = attend(b, q)
        k, v = rn(b.g, b.tokens, 2, 64), rn(b.g, b.tokens, 2, 64)
        kp = b.kp.clone()
        q_out = torch.full_like(q, 7.0)
        q3.paged_rope_append(q_out, q, k, v, kp, b.vp.clone(), b.plan)
        flag = q3.device_error()
        b.lens = [(n, 0 if bad else kv) for (n, kv), bad in zip(b.lens, b.bad)]
        exact, mag = b.attention_exact(q, 0.125)
        check_attention(out, exact, mag, "bad description")
        for i, bad in enumerate(b.bad):
            if bad:
                assert not out[b.rows(i)].any() and not q_out[b.rows(i)].any()
        return flag, kp

    for what in ("page", "low page", "long", "negative", "q"):
        b = batch()
        b.bad = [False, True, False]
        if what == "page":
            b.table[1, 1] = b.n_pages
        elif what == "low page":
            b.table[1, 0] = -1
        elif what == "long":
            b.kv_len[1] = b.max_pages * 16 + 1
        elif what == "negative":
            b.kv_len[1] = -5
        else:
            b.bad = [False, False, True]
            b.plan = q3.PagedPlan(3, b.tokens, 19, 8, 2, 64, 16, b.n_pages, b.max_pages)
        assert go(b)[0] == 4, what
    b = batch()
    b.bad = [True, True, True]
    b.q_start[1] = 5  # falls afterwards: no sequence counts
    before = b.kp.clone()
    flag, kp = go(b)
    assert flag == 4 and torch.equal(kp, before)


# ---------------------------------------------------------------- append

def rotate_exact(x, w, pos, freq, interleaved, amplitude, eps):
    """(exact rows, magnitude of the two rotated terms)."""
    y = x.to(F64)
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * w.to(F64)
    out, mag = y.clone(), y.abs()
    n = 0 if freq is None else len(freq)
    if n:
        ang = torch.outer(pos.to(F64), freq.to(F64))[:, None, :]
        c, s = torch.cos(ang) * amplitude, torch.sin(ang) * amplitude
        i = torch.arange(n, device="cuda")
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        u, v = y[..., a], y[..., b]
        out[..., a], out[..., b] = u * c - v * s, v * c + u * s
        mag[..., a] = mag[..., b] = (u.abs() + v.abs()) * amplitude
    return out, mag


def check_rotated(got, exact, mag, what):
    err = (got.to(F64) - exact).abs()
    bound = 2.0 ** -8 * exact.abs() + 2.0 ** -18 * mag + 1e-37
    worst = (err / bound).max().item()
    assert worst <= 1.0 + 2.0 ** -12, f"{what}: error is {worst:.3f} of the bound"


@pytest.mark.parametrize("heads,kvh,dim,rope,interleaved", [
    (32, 8, 128, 128, False), (32, 8, 128, 128, True), (16, 8, 128, 64, False), (4, 2, 64, 64, False),
    (4, 2, 64, 32, True), (12, 2, 96, 96, False), (12, 2, 96, 48, True), (6, 2, 40, 40, False), (6, 2, 40, 20, False),
    (6, 2, 40, 6, True), (3, 1, 8, 8, False), (3, 1, 8, 2, False), (5, 5, 72, 72, False), (8, 4, 128, 0, False),
    (8, 4, 104, 80, False)])
@pytest.mark.parametrize("norm", [True, False])
def test_append_matches_definition(heads, kvh, dim, rope, interleaved, norm):
    lens = [(1, 1), (3, 3), (0, 5), (17, 40), (2, 33000), (4, 2), (1, 0), (33, 333)]
    b = Batch(lens, heads, kvh, dim, 24, seed=dim + rope, extra_rows=2, slots_first=norm)
    wide = rn(b.g, b.tokens, (heads + 2 * kvh) * dim)
    q, k, v = wide[:, :heads * dim], wide[:, heads * dim:(heads + kvh) * dim], wide[:, (heads + kvh) * dim:]
    qw, kw = (rn(b.g, dim, std=0.2, mean=1.0), rn(b.g, dim, std=0.2, mean=1.0)) if norm else (None, None)
    freq, amp = None, 1.0
    if rope:
        f, amp = q3.rope_inv_freq(rope, 1e6, "yarn", factor=4.0, beta_fast=32.0, beta_slow=1.0, original_max=8192)
        freq = torch.from_numpy(f).cuda()
    q_out = torch.full((b.tokens, heads * dim), 7.0, dtype=BF, device="cuda")
    kp, vp = b.kp.clone(), b.vp.clone()
    b.update()
    q3.paged_rope_append(q_out, q, k, v, b.kp, b.vp, b.plan, freq, q_norm_w=qw, k_norm_w=kw, eps=1e-5,
                         interleaved=interleaved, amplitude=amp)
    for i, (n, kv) in enumerate(lens):
        skip = max(0, n - kv)
        r = slice(b.starts[i] + skip, b.starts[i + 1])
        assert not q_out[b.starts[i]:b.starts[i] + skip].any()
        pos = torch.arange(kv - n + skip, kv, device="cuda")
        if len(pos) == 0:
            continue
        exact, mag = rotate_exact(q[r].reshape(-1, heads, dim), qw, pos, freq, interleaved, amp, 1e-5)
        check_rotated(q_out[r].view(-1, heads, dim), exact, mag, f"q of sequence {i}")
        exact, mag = rotate_exact(k[r].reshape(-1, kvh, dim), kw, pos, freq, interleaved, amp, 1e-5)
        page, slot = b.table[i].long()[pos // 24], pos % 24
        check_rotated(b.kp[page, :, slot], exact, mag, f"k of sequence {i}")
        assert torch.equal(b.vp[page, :, slot], v[r].reshape(-1, kvh, dim))
        kp[page, :, slot], vp[page, :, slot] = b.kp[page, :, slot], b.vp[page, :, slot]
    assert (q_out[b.starts[-1]:] == 7.0).all()
    assert torch.equal(b.kp, kp) and torch.equal(b.vp, vp), "a slot no new token owns was written"
    assert q3.device_error() == 0


def test_append_in_place_and_many_tokens():
    b = Batch([(700, 700), (500, 1300)], 8, 8, 128, 64, seed=3)
    q, k, v = rn(b.g, b.tokens, 8, 128), rn(b.g, b.tokens, 8, 128), rn(b.g, b.tokens, 8, 128)
    freq = torch.from_numpy(q3.rope_inv_freq(128, 1e6)[0]).cuda()
    b.update()
    out = torch.empty_like(q)
    q3.paged_rope_append(out, q, k, v, b.kp, b.vp, b.plan, freq)
    q3.paged_rope_append(q, q, k, v, b.kp, b.vp, b.plan, freq)
    assert torch.equal(q, out)
    assert torch.equal(b.cached(b.vp, 1)[800:], v[700:])


def test_append_carries_nan_and_infinity():
    b = Batch([(2, 2)], 2, 1, 64, 8, seed=3)
    q, k, v = rn(b.g, 2, 2, 64), rn(b.g, 2, 1, 64), rn(b.g, 2, 1, 64)
    q[0, 0, 3], v[1, 0, 0] = NAN, float("inf")
    w = rn(b.g, 64, mean=1.0, std=0.1)
    out = torch.empty_like(q)
    b.update()
    q3.paged_rope_append(out, q, k, v, b.kp, b.vp, b.plan, q_norm_w=w, k_norm_w=w)
    assert torch.isnan(out[0, 0]).all() and torch.isfinite(out[0, 1]).all() and torch.isfinite(out[1]).all()
    assert b.cached(b.vp, 0)[1, 0, 0] == float("inf")


# ---------------------------------------------------------------- refusals

def test_refusals():
    b = Batch([(1, 20), (2, 30)], 8, 2, 64, 16, seed=1)
    b.update()
    q = rn(b.g, 3, 8, 64)
    k, v, out = rn(b.g, 3, 2, 64), rn(b.g, 3, 2, 64), torch.empty_like(q)

    def refuses(status, fn, *a, **kw):
        with pytest.raises(q3.Q3Error) as e:
            fn(*a, **kw)
        assert e.value.status == status, e.value

    refuses(1, q3.paged_attention, out, q[:2], b.kp, b.vp, b.plan)           # rows of another shape
    refuses(1, q3.paged_attention, out, q[:, :4], b.kp, b.vp, b.plan)        # too few heads
    refuses(5, q3.paged_attention, out, q.float(), b.kp, b.vp, b.plan)       # type
    refuses(5, q3.paged_attention, out, q.cpu(), b.kp, b.vp, b.plan)         # device
    refuses(1, q3.paged_attention, out, q, b.kp[1:], b.vp[1:], b.plan)       # pages
    refuses(1, q3.paged_attention, out, q, b.kp, b.vp.transpose(0, 2).contiguous().transpose(0, 2), b.plan)
    wide = torch.zeros(3, 8 * 64 + 4, dtype=BF, device="cuda")
    refuses(2, q3.paged_attention, out, wide[:, :512], b.kp, b.vp, b.plan)   # rows not 16 bytes apart
    refuses(2, q3.paged_attention, out, wide.view(-1)[1:1 + 3 * 512].view(3, 512), b.kp, b.vp, b.plan)
    f = torch.ones(40, device="cuda")
    refuses(1, q3.paged_rope_append, out, q, k, v, b.kp, b.vp, b.plan, f)    # rotates more than the head
    refuses(5, q3.paged_rope_append, out, q, k, v, b.kp, b.vp, b.plan, f.double())
    refuses(1, q3.paged_rope_append, out, q, k, v, b.kp, b.vp, b.plan, q_norm_w=rn(b.g, 32))
    refuses(1, b.plan.update, b.q_start[:2], b.kv_len, b.table)
    refuses(5, b.plan.update, b.q_start, b.kv_len.long(), b.table)
    torch.cuda.synchronize()
    assert q3.device_error() == 0


def test_sequences_without_new_tokens():
    pages = torch.zeros(4, 2, 16, 64, dtype=BF, device="cuda")
    plan = q3.PagedPlan(2, 4, 4, 8, 2, 64, 16, 4, 1)
    plan.update(torch.zeros(3, dtype=torch.int32, device="cuda"), torch.full((2,), 5, dtype=torch.int32, device="cuda"),
                torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    out = torch.full((4, 8, 64), 7.0, dtype=BF, device="cuda")
    q3.paged_attention(out, torch.zeros_like(out), pages, pages, plan)
    assert (out == 7.0).all() and q3.device_error() == 0


def test_many_short_chunks_beside_long_decodes():
    # CTAs that take many items of one or two steps each while the decodes keep memory busy: no wait may miss its phase
    g = np.random.default_rng(9)
    lens = [(1, 4096)] * 24 + [(int(n), int(n) + int(c)) for n, c in zip(g.integers(9, 200, 48), g.integers(0, 150, 48))]
    b = Batch(lens, 32, 8, 128, 32, seed=31, fill=NAN)
    q = rn(b.g, b.tokens, 32, 128)
    out = attend(b, q)
    again = [torch.empty_like(out) for _ in range(2)]
    for i in range(60):
        q3.paged_attention(again[i % 2], q, b.kp, b.vp, b.plan)
    torch.cuda.synchronize()
    assert q3.device_error() == 0
    assert torch.equal(out, again[0]) and torch.equal(out, again[1])
    check_attention(out, *b.attention_exact(q, 128 ** -0.5), "short chunks and long decodes")


# draft tokens being verified: a few rows per kv head, in one to three tiles of the kernel for few rows
@pytest.mark.parametrize("heads,kvh,dim,most", [(32, 8, 128, 4), (16, 8, 128, 8), (8, 8, 128, 11), (12, 2, 96, 2), (6, 2, 40, 7),
                                                (32, 4, 64, 3), (4, 2, 64, 12), (64, 8, 128, 2), (40, 2, 64, 1)])
@pytest.mark.parametrize("page", [8, 48])
def test_draft_tokens_match_definition(heads, kvh, dim, most, page):
    kv = (1, 2, 31, 32, 33, 64, 65, 127, 320, 1500, 4097)
    lens = [(min(1 + i * most // 8, most), max(n, i % 3)) for i, n in enumerate(kv)] + [(most, most - 1), (most, 0), (0, 50)]
    b = Batch(lens, heads, kvh, dim, page, seed=heads + page + most, fill=NAN)
    q = rn(b.g, b.tokens, heads, dim, std=1.5)
    out = attend(b, q)
    check_attention(out, *b.attention_exact(q, dim ** -0.5), f"drafts {heads}/{kvh}x{dim} page {page}")
    assert torch.equal(out, attend(b, q))
    assert q3.device_error() == 0


@pytest.mark.parametrize("heads,kvh,dim,n", [(32, 8, 128, 4), (8, 8, 128, 13), (32, 4, 64, 3), (4, 2, 64, 9)])
def test_bad_values_stay_behind_the_mask_of_drafts(heads, kvh, dim, n):
    for kv in (n, 40, 96, 97, 700):
        for value in (NAN, float("inf")):
            b = Batch([(n, kv), (1, 30)], heads, kvh, dim, 16, seed=n + kv, fill=NAN)
            q = rn(b.g, b.tokens, heads, dim)
            where = kv - n + n // 2
            page, slot = b.table[0, where // 16].item(), where % 16
            b.vp[page, 0, slot, 5] = value
            b.vp[page, 1, slot, dim - 1] = -value
            exact, mag = b.attention_exact(q, dim ** -0.5)
            check_attention(attend(b, q), exact, mag, f"value {value} at {where} of {kv}")


# more tokens than the shape allows, in a step whose shape needs no kernel for many rows
@pytest.mark.parametrize("heads,kvh,most", [(8, 2, 1), (8, 2, 4), (8, 8, 1), (32, 2, 0), (4, 2, 0)])
def test_too_many_tokens_are_padding(heads, kvh, most):
    b = Batch([(most, 40), (37, 50), (0, 9), (most, 7)], heads, kvh, 64, 16, seed=heads, max_q=most)
    b.bad = [False, True, False, False]
    q = rn(b.g, b.tokens, heads, 64)
    out = attend(b, q)
    assert q3.device_error() == 4
    b.lens[1] = (37, 0)
    check_attention(out, *b.attention_exact(q, 0.125), "too many tokens")
    assert not out[b.rows(1)].any()


# what lies past rope_dim passes through: an infinity there reaches nothing else
@pytest.mark.parametrize("dim,rope,interleaved", [(128, 64, True), (128, 20, True), (64, 32, False), (64, 20, False), (96, 48, True)])
def test_append_keeps_values_past_the_rotated_ones_apart(dim, rope, interleaved):
    b = Batch([(3, 9)], 4, 2, dim, 8, seed=dim + rope)
    b.update()
    q, k, v = rn(b.g, 3, 4, dim), rn(b.g, 3, 2, dim), rn(b.g, 3, 2, dim)
    freq = torch.from_numpy(q3.rope_inv_freq(rope, 1e4)[0]).cuda()
    clean, out = torch.empty_like(q), torch.empty_like(q)
    q3.paged_rope_append(clean, q, k, v, b.kp, b.vp, b.plan, freq, interleaved=interleaved)
    q[1, 2, rope + 2] = float("inf")
    q[2, 0, dim - 1] = NAN
    q3.paged_rope_append(out, q, k, v, b.kp, b.vp, b.plan, freq, interleaved=interleaved)
    assert torch.equal(clean[..., rope:], torch.where(torch.isfinite(q[..., rope:]), q[..., rope:], clean[..., rope:]))
    changed = (out != clean).nonzero().tolist()
    assert changed == [[1, 2, rope + 2], [2, 0, dim - 1]]
    assert torch.isinf(out[1, 2, rope + 2]) and torch.isnan(out[2, 0, dim - 1])


# A captured step with decodes and a chunk, whose two kernels run side by side: what the step before it left in the plan,
# the queries and the pages is overwritten between replays, and neither kernel may still see it.
def test_a_captured_mixed_step_follows_its_inputs():
    heads, kvh, dim, page, most = 32, 8, 128, 16, 120
    b = Batch([(1, 900)] * 6 + [(most, 900)], heads, kvh, dim, page, seed=12, max_q=most)
    freq = torch.from_numpy(q3.rope_inv_freq(dim, 1e6)[0]).cuda()
    layers = [(b.kp, b.vp), (b.vp.clone(), b.kp.clone())]
    x = [[rn(b.g, b.tokens, n, dim) for n in (heads, kvh, kvh)] for _ in layers]
    qs = [torch.empty_like(x[0][0]) for _ in layers]
    outs = [torch.empty_like(x[0][0]) for _ in layers]

    def step():
        b.update()
        for (kp, vp), (q, k, v), q_out, out in zip(layers, x, qs, outs):
            q3.paged_rope_append(q_out, q, k, v, kp, vp, b.plan, freq)
            q3.paged_attention(out, q_out, kp, vp, b.plan)

    step()  # kernel attributes are set before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    first = b.table.clone()
    for i, (chunk, kv) in enumerate([(most, [900, 17, 1, 640, 33, 128, 900]), (40, [1, 2, 899, 5, 900, 0, 40]), (most, [64] * 6 + [most]),
                                     (1, [900] * 7), (77, [300, 900, 31, 32, 33, 34, 800])]):
        b.lens = [(1, n) for n in kv[:6]] + [(chunk, kv[6])]
        b.starts = [0, 1, 2, 3, 4, 5, 6, 6 + chunk]
        b.q_start.copy_(torch.tensor(b.starts, dtype=torch.int32))
        b.kv_len.copy_(torch.tensor(kv, dtype=torch.int32))
        b.table.copy_(first.roll(i, 0))
        for rows in x:
            for t in rows:
                t.normal_(generator=b.g)
        for out in outs:
            out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert q3.device_error() == 0
        n = b.starts[-1]
        for (b.kp, b.vp), (_, _, v), q, out in zip(layers, x, qs, outs):
            exact, mag = b.attention_exact(q, dim ** -0.5)
            check_attention(out[:n], exact[:n], mag[:n], f"replay {i}")
            assert (out[n:] == 7.0).all()
            for s, (m, kv_s) in enumerate(b.lens):
                assert torch.equal(b.cached(b.vp, s)[max(0, kv_s - m):], v[b.rows(s)][max(0, m - kv_s):])


# a plan whose first update has only been captured describes nothing yet
@pytest.mark.parametrize("most", [1, 40])
def test_a_plan_that_was_only_captured_does_nothing(most):
    b = Batch([(1, 20), (most, 60)], 8, 2, 64, 16, seed=3)
    q, k, v = rn(b.g, b.tokens, 8, 64), rn(b.g, b.tokens, 2, 64), rn(b.g, b.tokens, 2, 64)
    out, q_out = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    kp, vp = b.kp.clone(), b.vp.clone()
    with pytest.raises(q3.Q3Error):
        q3.paged_attention(out, q, b.kp, b.vp, b.plan)
    warm = Batch(b.lens, 8, 2, 64, 16, seed=3)
    attend(warm, q)  # kernel attributes are set before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.update()
    for interleaved in (False, True):
        q3.paged_rope_append(q_out, q, k, v, b.kp, b.vp, b.plan, interleaved=interleaved)
    q3.paged_rope_append(q_out, q, k, v, b.kp, b.vp, b.plan, torch.ones(10, device="cuda"))
    q3.paged_attention(out, q, b.kp, b.vp, b.plan)
    torch.cuda.synchronize()
    assert torch.equal(b.kp, kp) and torch.equal(b.vp, vp)
    assert (out == 7.0).all() and (q_out == 7.0).all() and q3.device_error() == 0
    graph.replay()
    q3.paged_attention(out, q, b.kp, b.vp, b.plan)
    check_attention(out, *b.attention_exact(q, 0.125), "after the replay")


def test_a_first_update_on_another_stream():
    side = torch.cuda.Stream()
    b = Batch([(1, 20), (30, 60)], 8, 2, 64, 16, seed=3)
    q = rn(b.g, b.tokens, 8, 64)
    torch.cuda.synchronize()
    for _ in range(20):
        torch.cuda._sleep(1000000)  # the zeros of a new plan come late on this stream
        b.plan = q3.PagedPlan(2, b.tokens, 30, 8, 2, 64, 16, b.n_pages, b.max_pages)
        with torch.cuda.stream(side):
            out = attend(b, q)
        check_attention(out, *b.attention_exact(q, 0.125), "updated on another stream")


@pytest.mark.parametrize("n_seqs,max_q", [(0, 0), (0, 40), (3, 1), (3, 40)])
@pytest.mark.parametrize("tokens", [0, 2])
def test_steps_without_tokens_or_sequences(n_seqs, max_q, tokens):
    i32 = dict(dtype=torch.int32, device="cuda")
    plan = q3.PagedPlan(n_seqs, tokens, max_q, 8, 2, 64, 16, 4, 2)
    plan.update(torch.zeros(n_seqs + 1, **i32), torch.full((n_seqs,), 20, **i32), torch.zeros(n_seqs, 2, **i32))
    pages = torch.ones(4, 2, 16, 64, dtype=BF, device="cuda")
    q, kv = torch.ones(tokens, 8, 64, dtype=BF, device="cuda"), torch.ones(tokens, 2, 64, dtype=BF, device="cuda")
    out = torch.full_like(q, 7.0)
    q3.paged_rope_append(out, q, 2 * kv, 2 * kv, pages, pages, plan, torch.ones(32, device="cuda"))
    q3.paged_attention(out, q, pages, pages, plan)
    assert (out == 7.0).all() and (pages == 1.0).all()
    x = torch.ones(0, 50, device="cuda")
    q3.logits_process(x, x, torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros(0, **i32), torch.ones(0, device="cuda"),
                      mask=torch.zeros(0, 2, **i32))
    assert q3.device_error() == 0
