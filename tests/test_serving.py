"""The server's host side: pages, and which tokens each step takes."""
import sys
from pathlib import Path

import numpy as np
import pytest

HERE = Path(__file__).resolve().parent
sys.path.insert(0, str(HERE))
import conftest  # noqa: E402,F401
from llm_inference_b200.checkpoint import PRESETS  # noqa: E402
from llm_inference_b200.serving import PagedServer, Sequence, Sequences  # noqa: E402


def run(s, n, token=7):
    steps = []
    for _ in range(n):
        st = s.step()
        steps.append((list(zip(st.ids, st.counts)), [i for _, i in st.outputs]))
        s.commit(st, [token] * len(st.outputs))
    return steps


def test_decodes_run_beside_one_chunk():
    s = Sequences(n_pages=100, page_size=8, max_seqs=4, max_pages=10, chunk=16)
    a = s.add(Sequence([1]))
    b = s.add(Sequence(list(range(40))))
    c = s.add(Sequence(list(range(20))))
    got = run(s, 6)
    assert got[0] == ([(a, 1), (b, 16)], [a])
    assert got[1] == ([(a, 1), (b, 16)], [a])
    assert got[2] == ([(a, 1), (b, 8)], [a, b])       # b's last chunk: its first token
    assert got[3] == ([(a, 1), (b, 1), (c, 16)], [a, b])
    assert got[4] == ([(a, 1), (b, 1), (c, 4)], [a, b, c])
    assert got[5][1] == [a, b, c]
    assert s.live[b].generated == [7] * 4 and s.live[b].cached == 43
    assert len(s.live[b].pages) == 6 and len(set(s.live[a].pages + s.live[b].pages + s.live[c].pages)) == 10


def test_tokens_and_rows_of_a_step():
    s = Sequences(10, 8, 4, 10, 16)
    a = s.add(Sequence([5]))
    b = s.add(Sequence([9, 8, 7]))
    st = s.step()
    assert st.tokens == [5, 9, 8, 7] and st.outputs == [(0, a), (3, b)]
    s.commit(st, [50, 90])
    assert s.step().tokens == [50, 90]


def test_pages_run_out_and_come_back():
    s = Sequences(n_pages=3, page_size=8, max_seqs=4, max_pages=3, chunk=16)
    a = s.add(Sequence(list(range(16))))
    b = s.add(Sequence(list(range(16))))
    assert run(s, 1)[0][0] == [(a, 16)]               # two of three pages
    assert run(s, 1)[0][0] == [(a, 1)]                # the third; b finds none
    assert run(s, 1)[0][0] == [(a, 1)]
    s.remove(a)
    assert sorted(s.free) == [0, 1, 2]
    assert run(s, 1)[0][0] == [(b, 16)]
    for _ in range(20):                               # b's page table ends at 24 positions
        run(s, 1)
    assert s.live[b].cached == 24 and s.step().ids == []


def test_refusals():
    s = Sequences(10, 8, 1, 2, 16)
    with pytest.raises(ValueError):
        s.add(Sequence([]))
    with pytest.raises(ValueError):
        s.add(Sequence([1] * 17))
    s.add(Sequence([1]))
    with pytest.raises(RuntimeError):
        s.add(Sequence([1]))


def test_a_prompt_longer_than_the_pool_is_refused():
    s = Sequences(n_pages=2, page_size=8, max_seqs=4, max_pages=8, chunk=16)
    with pytest.raises(ValueError, match="pool"):
        s.add(Sequence(list(range(17))))
    assert not s.live
    a = s.add(Sequence(list(range(16))))
    assert run(s, 1) == [([(a, 16)], [a])]


@pytest.mark.parametrize("max_pages,n_pages", [(3, 3), (2, 9), (8, 2)])
def test_sequences_at_their_end_are_reported_and_give_their_pages_back(max_pages, n_pages):
    s = Sequences(n_pages=n_pages, page_size=8, max_seqs=4, max_pages=max_pages, chunk=16)
    most = 8 * min(max_pages, n_pages)
    a = s.add(Sequence([1, 2, 3]))
    assert s.running() == [a]
    steps = 0
    while s.running():
        run(s, 1)
        steps += 1
        assert steps <= most
    # its last token comes from its last position
    assert s.live[a].cached == most and len(s.live[a].generated) == most - 2
    assert sorted(s.free) == list(range(n_pages)) and s.step().ids == []
    b = s.add(Sequence(list(range(9))))  # room again, beside the one that has ended
    assert s.running() == [b] and run(s, 2) == [([(b, 9)], [b]), ([(b, 1)], [b])]
    s.remove(a)
    s.remove(b)
    assert sorted(s.free) == list(range(n_pages)) and s.running() == []


def test_two_half_loaded_prompts_do_not_block_each_other():
    s = Sequences(n_pages=4, page_size=8, max_seqs=4, max_pages=4, chunk=8)
    a = s.add(Sequence(list(range(24))))
    b = s.add(Sequence(list(range(24))))
    s.live[b].pages, s.live[b].cached = [s.free.pop(), s.free.pop()], 16  # both have two of the four pages
    s.live[a].pages, s.live[a].cached = [s.free.pop(), s.free.pop()], 16
    assert run(s, 2) == [([(a, 8)], [a]), ([(a, 1)], [a])]
    assert s.live[b].cached == 0 and s.live[b].pages == []


# what a sequence says depends on its own tokens alone, however often it loses its pages on the way
@pytest.mark.parametrize("seed", range(12))
def test_a_small_pool_stops_nobody(seed):
    import random
    rng = random.Random(seed)
    page, pool, chunk = 4, rng.randint(5, 12), rng.choice([1, 3, 8, 16])
    prompts = [[rng.randrange(97) for _ in range(rng.randint(1, 4 * pool // 2))] for _ in range(5)]

    def next_token(tokens):
        return (31 * sum(tokens) + 7 * tokens[-1] + len(tokens)) % 97

    s = Sequences(n_pages=pool, page_size=page, max_seqs=5, max_pages=pool, chunk=chunk)
    ids = [s.add(Sequence(list(p))) for p in prompts]
    lost = 0
    for _ in range(20000):
        if not s.running():
            break
        before = {i: s.live[i].cached for i in ids}
        st = s.step()
        lost += sum(s.live[i].cached < before[i] for i in ids)
        assert st.ids and len(set(st.ids)) == len(st.ids), "a step without work"
        held = [q for i in ids for q in s.live[i].pages]
        assert sorted(held + s.free) == list(range(pool))
        at = 0
        for i, n in zip(st.ids, st.counts):  # a step's tokens follow on what is in the cache
            seq = s.live[i]
            whole = seq.prompt + seq.generated
            assert st.tokens[at:at + n] == whole[seq.cached:seq.cached + n]
            assert len(seq.pages) * page >= seq.cached + n
            at += n
        s.commit(st, [next_token(s.live[i].prompt + s.live[i].generated) for _, i in st.outputs])
    assert not s.running() and lost > 0
    for i, p in zip(ids, prompts):
        want = list(p)
        while len(want) <= pool * page:
            want.append(next_token(want))
        assert s.live[i].prompt + s.live[i].generated == want


def server():
    """A server without its device side."""
    s = PagedServer.__new__(PagedServer)
    s.shape, s.seqs = PRESETS["tiny"], Sequences(n_pages=8, page_size=8, max_seqs=4, max_pages=8, chunk=16)
    return s


def test_a_prompt_may_be_an_iterator():
    s = server()
    a = s.add(t for t in (5, 6, 7))
    assert s.seqs.live[a].prompt == [5, 6, 7]
    for prompt in ([1, -1], [s.shape.vocab_size], iter([2, s.shape.vocab_size])):
        with pytest.raises(ValueError, match="vocabulary"):
            s.add(prompt)
    assert list(s.seqs.live) == [a]


def test_masks_are_checked_when_a_sequence_is_added():
    s = server()
    words = (s.shape.vocab_size + 31) // 32
    bits = np.arange(words, dtype=np.uint32) * np.uint32(0x90000001)
    for mask in (bits, bits.view(np.int32), bits.astype(np.int64), np.append(bits, bits[:3]), bits.tolist()):
        m = s.seqs.live[s.add([1], mask=mask)].mask
        assert m.dtype == np.int32 and np.array_equal(m.view(np.uint32), bits)
        s.seqs.live.clear()
    for mask in (bits[:-1], bits[None], bits.astype(np.float32), []):
        with pytest.raises(ValueError, match="mask"):
            s.add([1], mask=mask)
    assert not s.seqs.live
