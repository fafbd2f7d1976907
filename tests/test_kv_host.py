"""The 8-bit cache's bookkeeping of pages, and what it refuses, on the host alone (device = -1)."""
import random

import numpy as np
import pytest

import warpdecode_b200 as wd


def cache(**kw):
    c = dict(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=64, n_pages=12, max_seqs=5, max_context=100, page_tokens=16, device=-1)
    c.update(kw)
    return wd.KvCache(**c)


@pytest.mark.parametrize("bad", [dict(n_layers=0), dict(n_heads=7), dict(n_kv_heads=0), dict(head_dim=48), dict(head_dim=0), dict(page_tokens=8),
                                 dict(page_tokens=48), dict(n_pages=0), dict(max_seqs=0), dict(max_seqs=1025), dict(max_context=0), dict(codes=2),
                                 dict(device=-2), dict(max_context=1 << 25), dict(max_seqs=1024, max_context=1 << 24, page_tokens=16)])
def test_refuses_a_geometry(bad):
    with pytest.raises(wd.WdError):
        cache(**bad)


def test_pages_come_and_go():
    kv = cache()
    assert kv.free_pages() == 12
    kv.begin([0, 3], [17, 16])
    assert kv.length(0) == 17 and kv.length(3) == 16 and kv.length(1) == 0
    assert kv.free_pages() == 9 and kv.pages(0).tolist() == [0, 1] and kv.pages(3).tolist() == [2]
    kv.begin([3, 0], [1, 15])
    assert kv.pages(3).size == 2 and kv.pages(0).size == 2 and kv.free_pages() == 8
    kv.truncate(0, 16)
    assert kv.pages(0).size == 1 and kv.free_pages() == 9
    kv.truncate(0, 0)
    kv.free([3, 3, 1])
    assert kv.free_pages() == 12 and kv.length(3) == 0


def test_a_step_takes_all_of_its_pages_or_none():
    kv = cache()
    kv.begin([0], [100])                     # 7 pages
    with pytest.raises(wd.WdError, match="5 free"):
        kv.begin([1, 2], [48, 48])
    assert kv.length(1) == 0 and kv.free_pages() == 5
    for seqs, counts in (([0], [1]), ([1], [-1]), ([5], [1]), ([-1], [1]), ([1, 1], [1, 1]), ([1], [2 ** 31 - 1])):
        with pytest.raises(wd.WdError):
            kv.begin(seqs, counts)
    assert kv.free_pages() == 5
    with pytest.raises(ValueError):
        kv.begin([1, 2], [1])
    kv.begin([1, 2], [0, 0])
    kv.begin([], [])


@pytest.mark.parametrize("kw", [dict(n_pages=2 ** 31 - 1, n_layers=4096), dict(n_pages=2 ** 31 - 1, n_layers=4096, n_heads=4096, n_kv_heads=4096, head_dim=256, page_tokens=128)])
def test_pages_that_no_memory_holds(kw):
    with pytest.raises(wd.WdError, match="4 TiB"):
        cache(**kw)


def test_rows_of_heads_are_counted_in_32_bits():
    kv = cache(n_heads=4096, n_kv_heads=1, n_pages=2 ** 16, max_context=2 ** 22)
    with pytest.raises(wd.WdError, match="too many rows"):
        kv.begin([0], [2 ** 18])
    assert kv.length(0) == 0 and kv.free_pages() == 2 ** 16
    kv.begin([0], [2 ** 18 - 1])
    assert kv.length(0) == 2 ** 18 - 1


def test_lists_are_whole_numbers_of_32_bits():
    kv = cache()
    kv.begin(np.array([0, 1], np.int64), np.array([3, 2], np.uint8))
    for bad in (np.array([2 ** 32]), np.array([0.5]), np.array([[0]])):
        with pytest.raises(ValueError):
            kv.begin(bad, bad)
    with pytest.raises((TypeError, OverflowError)):
        kv.begin([0], [2 ** 31])
    with pytest.raises(TypeError):
        kv.free([0.5])
    assert kv.length(0) == 3 and kv.length(1) == 2


def test_fork_shares_and_copies_when_written():
    kv = cache()
    kv.begin([0], [20])
    kv.fork(0, [1, 2])
    assert kv.free_pages() == 10 and kv.pages(1).tolist() == kv.pages(2).tolist() == kv.pages(0).tolist()
    kv.begin([0, 1, 2], [1, 1, 1])           # two of three copy the page that is not full, the last holder keeps it
    assert kv.free_pages() == 8
    last = [int(kv.pages(i)[1]) for i in range(3)]
    assert len(set(last)) == 3 and [int(kv.pages(i)[0]) for i in range(3)] == [int(kv.pages(0)[0])] * 3
    kv.free([0])
    assert kv.free_pages() == 9
    for src, dst in ((1, [1]), (1, [2]), (1, [3, 3]), (1, [5]), (7, [3])):
        with pytest.raises(wd.WdError):
            kv.fork(src, dst)
    kv.fork(3, [4])                          # an empty one
    assert kv.length(4) == 0


def test_full_pages_are_shared_without_a_copy():
    kv = cache(n_pages=5)
    kv.begin([0], [32])
    kv.fork(0, [1])
    kv.begin([0, 1], [1, 1])
    assert kv.free_pages() == 1 and kv.pages(0)[:2].tolist() == kv.pages(1)[:2].tolist()


def test_a_copy_needs_a_page():
    kv = cache(n_pages=2)
    kv.begin([0], [20])
    kv.fork(0, [1])
    with pytest.raises(wd.WdError, match="0 free"):
        kv.begin([1], [1])
    kv.free([0])
    kv.begin([1], [1])                       # the only holder writes in place


@pytest.mark.parametrize("pages", [12, 3])      # into new pages; in place
def test_keep(pages):
    kv = cache(n_pages=pages)
    kv.begin([0], [40])
    for first, index in ((41, []), (-1, []), (10, [30]), (10, [3, 3]), (10, [4, 3]), (10, [-1])):
        with pytest.raises(wd.WdError):
            kv.keep(0, first, index)
    before = kv.pages(0).tolist()
    kv.keep(0, 10, [0, 1, 2])                # nothing moves
    assert kv.length(0) == 13 and kv.pages(0).tolist() == before[:1]
    kv.begin([0], [27])
    kv.keep(0, 14, [1, 5, 25])
    assert kv.length(0) == 17 and kv.pages(0).size == 2 and kv.free_pages() == pages - 2
    kv.keep(0, 17, [])
    kv.keep(0, 3, [])
    assert kv.length(0) == 3


def test_keep_does_not_write_into_a_page_that_others_hold():
    kv = cache(n_pages=2)
    kv.begin([0], [20])
    kv.fork(0, [1])
    with pytest.raises(wd.WdError, match="0 free"):
        kv.keep(1, 0, [1, 2])
    assert kv.length(1) == 20


def test_a_walk_of_calls_keeps_count_of_the_pages():
    rng, kv = random.Random(3), cache(n_pages=20, max_seqs=6)
    for _ in range(3000):
        what, seq = rng.randrange(6), rng.randrange(6)
        n = kv.length(seq)
        try:
            if what <= 1:
                seqs = rng.sample(range(6), rng.randint(1, 6))
                kv.begin(seqs, [rng.randint(0, 30) for _ in seqs])
            elif what == 2:
                kv.fork(seq, rng.sample(range(6), rng.randint(0, 2)))
            elif what == 3:
                kv.truncate(seq, rng.randint(0, n))
            elif what == 4:
                kv.free([seq])
            else:
                first = rng.randint(0, n)
                kv.keep(seq, first, sorted(rng.sample(range(n - first), rng.randint(0, n - first))))
        except wd.WdError:
            pass
        held = [kv.pages(i).tolist() for i in range(6)]
        for i, p in enumerate(held):
            assert len(p) == -(-kv.length(i) // 16) and len(set(p)) == len(p)
        assert len({p for h in held for p in h}) + kv.free_pages() == 20


def test_calls_on_the_device_are_refused_without_one():
    kv = cache()
    kv.begin([0], [4])
    for call in (lambda: kv.append(0, 16, 16), lambda: kv.attend(0, 16, 16), lambda: kv.read(0, [0], [0], [4], 16, 16), lambda: kv.status()):
        with pytest.raises(wd.WdError, match="without a device"):
            call()


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(vocab=0), dict(n_top=33), dict(n_top=-1), dict(type=wd.TYPE_Q8_0), dict(logits_ptr=None),
                                 dict(tokens_ptr=None), dict(n_top=2), dict(rows=2 ** 30 + 1), dict(vocab=2 ** 30 + 1), dict(logits_ptr=1026), dict(stride=99), dict(logprob_ptr=None)])
def test_scores_refuse(bad):
    a = dict(logits_ptr=1024, rows=2, vocab=100, tokens_ptr=1024, logprob_ptr=1024, entropy_ptr=None)
    a.update(bad)
    with pytest.raises(wd.WdError):
        wd.token_logprobs(**a)


def test_no_rows_is_no_work():
    wd.token_logprobs(1024, 0, 100, None, None, 1024)
    assert np.asarray(cache().pages(0)).size == 0
