"""What the verification of drafts refuses, on the host alone; and that what is left of the target after rejections needs two numbers."""
import numpy as np
import pytest

import warpdecode_b200 as wd


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(vocab=0), dict(n_seqs=-1), dict(type=wd.TYPE_Q8_0), dict(target_ptr=None), dict(tokens_ptr=None), dict(uniforms_ptr=None), dict(path_ptr=None),
                                 dict(count_ptr=None), dict(next_ptr=None), dict(rows=2 ** 30 + 1), dict(vocab=2 ** 30 + 1), dict(target_ptr=1026), dict(draft_ptr=1025), dict(tokens_ptr=1026),
                                 dict(parents_ptr=1026), dict(uniforms_ptr=1025), dict(temperature_ptr=1026), dict(path_ptr=1026), dict(count_ptr=1026), dict(next_ptr=1027), dict(first_ptr=1026),
                                 dict(target_stride=99), dict(draft_ptr=1024, draft_stride=99), dict(rows=5, n_seqs=2), dict(rows=1025), dict(n_seqs=2 ** 24 + 1, rows=0)])
def test_refuses(bad):
    a = dict(target_ptr=1024, rows=4, vocab=100, tokens_ptr=1024, uniforms_ptr=1024, path_ptr=1024, count_ptr=1024, next_ptr=1024, n_seqs=1)
    a.update(bad)
    with pytest.raises(wd.WdError):
        wd.verify_drafts(**a)


@pytest.mark.parametrize("bad", [dict(rows=2 ** 32), dict(vocab=2 ** 32 + 5), dict(n_seqs=2 ** 32), dict(type=2 ** 32), dict(target_stride=2 ** 64), dict(draft_stride=2 ** 64)])
def test_numbers_are_not_cut(bad):
    a = dict(target_ptr=1024, rows=4, vocab=100, tokens_ptr=1024, uniforms_ptr=1024, path_ptr=1024, count_ptr=1024, next_ptr=1024, n_seqs=1)
    a.update(bad)
    with pytest.raises(ValueError):
        wd.verify_drafts(**a)


def test_no_sequences_are_no_work():
    wd.verify_drafts(None, 0, 100, None, None, None, None, None, n_seqs=0)


def test_what_rejections_leave():
    gen = np.random.default_rng(0)
    for _ in range(50):
        n = int(gen.integers(2, 200))
        p, q = gen.dirichlet(np.full(n, 0.3)), gen.dirichlet(np.full(n, 0.3))
        r, c, s = p, 0.0, 1.0
        for _ in range(6):
            r = np.maximum(r - q, 0)
            r = r / r.sum()
            c += s
            left = np.maximum(p - c * q, 0)
            s = left.sum()
            if s < 1e-9:
                break
            assert np.abs(left / s - r).max() <= 1e-6
