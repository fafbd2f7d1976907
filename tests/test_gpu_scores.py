"""Log probabilities of given tokens, the entropy and the likeliest alternatives against the same in 64 bits."""
import numpy as np
import pytest
import torch

import warpdecode_b200 as wd

pytestmark = pytest.mark.gpu
TYPES = {"f32": (torch.float32, wd.TYPE_F32), "f16": (torch.float16, wd.TYPE_F16), "bf16": (torch.bfloat16, wd.TYPE_BF16)}


def score(x, tokens, n_top, dtype, stride=0, entropy=True, stream=None):
    rows, vocab = tokens.shape[0], x.shape[1] if stride == 0 else stride[1]
    lp, h = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    ids, best = torch.full((rows, max(n_top, 1)), 7, dtype=torch.int32, device="cuda"), torch.full((rows, max(n_top, 1)), 7.0, device="cuda")
    torch.cuda.synchronize()
    wd.token_logprobs(x.data_ptr(), rows, vocab, tokens.data_ptr(), lp.data_ptr(), h.data_ptr() if entropy else None, n_top,
                      ids.data_ptr() if n_top else None, best.data_ptr() if n_top else None, TYPES[dtype][1], stride[0] if stride else 0, stream)
    torch.cuda.synchronize()
    return lp.cpu().double().numpy(), h.cpu().double().numpy(), ids.cpu().numpy(), best.cpu().double().numpy()


def expected(x, tokens, n_top):
    x = x.double().cpu().numpy()
    m = x.max(axis=1, keepdims=True)
    p = x - m - np.log(np.exp(x - m).sum(axis=1, keepdims=True))
    h = -np.where(p > -np.inf, np.where(p > -np.inf, p, 0.0) * np.exp(p), 0.0).sum(axis=1)
    t = tokens.cpu().numpy()
    order = np.argsort(-x, axis=1, kind="stable")[:, :n_top].astype(np.int32)
    best = np.take_along_axis(p, order, axis=1)
    ids = np.where(best > -np.inf, order, -1)
    behind = ((0, 0), (0, max(0, n_top - x.shape[1])))          # fewer tokens than alternatives
    return p[np.arange(len(t)), t], h, np.pad(ids, behind, constant_values=-1), np.pad(best, behind, constant_values=-np.inf)


def check(got, want, n_top, spread):
    """A sum of e^y of up to 2^18 terms, 512 threads' partial sums of at most 512 each: the terms' own error (2^-22, and y's of 2^-24 |y|) and 2^9 additions
    of 2^-24 at most, far from all of one sign: 2^-16 bounds the logarithm; the subtraction of the maximum and the rest are F32 steps of the values' size."""
    tol = 2.0 ** -16 + spread * 2.0 ** -22
    for a, b in ((got[0], want[0]), (got[1], want[1])):
        fine = np.isfinite(b)
        assert np.array_equal(np.isfinite(a), fine) and np.array_equal(a[~fine], b[~fine])
        assert np.abs(a[fine] - b[fine]).max(initial=0) <= tol
    if n_top:
        assert np.array_equal(got[2], want[2])
        fine = np.isfinite(want[3])
        assert np.array_equal(got[3][~fine], want[3][~fine])
        assert np.abs(got[3][fine] - want[3][fine]).max(initial=0) <= tol


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab,n_top", [(1, 1, 1), (1, 2, 3), (3, 5, 5), (2, 31, 32), (1, 1000, 1), (5, 4097, 7), (2, 16384, 0), (4, 151936, 5),
                                              (150, 8193, 20), (1, 262143, 32), (300, 333, 4), (9, 65536, 24)])
def test_scores(dtype, rows, vocab, n_top):
    g = torch.Generator().manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(TYPES[dtype][0])
    x[:, vocab // 2:vocab // 2 + vocab // 10] = -float("inf")
    t = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    check(score(x.cuda(), t.cuda(), n_top, dtype), expected(x, t, n_top), n_top, 40.0)


@pytest.mark.parametrize("vocab", [100, 9000, 40001, 151936])
def test_rows_that_make_many_candidates(vocab):
    """Sorted up and down, constant, two values, a few finite ones, one large one: the list of candidates runs over."""
    i = torch.arange(vocab, dtype=torch.float32)
    few = torch.full((vocab,), -float("inf"))
    few[[3, vocab // 2, vocab - 1]] = torch.tensor([1.0, 2.0, 1.0])
    one = torch.full((vocab,), -5.0)
    one[vocab - 2] = 80.0
    x = torch.stack([i / vocab * 8, -i / vocab * 8, torch.full((vocab,), 2.5), (i % 2) * 3, few, one, -0.0 * (i % 2), torch.where(i < 40, -1e30, -1e30 + 0 * i), i.flip(0) % 77])
    t = torch.randint(0, vocab, (x.shape[0],), dtype=torch.int32)
    got = score(x.cuda(), t.cuda(), 32, "f32")
    check(got, expected(x, t, 32), 32, 100.0)
    for rows in (1, 2):                     # shared by the CTAs of a cluster
        for r in range(0, x.shape[0] - 1):
            got = score(x[r:r + rows].contiguous().cuda(), t[r:r + rows].cuda(), 32, "f32")
            check(got, expected(x[r:r + rows], t[r:r + rows], 32), 32, 100.0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [50, 5000, 140000])
def test_masks_of_the_lowest_number(dtype, vocab):
    """The lowest finite value as a mask: beside numbers it has no probability left, alone it is a distribution like any other."""
    lowest = torch.finfo(TYPES[dtype][0]).min
    x = torch.randn(4, vocab).to(TYPES[dtype][0])
    x[0, ::2] = lowest
    x[1] = lowest
    x[2] = lowest
    x[2, vocab // 3] = -float("inf")
    x[3, :vocab - 3] = lowest
    t = torch.tensor([1, 5, 7, vocab - 1], dtype=torch.int32)
    got, want = score(x.cuda(), t.cuda(), 2, dtype), expected(x, t, 2)
    assert np.abs(got[0] - want[0]).max() < 2e-5 and np.abs(got[1] - want[1]).max() < 2e-5
    assert np.array_equal(got[2], want[2]) and np.abs(got[3] - want[3]).max() < 2e-5


@pytest.mark.parametrize("vocab", [7, 5000, 70000])
def test_rows_without_a_distribution_and_tokens_outside(vocab):
    x = torch.randn(6, vocab)
    x[1, vocab // 2] = float("nan")
    x[2, vocab - 1] = float("inf")
    x[3] = -float("inf")
    t = torch.tensor([0, 1, 2, 3, -1, vocab], dtype=torch.int32)
    lp, h, ids, best = score(x.cuda(), t.cuda(), 4, "f32")
    assert np.isfinite(lp[0]) and np.isnan(lp[1:]).all()
    assert np.isfinite(h[[0, 4, 5]]).all() and np.isnan(h[1:4]).all()
    assert (ids[1:4] == -1).all() and np.isnan(best[1:4]).all() and (ids[[0, 4, 5]] >= 0).all()


def test_strides_odd_places_and_outputs_left_out():
    for dtype, (t, _) in TYPES.items():
        base = torch.randn(9, 1013).to(t).cuda()
        x = base[:, 3:1004]                 # rows of 1,001 that begin on no boundary
        tok = torch.randint(0, 1001, (9,), dtype=torch.int32).cuda()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = score(x, tok, 6, dtype, stride=(1013, 1001), stream=s.cuda_stream)
        check(got, expected(x, tok, 6), 6, 30.0)
        assert (score(x, tok, 0, dtype, stride=(1013, 1001), entropy=False)[1] == 7.0).all()
    with pytest.raises(wd.WdError, match="device memory"):
        wd.token_logprobs(np.zeros(8, np.float32).ctypes.data, 1, 8, None, None, tok.data_ptr())


def test_a_captured_call():
    x, t = torch.randn(3, 20000, device="cuda"), torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    lp = torch.zeros(3, device="cuda")
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        wd.token_logprobs(x.data_ptr(), 3, 20000, t.data_ptr(), lp.data_ptr(), stream=s.cuda_stream)
    for _ in range(3):
        x.copy_(torch.randn(3, 20000))
        g.replay()
        torch.cuda.synchronize()
        assert np.abs(lp.cpu().double().numpy() - expected(x, t, 0)[0]).max() < 2e-5
