"""Attention over the 8-bit cache where the weights, or the sizes of values and scores, lie far apart."""
import numpy as np
import pytest
import torch

from test_gpu_kv_cache import HALF_STEP, TYPES, Pair

pytestmark = pytest.mark.gpu
FEW, PROMPT, RUNS = "kv_attend_kernel", "kv_prompt_kernel", "kv_prompt_kernel, kv_prompt_join_kernel"
KERNELS = [(FEW, 4, 2), (RUNS, 8, 1000), (PROMPT, 16, 1200)]         # heads over two, and last rows, that run on each


def heavy_first(dtype, tokens, rows, nats, dim, alike):
    """One kv head, `rows` last tokens. The first token's score is `nats` above the others', which differ by 0.2 (alike: not at all); its values are 0."""
    p = Pair(4, 1, dim, 64, 0, dtype, n_pages=tokens // 64 + 2, max_seqs=1, max_context=tokens + 64, layers=1, seed=nats)
    size = 8.0
    q = torch.zeros(rows, 4, dim)
    q[..., 0] = size
    k = torch.zeros(tokens, 1, dim)
    k[..., 0] = 0.0 if alike else (torch.rand(tokens, 1, generator=p.gen) - 0.5) * 0.2 / size
    k[..., 1] = 1.0                     # (the pages' scale)
    k[0, 0, 0] = nats / size
    v = torch.full((tokens, 1, dim), 1.0) if alike else torch.randn(tokens, 1, dim, generator=p.gen) + 1.0
    v[0] = 0.0
    t = TYPES[dtype][0]
    return p, q.to(t), k.to(t), v.to(t)


def run(p, q, k, v, kernel):
    n, m = k.shape[0], q.shape[0]
    if n > m:
        p.step([0], [n - m], rows=[(k[:n - m], v[:n - m])])
    p.step([0], [m], rows=[(k[n - m:], v[n - m:])])
    qd = q.cuda()
    out = torch.full_like(qd, 3.0)
    p.kv.attend(0, qd.data_ptr(), out.data_ptr(), TYPES[p.dtype][1], scale=1.0)
    torch.cuda.synchronize()
    assert p.kv.kernel_name() == kernel and p.kv.status() == 0
    rows = np.unique(np.linspace(0, m - 1, 5).astype(int))
    want = p.ref[0].attend(0, q.double().numpy(), 1.0, 0, rows=rows)
    return out.double().cpu().numpy()[rows], want


SHORT = [(4097, 1, FEW), (4097, 900, RUNS), (4900, 4800, PROMPT)]
LONG = [(131073, 1, FEW), (131073, 400, RUNS)]


@pytest.mark.parametrize("dtype,tokens,rows,kernel,nats,dim,alike",
                         [(t, *s, n, d, a) for t in TYPES for s in SHORT for n in (10, 14, 18) for d in (64, 256) for a in (False, True)] +
                         [(t, *s, n, 64, a) for t in ("f32", "bf16") for s in LONG for n in (12, 18) for a in (False, True)])
def test_a_long_tail_behind_a_heavy_token(dtype, tokens, rows, kernel, nats, dim, alike):
    """The first token has nearly all of the weight, and values of 0: the answer is the tail's alone, and is held to the tail's size.

    Weights are F16 terms below a maximum of at least 2^13 (16 bits: 2^9): one is off by half a step of its own (2^-11; of two terms 2^-22), and by 2^-25 where
    F16 ends, which is 2^-38 (2^-34) e^(nats + 0.2) of the tail's least weight. Scores (F32) are below 2^5, off by 2^-19 of e each, exponentials by 2^-21; all
    of it once more for the denominator; then the answer's own rounding. A tensor core cuts each of the products that it adds where the sum ends, by up to 2^-23
    of a sum that holds 2,048 tokens of two terms at most (16 bits: 8,192 of one), and half of its last value on average: 2,048 2^-23 (4,096 2^-23)."""
    p, q, k, v = heavy_first(dtype, tokens, rows, nats, dim, alike)
    got, want = run(p, q, k, v, kernel)
    own = 2.0 ** -22 if dtype == "f32" else 2.0 ** -11
    end = 2.0 ** (-38 if dtype == "f32" else -34) * np.exp(nats + 0.2)
    tol = 2 * (own + 2.0 ** -19 + 2.0 ** -21) + end + (2048 if dtype == "f32" else 4096) * 2.0 ** -23 + HALF_STEP[dtype]
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


# sums of 2,400 tokens, 150 times 16 of two terms: 2 150 2^-24, and weights off by 2^-21
TOL = 2.0 ** -15
SPREADS = [(1e12, 0.0), (0.0, 1e12), (1e20, 1e-20), (1e-20, 1e20), (1e26, 0.0), (1e34, 1.0), (1.0, 1e34), (1e-25, 0.0), (1e37, 1e37), (0.0, 0.0)]


@pytest.mark.parametrize("kernel,heads,count", KERNELS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("first,second", SPREADS)
def test_pages_whose_values_are_far_apart_weigh_alike(first, second, dim, kernel, heads, count):
    """Scores are all alike, values of one stretch of pages are `first`, of another `second` in size, turn about: each token has its share of the weight."""
    n = 1200 + count
    p = Pair(heads, 2, dim, 16, 0, "f32", n_pages=400, layers=1)
    k, v = torch.zeros(n, 2, dim), p.rand(n, 2, dim).abs() + 0.5
    stretch = torch.arange(n) // 400 % 2 == 0
    v = torch.where(stretch[:, None, None], v * first, v * second)
    got, want = run(p, torch.zeros(count, heads, dim), k, v, kernel)
    assert np.isfinite(got).all()
    assert np.linalg.norm(got - want) <= TOL * np.linalg.norm(want)


@pytest.mark.parametrize("kernel,heads,count", KERNELS)
@pytest.mark.parametrize("size", [1.0, 1e12, 1e-20])
def test_small_values_that_have_the_weight(size, kernel, heads, count):
    """Large values whose scores are 120 below: what remains of them (1e-42 of the answer) is added to the small ones' sum, which does not lose by it."""
    n = 1200 + count
    p = Pair(heads, 2, 64, 16, 0, "f32", n_pages=400, layers=1)
    k, v = torch.zeros(n, 2, 64), (p.rand(n, 2, 64).abs() + 0.5) * size
    k[:, :, 0] = k[:, :, 1] = 1.0
    k[400:608, :, 0] = -1.0
    v[400:608] *= 1e10
    q = torch.zeros(count, heads, 64)
    q[..., 0] = 60.0
    got, want = run(p, q, k, v, kernel)
    assert np.linalg.norm(got - want) <= TOL * np.linalg.norm(want)


@pytest.mark.parametrize("kernel,heads,count", KERNELS)
@pytest.mark.parametrize("was", [1e30, 1e-24])
def test_values_of_another_size_that_are_gone(was, kernel, heads, count):
    """What a cache has held before, in pages that are in use again, changes nothing."""
    n = 1200 + count
    p = Pair(heads, 2, 64, 16, 0, "f32", n_pages=400, layers=1)
    k, v = p.rand(n, 2, 64), p.rand(n, 2, 64)
    p.step([0], [3000], rows=[(p.rand(3000, 2, 64), p.rand(3000, 2, 64) * was)])
    p.kv.free([0])
    p.ref[0].truncate(0, 0)
    got, want = run(p, p.rand(count, heads, 64) * 0.125, k, v, kernel)
    # scores of at most 5 5 64 / 8, off by 2^-22 of that; norms over values of either sign, whose sums are a part of them
    assert np.linalg.norm(got - want) <= 2.0 ** -13 * np.linalg.norm(want)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kernel,heads,count", KERNELS)
def test_queries_whose_elements_are_far_apart(dtype, kernel, heads, count):
    """One element of the queries is 3e6 times the others, and meets keys of 0: scores are the others' alone (about 2.5 in size), and exact but for F32 sums.

    Elements are off by 2^-40 of the largest: 64 30000 2^-40 30 4 / 8 of a score, 2^-14; weights by 2^-11 each way for rows of 16 bits; sums as above."""
    n = 1200 + count
    p = Pair(heads, 2, 64, 32, 0, dtype, n_pages=400, layers=1)
    q, k, v = p.rand(count, heads, 64) * 0.01, p.rand(n, 2, 64) * 30, p.rand(n, 2, 64)
    q[..., 7], k[..., 7] = 30000.0, 0.0
    t = TYPES[dtype][0]
    got, want = run(p, q.to(t), k.to(t), v.to(t), kernel)
    values = np.abs(v.double().numpy()).max()
    assert np.abs(got - want).max() <= (2.0 ** -12 + (0.0 if dtype == "f32" else 2.0 ** -10) + 2.0 ** -14 + HALF_STEP[dtype]) * values


@pytest.mark.parametrize("kernel,heads,count", KERNELS)
@pytest.mark.parametrize("was", [1.0, 1e26, 1e33])
def test_pages_of_zeros_beside_numbers(was, kernel, heads, count):
    """Pages of zeros have a third of the weight, in a cache that has held values of another size before: the others lose nothing by it."""
    n = 1200 + count
    p = Pair(heads, 2, 64, 16, 0, "f32", n_pages=400, layers=1)
    p.step([0], [100], rows=[(p.rand(100, 2, 64), p.rand(100, 2, 64) * was)])
    p.kv.free([0])
    p.ref[0].truncate(0, 0)
    k, v = torch.zeros(n, 2, 64), p.rand(n, 2, 64).abs() + 0.5
    v[torch.arange(n) // 16 % 3 == 1] = 0.0
    got, want = run(p, torch.zeros(count, heads, 64), k, v, kernel)
    assert np.linalg.norm(got - want) <= TOL * np.linalg.norm(want)
