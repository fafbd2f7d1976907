"""Attention over the 8-bit cache where a step's rows are trees of drafts, against 64 bits."""
import random

import numpy as np
import pytest
import torch

import warpdecode_b200 as wd
from test_gpu_kv_cache import GEOMETRY, TYPES, Pair

pytestmark = pytest.mark.gpu
FEW, TREE = "kv_attend_kernel", ("kv_tree_kernel", "kv_prompt_kernel")         # (of the second, by lengths)


def make_tree(n, rng, kind):
    """Parents: a chain, all beside one another, or anything."""
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] * n
    return [rng.randint(-1 if rng.random() < 0.2 else max(-1, i - 9), i - 1) for i in range(n)]


def seen(parents, before, window):
    """[rows][tokens]"""
    n = len(parents)
    out = np.zeros((n, before + n), bool)
    for r in range(n):
        way, a = [], r
        while a >= 0:
            way.append(a)
            a = parents[a] if -1 <= parents[a] < a else -1
        depth = len(way) - 1
        out[r, [before + a for i, a in enumerate(way) if not window or i < window]] = True
        out[r, max(0, before + depth - window + 1) if window else 0:before] = True
    return out


def attend(p, layer, seqs, counts, q, parents, scale, window):
    at, want = 0, []
    for s, n in zip(seqs, counts):
        if n == 0:
            continue
        k, v = p.ref[layer].numbers(s)
        see = seen(parents[at:at + n], k.shape[0] - n, window)
        out, g = np.zeros((n, p.heads, p.dim)), p.heads // p.kv_heads
        for h in range(p.heads):
            x = np.where(see, q[at:at + n, h].double().numpy() @ k[:, h // g].T * scale, -np.inf)
            w = np.exp(x - x.max(axis=1, keepdims=True))
            out[:, h] = w @ v[:, h // g] / w.sum(axis=1, keepdims=True)
        want.append(out)
        at += n
    return np.concatenate(want)


def check(p, seqs, counts, parents, window=0, kernel=None, layer=1):
    q = p.rand(sum(counts), p.heads, p.dim, size=1.5)
    qd, out, pd = q.cuda(), torch.full((sum(counts), p.heads, p.dim), 3.0, dtype=q.dtype, device="cuda"), torch.tensor(parents, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    p.kv.attend_tree(layer, qd.data_ptr(), out.data_ptr(), pd.data_ptr(), TYPES[p.dtype][1], window=window)
    torch.cuda.synchronize()
    if kernel:
        assert p.kv.kernel_name().startswith(kernel)
    want, got = attend(p, layer, seqs, counts, q, parents, p.dim ** -0.5, window), out.double().cpu().numpy()
    values = max(np.abs(p.ref[layer].numbers(s)[1]).max() for s in seqs)
    assert np.abs(got - want).max() <= p.tolerance(q, seqs, layer=layer) * values
    return qd, out, pd


@pytest.mark.parametrize("geometry", GEOMETRY)
@pytest.mark.parametrize("kind", ["any", "star", "chain"])
@pytest.mark.parametrize("lengths,counts", [([1], [1]), ([13], [13]), ([63, 65, 20], [5, 0, 20]), ([300, 8, 129, 64], [7, 3, 33, 64]), ([1000], [128]), ([700, 190], [40, 128])])
def test_trees(geometry, kind, lengths, counts):
    p, rng = Pair(*geometry), random.Random(len(lengths) + counts[0])
    seqs = list(range(len(lengths)))[::-1]
    before = [n - c for n, c in zip(lengths, counts)]
    if sum(before):
        p.step(seqs, before)
    p.step(seqs, counts)
    check(p, seqs, counts, [x for n in counts for x in make_tree(n, rng, kind)])
    assert p.kv.status() == 0


@pytest.mark.parametrize("geometry", [(8, 2, 64, 16, 0, "f32"), (8, 1, 128, 32, 1, "bf16"), (4, 1, 256, 64, 0, "f32"), (32, 1, 64, 64, 0, "bf16"), (32, 1, 128, 64, 0, "f32")])
@pytest.mark.parametrize("window", [1, 2, 5, 17, 64, 300])
def test_windows_count_positions(geometry, window):
    p, rng = Pair(*geometry), random.Random(window)
    p.step([0, 1, 2], [500, 64, 3])
    counts = [45, 9, 128]
    p.step([2, 0, 1], counts)
    check(p, [2, 0, 1], counts, [x for n in counts for x in make_tree(n, rng, "any")], window=window)


SIZES = [(FEW, [8100, 70, 0, 301], [2, 1, 3, 5]), (TREE, [8100], [128]), (TREE, [8100, 100], [128, 3]), (None, [130], [64]), (None, [300, 170, 0, 255], [128] * 4),
         (TREE, [300, 8000, 0, 255, 256, 257, 1000, 2900], [128] * 7 + [77])]


@pytest.mark.parametrize("geometry", [(32, 1, 64, 64, 0, "bf16"), (64, 1, 128, 64, 1, "f32"), (16, 1, 256, 128, 0, "bf16"), (32, 1, 96, 32, 0, "f16"), (32, 1, 64, 16, 1, "f32"), (16, 1, 256, 64, 1, "f32"),
                                      (32, 2, 32, 16, 0, "bf16"), (32, 1, 128, 128, 0, "bf16")])
@pytest.mark.parametrize("kernel,before,counts", SIZES)
def test_every_kernel(geometry, kernel, before, counts):
    p, rng = Pair(*geometry, n_pages=4000, max_context=9000, layers=2), random.Random(1)
    seqs = list(range(len(before)))
    p.step(seqs, before)
    p.step(seqs, counts)
    check(p, seqs, counts, [x for n in counts for x in make_tree(n, rng, "any")], kernel=kernel)
    check(p, seqs, counts, [x for n in counts for x in make_tree(n, rng, "any")], window=150)
    check(p, seqs, counts, [x for n in counts for x in make_tree(n, rng, "any")], window=1500)


@pytest.mark.parametrize("geometry", [(32, 8, 128, 64, 1, "f16"), (16, 4, 64, 64, 0, "f32"), (24, 6, 96, 32, 0, "bf16"), (16, 4, 32, 128, 1, "bf16")])
@pytest.mark.parametrize("kernel,before,counts", [(TREE, [30000], [64]), (TREE, [20001, 15000], [61, 128]), (None, [300 + 80 * i for i in range(16)], [26] * 16)])
def test_two_blocks_of_rows_by_one(geometry, kernel, before, counts):
    p, rng = Pair(*geometry, n_pages=-(-sum(before) // geometry[3]) + 100, max_context=31000, max_seqs=16, layers=2), random.Random(2)
    seqs = list(range(len(before)))
    p.step(seqs, before)
    p.step(seqs, counts)
    parents = [x for n in counts for x in make_tree(n, rng, "any")]
    check(p, seqs, counts, parents, kernel="kv_prompt_kernel" if before == [30000] and p.dim == 128 else kernel)
    check(p, seqs, counts, parents, window=9000)
    check(p, seqs, counts, [x for n in counts for x in make_tree(n, rng, "chain")], window=40)
    assert p.kv.status() == 0


@pytest.mark.parametrize("dtype,tokens", [("f32", 70000), ("bf16", 140000)])
def test_sums_that_are_brought_to_memory(dtype, tokens):
    """More tiles of a CTA than one sum may hold: a few values of one sign, whose sums a tensor core would cut off."""
    p = Pair(64, 1, 64, 128, 0, dtype, n_pages=tokens // 128 + 8, max_seqs=1, max_context=tokens + 256, layers=1)
    gen = torch.Generator().manual_seed(7)
    t = TYPES[dtype][0]
    rows = lambda n: ((torch.randn(n, 1, 64, generator=gen) * 0.3).to(t), (torch.rand(n, 1, 64, generator=gen) + 0.5).to(t))  # noqa: E731
    p.step([0], [tokens], rows=[rows(tokens)])
    p.step([0], [128], rows=[rows(128)])
    q = (torch.randn(128, 64, 64, generator=gen) * 0.3).to(t)
    parents = make_tree(128, random.Random(3), "any")
    qd, pd = q.cuda(), torch.tensor(parents, dtype=torch.int32, device="cuda")
    out = torch.empty_like(qd)
    torch.cuda.synchronize()
    p.kv.attend_tree(0, qd.data_ptr(), out.data_ptr(), pd.data_ptr(), TYPES[dtype][1])
    torch.cuda.synchronize()
    assert p.kv.kernel_name().startswith(TREE) and p.kv.status() == 0
    k, v = p.ref[0].numbers(0)
    see = seen(parents, tokens, 0)
    for r in (0, 1, 64, 127):
        for h in (0, 37, 63):
            x = np.where(see[r], k[:, 0] @ q[r, h].double().numpy() / 8, -np.inf)
            w = np.exp(x - x.max())
            want = w @ v[:, 0] / w.sum()
            # the answer's rounding, half a step of the weights' (16 bits), and what the sums may be cut off by: 2^-13 (F32 rows 2^-15)
            tol = 2.0 ** -14 if dtype == "f32" else 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -12
            assert np.abs(out[r, h].double().cpu().numpy() - want).max() <= tol * np.abs(want).max()


@pytest.mark.parametrize("count", [1, 6, 128])
def test_a_chain_is_attention(count):
    for geometry in [(8, 2, 64, 16, 0, "f32"), (32, 1, 128, 64, 1, "bf16")]:
        p = Pair(*geometry, layers=1)
        p.step([0, 1], [333, 50])
        p.step([0, 1], [count, 3])
        qd, out, _ = check(p, [0, 1], [count, 3], make_tree(count, None, "chain") + [-1, 0, 1], layer=0)
        same, kernel = torch.empty_like(out), p.kv.kernel_name()
        p.kv.attend(0, qd.data_ptr(), same.data_ptr(), TYPES[p.dtype][1])
        torch.cuda.synchronize()
        if kernel == p.kv.kernel_name():
            assert torch.equal(out, same)
        want = p.ref[0].attend(0, qd[:count].double().cpu().numpy(), p.dim ** -0.5, 0)
        for x in (out, same):
            assert np.abs(x[:count].double().cpu().numpy() - want).max() <= p.tolerance(qd.cpu(), [0], layer=0) * np.abs(p.ref[0].numbers(0)[1]).max()


def test_parents_that_are_no_row_in_front():
    p = Pair(8, 2, 64, 16, 0, "f32", layers=1)
    p.step([0], [40])
    p.step([0], [7])
    check(p, [0], [7], [0, 1, 7, 2 ** 31 - 1, -2 ** 31, -1, 5], layer=0)         # the last one alone follows a row


@pytest.mark.parametrize("dtype,heads", [("f32", 8), ("bf16", 64)])
def test_values_far_apart(dtype, heads):
    """Value scales more than 2^90 apart, which the kernel for prompts takes another way with."""
    p = Pair(heads, 1, 64, 16, 0, dtype, layers=1)
    gen = torch.Generator().manual_seed(4)
    rows = lambda n, size: (torch.randn(n, 1, 64, generator=gen).to(TYPES[dtype][0]), (torch.randn(n, 1, 64, generator=gen) * size).to(TYPES[dtype][0]))  # noqa: E731
    p.step([0], [160], rows=[rows(160, 1e-33)])
    p.step([0], [16], rows=[rows(16, 1e5)])
    p.step([0], [40], rows=[rows(40, 1.0)])
    rng = random.Random(2)
    check(p, [0], [40], make_tree(40, rng, "any"), layer=0)
    check(p, [0], [40], make_tree(40, rng, "any"), layer=0, window=20)          # no large value in sight of most rows


@pytest.mark.parametrize("heads", [8, 64])
def test_in_place_and_strided(heads):
    p, rng = Pair(heads, 2, 64, 16, 0, "bf16", layers=1), random.Random(5)
    p.step([0, 1], [100, 30])
    p.step([0, 1], [20, 50])
    parents = [x for n in (20, 50) for x in make_tree(n, rng, "any")]
    qd, out, pd = check(p, [0, 1], [20, 50], parents, layer=0)
    wide = torch.full((70, heads * 64 + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:8 + heads * 64] = qd.reshape(70, -1)
    torch.cuda.synchronize()
    at = wide.data_ptr() + 16
    p.kv.attend_tree(0, at, at, pd.data_ptr(), wd.TYPE_BF16, q_stride=wide.shape[1], out_stride=wide.shape[1])
    torch.cuda.synchronize()
    assert torch.equal(wide[:, 8:8 + heads * 64].reshape(70, heads, 64), out) and (wide[:, :8] == 7.0).all() and (wide[:, 8 + heads * 64:] == 7.0).all()


@pytest.mark.parametrize("heads,counts", [(8, [5, 2]), (64, [60, 2])])
def test_captured_and_replayed_on_other_steps(heads, counts):
    p, rng = Pair(heads, 2, 64, 16, 0, "f32", layers=1, n_pages=900), random.Random(6)
    p.step([0, 1, 2], [300, 20, 7])
    q, out = (torch.zeros(200, heads, 64, device="cuda") for _ in range(2))
    k, v = (torch.zeros(200, 2, 64, device="cuda") for _ in range(2))
    parents = torch.full((200,), -1, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    p.kv.begin([0, 1], counts, s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        p.kv.append(0, k.data_ptr(), v.data_ptr(), stream=s.cuda_stream)
        p.kv.attend_tree(0, q.data_ptr(), out.data_ptr(), parents.data_ptr(), stream=s.cuda_stream)
    for turn, (seqs, n) in enumerate((([0, 1], counts), ([2], [70]), ([1, 2, 0], [1, 9, 30]), ([0, 2], [129, 1]), ([2], [3]))):
        if turn:
            p.kv.begin(seqs, n, s.cuda_stream)
        rows = [p.rand(sum(n), h, 64) for h in (2, 2, heads)]
        tree = [x for m in n for x in make_tree(m, rng, "any")]
        with torch.cuda.stream(s):
            for to, x in zip((k, v, q), rows):
                to[:sum(n)].copy_(x)
            parents[:sum(n)].copy_(torch.tensor(tree, dtype=torch.int32))
            out.fill_(5.0)
            g.replay()
        s.synchronize()
        at = 0
        for i, m in zip(seqs, n):
            p.ref[0].append(i, rows[0][at:at + m].double().numpy(), rows[1][at:at + m].double().numpy())
            at += m
        if max(n) > 128:
            assert (out == 5.0).all()
            continue
        want = attend(p, 0, seqs, n, rows[2], tree, 0.125, 0)
        assert np.linalg.norm(out[:sum(n)].double().cpu().numpy() - want) <= 2.0 ** -15 * np.linalg.norm(want) and (out[sum(n):] == 5.0).all()
    p.kv.truncate(2, 3, s.cuda_stream)
    with torch.cuda.stream(s):
        out.fill_(5.0)
        g.replay()
    s.synchronize()
    assert (out == 5.0).all()


def test_refusals():
    p = Pair(8, 2, 64, 16, 0, "f32")
    a = dict(layer=0, q_ptr=1024, out_ptr=1024, parents_ptr=1024)
    with pytest.raises(wd.WdError, match="no step"):
        p.kv.attend_tree(**a)
    p.kv.begin([0, 1], [0, 0])
    p.kv.attend_tree(**{**a, "q_ptr": None, "parents_ptr": None})          # no rows
    p.kv.begin([0, 1], [3, 129])
    with pytest.raises(wd.WdError, match="128 rows"):
        p.kv.attend_tree(**a)
    p.kv.begin([0, 1], [3, 1])
    for bad in (dict(layer=2), dict(layer=-1), dict(q_ptr=None), dict(out_ptr=None), dict(parents_ptr=None), dict(parents_ptr=1026), dict(q_ptr=1026), dict(type=wd.TYPE_Q8_0), dict(scale=0.0),
                dict(scale=float("nan")), dict(window=-1), dict(q_stride=511), dict(out_stride=511), dict(q_stride=512, out_stride=600)):
        with pytest.raises(wd.WdError):
            p.kv.attend_tree(**{**a, **bad})
