"""Attention of trees of drafts by each of the kernels that a step may take: at lengths that the rule gives to that kernel, with its name asserted, where the other tests' small steps go to
the kernel for few rows. (The rule counts the device's SMs: 148.)"""
import random

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import TYPES, Pair
from test_gpu_kv_tree import attend, check, make_tree

pytestmark = pytest.mark.gpu

FEW, WHOLE, CUT, PAIRS, PAIRS_CUT = ("kv_attend_kernel", "kv_tree_kernel", "kv_tree_kernel, kv_tree_join_kernel", "kv_prompt_kernel", "kv_prompt_kernel, kv_prompt_join_kernel")


def steps(n, before, rows):
    """n sequences of a little less than `before` tokens, `rows` and a few less drafted ones."""
    return [before - 7 * i for i in range(n)], [rows - 5 * i % 24 for i in range(n)]


# kernel, heads, key/value heads, size of a head, tokens of a page, codes, type; sequences, tokens before the step, rows; window
SHAPES = [(FEW, (8, 2, 64, 16, 0, "bf16"), (3, 90, 20), 0), (FEW, (8, 1, 256, 32, 1, "f32"), (2, 60, 9), 20),
          (CUT, (8, 1, 32, 16, 0, "bf16"), (4, 3100, 128), 0), (WHOLE, (32, 1, 32, 64, 1, "f16"), (4, 1500, 128), 0), (PAIRS, (32, 1, 32, 16, 0, "bf16"), (11, 220, 128), 0),
          (PAIRS_CUT, (32, 1, 32, 128, 0, "f32"), (4, 1700, 128), 0), (CUT, (16, 1, 32, 32, 1, "f32"), (4, 3100, 128), 0),
          (CUT, (8, 1, 64, 64, 0, "bf16"), (2, 3100, 128), 0), (WHOLE, (16, 1, 64, 16, 1, "bf16"), (8, 800, 128), 0), (PAIRS, (32, 1, 64, 64, 0, "f16"), (5, 200, 128), 0),
          (PAIRS_CUT, (16, 1, 64, 128, 1, "bf16"), (4, 1300, 128), 0), (CUT, (8, 1, 64, 32, 0, "f32"), (2, 3200, 128), 0), (PAIRS, (32, 1, 64, 64, 1, "f32"), (5, 200, 128), 0),
          (PAIRS_CUT, (16, 1, 64, 128, 0, "f32"), (8, 760, 128), 0),
          (CUT, (8, 1, 96, 64, 0, "bf16"), (2, 3100, 128), 0), (PAIRS, (32, 1, 96, 16, 1, "f16"), (4, 170, 128), 0), (PAIRS_CUT, (16, 1, 96, 128, 0, "f32"), (8, 760, 128), 0),
          (CUT, (8, 1, 128, 64, 1, "bf16"), (2, 3100, 128), 0), (CUT, (8, 1, 128, 16, 0, "f32"), (2, 3100, 128), 0), (PAIRS, (32, 1, 128, 64, 0, "f32"), (4, 170, 128), 0),
          (PAIRS, (32, 1, 128, 128, 0, "bf16"), (4, 300, 128), 100), (PAIRS_CUT, (8, 1, 128, 32, 1, "f16"), (8, 760, 128), 0),
          (WHOLE, (16, 1, 256, 128, 0, "bf16"), (9, 220, 128), 0), (WHOLE, (32, 1, 256, 64, 1, "f32"), (8, 220, 128), 100), (CUT, (8, 1, 256, 64, 1, "bf16"), (1, 3300, 128), 0),
          (CUT, (8, 1, 256, 32, 0, "f32"), (1, 3300, 128), 0)]


def filled(geometry, before, **kw):
    p = Pair(*geometry, n_pages=sum(-(-(b + 700) // geometry[3]) for b in before), max_seqs=len(before), max_context=max(before) + 1000, layers=1, **kw)
    p.step(list(range(len(before))), before)
    return p


@pytest.mark.parametrize("kernel,geometry,size,window", SHAPES)
def test_trees_in_place_strided_and_beside_boundaries(kernel, geometry, size, window):
    (before, counts), rng = steps(*size), random.Random(size[0])
    p, seqs = filled(geometry, before), list(range(len(before)))
    p.step(seqs[::-1], counts)
    for kind in ("any", "star", "chain"):
        parents = [x for n in counts for x in make_tree(n, rng, kind)]
        qd, out, pd = check(p, seqs[::-1], counts, parents, window=window, layer=0)
        assert p.kv.kernel_name() == kernel
    width, type_ = p.heads * p.dim, TYPES[p.dtype]
    for lead, more in ((8, 24), (1, 24), (3, 5), (0, 1)):               # rows on boundaries of 16 bytes, beside them, and each at another place
        wide = torch.full((sum(counts), width + more), 7.0, dtype=type_[0], device="cuda")
        wide[:, lead:lead + width] = qd.reshape(-1, width)
        rest = wide.clone()
        apart = torch.full((sum(counts) * (width + 3) + 3,), 9.0, dtype=type_[0], device="cuda")
        torch.cuda.synchronize()
        at, size_of = wide.data_ptr(), wide.element_size()
        p.kv.attend_tree(0, at + lead * size_of, apart.data_ptr() + 3 * size_of, pd.data_ptr(), type_[1], window=window, q_stride=width + more, out_stride=width + 3)
        p.kv.attend_tree(0, at + lead * size_of, at + lead * size_of, pd.data_ptr(), type_[1], window=window, q_stride=width + more, out_stride=width + more)
        torch.cuda.synchronize()
        assert p.kv.kernel_name() == kernel
        rest[:, lead:lead + width] = out.reshape(-1, width)
        assert torch.equal(wide, rest)
        apart = apart[3:].reshape(-1, width + 3)
        assert torch.equal(apart[:, :width], out.reshape(-1, width)) and (apart[:, width:] == 9.0).all()
    assert p.kv.status() == 0


@pytest.mark.parametrize("kernel,geometry,size,window", SHAPES)
def test_replays_on_other_steps(kernel, geometry, size, window):
    (before, counts), rng = steps(*size), random.Random(7)
    p, seqs = filled(geometry, before), list(range(len(before)))
    p.step(seqs, counts)
    type_, most = TYPES[p.dtype], max(sum(counts), 300)
    q, out = (torch.zeros(most, p.heads, p.dim, dtype=type_[0], device="cuda") for _ in range(2))
    parents, s = torch.full((most,), -1, dtype=torch.int32, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        p.kv.attend_tree(0, q.data_ptr(), out.data_ptr(), parents.data_ptr(), type_[1], window=window, stream=s.cuda_stream)
    assert p.kv.kernel_name() == kernel
    for turn, (who, n) in enumerate(((seqs, counts), (seqs[-1:], [1]), (seqs[::-1][:2], [60, 17][:len(seqs)]), (seqs[:2], [129, 3][:len(seqs)]), (seqs[:3], [0, 31, 128][:len(seqs)]),
                                     (seqs[:1], [128]))):
        if turn:
            p.step(who, n)
        rows, tree = p.rand(sum(n), p.heads, p.dim, size=1.5), [x for m in n for x in make_tree(m, rng, "any")]
        q[:sum(n)].copy_(rows)
        parents[:sum(n)].copy_(torch.tensor(tree, dtype=torch.int32))
        out.fill_(5.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        if max(n) > 128 or sum(n) == 0:
            assert (out == 5.0).all()
            continue
        want, got = attend(p, 0, who, n, rows, tree, p.dim ** -0.5, window), out[:sum(n)].double().cpu().numpy()
        values = max(np.abs(p.ref[0].numbers(i)[1]).max() for i in who)
        assert np.abs(got - want).max() <= p.tolerance(rows, who, layer=0) * values and (out[sum(n):] == 5.0).all()
    p.kv.truncate(0, 3)
    out.fill_(5.0)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        g.replay()
    s.synchronize()
    assert (out == 5.0).all() and p.kv.status() == 0


@pytest.mark.parametrize("kernel,geometry,size,window", [x for x in SHAPES if x[1][5] != "f16"])
def test_values_far_apart(kernel, geometry, size, window):
    """Value scales more than 2^90 apart, which the kernels on tensor cores take another way with: tiny ones first, a few large ones, ordinary ones; and the tree itself, tiny."""
    before, counts = steps(*size)
    rng, seqs = random.Random(3), list(range(len(before)))
    p = Pair(*geometry, n_pages=sum(-(-(b + 700) // geometry[3]) for b in before), max_seqs=len(before), max_context=max(before) + 1000, layers=1)
    t = TYPES[p.dtype][0]
    rows = lambda n, size: (torch.randn(n, p.kv_heads, p.dim, generator=p.gen).to(t), (torch.randn(n, p.kv_heads, p.dim, generator=p.gen) * size).to(t))  # noqa: E731
    for share, scale in ((0.6, 1e-33), (0.1, 1e5), (0.3, 1.0)):
        n = [max(1, int(b * share)) for b in before]
        p.step(seqs, n, rows=[rows(sum(n), scale)])
    p.step(seqs, counts, rows=[rows(sum(counts), 1e-30)])
    parents = [x for n in counts for x in make_tree(n, rng, "any")]
    for w in (window, 20):              # (a short one: no large value in sight of most rows)
        check(p, seqs, counts, parents, window=w, layer=0)
        if w == window:
            assert p.kv.kernel_name() == kernel
    assert p.kv.status() == 0


@pytest.mark.parametrize("geometry,prefix,count", [((32, 8, 64, 64, 0, "bf16"), 1000, 16), ((32, 8, 32, 64, 1, "f16"), 1500, 32), ((32, 8, 64, 128, 0, "f32"), 2000, 16), ((32, 8, 256, 64, 1, "bf16"), 1000, 16)])
def test_many_sequences(geometry, prefix, count):
    """More sequences than a kernel holds entries of (64), all of one prefix, cut to lengths of their own; whole items, in turn."""
    n = 128 if geometry[2] < 256 else 80
    p = Pair(*geometry, n_pages=-(-prefix // geometry[3]) + 3 * n, max_seqs=n, max_context=prefix + count, layers=1)
    p.step([0], [prefix])
    p.kv.fork(0, list(range(1, n)))
    looked_at = [0, 1, 31, 32, 62, 63, 64, 65, 79] + [n - 1] * (n > 80)
    for i in looked_at[1:]:
        p.ref[0].fork(0, i)
    for i in range(1, n):
        length = prefix - 13 * i % 97
        p.kv.truncate(i, length)
        if i in looked_at:
            p.ref[0].truncate(i, length)
    rng, seqs = random.Random(5), list(range(n))
    rng.shuffle(seqs)
    counts = [count - i % 3 for i in range(n)]
    type_ = TYPES[p.dtype]
    k, v = p.rows(sum(counts)), p.rows(sum(counts))
    q, parents = p.rand(sum(counts), p.heads, p.dim, size=1.5), [x for m in counts for x in make_tree(m, rng, "any")]
    kd, vd, qd, pd = k.cuda(), v.cuda(), q.cuda(), torch.tensor(parents, dtype=torch.int32, device="cuda")
    out = torch.full_like(qd, 3.0)
    torch.cuda.synchronize()
    p.kv.begin(seqs, counts)
    p.kv.append(0, kd.data_ptr(), vd.data_ptr(), type_[1])
    p.kv.attend_tree(0, qd.data_ptr(), out.data_ptr(), pd.data_ptr(), type_[1])
    torch.cuda.synchronize()
    assert p.kv.kernel_name() == WHOLE and p.kv.status() == 0
    got, first = out.double().cpu().numpy(), np.concatenate([[0], np.cumsum(counts)])
    assert np.isfinite(got).all()
    for j, i in enumerate(seqs):
        if i not in looked_at:
            continue
        a, b = first[j], first[j + 1]
        p.ref[0].append(i, k[a:b].double().numpy(), v[a:b].double().numpy())
        want = attend(p, 0, [i], [b - a], q[a:b], parents[a:b], p.dim ** -0.5, 0)
        assert np.abs(got[a:b] - want).max() <= p.tolerance(q[a:b], [i], layer=0) * np.abs(p.ref[0].numbers(i)[1]).max()


def test_parts_of_unequal_sequences():
    """Heads of 256 in F32 against pages of 16 tokens, items of very unequal sequences, one of them without rows and one without tokens in front."""
    p = Pair(8, 2, 256, 16, 0, "f32", n_pages=700, max_seqs=5, max_context=4000, layers=1)
    p.step([0, 1, 2, 4], [3000, 1, 500, 2999])
    counts, rng = [128, 1, 0, 128, 77], random.Random(8)
    p.step([0, 1, 2, 3, 4], counts)
    for window in (0, 1, 2000):
        check(p, [0, 1, 2, 3, 4], counts, [x for n in counts for x in make_tree(n, rng, "any")], window=window, layer=0)
        if window == 0:
            assert p.kv.kernel_name() == CUT
    assert p.kv.status() == 0
