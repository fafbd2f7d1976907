"""Verification of drafted tokens against 64 bits, sequence by sequence: whole numbers, equal."""
import random

import numpy as np
import pytest
import torch

import verify_oracle
import warpdecode_b200 as wd

pytestmark = pytest.mark.gpu
TYPES = {"f32": (torch.float32, wd.TYPE_F32), "f16": (torch.float16, wd.TYPE_F16), "bf16": (torch.bfloat16, wd.TYPE_BF16)}


def call(target, tokens, parents, u, draft=None, first=None, heat=None, n_seqs=1, stream=None, strides=(0, 0), vocab=None):
    """On device tensors; path, count, next as numpy."""
    rows = tokens.numel()
    path, count, following = (torch.full((max(n, 1),), -7, dtype=torch.int32, device="cuda") for n in (rows, n_seqs, n_seqs))
    torch.cuda.synchronize()
    ptr = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    wd.verify_drafts(ptr(target), rows, vocab or target.shape[1], ptr(tokens), ptr(u), ptr(path), ptr(count), ptr(following), n_seqs=n_seqs, draft_ptr=ptr(draft),
                     parents_ptr=ptr(parents), first_ptr=ptr(first), temperature_ptr=ptr(heat), type={v[0]: v[1] for v in TYPES.values()}[target.dtype], target_stride=strides[0],
                     draft_stride=strides[1], stream=stream)
    torch.cuda.synchronize()
    return path.cpu().numpy()[:rows], count.cpu().numpy(), following.cpu().numpy()


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def tree(n, rng, most=4):
    kids, parents = [0] * n, [-1]
    for i in range(1, n):
        p = rng.choice([j for j in range(i) if kids[j] < most][-12:])
        kids[p] += 1
        parents.append(p)
    return parents


def make(lengths, vocab, dtype, seed, with_draft, chain, heats):
    """Logits of both, drafted tokens as they come out of the draft (or likely ones), and the numbers."""
    rng, gen = random.Random(seed), np.random.default_rng(seed)
    rows = sum(lengths)
    target = gen.standard_normal((rows, vocab)) * 1.5
    hot = gen.integers(0, vocab, (rows, 4))
    np.put_along_axis(target, hot, np.log(vocab) + 3 * gen.random((rows, 4)), 1)
    draft = target + gen.standard_normal((rows, vocab)) * 0.5
    if vocab > 40:
        target[:, -3:] = draft[:, -3:] = -np.inf
    target, draft = (torch.tensor(x, dtype=torch.float32).to(TYPES[dtype][0]) for x in (target, draft))
    tokens, parents, at = np.zeros(rows, np.int64), np.full(rows, -1), 0
    for n, t in zip(lengths, heats):
        ps = list(range(-1, n - 1)) if chain else tree(n, rng) if n else []
        for j, p in enumerate(ps):
            if p < 0:
                continue
            parents[at + j] = p
            q = verify_oracle.softmax(draft[at + p].double().numpy(), t if t >= 1e-6 else 0.1)
            tokens[at + j] = gen.choice(vocab, p=q / q.sum()) if with_draft or rng.random() < 0.3 else int(np.argsort(-q)[min(vocab - 1, ps[:j].count(p))])
        at += n
    return target, draft if with_draft else None, tokens, parents, gen.random(rows).astype(np.float32)


def check(got, lengths, target, draft, tokens, parents, u, heats):
    path, count, following = got
    at = 0
    target = target.double().cpu().numpy()
    draft = None if draft is None else draft.double().cpu().numpy()
    for i, n in enumerate(lengths):
        if n == 0:
            assert count[i] == 0 and following[i] == -1
            continue
        with np.errstate(invalid="ignore"):
            want, token = verify_oracle.sequence(target[at:at + n], None if draft is None else draft[at:at + n], tokens[at:at + n], parents[at:at + n], u[at:at + n], heats[i])
        assert path[at:at + n].tolist() == want + [-1] * (n - len(want)), (i, want)
        assert count[i] == len(want) and following[i] == token, (i, want, token, following[i])
        at += n


@pytest.mark.parametrize("vocab", [2, 7, 33, 1000, 5003, 70001])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("chain", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_against_64_bits(vocab, with_draft, chain, dtype):
    lengths = [1, 5, 0, 13, 40, 2, 8, 3]
    heats = [1.0, 0.7, 1.0, 1.3, 0.9, 0.0, 1e-7, 0.25]
    target, draft, tokens, parents, u = make(lengths, vocab, dtype, 100 * vocab + 10 * with_draft + chain, with_draft, chain, heats)
    first = np.concatenate([[0], np.cumsum(lengths)])
    got = call(target.cuda(), ints(tokens), ints(parents), torch.tensor(u, device="cuda"), None if draft is None else draft.cuda(), ints(first),
               torch.tensor(heats, dtype=torch.float32, device="cuda"), len(lengths))
    check(got, lengths, target, draft, tokens, parents, u, [float(np.float32(t)) for t in heats])


@pytest.mark.parametrize("n_seqs", [1, 3, 9, 40, 300])          # clusters of 16 down to single CTAs
@pytest.mark.parametrize("with_draft", [True, False])
def test_clusters_of_every_size(n_seqs, with_draft):
    lengths, heats, vocab = [5] * n_seqs, [1.0] * n_seqs, 40009 if n_seqs < 100 else 3001
    target, draft, tokens, parents, u = make(lengths, vocab, "bf16", n_seqs, with_draft, True, heats)
    got = call(target.cuda(), ints(tokens), None, torch.tensor(u, device="cuda"), None if draft is None else draft.cuda(), n_seqs=n_seqs)
    check(got, lengths, target, draft, tokens, parents, u, heats)


@pytest.mark.parametrize("with_draft,wide", [(True, False), (False, False), (False, True)])         # a very deep chain, a root with very many children
def test_the_longest_sequences(with_draft, wide):
    n, vocab = 1024, 3000
    lengths, heats = [n, 2], [0.8, 1.0]
    target, draft, tokens, _, u = make(lengths, vocab, "f32", 5, with_draft, True, heats)
    parents = np.array(([-1] + [0] * (n - 1) if wide else list(range(-1, n - 1))) + [-1, 0])
    if wide:
        u[:] = 0.999999         # most are turned down
        tokens[1:n] = np.random.default_rng(1).permutation(vocab)[:n - 1]
    else:
        u[1:] *= 1e-3           # most are taken
    got = call(target.cuda(), ints(tokens), ints(parents), torch.tensor(u, device="cuda"), None if draft is None else draft.cuda(), ints([0, n, n + 2]),
               torch.tensor(heats, dtype=torch.float32, device="cuda"), 2)
    check(got, lengths, target, draft, tokens, parents, u, [float(np.float32(t)) for t in heats])
    assert wide or got[1][0] > 20


def test_more_rows_than_a_sequence_may_have():
    target = torch.zeros(1030, 4, device="cuda")
    tokens = ints(np.zeros(1030))
    path, count, following = call(target, tokens, None, torch.zeros(1030, device="cuda"), first=ints([0, 1025, 1030]), n_seqs=2)
    assert count.tolist() == [0, 5] and following.tolist() == [-1, 0] and (path[:1025] == -1).all() and path[1025:].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lead", [0, 1, 3])
def test_strides_and_rows_beside_a_boundary(dtype, lead):
    lengths, heats, vocab = [6, 6, 6], [1.0, 0.6, 0.0], 4099
    target, draft, tokens, parents, u = make(lengths, vocab, dtype, 9 + lead, True, False, heats)
    held = []
    for x, stride in ((target, 4105), (draft, 4099)):
        buf = torch.full((18 * stride + 8,), float("nan"), dtype=x.dtype, device="cuda")
        torch.as_strided(buf, (18, vocab), (stride, 1), lead).copy_(x)
        held.append(buf[lead:])
    got = call(held[0], ints(tokens), ints(parents), torch.tensor(u, device="cuda"), held[1], heat=torch.tensor(heats, dtype=torch.float32, device="cuda"), n_seqs=3, strides=(4105, 0), vocab=vocab)
    check(got, lengths, target, draft, tokens, parents, u, [float(np.float32(t)) for t in heats])


@pytest.mark.parametrize("with_draft", [True, False])
def test_tokens_come_out_as_the_target_makes_them(with_draft):
    """Two drafts a sequence (siblings, then a chain), 2^18 sequences of one distribution: the first two tokens that come out have the target's shares, to six
    standard deviations."""
    n, vocab, gen = 1 << 18, 6, np.random.default_rng(3)
    target = np.log(np.array([[0.35, 0.3, 0.2, 0.1, 0.05, 0.0], [0.05, 0.15, 0.2, 0.25, 0.35, 0.0]]) + 1e-30)
    target[:, 5] = -np.inf
    q = np.array([0.1, 0.45, 0.05, 0.3, 0.1, 0.0])
    draft = np.log(q + 1e-30)
    # rows: 0; its children 1, 2; behind them the second distribution
    t = np.stack([target[0], target[1], target[1]]).astype(np.float32)
    big_t = torch.tensor(t, device="cuda").repeat(n, 1)
    big_q = torch.tensor(draft, dtype=torch.float32, device="cuda").repeat(3 * n, 1)
    tokens = gen.choice(vocab, size=(n, 3), p=q) if with_draft else np.tile([0, 1, 3], (n, 1))
    u = torch.tensor(gen.random(3 * n, dtype=np.float32), device="cuda")
    path, count, following = call(big_t, ints(tokens.reshape(-1)), ints(np.tile([-1, 0, 0], n)), u, big_q if with_draft else None, n_seqs=n)
    path = path.reshape(n, 3)
    one = np.where(count == 1, following, tokens[np.arange(n), np.maximum(path[:, 1], 0)])
    for got, p in ((one, np.exp(target[0])), (following[count == 2], np.exp(target[1]))):
        share, p = np.bincount(got, minlength=vocab) / got.size, p / p.sum()
        assert (np.abs(share - p) <= 6 * np.sqrt(p * (1 - p) / got.size) + 1e-12).all(), (share, p)
    assert count.max() == 2 and (count == 2).mean() > 0.3


@pytest.mark.parametrize("kind", ["swapped", "few", "scaled", "one"])
@pytest.mark.parametrize("vocab", [3000, 70001])
def test_drafts_that_are_the_target_but_for_some_tokens(kind, vocab):
    """Most tokens' quotient of the two probabilities lies on the border between something left and nothing, or a rounding beside it."""
    gen = np.random.default_rng(vocab)
    lengths, heats = [2, 4, 4, 4], [1.0, 0.7, 1.0, 1.3]
    target = gen.standard_normal((14, vocab)) * 1.5
    draft = target.copy()
    for r in range(14):
        a = gen.permutation(vocab)[:20]
        if kind == "swapped":
            target[r, a[:10]] += 4.0
            draft[r, a[10:]] = target[r, a[:10]]
            draft[r, a[:10]] = target[r, a[10:]]
        elif kind == "few":
            draft[r, a] += gen.standard_normal(20) * 3
        elif kind == "scaled":
            draft[r] = target[r] + 2.0
            draft[r, a] += gen.standard_normal(20) * 3
        else:
            draft[r, a[0]] += 6.0
    target, draft = (torch.tensor(x, dtype=torch.float32) for x in (target, draft))
    parents = np.array([-1, 0] + [-1, 0, 0, 0] * 3)
    first = [0, 2, 6, 10, 14]
    root = np.repeat([0, 2, 6, 10], [2, 4, 4, 4])
    for turn in range(6):
        # the tokens that the draft likes better than the target, so that many are turned down
        more = [verify_oracle.softmax(draft[r].double().numpy(), 1.0) - verify_oracle.softmax(target[r].double().numpy(), 1.0) for r in range(14)]
        tokens = np.array([int(np.argsort(-more[r])[gen.integers(0, 3)]) for r in root])
        u = gen.random(14).astype(np.float32)
        got = call(target.cuda(), ints(tokens), ints(parents), torch.tensor(u, device="cuda"), draft.cuda(), ints(first), torch.tensor(heats, dtype=torch.float32, device="cuda"), 4)
        check(got, lengths, target, draft, tokens, parents, u, [float(np.float32(t)) for t in heats])


def test_borders():
    """Numbers that lie on a border, or at the ends of [0, 1)."""
    even = torch.zeros(1, 4, device="cuda")
    most = float(np.nextafter(np.float32(1), np.float32(0)))
    for u, want in ((0.0, 0), (0.25, 1), (0.5, 2), (most, 3), (float(np.nextafter(np.float32(0.25), np.float32(0))), 0)):
        assert call(even, ints([9]), None, torch.tensor([u], device="cuda"))[2][0] == want
    pair = torch.zeros(2, 2, device="cuda")
    for u, count in ((0.5, 1), (float(np.nextafter(np.float32(0.5), np.float32(0))), 2)):          # u < p = 1/2
        path, n, following = call(pair, ints([0, 1]), None, torch.tensor([most, u], device="cuda"))
        assert n[0] == count and (count == 2 or following[0] == 0)          # the rejected token is not drawn
    # p = q: whatever was drawn is accepted
    x = torch.randn(5, 1000, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    u = torch.full((5,), most, device="cuda")
    assert call(x, ints([0, 3, 999, 40, 41]), None, u, x.clone())[1][0] == 5
    # what the draft could not have made, but the target could
    q = x.clone()
    q[0, 3] = float("-inf")
    assert call(x, ints([0, 3, 999, 40, 41]), None, u, q)[1][0] == 5
    # out of [0, 1): some token that has a probability
    for bad in (1.0, 2.0, -1.0, float("nan"), float("inf")):
        path, n, following = call(x, ints([0, 3, 999, 40, 41]), None, torch.full((5,), bad, device="cuda"), q)
        assert 1 <= n[0] <= 5 and 0 <= following[0] < 1000


def test_little_is_left():
    """Rejections that leave 2^-20 of the probability, or nothing at all."""
    vocab = 3000
    for rest in (2.0 ** -20, 0.0):
        target = torch.full((3, vocab), float("-inf"))
        target[:, 7] = 0.0
        if rest:
            target[:, 100:1124] = np.log(rest / 1024)
        tokens, u = [0, 7, 7], torch.tensor([0.4995, 1.0, 1.0])       # (1: out of the range, so that all are turned down)
        path, n, following = call(target.cuda(), ints(tokens), ints([-1, 0, 0]), u.cuda())
        assert n[0] == 1 and following[0] == (611 if rest else 7)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_the_largest_logit(dtype):
    x = torch.zeros(4, 40000, dtype=TYPES[dtype][0])
    x[0, [17, 9000, 39999]] = 5.0
    x[1, :] = -3.0                       # all equal: the first one
    x[2, :] = float("-inf")
    x[2, 12345] = torch.finfo(x.dtype).min
    x[3, 3], x[3, 4] = -0.0, 0.0
    x[3, [0, 1, 2]] = -1.0
    u, heat = torch.full((4,), 0.5, device="cuda"), torch.zeros(1, device="cuda")
    for draft in (None, torch.randn(4, 40000, device="cuda").to(x.dtype)):
        path, n, following = call(x.cuda(), ints([0, 17, 0, 12345]), None, u, draft, heat=heat)
        assert n[0] == 4 and path.tolist() == [0, 1, 2, 3] and following[0] == 3
        path, n, following = call(x.cuda(), ints([0, 9000, 0, 12345]), None, u, draft, heat=heat)
        assert n[0] == 1 and following[0] == 17


@pytest.mark.parametrize("heat", [1.0, 0.0, 0.5, float("inf"), float("nan")])
@pytest.mark.parametrize("with_draft", [True, False])
def test_rows_without_a_distribution_end_the_walk(heat, with_draft):
    gen = torch.Generator().manual_seed(2)
    for value in ("nan", "inf", "-inf"):
        for where in range(3):
            x = torch.randn(3, 5000, generator=gen)
            d = x.clone()
            if value == "-inf":
                x[where] = float("-inf")
            else:
                x[where, 4321] = float(value)
            tokens = [0] + [int(x[i].argmax()) for i in range(2)]
            u = torch.zeros(3)
            path, n, following = call(x.cuda(), ints(tokens), None, u.cuda(), d.cuda() if with_draft else None, heat=torch.tensor([heat], device="cuda"))
            assert n[0] == where + 1 and following[0] == -1 and path.tolist() == list(range(where + 1)) + [-1] * (2 - where)
    if with_draft and heat in (1.0, 0.5):
        x = torch.randn(3, 5000, generator=gen)
        d = x.clone()
        d[1, 7] = float("nan")
        d[2, :] = float("nan")             # a leaf's is not asked for
        assert call(x.cuda(), ints([0, 5, 6]), None, torch.zeros(3, device="cuda"), d.cuda())[1:] == (np.array([2]), np.array([-1]))
        d[1, 7] = 0.0
        assert call(x.cuda(), ints([0, 5, 6]), None, torch.zeros(3, device="cuda"), d.cuda())[1][0] == 3


def test_a_flat_temperature():
    x = torch.randn(1, 1000)
    x[0, 500:] = float("-inf")
    for u, want in ((0.0, 0), (0.5005, 250), (0.9995, 499)):
        assert call(x.cuda(), ints([0]), None, torch.tensor([u], device="cuda"), heat=torch.tensor([float("inf")], device="cuda"))[2][0] == want


def test_drafts_that_are_none():
    """Tokens outside of the vocabulary, parents that are no row in front."""
    x = torch.zeros(6, 50, device="cuda")
    x[:, 3] = 20.0
    u = torch.full((6,), 0.3, device="cuda")
    path, n, following = call(x, ints([0, -1, 50, 3, 2 ** 31 - 1, 3]), ints([-1, 0, 0, 0, 3, 3]), u)
    assert path.tolist() == [0, 3, 5, -1, -1, -1] and following[0] == 3
    path, n, following = call(x, ints([3] * 6), ints([5, 1, 2, 7, -9, -1]), u)
    assert path.tolist() == [0] + [-1] * 5 and n[0] == 1 and following[0] == 3
    for d in (None, x.clone()):
        assert call(x, ints([0, -1, 50, 51, 99, -2 ** 31]), ints([-1, 0, 0, 0, 0, 0]), u, d)[1:] == (np.array([1]), np.array([3]))


def test_on_a_stream_and_in_a_graph():
    lengths, heats, vocab = [5, 5, 5], [1.0] * 3, 9001
    s = torch.cuda.Stream()
    sets = [make(lengths, vocab, "f32", 50 + i, True, False, heats) for i in range(3)]
    target, draft = (torch.zeros(15, vocab, device="cuda") for _ in range(2))
    tokens, parents = (torch.zeros(15, dtype=torch.int32, device="cuda") for _ in range(2))
    u = torch.zeros(15, device="cuda")
    path, count, following = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (15, 3, 3))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        wd.verify_drafts(target.data_ptr(), 15, vocab, tokens.data_ptr(), u.data_ptr(), path.data_ptr(), count.data_ptr(), following.data_ptr(), n_seqs=3, draft_ptr=draft.data_ptr(),
                         parents_ptr=parents.data_ptr(), stream=s.cuda_stream)
    for x in sets:
        with torch.cuda.stream(s):
            for to, v in zip((target, draft), x[:2]):
                to.copy_(v)
            tokens.copy_(torch.tensor(x[2]))
            parents.copy_(torch.tensor(x[3]))
            u.copy_(torch.tensor(x[4]))
            g.replay()
        s.synchronize()
        check([v.cpu().numpy() for v in (path, count, following)], lengths, *x, heats)


def test_no_rows():
    count, following = (torch.full((3,), 5, dtype=torch.int32, device="cuda") for _ in range(2))
    wd.verify_drafts(None, 0, 100, None, None, None, count.data_ptr(), following.data_ptr(), n_seqs=3)
    torch.cuda.synchronize()
    assert count.tolist() == [0] * 3 and following.tolist() == [-1] * 3
