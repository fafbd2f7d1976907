"""Verification where a CTA's part of the rows does not fit shared memory, so that every pass reads them anew; a sequence by 1, 2, 4 and 16 CTAs."""
import numpy as np
import pytest
import torch

from test_gpu_verify import call, check, ints, make

pytestmark = pytest.mark.gpu

# sequences (those without rows count for the number of CTAs), vocabulary; 215,000 bytes of rows a CTA are the most that it holds
LARGE = [(600, 30011, "f32", True), (600, 60017, "bf16", True), (600, 60017, "f32", False), (600, 120011, "f16", False), (400, 70001, "f32", True), (400, 240011, "bf16", False),
         (200, 151936, "f32", True), (200, 240011, "f16", True), (200, 240011, "f32", False), (3, 500009, "f32", True), (3, 1800017, "bf16", False)]


@pytest.mark.parametrize("n_seqs,vocab,dtype,with_draft", LARGE)
@pytest.mark.parametrize("chain", [True, False])
def test_rows_that_are_not_held(n_seqs, vocab, dtype, with_draft, chain):
    lengths, heats = [0] * n_seqs, [1.0] * n_seqs
    for i, (n, heat) in enumerate([(1, 1.0), (5, 0.7), (9, 1.0), (3, 0.0), (4, 1.3), (2, 1.0)]):
        at = i * (n_seqs - 1) // 5 if n_seqs > 6 else i
        if at < n_seqs:
            lengths[at], heats[at] = n, heat
    target, draft, tokens, parents, u = make(lengths, vocab, dtype, vocab + chain, with_draft, chain, heats)
    first = np.concatenate([[0], np.cumsum(lengths)])
    got = call(target.cuda(), ints(tokens), ints(parents), torch.tensor(u, device="cuda"), None if draft is None else draft.cuda(), ints(first),
               torch.tensor(heats, dtype=torch.float32, device="cuda"), n_seqs)
    check(got, lengths, target, draft, tokens, parents, u, [float(np.float32(t)) for t in heats])


@pytest.mark.parametrize("n_seqs", [80, 200, 400, 600])          # clusters of 8, 4, 2 and single CTAs, rows held
@pytest.mark.parametrize("with_draft", [True, False])
def test_smaller_clusters(n_seqs, with_draft):
    lengths, heats, vocab = [3] * n_seqs, [1.0] * n_seqs, 16411 if n_seqs < 100 else 4001
    target, draft, tokens, parents, u = make(lengths, vocab, "f32", n_seqs, with_draft, True, heats)
    got = call(target.cuda(), ints(tokens), None, torch.tensor(u, device="cuda"), None if draft is None else draft.cuda(), n_seqs=n_seqs)
    check(got, lengths, target, draft, tokens, parents, u, heats)


@pytest.mark.parametrize("with_draft", [True, False])
def test_many_sequences_of_a_large_vocabulary(with_draft):
    """No sequence is empty, and more CTAs than the device holds at once."""
    n_seqs, vocab, gen = 600, 60017, np.random.default_rng(1)
    target, draft, tokens, parents, u = make([2] * 8, vocab, "bf16", 77, with_draft, True, [1.0] * 8)
    of = gen.integers(0, 8, n_seqs)
    rows = torch.tensor(np.stack([2 * of, 2 * of + 1], 1).reshape(-1))
    big = [None if x is None else x.cuda()[rows.cuda()] for x in (target, draft)]
    uu = gen.random(2 * n_seqs).astype(np.float32)
    path, count, following = call(big[0], ints(tokens[rows.numpy()]), None, torch.tensor(uu, device="cuda"), big[1], n_seqs=n_seqs)
    some = sorted(set(range(0, n_seqs, 37)) | {n_seqs - 1})
    at = np.array([[2 * i, 2 * i + 1] for i in some]).reshape(-1)
    got = (path[at], count[some], following[some])
    pick = rows.numpy()[at]
    check(got, [2] * len(some), target[pick], None if draft is None else draft[pick], tokens[pick], np.tile([-1, 0], len(some)), uu[at], [1.0] * len(some))
    for i, w in enumerate(of):           # the same rows and numbers give the same answer, whichever CTA has them
        assert count[i] in (1, 2) and 0 <= following[i] < vocab
