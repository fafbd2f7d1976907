"""Steps of a small decoder whose sequences each verify a tree of drafts: place, attend, verify, keep; each part against 64 bits from what the one before it gave."""
import random

import numpy as np
import pytest
import torch

import verify_oracle
import warpdecode_b200 as wd
from rope_oracle import rotated
from test_gpu_kv_cache import TYPES
from test_gpu_kv_tree import attend
from test_gpu_rope import Turned
from test_gpu_verify import ints, tree

pytestmark = pytest.mark.gpu
VOCAB = 509


class Decoder:
    """Weights of its own on the device; what lies between the operators is a plain product."""

    def __init__(self, shape, kind, prompts, heat, with_draft, seed):
        self.t = Turned(**shape, **kind, seed=seed, layers=2)
        self.p, self.heat, self.with_draft = self.t.p, heat, with_draft
        self.type, self.rng = TYPES[self.p.dtype], random.Random(seed)
        gen = torch.Generator().manual_seed(seed)
        w = self.p.heads * self.p.dim
        make = lambda *s: (torch.randn(*s, generator=gen) * s[0] ** -0.5).to(self.type[0]).cuda()  # noqa: E731
        self.embed, self.out, self.head = make(VOCAB, w) * VOCAB ** 0.5, [make(w, w) for _ in range(2)], make(w, VOCAB) * 4
        self.qkv = [[make(w, n * self.p.dim) for n in (self.p.heads, self.p.kv_heads, self.p.kv_heads)] for _ in range(2)]
        self.stream = torch.cuda.Stream()
        self.roots = [self.rng.randrange(VOCAB) for _ in prompts]
        self.go([[self.rng.randrange(VOCAB) for _ in range(n)] for n in prompts], [list(range(-1, n - 1)) for n in prompts])

    def go(self, tokens, parents):
        """A step of all sequences; returns the logits."""
        kv, counts, seqs, s = self.p.kv, [len(x) for x in tokens], list(range(len(tokens))), self.stream
        before = [kv.length(i) for i in seqs]
        rows, depth = sum(counts), [0] * 0
        for b, ps in zip(before, parents):
            d = []
            for q in ps:
                d.append(0 if q < 0 else d[q] + 1)
            depth += [b + x for x in d]
        positions, flat = torch.tensor(depth, dtype=torch.int32)[:, None], [q for ps in parents for q in ps]
        kv.begin(seqs, counts, stream=s.cuda_stream)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            pos, above, ids = ints(depth), ints(flat), torch.tensor([x for y in tokens for x in y], device="cuda")
            x = self.embed[ids]
            for layer in range(2):
                q, k, v = ((x @ w).view(rows, -1, self.p.dim) for w in self.qkv[layer])
                turned, seen = torch.full_like(q, 3.0), torch.full_like(q, 3.0)
                self.t.call(layer, k.data_ptr(), v.data_ptr(), q.data_ptr(), turned.data_ptr(), pos.data_ptr(), stream=s.cuda_stream)
                kv.attend_tree(layer, turned.data_ptr(), seen.data_ptr(), above.data_ptr(), self.type[1], stream=s.cuda_stream)
                x = x + seen.view(rows, -1) @ self.out[layer]
                s.synchronize()
                self.t.check_q(turned, q.cpu(), positions)
                self.t.keep_plain(layer, seqs, counts, k.cpu(), v.cpu(), positions)
                want = attend(self.p, layer, seqs, counts, turned.cpu(), flat, self.p.dim ** -0.5, 0)
                values = max(np.abs(self.p.ref[layer].numbers(i)[1]).max() for i in seqs)
                assert np.abs(seen.double().cpu().numpy() - want).max() <= self.p.tolerance(turned.cpu(), seqs, layer=layer) * values
            logits = x @ self.head
        s.synchronize()
        return logits

    def drafted(self, most):
        """Trees of up to `most` rows, the first the token that is known."""
        n = [self.rng.randint(1, most) for _ in self.roots]
        return [[r] + [self.rng.randrange(VOCAB) for _ in range(m - 1)] for r, m in zip(self.roots, n)], [tree(m, self.rng) for m in n]

    def step(self, most, by_target):
        before = [self.p.kv.length(i) for i in range(len(self.roots))]
        tokens, parents = self.drafted(most)
        if by_target:           # what the target itself would say of each row, so that ways through the tree are taken
            for _ in range(2):
                logits = self.go(tokens, parents).float().cpu().numpy()
                at = 0
                for ts, ps in zip(tokens, parents):
                    for j in range(1, len(ts)):
                        if self.rng.random() < 0.8:
                            ts[j] = int(np.argsort(-logits[at + ps[j]])[ps[:j].count(ps[j])])
                    at += len(ts)
                for i, n in enumerate(before):
                    self.p.kv.truncate(i, n)
                    for c in self.p.ref:
                        c.truncate(i, n)
        logits = self.go(tokens, parents)
        rows, n_seqs = logits.shape[0], len(tokens)
        draft = None
        with torch.cuda.stream(self.stream):
            if self.with_draft:
                draft = (logits.float() + 0.3 * torch.randn(rows, VOCAB, device="cuda")).to(logits.dtype)
            first = np.concatenate([[0], np.cumsum([len(t) for t in tokens])])
            u, heat = torch.tensor([self.rng.random() for _ in range(rows)], device="cuda"), torch.tensor(self.heat, device="cuda")
            path, count, following = (torch.full((n,), -7, dtype=torch.int32, device="cuda") for n in (rows, n_seqs, n_seqs))
            ids, above, ends = ints([x for t in tokens for x in t]), ints([x for t in parents for x in t]), ints(first)
            wd.verify_drafts(logits.data_ptr(), rows, VOCAB, ids.data_ptr(), u.data_ptr(), path.data_ptr(), count.data_ptr(), following.data_ptr(), n_seqs=n_seqs,
                             draft_ptr=None if draft is None else draft.data_ptr(), parents_ptr=above.data_ptr(), first_ptr=ends.data_ptr(), temperature_ptr=heat.data_ptr(),
                             type=self.type[1], stream=self.stream.cuda_stream)
        self.stream.synchronize()
        path, count, following = path.tolist(), count.tolist(), following.tolist()
        for i, (a, e) in enumerate(zip(first, first[1:])):
            want, token = verify_oracle.sequence(logits[a:e].double().cpu().numpy(), None if draft is None else draft[a:e].double().cpu().numpy(), tokens[i], parents[i],
                                                 u[a:e].cpu().numpy(), self.heat[i])
            assert path[a:e] == want + [-1] * (e - a - len(want)) and count[i] == len(want) and following[i] == token
            self.p.kv.keep(i, before[i], want)
            for c in self.p.ref:
                c.keep(i, before[i], want)
            assert self.p.kv.length(i) == before[i] + count[i]
        self.roots = following
        return sum(count)


@pytest.mark.parametrize("shape,kind,most", [(dict(heads=8, kv_heads=2, dim=64, page=16, codes=0, dtype="f32"), dict(), 13),
                                             (dict(heads=4, kv_heads=2, dim=128, page=64, codes=1, dtype="bf16"), dict(rotary=64, neighbours=True), 40),
                                             (dict(heads=8, kv_heads=4, dim=32, page=32, codes=0, dtype="f16"), dict(norm=False), 7),
                                             (dict(heads=6, kv_heads=1, dim=96, page=128, codes=0, dtype="bf16"), dict(), 100)])
@pytest.mark.parametrize("with_draft", [False, True])
def test_steps(shape, kind, most, with_draft):
    d = Decoder(shape, kind, [120, 3, 64, 15], [0.0, 1.0, 0.8, 1e-7], with_draft, seed=most)
    taken = [d.step(most, by_target) for by_target in (True, False, True, True)]
    d.p.check_numbers([2, 0, 1, 3])
    assert max(taken) > 4 and d.p.kv.status() == 0
