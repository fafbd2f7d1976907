"""The 8-bit key/value cache and attention over it against a plain cache in 64 bits."""
import numpy as np
import pytest
import torch

import kv_oracle
import warpdecode_b200 as wd

pytestmark = pytest.mark.gpu
TYPES = {"f32": (torch.float32, wd.TYPE_F32), "f16": (torch.float16, wd.TYPE_F16), "bf16": (torch.bfloat16, wd.TYPE_BF16)}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Pair:
    """The framework's cache and the plain one, fed alike."""

    def __init__(self, heads, kv_heads, dim, page, codes, dtype, n_pages=400, max_seqs=8, max_context=6000, layers=2, seed=0):
        self.kv = wd.KvCache(layers, heads, kv_heads, dim, n_pages, max_seqs, max_context, page_tokens=page, codes=codes)
        self.ref = [kv_oracle.Cache(kv_heads, dim, page, codes, max_seqs) for _ in range(layers)]
        self.heads, self.kv_heads, self.dim, self.layers, self.dtype = heads, kv_heads, dim, layers, dtype
        self.gen = torch.Generator().manual_seed(seed)

    def rand(self, *shape, size=1.0):
        return (torch.randn(*shape, generator=self.gen) * size).to(TYPES[self.dtype][0])

    def rows(self, n):
        x = self.rand(n, self.kv_heads, self.dim)
        big = torch.rand(n, self.kv_heads, 1, generator=self.gen) < 0.05
        return torch.where(big, x * 5, x * (0.2 + torch.rand(n, 1, 1, generator=self.gen))).to(x.dtype)

    def step(self, seqs, counts, rows=None):
        self.kv.begin(seqs, counts)
        for layer in range(self.layers):
            k, v = rows[layer] if rows else (self.rows(sum(counts)), self.rows(sum(counts)))
            kd, vd = k.cuda(), v.cuda()
            self.kv.append(layer, kd.data_ptr(), vd.data_ptr(), TYPES[self.dtype][1])
            torch.cuda.synchronize()
            at = 0
            for s, n in zip(seqs, counts):
                self.ref[layer].append(s, k[at:at + n].double().numpy(), v[at:at + n].double().numpy())
                at += n

    def check_numbers(self, seqs):
        """F32 out: code times scale, rounded once."""
        n = [self.kv.length(s) for s in seqs]
        k = torch.full((self.layers, sum(n), self.kv_heads, self.dim), 7.0, device="cuda")
        v = k.clone()
        self.kv.read(-1, seqs, [0] * len(seqs), n, k.data_ptr(), v.data_ptr())
        torch.cuda.synchronize()
        for layer in range(self.layers):
            want = np.concatenate([self.ref[layer].numbers(s) for s in seqs], axis=1).astype(np.float32)
            assert np.array_equal(k[layer].cpu().numpy(), want[0])
            assert np.array_equal(v[layer].cpu().numpy(), want[1])

    def attend(self, seqs, counts, scale=None, window=0, size=1.5, q=None, layer=1):
        q = self.rand(sum(counts), self.heads, self.dim, size=size) if q is None else q
        qd = q.cuda()
        out = torch.full_like(qd, 3.0)
        self.kv.attend(layer, qd.data_ptr(), out.data_ptr(), TYPES[self.dtype][1], scale=scale, window=window)
        torch.cuda.synchronize()
        at, want = 0, []
        for s, n in zip(seqs, counts):
            if n:
                want.append(self.ref[layer].attend(s, q[at:at + n].double().numpy(), self.dim ** -0.5 if scale is None else scale, window))
            at += n
        return out.double().cpu().numpy(), np.concatenate(want), q

    def tolerance(self, q, seqs, scale=None, layer=1):
        """Largest error of an output, as a share of the largest value it is made of.

        Scores: q in F16 terms is off by u = 2^-11 (one term) or 2^-22 (two) of its row's largest element at most half a step, D elements of k: a
        score is off by at most u D |q| |k| scale, and F32 sums of D terms by D 2^-24 of the same. A weight is off by that much (relative; twice, for
        the denominator's part), by u from its own rounding and by 2^-21 for its exponential; then the output's rounding."""
        s = self.dim ** -0.5 if scale is None else scale
        big_k = max(np.abs(self.ref[layer].numbers(i)[0]).max() for i in seqs)
        big_q = q.double().abs().max().item()
        u = 2.0 ** -22 if self.dtype == "f32" else 0.0 if self.dtype == "f16" else 2.0 ** -25
        score = self.dim * big_q * big_k * s * (u + self.dim * 2.0 ** -24 / 4)
        p = 2.0 ** -22 if self.dtype == "f32" else 2.0 ** -11
        return 2 * score + 2 * p + 2.0 ** -20 + HALF_STEP[self.dtype]

    def check_attend(self, seqs, counts, **kw):
        got, want, q = self.attend(seqs, counts, **kw)
        values = max(np.abs(self.ref[1].numbers(s)[1]).max() for s in seqs)
        assert np.abs(got - want).max() <= self.tolerance(q, seqs, kw.get("scale")) * values
        assert np.linalg.norm(got - want) <= 4 * (HALF_STEP[self.dtype] + 2.0 ** -19) * np.linalg.norm(want)


GEOMETRY = [(4, 4, 32, 16, 0, "f32"), (8, 2, 64, 16, 0, "f32"), (8, 2, 64, 64, 1, "bf16"), (6, 2, 96, 32, 0, "f16"), (6, 2, 96, 16, 1, "f32"),
            (4, 1, 128, 128, 0, "bf16"), (8, 1, 128, 32, 1, "f32"), (16, 2, 256, 64, 0, "f32"), (3, 3, 256, 16, 1, "f16"), (7, 1, 64, 128, 0, "f32")]


@pytest.mark.parametrize("geometry", GEOMETRY)
def test_codes_are_exact_at_every_way_to_append(geometry):
    p = Pair(*geometry)
    p.step([0], [1])
    p.check_numbers([0])
    p.step([0, 2], [1, 37])
    p.step([2, 0, 1], [1, 15, 130])
    p.step([1, 3, 2], [3, 0, 64])
    p.check_numbers([0, 1, 2])
    p.step([0], [200])
    p.check_numbers([2, 0, 1])
    assert p.kv.status() == 0


@pytest.mark.parametrize("geometry", GEOMETRY)
@pytest.mark.parametrize("lengths,counts", [([1], [1]), ([2, 64], [1, 1]), ([63, 65, 17], [1, 0, 1]), ([300, 5, 129, 64], [1, 4, 3, 64]), ([1000], [2]), ([700, 90], [40, 90])])
def test_attention(geometry, lengths, counts):
    p = Pair(*geometry)
    seqs = list(range(len(lengths)))[::-1]
    before = [n - c for n, c in zip(lengths, counts)]
    if sum(before):
        p.step(seqs, before)
    p.step(seqs, counts)
    p.check_attend(seqs, counts)


@pytest.mark.parametrize("geometry", [(8, 2, 64, 16, 0, "f32"), (8, 1, 128, 32, 1, "bf16"), (4, 1, 256, 64, 0, "f32")])
@pytest.mark.parametrize("window", [1, 17, 64, 300])
def test_attention_in_a_window(geometry, window):
    p = Pair(*geometry, layers=2)
    p.step([0, 1, 2], [500, 64, 3])
    p.step([2, 0, 1], [5, 1, 2])
    p.check_attend([2, 0, 1], [5, 1, 2], window=window)


@pytest.mark.parametrize("geometry", [(8, 2, 64, 32, 0, "bf16"), (4, 4, 128, 128, 1, "f16"), (8, 2, 128, 16, 0, "f32"), (16, 2, 256, 64, 0, "f32")])
def test_attention_over_long_and_ragged_contexts(geometry):
    """Runs that go over many tiles, and over many items, again and again without a wait between them."""
    p = Pair(*geometry, n_pages=9000, max_seqs=40, max_context=30000)
    lengths = [20011, 1, 7000, 64, 65] + [90 + 7 * i for i in range(30)]
    seqs = list(range(35))
    p.step(seqs, [n - 1 for n in lengths])
    p.step(seqs, [1] * 35)
    got, want, q = p.attend(seqs, [1] * 35)
    tol = p.tolerance(q, seqs) * max(np.abs(p.ref[1].numbers(s)[1]).max() for s in seqs)
    assert np.abs(got - want).max() <= tol
    qd = q.cuda()
    outs = [torch.empty_like(qd) for _ in range(50)]
    for o in outs:
        p.kv.attend(1, qd.data_ptr(), o.data_ptr(), TYPES[p.dtype][1])
    torch.cuda.synchronize()
    for o in outs:
        assert np.array_equal(o.double().cpu().numpy(), got)
    assert p.kv.status() == 0


@pytest.mark.parametrize("geometry", [(4, 4, 32, 16, 0, "f32"), (8, 2, 64, 32, 1, "bf16"), (6, 2, 96, 128, 0, "f16"), (16, 2, 256, 64, 1, "f32")])
def test_forks_go_their_own_ways(geometry):
    p = Pair(*geometry)
    p.step([0], [150])
    p.kv.fork(0, [3, 1])
    for r in p.ref:
        r.fork(0, 3)
        r.fork(0, 1)
    p.check_numbers([0, 1, 3])
    p.step([3, 0], [1, 2])
    p.step([1, 3], [40, 1])
    p.check_numbers([0, 1, 3])
    p.kv.truncate(0, 149)
    p.kv.free([3])
    for r in p.ref:
        r.truncate(0, 149)
        r.truncate(3, 0)
    p.step([0, 3], [3, 20])
    p.check_numbers([0, 1, 3])
    p.step([0, 1], [1, 1])
    p.check_attend([0, 1], [1, 1])


@pytest.mark.parametrize("n_pages", [400, 0])       # into new pages; in place, page after page
@pytest.mark.parametrize("geometry", [(4, 4, 32, 16, 0, "f32"), (8, 2, 64, 32, 1, "bf16"), (6, 2, 96, 128, 0, "f16"), (16, 2, 256, 64, 1, "f32")])
@pytest.mark.parametrize("length,first,step", [(40, 37, 2), (300, 0, 3), (300, 130, 2), (257, 128, 1), (200, 64, 50)])
def test_kept_tokens_move_together(geometry, n_pages, length, first, step):
    p = Pair(*geometry, n_pages=n_pages or -(-length // geometry[3]))
    p.step([2], [length - 3])
    p.step([2], [3])
    index = [i for i in range(length - first) if i % step == step - 1 or (step == 1 and i % 7 < 4)]
    if step == 1:
        index = [i for i in index if i % 7 < 4]
    p.kv.keep(2, first, index)
    for r in p.ref:
        r.keep(2, first, index)
    assert p.kv.length(2) == first + len(index)
    p.check_numbers([2])
    p.step([2], [1])
    p.check_numbers([2])
    p.check_attend([2], [1])


def test_keep_leaves_other_holders_alone():
    p = Pair(8, 2, 64, 32, 0, "f32")
    p.step([0], [100])
    p.kv.fork(0, [1])
    index = list(range(0, 60, 2))
    p.kv.keep(1, 40, index)
    for r in p.ref:
        r.fork(0, 1)
        r.keep(1, 40, index)
    p.check_numbers([0, 1])


@pytest.mark.parametrize("codes", [0, 1])
def test_rows_that_are_not_numbers(codes):
    p = Pair(4, 2, 64, 16, codes, "f32", layers=1)
    k, v = p.rows(20), p.rows(20)
    k[3, 0, 5], k[7, 1, 0], v[19, 1, 63], v[2, 0, 1] = float("inf"), float("-inf"), float("nan"), float("inf")
    v[16:, 0] = float("inf")                # a page and head without a finite number
    k[:, 1] = 0.0
    k[7, 1, 0] = float("nan")
    p.step([0], [20], rows=[(k, v)])
    p.check_numbers([0])
    assert p.kv.status() == 32 and p.kv.status() == 0


@pytest.mark.parametrize("codes", [0, 1])
def test_ties_and_sizes_of_codes(codes):
    """Quotients on and next to the middles between codes, scales from 2^-100 to near the largest number."""
    dim, page = 256, 16
    limit = kv_oracle.LIMIT[codes]
    for size in (1.0, 3.0, 2.0 ** -70, 1e-38, 1e-45, 1e30, 3.0e38 / limit):
        p = Pair(1, 1, dim, page, codes, "f32", layers=1)
        s = float(np.float32(size))
        mid = (np.arange(dim) % 127 + 0.5) * s if codes == 0 else np.linspace(0.001, 440, dim) * s
        if codes == 1:
            mid = kv_oracle.e4m3_round(mid / s) * s
            mid = (mid + np.roll(mid, -1)) / 2
        rows = np.stack([mid, np.nextafter(mid.astype(np.float32), np.float32(3e38)), np.nextafter(mid.astype(np.float32), np.float32(0)), -mid]).astype(np.float32)
        rows[:, 0] = np.float32(limit) * np.float32(s)
        x = torch.from_numpy(rows)[:, None, :]
        p.step([0], [4], rows=[(x, x.flip(0).contiguous())])
        p.check_numbers([0])
        y = x * torch.tensor([1.0, 1.37, 0.2, 1.0]).reshape(4, 1, 1) if size < 1e30 else x
        p.step([0], [4], rows=[(y, x)])
        p.check_numbers([0])


def test_attention_when_values_differ_by_orders_of_magnitude():
    """A page whose values are small must not be rounded away beside one whose values are large, where its tokens have the weight."""
    p = Pair(8, 2, 64, 16, 0, "f32", layers=1)
    k, v = p.rows(64).float(), p.rows(64).float()
    k[:] = 0.01 * k
    v[:16] *= 1e6
    v[16:32] *= 1e-8
    v[32:48] = 0.0
    q = p.rand(1, 8, 64)
    k[20] = q[0, ::4] * 6          # the weight is on token 20, whose values are small
    p.step([0], [64], rows=[(k, v)])
    p.step([0], [1], rows=[(k[:1], v[40:41])])
    got, want, _ = p.attend([0], [1], q=q, layer=0, scale=1.0)
    assert np.abs(got - want).max() <= 1e-5 * np.abs(want).max()
    assert np.abs(want).max() < 1e6


def test_strides_streams_and_rows_behind_the_last():
    p = Pair(8, 2, 64, 16, 0, "f32", layers=1)
    p.step([0, 1], [70, 30])
    n, q_w, kv_w = 3, 8 * 64, 2 * 64
    fused = p.rand(n + 2, q_w + 2 * kv_w + 5).cuda()
    out = torch.full((n + 2, q_w + 3), 9.0, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    w = fused.shape[1]
    p.kv.begin([1, 0], [2, 1], s.cuda_stream)
    p.kv.append(0, fused.data_ptr() + 4 * q_w, fused.data_ptr() + 4 * (q_w + kv_w), k_stride=w, v_stride=w, stream=s.cuda_stream)
    p.kv.attend(0, fused.data_ptr(), out.data_ptr(), q_stride=w, out_stride=q_w + 3, stream=s.cuda_stream)
    s.synchronize()
    f = fused.cpu().double().numpy()
    for seq, a, b in ((1, 0, 2), (0, 2, 3)):
        p.ref[0].append(seq, f[a:b, q_w:q_w + kv_w].reshape(-1, 2, 64), f[a:b, q_w + kv_w:q_w + 2 * kv_w].reshape(-1, 2, 64))
    p.check_numbers([0, 1])
    o = out.cpu().double().numpy()
    for seq, a, b in ((1, 0, 2), (0, 2, 3)):
        want = p.ref[0].attend(seq, f[a:b, :q_w].reshape(-1, 8, 64), 0.125, 0)
        assert np.abs(o[a:b, :q_w].reshape(-1, 8, 64) - want).max() < 2e-5
    assert (o[n:] == 9.0).all() and (o[:, q_w:] == 9.0).all()
    # in place: the output over the queries
    q = p.rand(3, 8, 64).cuda()
    want = torch.empty_like(q)
    p.kv.attend(0, q.data_ptr(), want.data_ptr())
    p.kv.attend(0, q.data_ptr(), q.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(q, want)


def test_a_captured_step_serves_the_steps_that_follow():
    p = Pair(8, 2, 64, 16, 0, "f32", layers=1)
    p.step([0, 1], [15, 200])
    k, v, q = (torch.zeros(2, h, 64, device="cuda") for h in (2, 2, 8))
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    p.kv.begin([0, 1], [1, 1], s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        p.kv.append(0, k.data_ptr(), v.data_ptr(), stream=s.cuda_stream)
        p.kv.attend(0, q.data_ptr(), out.data_ptr(), stream=s.cuda_stream)
        with pytest.raises(wd.WdError, match="captured"):
            p.kv.begin([0], [1], s.cuda_stream)
        with pytest.raises(wd.WdError, match="captured"):
            p.kv.free([0], s.cuda_stream)
    for i in range(20):
        seqs, counts = ([0, 1], [1, 1]) if i % 3 else ([1], [2])
        if i:
            p.kv.begin(seqs, counts, s.cuda_stream)
        else:
            seqs, counts = [0, 1], [1, 1]
        rows = [p.rand(2, h, 64) for h in (2, 2, 8)]
        with torch.cuda.stream(s):
            for to, x in zip((k, v, q), rows):
                to.copy_(x)
            g.replay()
        s.synchronize()
        at = 0
        for seq, n in zip(seqs, counts):
            p.ref[0].append(seq, rows[0][at:at + n].double().numpy(), rows[1][at:at + n].double().numpy())
            want = p.ref[0].attend(seq, rows[2][at:at + n].double().numpy(), 0.125, 0)
            assert np.abs(out[at:at + n].double().cpu().numpy() - want).max() < 2e-5
            at += n
    p.check_numbers([0, 1])


def test_calls_out_of_order_and_bad_arguments():
    kv = wd.KvCache(2, 8, 2, 64, 8, 2, 100, page_tokens=16)
    x = torch.zeros(4, 8, 64, device="cuda")
    a = x.data_ptr()
    for call in (lambda: kv.append(0, a, a), lambda: kv.attend(0, a, a)):
        with pytest.raises(wd.WdError, match="no step"):
            call()
    kv.begin([0], [4])
    for call in (lambda: kv.append(2, a, a), lambda: kv.append(-1, a, a), lambda: kv.append(0, a + 2, a), lambda: kv.append(0, a, None),
                 lambda: kv.append(0, a, a, wd.TYPE_Q8_0), lambda: kv.append(0, a, a, k_stride=127), lambda: kv.attend(0, a, a, scale=0.0),
                 lambda: kv.attend(0, a, a, scale=float("nan")), lambda: kv.attend(0, a, a, window=-1), lambda: kv.attend(0, a, a, q_stride=511),
                 lambda: kv.attend(0, None, a), lambda: kv.read(0, [0], [0], [5], a, a), lambda: kv.read(0, [0], [3], [2 ** 31 - 2], a, a),
                 lambda: kv.read(2, [0], [0], [1], a, a), lambda: kv.read(0, [2], [0], [0], a, a), lambda: kv.read(0, [0], [0], [1], None, None)):
        with pytest.raises(wd.WdError):
            call()
    kv.append(0, a, a)
    kv.truncate(0, 2)
    with pytest.raises(wd.WdError, match="no step"):
        kv.attend(0, a, a)
    kv.begin([0, 1], [0, 0])
    kv.attend(0, a, a)              # no rows: no work
    with pytest.raises(wd.WdError):
        wd.KvCache(1, 8, 2, 64, 8, 2, 100, device=99)
    with pytest.raises(wd.WdError, match="fit"):
        wd.KvCache(64, 8, 8, 256, 1 << 20, 2, 100, page_tokens=128)


@pytest.mark.parametrize("geometry", GEOMETRY)
@pytest.mark.parametrize("lengths,counts", [([128], [128]), ([130], [97]), ([400, 260, 7], [300, 1, 7]), ([513], [513]), ([1500, 700], [200, 333])])
def test_attention_of_a_prompt(geometry, lengths, counts):
    p = Pair(*geometry)
    seqs = list(range(len(lengths)))
    before = [n - c for n, c in zip(lengths, counts)]
    if sum(before):
        p.step(seqs, before)
    p.step(seqs, counts)
    p.check_attend(seqs, counts)
    assert p.kv.status() == 0


@pytest.mark.parametrize("geometry", [(8, 2, 64, 16, 0, "f32"), (8, 1, 128, 32, 1, "bf16"), (16, 2, 256, 64, 0, "f32"), (6, 2, 96, 128, 0, "f16")])
@pytest.mark.parametrize("window", [1, 63, 200, 1000])
def test_attention_of_a_prompt_in_a_window(geometry, window):
    p = Pair(*geometry)
    p.step([0, 1, 2], [500, 0, 30])
    p.step([2, 0, 1], [170, 259, 600])
    p.check_attend([2, 0, 1], [170, 259, 600], window=window)


def test_rows_of_a_prompt_far_apart_in_size():
    """A few rows of a tile whose scores leap (the sums are brought to a new maximum), rows of zeros, rows of 1e30 and of 1e-30."""
    p = Pair(8, 2, 64, 16, 0, "f32")
    k, v = p.rows(600), p.rows(600)
    k *= torch.linspace(0.1, 30, 600)[:, None, None]
    v[100:120] *= 1e5
    p.step([0], [600], rows=[(k, v)] * 2)
    q = p.rand(600, 8, 64)
    q[5], q[200:210], q[17] = 0.0, q[200:210] * 30, q[17] * 1e-30
    got, want, _ = p.attend([0], [600], q=q)
    values = np.abs(p.ref[1].numbers(0)[1]).max()
    # scores up to 30 * 30 * 8 * 5 / 8 = 4,500, in F32: 4,500 * 2^-23 of a weight, and what comes of q's terms
    assert np.abs(got - want).max() <= (4500 * 64 * 2.0 ** -24 + 2.0 ** -18) * values
    small = np.ones(600, bool)
    small[200:210] = False
    assert np.linalg.norm((got - want)[small]) <= 2e-4 * np.linalg.norm(want[small])


@pytest.mark.parametrize("geometry", GEOMETRY + [(16, 2, 128, 64, 1, "f16"), (8, 8, 64, 32, 0, "bf16"), (32, 4, 32, 16, 1, "bf16"), (12, 2, 256, 32, 1, "bf16")])
@pytest.mark.parametrize("before,count,window", [(0, 4000, 0), (700, 4031, 0), (300, 3500, 1500), (5000, 900, 0), (20, 6001, 100)])
def test_prompts_that_the_tensor_cores_take(geometry, before, count, window):
    """Chunks that are large enough for the kernel for prompts, whole items and items cut into runs; some of the rows are looked at."""
    p = Pair(*geometry, n_pages=900, max_context=7000, layers=1)
    if before:
        p.step([1], [before])
    p.step([1, 0], [count, 3])
    q = p.rand(count + 3, p.heads, p.dim, size=1.5)
    qd = q.cuda()
    out = torch.full_like(qd, 3.0)
    p.kv.attend(0, qd.data_ptr(), out.data_ptr(), TYPES[p.dtype][1], window=window)
    if count > 3000 and not window:
        assert p.kv.kernel_name().startswith("kv_prompt_kernel")
    torch.cuda.synchronize()
    rows = np.unique(np.concatenate([[0, 1, 127, 128, 255, 256, count // 2, count - 2, count - 1], np.random.default_rng(1).integers(0, count, 60)]))
    got = out.double().cpu().numpy()
    values = max(np.abs(p.ref[0].numbers(i)[1]).max() for i in (0, 1))
    tol = p.tolerance(q, [1], layer=0)
    want = p.ref[0].attend(1, q[:count].double().numpy(), p.dim ** -0.5, window, rows=rows)
    assert np.abs(got[rows] - want).max() <= tol * values
    assert np.linalg.norm(got[rows] - want) <= 4 * (HALF_STEP[p.dtype] + 2.0 ** -19) * np.linalg.norm(want)
    want = p.ref[0].attend(0, q[count:].double().numpy(), p.dim ** -0.5, window)
    assert np.abs(got[count:] - want).max() <= tol * values
    again = torch.empty_like(out)
    p.kv.attend(0, qd.data_ptr(), again.data_ptr(), TYPES[p.dtype][1], window=window)
    torch.cuda.synchronize()
    assert torch.equal(out, again) and p.kv.status() == 0


@pytest.mark.parametrize("chunk,name", [(6000, "kv_prompt_kernel"), (4000, "kv_prompt_kernel, kv_prompt_join_kernel")])       # 94 items; 63, in two runs each
def test_a_prompt_kernel_in_a_graph_serves_other_steps(chunk, name):
    """Captured at a long chunk, replayed at shorter ones, at a step of many sequences, and at one without rows."""
    p = Pair(4, 1, 64, 32, 0, "bf16", n_pages=900, max_context=9000, layers=1)
    p.step([0], [chunk])
    q = p.rand(6000, 4, 64).cuda()
    out = torch.full_like(q, 3.0)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        p.kv.attend(0, q.data_ptr(), out.data_ptr(), wd.TYPE_BF16, stream=s.cuda_stream)
    assert p.kv.kernel_name() == name
    for seqs, counts in (([0], [100]), ([1, 2, 3, 0], [700, 1, 64, 1]), ([4, 5, 6, 7, 1, 2], [900, 800, 300, 200, 100, 600]), ([2], [0]), ([3], [1])):
        p.step(seqs, counts)
        torch.cuda.synchronize()
        out.fill_(3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        got, at = out.double().cpu().numpy(), 0
        for seq, n in zip(seqs, counts):
            if n:
                want = p.ref[0].attend(seq, q[at:at + n].double().cpu().numpy(), 0.125, 0)
                assert np.linalg.norm(got[at:at + n] - want) <= 4 * 2.0 ** -8 * np.linalg.norm(want)
            at += n
        assert (got[at:] == 3.0).all()


@pytest.mark.parametrize("counts", [[1, 2], [700, 300]])        # the kernel for few rows, and the one for prompts
def test_a_window_beyond_every_context_is_none(counts):
    p = Pair(8, 2, 64, 16, 0, "f16")
    p.step([0, 1], counts)
    q = p.rand(sum(counts), 8, 64, size=1.5)
    seen = []
    for window in (0, 2 ** 31 - 1, 2 ** 31 - 64, 6000):
        p.check_attend([0, 1], counts, window=window, q=q)
        seen.append(p.attend([0, 1], counts, window=window, q=q)[0])
    assert all(np.array_equal(seen[0], x) for x in seen[1:])


def test_a_scale_that_no_number_holds():
    kv = wd.KvCache(1, 8, 2, 64, 8, 2, 100)
    x = torch.zeros(1, 8, 64, device="cuda")
    kv.begin([0], [1])
    with pytest.raises(wd.WdError, match="scale"):
        kv.attend(0, x.data_ptr(), x.data_ptr(), scale=3.0e38)


def test_a_step_without_rows_is_not_captured():
    """A graph of it would hold nothing, and its replays would leave the steps that follow undone."""
    kv = wd.KvCache(1, 8, 2, 64, 8, 2, 100)
    x = torch.zeros(1, 8, 64, device="cuda")
    s = torch.cuda.Stream()
    kv.begin([0], [0], s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        x.add_(0.0)
        with pytest.raises(wd.WdError, match="captured"):
            kv.append(0, x.data_ptr(), x.data_ptr(), stream=s.cuda_stream)
        with pytest.raises(wd.WdError, match="captured"):
            kv.attend(0, x.data_ptr(), x.data_ptr(), stream=s.cuda_stream)
    kv.append(0, x.data_ptr(), x.data_ptr(), stream=s.cuda_stream)


@pytest.mark.parametrize("page", [16, 128])
def test_a_captured_step_of_a_token_serves_one_of_many(page):
    """More pages, items and rows than the captured launch was made for."""
    p = Pair(8, 2, 64, page, 0, "f32", layers=1)
    k, v, q = (torch.zeros(300, h, 64, device="cuda") for h in (2, 2, 8))
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    p.kv.begin([0], [1], s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        p.kv.append(0, k.data_ptr(), v.data_ptr(), stream=s.cuda_stream)
        p.kv.attend(0, q.data_ptr(), out.data_ptr(), stream=s.cuda_stream)
    p.kv.free([0], s.cuda_stream)
    p.kv.begin([0, 1], [133, 167], s.cuda_stream)
    rows = [p.rand(300, h, 64) for h in (2, 2, 8)]
    with torch.cuda.stream(s):
        for to, x in zip((k, v, q), rows):
            to.copy_(x)
        g.replay()
    s.synchronize()
    for seq, at, n in ((0, 0, 133), (1, 133, 167)):
        p.ref[0].append(seq, rows[0][at:at + n].double().numpy(), rows[1][at:at + n].double().numpy())
        want = p.ref[0].attend(seq, rows[2][at:at + n].double().numpy(), 0.125, 0)
        values = np.abs(p.ref[0].numbers(seq)[1]).max()
        assert np.abs(out[at:at + n].double().cpu().numpy() - want).max() <= p.tolerance(rows[2], [seq], layer=0) * values
    p.check_numbers([0, 1])


def test_a_refused_call_leaves_nothing_behind():
    """An error of the runtime that one call has returned is not found by the next one's look at its launches."""
    kv = wd.KvCache(1, 8, 2, 64, 8, 2, 100)
    x = torch.ones(1, 8, 64, device="cuda")
    for _ in range(2):
        with pytest.raises(wd.WdError, match="device"):
            wd.KvCache(1, 8, 2, 64, 8, 2, 100, device=99)
        kv.begin([0], [1])
        with pytest.raises(wd.WdError, match="device"):
            wd.KvCache(1, 8, 2, 64, 8, 2, 100, device=99)
        kv.append(0, x.data_ptr(), x.data_ptr())
    kv.attend(0, x.data_ptr(), x.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(x, torch.ones_like(x))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("counts", [[1, 3], [400, 300]])        # the kernel for few rows, and the one for prompts
def test_queries_that_are_not_numbers_stay_by_themselves(dtype, counts):
    p = Pair(8, 2, 64, 16, 0, dtype)
    p.step([0, 1], [200, 40])
    p.step([0, 1], counts)
    q = p.rand(sum(counts), 8, 64)
    clean = p.attend([0, 1], counts, q=q)[0]
    values = max(np.abs(p.ref[1].numbers(i)[1]).max() for i in (0, 1))
    tol = 2 * p.tolerance(q, [0, 1]) * values           # both are that near to the real answer (a row may take another's reason to be scaled anew)
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = q.clone()
        x[0, 3, 5] = bad
        x[-1, 0, 63] = bad
        got = p.attend([0, 1], counts, q=x)[0]
        hit = np.zeros(got.shape[:2], bool)
        hit[0, 3] = hit[-1, 0] = True
        assert np.abs(got[~hit] - clean[~hit]).max() <= tol
        assert np.isnan(got[hit]).all()
