"""Norms and rotary positions on the way into the 8-bit cache against 64 bits: codes are exact, queries to their type."""
import numpy as np
import pytest
import torch

import warpdecode_b200 as wd
from rope_oracle import frequencies, rotated
from test_gpu_kv_cache import HALF_STEP, TYPES, Pair

pytestmark = pytest.mark.gpu


class Turned:
    """A cache and its plain one, fed by append_rope."""

    def __init__(self, heads, kv_heads, dim, page, codes, dtype, rotary=0, theta=10000.0, sections=(), neighbours=False, factor=1.0, inv_freq=None, norm=True, eps=1e-6, **kw):
        self.p = Pair(heads, kv_heads, dim, page, codes, dtype, **kw)
        self.rope = wd.Rope(dim, rotary, theta=theta, sections=sections, neighbours=neighbours, factor=factor, inv_freq=inv_freq)
        self.freq = frequencies(rotary or dim, theta) if inv_freq is None else np.asarray(inv_freq)
        self.plain = dict(sections=sections, neighbours=neighbours, eps=eps, factor=float(np.float32(factor)))
        self.axes, self.eps = max(1, len(sections)), eps
        self.norms = [(1.0 + 0.3 * torch.randn(dim, generator=self.p.gen)) for _ in range(2)] if norm else [None, None]
        self.norms_dev = [None if w is None else w.cuda() for w in self.norms]

    def positions(self, n):
        return torch.randint(-100, 200000, (n, self.axes), generator=self.p.gen, dtype=torch.int32)

    def own_places(self, seqs, counts):
        return torch.cat([torch.arange(self.p.kv.length(s) - n, self.p.kv.length(s)) for s, n in zip(seqs, counts)])[:, None].expand(-1, self.axes)

    def rows(self, n):
        return self.p.rows(n), self.p.rows(n), self.p.rand(n, self.p.heads, self.p.dim, size=1.5)

    def send(self, layer, k, v, q, positions, stream=None, **kw):
        """One call on device copies; returns q's output."""
        dev = [x.cuda() for x in (k, v, q)]
        out = torch.full_like(dev[2], 3.0)
        pos = None if positions is None else positions.cuda()
        torch.cuda.synchronize()
        self.call(layer, dev[0].data_ptr(), dev[1].data_ptr(), dev[2].data_ptr(), out.data_ptr(), None if pos is None else pos.data_ptr(), stream=stream, **kw)
        torch.cuda.synchronize()
        return out

    def call(self, layer, k, v, q, out, positions, stream=None, **kw):
        w = [None if x is None else x.data_ptr() for x in self.norms_dev]
        self.p.kv.append_rope(layer, self.rope, k, v, q, out, positions, q_norm_ptr=w[0], k_norm_ptr=w[1], eps=self.eps, type=TYPES[self.p.dtype][1], stream=stream, **kw)

    def check_q(self, got, q, positions):
        """Relative to the two elements that one is made of, in half steps of F32: the angle 1.6 (of pi times a float), its functions 2 each, the sum of squares 7, its
        root, the quotient's two products 4, the rotation's two 3, the factor 1: below 2^5; then the output's rounding."""
        want, size = rotated(q.double().numpy(), positions.numpy(), self.freq, norm=self.norms[0], **self.plain)
        off = np.abs(got.double().cpu().numpy() - want)
        assert (off <= 2.0 ** -19 * size + HALF_STEP[self.p.dtype] * np.abs(want) + 1e-37 + (2.0 ** -25 if self.p.dtype == "f16" else 0)).all()

    def keep_plain(self, layer, seqs, counts, k, v, positions):
        turned = rotated(k.double().numpy(), positions.numpy(), self.freq, norm=self.norms[1], **self.plain)[0].astype(np.float32)
        at = 0
        for s, n in zip(seqs, counts):
            self.p.ref[layer].append(s, turned[at:at + n], v[at:at + n].double().numpy())
            at += n

    def step(self, seqs, counts, own=False):
        self.p.kv.begin(seqs, counts)
        n = sum(counts)
        pos = self.own_places(seqs, counts) if own else self.positions(n)
        for layer in range(self.p.layers):
            k, v, q = self.rows(n)
            out = self.send(layer, k, v, q, None if own else pos)
            self.check_q(out, q, pos)
            self.keep_plain(layer, seqs, counts, k, v, pos)


KINDS = [(dict(heads=4, kv_heads=4, dim=32, page=16, codes=0, dtype="f32"), dict()),
         (dict(heads=8, kv_heads=2, dim=64, page=16, codes=0, dtype="bf16"), dict(neighbours=True, norm=False)),
         (dict(heads=6, kv_heads=2, dim=96, page=32, codes=1, dtype="f16"), dict(rotary=48)),
         (dict(heads=6, kv_heads=2, dim=96, page=16, codes=0, dtype="f32"), dict(neighbours=True)),
         (dict(heads=8, kv_heads=1, dim=128, page=64, codes=0, dtype="bf16"), dict(sections=(16, 24, 24), theta=1e6)),
         (dict(heads=7, kv_heads=1, dim=128, page=128, codes=1, dtype="f32"), dict(rotary=64, sections=(5, 0, 26, 1), neighbours=True, factor=1.25)),
         (dict(heads=16, kv_heads=2, dim=256, page=64, codes=0, dtype="f32"), dict(rotary=64)),
         (dict(heads=3, kv_heads=3, dim=256, page=128, codes=1, dtype="bf16"), dict(sections=(64, 64))),
         (dict(heads=4, kv_heads=1, dim=64, page=32, codes=0, dtype="f16"), dict(rotary=6, inv_freq=[1.0, -0.37, 0.0], norm=False)),
         (dict(heads=2, kv_heads=2, dim=64, page=128, codes=0, dtype="f32"), dict(rotary=2, eps=0.1))]


@pytest.mark.parametrize("shape,kind", KINDS)
def test_codes_are_exact_and_queries_turned(shape, kind):
    t = Turned(**shape, **kind)
    t.step([0], [1])
    t.p.check_numbers([0])
    t.step([0, 2], [1, 37])
    t.step([2, 0, 1], [1, 15, 130], own=True)
    t.step([1, 3, 2], [3, 0, 64])
    t.p.check_numbers([0, 1, 2])
    t.step([0], [300], own=True)            # more than shared memory holds of a page of 128 tokens of 256
    t.p.check_numbers([2, 0, 1])
    assert t.p.kv.status() == 0


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rotary,neighbours,norm", [(0, False, True), (0, False, False), (0, True, True), (32, False, True), (16, True, False)])
def test_many_tokens_of_a_page(dim, dtype, rotary, neighbours, norm):
    g = {32: 1, 64: 3, 96: 2, 128: 7, 256: 4}[dim]
    t = Turned(2 * g, 2, dim, 128, dim // 32 % 2, dtype, rotary=rotary, neighbours=neighbours, norm=norm, max_context=1000, n_pages=40, layers=1)
    t.step([0], [128])
    t.step([1, 0, 2], [67, 201, 99], own=True)
    t.step([2, 1], [130, 1])
    t.p.check_numbers([0, 1, 2])
    assert t.p.kv.status() == 0


def test_many_tokens_in_place_of_parts_of_a_fused_row():
    t = Turned(6, 2, 96, 64, 0, "bf16", layers=1)
    n, width = 150, 10 * 96
    k, v, q = t.rows(n)
    for lead in (0, 8, 3):              # (rows on boundaries of 16 bytes, and not)
        row = torch.full((n, width + 16), 9.0, dtype=torch.bfloat16)
        row[:, lead:lead + width] = torch.cat([x.reshape(n, -1) for x in (q, k, v)], dim=1)
        dev, at = row.cuda(), 2 * lead
        t.p.kv.begin([0], [n])
        pos = t.own_places([0], [n])
        torch.cuda.synchronize()
        here = lambda e: dev.data_ptr() + at + 2 * e  # noqa: E731
        t.call(0, here(6 * 96), here(8 * 96), here(0), here(0), None, q_stride=width + 16, q_out_stride=width + 16, k_stride=width + 16, v_stride=width + 16)
        torch.cuda.synchronize()
        got = dev.cpu()
        t.check_q(got[:, lead:lead + 576].reshape(n, 6, 96), q, pos)
        assert torch.equal(got[:, :lead], row[:, :lead]) and torch.equal(got[:, lead + 576:], row[:, lead + 576:])
        t.keep_plain(0, [0], [n], k, v, pos)
        t.p.check_numbers([0])


def test_the_same_rows_again_leave_the_cache_as_it_is():
    t = Turned(8, 2, 128, 64, 0, "bf16", layers=1)
    t.step([0], [50])
    t.p.kv.begin([0, 1], [30, 7])
    k, v, q = t.rows(37)
    pos = t.positions(37)
    for _ in range(3):
        t.send(0, k, v, q, pos)
    t.keep_plain(0, [0, 1], [30, 7], k, v, pos)
    t.p.check_numbers([0, 1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lead", [0, 1])            # elements that the rows lie beside a boundary of 16 bytes
def test_parts_of_a_fused_row_in_place(dtype, lead):
    t = Turned(8, 2, 64, 16, 0, dtype, layers=1)
    t.p.kv.begin([0, 1], [19, 2])
    k, v, q = t.rows(21)
    pos = t.positions(21)
    row = torch.cat([q.reshape(21, -1), k.reshape(21, -1), v.reshape(21, -1), torch.zeros(21, 5, dtype=q.dtype)], dim=1)
    buf = torch.full((21 * row.shape[1] + 8,), 7.0, dtype=q.dtype, device="cuda")
    view = buf[lead:lead + row.numel()].view(row.shape)
    view.copy_(row)
    torch.cuda.synchronize()
    width, size = row.shape[1], row.element_size()
    at, pd = view.data_ptr(), pos.cuda()
    strides = dict(q_stride=width, q_out_stride=width, k_stride=width, v_stride=width)
    t.call(0, at + 512 * size, at + 640 * size, at, at, pd.data_ptr(), **strides)
    torch.cuda.synchronize()
    t.check_q(view[:, :512].reshape(21, 8, 64), q, pos)
    t.keep_plain(0, [0, 1], [19, 2], k, v, pos)
    t.p.check_numbers([0, 1])
    assert torch.equal(view[:, 512:].cpu(), row[:, 512:]) and (buf[lead + row.numel():] == 7.0).all() and (buf[:lead] == 7.0).all()


def test_without_queries_and_with_one_norm():
    t = Turned(8, 2, 64, 16, 0, "f32", layers=1)
    t.norms[0], t.norms_dev[0] = None, None
    t.p.kv.begin([0], [20])
    k, v, q = t.rows(20)
    pos = t.positions(20)
    kd, vd, pd = k.cuda(), v.cuda(), pos.cuda()
    torch.cuda.synchronize()
    t.call(0, kd.data_ptr(), vd.data_ptr(), None, None, pd.data_ptr())
    t.keep_plain(0, [0], [20], k, v, pos)
    t.p.check_numbers([0])
    t.check_q(t.send(0, k, v, q, pos), q, pos)


def test_it_is_append_where_nothing_turns():
    """Positions 0 and no norm: the rows themselves, in both orders of pairs; attention over them is the same to the bit."""
    rows = None
    outs = []
    for way in ("append", "halves", "neighbours"):
        t = Turned(8, 2, 128, 32, 0, "bf16", layers=1, norm=False, neighbours=way == "neighbours")
        t.p.kv.begin([0], [77])
        rows = rows or t.rows(77)
        k, v, q = (x.cuda() for x in rows)
        torch.cuda.synchronize()
        if way == "append":
            t.p.kv.append(0, k.data_ptr(), v.data_ptr(), wd.TYPE_BF16)
        else:
            q = t.send(0, *rows, torch.zeros(77, 1, dtype=torch.int32))
            assert torch.equal(q.cpu(), rows[2])
        out = torch.empty_like(q)
        t.p.kv.attend(0, q.data_ptr(), out.data_ptr(), wd.TYPE_BF16)
        torch.cuda.synchronize()
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("size", [1e25, 1e-25, 1e-42])
def test_rows_whose_squares_f32_does_not_hold(size):
    t = Turned(4, 2, 64, 16, 0, "f32", layers=1, eps=1e-30)
    t.p.kv.begin([0], [9])
    k, v, q = t.rows(9)
    k, q = k * size, q * size
    pos = t.positions(9)
    out = t.send(0, k, v, q, pos)
    t.check_q(out, q, pos)
    t.keep_plain(0, [0], [9], k, v, pos)
    t.p.check_numbers([0])


def test_numbers_that_are_none_stay_in_their_head_and_row():
    t = Turned(8, 2, 64, 16, 0, "f32", layers=1)
    t.p.kv.begin([0], [40])
    k, v, q = t.rows(40)
    k[3, 1, 5], k[20, 0, 7], v[30, 1, 3] = float("nan"), float("inf"), float("-inf")
    q[7, 2, 60], q[8, 3, 1] = float("nan"), float("inf")
    pos = t.positions(40)
    out = t.send(0, k, v, q, pos)
    assert t.p.kv.status() == 32
    with np.errstate(invalid="ignore"):
        t.keep_plain(0, [0], [40], k, v, pos)
    t.p.check_numbers([0])
    bad = ~torch.isfinite(out)
    assert bad[7, 2].any() and bad[8, 3].any()
    q[7, 2], q[8, 3], out[7, 2], out[8, 3] = 0.0, 0.0, 0.0, 0.0
    t.check_q(out, q, pos)


def test_captured_and_replayed_on_other_steps():
    """A replay on a step with more rows of a page than the captured one had, and on another order of sequences."""
    t = Turned(16, 2, 256, 128, 0, "bf16", rotary=64, layers=1, max_seqs=4)
    k, v, q = (torch.zeros(200, h, 256, dtype=torch.bfloat16, device="cuda") for h in (2, 2, 16))
    out, pos = torch.zeros_like(q), torch.zeros(200, 1, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    t.p.kv.begin([0, 1], [1, 1], s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        t.call(0, k.data_ptr(), v.data_ptr(), q.data_ptr(), out.data_ptr(), pos.data_ptr(), stream=s.cuda_stream)
    first = True
    for seqs, counts in (([0, 1], [1, 1]), ([1, 0], [60, 3]), ([2], [200]), ([0, 2, 1, 3], [1, 1, 1, 5])):
        if not first:
            t.p.kv.begin(seqs, counts, s.cuda_stream)
        first = False
        n = sum(counts)
        rows = t.rows(n)
        p = t.positions(n)
        with torch.cuda.stream(s):
            for to, x in zip((k, v, q, pos), (*rows, p)):
                to[:n].copy_(x)
            out.fill_(5.0)
            g.replay()
        s.synchronize()
        t.check_q(out[:n], rows[2], p)
        assert (out[n:] == 5.0).all()
        t.keep_plain(0, seqs, counts, rows[0], rows[1], p)
    t.p.check_numbers([0, 1, 2, 3])
    t.p.kv.truncate(0, 2, s.cuda_stream)
    with torch.cuda.stream(s):
        out.fill_(5.0)
        g.replay()
    s.synchronize()
    assert (out == 5.0).all()


def test_refusals():
    t = Turned(8, 2, 64, 16, 0, "f32", layers=2)
    other = wd.Rope(128)
    a = dict(layer=0, rope=t.rope, k_ptr=1024, v_ptr=1024, q_ptr=2048, q_out_ptr=4096, positions_ptr=1024)
    kv = t.p.kv
    with pytest.raises(wd.WdError, match="no step"):
        kv.append_rope(**a)
    kv.begin([0], [0])
    kv.append_rope(**{**a, "k_ptr": None})                 # no rows: nothing is asked of their address
    kv.begin([0], [3])
    for bad in (dict(layer=2), dict(layer=-1), dict(rope=other), dict(k_ptr=None), dict(v_ptr=None), dict(q_ptr=None), dict(q_out_ptr=None), dict(k_ptr=1026), dict(q_out_ptr=4097),
                dict(positions_ptr=1025), dict(q_norm_ptr=1026), dict(k_norm_ptr=1024, eps=0.0), dict(q_norm_ptr=1024, eps=-1.0), dict(q_norm_ptr=1024, eps=float("nan")),
                dict(type=wd.TYPE_Q8_0), dict(k_stride=127), dict(v_stride=-1), dict(q_stride=511), dict(q_out_stride=511), dict(q_out_ptr=2048, q_out_stride=600)):
        with pytest.raises(wd.WdError):
            kv.append_rope(**{**a, **bad})
    assert kv.status() == 0
