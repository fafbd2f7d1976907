"""Calls of two host threads at once, of one kernel and other sizes: what a launch needs of a kernel belongs to the call."""
import ctypes
import threading

import numpy as np
import pytest
import torch

import warpdecode_b200 as wd

pytestmark = pytest.mark.gpu


def side_by_side(*calls, turns):
    """Every call `turns` times, each by a thread of its own; what the threads raised."""
    start, raised = threading.Barrier(len(calls)), []

    def run(call):
        try:
            start.wait()
            for _ in range(turns):
                call()
        except Exception as e:          # noqa: BLE001 (said by the test)
            raised.append(e)

    threads = [threading.Thread(target=run, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return raised


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("dtype,type_", [(torch.float32, wd.TYPE_F32), (torch.bfloat16, wd.TYPE_BF16)])
def test_verification_of_two_vocabularies(with_draft, dtype, type_):
    def one(vocab, seed):
        gen = torch.Generator("cuda").manual_seed(seed)
        x = (3 * torch.randn(3, vocab, generator=gen, device="cuda")).to(dtype)
        d = x.clone()
        tokens = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
        u = torch.tensor([0.4, 0.0, 0.0], device="cuda")
        out = [torch.full((n,), -7, dtype=torch.int32, device="cuda") for n in (3, 1, 1)]
        s = torch.cuda.Stream()
        torch.cuda.synchronize()

        def call():
            wd.verify_drafts(x.data_ptr(), 3, vocab, tokens.data_ptr(), u.data_ptr(), *(o.data_ptr() for o in out), draft_ptr=d.data_ptr() if with_draft else None, type=type_,
                             stream=s.cuda_stream)

        call()
        torch.cuda.synchronize()
        return call, out, [o.clone() for o in out], (x, d, tokens, u, s)

    pairs = [one(vocab, i) for i, vocab in enumerate((151936, 50, 151936, 50))]
    assert side_by_side(*(p[0] for p in pairs), turns=3000) == []
    for _, out, want, _ in pairs:
        assert all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.parametrize("neighbours", [False, True])
def test_rotary_append_into_two_caches(neighbours):
    def one(dim, page, count):
        kv = wd.KvCache(1, 2, 2, dim, 8, 1, 8 * page, page_tokens=page)
        rope = wd.Rope(dim, neighbours=neighbours)
        gen = torch.Generator("cuda").manual_seed(dim)
        k, v, q = (torch.randn(count, 2, dim, generator=gen, device="cuda") for _ in range(3))
        out, s = torch.zeros_like(q), torch.cuda.Stream()
        torch.cuda.synchronize()
        kv.begin([0], [count], s.cuda_stream)

        rows = wd.RopeRows(None, None, None, k.data_ptr(), v.data_ptr(), q.data_ptr(), out.data_ptr(), 0, 0, 0, 0, 1e-6, wd.TYPE_F32)
        args, f = (kv.h, 0, rope.h, ctypes.byref(rows), s.cuda_stream), wd.lib().wd_kv_append_rope

        def call():                     # (by the C entry: less of the turn is the interpreter's, which one thread has at a time)
            if f(*args):
                raise RuntimeError(wd.lib().wd_last_error().decode())

        def read():
            got = [torch.zeros(count, 2, dim, device="cuda") for _ in range(2)]
            torch.cuda.synchronize()
            kv.read(0, [0], [0], [count], *(g.data_ptr() for g in got), stream=s.cuda_stream)
            torch.cuda.synchronize()
            return [out.cpu().numpy()] + [g.cpu().numpy() for g in got]

        call()
        return call, read, read(), (k, v, q, kv, rope, rows)

    pairs = [one(256, 128, 64), one(64, 64, 40), one(256, 128, 64), one(64, 64, 40)]
    assert side_by_side(*(p[0] for p in pairs), turns=15000) == []
    for _, read, want, _ in pairs:
        assert all(np.array_equal(x, y) for x, y in zip(read(), want))
