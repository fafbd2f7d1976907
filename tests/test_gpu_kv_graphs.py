"""Replays of captured calls of the 8-bit cache around the end of a step."""
import numpy as np
import pytest
import torch

from test_gpu_kv_cache import Pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("chunk", [3, 4000])            # the kernel for few rows; the one for prompts
@pytest.mark.parametrize("end", ["truncate", "free", "keep", "nothing"])
def test_a_replay_behind_the_end_of_a_step_does_nothing(chunk, end):
    p = Pair(8, 2, 64, 16, 0, "f32", n_pages=900, layers=1)
    p.step([0, 1], [21, 9])
    k, v, q = (torch.zeros(chunk, h, 64, device="cuda") for h in (2, 2, 8))
    out = torch.full_like(q, 3.0)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    p.kv.begin([0], [chunk], s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        p.kv.append(0, k.data_ptr(), v.data_ptr(), stream=s.cuda_stream)
        p.kv.attend(0, q.data_ptr(), out.data_ptr(), stream=s.cuda_stream)
    rows = [p.rand(chunk, h, 64) for h in (2, 2, 8)]

    def replay(factor):
        with torch.cuda.stream(s):
            for to, x in zip((k, v, q), rows):
                to.copy_(x * factor)
            g.replay()
        s.synchronize()

    replay(1.0)
    p.ref[0].append(0, rows[0].double().numpy(), rows[1].double().numpy())
    want = p.ref[0].attend(0, rows[2].double().numpy(), 0.125, 0)
    assert np.linalg.norm(out.double().cpu().numpy() - want) <= 2.0 ** -16 * np.linalg.norm(want)
    if end == "truncate":
        p.kv.truncate(0, 23, s.cuda_stream)             # two of the step's tokens stay, in the page that held some before
        p.ref[0].truncate(0, 23)
    elif end == "free":
        p.kv.free([1], s.cuda_stream)
        p.ref[0].truncate(1, 0)
    elif end == "keep":
        p.kv.keep(0, 21, [0, 2], s.cuda_stream)
        p.ref[0].keep(0, 21, [0, 2])
    else:
        p.kv.begin([], [], s.cuda_stream)
    out.fill_(5.0)
    torch.cuda.synchronize()
    replay(100.0)                                       # would make the scales of the pages grow
    assert (out == 5.0).all()
    p.check_numbers([0, 1])
    p.kv.begin([1], [1], s.cuda_stream)                 # and the steps that follow are served
    replay(1.0)
    p.ref[0].append(1, rows[0][:1].double().numpy(), rows[1][:1].double().numpy())
    want = p.ref[0].attend(1, rows[2][:1].double().numpy(), 0.125, 0)
    assert np.linalg.norm(out[:1].double().cpu().numpy() - want) <= 2.0 ** -16 * np.linalg.norm(want)
    p.check_numbers([0, 1])


def test_a_replayed_read_finds_the_pages_that_a_sequence_has_then():
    p = Pair(4, 2, 64, 16, 0, "f32", layers=2)
    p.step([0, 1], [40, 40])
    k, v = (torch.zeros(2, 40, 2, 64, device="cuda") for _ in range(2))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        p.kv.read(-1, [1], [0], [40], k.data_ptr(), v.data_ptr(), stream=s.cuda_stream)

    def same(seq):
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        for layer in range(2):
            assert np.array_equal(np.stack([k[layer].cpu().numpy(), v[layer].cpu().numpy()]), p.ref[layer].numbers(seq)[:, :40].astype(np.float32))

    same(1)
    p.kv.free([1], s.cuda_stream)
    p.kv.fork(0, [1], s.cuda_stream)            # nothing else is called before the replay
    same(0)
    for r in p.ref:
        r.truncate(1, 0)
        r.fork(0, 1)
    torch.cuda.synchronize()
    p.step([1, 0], [5, 30])
    same(1)
    p.kv.truncate(1, 41, s.cuda_stream)
    same(1)
