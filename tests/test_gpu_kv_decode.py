"""A speculative step put together out of the library's operators: embedding rows, products, the 8-bit cache, the MoE block, the head, and the scores
that judge the draft; then the accepted tokens are kept."""
import numpy as np
import pytest
import torch

import kv_oracle
import warpdecode_b200 as wd
from test_gpu_scores import check, expected
from warpdecode_b200 import synth

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV, DIM, VOCAB, PAGE = 512, 8, 2, 64, 2048, 16


def q8(rows, cols, seed):
    w = torch.empty(rows * cols // 32 * 34, dtype=torch.uint8, device="cuda")
    wd.synth_tensor_device(wd.TYPE_Q8_0, rows, cols, 1.0 if rows == VOCAB else 0.05, seed, 7, w.data_ptr())
    return w


def q4(rows, cols, seed):
    """Random Q4_0 blocks with scales of a sensible size."""
    g = np.random.default_rng(seed)
    raw = g.integers(0, 256, (rows * cols // 32, 18), dtype=np.uint8)
    raw[:, :2] = (g.random(raw.shape[0]) * 0.01 + 0.005).astype(np.float16).view(np.uint8).reshape(-1, 2)
    return wd.DenseQ4_0(rows, cols, raw.reshape(-1))


def test_a_speculative_step():
    block = synth.make_moe_block(1, HIDDEN, 256, 32, 6, 256)
    moe = wd.Engine(HIDDEN, 256, 32, 6, 256, 1, max_tokens=4)
    moe.load_block(0, block)
    table, head = q8(VOCAB, HIDDEN, 3), q8(VOCAB, HIDDEN, 4)
    head = wd.HeadQ8_0(VOCAB, HIDDEN, ggml_dev_ptr=head.data_ptr())
    wqkv, wo = q4((HEADS + 2 * KV) * DIM, HIDDEN, 5), q4(HIDDEN, HEADS * DIM, 6)
    kv = wd.KvCache(1, HEADS, KV, DIM, 40, 3, 200, page_tokens=PAGE)
    ref = kv_oracle.Cache(KV, DIM, PAGE, 0, 3)
    s = torch.cuda.Stream()
    sp = s.cuda_stream
    width = (HEADS + 2 * KV) * DIM

    def step(seq, tokens):
        """Logits of the tokens' rows; the plain cache takes the same keys and values, and the attention's output is compared."""
        n = len(tokens)
        ids = torch.tensor(tokens, dtype=torch.int32, device="cuda")
        x, qkv, ctx = torch.zeros(n, HIDDEN, device="cuda"), torch.zeros(n, width, device="cuda"), torch.zeros(n, HEADS * DIM, device="cuda")
        o, y, logits, token = torch.zeros(n, HIDDEN, device="cuda"), torch.zeros(n, HIDDEN, device="cuda"), torch.zeros(n, VOCAB, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        kv.begin([seq], [n], sp)
        with torch.cuda.stream(s):
            for i in range(n):
                wd.embed_q8_0(table.data_ptr(), VOCAB, HIDDEN, ids.data_ptr() + 4 * i, x[i].data_ptr(), sp)
                wqkv.matvec(x[i].data_ptr(), qkv[i].data_ptr(), sp)
            base = qkv.data_ptr()
            kv.append(0, base + 4 * HEADS * DIM, base + 4 * (HEADS + KV) * DIM, k_stride=width, v_stride=width, stream=sp)
            kv.attend(0, base, ctx.data_ptr(), q_stride=width, stream=sp)
            for i in range(n):
                wo.matvec(ctx[i].data_ptr(), o[i].data_ptr(), sp)
            x += 0.1 * o
            for i in range(0, n, 4):
                moe.forward_device(0, x[i].data_ptr(), y[i].data_ptr(), sp, min(4, n - i))
            x += y
            x /= x.std(dim=1, keepdim=True)
            for i in range(n):
                head.argmax(x[i].data_ptr(), token.data_ptr() + 4 * i, logits[i].data_ptr(), None, sp)
        s.synchronize()
        rows = qkv.double().cpu().numpy().reshape(n, -1, DIM)
        ref.append(seq, rows[:, HEADS:HEADS + KV], rows[:, HEADS + KV:])
        want = ref.attend(seq, rows[:, :HEADS], DIM ** -0.5, 0)
        got = ctx.double().cpu().numpy().reshape(n, HEADS, DIM)
        assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)
        return logits, token

    def same(seq):
        n = kv.length(seq)
        k, v = torch.zeros(n, KV, DIM, device="cuda"), torch.zeros(n, KV, DIM, device="cuda")
        kv.read(0, [seq], [0], [n], k.data_ptr(), v.data_ptr())
        torch.cuda.synchronize()
        assert n == ref.length[seq]
        assert np.array_equal(np.stack([k.cpu().numpy(), v.cpu().numpy()]), ref.numbers(seq).astype(np.float32))

    step(0, list(range(5, 5 + 37)))                                     # the prompt
    kv.fork(0, [1, 2])                                                  # two drafts behind it
    ref.fork(0, 1)
    ref.fork(0, 2)
    drafts = {1: [100, 7, 9, 1500], 2: [100, 300, 2047]}
    for seq, tokens in drafts.items():
        logits, best = step(seq, tokens)
        n = len(tokens)
        judged = torch.tensor(tokens[1:] + [0], dtype=torch.int32, device="cuda")
        lp, h = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        ids, top = torch.zeros(n, 5, dtype=torch.int32, device="cuda"), torch.zeros(n, 5, device="cuda")
        wd.token_logprobs(logits.data_ptr(), n, VOCAB, judged.data_ptr(), lp.data_ptr(), h.data_ptr(), 5, ids.data_ptr(), top.data_ptr(), stream=sp)
        s.synchronize()
        got = [x.cpu().double().numpy() if x.dtype != torch.int32 else x.cpu().numpy() for x in (lp, h, ids, top)]
        check(got, expected(logits, judged, 5), 5, 60.0)
        assert np.array_equal(got[2][:, 0], best.cpu().numpy())         # the likeliest token is the head's
    kv.keep(1, 37, [0, 2, 3], sp)                                       # a path of the first draft is accepted
    ref.keep(1, 37, [0, 2, 3])
    kv.free([2], sp)
    ref.truncate(2, 0)
    same(1)
    same(0)
    kv.free([0], sp)
    ref.truncate(0, 0)
    step(1, [11])
    same(1)
    assert kv.free_pages() == 40 - len(kv.pages(1)) and kv.status() == 0 and moe.device_status() == 0
