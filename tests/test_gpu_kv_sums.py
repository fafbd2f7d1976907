"""Long sums of values of one sign: attention over values that are all alike is that value, whatever the weights."""
import numpy as np
import pytest
import torch

import warpdecode_b200 as wd
from test_gpu_kv_cache import HALF_STEP, TYPES

pytestmark = pytest.mark.gpu
FEW, PROMPT, RUNS = "kv_attend_kernel", "kv_prompt_kernel", "kv_prompt_kernel, kv_prompt_join_kernel"


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 96, 256])
@pytest.mark.parametrize("kernel,seqs,kv_heads,tokens,rows", [(FEW, 64, 4, 20000, 1), (FEW, 1, 4, 300, 1), (PROMPT, 1, 1, 30000, 4800), (RUNS, 1, 1, 131072, 300), (PROMPT, 3, 2, 1800, 1700)])
@pytest.mark.parametrize("spread", [0.0, 0.4])
def test_values_alike(dtype, dim, kernel, seqs, kv_heads, tokens, rows, spread):
    """A tensor core cuts the products that it adds where the sum ends; over random weights that comes to 2^-23 of the sum for 16 tokens and a term at most. The
    kernel for few rows adds 64 tokens at a time (2 4 2^-23), the one for prompts 2,048 (F32; half of 2 128 2^-23, as sums grow evenly) or 8,192 (16 bits, half
    of 512 2^-23). Pieces are added in F32: 30 at most, 2^-24 each; the denominator likewise; the weights' terms are off by 2^-22 (two), or 2^-11 each way, and
    the answer by its own rounding. Weights that are all alike are powers of two here, and their sums exact."""
    t, code = TYPES[dtype]
    heads = kv_heads * (4 if rows > 1 else 1)
    kv = wd.KvCache(1, heads, kv_heads, dim, seqs * (tokens // 128 + 1), seqs, tokens, page_tokens=128)
    g = torch.Generator(device="cuda").manual_seed(dim + tokens)
    ids, before = list(range(seqs)), tokens - rows
    v = torch.ones(tokens, kv_heads, dim, device="cuda", dtype=t)
    k = (torch.randn(tokens, kv_heads, dim, device="cuda", generator=g) * spread * dim ** -0.5).to(t)
    for s in ids:
        kv.begin([s], [before])
        kv.append(0, k.data_ptr(), v.data_ptr(), code)
    kv.begin(ids, [rows] * seqs)
    kn, vn = k[before:].repeat(seqs, 1, 1), v[before:].repeat(seqs, 1, 1)
    kv.append(0, kn.data_ptr(), vn.data_ptr(), code)
    q = torch.randn(seqs * rows, heads, dim, device="cuda", generator=g).to(t)
    out = torch.full_like(q, 3.0)
    kv.attend(0, q.data_ptr(), out.data_ptr(), code, scale=1.0)
    torch.cuda.synchronize()
    assert kv.kernel_name() == kernel and kv.status() == 0
    want = 127.0 * float(np.float32(1.0) / np.float32(127.0))
    steps = 8 if kernel == FEW else 128 if dtype == "f32" else 256
    if dtype != "f32" and kernel == FEW:
        steps = 4
    weights = 2.0 ** -22 if dtype == "f32" else 2.0 ** -11
    assert (out.double() - want).abs().max().item() <= steps * 2.0 ** -23 + 60 * 2.0 ** -24 + weights + HALF_STEP[dtype]
