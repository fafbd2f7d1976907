"""Two engines or decoders of one process, a large one and then a small one: what a kernel may have of shared memory does not go by the one that was made last."""
import numpy as np
import pytest

import oracle_lib as ol
import warpdecode_b200 as wd
from warpdecode_b200 import synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("one_launch", [False, True])            # operations by a graph of kernels, or a token by one kernel
def test_decoders(monkeypatch, one_launch):
    monkeypatch.setenv("WD_DENSE_TOKEN_KERNEL", str(int(one_launch)))

    def decoder(hidden, heads, kv, ffn, ctx):
        d = wd.DenseDecoder(hidden, heads, kv, 64, ffn, 96, 1, ctx, 1e-5, 500000.0)
        d.synth(11, 0.05)
        return d

    tokens = np.random.Generator(np.random.PCG64(3)).integers(0, 96, 20).astype(np.int32)
    large = decoder(2048, 32, 8, 8192, 4000)
    assert (large.kernel_name() == "dense_token_kernel") == one_launch
    want, _ = large.decode(tokens, 5)
    small = decoder(512, 8, 2, 1024, 64)
    of_small, _ = small.decode(tokens, 5)
    got, _ = large.decode(tokens, 5)
    assert np.array_equal(got, want)
    small.close()
    large.close()
    again = decoder(512, 8, 2, 1024, 64)
    got, _ = again.decode(tokens, 5)
    assert np.array_equal(got, of_small)
    again.close()


@pytest.mark.parametrize("tokens", [1, 4])
def test_plain_engines(tokens):
    engines = []
    for seed, hidden, ffn in ((1, 2560, 640), (2, 512, 192)):
        m = synth.make_moe_block(seed, hidden, ffn, 16, 4, 128, expert_type=wd.TYPE_IQ3_S, down_type=wd.TYPE_IQ4_NL, router_f32=True)
        e = wd.Engine(hidden, ffn, 16, 4, 128, 1, expert_type=wd.TYPE_IQ3_S, down_type=wd.TYPE_IQ4_NL, router_f32=True, max_tokens=4)
        assert e.kernel_name() == "plain_gate_up_kernel"
        e.load_block(0, m)
        engines.append((e, m, np.random.Generator(np.random.PCG64(seed)).standard_normal((tokens, hidden)).astype(np.float32)))
    oracle = ol.Oracle()
    for e, m, x in engines:
        out = e.forward_host(0, x[0] if tokens == 1 else x).reshape(tokens, -1)
        for i in range(tokens):
            assert np.array_equal(ol.fbits(out[i]), ol.fbits(oracle.moe_block(m, x[i])["out"]))
    for e, _, _ in engines:
        e.close()
