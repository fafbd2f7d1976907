"""Two engines or decoders of one process, a large one and then a small one: what a kernel may have of shared memory does not go by the one that was made last."""
import numpy as np
import pytest

import oracle_lib as ol
import warpdecode_b200 as wd
from warpdecode_b200 import synth

pytestmark = pytest.mark.gpu


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
