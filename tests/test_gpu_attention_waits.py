"""The tile passes' bounded waits: with the failure-detection hook that keeps all
but a thread block's first tile of keys from being loaded and a 20 ms budget,
the waits run out, the kernels let the copies and products under way finish
and return; the run reports it, and the session then computes as before.
Nothing faults, traps or hangs: every wait in the kernels is bounded."""
import numpy as np
import pytest

from emx_onnx_cgen_b200 import kernel_ids as K
from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.runtime import FAULT_DROP_KEY_TILES, EmxError, Session
from gpu_util import plan_for, require_gpu

pytestmark = pytest.mark.gpu

EMX_ERR_DEVICE_TIMEOUT = 6


@pytest.mark.parametrize("kw,own", [
    (dict(batch=4, q_heads=8, kv_heads=8, q_seq=60, kv_seq=1500), K.AF_PASS_TILES),
    (dict(batch=4, q_heads=8, kv_heads=8, q_seq=60, kv_seq=1500, head_dim=128), K.AF_PASS_TILES),
    (dict(batch=20, q_heads=16, kv_heads=16, q_seq=300, kv_seq=1500), K.AF_PASS_WIDE),
    (dict(batch=20, q_heads=16, kv_heads=4, q_seq=300, kv_seq=1500, head_dim=128), K.AF_PASS_WIDE),
    (dict(batch=20, q_heads=6, kv_heads=2, q_seq=300, kv_seq=1500, head_dim=128), K.AF_PASS_WIDE),  # rows copied one by one
])
def test_waits_that_run_out(kw, own):
    require_gpu()
    wl = W.decoder_attention(count=True, **kw)
    plan = plan_for(wl, attention_mode="flash")
    assert plan.ops[0].ip[K.AF_PASS_OWN] == own
    x = wl.make_inputs(43)
    sess = Session(plan)
    want = sess.run(x)["Y"]
    for _ in range(3):
        sess.set_wait_budget(20_000_000)
        sess.set_fault(FAULT_DROP_KEY_TILES)
        with pytest.raises(EmxError, match="gave up") as e:
            sess.run(x)
        assert e.value.status == EMX_ERR_DEVICE_TIMEOUT
        sess.set_wait_budget(0)
        sess.set_fault(0)
        for _ in range(2):
            assert np.array_equal(sess.run(x)["Y"].view(np.uint16), want.view(np.uint16))
