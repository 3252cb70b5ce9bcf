"""A session's first run, right behind its load."""
import numpy as np
import pytest

from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.runtime import Session
from gpu_util import plan_for, require_gpu

pytestmark = pytest.mark.gpu


def test_first_run_behind_the_load_of_a_large_arena():
    """The load zeroes the arena; an input staged at its far end by the first run stays."""
    require_gpu()
    import torch
    wl = W.decoder_attention(batch=32, q_heads=8, kv_heads=8, q_seq=1, kv_seq=16384, head_dim=128, count=True)
    plan = plan_for(wl, attention_mode="flash")
    assert plan.arena_bytes > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    shapes = dict(zip(plan.input_names, plan.input_shapes))
    dev = {n: torch.randn(shapes[n], generator=g, device="cuda", dtype=torch.float16) for n in "QKV"}
    count = np.full(32, 64, np.int64)  # host memory: staged in the arena, behind the room for K and V
    ptrs = [count.ctypes.data if n == "count" else dev[n].data_ptr() for n in plan.input_names]
    outs = [torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda") for _ in range(9)]
    torch.cuda.synchronize()
    for y in outs:
        sess = Session(plan)
        sess.run_ptrs(ptrs, [y.data_ptr()])
        sess.sync()
        if y is outs[0]:
            sess.run_ptrs(ptrs, [y.data_ptr()])  # a second run of the first session: the reference
            sess.sync()
        sess.close()
    assert all(torch.equal(y, outs[0]) for y in outs) and outs[0].abs().max() > 0.1


def test_first_runs_of_many_small_sessions():
    require_gpu()
    for make, mode in ((lambda: W.decoder_attention(batch=9, q_seq=2, kv_seq=59, mask="f16"), "flash"),
                       (lambda: W.norm_rope(batch=1, seq=1, q_heads=5, kv_heads=4, dtype="f32"), "exact"),
                       (lambda: W.mlp_fp32(), "exact")):
        wl = make()
        plan = plan_for(wl, attention_mode=mode)
        x = wl.make_inputs(3)
        sess = Session(plan)
        sess.run(x)
        want = sess.run(x)
        for _ in range(20):
            got = Session(plan).run(x)
            assert all(np.array_equal(got[n].view(np.uint8), want[n].view(np.uint8)) for n in want)
