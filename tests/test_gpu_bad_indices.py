"""Valid key counts and positions out of range, whichever pass reads them: the
sequence they belong to is handled as documented (the count clamped, the rows
NaN), every other result of the run and of the runs behind it is as without
them, and the next sync reports the input."""
import numpy as np
import pytest

from emx_onnx_cgen_b200 import kernel_ids as K
from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.runtime import EmxError, Session
from gpu_util import plan_for, require_gpu

pytestmark = pytest.mark.gpu

EMX_ERR_INVALID_ARGUMENT = 1


@pytest.mark.parametrize("kw,own", [
    (dict(batch=6, q_heads=4, kv_heads=2, q_seq=2, kv_seq=700), K.AF_PASS_ROWS8),
    (dict(batch=6, q_heads=4, kv_heads=2, q_seq=8, kv_seq=700, head_dim=128), K.AF_PASS_ROWS16),
    (dict(batch=6, q_heads=4, kv_heads=2, q_seq=50, kv_seq=1500), K.AF_PASS_TILES),
    (dict(batch=20, q_heads=8, kv_heads=8, q_seq=300, kv_seq=1500), K.AF_PASS_WIDE),   # several items a CTA
    (dict(batch=20, q_heads=8, kv_heads=4, q_seq=200, kv_seq=1500, head_dim=128), K.AF_PASS_WIDE),
    (dict(batch=1, q_heads=2, kv_heads=2, q_seq=300, kv_seq=4000), K.AF_PASS_WIDE),    # key ranges
])
@pytest.mark.parametrize("graphs", [True, False])
def test_counts_out_of_range_touch_their_own_sequence(kw, own, graphs):
    require_gpu()
    import torch
    wl = W.decoder_attention(count=True, **kw)
    plan = plan_for(wl, attention_mode="flash")
    assert plan.ops[0].ip[K.AF_PASS_OWN] == own
    x = wl.make_inputs(41)
    bad = x["count"].copy()
    bad[0] = -3
    bad[-1] = kw["kv_seq"] + 1 if kw["batch"] > 1 else 2 ** 40
    clamped = np.clip(bad, 0, kw["kv_seq"])
    sess = Session(plan)
    sess.set_graphs(graphs)
    want = {n: sess.run(dict(x, count=c))["Y"] for n, c in (("clamped", clamped), ("good", x["count"]))}
    dev = {n: torch.from_numpy(v).cuda() for n, v in x.items()}
    counts = {"clamped": torch.from_numpy(bad).cuda(), "good": dev["count"]}
    runs = [(n, torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda"))
            for n in ("clamped", "good", "clamped", "good", "good")]
    torch.cuda.synchronize()
    for n, y in runs:  # no sync between them
        sess.run_ptrs([(counts[n] if name == "count" else dev[name]).data_ptr() for name in plan.input_names], [y.data_ptr()])
    with pytest.raises(EmxError, match="out of range") as e:
        sess.sync()
    assert e.value.status == EMX_ERR_INVALID_ARGUMENT
    for n, y in runs:
        assert np.array_equal(y.cpu().numpy().view(np.uint16), want[n].view(np.uint16)), n
    sess.sync()  # reported once


def test_positions_out_of_range_leave_the_attention_behind_them_alone():
    """A decoder layer's run: the rotation's bad rows are NaN, the other sequences' results are theirs."""
    require_gpu()
    wl = W.decoder_layer(batch=5, tokens=70, head_dim=128, q_heads=8, prefix=500, frames=700)
    x = wl.make_inputs(42)
    plan = plan_for(wl, attention_mode="flash")
    sess = Session(plan)
    want = sess.run(x)["Y"]
    import torch
    x["pos"][3, 5] = 10 ** 9
    dev = [torch.from_numpy(x[n]).cuda() for n in plan.input_names]
    y = torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    sess.run_ptrs([t.data_ptr() for t in dev], [y.data_ptr()])
    with pytest.raises(EmxError, match="out of range"):
        sess.sync()
    got = y.cpu().numpy()
    others = [0, 1, 2, 4]
    assert np.array_equal(got[others].view(np.uint16), want[others].view(np.uint16))
    assert np.isnan(got[3, 5:]).all() and np.isfinite(got[3, :5]).all()  # tokens behind it see its key


def test_a_report_leaves_no_trace_in_the_next_run():
    """Reports and good runs in turn, back to back on the plan's own stream and on another one: a report is neither
    repeated nor lost, and no good run gives up on its account."""
    require_gpu()
    import torch
    wl = W.decoder_attention(batch=4, q_heads=8, kv_heads=8, q_seq=200, kv_seq=900, count=True)
    plan = plan_for(wl, attention_mode="flash")
    x = wl.make_inputs(44)
    sess = Session(plan)
    want = sess.run(x)["Y"]
    dev = {n: torch.from_numpy(v).cuda() for n, v in x.items()}
    bad = torch.full((4,), 901, dtype=torch.int64, device="cuda")
    y = torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    ptrs = {k: [(c if n == "count" else dev[n]).data_ptr() for n in plan.input_names] for k, c in (("bad", bad), ("good", dev["count"]))}
    for i in range(40):
        stream = (0, torch.cuda.Stream().cuda_stream)[i % 2]
        sess.run_ptrs(ptrs["bad"], [y.data_ptr()], stream=stream)
        with pytest.raises(EmxError, match="out of range"):
            sess.sync()
        sess.run_ptrs(ptrs["good"], [y.data_ptr()], stream=stream)
        sess.sync()
        assert np.array_equal(y.cpu().numpy().view(np.uint16), want.view(np.uint16))
