"""RMSNormalization and RotaryEmbedding on the B200 kernels against their
float64 definitions (decoder_reference.py), within the bound that one final
rounding and the fp32 steps before it give: both types, the layouts a planner
fuses, pairings, partial rotation, head sizes off the 16-byte pieces, one
token, strided heads, and the error for a position out of the tables."""
import numpy as np
import pytest

from decoder_reference import HALF, TINY, check, norm_rope, rms_norm
from emx_onnx_cgen_b200 import kernel_ids as K
from emx_onnx_cgen_b200 import lowering
from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.plan import B200PlanEmitter
from emx_onnx_cgen_b200.runtime import EmxError, Session
from emx_onnx_cgen_b200.spec import GraphSpec, NodeSpec, TensorSpec
from gpu_util import plan_for, require_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [
    dict(),
    dict(batch=32, seq=1, q_heads=32, kv_heads=8, head_dim=128),
    dict(batch=1, seq=1, q_heads=1, kv_heads=1, head_dim=8),
    dict(dtype="f32", head_dim=80, rotary_dim=32, interleaved=True, q_heads=12, kv_heads=4, seq=33),
    dict(dtype="f32", head_dim=256, q_heads=3, kv_heads=1),
    dict(dtype="f16", head_dim=512, q_heads=2, kv_heads=2, interleaved=True),
    dict(dtype="f16", head_dim=520, q_heads=2, kv_heads=1),           # longer than a warp's pieces
    dict(dtype="f16", head_dim=80, rotary_dim=40),                    # halves of 20: off the pieces
    dict(dtype="f32", head_dim=6, rotary_dim=2, q_heads=3, kv_heads=3, interleaved=True),
    dict(dtype="f16", head_dim=96, rotary_dim=48, seq=37),            # an odd number of pieces behind the rotation
    dict(dtype="f16", head_dim=72, rotary_dim=16, interleaved=True),
    dict(layout="heads", seq=19), dict(layout="flat", seq=19), dict(layout="flat", seq=7, dtype="f32", head_dim=32),
    dict(norm=False), dict(norm=False, layout="heads", interleaved=True, dtype="f32"),
    dict(positions="rows", seq=21), dict(positions="rows", seq=5, head_dim=24, rotary_dim=8, dtype="f32"),
    dict(batch=7, seq=300, q_heads=32, kv_heads=8, head_dim=128),     # four rows per lane group
    dict(batch=5, seq=511, q_heads=12, kv_heads=5, head_dim=128, interleaved=True, dtype="f32"),
    # lane groups that go around (norm_rope.cu): head counts off the four rows of a group, token counts off the grid
    dict(batch=3, seq=1401, q_heads=30, kv_heads=7, head_dim=128),
    dict(batch=3, seq=1401, q_heads=30, kv_heads=7, head_dim=128, rotary_dim=96, interleaved=True),
    dict(batch=1, seq=3001, q_heads=21, kv_heads=5, head_dim=128, rotary_dim=64, interleaved=True, dtype="f32"),
    dict(batch=2, seq=2003, q_heads=33, kv_heads=1, head_dim=72, rotary_dim=48, positions="rows", layout="heads"),
    dict(batch=1, seq=5003, q_heads=31, kv_heads=30, head_dim=64, norm=False, dtype="f32", layout="flat"),
])
def test_definition(kw):
    require_gpu()
    wl = W.norm_rope(**kw)
    plan = plan_for(wl)
    assert [o.kernel for o in plan.ops] == [K.K_NORM_ROPE]
    x = wl.make_inputs(3)
    got = Session(plan).run(x)
    for name, (y, tol) in norm_rope(wl, x).items():
        check(got[name], y, tol, f"{kw} {name}")


def test_values_outside_the_rotation_pass_through():
    """Infinities behind the rotated elements stay, and rows apart stay apart."""
    require_gpu()
    for inter in (False, True):
        wl = W.norm_rope(norm=False, head_dim=64, rotary_dim=32, interleaved=inter)
        x = wl.make_inputs(1)
        x["Q"][0, 3, 2, 40] = np.inf
        x["Q"][1, 2, 1, 5] = np.nan
        got = Session(plan_for(wl)).run(x)["YQ"]
        assert got[0, 2, 3, 40] == np.inf
        nan = np.zeros(got.shape, bool)
        nan[1, 1, 2, [5, 4] if inter else [5, 21]] = True
        assert np.array_equal(np.isnan(got), nan)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("shape,axis", [((5, 1), -1), ((3, 7), -1), ((4, 1000), 1), ((2, 3, 1024), -1), ((3, 1025), -1),
                                        ((2, 8192), -1), ((1, 2, 3000), 1), ((9, 4104), -1)])
def test_rms_norm(shape, axis, dtype):
    require_gpu()
    npt = np.float16 if dtype == "f16" else np.float32
    r = np.random.default_rng(2)
    axes = len(shape) - axis % len(shape)
    scale = r.uniform(0.5, 1.5, shape[-axes:]).astype(npt)
    g = GraphSpec("rms", [TensorSpec("X", dtype, shape)], [TensorSpec("Y", dtype, shape)],
                  [NodeSpec("RMSNormalization", "n", ("X", "s"), ("Y",), {"axis": axis, "epsilon": 1e-5})], {"s": scale},
                  opset_imports=(("", 23),))
    plan = B200PlanEmitter().emit_plan(lowering.lower(g))
    x = r.standard_normal(shape).astype(npt)
    want = rms_norm(x, scale, 1e-5, axes)
    check(Session(plan).run({"X": x})["Y"], want, HALF[dtype] * np.abs(want) + TINY[dtype] + 40 * 2.0 ** -24 * np.abs(want),
          f"{shape} {axis}")


def test_position_out_of_the_tables_is_reported():
    require_gpu()
    for head_dim in (64, 20):  # both kernels
        wl = W.norm_rope(head_dim=head_dim)
        x = wl.make_inputs(0)
        sess = Session(plan_for(wl))
        good = sess.run(x)
        for bad in (-1, wl.graph.initializers["cos"].shape[0], 2 ** 40):
            y = {k: v.copy() for k, v in x.items()}
            y["pos"][1, 3] = bad
            with pytest.raises(EmxError, match="out of range"):
                sess.run(y)
        again = sess.run(x)  # the session stays usable
        assert all(np.array_equal(good[n], again[n]) for n in good)


def test_position_out_of_the_tables_among_many_tokens():
    """The rows of a bad position are NaN, every other row is as without it."""
    require_gpu()
    import torch
    wl = W.norm_rope(batch=3, seq=1401, q_heads=30, kv_heads=7, head_dim=128)
    x = wl.make_inputs(2)
    plan = plan_for(wl)
    sess = Session(plan)
    want = sess.run(x)
    x["pos"][2, 1400] = -5
    x["pos"][0, 0] = wl.graph.initializers["cos"].shape[0]
    dev = [torch.from_numpy(x[n]).cuda() for n in plan.input_names]
    outs = [torch.zeros(s, dtype=torch.float16, device="cuda") for s in plan.output_shapes]
    sess.run_ptrs([t.data_ptr() for t in dev], [o.data_ptr() for o in outs], stream=1)
    with pytest.raises(EmxError, match="out of range"):
        sess.sync()
    for n, o in zip(plan.output_names, outs):
        got, ref = o.cpu().numpy(), want[n].copy()
        assert np.isnan(got[2, :, 1400]).all() and np.isnan(got[0, :, 0]).all()
        got[2, :, 1400], got[0, :, 0] = ref[2, :, 1400], ref[0, :, 0]
        assert np.array_equal(got, ref)


def test_batch_slices():
    require_gpu()
    wl = W.norm_rope(batch=4, seq=6)
    x = wl.make_inputs(5)
    plan = plan_for(wl)
    assert plan.batch == 4
    sess = Session(plan)
    whole = sess.run(x)
    part = sess.run(x, 1, 2)
    for n in whole:
        assert np.array_equal(part[n][1:3], whole[n][1:3]) and not part[n][0].any() and not part[n][3].any()


def test_misaligned_device_buffers():
    """Tensors that start off 16 bytes take the element-wise kernel."""
    require_gpu()
    import torch
    wl = W.norm_rope(batch=2, seq=5)
    x = wl.make_inputs(4)
    plan = plan_for(wl)
    sess = Session(plan)
    want = norm_rope(wl, x)
    bufs = {}
    for n in plan.input_names:
        t = torch.from_numpy(x[n]).cuda()
        pad = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        pad[1:] = t.reshape(-1)
        bufs[n] = pad
    outs = [torch.full((int(np.prod(s)) + 2,), 7.0, dtype=torch.float16, device="cuda") for s in plan.output_shapes]
    sess.run_ptrs([bufs[n].data_ptr() + bufs[n].element_size() for n in plan.input_names],
                  [o.data_ptr() + 2 for o in outs], stream=torch.cuda.current_stream().cuda_stream or 1)
    sess.sync()
    for n, s, o in zip(plan.output_names, plan.output_shapes, outs):
        o = o.cpu().numpy()
        assert o[0] == 7 and o[-1] == 7
        check(o[1:-1].reshape(s), *want[n], n)


def test_pointers_are_taken_anew_each_call():
    """Too few are refused, whatever the call before passed; extra ones are ignored."""
    require_gpu()
    import torch
    wl = W.norm_rope(batch=2, seq=5)
    plan = plan_for(wl)
    sess = Session(plan)
    x = [wl.make_inputs(s) for s in (1, 2)]
    dev = [[torch.from_numpy(v[n]).cuda() for n in plan.input_names] for v in x]
    outs = [[torch.zeros(s, dtype=torch.float16, device="cuda") for s in plan.output_shapes] for _ in x]
    ptrs = lambda ts: [t.data_ptr() for t in ts]
    for d, o in zip(dev, outs):
        sess.run_ptrs(ptrs(d), ptrs(o) + [1], stream=1)
        for i, j in ((1, 0), (0, 1)):
            with pytest.raises(ValueError, match="pointers"):
                sess.run_ptrs(ptrs(d)[i:], tuple(ptrs(o))[j:])
    sess.sync()
    for v, o in zip(x, outs):
        for n, (y, tol) in norm_rope(wl, v).items():
            check(o[plan.output_names.index(n)].cpu().numpy(), y, tol, n)
