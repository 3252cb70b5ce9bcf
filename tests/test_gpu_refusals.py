"""What a run that a kernel cannot take says: the reason, and no other kernel's."""
import numpy as np
import pytest

from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.runtime import EmxError, Session
from gpu_util import plan_for, require_gpu

pytestmark = pytest.mark.gpu

EMX_ERR_UNSUPPORTED = 5


def buffers(plan, x):
    import torch
    dev = [torch.from_numpy(x[n]).cuda() for n in plan.input_names]
    dt = {"f16": torch.float16, "f32": torch.float32, "u8": torch.uint8}
    outs = [torch.zeros(s, dtype=dt[t], device="cuda") for s, t in zip(plan.output_shapes, plan.output_dtypes)]
    return dev, outs


def refused(sess, ins, outs):
    with pytest.raises(EmxError) as e:
        sess.run_ptrs(ins, outs)
    assert e.value.status == EMX_ERR_UNSUPPORTED
    return str(e.value)


def test_a_kernel_that_refuses_a_size_says_nothing_of_buffers():
    require_gpu()
    wl = W.qlinear_matmul_u8(m=8 * 65535 + 1, k=3, n=2)
    plan = plan_for(wl)
    dev, outs = buffers(plan, {"A": np.zeros((8 * 65535 + 1, 3), np.uint8)})
    msg = refused(Session(plan), [t.data_ptr() for t in dev], [t.data_ptr() for t in outs])
    assert "qlinear_matmul" in msg and "size" in msg and "buffer" not in msg and "16" not in msg


@pytest.mark.parametrize("make,mode,which,off", [
    (lambda: W.decoder_attention(), "flash", "Q", 2),
    (lambda: W.decoder_attention(count=True), "flash", "count", 4),
    (lambda: W.decoder_attention(mask="f32"), "flash", "mask", 2),
    (lambda: W.decoder_attention(mask="f16"), "flash", "mask", 1),
    (lambda: W.norm_rope(), "exact", "K", 1),
    (lambda: W.norm_rope(dtype="f32"), "exact", "Q", 2),
    (lambda: W.norm_rope(), "exact", "pos", 4),
])
def test_a_kernel_that_needs_a_boundary_names_it(make, mode, which, off):
    require_gpu()
    import torch
    wl = make()
    plan = plan_for(wl, attention_mode=mode)
    x = wl.make_inputs(1)
    dev, outs = buffers(plan, x)
    i = plan.input_names.index(which)
    wide = torch.zeros(dev[i].numel() * dev[i].element_size() + 16, dtype=torch.uint8, device="cuda")
    ptrs = [t.data_ptr() for t in dev]
    sess = Session(plan)
    want = sess.run(x)
    msg = refused(sess, ptrs[:i] + [wide.data_ptr() + off] + ptrs[i + 1:], [t.data_ptr() for t in outs])
    assert "boundary" in msg and "too large" not in msg
    sess.run_ptrs(ptrs, [t.data_ptr() for t in outs])
    sess.sync()
    for n, t in zip(plan.output_names, outs):
        assert np.array_equal(t.cpu().numpy(), want[n])


def test_a_plan_without_room_for_mask_references_is_refused_when_loaded():
    """As written before partial results carried them: split keys under an additive mask."""
    require_gpu()
    import dataclasses
    import struct

    from emx_onnx_cgen_b200 import kernel_ids as K
    for mask, ok in (("f16", False), ("f32", False), ("bool", True)):
        wl = W.decoder_attention(batch=1, q_heads=2, kv_heads=2, q_seq=3, kv_seq=4000, mask=mask)
        plan = plan_for(wl, attention_mode="flash")
        op = plan.ops[-1]
        assert op.ip[K.AF_SPLITS_K] > 1
        blob = bytearray(plan.plan_bytes)
        at = len(blob) - 440 + 8 + 12 * 4 + 8 * K.AF_PART_WIDTH  # the last op's integers
        assert struct.unpack_from("<q", blob, at)[0] == op.ip[K.AF_PART_WIDTH]
        struct.pack_into("<q", blob, at, 0)
        old = dataclasses.replace(plan, plan_bytes=bytes(blob))
        if ok:
            Session(old).run(wl.make_inputs(1))
            continue
        with pytest.raises(EmxError, match="plan it again") as e:
            Session(old)
        assert e.value.status == EMX_ERR_UNSUPPORTED
