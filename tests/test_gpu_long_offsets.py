"""Keys, values, masks and rows whose element offsets pass 2^31, on the device."""
import numpy as np
import pytest

from emx_onnx_cgen_b200 import kernel_ids as K
from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.runtime import Session
from gpu_util import plan_for, require_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw,own", [
    (dict(batch=2, q_seq=1, kv_seq=8, past=700_000, shared_past=False), K.AF_PASS_ROWS8),
    (dict(batch=2, q_seq=1, kv_seq=700_000, mask="bool"), K.AF_PASS_ROWS8),
    (dict(batch=2, q_seq=40, kv_seq=700_000), K.AF_PASS_TILES),
    (dict(batch=2, q_seq=40, kv_seq=700_000, mask="f16"), K.AF_PASS_TILES),
    (dict(batch=2, q_seq=150, kv_seq=700_000, rank=3), K.AF_PASS_WIDE),
    (dict(batch=2, q_seq=150, kv_seq=140, past=700_000, shared_past=False), K.AF_PASS_WIDE),
])
def test_keys_far_into_a_long_cache(kw, own):
    """One key of each sequence and head has all of the weight: its value comes out, wherever it lies."""
    require_gpu()
    import torch
    h, d = 16, 128
    kw = dict(kw, q_heads=h, kv_heads=h, head_dim=d)
    b, past = kw["batch"], kw.get("past", 0)
    t = past + kw["kv_seq"]
    assert b * h * t * d > 2 ** 31
    wl = W.decoder_attention(**kw)
    plan = plan_for(wl, attention_mode="flash")
    assert plan.ops[-1].ip[K.AF_PASS_OWN] == own
    shapes = dict(zip(plan.input_names, plan.input_shapes))
    g = torch.Generator(device="cuda").manual_seed(3)
    x = {"Q": torch.ones(shapes["Q"], dtype=torch.float16, device="cuda")}
    for n in ("K", "V", "PK", "PV"):
        if n in shapes:
            x[n] = torch.zeros(shapes[n], dtype=torch.float16, device="cuda")
    if "mask" in shapes:
        x["mask"] = torch.ones(shapes["mask"], dtype=torch.bool, device="cuda") if kw["mask"] == "bool" else \
            torch.zeros(shapes["mask"], dtype=torch.float16, device="cuda")

    def at(name, i, j, k):  # key k of sequence i and head j
        m = x[name]
        return m[i, j, k] if m.dim() == 4 else m[i, k].view(h, d)[j]

    want = torch.randn((b, h, d), generator=g, device="cuda", dtype=torch.float16)
    r = np.random.default_rng(4)
    for i in range(b):
        for j in range(h):
            k = t - 1 - 37 * j if i else int(r.integers(0, t))
            if "past" in kw and k < past:
                at("PK", i, j, k).fill_(4.0)
                at("PV", i, j, k).copy_(want[i, j])
            else:
                at("K", i, j, k - past).fill_(4.0)
                at("V", i, j, k - past).copy_(want[i, j])
    y = torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    sess = Session(plan)
    sess.run_ptrs([x[n].data_ptr() for n in plan.input_names], [y.data_ptr()])
    sess.sync()
    if kw.get("rank") == 3:
        y = y.view(b, kw["q_seq"], h, d).transpose(1, 2)
    # the other keys' weights are e^-45 each: together below 1e-13
    assert torch.equal(y, want[:, :, None].expand_as(y))


@pytest.mark.parametrize("layout", ["transpose", "heads"])
def test_norm_and_rotation_of_more_than_2_31_elements(layout):
    require_gpu()
    import torch
    b, t, hq, hkv, d = 3, 150_000, 40, 4, 128
    wl = W.norm_rope(batch=b, seq=t, q_heads=hq, kv_heads=hkv, head_dim=d, layout=layout)
    assert b * t * hq * d > 2 ** 31
    plan = plan_for(wl)
    shapes = dict(zip(plan.input_names, plan.input_shapes))
    g = torch.Generator(device="cuda").manual_seed(5)
    x = {n: torch.randn(shapes[n], generator=g, device="cuda", dtype=torch.float16) for n in "QK"}
    x["pos"] = torch.arange(t, device="cuda").expand(b, t).contiguous() + torch.arange(b, device="cuda")[:, None]
    outs = [torch.zeros(s, dtype=torch.float16, device="cuda") for s in plan.output_shapes]
    torch.cuda.synchronize()
    sess = Session(plan)
    sess.run_ptrs([x[n].data_ptr() for n in plan.input_names], [o.data_ptr() for o in outs])
    sess.sync()
    cos, sin = (torch.from_numpy(wl.graph.initializers[n]).cuda().double() for n in ("cos", "sin"))
    for n, out in zip("QK", outs):
        scale = torch.from_numpy(wl.graph.initializers[n.lower() + "_scale"]).cuda().double()
        for i, s in ((0, 0), (1, 70_000), (2, t - 64)):  # 64 tokens of each sequence, the last ones of the last
            v = x[n][i, s:s + 64].transpose(0, 1) if layout == "transpose" else x[n][i, :, s:s + 64]
            v = v.double()
            v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * scale
            c, sn = cos[x["pos"][i, s:s + 64]], sin[x["pos"][i, s:s + 64]]
            a, e = v[..., :d // 2], v[..., d // 2:]
            y = torch.cat([a * c - e * sn, a * sn + e * c], -1)
            mag = torch.cat([(a * c).abs() + (e * sn).abs(), (a * sn).abs() + (e * c).abs()], -1)
            got = out[i, :, s:s + 64].double()
            assert ((got - y).abs() <= 2.0 ** -11 * y.abs() + 2.0 ** -25 + 40 * 2.0 ** -24 * mag).all(), (n, i)
