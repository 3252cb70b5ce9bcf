"""RMSNormalization, alone and in front of a rotation, on rows whose squares
leave the range of fp32: infinite elements, and finite fp32 rows of any size,
against the float64 definition within the bound of the fp32 steps."""
import numpy as np
import pytest

from decoder_reference import HALF, TINY, check, norm_rope, rms_norm
from emx_onnx_cgen_b200 import lowering
from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.plan import B200PlanEmitter
from emx_onnx_cgen_b200.runtime import Session
from emx_onnx_cgen_b200.spec import GraphSpec, NodeSpec, TensorSpec
from gpu_util import plan_for, require_gpu

pytestmark = pytest.mark.gpu


def _rms(x, scale, eps, axes=1):
    dtype = "f16" if x.dtype == np.float16 else "f32"
    g = GraphSpec("rms", [TensorSpec("X", dtype, x.shape)], [TensorSpec("Y", dtype, x.shape)],
                  [NodeSpec("RMSNormalization", "n", ("X", "s"), ("Y",), {"axis": -axes, "epsilon": eps})], {"s": scale},
                  opset_imports=(("", 23),))
    return Session(B200PlanEmitter().emit_plan(lowering.lower(g))).run({"X": x})["Y"]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [7, 64, 1024, 1025, 8192])
def test_norm_of_a_row_with_an_infinity(n, dtype):
    """x / sqrt(inf): 0 for every finite element, NaN for the infinite one; other rows as without it."""
    require_gpu()
    npt = np.float16 if dtype == "f16" else np.float32
    r = np.random.default_rng(3)
    x, scale = r.standard_normal((5, n)).astype(npt), r.uniform(0.5, 1.5, n).astype(npt)
    want = rms_norm(x, scale, 1e-5)
    want[1], want[3] = 0, 0
    x[1, n // 2], x[3, 0] = np.inf, -np.inf
    got = _rms(x, scale, 1e-5)
    assert np.isnan(got[1, n // 2]) and np.isnan(got[3, 0])
    got[1, n // 2] = got[3, 0] = 0
    check(got, want, HALF[dtype] * np.abs(want) + TINY[dtype] + 40 * 2.0 ** -24 * np.abs(want), f"{n}")


@pytest.mark.parametrize("size,eps", [(1e19, 1e-5), (1e20, 1e-5), (3e38, 1e-5), (1e-21, 0.0), (1e-30, 0.0), (1e-42, 0.0),
                                      (1e-16, 1e-32), (1e-30, 1e-38)])
@pytest.mark.parametrize("n", [6, 96, 1024, 1030, 8192])
def test_norm_of_very_large_and_very_small_rows(n, size, eps):
    """Finite fp32 rows whose squares, or their sum, lie beyond fp32's range have ordinary norms."""
    require_gpu()
    r = np.random.default_rng(4)
    x = (size * r.uniform(-1, 1, (4, n))).astype(np.float32)
    x[2] = r.standard_normal(n)
    scale = r.uniform(0.5, 1.5, n).astype(np.float32)
    want = rms_norm(x, scale, float(np.float32(eps)))
    check(_rms(x, scale, eps), want, TINY["f32"] + 41 * 2.0 ** -24 * np.abs(want), f"{n} {size}")


@pytest.mark.parametrize("kw", [
    dict(), dict(interleaved=True, layout="heads"), dict(head_dim=80, rotary_dim=32, interleaved=True), dict(head_dim=20),
    dict(layout="flat", rotary_dim=32), dict(batch=3, seq=1401, q_heads=30, kv_heads=7, head_dim=128),   # groups go around
])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_norm_and_rotation_of_extreme_rows(kw, dtype):
    """As above through the rotation: an infinite element and its partner are NaN, the rest of that row 0, and
    finite fp32 rows of any size are what the definition says."""
    require_gpu()
    wl = W.norm_rope(**dict(kw, dtype=dtype, eps=1e-6))
    p = wl.params
    x = wl.make_inputs(6)
    token = (lambda t, h: (0, h, t)) if p["layout"] == "heads" else (lambda t, h: (0, t, h))
    if dtype == "f32":
        x["Q"][token(2, 1)] *= np.float32(1e20)
        x["Q"][token(3, 2)] = np.float32(3e38)
        x["K"][token(4, 0)] *= np.float32(1e37)
    want = norm_rope(wl, x)
    rot, half = p["rot"], p["rot"] // 2
    e = 5
    partner = (e ^ 1 if p["interleaved"] else (e + half if e < half else e - half)) if e < rot else e
    x["Q"][token(7, 3)][e] = np.inf
    got = Session(plan_for(wl)).run(x)
    for n in ("YQ", "YK"):
        y, tol = (a.copy() for a in want[n])
        g = got[n]
        if n == "YQ":
            at = (0, 3, 7) if p["layout"] != "flat" else (0, 7, slice(3 * p["head_dim"], 4 * p["head_dim"]))
            row = g[at].copy()
            assert np.isnan(row[[e, partner]]).all()
            row[[e, partner]] = 0
            assert not row.any()
            g[at], y[at] = 0, 0
        check(g, y, tol, f"{kw} {n}")
