"""Attention in flash mode against its float64 definition, within the bound of
its roundings (decoder_reference.py): lengths from one token over every tile
edge, head sizes and layouts, grouped heads, masks of every kind and shape
(rows that see nothing, the type's lowest value, infinities), valid counts
down to zero with NaN in the padding, a past per sequence and one shared by
the batch, split key ranges, batch slices, and a decoder layer's run of
operators together."""
import numpy as np
import pytest

from decoder_reference import attention, check, decoder_attention, rms_norm, rotate
from emx_onnx_cgen_b200 import kernel_ids as K
from emx_onnx_cgen_b200 import lowering
from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.onnx_reader import infer_types
from emx_onnx_cgen_b200.plan import B200PlanEmitter
from emx_onnx_cgen_b200.runtime import EmxError, Session
from emx_onnx_cgen_b200.spec import GraphSpec, NodeSpec, TensorSpec
from gpu_util import plan_for, require_gpu

pytestmark = pytest.mark.gpu


def run(wl, x, kernels=None):
    plan = plan_for(wl, attention_mode="flash")
    assert [o.kernel for o in plan.ops] == (kernels or [K.K_ATTENTION_FLASH])
    return Session(plan).run(x)["Y"]


def verify(kw, x=None, seed=3):
    wl = W.decoder_attention(**kw)
    x = x or wl.make_inputs(seed)
    check(run(wl, x), *decoder_attention(wl, x), str(kw))


@pytest.mark.parametrize("kw", [
    dict(),
    dict(batch=1, q_heads=1, kv_heads=1, q_seq=1, kv_seq=1, head_dim=8),
    dict(batch=2, q_heads=2, kv_heads=2, q_seq=1, kv_seq=63),
    dict(batch=2, q_heads=2, kv_heads=2, q_seq=1, kv_seq=64),
    dict(batch=2, q_heads=2, kv_heads=1, q_seq=129, kv_seq=65, head_dim=128),
    dict(batch=1, q_heads=6, kv_heads=2, q_seq=77, kv_seq=333, head_dim=80),
    dict(batch=1, q_heads=5, kv_heads=5, q_seq=200, kv_seq=130, head_dim=32),
    dict(batch=1, q_heads=8, kv_heads=1, q_seq=40, kv_seq=300, head_dim=96, v_dim=40),
    dict(batch=1, q_heads=2, kv_heads=2, q_seq=40, kv_seq=300, head_dim=64, v_dim=128),
    dict(batch=2, q_heads=3, kv_heads=1, q_seq=70, kv_seq=129, head_dim=72, rank=3),
    dict(batch=2, q_heads=4, kv_heads=4, q_seq=70, kv_seq=129, head_dim=64, v_dim=24, rank=3),
    dict(batch=1, q_heads=2, kv_heads=1, q_seq=300, kv_seq=300, causal=True, head_dim=128),
    dict(batch=2, q_heads=4, kv_heads=2, q_seq=130, kv_seq=70, causal=True),
    dict(batch=1, q_heads=3, kv_heads=1, q_seq=65, kv_seq=400, causal=True, rank=3),
    dict(batch=1, q_heads=2, kv_heads=2, q_seq=1, kv_seq=5000, head_dim=128),    # split along the keys
    dict(batch=3, q_heads=16, kv_heads=2, q_seq=1, kv_seq=4097, head_dim=64),
    dict(batch=1, q_heads=2, kv_heads=2, q_seq=600, kv_seq=600, head_dim=64, scale=0.7),
    dict(batch=1, q_heads=2, kv_heads=2, q_seq=33, kv_seq=100, head_dim=64, scale=-0.2),
    dict(batch=1, q_heads=2, kv_heads=2, q_seq=33, kv_seq=100, head_dim=64, scale=0.0),
])
def test_lengths_heads_layouts(kw):
    require_gpu()
    verify(kw)


@pytest.mark.parametrize("shape", ["seq", "query", "head", "full", "rank2", "rank3", "short", "short_query"])
@pytest.mark.parametrize("mask", ["bool", "f16", "f32"])
@pytest.mark.parametrize("past,tq,d", [(0, 35, 64), (72, 35, 64), (101, 35, 128), (0, 3, 64), (72, 3, 128), (101, 7, 64),
                                       (40, 1, 128)])
def test_masks(mask, shape, past, tq, d):
    require_gpu()
    b, h, tk = 2, 4, 136
    t = past + tk
    ms = {"seq": (b, 1, 1, t), "query": (b, 1, tq, t), "head": (1, h, 1, t), "full": (b, h, tq, t), "rank2": (tq, t),
          "rank3": (h, tq, t), "short": (b, 1, 1, t - 70), "short_query": (1, 1, tq, max(past // 2, 60))}[shape]
    verify(dict(batch=b, q_heads=h, kv_heads=2, q_seq=tq, kv_seq=tk, mask=mask, mask_shape=ms, past=past, head_dim=d,
                shared_past=past != 101))


@pytest.mark.parametrize("mask", ["bool", "f16", "f32"])
@pytest.mark.parametrize("kv_seq,q_seq", [(150, 40), (3000, 2), (3000, 20)])
def test_rows_that_see_nothing(mask, kv_seq, q_seq):
    """Such rows give 0, whether one of a tile, a whole sequence, or only in
    some of the key ranges; so do their neighbours' values stay as they are."""
    require_gpu()
    kw = dict(batch=3, q_heads=2, kv_heads=2, q_seq=q_seq, kv_seq=kv_seq, mask=mask, mask_shape=(3, 1, q_seq, kv_seq))
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(5)
    off = False if mask == "bool" else -np.inf
    x["mask"][0, 0, q_seq // 2] = off
    x["mask"][1] = off
    x["mask"][2, 0, :, :kv_seq - 9] = off
    got = run(wl, x)
    check(got, *decoder_attention(wl, x), str(kw))
    assert not got[1].any() and not got[0, :, q_seq // 2].any()


@pytest.mark.parametrize("heads", [2, 40])
@pytest.mark.parametrize("mask", ["f16", "f32"])
def test_lowest_value_masks(mask, heads):
    """Padding at the type's lowest value.  A row of nothing else is a softmax of
    its scores, with all their digits, at fp16's lowest value; at fp32's the sum
    has none of them left, in 64 bits too, and its keys weigh the same."""
    require_gpu()
    # 20 queries of two heads to a key/value head, or eight of one
    kw = dict(batch=2, q_heads=heads, kv_heads=heads // 2 if heads == 2 else heads, q_seq=20 if heads == 2 else 8, kv_seq=200,
              mask=mask, mask_shape=(2, 1, 20 if heads == 2 else 8, 200))
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(6)
    low = float(np.finfo(np.float16).min)
    x["mask"][:, :, :, 120:] = low
    x["mask"][0, 0, 3, :] = low
    x["mask"][1, 0, 4, :130] = low  # the visible keys come in the last tiles
    x["mask"][1, 0, 4, 130:] = 0
    check(run(wl, x), *decoder_attention(wl, x), str(kw))
    if mask == "f32":  # the fp32 type's own lowest value
        x["mask"][:, :, :, 120:] = np.finfo(np.float32).min
        x["mask"][1, 0, 4, 130:] = 0
        x["mask"][:, 0, 7, :] = np.finfo(np.float32).min
        x["mask"][0, 0, 6, :] = -1e9  # beside this the scores keep enough digits
        x["mask"][0, 0, 5, :] = -1e9
        x["mask"][0, 0, 5, 9:] = np.finfo(np.float32).min
        x["mask"][1, 0, 6, :] = np.finfo(np.float32).max
        x["mask"][1, 0, 5, :] = -3e38
        got, (want, tol) = run(wl, x), decoder_attention(wl, x)
        check(got, want, tol, str(kw))
        assert np.abs(want[0, 0, 7] - x["V"][0, 0].astype(np.float64).mean(0)).max() < 1e-12


@pytest.mark.parametrize("q_seq,d", [(9, 64), (1, 128), (5, 64)])
def test_counts(q_seq, d):
    """Valid counts from none to all; what the padding holds reaches nothing."""
    require_gpu()
    kw = dict(batch=7, q_heads=4, kv_heads=2, q_seq=q_seq, kv_seq=200, count=True, head_dim=d)
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(7)
    x["count"][:] = [200, 0, 1, 63, 64, 65, 130]
    want = decoder_attention(wl, x)
    for b, n in enumerate(x["count"]):
        x["K"][b, :, n:] = np.nan
        x["V"][b, :, n:] = np.nan
    got = run(wl, x)
    assert not got[1].any()
    check(got, *want, str(kw))
    sess = Session(plan_for(wl, attention_mode="flash"))
    for bad in (-1, 201, 2 ** 40):
        y = dict(x, count=x["count"].copy())
        y["count"][3] = bad
        with pytest.raises(EmxError, match="out of range"):
            sess.run(y)
    check(sess.run(x)["Y"], *want, "after the errors")


@pytest.mark.parametrize("q_seq", [50, 2])
def test_padding_behind_a_boolean_mask(q_seq):
    """Keys past the last that any row of a sequence sees are not read; below 17
    rows, 16- or 32-key blocks that no row sees are not."""
    require_gpu()
    kw = dict(batch=3, q_heads=2, kv_heads=2, q_seq=q_seq, kv_seq=300, mask="bool")
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(8)
    ends = [300, 77, 128]
    x["mask"][:] = np.arange(300)[None, None, None, :] < np.array(ends)[:, None, None, None]
    want = decoder_attention(wl, x)
    for b, n in enumerate(ends):
        n = n if q_seq > 16 else -(-n // 32) * 32
        x["K"][b, :, n:] = np.nan
        x["V"][b, :, n:] = np.inf
    check(run(wl, x), *want, str(kw))


@pytest.mark.parametrize("q_seq,d", [(1, 64), (2, 128), (7, 64), (12, 64), (50, 64), (300, 64), (300, 128)])
def test_padding_to_the_key_behind_a_boolean_mask(q_seq, d):
    """What lies behind the last key that any row of a sequence sees reaches
    nothing, from the very next key on, whichever pass runs."""
    require_gpu()
    kw = dict(batch=5, q_heads=2, kv_heads=2, q_seq=q_seq, kv_seq=300, mask="bool", head_dim=d)
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(21)
    ends = [300, 77, 128, 1, 0]
    x["mask"][:] = np.arange(300)[None, None, None, :] < np.array(ends)[:, None, None, None]
    x["mask"][0, ..., :40] = False  # (keys before the first visible one stay finite)
    want = decoder_attention(wl, x)
    for b, n in enumerate(ends):
        x["K"][b, :, n:] = np.nan
        x["V"][b, :, n:] = np.nan
    check(run(wl, x), *want, str(kw))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kw", [
    dict(q_heads=6, kv_heads=2, q_seq=100, kv_seq=400, mask="bool", mask_shape="query"),      # three heads a group
    dict(q_heads=6, kv_heads=2, q_seq=100, kv_seq=400, mask="bool", mask_shape="full", causal=True),
    dict(q_heads=4, kv_heads=2, q_seq=200, kv_seq=130, mask="bool", mask_shape="seq", past=190),
    dict(q_heads=4, kv_heads=2, q_seq=129, kv_seq=260, mask="bool", mask_shape="full", rank=3),
    dict(q_heads=2, kv_heads=2, q_seq=300, kv_seq=700, count=True),
    dict(q_heads=3, kv_heads=1, q_seq=43, kv_seq=257, count=True, rank=3),                     # 129 rows
    dict(q_heads=2, kv_heads=1, q_seq=300, kv_seq=1, causal=True),
    dict(q_heads=2, kv_heads=2, q_seq=257, kv_seq=385, scale=-0.3),
])
def test_two_row_tiles_an_item(kw, d):
    """The 256-row pass: masks of every shape, counts with NaN behind them, groups that do not divide a tile."""
    require_gpu()
    b, t = 3, kw.get("past", 0) + kw["kv_seq"]
    ms = {"seq": (b, 1, 1, t), "query": (b, 1, kw["q_seq"], t), "full": (b, kw["q_heads"], kw["q_seq"], t)}
    kw = dict(kw, batch=b, head_dim=d)
    if "mask_shape" in kw:
        kw["mask_shape"] = ms[kw["mask_shape"]]
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(22)
    if "mask" in kw:
        x["mask"][1, :, -1] = False  # a row (or a sequence) without a key
        x["mask"][2, ..., 140:] = False
    if "count" in x:
        x["count"][:] = [kw["kv_seq"], 0, 129]
    want = decoder_attention(wl, x)
    if "count" in x:
        for i, n in enumerate(x["count"]):
            if kw.get("rank") == 3:
                x["K"][i, n:] = x["V"][i, n:] = np.nan
            else:
                x["K"][i, :, n:] = x["V"][i, :, n:] = np.nan
    check(run(wl, x), *want, str(kw))


@pytest.mark.parametrize("kw", [
    dict(batch=40, q_heads=4, kv_heads=1, q_seq=1, kv_seq=20, past=500, head_dim=128),                  # 160 rows
    dict(batch=33, q_heads=8, kv_heads=2, q_seq=3, kv_seq=20, past=500, head_dim=64),                   # 12 a sequence
    dict(batch=50, q_heads=3, kv_heads=1, q_seq=3, kv_seq=20, past=300, head_dim=128, rank=3),          # 9 a sequence
    dict(batch=33, q_heads=4, kv_heads=1, q_seq=2, kv_seq=20, past=260, head_dim=64, mask="bool", mask_shape=(33, 4, 2, 280)),
])
def test_shared_past_in_the_256_row_pass(kw):
    """The batch's rows packed in two row tiles against the one copy, own keys beside it."""
    require_gpu()
    wl = W.decoder_attention(**kw)
    op = plan_for(wl, attention_mode="flash").ops[0]
    assert op.ip[K.AF_PASS_PAST] == K.AF_PASS_WIDE
    verify(kw)


@pytest.mark.parametrize("q_seq,d", [(1, 64), (3, 128), (40, 64), (200, 64), (200, 128)])
def test_infinite_and_nan_scores(q_seq, d):
    """A visible NaN or infinite score makes its row NaN, as exp does, and no other row."""
    require_gpu()
    kw = dict(batch=2, q_heads=2, kv_heads=2, q_seq=q_seq, kv_seq=200, head_dim=d)
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(23)
    want = decoder_attention(wl, x)
    x["Q"][0, 1, q_seq // 2, 3] = np.nan
    x["Q"][1, 0, 0] = 0  # only its first element meets the infinite key below
    x["Q"][1, 0, 0, 0] = 1
    x["K"][1, 0, 150, 0] = np.inf
    got = run(wl, x)
    assert np.isnan(got[0, 1, q_seq // 2]).all() and np.isnan(got[1, 0, 0]).all()
    fine = np.ones(got.shape, bool)
    fine[0, 1, q_seq // 2] = False
    fine[1, 0] = False  # (every row of that head meets the infinity)
    y, tol = want
    check(got[fine], y[fine], tol[fine], str(kw))


def test_boolean_mask_longer_than_an_item_holds():
    """More keys than one few-row item keeps mask bits for: split, whatever the batch."""
    require_gpu()
    verify(dict(batch=160, q_heads=1, kv_heads=1, q_seq=1, kv_seq=4200, head_dim=8, mask="bool", mask_shape=(160, 1, 1, 4200)))


def test_scores_of_hidden_keys_do_not_matter():
    """Infinite and NaN scores of keys that a row does not see leave it alone."""
    require_gpu()
    for mask, tq in (("bool", 30), ("f16", 30), ("bool", 6), ("f16", 6)):
        kw = dict(batch=1, q_heads=2, kv_heads=2, q_seq=tq, kv_seq=150, mask=mask, mask_shape=(1, 1, tq, 150))
        wl = W.decoder_attention(**kw)
        x = wl.make_inputs(9)
        x["mask"][..., [3, 70, 149]] = False if mask == "bool" else -np.inf
        want = decoder_attention(wl, x)
        x["K"][:, :, 3], x["K"][:, :, 70], x["K"][:, :, 149] = np.inf, np.nan, -np.inf
        check(run(wl, x), *want, mask)


@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("kw", [
    dict(batch=5, q_heads=8, kv_heads=2, q_seq=1, kv_seq=33, past=200, head_dim=128),
    dict(batch=70, q_heads=4, kv_heads=1, q_seq=1, kv_seq=1, past=65, head_dim=64),   # several row tiles of a prefix
    dict(batch=7, q_heads=12, kv_heads=4, q_seq=3, kv_seq=40, past=1001, head_dim=64),
    dict(batch=2, q_heads=4, kv_heads=4, q_seq=90, kv_seq=90, past=500, causal=True, head_dim=80),
    dict(batch=1, q_heads=2, kv_heads=1, q_seq=4, kv_seq=4, past=1, causal=True, head_dim=32, v_dim=64),
    dict(batch=3, q_heads=4, kv_heads=2, q_seq=2, kv_seq=70, past=130, rank=3),
    dict(batch=3, q_heads=4, kv_heads=2, q_seq=1, kv_seq=20, past=9000, head_dim=128),  # split prefix
    dict(batch=130, q_heads=8, kv_heads=2, q_seq=1, kv_seq=300, past=700, head_dim=128),
    dict(batch=4, q_heads=8, kv_heads=2, q_seq=3, kv_seq=50, past=300, head_dim=128),   # 12 rows a sequence
    dict(batch=2, q_heads=4, kv_heads=2, q_seq=30, kv_seq=30, past=300, causal=True),   # 60 rows a sequence
    dict(batch=2, q_heads=4, kv_heads=2, q_seq=3, kv_seq=3, past=100, causal=True, head_dim=24),
])
def test_past(kw, shared):
    require_gpu()
    verify(dict(kw, shared_past=shared))


@pytest.mark.parametrize("batch", [6, 40])
@pytest.mark.parametrize("shared", [True, False])
def test_past_with_masks(shared, batch):
    """A mask over prefix and suffix: hidden prefix keys, hidden suffixes, a row
    that sees the prefix alone, the suffix alone, or nothing."""
    require_gpu()
    kw = dict(batch=batch, q_heads=4, kv_heads=2, q_seq=2, kv_seq=70, past=321, mask="bool", mask_shape=(batch, 1, 2, 391),
              shared_past=shared)
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(11)
    x["mask"][0, 0, 0, 321:] = False
    x["mask"][1, 0, 1, :321] = False
    x["mask"][2, 0, 0] = False
    x["mask"][3, 0, :, 200:321] = False
    got = run(wl, x)
    check(got, *decoder_attention(wl, x), str(kw))
    assert not got[2, :, 0].any()


def test_expand_that_others_read_is_materialised():
    """Only an Expand whose every reader is an attention's past disappears."""
    require_gpu()
    wl = W.decoder_attention(batch=2, past=66, kv_seq=10, q_seq=3)
    wl.graph.outputs.append(TensorSpec("PKx", "f16", wl.graph.tensor("PKx").shape))
    plan = plan_for(wl, attention_mode="flash")
    assert [o.kernel for o in plan.ops] == [K.K_TRANSPOSE, K.K_ATTENTION_FLASH]
    x = wl.make_inputs(2)
    out = Session(plan).run(x)
    assert np.array_equal(out["PKx"], np.broadcast_to(x["PK"], out["PKx"].shape))
    check(out["Y"], *decoder_attention(wl, x), "")


@pytest.mark.parametrize("shape,target", [((1, 3), (2, 1)), ((4, 1, 2), (3, 1, 5, 1)), ((1,), (7,))])
@pytest.mark.parametrize("dtype", ["f16", "f32", "u8"])
def test_expand(shape, target, dtype):
    require_gpu()
    out = np.broadcast_shapes(shape, target)
    g = GraphSpec("e", [TensorSpec("X", dtype, shape)], [TensorSpec("Y", dtype, out)],
                  [NodeSpec("Expand", "e", ("X", "s"), ("Y",))], {"s": np.array(target, np.int64)})
    x = np.arange(int(np.prod(shape))).astype({"f16": np.float16, "f32": np.float32, "u8": np.uint8}[dtype]).reshape(shape)
    got = Session(B200PlanEmitter().emit_plan(lowering.lower(g))).run({"X": x})["Y"]
    assert np.array_equal(got, np.broadcast_to(x, out))


def test_batch_slices():
    """A slice of the batch with masks, counts or a past per sequence gives the whole run's rows."""
    require_gpu()
    for kw in (dict(mask="bool", mask_shape=(4, 1, 5, 3000)), dict(count=True), dict(past=40, shared_past=False),
               dict(mask="f16", mask_shape=(4, 1, 1, 3000))):
        wl = W.decoder_attention(batch=4, kv_seq=3000, **kw) if "past" not in kw else W.decoder_attention(batch=4, **kw)
        x = wl.make_inputs(12)
        plan = plan_for(wl, attention_mode="flash")
        assert plan.batch == 4, kw
        sess = Session(plan)
        whole = sess.run(x)["Y"]
        check(whole, *decoder_attention(wl, x), str(kw))
        part = sess.run(x, 1, 2)["Y"]
        assert np.array_equal(part[1:3], whole[1:3]) and not part[0].any() and not part[3].any()


@pytest.mark.parametrize("overlap", [False, True])
def test_page_locked_host_buffers(overlap):
    """Runs on page-locked host memory, sliced along the batch or overlapping one another, give the device run's bits."""
    require_gpu()
    import torch
    wl = W.decoder_attention(batch=6, q_heads=8, kv_heads=4, q_seq=40, kv_seq=700, mask="bool", mask_shape=(6, 1, 40, 700),
                             head_dim=64)
    plan = plan_for(wl, attention_mode="flash")
    sess = Session(plan)
    sess.set_host_io_overlap(overlap)
    jobs = []
    for seed in (1, 2, 3):
        x = wl.make_inputs(seed)
        host = [torch.from_numpy(x[n]).pin_memory() for n in plan.input_names]
        jobs.append((x, host, torch.zeros(plan.output_shapes[0], dtype=torch.float16).pin_memory()))
    for _, host, y in jobs:
        sess.run_ptrs([t.data_ptr() for t in host], [y.data_ptr()])
    sess.sync()
    for x, _, y in jobs:
        check(y.numpy(), *decoder_attention(wl, x), "page-locked")
        assert np.array_equal(y.numpy().view(np.uint16), Session(plan).run(x)["Y"].view(np.uint16))


def test_repeated_and_uncaptured_runs_identical():
    """Merging split key ranges has a fixed order; a replayed graph and direct launches agree."""
    require_gpu()
    wl = W.decoder_attention(batch=3, q_heads=8, kv_heads=2, q_seq=1, kv_seq=2000, past=3000, head_dim=128)
    x = wl.make_inputs(13)
    sess = Session(plan_for(wl, attention_mode="flash"))
    first = sess.run(x)["Y"]
    for _ in range(3):
        assert np.array_equal(sess.run(x)["Y"].view(np.uint16), first.view(np.uint16))
    sess.set_graphs(False)
    assert np.array_equal(sess.run(x)["Y"].view(np.uint16), first.view(np.uint16))
    other = dict(wl.make_inputs(14))
    check(sess.run(other)["Y"], *decoder_attention(wl, other), "other inputs, same session")


def test_two_sessions_on_two_streams():
    """Sessions share nothing: two of one plan, interleaved on two streams."""
    require_gpu()
    import torch
    wl = W.decoder_attention(batch=2, q_heads=8, kv_heads=2, q_seq=1, kv_seq=900, past=3000, mask="bool",
                             mask_shape=(2, 1, 1, 3900), head_dim=128)
    plan = plan_for(wl, attention_mode="flash")
    jobs = []
    for seed in (1, 2):
        x = wl.make_inputs(seed)
        s = torch.cuda.Stream()
        dev = [torch.from_numpy(x[n]).cuda() for n in plan.input_names]
        y = torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda")
        jobs.append((Session(plan), s, dev, y, decoder_attention(wl, x)))
    torch.cuda.synchronize()
    for _ in range(5):
        for sess, s, dev, y, _ in jobs:
            sess.run_ptrs([t.data_ptr() for t in dev], [y.data_ptr()], stream=s.cuda_stream)
    torch.cuda.synchronize()
    for _, _, _, y, want in jobs:
        check(y.cpu().numpy(), *want, "")


def test_captured_into_a_callers_graph():
    """With its own graph replay off, a session's run can be part of a caller's
    graph: replayed on other inputs, beside an eager run of another session."""
    require_gpu()
    import torch
    for kw in (dict(batch=3, q_heads=8, kv_heads=2, q_seq=1, kv_seq=2000, past=3000, head_dim=128),
               dict(batch=40, q_heads=8, kv_heads=2, q_seq=1, kv_seq=70, past=900, head_dim=128, mask="bool"),
               dict(batch=2, q_heads=4, kv_heads=2, q_seq=100, kv_seq=77, mask="f16", mask_shape=(2, 1, 100, 77))):
        wl = W.decoder_attention(**kw)
        plan = plan_for(wl, attention_mode="flash")
        sess, other = Session(plan), Session(plan)
        sess.set_graphs(False)
        x = [wl.make_inputs(s) for s in (1, 2)]
        dev = [torch.from_numpy(x[0][n]).cuda() for n in plan.input_names]
        y = torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            sess.run_ptrs([t.data_ptr() for t in dev], [y.data_ptr()], stream=torch.cuda.current_stream().cuda_stream)
        for v in (1, 0):
            for t, n in zip(dev, plan.input_names):
                t.copy_(torch.from_numpy(x[v][n]))
            graph.replay()
            check(other.run(x[1 - v])["Y"], *decoder_attention(wl, x[1 - v]), "beside the replay")
            torch.cuda.synchronize()
            check(y.cpu().numpy(), *decoder_attention(wl, x[v]), str(kw))


def test_misaligned_buffers_are_refused():
    require_gpu()
    import torch
    wl = W.decoder_attention()
    x = wl.make_inputs(0)
    plan = plan_for(wl, attention_mode="flash")
    sess = Session(plan)
    dev = [torch.from_numpy(x[n]).cuda() for n in plan.input_names]
    y = torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda")
    extra = torch.zeros(dev[0].numel() + 8, dtype=torch.float16, device="cuda")
    for i in range(3):
        ptrs = [t.data_ptr() for t in dev]
        ptrs[i] = extra.data_ptr() + 2
        with pytest.raises(EmxError, match="16"):
            sess.run_ptrs(ptrs, [y.data_ptr()])
    sess.run_ptrs([t.data_ptr() for t in dev], [y.data_ptr()])
    sess.sync()
    check(y.cpu().numpy(), *decoder_attention(wl, x), "after the refusals")


def _stage(g, names, inputs, outputs):
    """The nodes ``names`` of a graph as a graph of their own."""
    nodes = [n for n in g.nodes if n.name in names]
    used = {i for n in nodes for i in n.inputs}
    return GraphSpec("stage", [g.tensor(n) for n in inputs], [g.tensor(n) for n in outputs], nodes,
                     {k: v for k, v in g.initializers.items() if k in used},
                     [t for t in g.values if t.name not in inputs and t.name not in outputs], g.opset_imports)


@pytest.mark.parametrize("kw", [dict(), dict(batch=9, tokens=1, prefix=2000, frames=1500),
                                dict(tokens=70, head_dim=128, q_heads=8)])
def test_decoder_layer(kw):
    """Norm and rotation, attention behind a shared prefix, norm, cross attention
    in one plan: the same bits as its stages run one by one, each of which is
    within its bound on the inputs it got."""
    require_gpu()
    wl = W.decoder_layer(**kw)
    p, g = wl.params, infer_types(wl.graph)
    x = wl.make_inputs(4)
    plan = plan_for(wl, attention_mode="flash")
    assert [o.kernel for o in plan.ops] == [K.K_NORM_ROPE, K.K_ATTENTION_FLASH, K.K_TRANSPOSE, K.K_RMS_NORM,
                                            K.K_ATTENTION_FLASH]
    whole = Session(plan).run(x)["Y"]
    v = dict(x)
    for names, ins, outs in (
            (["Q_norm", "Q_heads", "Q_rope", "K_norm", "K_heads", "K_rope"], ["Q", "K", "pos"], ["Qr", "Kr"]),
            (["share_k", "share_v", "self"], ["Qr", "Kr", "V", "prefix_k", "prefix_v"], ["S"]),
            (["tokens", "join", "x_norm"], ["S"], ["X"]), (["cross"], ["X", "enc_k", "enc_v", "count"], ["Y"])):
        st = B200PlanEmitter(attention_mode="flash").emit_plan(lowering.lower(_stage(g, names, ins, outs)))
        v.update(Session(st).run({n: v[n] for n in ins}))
    assert np.array_equal(whole.view(np.uint16), v["Y"].view(np.uint16))
    b, t, hq, d = p["batch"], p["tokens"], p["q_heads"], p["head_dim"]
    cos, sin = (g.initializers[n][x["pos"]] for n in ("cos", "sin"))
    for n in ("Q", "K"):
        y, mag = rotate(rms_norm(x[n], g.initializers[n.lower() + "_scale"], 1e-6), cos, sin, d, False)
        tol = 2.0 ** -11 * np.abs(y) + 2.0 ** -25 + 40 * 2.0 ** -24 * mag
        check(v[n + "r"], y.transpose(0, 2, 1, 3), tol.transpose(0, 2, 1, 3), n)
    past = [np.broadcast_to(x[n], (b, *x[n].shape[1:])) for n in ("prefix_k", "prefix_v")]
    check(v["S"], *attention(v["Qr"], np.concatenate([past[0], v["Kr"]], 2), np.concatenate([past[1], x["V"]], 2),
                             d ** -0.5, past=p["prefix"], causal=True), "self")
    y = rms_norm(v["S"].transpose(0, 2, 1, 3).reshape(b, t, hq * d), g.initializers["x_scale"], 1e-5)
    check(v["X"], y, (2.0 ** -11 + 40 * 2.0 ** -24) * np.abs(y) + 2.0 ** -25, "norm")
    heads = [v[n].reshape(b, -1, hq, d).transpose(0, 2, 1, 3) for n in ("X", "enc_k", "enc_v")]
    y, tol = attention(*heads, d ** -0.5, counts=x["count"])
    check(v["Y"], *(a.transpose(0, 2, 1, 3).reshape(b, t, hq * d) for a in (y, tol)), "cross")


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("kw", [dict(batch=80, tokens=1, q_heads=8, prefix=900), dict(batch=40, tokens=2, q_heads=4, prefix=4200),
                                dict(batch=60, tokens=1, q_heads=8, prefix=700, head_dim=128)])
def test_passes_side_by_side_read_what_came_before_both(kw, graphs):
    """Own keys' few-row pass beside the shared past's tile pass, with Q and K from the same run's rotation: the bits of
    a run of its own, on changing inputs in the same buffers."""
    require_gpu()
    import torch
    wl = W.decoder_layer(**kw)
    plan = plan_for(wl, attention_mode="flash")
    op = next(o for o in plan.ops if o.kernel == K.K_ATTENTION_FLASH)
    assert op.ip[K.AF_PASS_OWN] in (K.AF_PASS_ROWS8, K.AF_PASS_ROWS16) and op.ip[K.AF_PASS_PAST] in (K.AF_PASS_TILES, K.AF_PASS_WIDE)
    g = infer_types(wl.graph)
    stages = []
    for names, ins, outs in (
            (["Q_norm", "Q_heads", "Q_rope", "K_norm", "K_heads", "K_rope"], ["Q", "K", "pos"], ["Qr", "Kr"]),
            (["share_k", "share_v", "self"], ["Qr", "Kr", "V", "prefix_k", "prefix_v"], ["S"]),
            (["tokens", "join", "x_norm"], ["S"], ["X"]), (["cross"], ["X", "enc_k", "enc_v", "count"], ["Y"])):
        st = B200PlanEmitter(attention_mode="flash").emit_plan(lowering.lower(_stage(g, names, ins, outs)))
        stages.append((Session(st), ins))
    xs = [wl.make_inputs(s) for s in range(50, 53)]
    want = []
    for x in xs:
        v = dict(x)
        for sess, ins in stages:
            v.update(sess.run({n: v[n] for n in ins}))
        want.append(v["Y"])
    sess = Session(plan)
    sess.set_graphs(graphs)
    dev = [torch.from_numpy(xs[0][n]).cuda() for n in plan.input_names]
    y = torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda")
    for _ in range(4):
        for x, w in zip(xs, want):
            for t, n in zip(dev, plan.input_names):
                t.copy_(torch.from_numpy(x[n]))
            sess.run_ptrs([t.data_ptr() for t in dev], [y.data_ptr()], stream=torch.cuda.current_stream().cuda_stream or 1)
            torch.cuda.synchronize()
            assert np.array_equal(y.cpu().numpy().view(np.uint16), w.view(np.uint16))
    sess.sync()


@pytest.mark.parametrize("shared", [True, False])
def test_empty_past_on_the_device(shared):
    """A first step's past of no tokens: its device tensors have no address."""
    require_gpu()
    import torch
    kw = dict(batch=2, q_heads=4, kv_heads=2, q_seq=5, kv_seq=5, causal=True)
    wl = W.decoder_attention(**kw, past=16, shared_past=shared)
    g = wl.graph
    for n in ("PK", "PV"):
        i = next(k for k, t in enumerate(g.inputs) if t.name == n)
        g.inputs[i] = TensorSpec(n, "f16", (1 if shared else 2, 2, 0, 64))
        if shared:
            g.initializers[n + "_shape"] = np.array([2, 2, 0, 64], np.int64)
    g.values.clear()
    plan = plan_for(wl, attention_mode="flash")
    plain = W.decoder_attention(**kw)
    x = plain.make_inputs(3)
    dev = {n: torch.from_numpy(x[n]).cuda() for n in "QKV"}
    dev.update({n: torch.empty(0, dtype=torch.float16, device="cuda") for n in ("PK", "PV")})
    assert dev["PK"].data_ptr() == 0
    y = torch.zeros(plan.output_shapes[0], dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    sess = Session(plan)
    sess.run_ptrs([dev[n].data_ptr() for n in plan.input_names], [y.data_ptr()])
    sess.sync()
    check(y.cpu().numpy(), *decoder_attention(plain, x), str(kw))
    with pytest.raises(EmxError, match="NULL"):
        sess.run_ptrs([0 if n == "K" else dev[n].data_ptr() for n in plan.input_names], [y.data_ptr()])
