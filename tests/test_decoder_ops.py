"""Decoder operators on the host (no GPU): shapes and attributes, what the
planner fuses and shares, split decisions, refusals, the ONNX round trip, and
the index arithmetic of attention_flash.cu's work items."""
import numpy as np
import pytest

from decoder_reference import attention, rotate
from emx_onnx_cgen_b200 import kernel_ids as K
from emx_onnx_cgen_b200 import lowering
from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.lowering import UnsupportedOpError
from emx_onnx_cgen_b200.onnx_reader import infer_types, read_onnx
from emx_onnx_cgen_b200.onnx_writer import write_onnx
from emx_onnx_cgen_b200.plan import B200PlanEmitter, flash_schedule, flash_splits
from emx_onnx_cgen_b200.spec import GraphSpec, NodeSpec, TensorSpec


def plan_of(wl, **kw):
    g = wl if isinstance(wl, GraphSpec) else wl.graph
    return B200PlanEmitter(**{"attention_mode": "flash", **kw}).emit_plan(lowering.lower(g))


def kernels(wl, **kw):
    return [o.kernel for o in plan_of(wl, **kw).ops]


# ------------------------------------------------------------------ norm and rotation
@pytest.mark.parametrize("layout", ["transpose", "heads", "flat"])
@pytest.mark.parametrize("norm", [True, False])
def test_norm_transpose_and_rotation_are_one_launch(layout, norm):
    wl = W.norm_rope(layout=layout, norm=norm, q_heads=6, kv_heads=2, head_dim=32, seq=5, batch=2)
    plan = plan_of(wl)
    assert [o.kernel for o in plan.ops] == [K.K_NORM_ROPE]
    op = plan.ops[0]
    assert op.ip[K.NR_ITEMS] == 2 and (op.ip[K.NR_H0], op.ip[K.NR_H1]) == (6, 2)
    assert (op.tensors[4] >= 0) == norm and (op.tensors[7] >= 0) == norm
    h, t, d = 6, 5, 32
    flat, heads = (t * h * d, h * d, d), (h * t * d, d, t * d)
    xs, ys = {"transpose": (flat, heads), "heads": (heads, heads), "flat": (flat, flat)}[layout]
    assert tuple(op.ip[s] for s in (K.NR_X0_SB, K.NR_X0_ST, K.NR_X0_SH)) == xs
    assert tuple(op.ip[s] for s in (K.NR_Y0_SB, K.NR_Y0_ST, K.NR_Y0_SH)) == ys
    assert plan.batch == 2


def test_norm_read_by_others_stays_apart():
    wl = W.norm_rope()
    wl.graph.outputs.append(TensorSpec("Qn", "f16", wl.graph.tensor("Qn").shape))
    assert kernels(wl) == [K.K_RMS_NORM, K.K_NORM_ROPE]
    op = plan_of(wl).ops[-1]
    assert op.ip[K.NR_ITEMS] == 2 and op.tensors[4] == -1 and op.tensors[7] >= 0


def test_rotations_are_paired_only_where_order_allows():
    """A reader of the first rotation's output before the second keeps them apart."""
    wl = W.norm_rope(layout="heads", norm=False, q_heads=4, kv_heads=4)
    g = wl.graph
    shape = g.tensor("Q").shape
    g.nodes[1] = NodeSpec("RotaryEmbedding", "K_rope", ("YQ", "cos", "sin", "pos"), ("YK",), g.nodes[1].attrs)
    g.inputs = [t for t in g.inputs if t.name != "K"]
    plan = plan_of(wl)
    assert [o.kernel for o in plan.ops] == [K.K_NORM_ROPE, K.K_NORM_ROPE] and plan.ops[0].ip[K.NR_ITEMS] == 1
    assert shape == g.tensor("YK").shape


def test_batch_slicing_of_rotations():
    assert plan_of(W.norm_rope(batch=4, positions="rows")).batch == 4
    # position ids fixed as an initializer do not follow a slice: the plan runs whole
    wl = W.norm_rope(batch=4, seq=3)
    wl.graph.inputs = [t for t in wl.graph.inputs if t.name != "pos"]
    wl.graph.initializers["pos"] = np.zeros((4, 3), np.int64)
    assert plan_of(wl).batch == 0


def _rope(**kw):
    wl = W.norm_rope(**{"layout": "heads", "norm": False, **kw})
    return wl.graph


@pytest.mark.parametrize("change,match", [
    (lambda g: g.initializers.update(cos=g.initializers["cos"][:, :5]), "caches"),
    (lambda g: g.initializers.update(cos=g.initializers["cos"].astype(np.float32)), "caches"),
    (lambda g: g.initializers.update(cos=g.initializers["cos"][None], sin=g.initializers["sin"][None]), "caches"),
    (lambda g: g.nodes.__setitem__(0, NodeSpec("RotaryEmbedding", "r", ("Q", "cos", "sin"), ("YQ",), {})), "without"),
    (lambda g: g.nodes.__setitem__(0, NodeSpec("RotaryEmbedding", "r", ("Q", "cos", "sin", "pos"), ("YQ",),
                                               {"rotary_embedding_dim": 66})), "66 rotated"),
    (lambda g: g.nodes.__setitem__(0, NodeSpec("RotaryEmbedding", "r", ("Q", "cos", "sin", "pos"), ("YQ",),
                                               {"rotary_embedding_dim": 7})), "7 rotated"),
    (lambda g: g.nodes.__setitem__(0, NodeSpec("RotaryEmbedding", "r", ("Q", "cos", "sin", "pos"), ("YQ",),
                                               {"num_heads": 5})), "num_heads"),
    (lambda g: g.inputs.__setitem__(0, TensorSpec("pos", "i32", g.tensor("pos").shape)), "position_ids"),
])
def test_rotation_refusals(change, match):
    g = _rope()
    assert g.inputs[0].name == "pos"
    change(g)
    with pytest.raises(UnsupportedOpError, match=match):
        plan_of(g)


def test_norm_refusals():
    def graph(xs, ss, attrs, dt="f16", sdt=np.float16):
        return GraphSpec("n", [TensorSpec("X", dt, xs)], [TensorSpec("Y", dt, xs)],
                         [NodeSpec("RMSNormalization", "n", ("X", "s"), ("Y",), attrs)], {"s": np.ones(ss, sdt)})

    assert kernels(graph((2, 3, 4), (3, 4), {"axis": 1})) == [K.K_RMS_NORM]
    for args, match in ((((2, 4), (1,), {}), "scale"), (((2, 4), (4,), {"stash_type": 10}), "stash_type"),
                        (((2, 4), (4,), {"axis": 2}), "axis 2"), (((2, 4), (4,), {}, "f64", np.float64), "f64"),
                        (((2, 4), (4,), {}, "f16", np.float32), "f32 scale")):
        with pytest.raises(UnsupportedOpError, match=match):
            plan_of(graph(*args))


# ------------------------------------------------------------------ attention
def test_shared_past_has_no_expand():
    plan = plan_of(W.decoder_attention(past=128, batch=6))
    assert [o.kernel for o in plan.ops] == [K.K_ATTENTION_FLASH]
    op = plan.ops[0]
    assert op.ip[K.AF_PAST_SHARED] == 1 and op.ip[K.AF_TP] == 128
    assert plan.tensors[op.tensors[5]].shape == (1, 2, 128, 64)
    # in the other modes the past has no kernel
    for mode in ("exact", "tensor"):
        with pytest.raises(UnsupportedOpError, match="past"):
            plan_of(W.decoder_attention(past=128), attention_mode=mode)


def test_expand_of_heads_is_not_a_shared_past():
    wl = W.decoder_attention(batch=2, kv_heads=2, past=16)
    g = wl.graph
    for n in ("PK", "PV"):
        i = next(k for k, t in enumerate(g.inputs) if t.name == n)
        g.inputs[i] = TensorSpec(n, "f16", (1, 1, 16, 64))
    plan = plan_of(wl)
    assert [o.kernel for o in plan.ops] == [K.K_TRANSPOSE, K.K_TRANSPOSE, K.K_ATTENTION_FLASH]
    assert plan.ops[-1].ip[K.AF_PAST_SHARED] == 0


def test_past_of_no_tokens():
    wl = W.decoder_attention(batch=2, past=16, shared_past=False)
    for n in ("PK", "PV"):
        i = next(k for k, t in enumerate(wl.graph.inputs) if t.name == n)
        wl.graph.inputs[i] = TensorSpec(n, "f16", (2, 2, 0, 64))
    op = plan_of(wl).ops[0]
    assert op.ip[K.AF_TP] == 0 and op.tensors[5] == -1


@pytest.mark.parametrize("kw,match", [
    (dict(head_dim=136), "head sizes"), (dict(head_dim=20), "head sizes"), (dict(v_dim=4), "head sizes"),
    (dict(count=True, past=8), "nonpad"), (dict(count=True, causal=True), "nonpad"),
    (dict(mask="u8", mask_shape=(2, 1, 1, 70)), "u8 mask"),
])
def test_attention_refusals(kw, match):
    with pytest.raises(UnsupportedOpError, match=match):
        plan_of(W.decoder_attention(**kw))


@pytest.mark.parametrize("ms", [(3, 1, 1, 70), (2, 3, 1, 70), (2, 1, 4, 70), (2, 1, 1, 71), (70,), (2, 1, 1, 1),
                                (1, 2, 1, 1, 70)])
def test_mask_shapes_that_do_not_broadcast(ms):
    with pytest.raises(UnsupportedOpError, match="attn_mask"):
        plan_of(W.decoder_attention(mask="bool", mask_shape=ms))


def test_masks_are_refused_outside_flash_mode():
    """A mask input is never dropped: the modes without a masked kernel refuse it."""
    for mode in ("exact", "tensor"):
        for kw in (dict(mask="bool"), dict(count=True)):
            with pytest.raises(UnsupportedOpError, match="masks"):
                plan_of(W.decoder_attention(**kw), attention_mode=mode)
    with pytest.raises(UnsupportedOpError, match="masks"):
        plan_of(W.decoder_attention(mask="bool"), use_tensor_cores=False)


def _attention_graph(shapes, attrs=None, outputs=("Y",), dtype="f16", extra=()):
    ins = [TensorSpec(n, dtype, s) for n, s in zip("QKV", shapes)] + list(extra)
    names = ["Q", "K", "V"] + [t.name for t in extra]
    return GraphSpec("a", ins, [TensorSpec("Y", dtype, (2, 4, 3, 64))],
                     [NodeSpec("Attention", "a", tuple(names), outputs, attrs or {})], {})


def test_shape_and_output_refusals():
    q, k = (2, 4, 3, 64), (2, 2, 9, 64)
    assert kernels(_attention_graph((q, k, k))) == [K.K_ATTENTION_FLASH]
    for shapes, attrs, match in (((q, (2, 3, 9, 64), (2, 3, 9, 64)), {}, "over 3"), ((q, (1, 2, 9, 64), k), {}, "fit"),
                                 ((q, (2, 2, 9, 32), k), {}, "fit"), ((q, k, (2, 2, 8, 64)), {}, "fit"),
                                 (((2, 3, 256), k, k), {}, "q_num_heads"),
                                 (((2, 3, 256), k, k), {"q_num_heads": 3}, "q_num_heads"),
                                 ((q, k, k), {"softcap": 30.0}, "softcap")):
        with pytest.raises(UnsupportedOpError, match=match):
            plan_of(_attention_graph(shapes, attrs))
    with pytest.raises(UnsupportedOpError, match="present"):
        plan_of(_attention_graph((q, k, k), outputs=("Y", "pk", "pv")))
    with pytest.raises(UnsupportedOpError, match="fp16"):
        plan_of(_attention_graph((q, k, k), dtype="f32"))
    with pytest.raises(UnsupportedOpError, match="empty"):
        plan_of(_attention_graph((q, (2, 2, 0, 64), (2, 2, 0, 64))))


def test_splits_keep_every_item_resident():
    assert flash_splits([(1, 100)], 296, 4) == [25]                   # four tiles an item at least
    assert flash_splits([(296, 100)], 296, 4) == [1]
    assert flash_splits([(148, 64)], 296, 4) == [2]
    assert flash_splits([(4000, 3)], 296, 4) == [1]
    assert flash_splits([(1, 1)], 296, 4) == [1]
    for items in range(1, 400, 7):
        for tiles in (1, 2, 7, 33, 250):
            (s,) = flash_splits([(items, tiles)], 296, 4)
            assert 1 <= s <= tiles and (s == 1 or items * s <= 296)
    a, b = flash_splits([(128, 1), (32, 128)], 296, 4)
    assert a == 1 and 1 < b <= 128


def test_schedules():
    rows8, rows16, tiles, wide, none = (K.AF_PASS_ROWS8, K.AF_PASS_ROWS16, K.AF_PASS_TILES, K.AF_PASS_WIDE,
                                        K.AF_PASS_NONE)
    pick = lambda *a: (lambda s: (s.own, s.past))(flash_schedule(*a))
    assert pick(16, 16, 1, 1500, 0, False) == (rows8, none)
    assert pick(2, 2, 12, 1500, 0, False) == (rows16, none)
    assert pick(2, 2, 17, 1500, 0, False) == (tiles, none)
    assert pick(4, 2, 4, 10, 500, False) == (rows8, none)       # a past of its own is part of the row's keys
    assert pick(8, 8, 4, 33, 2048, True) == (rows16, rows16)    # 32 packed rows
    assert pick(16, 8, 4, 33, 2048, True, "", 64) == (rows16, rows16)
    assert pick(16, 8, 4, 33, 2048, True) == (rows16, rows16)
    assert pick(17, 8, 4, 33, 2048, True) == (rows8, tiles)
    assert pick(16, 8, 4, 33, 4097, True) == (rows8, tiles)
    assert pick(25, 8, 4, 33, 2048, True, "", 64) == (rows8, tiles)
    assert pick(2, 8, 4, 33, 2048, True) == (rows8, rows8)
    assert pick(33, 8, 4, 33, 2048, True) == (rows8, wide)
    assert pick(33, 8, 4, 33, 2048, True, "f16") == (rows8, tiles)  # additive masks: no wide form
    assert pick(2, 2, 129, 1500, 0, False) == (wide, none)
    assert pick(2, 2, 129, 1500, 0, False, "f32") == (tiles, none)
    assert pick(1, 8, 4, 33, 2048, True) == (rows8, none)       # nobody to share with
    assert pick(3, 8, 100, 33, 2048, True) == (tiles, tiles)
    assert pick(3, 8, 128, 33, 2048, True) == (tiles, none)
    for args in ((1, 1, 1, 5000, 0, False), (128, 8, 4, 256, 8192, True), (7, 4, 9, 40, 1001, True)):
        s = flash_schedule(*args)
        assert s.slots == s.splits_own + s.splits_past and (s.splits_past > 0) == (s.past != none)
    # the few-row pass holds a key range's boolean mask on chip
    for b, tk, tp, shared in ((400, 9000, 0, False), (400, 4097, 0, False), (2, 9000, 20000, True), (300, 5000, 70000, False)):
        s = flash_schedule(b, 8, 4, tk, tp, shared, "bool")
        blocks = lambda *parts: sum(-(-t // 16) for t in parts)
        own, past = (blocks(tk), blocks(tp)) if s.past != none else (blocks(tk, tp), 0)
        assert -(-own // s.splits_own) * 16 <= K.AF_ROWS_MASK_KEYS
        assert s.past not in (rows8, rows16) or -(-past // s.splits_past) * 16 <= K.AF_ROWS_MASK_KEYS


def test_partials_are_reserved_for_split_or_two_part_keys():
    t = lambda plan: plan.ops[0].tensors[8]
    assert t(plan_of(W.decoder_attention(batch=2, q_heads=2, kv_heads=2, kv_seq=64))) == -1
    plan = plan_of(W.decoder_attention(batch=2, q_heads=2, kv_heads=2, q_seq=1, kv_seq=4096))
    s = plan.ops[0].ip[K.AF_SPLITS_K]
    assert s > 1 and plan.tensors[t(plan)].shape == (s, 2 * 1 * 2, 66)
    plan = plan_of(W.decoder_attention(batch=2, q_heads=2, kv_heads=2, q_seq=1, past=64, kv_seq=5))
    assert plan.tensors[t(plan)].shape == (2, 4, 66)
    assert t(plan_of(W.decoder_attention(batch=2, q_heads=2, kv_heads=2, q_seq=1, past=64, kv_seq=5, shared_past=False))) == -1


def test_batched_operands():
    """A plan may run batch slices only where every operand follows the slice."""
    assert plan_of(W.decoder_attention(batch=4)).batch == 4
    assert plan_of(W.decoder_attention(batch=4, mask="bool", mask_shape=(4, 1, 5, 70))).batch == 4
    assert plan_of(W.decoder_attention(batch=4, count=True)).batch == 4
    assert plan_of(W.decoder_attention(batch=4, past=8, shared_past=False)).batch == 4
    # axis 0 is the batch by number only (a mask per head, or per query)
    assert plan_of(W.decoder_attention(batch=4, q_heads=4, mask="bool", mask_shape=(4, 1, 70))).batch == 0
    assert plan_of(W.decoder_attention(batch=5, q_seq=5, mask="bool", mask_shape=(5, 70))).batch == 0
    assert plan_of(W.decoder_attention(batch=4, past=8)).batch == 0
    # a fixed mask: with a row per sequence it does not follow a slice, with one for all it does
    for ms, want in (((4, 1, 1, 70), 0), ((1, 1, 1, 70), 4)):
        wl = W.decoder_attention(batch=4, mask="bool", mask_shape=ms)
        wl.graph.inputs = [t for t in wl.graph.inputs if t.name != "mask"]
        wl.graph.initializers["mask"] = np.ones(ms, bool)
        assert plan_of(wl).batch == want


@pytest.mark.parametrize("b,hq,hkv,tq,shared", [(3, 6, 2, 5, True), (70, 8, 8, 1, True), (2, 4, 1, 50, False)])
def test_row_packing_covers_every_query_once(b, hq, hkv, tq, shared):
    """row_of() of attention_flash.cu: tiles of 128 rows over (sequence, token, head of the group)."""
    group = hq // hkv
    rows_all = tq * group * (b if shared else 1)
    seen = np.zeros((b, hq, tq), int)
    for bb in range(1 if shared else b):
        for kvh in range(hkv):
            for tile in range(-(-rows_all // 128)):
                for r in range(tile * 128, min(rows_all, tile * 128 + 128)):
                    g, bt = r % group, r // group
                    bi, t = (bt // tq, bt % tq) if shared else (bb, bt)
                    seen[bi, kvh * group + g, t] += 1
    assert (seen == 1).all()


def test_onnx_round_trip(tmp_path):
    for wl, mode in ((W.norm_rope(), "exact"), (W.norm_rope(layout="flat", positions="rows"), "exact"),
                     (W.decoder_attention(past=20, mask="bool", mask_shape=(2, 1, 5, 90)), "flash"),
                     (W.decoder_attention(rank=3, count=True), "flash"), (W.decoder_layer(), "flash")):
        path = tmp_path / "m.onnx"
        write_onnx(wl.graph, path)
        spec = read_onnx(path)
        spec.values = []  # every intermediate's type is propagated again
        back = plan_of(infer_types(spec), attention_mode=mode)
        here = plan_of(wl, attention_mode=mode)
        assert back.plan_bytes == here.plan_bytes and back.weight_bytes == here.weight_bytes


# ------------------------------------------------------------------ the reference itself
def test_reference_attention_against_a_loop():
    r = np.random.default_rng(0)
    q, k, v = (r.standard_normal(s) for s in ((1, 2, 3, 4), (1, 1, 6, 4), (1, 1, 6, 5)))
    mask = r.random((1, 1, 3, 5)) < 0.6
    mask[0, 0, 1] = False
    y, _ = attention(q, k, v, 0.5, mask=mask, past=3, causal=True)
    for h in range(2):
        for t in range(3):
            keys = [j for j in range(5) if j <= t + 3 and mask[0, 0, t, j]]
            w = np.array([np.exp(0.5 * q[0, h, t] @ k[0, 0, j]) for j in keys])
            want = sum(wi * v[0, 0, j] for wi, j in zip(w, keys)) / w.sum() if keys else np.zeros(5)
            assert np.allclose(y[0, h, t], want, atol=1e-14)


def test_reference_rotation_against_angles():
    x = np.random.default_rng(1).standard_normal((1, 2, 1, 6))
    ang = np.array([[[0.3, 1.1], [0.5, -0.2]]])
    for inter, pairs in ((False, ((0, 2), (1, 3))), (True, ((0, 1), (2, 3)))):
        y, _ = rotate(x, np.cos(ang), np.sin(ang), 4, inter)
        for t in range(2):
            for i, (a, b) in enumerate(pairs):
                z = (x[0, t, 0, a] + 1j * x[0, t, 0, b]) * np.exp(1j * ang[0, t, i])
                assert np.allclose([y[0, t, 0, a], y[0, t, 0, b]], [z.real, z.imag])
        assert np.array_equal(y[..., 4:], x[..., 4:])


def test_one_expand_for_two_attentions():
    """Both read the one copy in place; with another reader as well, the Expand runs and both still read the one copy."""
    wl = W.decoder_attention(batch=3, past=40, kv_seq=9, q_seq=2)
    g = wl.graph
    first = next(n for n in g.nodes if n.op_type == "Attention")
    g.nodes.append(NodeSpec("Attention", "again", ("Y", *first.inputs[1:]), ("Z",), first.attrs))
    g.outputs.append(TensorSpec("Z", "f16", g.tensor("Y").shape))
    plan = plan_of(wl)
    assert [o.kernel for o in plan.ops] == [K.K_ATTENTION_FLASH] * 2
    assert all(o.ip[K.AF_PAST_SHARED] == 1 for o in plan.ops)
    assert plan.ops[0].tensors[5:7] == plan.ops[1].tensors[5:7]
    g.outputs.append(TensorSpec("PKx", "f16", g.tensor("PKx").shape))
    plan = plan_of(wl)
    assert sorted(o.kernel for o in plan.ops) == sorted([K.K_TRANSPOSE] + [K.K_ATTENTION_FLASH] * 2)
    assert all(o.ip[K.AF_PAST_SHARED] == 1 for o in plan.ops if o.kernel == K.K_ATTENTION_FLASH)


def test_more_rows_or_keys_than_the_kernels_number():
    """Row, key and token numbers are 32-bit in the kernels: larger plans are refused, whatever the memory."""
    big = 2 ** 31
    for kw in (dict(batch=1, q_heads=1, kv_heads=1, q_seq=big, kv_seq=8, head_dim=8),
               dict(batch=2, q_heads=2, kv_heads=1, q_seq=big // 4, kv_seq=8, head_dim=8),
               dict(batch=1, q_heads=1, kv_heads=1, q_seq=1, kv_seq=big, head_dim=8),
               dict(batch=1, q_heads=1, kv_heads=1, q_seq=1, kv_seq=big // 2, past=big // 2, head_dim=8)):
        with pytest.raises(UnsupportedOpError, match="no B200 kernel"):
            plan_of(W.decoder_attention(**kw))
    x = TensorSpec("X", "f16", (1, 1, big, 8))
    g = GraphSpec("r", [x, TensorSpec("pos", "i64", (1, big))], [TensorSpec("Y", "f16", x.shape)],
                  [NodeSpec("RotaryEmbedding", "r", ("X", "cos", "sin", "pos"), ("Y",), {})],
                  {n: np.zeros((4, 4), np.float16) for n in ("cos", "sin")})
    with pytest.raises(UnsupportedOpError, match="tokens"):
        plan_of(g)
    assert plan_of(W.decoder_attention(batch=1, q_heads=1, kv_heads=1, q_seq=1, kv_seq=2 ** 20, head_dim=8)).ops
