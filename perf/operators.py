"""Attention-side operators of a decoder layer, as this framework's user meets them in ONNX graphs, and
the cases they are measured on.

* ``norm_rope``: RMSNormalization of every query and key head, the exchange of the token and head axes,
  and RotaryEmbedding, for Q and K of one layer.
* ``cross``: Attention of decoder tokens over an encoder's states of another length, with the encoder's
  valid lengths given as counts, as a boolean mask or as an additive mask.
* ``prefix``: Attention of a batch whose sequences share one long prefix (``Expand`` of the one copy into
  ``past_key`` / ``past_value``), each with its own suffix.

``run`` computes them in elementary torch operations, or, with ``own`` set, through a launch plan of this
package.
"""
import math

import numpy as np
import torch

own = False  # True: run() calls this package's kernels

F16, F32 = torch.float16, torch.float32


# ------------------------------------------------------------------ cases
def _norm_rope(name, b, t, hq, hkv, d, rot, interleaved, dtype):
    c = dict(op="norm_rope", b=b, t=t, hq=hq, hkv=hkv, d=d, rot=rot, interleaved=interleaved, dtype=dtype)
    return dict(c, name=name) if name else c


def _cross(name, b, hq, hkv, tq, tk, d, mask):
    c = dict(op="cross", b=b, hq=hq, hkv=hkv, tq=tq, tk=tk, d=d, mask=mask)
    return dict(c, name=name) if name else c


def _prefix(name, b, hq, hkv, tq, p, s, d, mask):
    c = dict(op="prefix", b=b, hq=hq, hkv=hkv, tq=tq, p=p, s=s, d=d, mask=mask)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoding step of 32 sequences: 1.3 MB moved, the launch is what counts
        _norm_rope("norm-rope one token", 32, 1, 32, 8, 128, 128, False, "f16"),
        # prompts of a serving batch
        _norm_rope("norm-rope prompts", 4, 2048, 32, 8, 128, 128, False, "f16"),
        # odd token count and head size, the first 32 of 80 elements rotated in pairs, fp32
        _norm_rope("norm-rope odd interleaved", 3, 333, 12, 4, 80, 32, True, "f32"),
        # a batch of long prompts
        _norm_rope("norm-rope long prompts", 8, 4096, 32, 8, 128, 128, False, "f16"),
        # one decoding step over encoder states, padded to the longest, valid counts per sequence
        _cross("cross one token", 16, 16, 16, 1, 1500, 64, "count"),
        # a transcript's tokens over padded encoder states, one boolean row per sequence
        _cross("cross tokens over frames", 8, 16, 16, 448, 1500, 64, "bool"),
        # shared key/value heads, head size and lengths off every tile, an additive mask per query row
        _cross("cross odd additive", 3, 12, 4, 77, 333, 80, "add"),
        # long decoder prompts over long encoder states
        _cross("cross long", 4, 32, 8, 2048, 4096, 128, "count"),
        # one decoding step of 16 sequences behind one system prompt, all suffixes as long
        _prefix("prefix one token", 16, 32, 8, 1, 2048, 33, 128, "none"),
        # the same of a large batch with a long prefix, suffixes of different lengths
        _prefix("prefix large batch", 128, 32, 8, 1, 8192, 256, 128, "bool"),
        # three drafted tokens per sequence, every size odd, a boolean row per query
        _prefix("prefix drafted tokens", 7, 12, 4, 3, 1001, 40, 64, "bool"),
        # prompts continued behind a cached prefix, causal among themselves
        _prefix("prefix prompts", 4, 32, 8, 512, 8192, 512, 128, "causal"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    group = rng.choice([1, 1, 2, 3, 4, 8])
    hkv = rng.choice([1, 2, 4, 5, 8, 16])
    return min(group, max(1, 32 // hkv)) * hkv, hkv


def draw(rng):
    while True:
        op = rng.choice(["norm_rope", "cross", "prefix"])
        hq, hkv = _heads(rng)
        b = _log(rng, 1, 64)
        if op == "norm_rope":
            d = rng.choice([32, 64, 80, 96, 128])
            rot = rng.choice([d, d, d // 2 // 2 * 2])
            c = _norm_rope(None, b, _log(rng, 1, 4096), hq, hkv, d, rot, rng.random() < 0.3,
                           rng.choice(["f16", "f16", "f32"]))
            size = c["b"] * c["t"] * (hq + hkv) * d * (2 if c["dtype"] == "f16" else 4)
            if size <= 8 * 4096 * 40 * 128 * 2:
                return c
        elif op == "cross":
            c = _cross(None, b, hq, hkv, _log(rng, 1, 2048), _log(rng, 16, 4096), rng.choice([32, 64, 80, 96, 128]),
                       rng.choice(["none", "count", "count", "bool", "add"]))
            if b * hq * c["tq"] * c["tk"] * c["d"] <= 4 * 32 * 2048 * 4096 * 128:
                return c
        else:
            mask = rng.choice(["none", "bool", "bool", "causal"])
            tq = rng.choice([1, 1, 1, 2, 3, 5]) if mask != "causal" else _log(rng, 2, 512)
            s = tq if mask == "causal" else _log(rng, max(tq, 2), 512)
            c = _prefix(None, b, hq, hkv, tq, _log(rng, 64, 16384), s, rng.choice([64, 80, 128]), mask)
            keys = c["p"] + s
            if b * hq * tq * keys * c["d"] <= 4 * 32 * 2048 * 4096 * 128 and b * hkv * keys * c["d"] <= 1.2e9:
                return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _lengths(case, g, longest):
    """Valid lengths between half and all of `longest`; the first sequence has the longest."""
    n = torch.randint(max(1, longest // 2), longest + 1, (case["b"],), generator=g, device="cuda")
    n[0] = longest
    return n


def _rotary_tables(case):
    """Cosine and sine of every position's angles, base 10000, as a model's initializers hold them."""
    half = case["rot"] // 2
    freq = 10000.0 ** (-np.arange(half, dtype=np.float64) / half)
    angle = np.arange(max(64, case["t"] + 17), dtype=np.float64)[:, None] * freq[None, :]
    npt = np.float16 if case["dtype"] == "f16" else np.float32
    return np.cos(angle).astype(npt), np.sin(angle).astype(npt)


def _inputs(case, seed):
    g = _gen(seed)

    def normal(*shape, dtype=F16):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    if case["op"] == "norm_rope":
        dt = F16 if case["dtype"] == "f16" else F32
        cos, sin = _rotary_tables(case)
        x = {"Q": normal(b, case["t"], hq, d, dtype=dt) * 3, "K": normal(b, case["t"], hkv, d, dtype=dt) * 3,
             # each sequence continues at a position of its own
             "pos": torch.randint(0, 17, (b, 1), generator=g, device="cuda") + torch.arange(case["t"], device="cuda")}
        w = {"q_scale": (1 + 0.2 * normal(d, dtype=F32)).to(dt), "k_scale": (1 + 0.2 * normal(d, dtype=F32)).to(dt),
             "cos": torch.from_numpy(cos).cuda(), "sin": torch.from_numpy(sin).cuda()}
        return x, w
    tq = case["tq"]
    x = {"Q": normal(b, hq, tq, d)}
    if case["op"] == "cross":
        tk = case["tk"]
        x["K"], x["V"] = normal(b, hkv, tk, d), normal(b, hkv, tk, d)
        if case["mask"] == "count":
            x["count"] = _lengths(case, g, tk)
        elif case["mask"] == "bool":
            x["mask"] = (torch.arange(tk, device="cuda") < _lengths(case, g, tk)[:, None])[:, None, None, :].contiguous()
        elif case["mask"] == "add":
            # a distance-like bias per query row; padded keys at the type's lowest value
            bias = -normal(b, 1, tq, tk).abs()
            pad = torch.arange(tk, device="cuda") >= _lengths(case, g, tk)[:, None]
            x["mask"] = bias.masked_fill(pad[:, None, None, :], torch.finfo(F16).min)
        return x, {}
    p, s = case["p"], case["s"]
    x["prefix_k"], x["prefix_v"] = normal(1, hkv, p, d), normal(1, hkv, p, d)
    x["K"], x["V"] = normal(b, hkv, s, d), normal(b, hkv, s, d)
    if case["mask"] == "bool":
        # suffixes of different lengths; of the last `tq` tokens each sees those up to its own
        last = _lengths(case, g, s)[:, None, None] - tq + torch.arange(tq, device="cuda")[None, :, None]
        own_keys = torch.arange(s, device="cuda") <= last.clamp(min=0)
        x["mask"] = torch.cat([torch.ones(b, tq, p, dtype=torch.bool, device="cuda"), own_keys], 2)[:, None].contiguous()
    return x, {}


# ------------------------------------------------------------------ this package's form
def _graph(case, x, w):
    from emx_onnx_cgen_b200.spec import GraphSpec, NodeSpec, TensorSpec

    dt = {torch.float16: "f16", torch.float32: "f32", torch.int64: "i64", torch.bool: "bool"}
    ins = [TensorSpec(n, dt[v.dtype], tuple(v.shape)) for n, v in x.items()]
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    inits = {n: v.cpu().numpy() for n, v in w.items()}
    if case["op"] == "norm_rope":
        rope = {"interleaved": int(case["interleaved"]),
                "rotary_embedding_dim": 0 if case["rot"] == d else case["rot"]}
        nodes = []
        for n, s in (("Q", "q_scale"), ("K", "k_scale")):
            nodes += [NodeSpec("RMSNormalization", n + "_norm", (n, s), (n + "n",), {"axis": -1, "epsilon": 1e-6}),
                      NodeSpec("Transpose", n + "_heads", (n + "n",), (n + "t",), {"perm": [0, 2, 1, 3]}),
                      NodeSpec("RotaryEmbedding", n + "_rope", (n + "t", "cos", "sin", "pos"), ("Y" + n,), rope)]
        outs = [TensorSpec("YQ", case["dtype"], (b, hq, case["t"], d)),
                TensorSpec("YK", case["dtype"], (b, hkv, case["t"], d))]
    elif case["op"] == "cross":
        # inputs: Q, K, V, attn_mask, past_key, past_value, nonpad_kv_seqlen
        nodes = [NodeSpec("Attention", "cross", ("Q", "K", "V", "mask" if "mask" in x else "", "", "",
                                                 "count" if "count" in x else ""), ("Y",), {"is_causal": 0})]
        outs = [TensorSpec("Y", "f16", (b, hq, case["tq"], d))]
    else:
        inits["full"] = np.array([b, hkv, case["p"], d], np.int64)
        nodes = [NodeSpec("Expand", "share_k", ("prefix_k", "full"), ("past_k",)),
                 NodeSpec("Expand", "share_v", ("prefix_v", "full"), ("past_v",)),
                 NodeSpec("Attention", "attn", ("Q", "K", "V", "mask" if "mask" in x else "", "past_k", "past_v"),
                          ("Y",), {"is_causal": int(case["mask"] == "causal")})]
        outs = [TensorSpec("Y", "f16", (b, hq, case["tq"], d))]
    return GraphSpec(case["op"], ins, outs, nodes, inits, opset_imports=(("", 24),))


def prepare(case, seed):
    x, w = _inputs(case, seed)
    state = {"case": case, "x": x, "w": w}
    if own:
        # the loaded plan and its output buffers, which a serving program keeps
        from emx_onnx_cgen_b200.lowering import lower
        from emx_onnx_cgen_b200.plan import B200PlanEmitter
        from emx_onnx_cgen_b200.runtime import Session

        plan = B200PlanEmitter(attention_mode="flash").emit_plan(lower(_graph(case, x, w)))
        state["session"] = Session(plan, device=torch.cuda.current_device())
        dt = {"f16": F16, "f32": F32}
        state["y"] = [torch.empty(s, dtype=dt[t], device="cuda") for s, t in zip(plan.output_shapes, plan.output_dtypes)]
        state["order"] = plan.input_names
    return state


def run(state):
    if own:
        x, y = state["x"], state["y"]
        # 1 is CUDA's handle of the default stream (0 would ask for the plan's own stream)
        state["session"].run_ptrs([x[n].data_ptr() for n in state["order"]], [t.data_ptr() for t in y],
                                  stream=torch.cuda.current_stream().cuda_stream or 1)
        return y
    return {"norm_rope": _plain_norm_rope, "cross": _plain_cross, "prefix": _plain_prefix}[state["case"]["op"]](state)


# ------------------------------------------------------------------ plain forms
def _rms_rotate(x, scale, cos, sin, rot, interleaved):
    """x [B,T,H,D] -> normalised over D, axes 1 and 2 exchanged, first `rot` elements rotated; cos, sin [B,T,rot/2]."""
    f = x.float()
    y = f / torch.sqrt((f * f).mean(-1, keepdim=True) + 1e-6) * scale.float()
    y = y.transpose(1, 2)
    c, s = cos.float()[:, None], sin.float()[:, None]
    head, rest = y[..., :rot], y[..., rot:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :rot // 2], head[..., rot // 2:])
    re, im = a * c - b * s, a * s + b * c
    head = torch.stack([re, im], -1).flatten(-2) if interleaved else torch.cat([re, im], -1)
    return torch.cat([head, rest], -1).to(x.dtype)


def _plain_norm_rope(state):
    c, x, w = state["case"], state["x"], state["w"]
    cos, sin = w["cos"][x["pos"]], w["sin"][x["pos"]]
    return [_rms_rotate(x[n], w[s], cos, sin, c["rot"], c["interleaved"]) for n, s in (("Q", "q_scale"), ("K", "k_scale"))]


def _attend(q, k, v, visible, bias):
    """softmax(q k^T / sqrt(d) + bias over the visible keys) v, zero where a row sees no key; q [B,Hq,Tq,D]."""
    b, hq, tq, d = q.shape
    hkv, tk = k.shape[1], k.shape[2]
    s = torch.matmul(q.float().reshape(b, hkv, -1, d), k.float().transpose(2, 3)).reshape(b, hq, tq, tk)
    s *= 1.0 / math.sqrt(d)
    if bias is not None:
        # a row's largest bias changes nothing in its softmax; taken out, the scores keep their digits beside it
        f = bias.float()
        s += f - f.amax(-1, keepdim=True)
    if visible is not None:
        s = torch.where(visible, s, -torch.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    del s
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(b, hkv, -1, tk), v.float()).reshape(b, hq, tq, -1)
    return (o / torch.where(total == 0, 1.0, total)).to(q.dtype)


def _plain_cross(state):
    c, x = state["case"], state["x"]
    visible = bias = None
    if c["mask"] == "count":
        visible = (torch.arange(c["tk"], device="cuda") < x["count"][:, None])[:, None, None]
    elif c["mask"] == "bool":
        visible = x["mask"]
    elif c["mask"] == "add":
        bias = x["mask"]
    return [_attend(x["Q"], x["K"], x["V"], visible, bias)]


def _plain_prefix(state):
    c, x = state["case"], state["x"]
    k, v = (torch.cat([x["prefix_" + n].expand(c["b"], -1, -1, -1), x[n.upper()]], 2) for n in "kv")
    visible = None
    if c["mask"] == "bool":
        visible = x["mask"]
    elif c["mask"] == "causal":
        visible = torch.arange(c["p"] + c["s"], device="cuda") <= torch.arange(c["tq"], device="cuda")[:, None] + c["p"]
    return [_attend(x["Q"], k, v, visible, None)]


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_rotation(x, scale, cos, sin, case):
    """One head axis at a time: normalise, then multiply the pairs, as complex numbers, by cos + i sin."""
    rot, y = case["rot"], []
    turn = torch.complex(cos.double(), sin.double())
    for h in range(x.shape[2]):
        f = x[:, :, h].double()
        f = f * (f.square().sum(-1, keepdim=True) / f.shape[-1] + 1e-6).rsqrt() * scale.double()
        z = f[..., :rot].unflatten(-1, (-1, 2)) if case["interleaved"] else f[..., :rot].unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        y.append(torch.cat([z.flatten(-2), f[..., rot:]], -1))
    return torch.stack(y, 1)


def exact(case, seed):
    x, w = _inputs(case, seed)
    if case["op"] == "norm_rope":
        cos, sin = w["cos"][x["pos"]], w["sin"][x["pos"]]
        return [_exact_rotation(x["Q"], w["q_scale"], cos, sin, case), _exact_rotation(x["K"], w["k_scale"], cos, sin, case)]
    group, out = case["hq"] // case["hkv"], []
    for b in range(case["b"]):
        heads = []
        for h in range(case["hkv"]):
            k, v = x["K"][b, h].double(), x["V"][b, h].double()
            if case["op"] == "prefix":
                k, v = torch.cat([x["prefix_k"][0, h].double(), k]), torch.cat([x["prefix_v"][0, h].double(), v])
            q = x["Q"][b, h * group:(h + 1) * group].double()
            s = torch.einsum("gtd,kd->gtk", q, k) / math.sqrt(case["d"])
            if case["mask"] == "add":
                s = s + x["mask"][b, 0].double()
            elif case["mask"] == "bool":
                s = s.masked_fill(~x["mask"][b, 0], -torch.inf)
            elif case["mask"] == "count":
                s[..., int(x["count"][b]):] = -torch.inf
            elif case["mask"] == "causal":
                s = s.masked_fill(torch.ones(case["tq"], k.shape[0], dtype=torch.bool, device="cuda").triu(case["p"] + 1), -torch.inf)
            heads.append(torch.einsum("gtk,kd->gtd", torch.nan_to_num(torch.softmax(s, -1), nan=0.0), v))
        out.append(torch.cat(heads))
    return [torch.stack(out)]


# ------------------------------------------------------------------ work
def work(case):
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    if case["op"] == "norm_rope":
        e = 2 if case["dtype"] == "f16" else 4
        n = b * case["t"] * (hq + hkv) * d
        # positions, the rows of the tables that they name, both scales
        side = b * case["t"] * 8 + 2 * min(case["t"] + 17, b * case["t"]) * case["rot"] // 2 * e + 2 * d * e
        return {"bytes": 2 * n * e + side, "flops": 8 * n}
    tq = case["tq"]
    if case["op"] == "cross":
        tk = case["tk"]
        # valid lengths lie evenly between half of the states and all; an additive mask keeps every key
        keys = 0.75 * tk if case["mask"] in ("count", "bool") else tk
        kv = 2 * b * hkv * keys * d * 2
        side = {"none": 0, "count": 8 * b, "bool": b * tk, "add": 2 * b * tq * tk}[case["mask"]]
        pairs = b * hq * tq * keys
    else:
        p, s = case["p"], case["s"]
        mine = {"none": s, "bool": 0.75 * s, "causal": (s + 1) / 2}[case["mask"]]
        read = s if case["mask"] == "causal" else mine
        kv = 2 * hkv * (p + b * read) * d * 2
        side = b * tq * (p + s) if case["mask"] == "bool" else 0
        pairs = b * hq * tq * (p + mine)
    return {"bytes": kv + side + 2 * b * hq * tq * d * 2, "flops": 4 * pairs * d}
