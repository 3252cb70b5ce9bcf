"""The decoder operators in float64, straight from their definitions: the
plain implementation that the tests of norm_rope.cu and attention_flash.cu
compare with, and the error bounds that those kernels' roundings imply."""
import numpy as np

HALF = {"f16": 2.0 ** -11, "f32": 2.0 ** -24}   # half a step of the output type, relative
TINY = {"f16": 2.0 ** -25, "f32": 2.0 ** -150}  # half the smallest subnormal


def rms_norm(x, scale, eps, axes=1):
    x = x.astype(np.float64)
    ax = tuple(range(x.ndim - axes, x.ndim))
    return x / np.sqrt((x * x).mean(axis=ax, keepdims=True) + eps) * scale.astype(np.float64)


def rotate(x, cos, sin, rot, interleaved):
    """x [B,T,H,D]; cos, sin [B,T,rot/2] -> (rotated, |a c| + |b s| magnitudes)."""
    x = x.astype(np.float64).copy()
    c, s = cos.astype(np.float64)[:, :, None], sin.astype(np.float64)[:, :, None]
    a = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    b = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    xa, xb = x[..., a].copy(), x[..., b].copy()
    mag = np.abs(x)
    x[..., a], x[..., b] = xa * c - xb * s, xa * s + xb * c
    mag[..., a] = np.abs(xa * c) + np.abs(xb * s)
    mag[..., b] = np.abs(xa * s) + np.abs(xb * c)
    return x, mag


def norm_rope(wl, x):
    """{"YQ": (value, bound), "YK": ...} of a norm_rope workload.  The bound: one
    rounding of the result, and 40 fp32 roundings of the magnitudes that meet
    in it (the row sum's chain, square root, division, two products, the
    rotation's products and sum)."""
    p, g = wl.params, wl.graph
    dt = g.tensor("Q").dtype
    if p["positions"] == "ids":
        cos, sin = (g.initializers[n][x["pos"]] for n in ("cos", "sin"))
    else:
        cos, sin = x["cos"], x["sin"]
    out = {}
    for n in ("Q", "K"):
        v = x[n].transpose(0, 2, 1, 3) if p["layout"] == "heads" else x[n]
        v = rms_norm(v, g.initializers[n.lower() + "_scale"], p["eps"]) if p["norm"] else v
        y, mag = rotate(v, cos, sin, p["rot"], p["interleaved"])
        tol = HALF[dt] * np.abs(y) + TINY[dt] + 40 * 2.0 ** -24 * mag
        if p["layout"] == "flat":
            shape = g.tensor(f"Y{n}").shape
            out[f"Y{n}"] = (y.reshape(shape), tol.reshape(shape))
        else:
            out[f"Y{n}"] = (y.transpose(0, 2, 1, 3), tol.transpose(0, 2, 1, 3))
    return out


def attention(q, k, v, scale, mask=None, counts=None, past=0, causal=False):
    """q [B,Hq,Tq,D], k [B,Hkv,T,D], v [B,Hkv,T,Dv] (past keys first) -> (value,
    bound).  A row that sees no key gives 0.  The bound, per element: half an
    fp16 step of the result; half an fp16 step of every weight in numerator
    and denominator (2 x 2^-11 of sum w |v|; weights below the normal range
    lose up to 2^-25 of the largest each); and the fp32 score's error, D
    roundings of scale sum |q k| plus 4 of the exponent's size, in every weight."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    b, hq, tq, d = q.shape
    hkv, t = k.shape[1:3]
    k, v = (np.repeat(a, hq // hkv, axis=1) for a in (k, v))
    s = np.einsum("bhqd,bhkd->bhqk", q, k) * scale
    mag = np.einsum("bhqd,bhkd->bhqk", np.abs(q), np.abs(k)) * abs(scale)
    see = np.ones(s.shape, bool)
    if causal:
        see &= np.arange(t)[None, :] <= np.arange(tq)[:, None] + past
    if counts is not None:
        see &= (np.arange(t) < counts[:, None])[:, None, None]
    if mask is not None:
        m = mask.reshape((1,) * (4 - mask.ndim) + mask.shape)
        if m.dtype == np.bool_:
            m = np.concatenate([m, np.zeros((*m.shape[:3], t - m.shape[3]), bool)], 3)
            see &= m
        else:
            m = np.concatenate([m.astype(np.float64), np.full((*m.shape[:3], t - m.shape[3]), -np.inf)], 3)
            see &= m != -np.inf
            s = s + np.where(np.isinf(m), 0.0, m)
    s = np.where(see, s, -np.inf)
    top = s.max(axis=-1, keepdims=True)
    w = np.where(see, np.exp(s - np.where(np.isinf(top), 0.0, top)), 0.0)
    total = w.sum(axis=-1, keepdims=True)
    w = w / np.where(total == 0, 1.0, total)
    y = np.einsum("bhqk,bhkd->bhqd", w, v)
    wv = np.einsum("bhqk,bhkd->bhqd", w, np.abs(v))
    worst = np.where(see, d * mag + 4 * np.abs(s - np.where(np.isinf(top), 0.0, top)), 0.0)
    worst = np.where(w > 2.0 ** -30, worst, 0.0).max(axis=-1, keepdims=True) * 2.0 ** -24
    tol = 2.0 ** -11 * np.abs(y) + 2.0 ** -25 + (2.0 ** -10 + 2 * worst) * wv + t * 2.0 ** -25 * np.abs(v).max()
    return y, np.where(total == 0, 0.0, tol)


def decoder_attention(wl, x):
    """(value, bound) of a decoder_attention workload, in the output's layout."""
    p = wl.params

    def heads(a, h):
        return a if p["rank"] == 4 else a.reshape(*a.shape[:2], h, -1).transpose(0, 2, 1, 3)

    q, k, v = heads(x["Q"], p["q_heads"]), heads(x["K"], p["kv_heads"]), heads(x["V"], p["kv_heads"])
    if p["past"]:
        pk, pv = (np.broadcast_to(x[n], (p["batch"], *x[n].shape[1:])) for n in ("PK", "PV"))
        k, v = np.concatenate([pk, k], 2), np.concatenate([pv, v], 2)
    y, tol = attention(q, k, v, p["scale"], x.get("mask"), x.get("count"), p["past"], p["causal"])
    if p["rank"] == 3:
        y, tol = (a.transpose(0, 2, 1, 3).reshape(p["batch"], p["q_seq"], -1) for a in (y, tol))
    return y, tol


def check(got, want, tol, what=""):
    got = got.astype(np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} outside the bound; first at {i}: got {got[i]}, "
                             f"value {want[i]}, bound {tol[i]}")
