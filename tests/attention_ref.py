"""Plain 64-bit restatements of the operators around attention, with what a 32-bit (and f16) computation may be off by."""
import numpy as np

U32, HALF = 2.0 ** -24, {np.dtype(np.float16): 2.0 ** -11, np.dtype(np.float32): 2.0 ** -24}   # half a step, relative


def norm_rope(x, w, cos, sin, eps):
    """(result, bound) of one tensor [B, H, n, D].  The bound: the f32 sum of D squares is off by at most D / 16 + 16 roundings in
    a row (partial sums of 16 lanes at least), the root halves that and adds two, products and the sum a few more on the two
    terms' sizes; then half a step of the type, and its smallest step where results are subnormal."""
    xd = x.astype(np.float64)
    y = xd / np.sqrt((xd * xd).mean(axis=-1, keepdims=True) + eps) * (1.0 if w is None else w.astype(np.float64))
    half = x.shape[-1] // 2
    z = np.concatenate([-y[..., half:], y[..., :half]], axis=-1)
    a, b = y * cos.astype(np.float64), z * sin.astype(np.float64)
    out = a + b
    bound = HALF[x.dtype] * np.abs(out) + (x.shape[-1] / 16 + 24) * U32 * (np.abs(a) + np.abs(b)) + 2.0 ** -25
    return out, bound


def attend(q, keys, values, dtype, scale=None, cap=0.0, bias=None, sees=None):
    """(result, bound) of q [n, D] over keys and values [T, D] in 64 bits.

    The bound, per element, with A = sum_j w_j |v_j|: a score of D products is off by at most D + 8 half steps of 32 bits
    on the sum of the products' sizes, and by a few on its own size (scale, change of base, difference from the maximum);
    the cap only shrinks that but has an error of its own of at most 4e-7 of the cap (caps of up to 512) or of the score.  e^ds - 1 <= 2 ds counts twice,
    for the weight and for the sum it is divided by.  f16: a weight is rounded to f16 before the product with V (half a
    step in the numerator; the sum is over the same values or not: another).  Sums of T terms in f32: T half steps at
    most, numerator and sum.  Then half a step of the result's type."""
    q, keys, values = (t.astype(np.float64) for t in (q, keys, values))
    d, t = q.shape[1], keys.shape[0]
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    if t == 0:
        return np.zeros((q.shape[0], values.shape[1])), np.full((q.shape[0], values.shape[1]), 1e-30)
    sees = np.ones((q.shape[0], t), bool) if sees is None else sees
    safe_k = np.where(np.isfinite(keys), keys, 0.0)
    safe_v = np.where(np.isfinite(values), values, 0.0)
    s = q @ safe_k.T * scale
    ds = (d + 8) * U32 * (np.abs(q) @ np.abs(safe_k).T) * abs(scale)
    if cap:
        s = cap * np.tanh(s / cap)
        ds = ds + 4e-7 * (cap if cap <= 512 else np.abs(s))
    if bias is not None:
        s = s + bias
        ds = ds + 2 * U32 * np.abs(bias)
    ds = ds + 4 * U32 * np.abs(s)
    s = np.where(sees, s, -np.inf)
    top = s.max(axis=1, keepdims=True)
    top = np.where(np.isneginf(top), 0.0, top)
    ds = ds + 4 * U32 * np.abs(top)
    e = np.exp(s - top)
    total = e.sum(axis=1, keepdims=True)
    w = e / np.where(total == 0, 1.0, total)
    out, size = w @ safe_v, w @ np.abs(safe_v)
    worst = np.where(sees, ds, 0.0).max(axis=1, keepdims=True)
    off = 4 * worst + 2 * (t + 16) * U32
    if dtype == np.float16:
        off = off + 2 * HALF[np.dtype(np.float16)]
    return out, HALF[np.dtype(dtype)] * np.abs(out) + off * size + 2.0 ** -24


def assert_within(got, want, bound, what=""):
    got = np.asarray(got).astype(np.float64)
    assert np.isfinite(got).all(), f"{what}: not finite"
    far = np.abs(got - want) / bound
    at = np.unravel_index(far.argmax(), far.shape) if far.size else None
    assert not far.size or far.max() <= 1.0, f"{what}: {got[at]} against {want[at]} at {at}: {far.max():.3g} times the bound {bound[at]:.3g}"


def scored(q, k, v, scale=None, cap=0.0, slopes=None, documents=None, prefix_lens=None, causal=True):
    """(result, bound) of ScoredSdpa on [B, H, n, D] tensors."""
    b_, hq, n, _ = q.shape
    hkv, t = k.shape[1:3]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    at, j = np.arange(n)[:, None] + t - n, np.arange(t)[None, :]
    for b in range(b_):
        sees = (j <= at) if causal else np.ones((n, t), bool)
        if causal and prefix_lens is not None:
            sees = sees | (j < prefix_lens[b])
        if documents is not None:
            ids = documents[b]
            sees = sees & (ids[None, :] == ids[t - n :, None]) & (ids >= 0)[None, :]
        for h in range(hq):
            bias = None if slopes is None else -np.float64(slopes[h]) * np.abs(at - j)
            out[b, h], bound[b, h] = attend(q[b, h], k[b, h * hkv // hq], v[b, h * hkv // hq], q.dtype, scale, cap, bias, sees)
    return out, bound


def shared(q, pk, pv, ks, vs, scale=None, causal=True):
    """(result, bound) of attention over a prefix [Hkv, P, D] and each sequence's own rows ks[i], vs[i] [Hkv, len, D]."""
    n, hq, sq, _ = q.shape
    hkv, p = pk.shape[:2]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        own = ks[i].shape[1]
        sees = np.ones((sq, p + own), bool)
        if causal:
            sees[:, p:] = np.arange(own)[None, :] <= np.arange(sq)[:, None] + own - sq
        for h in range(hq):
            g = h * hkv // hq
            out[i, h], bound[i, h] = attend(q[i, h], np.concatenate([pk[g], ks[i][g]]), np.concatenate([pv[g], vs[i][g]]), q.dtype, scale, sees=sees)
    return out, bound
