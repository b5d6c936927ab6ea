"""Plain 64-bit implementations of the coordinator-side operators (include/m26c_coord.h) on numpy arrays, with the
error each kernel may make beside its value: counted roundings (half a step each: FP32 2^-24, BF16 2^-8, E4M3 2^-4)."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
U32, UBF16, UE4M3 = 2.0 ** -24, 2.0 ** -8, 2.0 ** -4


def bf16(x):
    """FP32 values rounded to BF16, as (bits, values)."""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    bits = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return bits, (bits.astype(np.uint32) << 16).view(np.float32)


def widen(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def join(h, planes, pre_w, post_w, gate, scale, eps):
    """(h', bound on its error, n, bound on its FP32 error). A sum of squares is a chain of at most 16 products per thread and
    27 further additions (six over a wave, up to fifteen over waves, the mean and eps), whose relative error a square root halves;
    a square root, a division and the products add under eight roundings."""
    h, pre_w = np.asarray(h, np.float64), np.asarray(pre_w, np.float64)
    z = np.sum([np.asarray(p, np.float64) for p in planes], axis=0)
    size = np.sum([np.abs(np.asarray(p, np.float64)) for p in planes], axis=0)
    norm_err = ((16 + 27) / 2 + 8) * U32
    if post_w is not None:
        k = 1 / np.sqrt(np.mean(z * z, -1, keepdims=True) + eps)
        # the planes' additions round too: relative to the row, at most their share of its norm
        row = np.sqrt(np.sum((3 * U32 * size) ** 2, -1, keepdims=True) / np.maximum(np.sum(z * z, -1, keepdims=True), 1e-300))
        row[np.mean(z * z, -1, keepdims=True) < eps] = 0
        z_err = (3 * U32 * size + np.abs(z) * (norm_err + row)) * k * np.abs(post_w)
        z = z * k * np.asarray(post_w, np.float64)
    else:
        z_err = 3 * U32 * size
    g = scale * (1.0 if gate is None else np.asarray(gate, np.float64))
    out = h + g * z
    out_err = np.abs(g) * (z_err + 3 * U32 * np.abs(z)) + U32 * np.abs(out)
    k = 1 / np.sqrt(np.mean(out * out, -1, keepdims=True) + eps)
    n = out * k * pre_w
    row = np.sqrt(np.sum(out_err ** 2, -1, keepdims=True)) / np.sqrt(np.sum(out * out, -1, keepdims=True) + eps * out.shape[-1])
    n_err = out_err * k * np.abs(pre_w) + np.abs(n) * (norm_err + row)
    return out, out_err * 1.01, n, n_err * 1.01


def w4_weights(payload, scales):
    n, half = payload.shape
    codes = np.stack([payload & 15, payload >> 4], -1).reshape(n, half * 2)
    return E2M1[codes] * np.exp2(np.repeat(scales.astype(np.float64), 32, axis=1) - 127)


def e4m3(codes):
    c = codes.astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.exp2(e - 10.0))
    v = np.where((c & 0x7F) == 0x7F, np.nan, v)
    return np.where(c & 0x80, -v, v)


def wire_values(payload, scales):
    return e4m3(payload) * np.exp2(np.repeat(scales.astype(np.float64), 32, axis=-1) - 127)


def w4_product(x, w):
    """(y, bound): products of the operands are exact, and no order of k FP32 additions is further off than k roundings of the
    sum of magnitudes (twice that where an addition inside the matrix pipe cuts instead of rounding)."""
    x = np.asarray(x, np.float64)
    return x @ w.T, 2 * (w.shape[1] + 8) * U32 * (np.abs(x) @ np.abs(w).T)


def logprobs(logits, given, top, scale):
    """Per row: given log probabilities, entropy, top ids, their log probabilities, and a bound for each of the three numbers.

    A term exp(t - m) = 2^d is off by the roundings of scale * log2 e and its constant (relative 2 |t - m| U32), of d (|t - m| U32)
    and two of the exponential; a lane adds at most vocab / 128 + 40 terms one after another (a row of more than two chunks of
    512 values is at least two waves' work), and 20 joins follow, each of which rescales by a factor that is off like a term.
    The mean of |t - m| under the distribution is what the first part amounts to in Z. A log probability is (v - m) scale - ln Z:
    two roundings of the first part, two of the second, one of the difference."""
    rows, vocab = logits.shape
    x = np.asarray(logits, np.float64)
    t = x * scale
    gl = np.full(given.shape, np.nan)
    ent, ids, lp = np.zeros(rows), np.full((rows, top), -1, np.int64), np.full((rows, top), -np.inf)
    tol_g, tol_h, tol_t = np.zeros(given.shape), np.zeros(rows), np.zeros((rows, top))
    chain = vocab / 128 + 40 + 20
    for r in range(rows):
        row = t[r]
        numbers = np.where(np.isnan(row), -np.inf, row)
        order = np.lexsort((np.arange(vocab), -np.where(np.isnan(x[r]), -np.inf, x[r])))[:top]
        kept = order[numbers[order] > -np.inf]
        ids[r, :kept.size] = kept
        inside = (given[r] >= 0) & (given[r] < vocab)
        if np.isnan(row).any() or np.isposinf(row).any():
            ent[r] = np.nan
            lp[r, :kept.size] = np.nan
            continue
        m = row.max()
        if m == -np.inf:
            gl[r, inside] = -np.inf
            continue
        d = row - m
        e = np.exp(d)
        z = e.sum()
        p = e / z
        mean = -np.sum(np.where(p > 0, p * np.where(np.isfinite(d), d, 0), 0))
        lnz = np.log(z)
        z_err = (chain + 4 + 4 * mean) * U32
        logp = d - lnz
        ent[r] = lnz + mean
        spread = np.sum(np.where(p > 0, p * np.where(np.isfinite(d), d, 0) ** 2, 0))
        tol_h[r] = z_err * (1 + mean) + (chain + 8) * U32 * mean + 4 * spread * U32 + 6 * U32 * (lnz + mean)
        gl[r, inside] = logp[given[r, inside]]
        lp[r, :kept.size] = logp[kept]

        def bound(v):
            with np.errstate(invalid="ignore"):
                b = z_err + U32 * (3 * np.abs(v + lnz) + 2 * lnz + 3 * np.abs(v))
            return np.where(np.isfinite(v), b, 0)
        tol_g[r] = bound(np.where(inside, gl[r], 0))
        tol_t[r] = bound(lp[r])
    return gl, ent, ids, lp, tol_g * 1.05, tol_h * 1.05, tol_t * 1.05
