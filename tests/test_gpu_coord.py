"""GPU parity of the coordinator-side operators (include/m26c_coord.h) against their plain 64-bit forms
(tests/coord_reference.py), through the C ABI. Selections, codes and copies are exact; numbers stay within counted roundings."""
import ctypes as C

import numpy as np
import pytest

import b1_oracle as O
import coord_reference as R
from mimo26f_afd_amd import b1, coord, glue, synth

pytestmark = pytest.mark.gpu


def dev(a):
    return b1.DeviceBuffer.from_host(np.ascontiguousarray(a))


def room(nbytes, fill=0x5A):
    return dev(np.full(max(int(nbytes), 1), fill, np.uint8))


# ---- block join ----------------------------------------------------------------------------------------

def join_inputs(rows, cols, planes, post, gate, seed):
    rng = np.random.default_rng(seed)
    h = (rng.standard_normal((rows, cols)) * np.where(rng.random(cols) < 0.01, 20, 1)).astype(np.float32)
    p = [R.bf16((rng.standard_normal((rows, cols)) * 0.3).astype(np.float32)) for _ in range(planes)]
    pre = (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    pw = (0.5 + 0.1 * rng.standard_normal(cols)).astype(np.float32) if post else None
    shape = {"none": None, "row": (rows, 1), "column": (1, cols), "full": (rows, cols)}[gate]
    g = rng.random(shape).astype(np.float32) if shape else None
    return h, p, pre, pw, g


def run_join(h, planes, pre, pw, gate, scale, eps, kind, wire=True, norm=True, in_place=False, shift=0, pad=0):
    """Outputs as arrays. `shift`: elements by which every array misses its 16-byte boundary; `pad`: elements between rows, checked to
    stay as they were."""
    rows, cols = h.shape

    def laid(a, extra=0):
        size = a.dtype.itemsize
        flat = np.zeros(shift + rows * (cols + pad) + 8, a.dtype)
        view = flat[shift:shift + rows * (cols + pad)].reshape(rows, cols + pad)
        view[:, :cols] = a
        buf = dev(flat)
        return buf, buf.ptr + shift * size

    hb, hp = laid(h)
    pb = [laid(bits) for bits, _ in planes]
    wb = [dev(np.concatenate([np.zeros(shift, np.float32), w])) if w is not None else None for w in (pre, pw)]
    wp = [w.ptr + 4 * shift if w else None for w in wb]
    gate_cols, gate_pitch = {"none": (0, 0), "row": (1, 1), "column": (cols, 0), "full": (cols, cols)}[kind]
    gb = dev(np.concatenate([np.zeros(shift, np.float32), gate.reshape(-1)])) if gate is not None else None
    pitch = cols + pad
    ob = hb if in_place else room((shift + rows * pitch + 8) * 4)
    nb = room((shift + rows * pitch + 8) * 2) if norm else None
    wire_pitch = (cols + cols // 32 + 7) // 8 * 8 + 8 * (pad > 0) + (1 if shift else 0)
    fb = room(rows * wire_pitch + 64) if wire else None
    plan = coord.Join(cols, wp[0], post_weight=wp[1], planes=len(planes), gate_cols=gate_cols, gate_pitch=gate_pitch, scale=scale, eps=eps,
                      plane_pitch=pitch, h_pitch=pitch, norm_pitch=pitch, payload_pitch=wire_pitch, scales_pitch=wire_pitch)
    plan(rows, hp, [q for _, q in pb], hp if in_place else ob.ptr + 4 * shift, norm=nb.ptr + 2 * shift if norm else None,
         gate=gb.ptr + 4 * shift if gb else None, payload=fb.ptr if wire else None, scales=fb.ptr + cols if wire else None)
    out = {}

    def back(buf, dtype, keep):
        flat = buf.to_host(dtype)
        view = flat[shift:shift + rows * pitch].reshape(rows, pitch)
        if not keep:
            gap = np.full(4, 0x5A, np.uint8).view(np.uint16 if dtype == np.uint16 else np.uint32)[0]
            assert (view[:, cols:].view(gap.dtype) == gap).all(), "written between rows"
        return view[:, :cols]
    out["h"] = back(ob, np.float32, in_place)
    if norm:
        out["norm"] = back(nb, np.uint16, False)
    if wire:
        raw = fb.to_host(np.uint8)[:rows * wire_pitch].reshape(rows, wire_pitch)
        out["payload"], out["scales"] = raw[:, :cols], raw[:, cols:cols + cols // 32]
        assert (raw[:, cols + cols // 32:] == 0x5A).all()
    return out


def check_join(got, h, planes, pre, pw, gate, scale, eps):
    with np.errstate(all="ignore"):
        want, tol, n, n_tol = R.join(h, [v for _, v in planes], pre, pw, gate, scale, eps)
    assert np.all(np.abs(got["h"] - want) <= tol), np.max(np.abs(got["h"] - want) / tol)
    if "norm" in got:
        err = np.abs(R.widen(got["norm"]) - n)
        lim = n_tol + R.UBF16 * (np.abs(n) + n_tol) + 2.0 ** -134
        assert np.all(err <= lim), np.max(err / lim)
    if "payload" in got:
        rows, cols = h.shape
        blocks = lambda a: a.reshape(rows, cols // 32, 32)  # noqa: E731
        amax, slack = blocks(np.abs(n)).max(-1), blocks(n_tol).max(-1)
        scale_of = lambda a: np.clip(np.ceil(np.log2(np.maximum(a, 1e-300) / 448)) + 127, 0, 254)  # noqa: E731
        assert np.all((got["scales"] >= scale_of(amax - slack)) & (got["scales"] <= scale_of(amax + slack)))
        step = np.exp2(got["scales"].astype(np.float64) - 127)[..., None]
        value = blocks(R.wire_values(got["payload"], got["scales"]))
        mag = np.minimum(blocks(np.abs(n)), 448 * step)
        lim = blocks(n_tol) + np.maximum(R.UE4M3 * (mag + blocks(n_tol)), 2.0 ** -10 * step)
        assert np.all(np.abs(value - blocks(n)) <= lim), np.max(np.abs(value - blocks(n)) / lim)


@pytest.mark.parametrize("rows,cols,planes,post,gate", [
    (1, 4096, 1, False, "none"), (3, 4096, 4, True, "column"), (130, 4096, 2, True, "row"), (2, 32, 3, True, "full"), (5, 64, 1, False, "row"),
    (7, 2080, 4, True, "full"), (3, 8192, 1, True, "column"), (2, 8224, 2, False, "full"), (2, 16384, 4, True, "full"), (1, 96, 1, True, "none")])
@pytest.mark.parametrize("shift,pad", [(0, 0), (0, 8), (1, 3)])
def test_join_within_counted_roundings(rows, cols, planes, post, gate, shift, pad):
    args = join_inputs(rows, cols, planes, post, gate, rows * 7 + cols)
    check_join(run_join(*args, 0.75, 1e-5, gate, shift=shift, pad=pad), *args, 0.75, 1e-5)


@pytest.mark.parametrize("rows,cols,planes,post,gate", [(1, 1, 1, True, "none"), (4, 3, 2, True, "full"), (9, 31, 1, False, "column"), (5, 2047, 4, True, "row"),
                                                        (2, 4099, 2, True, "full"), (2, 9001, 1, True, "column"), (1, 16383, 3, True, "full")])
def test_join_odd_rows(rows, cols, planes, post, gate):
    args = join_inputs(rows, cols, planes, post, gate, rows * 5 + cols)
    check_join(run_join(*args, -1.5, 1e-6, gate, wire=False), *args, -1.5, 1e-6)
    check_join(run_join(*args, -1.5, 1e-6, gate, wire=False, in_place=True, pad=5), *args, -1.5, 1e-6)


def test_join_in_place_and_each_output_alone_give_the_same_bits():
    args = join_inputs(33, 4096, 2, True, "column", 4)
    whole = run_join(*args, 0.5, 1e-5, "column")
    again = run_join(*args, 0.5, 1e-5, "column", in_place=True)
    for k in whole:
        assert np.array_equal(whole[k].view(np.uint8), again[k].view(np.uint8)), k
    only = run_join(*args, 0.5, 1e-5, "column", wire=False)
    assert np.array_equal(only["norm"], whole["norm"]) and np.array_equal(only["h"].view(np.uint32), whole["h"].view(np.uint32))
    only = run_join(*args, 0.5, 1e-5, "column", norm=False)
    assert np.array_equal(only["payload"], whole["payload"]) and np.array_equal(only["scales"], whole["scales"])
    # each row by itself: a row's bits do not depend on its neighbours
    h, planes, pre, pw, g = args
    one = run_join(h[7:8], [(b[7:8], v[7:8]) for b, v in planes], pre, pw, g, 0.5, 1e-5, "column")
    for k in whole:
        assert np.array_equal(whole[k][7:8].view(np.uint8), one[k].view(np.uint8)), k


@pytest.mark.parametrize("shift", [0, 1])
def test_join_codes_and_casts_are_exact_where_the_norm_is(shift):
    """Rows whose mean square plus eps is exactly one (three in four values +-1, the rest 0, eps a quarter) leave the norm the
    weight itself up to sign, so the weights carry every exponent and tie through the BF16 and wire roundings: the checker's bits."""
    rng = np.random.default_rng(8)
    rows, cols = 6, 4096
    h = np.where(np.arange(cols) % 4 == 3, 0.0, np.where(rng.random((rows, cols)) < 0.5, 1.0, -1.0)).astype(np.float32)
    h = rng.permuted(h, axis=1)
    zero = [(np.zeros((rows, cols), np.uint16), np.zeros((rows, cols), np.float32))]
    w = synth.bf16_round((rng.standard_normal(cols) * np.exp2(rng.integers(-30, 30, cols))).astype(np.float32))
    w[:64] = np.ldexp(1.0, -10) * np.arange(64)
    w[64:96] = np.linspace(-480, 480, 32)
    w[96:128] = np.ldexp(np.arange(32, dtype=np.float32) + 0.5, -3)
    w[128:160] = 1e-45
    w[160:192] = 3.0e38
    got = run_join(h, zero, w, None, None, 1.0, 0.25, "none", shift=shift)
    n = (h * w).astype(np.float32)
    assert np.array_equal(got["h"], h)
    assert np.array_equal(got["norm"], O.bf16_rne_nan(n.reshape(-1)).reshape(rows, cols))
    p, s = O.q0_quantize(n)
    assert np.array_equal(got["scales"], s) and np.array_equal(got["payload"], p)


def test_join_keeps_a_bad_row_to_itself_and_a_zero_row_at_zero():
    args = join_inputs(5, 4096, 1, True, "none", 3)
    h, planes, pre, pw, _ = args
    h[1, 17] = np.nan
    h[2, 5] = np.inf
    h[3] = 0
    planes[0][0][3] = 0
    planes[0][1][3] = 0
    got = run_join(h, planes, pre, pw, None, 1.0, 1e-5, "none")
    check = [0, 4]
    check_join({k: v[check] for k, v in got.items()}, h[check], [(b[check], v[check]) for b, v in planes], pre, pw, None, 1.0, 1e-5)
    assert np.isnan(R.widen(got["norm"][1])).all() and (got["payload"][1] == 0).all()
    assert np.isnan(R.widen(got["norm"][2])[5])
    assert (got["h"][3] == 0).all() and (R.widen(got["norm"][3]) == 0).all() and (R.wire_values(got["payload"][3], got["scales"][3]) == 0).all()


@pytest.mark.parametrize("cols", [9, 2047, 4097, 12001])
def test_join_infinite_gate_stays_at_its_column_on_odd_rows(cols):
    """A column next to the row's end: an infinite h' there makes the norm's factor zero, the other columns' n zero and its own NaN."""
    h, planes, pre, pw, gate = join_inputs(3, cols, 2, True, "column", cols)
    at = cols - cols % 8 - 1
    gate[0, at] = np.inf
    got = run_join(h, planes, pre, pw, gate, 1.0, 1e-5, "column", wire=False)
    rest = np.arange(cols) != at
    assert np.isinf(got["h"][:, at]).all() and np.isfinite(got["h"][:, rest]).all()
    n = R.widen(got["norm"])
    assert np.isnan(n[:, at]).all() and (n[:, rest] == 0).all()


@pytest.mark.parametrize("rows,cols,planes,post,gate", [(600, 2050, 4, True, "full"), (515, 5001, 3, True, "row"), (513, 9999, 4, False, "column"),
                                                        (520, 4160, 2, True, "full")])
def test_join_many_longer_rows(rows, cols, planes, post, gate):
    args = join_inputs(rows, cols, planes, post, gate, cols)
    wire = cols % 32 == 0
    check_join(run_join(*args, 0.5, 1e-5, gate, wire=wire), *args, 0.5, 1e-5)
    check_join(run_join(*args, 0.5, 1e-5, gate, wire=wire, in_place=True, shift=3), *args, 0.5, 1e-5)


def test_join_many_rows_walk_the_grid():
    """More rows than workgroups in a launch; small rows keep it quick."""
    args = join_inputs(70001, 32, 1, True, "row", 5)
    check_join(run_join(*args, 1.0, 1e-5, "row"), *args, 1.0, 1e-5)


# ---- products with MXFP4 weights ---------------------------------------------------------------------------

def w4_inputs(n, k, seed, low=110, high=124):
    rng = np.random.default_rng(seed)
    payload = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    scales = rng.integers(low, high, (n, k // 32), dtype=np.uint8)
    return rng, payload, scales


def weights_of(payload, scales):
    p, s = dev(payload), dev(scales)                                  # freed on return: the handle holds its own copy
    return coord.Weights4(p.ptr, s.ptr, payload.shape[0], payload.shape[1] * 2)


def run_w4(weights, x, rows, fp8=None, bf16_out=False, x_pad=0, y_pad=0):
    n, k = weights.n, weights.k
    size = 2 if bf16_out else 4
    y = room((rows * (n + y_pad) + 4) * size)
    if fp8 is None:
        xb = np.full((rows, k + x_pad), 0x7FC0, np.uint16)          # NaN between the rows: not to be read as values
        xb[:, :k] = x
        xd = dev(xb)
        weights.matvec(xd.ptr, rows, y.ptr, bf16_out, x_pitch=k + x_pad, y_pitch=n + y_pad)
    else:
        payload, scales = fp8
        pitch = (k + k // 32 + 7) // 8 * 8 + x_pad
        frame = np.full((rows, pitch), 0x7F, np.uint8)
        frame[:, :k], frame[:, k:k + k // 32] = payload, scales
        xd = dev(frame)
        weights.matvec_fp8(xd.ptr, xd.ptr + k, rows, y.ptr, bf16_out, payload_pitch=pitch, scales_pitch=pitch, y_pitch=n + y_pad)
    raw = y.to_host(np.uint16 if bf16_out else np.uint32)
    assert (raw[rows * (n + y_pad):].view(np.uint8) == 0x5A).all()
    raw = raw[:rows * (n + y_pad)].reshape(rows, n + y_pad)
    assert (np.ascontiguousarray(raw[:, n:]).view(np.uint8) == 0x5A).all(), "written between rows"
    return R.widen(raw[:, :n]) if bf16_out else np.ascontiguousarray(raw[:, :n]).view(np.float32)


SHAPES = [(1, 1, 32), (1, 16, 64), (3, 17, 96), (16, 256, 4096), (17, 100, 128), (5, 1000, 2080), (33, 48, 160), (64, 130, 512), (65, 40, 544), (130, 31, 1024),
          (1, 4096, 4096), (2, 5, 16384), (48, 4099, 608), (16, 33000, 256),
          # every form of the rule on sizes: steps of 128 up to 8, 16, 24, 32, 48, 64 and more, in runs of 16 and 32 rows, tiles past one turn
          (3, 13000, 1056), (16, 12500, 2080), (9, 12400, 3200), (7, 12400, 4128), (5, 12330, 6176), (2, 12330, 8224), (33, 8200, 96), (29, 13000, 1056),
          (64, 8200, 2080), (50, 4200, 3200), (64, 4200, 4128), (300, 200, 640), (2, 40, 16416), (33, 3104, 16416), (1, 1, 64), (3, 7, 96), (16, 16500, 2080), (3, 16500, 1056)]


@pytest.mark.parametrize("rows,n,k", SHAPES)
@pytest.mark.parametrize("form", ["bf16", "fp8"])
def test_w4_product_within_counted_roundings(rows, n, k, form):
    rng, payload, scales = w4_inputs(n, k, rows + n + k)
    weights = weights_of(payload, scales)
    w = R.w4_weights(payload, scales)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    if form == "bf16":
        bits, value = R.bf16(x)
        run = lambda **kw: run_w4(weights, bits, rows, **kw)  # noqa: E731
    else:
        wire = O.q0_quantize(x)
        value = R.wire_values(*wire)
        run = lambda **kw: run_w4(weights, None, rows, fp8=wire, **kw)  # noqa: E731
    want, tol = R.w4_product(value, w)
    got = run()
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)
    padded = run(x_pad=8, y_pad=3)
    assert np.array_equal(padded.view(np.uint32), got.view(np.uint32))
    half = run(bf16_out=True)
    assert np.array_equal(half, R.bf16(got)[1])


@pytest.mark.parametrize("rows,n,k", [(3, 12400, 12320), (16, 12301, 16384), (3, 16500, 8224), (40, 70001, 8224), (17, 13000, 8224)])
@pytest.mark.parametrize("form", ["bf16", "fp8"])
def test_w4_wide_rows_in_phases(rows, n, k, form):
    """x too wide for the registers over many columns, and more tiles than a workgroup keeps sums for; the reference takes every 61st
    column and the last ones; with a single one in each row of weights every column is pinned."""
    rng, payload, scales = w4_inputs(n, k, rows + n)
    weights = weights_of(payload, scales)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    if form == "bf16":
        bits, value = R.bf16(x)
        got = run_w4(weights, bits, rows, y_pad=5)
    else:
        wire = O.q0_quantize(x)
        value = R.wire_values(*wire)
        got = run_w4(weights, None, rows, fp8=wire, y_pad=5)
    some = np.unique(np.r_[0:n:61, n - 20:n])
    want, tol = R.w4_product(value, R.w4_weights(payload[some], scales[some]))
    assert np.all(np.abs(got[:, some] - want) <= tol), np.max(np.abs(got[:, some] - want) / tol)
    # one in each row of weights, at a place that depends on the column: y names x's value there
    weights.close()
    place = (np.arange(n) * 7919) % k
    payload = np.zeros((n, k // 2), np.uint8)
    payload[np.arange(n), place // 2] = 2 << (4 * (place % 2))
    weights = weights_of(payload, np.full((n, k // 32), 127, np.uint8))
    got = run_w4(weights, bits, rows) if form == "bf16" else run_w4(weights, None, rows, fp8=wire)
    assert np.array_equal(got, value[:, place].astype(np.float32))


def test_w4_product_is_exact_on_small_integers():
    """Weights that are multiples of a half up to six and integers up to eight keep every partial sum a multiple of a half below
    2^23: any order of additions is exact, so every code, position and lane is pinned bit for bit. Weight rows and x rows are
    also ones at single places, which names the place."""
    rng, payload, _ = w4_inputs(300, 1056, 9)
    scales = np.full((300, 33), 127, np.uint8)
    payload[:264] = 0
    for j in range(264):                                              # row j: one nonzero code, at its own k
        k = 4 * j + 1
        payload[j, k // 2] = (1 + j % 15) << (4 * (k & 1))
    weights = weights_of(payload, scales)
    x = rng.integers(-8, 9, (20, 1056)).astype(np.float32)
    got = run_w4(weights, R.bf16(x)[0], 20)
    assert np.array_equal(got, (x.astype(np.float64) @ R.w4_weights(payload, scales).T).astype(np.float32))
    eye = np.zeros((33, 1056), np.float32)
    eye[np.arange(33), np.arange(33) * 32 + 7] = 1
    got = run_w4(weights, R.bf16(eye)[0], 33)
    assert np.array_equal(got, (eye.astype(np.float64) @ R.w4_weights(payload, scales).T).astype(np.float32))


# one shape or more for each form of the rule on sizes: streamed by one step and by two, resident in every number of steps and
# waves, 16 and 32 rows a run, several runs, in phases of three and of four steps a wave, the last phase partly empty
EXACT = [(20, 300, 1056), (16, 256, 4096), (40, 300, 12320), (16, 16500, 1024), (16, 16500, 2048), (13, 16400, 2080), (16, 9001, 4096), (9, 8300, 5152),
         (16, 8300, 6176), (16, 17003, 8224), (5, 17003, 9248), (16, 12301, 12320), (33, 8200, 992), (64, 8200, 2048), (64, 8200, 4096), (100, 4200, 2944),
         (64, 8300, 12320), (33, 17000, 8224)]


@pytest.mark.parametrize("rows,n,k", EXACT)
@pytest.mark.parametrize("form", ["bf16", "fp8"])
def test_w4_sums_are_exact_on_small_numbers(rows, n, k, form):
    """Weights are multiples of 1/4 up to 12 and values multiples of 1/2 up to 8, so that a sum over k is a multiple of 1/8 of at most 96 k, which
    is under 2^24 of them for k up to 21845: any order of FP32 additions is exact, and sums held in anything less are not."""
    assert 96 * k * 8 < 1 << 24
    period = min(n, 1021)                                             # weight rows repeat after a prime number of them: no whole tiles
    rng, payload, _ = w4_inputs(period, k, rows + n + k)
    scales = rng.integers(126, 129, (period, k // 32), dtype=np.uint8)
    again = np.arange(n) % period
    weights = weights_of(payload[again], scales[again])
    integers = rng.integers(-4, 5, (rows, k))
    s = rng.integers(126, 129, (rows, k // 32), dtype=np.uint8)
    value = (integers * np.exp2(np.repeat(s, 32, 1).astype(np.float64) - 127)).astype(np.float32)
    if form == "bf16":
        got = run_w4(weights, R.bf16(value)[0], rows)
    else:
        code = np.array([0, 0x38, 0x40, 0x44, 0x48], np.uint8)         # E4M3 of 0..4
        p = code[np.abs(integers)] | np.where(integers < 0, 0x80, 0).astype(np.uint8)
        assert np.array_equal(R.wire_values(p, s), value)
        got = run_w4(weights, None, rows, fp8=(p, s))
    want = value.astype(np.float64) @ R.w4_weights(payload, scales).T
    assert np.array_equal(got, want[:, again]), np.argwhere(got != want[:, again])[:4]


def test_w4_scale_bytes_every_one_accepted_or_refused():
    """Scale bytes 2..252 over nonzero codes are exact single products, groups of zeros carry any byte, and any other byte over a
    nonzero code is refused (code 3)."""
    ok = np.arange(2, 253, dtype=np.uint8)
    n, k = ok.size, 64
    payload = np.zeros((n, k // 2), np.uint8)
    payload[:, 3] = np.arange(n) % 15 + 1                             # one code at k = 6
    scales = np.stack([ok, np.resize(np.array([0, 255, 1, 254], np.uint8), n)], 1)
    weights = weights_of(payload, scales)
    for x6 in (1.0, -2.0 ** -40, 2.0 ** 60):
        x = np.zeros((2, k), np.float32)
        x[1, 6] = x6
        with np.errstate(over="ignore"):
            want = (R.E2M1[payload[:, 3] & 15] * np.exp2(ok.astype(np.float64) - 127) * x6)
            got = run_w4(weights, R.bf16(x)[0], 2)
            small = np.abs(want) < 2.0 ** -126                        # subnormal results may flush
            assert np.array_equal(got[1][~small], want.astype(np.float32)[~small]) and (got[0] == 0).all()
            assert np.all(np.abs(got[1][small]) <= 2.0 ** -126)
    for bad in (0, 1, 253, 254, 255):
        s = scales.copy()
        s[n - 1, 0] = bad
        payload[n - 1, 3] = 5
        with pytest.raises(coord.CoordError) as e:
            weights_of(payload, s)
        assert e.value.code == 3 and "scale byte" in str(e.value)


def test_w4_bad_values_of_x_stay_in_their_row():
    rng, payload, scales = w4_inputs(50, 256, 2)
    payload |= 0x11                                                   # no zero codes: an infinity keeps its sign rule
    weights = weights_of(payload, scales)
    w = R.w4_weights(payload, scales)
    x = rng.standard_normal((4, 256)).astype(np.float32)
    x[1, 9], x[2, 100] = np.nan, np.inf
    bits, value = R.bf16(x)
    bits[1, 9] = 0x7FC0
    got = run_w4(weights, bits, 4)
    want, tol = R.w4_product(value[[0, 3]], w)
    assert np.all(np.abs(got[[0, 3]] - want) <= tol)
    assert np.isnan(got[1]).all() and np.array_equal(got[2], np.copysign(np.inf, w[:, 100]))
    p, s = O.q0_quantize(np.nan_to_num(x, nan=0.5, posinf=1.0))
    p[1, 9] = 0x7F                                                    # a NaN code
    s[2, 3] = 255                                                     # a scale that is none
    got = run_w4(weights, None, 4, fp8=(p, s))
    value = R.wire_values(p[[0, 3]], s[[0, 3]])
    want, tol = R.w4_product(value, w)
    assert np.all(np.abs(got[[0, 3]] - want) <= tol) and np.isnan(got[[1, 2]]).all()


@pytest.mark.parametrize("form", ["bf16", "fp8"])
def test_w4_more_rows_than_a_launch_takes(form):
    rows, n, k = (1 << 19) + 21, 3, 32
    rng, payload, scales = w4_inputs(n, k, 9)
    weights = weights_of(payload, scales)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    if form == "bf16":
        bits, value = R.bf16(x)
        got = run_w4(weights, bits, rows, y_pad=1)
    else:
        wire = O.q0_quantize(x)
        value = R.wire_values(*wire)
        got = run_w4(weights, None, rows, fp8=wire, y_pad=1)
    want, tol = R.w4_product(value, R.w4_weights(payload, scales))
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("rows,n,k", [(3, 40, 160), (20, 16400, 256)])
def test_w4_subnormal_values_of_x_count(rows, n, k):
    """BF16 values below 2^-126 under weights large enough to make ordinary products of them."""
    rng, payload, _ = w4_inputs(n, k, rows)
    weights_scales = np.full((n, k // 32), 252, np.uint8)
    weights = weights_of(payload, weights_scales)
    bits = (rng.integers(0, 128, (rows, k)) | rng.integers(0, 2, (rows, k)) << 15).astype(np.uint16)
    want, tol = R.w4_product(R.widen(bits), R.w4_weights(payload, weights_scales))
    got = run_w4(weights, bits, rows)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


def test_w4_wire_rows_at_the_ends_of_the_scale_range():
    rng, payload, scales = w4_inputs(40, 128, 6, 126, 129)
    weights = weights_of(payload, scales)
    w = R.w4_weights(payload, scales)
    p = rng.integers(0, 0x7F, (8, 128), dtype=np.uint8) | (rng.integers(0, 2, (8, 128), dtype=np.uint8) << 7)
    for byte in (10, 60, 127, 200, 236):
        s = np.full((8, 4), byte, np.uint8)
        want, tol = R.w4_product(R.wire_values(p, s), w)
        got = run_w4(weights, None, 8, fp8=(p, s))
        assert np.all(np.abs(got - want) <= tol + 128 * 6 * 2.0 ** -126), byte
    zero = np.zeros((8, 128), np.uint8)
    assert (run_w4(weights, None, 8, fp8=(zero, np.zeros((8, 4), np.uint8))) == 0).all()


def on_the_grid(x):
    """What the products take wire values as: multiples of 2^-133, the step of BF16's smallest numbers, nearest even. It takes a
    scale byte below 3 for a code to have bits under that."""
    return np.rint(np.asarray(x, np.float64) * 2.0 ** 133) * 2.0 ** -133


@pytest.mark.parametrize("columns", [256, 16400])                     # rows streamed, rows resident
def test_w4_wire_rows_every_code_under_every_scale_byte(columns):
    """One nonzero weight in each column of y, a power of two: y names the value that a code under a byte is taken as. Byte 0 is
    2^-127 like any other byte's power of two, and what has a block of nonzero codes under it counts."""
    codes = np.resize(np.array([c for c in range(256) if c & 0x7F != 0x7F], np.uint8), 256)
    place = np.arange(columns) % 256
    w = np.zeros((columns, 128), np.uint8)
    w[np.arange(columns), place // 2] = 2 << (4 * (place % 2))        # the code of 1
    for exponent, some in ((125, np.arange(0, 40)), (0, np.arange(14, 247))):   # sums stay normal numbers
        weights = weights_of(w, np.full((columns, 8), 127 + exponent, np.uint8))
        for part in np.array_split(some, 1 + some.size // 40):
            p, s = np.tile(codes, (part.size, 1)), np.repeat(part.astype(np.uint8)[:, None], 8, 1)
            got = run_w4(weights, None, part.size, fp8=(p, s))
            want = on_the_grid(R.wire_values(p, s)) * 2.0 ** exponent
            assert np.array_equal(got, want[:, place].astype(np.float32)), part
            assert np.array_equal(on_the_grid(R.wire_values(p, s))[part > 2], R.wire_values(p, s)[part > 2])


@pytest.mark.parametrize("rows,n,k", [(3, 40, 160), (20, 16400, 256)])
def test_w4_wire_rows_of_the_smallest_blocks(rows, n, k):
    """Scale bytes 0..9 in one row, nonzero codes, under weights that make ordinary numbers of them."""
    rng, payload, _ = w4_inputs(n, k, rows + 1)
    w_scales = rng.integers(240, 253, (n, k // 32), dtype=np.uint8)
    weights = weights_of(payload, w_scales)
    p = rng.integers(1, 0x7F, (rows, k), dtype=np.uint8) | (rng.integers(0, 2, (rows, k), dtype=np.uint8) << 7)
    s = rng.integers(0, 10, (rows, k // 32), dtype=np.uint8)
    s[0] = 0
    want, tol = R.w4_product(on_the_grid(R.wire_values(p, s)), R.w4_weights(payload, w_scales))
    got = run_w4(weights, None, rows, fp8=(p, s))
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


def test_w4_takes_the_smallest_rows_the_join_writes():
    """A norm weight so small that the join's wire rows carry scale byte 0 over nonzero codes, read in place by a product."""
    rows, cols, n = 5, 1024, 300
    h, planes, _, _, _ = join_inputs(rows, cols, 1, False, "none", 21)
    pre = np.geomspace(1e-38, 1e-34, cols).astype(np.float32)
    out = run_join(h, planes, pre, None, None, 1.0, 1e-5, "none")
    p, s = np.ascontiguousarray(out["payload"]), np.ascontiguousarray(out["scales"])
    blocks = (p.reshape(rows, -1, 32) & 0x7F).any(-1)
    assert (blocks & (s == 0)).sum() > 20 and (s > 2).sum() > 20
    rng, payload, _ = w4_inputs(n, cols, 22)
    w_scales = np.full((n, cols // 32), 240, np.uint8)
    want, tol = R.w4_product(on_the_grid(R.wire_values(p, s)), R.w4_weights(payload, w_scales))
    got = run_w4(weights_of(payload, w_scales), None, rows, fp8=(p, s))
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


def test_w4_refuses_calls_that_do_not_fit():
    rng, payload, scales = w4_inputs(32, 64, 1)
    weights = weights_of(payload, scales)
    x, y = room(4096), room(4096)
    bad = [lambda: weights.matvec(x.ptr + 8, 1, y.ptr), lambda: weights.matvec(x.ptr, 1, y.ptr, x_pitch=60), lambda: weights.matvec(x.ptr, 1, y.ptr, x_pitch=68),
           lambda: weights.matvec(x.ptr, 1, y.ptr + 2), lambda: weights.matvec(x.ptr, 1, y.ptr, y_pitch=31), lambda: weights.matvec(x.ptr, -1, y.ptr),
           lambda: weights.matvec(None, 1, y.ptr), lambda: weights.matvec(x.ptr, 1, None), lambda: weights.matvec(x.ptr, 1, y.ptr + 1, True),
           lambda: weights.matvec_fp8(x.ptr + 4, x.ptr, 1, y.ptr), lambda: weights.matvec_fp8(x.ptr, x.ptr, 1, y.ptr, payload_pitch=68),
           lambda: weights.matvec_fp8(x.ptr, None, 1, y.ptr), lambda: weights.matvec_fp8(x.ptr, x.ptr, 1, y.ptr, scales_pitch=1)]
    bad += [lambda: weights.matvec(x.ptr, 2, y.ptr, x_pitch=1 << 25), lambda: weights.matvec(x.ptr, 2, y.ptr, y_pitch=(1 << 24) + 1),
            lambda: weights.matvec_fp8(x.ptr, x.ptr, 2, y.ptr, payload_pitch=1 << 25)]
    for call in bad:
        with pytest.raises(coord.CoordError) as e:
            call()
        assert e.value.code == 1
    weights.matvec(x.ptr, 0, y.ptr)
    assert (y.to_host(np.uint8) == 0x5A).all()
    weights.close()
    with pytest.raises(coord.CoordError):
        weights.matvec(x.ptr, 1, y.ptr)


# ---- log probabilities -------------------------------------------------------------------------------------

def run_logprobs(logits, given, top, scale=1.0, half=False, shift=0, pad=0, ragged=None):
    """(given, entropy, ids, top) as the kernel gives them; `logits` FP32 values (exact BF16 where half)."""
    rows, vocab = logits.shape
    dtype = np.uint16 if half else np.float32
    flat = np.full(shift + rows * (vocab + pad) + 8, 0x7FC0 if half else np.nan, dtype)   # NaN around the rows: not to be read
    flat[shift:shift + rows * (vocab + pad)].reshape(rows, vocab + pad)[:, :vocab] = R.bf16(logits)[0] if half else logits
    x = dev(flat)
    given = np.ascontiguousarray(given, np.int32)
    m = given.shape[1]
    gd, gl, en, ti, tl = dev(given), room(rows * m * 4), room(rows * 4), room(rows * top * 4), room(rows * top * 4)
    need = coord.token_logprobs_workspace(rows, vocab, top)
    ws = room(need, 0xFF)                                             # its content is irrelevant
    coord.token_logprobs(x.ptr + shift * x_size(half), half, rows, vocab, vocab + pad, gd.ptr, m, gl.ptr, en.ptr, top, ti.ptr if top else None,
                         tl.ptr if top else None, ws.ptr if need else None, need, scale=scale)
    return (gl.to_host(np.float32)[:rows * m].reshape(rows, m), en.to_host(np.float32)[:rows],
            ti.to_host(np.int32)[:rows * top].reshape(rows, top), tl.to_host(np.float32)[:rows * top].reshape(rows, top))


def x_size(half):
    return 2 if half else 4


def check_logprobs(got, logits, given, top, scale):
    with np.errstate(all="ignore"):
        check_logprobs_against(got, R.logprobs(logits, given, top, scale))


def check_logprobs_against(got, want):
    gl, en, ids, lp = got
    wg, wh, wi, wl, tg, th, tt = want
    assert np.array_equal(ids, wi)

    def near(a, b, tol):
        same = (np.isnan(a) & np.isnan(b)) | (a == b)
        with np.errstate(invalid="ignore"):
            ok = same | (np.abs(a - b) <= tol)
        assert ok.all(), (np.argwhere(~ok)[:3], a[~ok][:3], b[~ok][:3], np.broadcast_to(tol, a.shape)[~ok][:3])
    near(gl, wg, tg)
    near(en, wh, th)
    near(lp, wl, tt)


def some_logits(rng, rows, vocab, half, masked=0.0):
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 6
    x[rng.random((rows, vocab)) < masked] = -np.inf
    return R.bf16(x)[1] if half else x


LENGTHS = [(1, 1), (1, 2), (4, 5), (2, 8), (3, 63), (2, 64), (5, 511), (4, 512), (3, 513), (2, 520), (3, 1031), (2, 4099), (40, 2050), (3, 50003), (1, 131072),
           (2, 131075), (1100, 700),
           # every form of the rule on sizes: rows over two, four and eight waves, over several workgroups, more rows than workgroups
           (1600, 3000), (800, 9000), (600, 9000), (200, 4200), (100, 9000), (5000, 600), (4100, 40), (31, 1537),
           # rows in registers, more of them than workgroups; parts of four chunks, the last with values in few lanes; parts that are walked
           (17000, 40), (1, 1024), (3, 1025), (9, 8192), (9, 8193), (700, 8000), (3, 250000), (2, 262144), (1, 262150), (1, 400001), (90, 100003)]


@pytest.mark.parametrize("rows,vocab", LENGTHS)
@pytest.mark.parametrize("half", [False, True])
def test_logprobs_lengths_starts_and_counts(rows, vocab, half):
    rng = np.random.default_rng(rows * 11 + vocab)
    for top, shift, pad, scale, masked in ((0, 0, 0, 1.0, 0.0), (1, 1, 3, 0.7, 0.5), (5, 3, 0, 1.25, 0.0), (32, 0, 8, 1.0, 0.9), (20, 7, 1, 2.0, 0.0)):
        top = min(top, vocab)
        x = some_logits(rng, rows, vocab, half, masked)
        given = rng.integers(0, vocab, (rows, 3))
        given[:, 1] = np.argmax(x, 1)
        given[rng.random((rows, 3)) < 0.1] = -1
        given[0, 2] = vocab
        got = run_logprobs(x, given, top, scale, half, shift, pad)
        check_logprobs(got, x, given, top, scale)


def hard_rows(vocab, half):
    """Ties everywhere, values in order either way, one survivor, nothing left, lowest finite values, infinities and NaNs."""
    rng = np.random.default_rng(vocab)
    low = np.float32(R.bf16(np.float32(-3.38e38))[1]) if half else np.finfo(np.float32).min
    rows = []
    rows.append(np.zeros(vocab))                                     # all equal
    rows.append(np.linspace(-20, 20, vocab))                         # ascending: every chunk beats all before
    rows.append(np.linspace(20, -20, vocab))
    rows.append(rng.integers(0, 4, vocab).astype(float))             # four values
    rows.append(np.full(vocab, -np.inf))                             # nothing left
    one = np.full(vocab, -np.inf)
    one[vocab // 3] = -7.0
    rows.append(one)                                                 # one token left
    rows.append(np.full(vocab, low))                                 # masked with the lowest finite value, all of it
    some = np.full(vocab, low)
    some[::97] = rng.standard_normal(some[::97].size)
    rows.append(some)
    nan = rng.standard_normal(vocab)
    nan[5::31] = np.nan
    rows.append(nan)
    inf = rng.standard_normal(vocab)
    inf[vocab // 2] = np.inf
    rows.append(inf)
    rows.append(np.full(vocab, np.nan))
    signed = np.zeros(vocab)
    signed[1::2] = -0.0
    rows.append(signed)                                              # the two zeros are equal
    block = np.full(vocab, -50.0)
    block[vocab - 40:] = 3.0                                         # all alternatives in the last chunk, tied
    rows.append(block)
    x = np.stack(rows).astype(np.float32)
    x = R.bf16(x)[1] if half else x
    if half:
        x[np.isnan(np.stack(rows))] = np.nan
    return x


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("vocab", [700, 2000, 8100, 20011, 131072, 250000])
def test_logprobs_of_rows_that_are_hard_to_select_from(half, vocab):
    x = hard_rows(vocab, half)
    rows = range(len(x))
    given = np.stack([[vocab // 3, 0, vocab - 1]] * len(rows))
    for top in (1, 8, 32):
        check_logprobs(run_logprobs(np.ascontiguousarray(x), given, top, 1.0, half), x.astype(np.float64), given, top, 1.0)
        single = np.concatenate([run_logprobs(x[r:r + 1], given[r:r + 1], top, 1.0, half)[2] for r in range(len(rows))])
        assert np.array_equal(single, run_logprobs(x, given, top, 1.0, half)[2])   # however a row is cut, the same ids


def rows_of_large_numbers(vocab, half):
    """Logits so large that the rounding of scaled ones is more than the differences that matter, and masks like them."""
    rng = np.random.default_rng(vocab + 1)
    rows = [np.full(vocab, v) for v in (-1e9, -1e10, -3e20, 1e10, 9e29, 2e7)]                   # equal ones: the entropy is ln vocab
    for low in (-1e9, -1e10, -3e20, -1e38):                                                     # masks: a few tokens, one late token, half of them
        for kept in (np.arange(3, vocab, 997), np.array([vocab - 2]), np.arange(0, vocab, 2)):
            row = np.full(vocab, low)
            row[kept] = rng.standard_normal(kept.size) * 3
            rows.append(row)
    for base, step in ((11629080.0, 1.0), (-11629080.0, 1.0), (5e8, 32.0), (-5e8, 32.0)):       # 2^24 in units of log2, and past it
        rows.append(base + step * rng.integers(-60, 1, vocab))
        rows.append(base + step * np.sort(rng.integers(-9, 9, vocab)))
    x = np.stack(rows).astype(np.float32)
    return R.bf16(x)[1] if half else x


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("vocab,copies,top,scale", [(700, 1, 8, 1.0), (5003, 1, 20, 0.7), (5003, 80, 8, 1.0), (20011, 1, 8, 1.25), (20011, 60, 5, 1.0),
                                                    (100003, 4, 8, 1.0), (5003, 1, 4, 2.0 ** 20), (5003, 80, 4, 2.0 ** -20)])
def test_logprobs_of_large_numbers(half, vocab, copies, top, scale):
    x = rows_of_large_numbers(vocab, half)
    n = len(x)
    given = np.stack([[vocab // 3, 0, vocab - 2]] * n)
    got = run_logprobs(np.tile(x, (copies, 1)), np.tile(given, (copies, 1)), top, scale, half, shift=3)
    with np.errstate(over="ignore"):
        gl, en, ids, lp = (g.reshape(copies, n, -1) for g in got)
        for i in (0, copies - 1):                                                               # a log probability past FP32 is -infinity
            want = R.logprobs(x, given, top, scale)
            check_logprobs_against((gl[i], en[i, :, 0], ids[i], lp[i]), tuple(w.astype(np.float32) if k in (0, 3) else w for k, w in enumerate(want)))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("vocab,copies,top", [(3001, 120, 8), (3001, 100, 32), (17000, 50, 1), (17000, 50, 20), (17000, 130, 8), (100000, 8, 32)])
def test_logprobs_of_hard_rows_among_many(half, vocab, copies, top):
    """The forms that walk over a row, which many rows take. The same row gives the same bits wherever it stands."""
    x = hard_rows(vocab, half)
    n = len(x)
    given = np.stack([[vocab // 3, 0, vocab - 1]] * n)
    got = run_logprobs(np.tile(x, (copies, 1)), np.tile(given, (copies, 1)), top, 1.0, half, pad=-vocab % 8)
    check_logprobs([g[:n] for g in got], x.astype(np.float64), given, top, 1.0)
    for g in got:
        bits = g.view(np.uint32).reshape(copies, n, -1)
        assert (bits == bits[:1]).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,vocab", [(2000, 700), (300, 5003), (700, 5003), (30, 50003), (200, 50003)])
def test_logprobs_are_never_above_zero_and_entropies_never_below(rows, vocab, half):
    """Constrained decoding: one allowed token, or one far ahead of a few others, at any logit, with every one of them given."""
    rng = np.random.default_rng(rows + vocab)
    x = np.full((rows, vocab), -np.inf, np.float32)
    at = rng.integers(0, vocab, (rows, 3))
    x[np.arange(rows), at[:, 0]] = rng.standard_normal(rows) * np.exp2(rng.integers(-3, 12, rows))
    some = np.arange(rows) % 4 == 0
    for i in (1, 2):
        x[some, at[some, i]] = x[some, at[some, 0]] - rng.integers(15, 40, some.sum())
    x = R.bf16(x)[1] if half else x
    for scale in (1.0, 0.7):
        got = run_logprobs(x, at, 2, scale, half)
        check_logprobs(got, x, at, 2, scale)
        given, entropy, _, top = got
        assert (given <= 0).all() and (top <= 0).all() and (entropy >= 0).all(), (given.max(), top.max(), entropy.min())
        assert not np.signbit(entropy).any()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,vocab", [(3, 700), (40, 5003), (700, 5003), (3, 50003), (200, 50003)])
@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -122, 2.0 ** -135])
def test_logprobs_of_logits_whose_differences_pass_fp32(rows, vocab, half, scale):
    """Logits over FP32's whole range, brought to ordinary sizes by the scale: a difference of two may be past the range."""
    rng = np.random.default_rng(rows + vocab)
    x = rng.uniform(-3.38e38, 3.38e38, (rows, vocab)).astype(np.float32)
    x[:, 5], x[:, vocab // 2] = 3.38e38, -3.38e38
    x[rng.random((rows, vocab)) < 0.1] = -np.inf
    x = R.bf16(x)[1] if half else x
    given = np.stack([[5, vocab // 2, 0]] * rows)
    check_logprobs(run_logprobs(x, given, 8, scale, half), x, given, 8, scale)


def test_logprobs_signalling_nans_do_not_hide_values():
    x = np.random.default_rng(3).standard_normal((4, 3000)).astype(np.float32)
    raw = x.view(np.uint32)
    raw[1, 10:2000:8] = 0x7F800001                                   # a signalling NaN in most lanes' chunks
    raw[2, 10:2000:8] = 0xFFA00000
    given = np.zeros((4, 1), np.int32)
    with np.errstate(invalid="ignore"):
        check_logprobs(run_logprobs(x, given, 8), x.astype(np.float64), given, 8, 1.0)


def test_logprobs_without_optional_outputs_and_twice_the_same():
    rng = np.random.default_rng(6)
    x = some_logits(rng, 3, 40000, False)
    xd = dev(x)
    need = coord.token_logprobs_workspace(3, 40000, 4)
    ws, ids, lp = room(need), room(48), room(48)
    coord.token_logprobs(xd.ptr, False, 3, 40000, 40000, None, 0, None, None, 4, ids.ptr, lp.ptr, ws.ptr, need)
    first = ids.to_host(np.int32), lp.to_host(np.uint32)
    coord.token_logprobs(xd.ptr, False, 3, 40000, 40000, None, 0, None, None, 4, ids.ptr, lp.ptr, ws.ptr, need)
    assert np.array_equal(first[0], ids.to_host(np.int32)) and np.array_equal(first[1], lp.to_host(np.uint32))
    assert np.array_equal(first[0].reshape(3, 4), R.logprobs(x, np.zeros((3, 0), int), 4, 1.0)[2])


# ---- far apart ----------------------------------------------------------------------------------------------

def put(at, a):
    a = np.ascontiguousarray(a)
    assert b1.load().m26s_b1_copy_to_device(at, a.ctypes.data, a.nbytes) == 0


def take(at, shape, dtype):
    a = np.empty(shape, dtype)
    assert b1.load().m26s_b1_copy_to_host(a.ctypes.data, at, a.nbytes) == 0
    return a


def test_rows_further_apart_than_32_bits_reach():
    """Pitches that put a row past 2^32 bytes from the first; what lies between is not touched."""
    far = b1.DeviceBuffer(5 << 30)
    rng = np.random.default_rng(12)
    for vocab, half in ((1000, True), (20001, True), (20001, False)):
        size, pitch = x_size(half), ((1 << 32) // x_size(half)) + 5
        x = some_logits(rng, 2, vocab, half)
        for r in range(2):
            put(far.ptr + r * pitch * size, R.bf16(x[r])[0] if half else x[r])
        given = np.array([[3, 3, vocab - 1], [vocab // 2, -1, 0]], np.int32)
        gd, gl, en, ti, tl = dev(given), room(24), room(8), room(40), room(40)
        need = coord.token_logprobs_workspace(2, vocab, 5)
        ws = room(need)
        coord.token_logprobs(far.ptr, half, 2, vocab, pitch, gd.ptr, 3, gl.ptr, en.ptr, 5, ti.ptr, tl.ptr, ws.ptr, need)
        check_logprobs((gl.to_host(np.float32).reshape(2, 3), en.to_host(np.float32), ti.to_host(np.int32).reshape(2, 5),
                        tl.to_host(np.float32).reshape(2, 5)), x, given, 5, 1.0)
    # the join in place, a plane's rows and the normed rows between those of h
    cols = 96
    h, planes, pre, _, _ = join_inputs(2, cols, 1, False, "none", 2)
    hp, pp = (1 << 30) + 64, (1 << 31) + 64
    for r in range(2):
        put(far.ptr + r * hp * 4, h[r])
        put(far.ptr + 4096 + r * pp * 2, planes[0][0][r])
    w = dev(pre)
    plan = coord.Join(cols, w.ptr, scale=0.5, eps=1e-5, plane_pitch=pp, h_pitch=hp, norm_pitch=pp)
    plan(2, far.ptr, [far.ptr + 4096], far.ptr, norm=far.ptr + 8192)
    got = {"h": np.stack([take(far.ptr + r * hp * 4, cols, np.float32) for r in range(2)]),
           "norm": np.stack([take(far.ptr + 8192 + r * pp * 2, cols, np.uint16) for r in range(2)])}
    check_join(got, h, planes, pre, None, None, 0.5, 1e-5)
    # products: the largest pitches of x and y
    rows, n, k, pitch = 70, 40, 96, 1 << 24
    rng, payload, scales = w4_inputs(n, k, 3)
    weights = weights_of(payload, scales)
    bits, value = R.bf16(rng.standard_normal((rows, k)).astype(np.float32))
    for r in range(rows):
        put(far.ptr + 4096 + r * pitch * 2, bits[r])
        put(far.ptr + r * pitch * 4 + n * 4, np.full(4, 7.0, np.float32))
    weights.matvec(far.ptr + 4096, rows, far.ptr, x_pitch=pitch, y_pitch=pitch)
    y = np.stack([take(far.ptr + r * pitch * 4, n + 4, np.float32) for r in range(rows)])
    want, tol = R.w4_product(value, R.w4_weights(payload, scales))
    assert np.all(np.abs(y[:, :n] - want) <= tol) and (y[:, n:] == 7.0).all()


# ---- together ------------------------------------------------------------------------------------------------

def test_a_step_from_the_ranks_rows_to_the_answer():
    """The ranks' rows -> join -> BF16 rows to the router's product and its top-8, wire rows read in place by another
    product -> second join -> head -> log probabilities: each stage against its reference on the GPU's own inputs."""
    rng = np.random.default_rng(12)
    rows, cols, vocab, eps = 19, 4096, 5003, 1e-5
    h = rng.standard_normal((rows, cols)).astype(np.float32)
    planes = [R.bf16((rng.standard_normal((rows, cols)) * 0.2).astype(np.float32)) for _ in range(4)]
    w1, w2 = ((1 + 0.1 * rng.standard_normal(cols)).astype(np.float32) for _ in range(2))
    mats = {}
    for name, n in (("router", 256), ("proj", cols), ("head", vocab)):
        _, payload, scales = w4_inputs(n, cols, n, 116, 120)
        mats[name] = (weights_of(payload, scales), R.w4_weights(payload, scales))
    hd, pd, d1, d2 = dev(h), [dev(b) for b, _ in planes], dev(w1), dev(w2)
    pitch = 4224
    frame, norm, logits, branch, norm2 = room(rows * pitch), room(rows * cols * 2), room(rows * 256 * 4), room(rows * cols * 2), room(rows * cols * 2)
    ids, wts, bias = room(rows * 32), room(rows * 32), dev(np.zeros(256, np.float32))
    out = room(rows * vocab * 4)
    first = coord.Join(cols, d1.ptr, planes=4, eps=eps, payload_pitch=pitch, scales_pitch=pitch)
    second = coord.Join(cols, d2.ptr, post_weight=d1.ptr, eps=eps, scale=0.5)
    first(rows, hd.ptr, [p.ptr for p in pd], hd.ptr, norm.ptr, payload=frame.ptr, scales=frame.ptr + cols)
    h1 = hd.to_host(np.float32).reshape(rows, cols)
    mats["router"][0].matvec(norm.ptr, rows, logits.ptr)
    glue.router_topk(logits.ptr, bias.ptr, rows, 256, 8, ids.ptr, wts.ptr)
    mats["proj"][0].matvec_fp8(frame.ptr, frame.ptr + cols, rows, branch.ptr, True, payload_pitch=pitch, scales_pitch=pitch)
    second(rows, hd.ptr, [branch.ptr], hd.ptr, norm2.ptr)
    mats["head"][0].matvec(norm2.ptr, rows, out.ptr)
    given = rng.integers(0, vocab, (rows, 1)).astype(np.int32)
    gd, gl, en, ti, tl = dev(given), room(rows * 4), room(rows * 4), room(rows * 20), room(rows * 20)
    need = coord.token_logprobs_workspace(rows, vocab, 5)
    ws = room(need)
    coord.token_logprobs(out.ptr, False, rows, vocab, vocab, gd.ptr, 1, gl.ptr, en.ptr, 5, ti.ptr, tl.ptr, ws.ptr if need else None, need)

    n1 = norm.to_host(np.uint16).reshape(rows, cols)
    raw = frame.to_host(np.uint8).reshape(rows, pitch)
    got = {"h": h1, "norm": n1, "payload": raw[:, :cols], "scales": raw[:, cols:cols + 128]}
    check_join(got, h, planes, w1, None, None, 1.0, eps)
    lg = logits.to_host(np.float32).reshape(rows, 256)
    want, tol = R.w4_product(R.widen(n1), mats["router"][1])
    assert np.all(np.abs(lg - want) <= tol)
    assert np.array_equal(ids.to_host(np.int32).reshape(rows, 8), O.router_topk(lg, np.zeros(256, np.float32), 8)[0])
    br = branch.to_host(np.uint16).reshape(rows, cols)
    want, tol = R.w4_product(R.wire_values(got["payload"], got["scales"]), mats["proj"][1])
    assert np.all(np.abs(R.widen(br) - want) <= tol + R.UBF16 * (np.abs(want) + tol))
    n2 = norm2.to_host(np.uint16).reshape(rows, cols)
    check_join({"h": hd.to_host(np.float32).reshape(rows, cols), "norm": n2}, h1, [(br, R.widen(br))], w2, w1, None, 0.5, eps)
    lo = out.to_host(np.float32).reshape(rows, vocab)
    want, tol = R.w4_product(R.widen(n2), mats["head"][1])
    assert np.all(np.abs(lo - want) <= tol)
    check_logprobs((gl.to_host(np.float32).reshape(rows, 1), en.to_host(np.float32), ti.to_host(np.int32).reshape(rows, 5),
                    tl.to_host(np.float32).reshape(rows, 5)), lo, given, 5, 1.0)


class Hip:
    """The few stream and graph calls a captured step needs, from the HIP runtime that the library has loaded."""

    def __init__(self):
        b1.device_memory()                                            # the library, and with it the runtime, is loaded
        path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64.so" in line)
        self.lib = C.CDLL(path)

    def __call__(self, name, *args):
        rc = getattr(self.lib, name)(*args)
        assert rc == 0, (name, rc)

    def stream(self):
        s = C.c_void_p()
        self("hipStreamCreate", C.byref(s))
        return s


def test_captured_step_replays_on_new_inputs_beside_eager_calls():
    """Join, head and log probabilities captured into one graph on a stream of its own; each replay reads new inputs and equals
    an eager run of the same inputs, launched at the same time on another stream into buffers of its own."""
    hip = Hip()
    rng = np.random.default_rng(4)
    rows, cols, vocab, top = 4, 1024, 30011, 6
    payload = rng.integers(0, 256, (vocab, cols // 2), dtype=np.uint8)
    weights = weights_of(payload, np.full((vocab, cols // 32), 118, np.uint8))
    w = dev((1 + 0.1 * rng.standard_normal(cols)).astype(np.float32))
    plan = coord.Join(cols, w.ptr, eps=1e-5)
    need = coord.token_logprobs_workspace(rows, vocab, top)
    assert need > 0
    inputs = dict(h=rows * cols * 4, p=rows * cols * 2, ids=rows * 4)
    outputs = dict(ho=rows * cols * 4, n=rows * cols * 2, lo=rows * vocab * 4, gl=rows * 4, en=rows * 4, ti=rows * top * 4, tl=rows * top * 4)
    a, e = ({k: room(size, 0) for k, size in dict(inputs, **outputs, ws=need).items()} for _ in range(2))

    def step(b, stream):
        plan(rows, b["h"].ptr, [b["p"].ptr], b["ho"].ptr, b["n"].ptr, stream=stream)
        weights.matvec(b["n"].ptr, rows, b["lo"].ptr, stream=stream)
        coord.token_logprobs(b["lo"].ptr, False, rows, vocab, vocab, b["ids"].ptr, 1, b["gl"].ptr, b["en"].ptr, top, b["ti"].ptr, b["tl"].ptr,
                             b["ws"].ptr, need, stream=stream)

    side, other, graph, runnable = hip.stream(), hip.stream(), C.c_void_p(), C.c_void_p()
    hip("hipStreamBeginCapture", side, C.c_int(2))                    # relaxed
    step(a, side.value)
    hip("hipStreamEndCapture", side, C.byref(graph))
    hip("hipGraphInstantiate", C.byref(runnable), graph, None, None, C.c_size_t(0))
    seen = []
    for turn in range(4):
        new = dict(h=rng.standard_normal((rows, cols)).astype(np.float32), p=R.bf16(rng.standard_normal((rows, cols)).astype(np.float32))[0],
                   ids=rng.integers(0, vocab, (rows, 1)).astype(np.int32))
        for b in (a, e):
            for k, v in new.items():
                assert b1.load().m26s_b1_copy_to_device(b[k].ptr, v.ctypes.data, v.nbytes) == 0
        hip("hipGraphLaunch", runnable, side)
        step(e, other.value)
        hip("hipStreamSynchronize", side)
        hip("hipStreamSynchronize", other)
        for k in outputs:
            assert np.array_equal(a[k].to_host(np.uint8), e[k].to_host(np.uint8)), (turn, k)
        lo = a["lo"].to_host(np.float32).reshape(rows, vocab)
        check_logprobs((a["gl"].to_host(np.float32).reshape(rows, 1), a["en"].to_host(np.float32), a["ti"].to_host(np.int32).reshape(rows, top),
                        a["tl"].to_host(np.float32).reshape(rows, top)), lo, new["ids"], top, 1.0)
        seen.append(lo)
    assert not np.array_equal(seen[0], seen[1])
    hip("hipGraphExecDestroy", runnable)
    hip("hipGraphDestroy", graph)
    hip("hipStreamDestroy", side)
    hip("hipStreamDestroy", other)


def test_weights_are_not_laid_out_within_a_capture_and_leave_it_whole():
    """Laying weights out waits for the stream, which a capture does not allow: refused before anything is done, so that the graph
    goes on and no later call reports the failure."""
    hip = Hip()
    rng, payload, scales = w4_inputs(40, 128, 3)
    weights, p, s = weights_of(payload, scales), dev(payload), dev(scales)
    bits, value = R.bf16(rng.standard_normal((2, 128)).astype(np.float32))
    x, y = dev(bits), room(2 * 40 * 4)
    side, graph, runnable = hip.stream(), C.c_void_p(), C.c_void_p()
    hip("hipStreamBeginCapture", side, C.c_int(2))                    # relaxed
    with pytest.raises(coord.CoordError) as e:
        coord.Weights4(p.ptr, s.ptr, 40, 128, stream=side.value)
    assert e.value.code == 1 and "captured" in str(e.value)
    weights.matvec(x.ptr, 2, y.ptr, stream=side.value)
    hip("hipStreamEndCapture", side, C.byref(graph))
    hip("hipPeekAtLastError")
    hip("hipGraphInstantiate", C.byref(runnable), graph, None, None, C.c_size_t(0))
    want, tol = R.w4_product(value, R.w4_weights(payload, scales))
    for _ in range(3):
        put(y.ptr, np.full(2 * 40, 7.0, np.float32))
        hip("hipGraphLaunch", runnable, side)
        hip("hipStreamSynchronize", side)
        assert np.all(np.abs(y.to_host(np.float32).reshape(2, 40) - want) <= tol)
    hip("hipGraphExecDestroy", runnable)
    hip("hipGraphDestroy", graph)
    hip("hipStreamDestroy", side)
