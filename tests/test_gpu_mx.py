"""Microscaled matrices on the GPU: quantizers bit for bit, products, gradients and activations against 64-bit restatements.

Tolerances.  Packed operands are exact, so a product's error is that of its fp32 sum and of the last rounding.  The tensor cores add
a step's products to the running sum with an error of at most a few units of fp32 (2^-23) of the largest magnitude at hand, which
the sum S of the products' magnitudes bounds; a step has 16 values at least: (steps + 8) * 2^-22 * S.  An output type with
precision eps adds eps / 2 of the value (and fp16's smallest step 2^-24, half of it, where values are subnormal)."""
import numpy as np
import pytest

import mx_util

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GUARD = 77.0


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cntk_b200 import lib as L
    return L


def code(lib, t):
    return {"f32": lib.F32, "f16": lib.F16, "bf16": lib.BF16}[t]


def stream():
    return torch.cuda.current_stream().cuda_stream


def dense(rng, n, m, t, pad=0, offset=0, scale=1.0):
    """[n, m] view on the device of type t, `pad` values between columns, starting `offset` values into its buffer; and the values."""
    v = rng.standard_normal((n, m)) * np.exp2(rng.standard_normal((n, 1))) * scale
    return place(torch.from_numpy(v), t, pad, offset)


def place(v, t, pad=0, offset=0):
    n, m = v.shape
    flat = torch.full((offset + n * (m + pad) + 8,), GUARD, dtype=TYPES[t], device=DEV)
    d = flat[offset:offset + n * (m + pad)].view(n, m + pad)[:, :m]
    d.copy_(v.to(TYPES[t]))
    return flat, d, d.double().cpu().numpy()


def room(n, m, t, pad=0, offset=0):
    flat = torch.full((offset + n * (m + pad) + 8,), GUARD, dtype=TYPES[t], device=DEV)
    return flat, flat[offset:offset + n * (m + pad)].view(n, m + pad)[:, :m]


def untouched(flat, view, pad, offset):
    """Nothing outside the matrix was written."""
    n, m = view.shape
    mask = torch.ones_like(flat, dtype=torch.bool)
    mask[offset:offset + n * (m + pad)].view(n, m + pad)[:, :m] = False
    assert bool((flat[mask] == GUARD).all()), "written outside the matrix"


def to_dev(codes, scales):
    return torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV)


def packed(rng, n, m, fmt, scale=1.0):
    """A random packed matrix (rows m, columns n) on the device and its values."""
    x = rng.standard_normal((n, m)) * np.exp2(rng.standard_normal((n, 1))) * scale
    x = x.astype(np.float32)
    return to_dev(*mx_util.pack(x, fmt)), mx_util.values(x, fmt)


def check(got, want, mags, steps, t, what):
    """got within the derived bound of want (both [n, m]); mags: sum of the products' magnitudes."""
    eps = torch.finfo(TYPES[t]).eps
    got = got.double().cpu().numpy()
    tol = (steps + 8) * 2.0 ** -22 * mags + (eps / 2) * (np.abs(want) + (steps + 8) * 2.0 ** -22 * mags)
    if t == "f16":
        tol = tol + 2.0 ** -25
    assert np.array_equal(np.isnan(got), np.isnan(want)), what + ": NaN in other places"
    ok = np.isnan(want) | (got == want) | (np.abs(got - want) <= tol)
    assert ok.all(), f"{what}: {np.count_nonzero(~ok)} of {ok.size} off, first at {np.argwhere(~ok)[0].tolist()}: {got[~ok][0]} for {want[~ok][0]}, worst ratio {np.nanmax(np.abs(got - want) / tol)}"


# ---- quantizers -------------------------------------------------------------------------------------------------------------


def run_quantize(lib, d, m, n, t, ld, fmt, transpose):
    pm, pn = (n, m) if transpose else (m, n)
    codes = torch.full((lib.mx_code_bytes(pm, pn, fmt) + 32,), 0xA5, dtype=torch.uint8, device=DEV)
    scales = torch.full((lib.mx_scale_bytes(pm, pn) + 32,), 0xA5, dtype=torch.uint8, device=DEV)
    lib.mx_quantize(d.data_ptr(), code(lib, t), ld, codes.data_ptr(), scales.data_ptr(), m, n, fmt, transpose, stream())
    assert bool((codes[-32:] == 0xA5).all()) and bool((scales[-32:] == 0xA5).all())
    return codes[:-32], scales[:-32]


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("fmt", [mx_util.FP4, mx_util.INT8])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,pad,offset", [(1, 1, 0, 0), (32, 1, 0, 0), (1, 33, 0, 0), (31, 5, 0, 1), (128, 128, 0, 0), (129, 127, 0, 0), (429, 70, 3, 0),
                                            (512, 363, 0, 0), (40, 300, 8, 8), (363, 17, 5, 3), (1000, 130, 24, 0)])
def test_quantize_and_back(lib, m, n, pad, offset, t, fmt, transpose):
    rng = np.random.default_rng(m * 1000 + n)
    _, d, v = dense(rng, n, m, t, pad, offset)
    codes, scales = run_quantize(lib, d, m, n, t, m + pad, fmt, transpose)
    x = v.T if transpose else v
    want = mx_util.pack(x, fmt)
    assert np.array_equal(scales.cpu().numpy(), want[1])
    assert np.array_equal(codes.cpu().numpy(), want[0])
    values = mx_util.values(x, fmt)
    for t2 in ("f32", "bf16"):  # both hold every value exactly
        flat, out = room(x.shape[0], x.shape[1], t2, pad, offset)
        lib.mx_unquantize(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), code(lib, t2), x.shape[1] + pad, x.shape[1], x.shape[0], fmt, stream())
        assert np.array_equal(out.double().cpu().numpy(), values)
        untouched(flat, out, pad, offset)


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("fmt", [mx_util.FP4, mx_util.INT8])
def test_quantize_borders(lib, fmt, transpose):
    """Ties, the largest elements, subnormals, the ends of the scale range, zeros of both signs, NaN and infinities."""
    rows = []
    for s in (1.0, 2.0 ** 100, 2.0 ** -100, 2.0 ** -126, 2.0 ** -127, 2.0 ** -133, 2.0 ** -149, 2.0 ** 125):
        k = np.arange(32)
        rows.append(s * k / 16)                       # ties of fp4 at 1/4, 3/4, 5/4 ...
        rows.append(-s * (1 + k / 64 + 1 / 128))      # ties of int8
        rows.append(s * np.where(k == 7, 1.9999, (k - 16) / 128))
        rows.append(np.where(k == 31, s, 0.0))
    rows += [np.zeros(32), -np.zeros(32), np.full(32, 3.4028234e38), np.full(32, 1e-45), np.where(np.arange(32) % 2, 3.4028234e38, -1.0)]
    for bad in (np.nan, np.inf, -np.inf):
        rows.append(np.where(np.arange(32) == 5, bad, 1.5))
    x = np.array(rows, np.float32)
    x = np.concatenate([x, x[::-1]], axis=1)  # two blocks: a bad one leaves its neighbour alone
    v = torch.from_numpy(np.ascontiguousarray(x.T if transpose else x)).to(DEV)
    n, m = v.shape
    codes, scales = run_quantize(lib, v, m, n, "f32", m, fmt, transpose)
    want = mx_util.pack(x, fmt)
    assert np.array_equal(scales.cpu().numpy(), want[1])
    assert np.array_equal(codes.cpu().numpy(), want[0])
    out = torch.zeros(x.shape, dtype=torch.float32, device=DEV)
    lib.mx_unquantize(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), lib.F32, x.shape[1], x.shape[1], x.shape[0], fmt, stream())
    got, values = out.double().cpu().numpy(), mx_util.values(x, fmt)
    assert np.array_equal(got, values, equal_nan=True)


@pytest.mark.parametrize("fmt", [mx_util.FP4, mx_util.INT8])
@pytest.mark.parametrize("m,n,pad,offset", [(96, 40, 0, 0), (77, 33, 2, 1)])
def test_values_in_half_precision(lib, m, n, pad, offset, fmt):
    """fp16 cannot hold every value: each is rounded to nearest, too large ones to infinity."""
    rng = np.random.default_rng(15)
    x = rng.standard_normal((n, m)) * np.exp2(rng.integers(-30, 20, (n, 1)))
    (codes, scales), v = to_dev(*mx_util.pack(x, fmt)), mx_util.values(x, fmt)
    flat, out = room(n, m, "f16", pad, offset)
    lib.mx_unquantize(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), lib.F16, m + pad, m, n, fmt, stream())
    with np.errstate(over="ignore"):
        assert np.array_equal(out.cpu().numpy(), v.astype(np.float16))
    untouched(flat, out, pad, offset)


def test_offsets_beyond_32_bits(lib):
    """The last columns of a matrix of more than 2^32 values, with a gap between the columns."""
    m, n, ld = 64, 3, (1 << 31) + 64
    flat = torch.zeros(2 * ld + m, dtype=torch.bfloat16, device=DEV)
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((n, m))).to(torch.bfloat16)
    for j in range(n):
        flat[j * ld:j * ld + m] = x[j].to(DEV)
    codes, scales = run_quantize(lib, flat, m, n, "bf16", ld, mx_util.INT8, False)
    want = mx_util.pack(x.double().numpy(), mx_util.INT8)
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])
    lib.mx_unquantize(codes.data_ptr(), scales.data_ptr(), flat.data_ptr(), lib.BF16, ld, m, n, mx_util.INT8, stream())
    got = torch.stack([flat[j * ld:j * ld + m] for j in range(n)]).double().cpu().numpy()
    assert np.array_equal(got, mx_util.values(x.double().numpy(), mx_util.INT8))


# ---- 4-bit product ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("O,T,K,pad", [(128, 16, 256, 0), (1, 1, 1, 0), (128, 1, 32, 0), (129, 1, 2048, 0), (2048, 1, 2048, 0), (100, 3, 64, 5), (132, 17, 512, 0),
                                       (512, 33, 363, 8), (300, 129, 429, 1), (256, 256, 1024, 0), (2048, 300, 429, 0), (520, 511, 96, 0), (1000, 1000, 1000, 0), (2200, 2500, 900, 0), (2150, 2400, 900, 0), (5000, 1, 1100, 0),
                                       (5000, 2, 429, 3), (5001, 4, 2048, 0), (77, 4, 5000, 0), (40, 5, 333, 0),
                                       (33, 4, 8192, 0), (33, 4, 8193, 0), (20, 1, 40000, 0), (9300, 3, 200, 0), (9304, 4, 1024, 0)])
def test_times(lib, O, T, K, pad, t):
    rng = np.random.default_rng(O + T + K)
    (wc, ws), w = packed(rng, O, K, mx_util.FP4, 0.05)
    (xc, xs), x = packed(rng, T, K, mx_util.FP4)
    bias = rng.standard_normal(O).astype(np.float32)
    bd = torch.from_numpy(bias).to(DEV)
    mags = np.abs(x) @ np.abs(w).T
    for b, want in ((0, x @ w.T), (bd.data_ptr(), x @ w.T + bias)):
        flat, y = room(T, O, t, pad)
        lib.mx_times(wc.data_ptr(), ws.data_ptr(), xc.data_ptr(), xs.data_ptr(), b, y.data_ptr(), code(lib, t), O + pad, O, T, K, stream())
        lib.mx_check(stream())
        check(y, want, mags + (np.abs(bias) if b else 0), K / 16, t, f"times {O}x{T}x{K}")
        untouched(flat, y, pad, 0)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("O,T,K,pad,offset", [(256, 130, 300, 0, 1), (256, 40, 2048, 2, 1), (256, 40, 2048, 4, 2), (2304, 2500, 300, 2, 3)])
def test_results_at_any_alignment(lib, O, T, K, pad, offset, t):
    """Bases and distances between columns that rule out the wider stores, in whole and in split products."""
    rng = np.random.default_rng(21)
    (wc, ws), w = packed(rng, O, K, mx_util.FP4, 0.05)
    (xc, xs), x = packed(rng, T, K, mx_util.FP4)
    flat, y = room(T, O, t, pad, offset)
    lib.mx_times(wc.data_ptr(), ws.data_ptr(), xc.data_ptr(), xs.data_ptr(), 0, y.data_ptr(), code(lib, t), O + pad, O, T, K, stream())
    check(y, x @ w.T, np.abs(x) @ np.abs(w).T, K / 16, t, "times")
    untouched(flat, y, pad, offset)
    # the gradients of the same layer
    _, d, dy = dense(rng, T, O, "bf16", 0, 0, 1e-2)
    flat, dw = room(K, O, "f32", 0, offset)
    lib.mx_weight_grad(d.data_ptr(), lib.BF16, O, xc.data_ptr(), xs.data_ptr(), 4, dw.data_ptr(), O, K, T, False, stream())
    check(dw, x.T @ dy, np.abs(x).T @ np.abs(dy), T / 16, "f32", "weight gradient")
    untouched(flat, dw, 0, offset)
    flat, dx = room(T, K, t, pad, offset)
    lib.mx_input_grad(d.data_ptr(), lib.BF16, O, wc.data_ptr(), ws.data_ptr(), 4, dx.data_ptr(), code(lib, t), K + pad, O, K, T, stream())
    check(dx, dy @ w, np.abs(dy) @ np.abs(w), O / 16, t, "input gradient")
    untouched(flat, dx, pad, offset)


def test_times_without_inputs_is_the_bias(lib):
    bias = torch.arange(200, dtype=torch.float32, device=DEV)
    y = torch.full((5, 200), GUARD, device=DEV)
    lib.mx_times(0, 0, 0, 0, bias.data_ptr(), y.data_ptr(), lib.F32, 200, 200, 5, 0, stream())
    assert torch.equal(y, bias.expand(5, 200))
    lib.mx_times(0, 0, 0, 0, 0, y.data_ptr(), lib.F32, 200, 200, 5, 0, stream())
    assert not y.any()


@pytest.mark.parametrize("T", [3, 7, 200])
def test_times_scales_and_bad_blocks(lib, T):
    """Each block's scale goes with its own 32 values; a NaN block spoils its row of results and no other."""
    O, K = 130, 300
    rng = np.random.default_rng(5)
    xw = rng.standard_normal((O, K)) * np.exp2(rng.integers(-20, 20, (O, 10)).repeat(32, 1)[:, :K])
    xx = rng.standard_normal((T, K)) * np.exp2(rng.integers(-20, 20, (T, 10)).repeat(32, 1)[:, :K])
    xw[129, 299] = np.nan
    xx[1, 40] = np.inf
    (wc, ws), (xc, xs) = to_dev(*mx_util.pack(xw, 4)), to_dev(*mx_util.pack(xx, 4))
    w, x = mx_util.values(xw, 4), mx_util.values(xx, 4)
    y = torch.zeros(T, O, device=DEV)
    lib.mx_times(wc.data_ptr(), ws.data_ptr(), xc.data_ptr(), xs.data_ptr(), 0, y.data_ptr(), lib.F32, O, O, T, K, stream())
    check(y, x @ w.T, np.abs(x) @ np.abs(w).T, K / 16, "f32", "times with scales")


@pytest.mark.parametrize("T", [2, 20])
def test_times_at_the_ends_of_the_range(lib, T):
    """Scales whose product is in range though each is far from it, and sums that leave the range."""
    O, K = 40, 64
    rng = np.random.default_rng(6)
    xw = rng.standard_normal((O, K)).clip(-1.4, 1.4) * np.exp2(np.linspace(-120, 120, O).round())[:, None]
    xx = np.stack([rng.standard_normal(K).clip(-1.4, 1.4) * 2.0 ** (-100 if t % 2 else 60) for t in range(T)])
    (wc, ws), (xc, xs) = to_dev(*mx_util.pack(xw, 4)), to_dev(*mx_util.pack(xx, 4))
    w, x = mx_util.values(xw, 4), mx_util.values(xx, 4)
    y = torch.zeros(T, O, device=DEV)
    lib.mx_times(wc.data_ptr(), ws.data_ptr(), xc.data_ptr(), xs.data_ptr(), 0, y.data_ptr(), lib.F32, O, O, T, K, stream())
    got, want, mags = y.double().cpu().numpy(), x @ w.T, np.abs(x) @ np.abs(w).T
    top = 3.4028235e38
    # results below the smallest normal may be flushed; where the terms leave the range a sum of fp32 numbers is infinite, or NaN (two
    # terms of opposite signs)
    ok = np.abs(got - want) <= 10 * 2.0 ** -22 * mags + 2.0 ** -126
    over = mags > top / 2
    assert (ok | over).all()
    assert (~np.isfinite(got) | ok)[over].all()


# ---- gradients ----------------------------------------------------------------------------------------------------------------

GRADS = [(128, 128, 64, 0, 0), (1, 1, 1, 0, 0), (132, 512, 256, 0, 0), (64, 33, 5, 0, 0), (512, 363, 64, 0, 0), (300, 130, 129, 3, 0), (2048, 429, 1001, 0, 0), (257, 129, 300, 7, 1),
         (1000, 100, 2000, 8, 8), (72, 700, 513, 0, 0)]


@pytest.mark.parametrize("fmt", [mx_util.FP4, mx_util.INT8])
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("O,I,T,pad,offset", GRADS)
def test_weight_grad(lib, O, I, T, pad, offset, t, fmt):
    rng = np.random.default_rng(O + I + T)
    _, d, dy = dense(rng, T, O, t, pad, offset, 1e-2)
    (xc, xs), x = packed(rng, T, I, fmt)
    want, mags = x.T @ dy, np.abs(x).T @ np.abs(dy)
    flat, dw = room(I, O, "f32")
    planes = {"bf16": 1, "f16": 2, "f32": 3}[t]
    args = (d.data_ptr(), code(lib, t), O + pad, xc.data_ptr(), xs.data_ptr(), fmt, dw.data_ptr(), O, I, T)
    lib.mx_weight_grad(*args, False, stream())
    lib.mx_check(stream())
    check(dw, want, mags, planes * T / 16, "f32", "weight gradient")
    lib.mx_weight_grad(*args, True, stream())
    check(dw, 2 * want, 2 * mags, planes * T / 16 + 2, "f32", "weight gradient, added")
    untouched(flat, dw, 0, 0)


@pytest.mark.parametrize("fmt", [mx_util.FP4, mx_util.INT8])
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("O,I,T,pad,offset", GRADS)
def test_input_grad(lib, O, I, T, pad, offset, t, fmt):
    rng = np.random.default_rng(O + I + T)
    _, d, dy = dense(rng, T, O, t, pad, offset, 1e-2)
    (wc, ws), w = packed(rng, O, I, fmt, 0.05)
    want, mags = dy @ w, np.abs(dy) @ np.abs(w)
    planes = {"bf16": 1, "f16": 2, "f32": 3}[t]
    for t2 in dict.fromkeys((t, "f32")):
        flat, dx = room(T, I, t2, pad, offset)
        lib.mx_input_grad(d.data_ptr(), code(lib, t), O + pad, wc.data_ptr(), ws.data_ptr(), fmt, dx.data_ptr(), code(lib, t2), I + pad, O, I, T, stream())
        lib.mx_check(stream())
        check(dx, want, mags, planes * O / 16, t2, "input gradient")
        untouched(flat, dx, pad, offset)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("O,I,T", [(2048, 1100, 2100), (2049, 1100, 2100), (2301, 1100, 900), (2304, 1300, 900)])
def test_more_tiles_than_sms(lib, O, I, T, t):
    """Several tiles per CTA, by single CTAs and by pairs, the last pair with and without rows for its second CTA; with and without
    16-byte columns of dy."""
    rng = np.random.default_rng(O)
    _, d, dy = dense(rng, T, O, t, 0, 0, 1e-2)
    planes = {"bf16": 1, "f16": 2, "f32": 3}[t]
    (xc, xs), x = packed(rng, T, I, mx_util.INT8)
    _, dw = room(I, O, "f32")
    lib.mx_weight_grad(d.data_ptr(), code(lib, t), O, xc.data_ptr(), xs.data_ptr(), 8, dw.data_ptr(), O, I, T, False, stream())
    lib.mx_check(stream())
    check(dw, x.T @ dy, np.abs(x).T @ np.abs(dy), planes * T / 16, "f32", "weight gradient")
    (wc, ws), w = packed(rng, O, I, mx_util.FP4, 0.05)
    for t2 in dict.fromkeys((t, "f32")):
        _, dx = room(T, I, t2)
        lib.mx_input_grad(d.data_ptr(), code(lib, t), O, wc.data_ptr(), ws.data_ptr(), 4, dx.data_ptr(), code(lib, t2), I, O, I, T, stream())
        lib.mx_check(stream())
        check(dx, dy @ w, np.abs(dy) @ np.abs(w), planes * O / 16, t2, "input gradient")


def test_gradients_of_nothing(lib):
    dw = torch.full((40, 70), GUARD, device=DEV)
    lib.mx_weight_grad(0, lib.BF16, 70, 0, 0, lib.MXINT8, dw.data_ptr(), 70, 40, 0, False, stream())
    assert not dw.any()
    flat, dx = room(9, 40, "bf16", 3)
    lib.mx_input_grad(0, lib.BF16, 0, 0, 0, lib.MXFP4, dx.data_ptr(), lib.BF16, 43, 0, 40, 9, stream())
    assert not dx.any()
    untouched(flat, dx, 3, 0)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_gradients_of_non_finite_values(lib, t):
    """Infinities and NaN reach exactly the results they take part in; so do the extremes of the types."""
    O, I, T = 140, 70, 90
    rng = np.random.default_rng(11)
    dy = rng.standard_normal((T, O))
    dy[3, 5], dy[7, 100], dy[89, 139] = np.inf, np.nan, -np.inf
    big = {"bf16": 3e38, "f16": 65504.0, "f32": 3.4028234e38}[t]
    dy[20, 60], dy[21, 61] = big, -big
    _, d, dy = place(torch.from_numpy(dy), t)
    xx = rng.standard_normal((T, I)) * 1e-3
    xx[3], xx[89] = np.abs(xx[3]) + 1e-3, np.abs(xx[89]) + 1e-3  # no zero meets an infinity
    xx[50, 33] = np.nan
    (xc, xs), x = to_dev(*mx_util.pack(xx, 8)), mx_util.values(xx, 8)
    dw = torch.zeros(I, O, device=DEV)
    lib.mx_weight_grad(d.data_ptr(), code(lib, t), O, xc.data_ptr(), xs.data_ptr(), 8, dw.data_ptr(), O, I, T, False, stream())
    with np.errstate(invalid="ignore"):
        check(dw, x.T @ dy, np.nan_to_num(np.abs(x).T @ np.abs(dy), nan=0.0, posinf=0.0), 3 * T / 16, "f32", "weight gradient with infinities")


@pytest.mark.parametrize("fmt", [mx_util.FP4, mx_util.INT8])
def test_gradient_operands_at_the_ends_of_the_range(lib, fmt):
    """Scales from the smallest to the largest: the expansion to bf16 is exact, subnormals included."""
    T, I, O = 64, 256, 128
    rng = np.random.default_rng(2)
    x = np.zeros((T, I), np.float32)
    for t in range(T):
        x[t] = (rng.integers(-127, 128, I) / 64 * 2.0 ** (t - 127 if t < 32 else 4 * (t - 32))).astype(np.float32)
    (xc, xs), v = to_dev(*mx_util.pack(x, fmt)), mx_util.values(x, fmt)
    dy = np.zeros((T, O))
    # one token per output: results are the operand's values, moved out of fp32's subnormals
    dy[np.arange(T), np.arange(T) * 2] = np.where(np.arange(T) < 32, 2.0 ** 20, 1.0)
    _, d, dy = place(torch.from_numpy(dy), "bf16")
    dw = torch.zeros(I, O, device=DEV)
    lib.mx_weight_grad(d.data_ptr(), lib.BF16, O, xc.data_ptr(), xs.data_ptr(), fmt, dw.data_ptr(), O, I, T, False, stream())
    assert np.array_equal(dw.double().cpu().numpy(), v.T @ dy)


def test_long_sums_keep_their_precision(lib):
    """All-positive sums of 32768 terms: the running sum's own rounding, not more, in the result."""
    T, O, I = 32768, 64, 128
    rng = np.random.default_rng(8)
    _, d, dy = place(torch.from_numpy(rng.random((T, O)) + 0.5), "bf16")
    x = rng.random((T, I)) + 0.5
    (xc, xs), v = to_dev(*mx_util.pack(x, 8)), mx_util.values(x, 8)
    dw = torch.zeros(I, O, device=DEV)
    lib.mx_weight_grad(d.data_ptr(), lib.BF16, O, xc.data_ptr(), xs.data_ptr(), 8, dw.data_ptr(), O, I, T, False, stream())
    want = v.T @ dy
    # T / 16 steps, each off by at most one unit in the last place of the sum
    assert np.abs(dw.double().cpu().numpy() / want - 1).max() <= T / 16 * 2.0 ** -23


# ---- pointwise layers ---------------------------------------------------------------------------------------------------------


def f64(x, act):
    """f and f' in 64 bits."""
    x = torch.from_numpy(x)
    s = torch.sigmoid(x)
    if act == 0:
        y, g = torch.where(x > 0, x, x * 0), (x > 0).double() + x * 0
    elif act == 1:
        y, g = s, s * torch.sigmoid(-x)
    elif act == 2:
        y = torch.tanh(x)
        g = 4 * torch.sigmoid(2 * x) * torch.sigmoid(-2 * x)
    elif act == 3:
        c = 0.5 * torch.special.erfc(-x / 2 ** 0.5)
        y, g = x * c, c + x * torch.exp(-x * x / 2) / (2 * np.pi) ** 0.5
    else:
        y, g = x * s, s + x * s * torch.sigmoid(-x)
    return y.numpy(), g.numpy()


@pytest.mark.parametrize("act", range(5))
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,pad,offset", [(1, 1, 0, 0), (512, 37, 0, 0), (129, 130, 0, 0), (200, 9, 3, 1), (64, 260, 8, 8)])
def test_activation(lib, m, n, pad, offset, t, act):
    rng = np.random.default_rng(m + n + act)
    _, d, x = dense(rng, n, m, t, pad, offset, 2.0)
    _, g, dy = dense(rng, n, m, t, pad, offset)
    codes = torch.zeros(lib.mx_code_bytes(m, n, 8), dtype=torch.uint8, device=DEV)
    scales = torch.zeros(lib.mx_scale_bytes(m, n), dtype=torch.uint8, device=DEV)
    flat, y = room(n, m, t, pad, offset)
    ld = m + pad
    lib.mx_act_forward(d.data_ptr(), code(lib, t), ld, act, y.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), m, n, stream())
    want = mx_util.pack(x, 8)
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])
    flat2, dx = room(n, m, t, pad, offset)
    lib.mx_act_backward(g.data_ptr(), code(lib, t), ld, codes.data_ptr(), scales.data_ptr(), act, dx.data_ptr(), ld, m, n, stream())
    untouched(flat, y, pad, offset)
    untouched(flat2, dx, pad, offset)
    # fp32 arithmetic of a dozen roundings, each at most half a unit of a value no larger than |x| + 1; then the type's rounding
    eps = torch.finfo(TYPES[t]).eps
    wy = f64(x, act)[0]
    kept = mx_util.values(x, 8)
    slope = f64(kept, act)[1]
    for got, ref, size in ((y, wy, np.abs(x) + 1), (dx, dy * slope, np.abs(dy) * (np.abs(kept) + 1))):
        tol = 12 * 2.0 ** -24 * size + eps / 2 * np.abs(ref) + (2.0 ** -25 if t == "f16" else 0)
        err = np.abs(got.double().cpu().numpy() - ref)
        assert (err <= tol).all(), f"worst {np.max(err / tol)}"


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("pads", [(0, 3), (3, 0), (16, 8), (8, 5)])
def test_activation_with_columns_of_different_distances(lib, pads, t):
    """x and y (dy and dx) aligned and not, in every combination; values of the aligned call."""
    m, n = 160, 70
    rng = np.random.default_rng(12)
    _, d, x = dense(rng, n, m, t, pads[0], 0, 2.0)
    same = [torch.zeros(lib.mx_code_bytes(m, n, 8), dtype=torch.uint8, device=DEV), torch.zeros(lib.mx_scale_bytes(m, n), dtype=torch.uint8, device=DEV)]
    flat, y = room(n, m, t, pads[1])
    lib.mx_act_forward(d.data_ptr(), code(lib, t), m + pads[0], lib.ACT_SILU, y.data_ptr(), m + pads[1], same[0].data_ptr(), same[1].data_ptr(), m, n, stream())
    flat2, dx = room(n, m, t, pads[1])
    lib.mx_act_backward(d.data_ptr(), code(lib, t), m + pads[0], same[0].data_ptr(), same[1].data_ptr(), lib.ACT_SILU, dx.data_ptr(), m + pads[1], m, n, stream())
    untouched(flat, y, pads[1], 0)
    untouched(flat2, dx, pads[1], 0)
    near = d.contiguous()
    codes, scales, y0, dx0 = torch.zeros_like(same[0]), torch.zeros_like(same[1]), torch.zeros_like(near), torch.zeros_like(near)
    lib.mx_act_forward(near.data_ptr(), code(lib, t), m, lib.ACT_SILU, y0.data_ptr(), m, codes.data_ptr(), scales.data_ptr(), m, n, stream())
    lib.mx_act_backward(near.data_ptr(), code(lib, t), m, codes.data_ptr(), scales.data_ptr(), lib.ACT_SILU, dx0.data_ptr(), m, m, n, stream())
    want = mx_util.pack(x, 8)
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])
    assert torch.equal(codes, same[0]) and torch.equal(scales, same[1]) and torch.equal(y, y0) and torch.equal(dx, dx0)


@pytest.mark.parametrize("act", range(5))
def test_activation_in_place_and_extremes(lib, act):
    """y over x and dx over dy; far arguments; a NaN block gives NaN gradients and leaves its neighbours alone."""
    x = np.zeros((3, 64), np.float32)
    x[0, :12] = [0.0, -0.0, 1e-30, -1e-30, 90.0, -90.0, 700.0, -700.0, 1e30, -1e30, 20.0, -20.0]
    x[1, :3] = [np.nan, np.inf, 1.0]
    x[2, :4] = [3.4e38, -3.4e38, 1e-45, 5.0]
    d = torch.from_numpy(x).to(DEV)
    codes = torch.zeros(lib.mx_code_bytes(64, 3, 8), dtype=torch.uint8, device=DEV)
    scales = torch.zeros(lib.mx_scale_bytes(64, 3), dtype=torch.uint8, device=DEV)
    lib.mx_act_forward(d.data_ptr(), lib.F32, 64, act, d.data_ptr(), 64, codes.data_ptr(), scales.data_ptr(), 64, 3, stream())
    y = d.double().cpu().numpy()
    ref = f64(x.astype(np.float64), act)[0]
    inf = np.isinf(x)
    assert np.array_equal(np.isnan(y[~inf]), np.isnan(ref[~inf]))
    fine = np.isfinite(x)
    assert (np.abs(y - ref)[fine] <= (12 * 2.0 ** -24 * (np.abs(x) + 1))[fine]).all()
    g = torch.ones(3, 64, device=DEV)
    lib.mx_act_backward(g.data_ptr(), lib.F32, 64, codes.data_ptr(), scales.data_ptr(), act, g.data_ptr(), 64, 64, 3, stream())
    got = g.double().cpu().numpy()
    kept = mx_util.values(x, 8)
    ref = f64(kept, act)[1]
    assert np.isnan(got[1, :32]).all() and not np.isnan(got[1, 32:]).any()
    fine = np.isfinite(kept)
    assert np.isfinite(got[fine]).all()
    assert (np.abs(got - ref)[fine] <= 12 * 2.0 ** -24 * (np.minimum(np.abs(kept), 100.0) + 1)[fine]).all()


@pytest.mark.parametrize("act", range(1, 5))
def test_slope_against_differences(lib, act):
    """f' against (f(x + h) - f(x - h)) / 2h of the forward call itself, at values the 8-bit form holds exactly."""
    x = (np.arange(-127, 129).clip(-127, 127) / 32).astype(np.float32).reshape(8, 32)
    x[:, 0] = 127 / 32  # every block has the same scale
    h = 2.0 ** -7

    def forward(v):
        d = torch.from_numpy(v.astype(np.float32)).to(DEV)
        y = torch.zeros_like(d)
        codes = torch.zeros(lib.mx_code_bytes(32, 8, 8), dtype=torch.uint8, device=DEV)
        scales = torch.zeros(lib.mx_scale_bytes(32, 8), dtype=torch.uint8, device=DEV)
        lib.mx_act_forward(d.data_ptr(), lib.F32, 32, act, y.data_ptr(), 32, codes.data_ptr(), scales.data_ptr(), 32, 8, stream())
        return y.double().cpu().numpy(), codes, scales

    _, codes, scales = forward(x)
    diff = (forward(x + h)[0] - forward(x - h)[0]) / (2 * h)
    dx = torch.ones(8, 32, device=DEV)
    lib.mx_act_backward(dx.data_ptr(), lib.F32, 32, codes.data_ptr(), scales.data_ptr(), act, dx.data_ptr(), 32, 32, 8, stream())
    # third derivatives are below 4: h^2 / 6 * 4; the forward's rounding of values below 5: 12 * 2^-24 * 5 / h
    assert np.abs(dx.double().cpu().numpy() - diff).max() <= h * h * 4 / 6 + 12 * 2.0 ** -24 * 5 / h


# ---- together -----------------------------------------------------------------------------------------------------------------


def quantized(lib, d, m, n, ld, t, fmt, transpose=False):
    pm, pn = (n, m) if transpose else (m, n)
    codes = torch.empty(lib.mx_code_bytes(pm, pn, fmt), dtype=torch.uint8, device=DEV)
    scales = torch.empty(lib.mx_scale_bytes(pm, pn), dtype=torch.uint8, device=DEV)
    lib.mx_quantize(d.data_ptr(), code(lib, t), ld, codes.data_ptr(), scales.data_ptr(), m, n, fmt, transpose, stream())
    return codes, scales


class TwoLayers:
    """y = W2 gelu(W1 x + b1): forward with 4-bit products, x and the hidden layer's input kept in 8 bits, the hidden layer's output in
    its 4-bit form; backward from what was kept; the weight gradients go through the 1-bit aggregation step."""

    def __init__(self, lib, I, H, O, T, t):
        self.lib, self.I, self.H, self.O, self.T, self.t = lib, I, H, O, T, t
        new = lambda n, m, ty=t: torch.zeros(n, m, dtype=TYPES[ty], device=DEV)
        self.x, self.dy = new(T, I), new(T, O)
        self.w1, self.w2, self.b1 = new(I, H, "f32"), new(H, O, "f32"), torch.zeros(H, device=DEV)
        self.z, self.h, self.y, self.dh, self.dz = new(T, H), new(T, H), new(T, O), new(T, H), new(T, H)
        flat = torch.zeros(I * H + H * O, device=DEV)
        self.dw1, self.dw2 = flat[: I * H].view(I, H), flat[I * H:].view(H, O)

    def run(self):
        lib, I, H, O, T, t = self.lib, self.I, self.H, self.O, self.T, code(self.lib, self.t)
        p = lambda pair: (pair[0].data_ptr(), pair[1].data_ptr())
        self.w1q, self.w2q = quantized(lib, self.w1, H, I, H, "f32", lib.MXFP4, True), quantized(lib, self.w2, O, H, O, "f32", lib.MXFP4, True)
        self.xq, self.x8 = quantized(lib, self.x, I, T, I, self.t, lib.MXFP4), quantized(lib, self.x, I, T, I, self.t, lib.MXINT8)
        lib.mx_times(*p(self.w1q), *p(self.xq), self.b1.data_ptr(), self.z.data_ptr(), t, H, H, T, I, stream())
        self.z8 = [torch.empty(lib.mx_code_bytes(H, T, 8), dtype=torch.uint8, device=DEV), torch.empty(lib.mx_scale_bytes(H, T), dtype=torch.uint8, device=DEV)]
        lib.mx_act_forward(self.z.data_ptr(), t, H, lib.ACT_GELU, self.h.data_ptr(), H, *p(self.z8), H, T, stream())
        self.hq = quantized(lib, self.h, H, T, H, self.t, lib.MXFP4)
        lib.mx_times(*p(self.w2q), *p(self.hq), 0, self.y.data_ptr(), t, O, O, T, H, stream())
        lib.mx_weight_grad(self.dy.data_ptr(), t, O, *p(self.hq), lib.MXFP4, self.dw2.data_ptr(), O, H, T, False, stream())
        lib.mx_input_grad(self.dy.data_ptr(), t, O, *p(self.w2q), lib.MXFP4, self.dh.data_ptr(), t, H, O, H, T, stream())
        lib.mx_act_backward(self.dh.data_ptr(), t, H, *p(self.z8), lib.ACT_GELU, self.dz.data_ptr(), H, H, T, stream())
        lib.mx_weight_grad(self.dz.data_ptr(), t, H, *p(self.x8), lib.MXINT8, self.dw1.data_ptr(), H, I, T, False, stream())

    def fill(self, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        for a, s in ((self.x, 1.0), (self.dy, 0.1), (self.w1, 0.05), (self.w2, 0.05), (self.b1, 0.1)):
            a.copy_(torch.empty(a.shape, device=DEV).normal_(0.0, s, generator=g))

    def check(self):
        """Each step against the formula at what the step before it left."""
        v = lambda a: a.double().cpu().numpy()
        q = lambda a, fmt: mx_util.values(v(a), fmt)
        w1, w2 = q(self.w1.t(), 4), q(self.w2.t(), 4)  # [outputs, inputs]
        x4, x8, h4, z8 = q(self.x, 4), q(self.x, 8), q(self.h, 4), q(self.z, 8)
        I, H, O, T, t = self.I, self.H, self.O, self.T, self.t
        planes = {"bf16": 1, "f16": 2, "f32": 3}[t]
        check(self.z, x4 @ w1.T + v(self.b1), np.abs(x4) @ np.abs(w1).T + 1, I / 16, t, "z")
        check(self.y, h4 @ w2.T, np.abs(h4) @ np.abs(w2).T, H / 16, t, "y")
        dy, dh, dz = v(self.dy), v(self.dh), v(self.dz)
        check(self.dw2, h4.T @ dy, np.abs(h4).T @ np.abs(dy), planes * T / 16, "f32", "dw2")
        check(self.dh, dy @ w2, np.abs(dy) @ np.abs(w2), planes * O / 16, t, "dh")
        eps = torch.finfo(TYPES[t]).eps
        want = f64(v(self.z), 3)[0]
        assert (np.abs(v(self.h) - want) <= 12 * 2.0 ** -24 * (np.abs(v(self.z)) + 1) + eps / 2 * np.abs(want) + 2.0 ** -25).all()
        want = dh * f64(z8, 3)[1]
        assert (np.abs(dz - want) <= 12 * 2.0 ** -24 * np.abs(dh) * (np.abs(z8) + 1) + eps / 2 * np.abs(want) + 2.0 ** -25).all()
        check(self.dw1, x8.T @ dz, np.abs(x8).T @ np.abs(dz), planes * T / 16, "f32", "dw1")


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("I,H,O,T", [(363, 512, 132, 256), (429, 264, 100, 77), (64, 32, 16, 1)])
def test_a_training_step(lib, I, H, O, T, t):
    """Forward, backward, aggregation: the gradients that come out are what the aggregation step takes and quantizes."""
    net = TwoLayers(lib, I, H, O, T, t)
    net.fill(7)
    net.run()
    lib.mx_check(stream())
    net.check()
    grads = [net.dw1.clone(), net.dw2.clone()]
    shapes = [(H, I), (O, H)]
    comm = lib.Comm.create(None, 0, 1, 0)
    agg = lib.Aggregator(comm, shapes, 1)
    agg.step([net.dw1.data_ptr(), net.dw2.data_ptr()], stream())
    torch.cuda.synchronize()
    for (m, n), g, d in zip(shapes, grads, (net.dw1, net.dw2)):
        residual, out = torch.zeros_like(g), torch.zeros_like(g)
        packed = torch.zeros(lib.packed_bytes(m, n, 1), dtype=torch.uint8, device=DEV)
        lib.quantize(g.data_ptr(), residual.data_ptr(), residual.data_ptr(), packed.data_ptr(), m, n, 1, True, stream())
        lib.unquantize(packed.data_ptr(), out.data_ptr(), m, n, 1, False, stream())
        torch.cuda.synchronize()
        assert torch.equal(out, d)
    agg.destroy()
    comm.destroy()


def test_a_captured_step_replayed(lib):
    """One graph, three replays over other inputs in the same buffers, an eager step on another stream between them."""
    net, other = TwoLayers(lib, 200, 264, 144, 300, "bf16"), TwoLayers(lib, 200, 264, 144, 300, "bf16")
    net.fill(1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        net.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        net.run()
    for seed in (2, 3, 4):
        net.fill(seed)
        other.fill(seed + 10)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        other.run()
        torch.cuda.synchronize()
        net.check()
        other.check()


def test_products_on_two_streams(lib):
    """Kernels that each want whole SMs, and clusters of them, on two streams at once: the same bits as one after the other."""
    rng = np.random.default_rng(4)
    work = []
    for O, I, T, t in ((2048, 1100, 2100, "bf16"), (132, 512, 256, "f32"), (700, 300, 4096, "bf16"), (512, 363, 64, "f16")):
        _, d, _ = dense(rng, T, O, t, 0, 0, 1e-2)
        (xc, xs), _ = packed(rng, T, I, 8)
        (wc, ws), _ = packed(rng, O, I, 4, 0.05)
        (x4c, x4s), _ = packed(rng, T, I, 4)
        out = [torch.zeros(I, O, device=DEV), torch.zeros(T, I, dtype=TYPES[t], device=DEV), torch.zeros(T, O, device=DEV)]

        def run(O=O, I=I, T=T, t=t, d=d, xc=xc, xs=xs, wc=wc, ws=ws, x4c=x4c, x4s=x4s, out=out):
            lib.mx_weight_grad(d.data_ptr(), code(lib, t), O, xc.data_ptr(), xs.data_ptr(), 8, out[0].data_ptr(), O, I, T, False, stream())
            lib.mx_input_grad(d.data_ptr(), code(lib, t), O, wc.data_ptr(), ws.data_ptr(), 4, out[1].data_ptr(), code(lib, t), I, O, I, T, stream())
            lib.mx_times(wc.data_ptr(), ws.data_ptr(), x4c.data_ptr(), x4s.data_ptr(), 0, out[2].data_ptr(), lib.F32, O, O, T, I, stream())

        work.append((run, out))
    for run, _ in work:
        run()
    torch.cuda.synchronize()
    want = [[o.clone() for o in out] for _, out in work]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(6):
        for _, out in work:
            for o in out:
                o.zero_()
        torch.cuda.synchronize()
        for k, (run, _) in enumerate(work):
            with torch.cuda.stream(streams[(k + turn) % 2]):
                run()
        lib.mx_check(streams[0].cuda_stream)
        torch.cuda.synchronize()
        for (_, out), w in zip(work, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))


def test_products_with_columns_far_apart(lib):
    """Columns 2^31 values apart: the third begins beyond 2^32."""
    O, I, T, ld = 64, 40, 3, (1 << 31) + 64
    rng = np.random.default_rng(9)
    big = torch.zeros(2 * ld + 128, dtype=torch.bfloat16, device=DEV)
    dy = torch.from_numpy(rng.standard_normal((T, O))).to(torch.bfloat16)
    (xc, xs), x = packed(rng, T, I, 8)
    (wc, ws), w = packed(rng, O, I, 4)
    v = dy.double().numpy()
    for off in (0, 1):  # the copy engine's way, and the loaders'
        for j in range(T):
            big[off + j * ld:off + j * ld + O] = dy[j].to(DEV)
        at = big.data_ptr() + 2 * off
        dw = torch.zeros(I, O, device=DEV)
        lib.mx_weight_grad(at, lib.BF16, ld, xc.data_ptr(), xs.data_ptr(), 8, dw.data_ptr(), O, I, T, False, stream())
        check(dw, x.T @ v, np.abs(x).T @ np.abs(v), 1, "f32", "weight gradient")
        dx = torch.zeros(T, I, device=DEV)
        lib.mx_input_grad(at, lib.BF16, ld, wc.data_ptr(), ws.data_ptr(), 4, dx.data_ptr(), lib.F32, I, O, I, T, stream())
        check(dx, v @ w, np.abs(v) @ np.abs(w), O / 16, "f32", "input gradient")
    near = dy.to(DEV)
    lib.mx_input_grad(near.data_ptr(), lib.BF16, O, wc.data_ptr(), ws.data_ptr(), 4, big.data_ptr(), lib.BF16, ld, O, I, T, stream())
    check(torch.stack([big[j * ld:j * ld + I] for j in range(T)]), v @ w, np.abs(v) @ np.abs(w), O / 16, "bf16", "input gradient far apart")


@pytest.mark.parametrize("O,T", [(2200, 2500), (300, 40)])
def test_large_products_of_nothing(lib, O, T):
    bias = torch.arange(O, dtype=torch.float32, device=DEV)
    y = torch.full((T, O), GUARD, device=DEV)
    lib.mx_times(0, 0, 0, 0, bias.data_ptr(), y.data_ptr(), lib.F32, O, O, T, 0, stream())
    assert torch.equal(y, bias.expand(T, O))
    y.fill_(GUARD)
    lib.mx_weight_grad(0, lib.BF16, O, 0, 0, 8, y.data_ptr(), O, T, 0, False, stream())
    assert not y.any()
    y.fill_(GUARD)
    lib.mx_input_grad(0, lib.BF16, 0, 0, 0, 4, y.data_ptr(), lib.F32, O, 0, O, T, stream())
    assert not y.any()


INF = float("inf")
# f at +infinity and at -infinity: x * Phi(x) and x * sigmoid(x) have -infinity times 0 there
AT_INFINITY = [(INF, 0.0), (1.0, 0.0), (1.0, -1.0), (INF, np.nan), (INF, np.nan)]


@pytest.mark.parametrize("act", range(5))
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 3])
def test_activation_of_infinities(lib, t, act, pad):
    """What an overflowed product feeds the layer: f at both infinities, and next to them values that are not touched by it."""
    x = np.full((4, 64), 0.5)
    x[0, 5], x[1, 40], x[2, 0], x[2, 63], x[3, 20] = INF, -INF, INF, -INF, np.nan
    _, d, _ = place(torch.from_numpy(x), t, pad)
    flat, y = room(4, 64, t, pad)
    codes = torch.zeros(lib.mx_code_bytes(64, 4, 8), dtype=torch.uint8, device=DEV)
    scales = torch.zeros(lib.mx_scale_bytes(64, 4), dtype=torch.uint8, device=DEV)
    lib.mx_act_forward(d.data_ptr(), code(lib, t), 64 + pad, act, y.data_ptr(), 64 + pad, codes.data_ptr(), scales.data_ptr(), 64, 4, stream())
    got = y.double().cpu().numpy()
    high, low = AT_INFINITY[act]
    assert np.array_equal([got[0, 5], got[2, 0]], [high, high])
    assert np.array_equal([got[1, 40], got[2, 63]], [low, low], equal_nan=True)
    assert np.isnan(got[3, 20])
    # 0.5: as in test_activation
    want = f64(np.array([0.5]), act)[0][0]
    fine = x == 0.5
    assert (np.abs(got - want)[fine] <= 12 * 2.0 ** -24 * 1.5 + torch.finfo(TYPES[t]).eps / 2 * abs(want)).all()
    untouched(flat, y, pad, 0)


def sweep(lo, hi, n):
    """[columns, 32]: magnitudes from lo to hi, their logarithms evenly spread, both signs."""
    v = np.exp(np.linspace(np.log(lo), np.log(hi), n))
    return np.concatenate([v, -v]).reshape(-1, 32)


@pytest.mark.parametrize("act", range(1, 5))
def test_functions_in_fp32_keep_their_relative_precision(lib, act):
    """fp32 in, fp32 out: a few units (of 2^-23) of the result itself, tails of the sigmoid and of GELU included.

    An exponential is good to 3 units (the hardware's 2, its argument's rest put back), a reciprocal to 1, sums and products to half a unit.
    Sigmoid and SiLU: 3, 1 + e and its reciprocal 1.5, two products 1.  Slopes of sigmoid and tanh: 3, twice 1.5, two products 1: 7.  tanh
    itself: 2.  GELU: t = 1 / (1 + c x) is off by 1.5 units, which the tail's form makes 3.6 of, its polynomial's fit and steps 2, the
    exponential 3, three products 1.5: 10.  Slopes of GELU and SiLU: sums of two terms, each as good as that."""
    x = sweep(1e-30, 88.0, 4096).astype(np.float32)
    n = x.shape[0]
    d = torch.from_numpy(x).to(DEV)
    y, dx = torch.zeros_like(d), torch.ones_like(d)
    codes = torch.zeros(lib.mx_code_bytes(32, n, 8), dtype=torch.uint8, device=DEV)
    scales = torch.zeros(lib.mx_scale_bytes(32, n), dtype=torch.uint8, device=DEV)
    lib.mx_act_forward(d.data_ptr(), lib.F32, 32, act, y.data_ptr(), 32, codes.data_ptr(), scales.data_ptr(), 32, n, stream())
    lib.mx_act_backward(dx.data_ptr(), lib.F32, 32, codes.data_ptr(), scales.data_ptr(), act, dx.data_ptr(), 32, 32, n, stream())
    unit, least = 2.0 ** -23, 8 * 2.0 ** -149  # subnormal factors and results: roundings of the smallest step
    units = 10 if act == 3 else 7
    want = f64(x.astype(np.float64), act)[0]
    err = np.abs(y.double().cpu().numpy() - want)
    assert (err <= units * unit * np.abs(want) + least * (np.abs(x) + 1)).all(), f"worst {np.max(err / (unit * np.abs(want) + least))} units"
    kept = mx_util.values(x, 8)
    want = f64(kept, act)[1]
    s = torch.sigmoid(torch.from_numpy(kept)).numpy()
    if act == 3:
        size = 0.5 * torch.special.erfc(-torch.from_numpy(kept) / 2 ** 0.5).numpy() + 0.4 * np.abs(kept) * np.exp(-kept ** 2 / 2)
    elif act == 4:
        size = s + np.abs(kept) * s * torch.sigmoid(-torch.from_numpy(kept)).numpy()
    else:
        size = np.abs(want)
    err = np.abs(dx.double().cpu().numpy() - want)
    assert (err <= units * unit * size + least * (np.abs(kept) + 1)).all(), f"worst {np.max(err / (unit * size + least))} units"


@pytest.mark.parametrize("act", range(5))
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_functions_in_half_precision_are_rounded_once(lib, t, act):
    """16-bit results: half a step of the value itself, tails included, and what fp32 loses before that rounding.

    exp(-x^2 / 2) and exp(-|x|) with the hardware's exponential: its argument, up to 126 powers of two, is rounded twice (2^-24 each, times
    126 ln 2: 2^-17 of the result), itself within 2^-22; the polynomial of GELU's tail within 2.5e-5; tanh from 0.02 on loses
    1 / 0.04 of 2^-22 to a difference.  Together below 2^-14.  Exponentials below 2^-126 are 0, and with them results below that times |x|."""
    x = torch.from_numpy(sweep(1e-4, 88.0, 8192)).to(TYPES[t])
    n = x.shape[0]
    d = x.to(DEV)
    x = x.double().numpy()
    y, dx = torch.zeros_like(d), torch.ones_like(d)
    codes = torch.zeros(lib.mx_code_bytes(32, n, 8), dtype=torch.uint8, device=DEV)
    scales = torch.zeros(lib.mx_scale_bytes(32, n), dtype=torch.uint8, device=DEV)
    lib.mx_act_forward(d.data_ptr(), code(lib, t), 32, act, y.data_ptr(), 32, codes.data_ptr(), scales.data_ptr(), 32, n, stream())
    lib.mx_act_backward(dx.data_ptr(), code(lib, t), 32, codes.data_ptr(), scales.data_ptr(), act, dx.data_ptr(), 32, 32, n, stream())
    eps = torch.finfo(TYPES[t]).eps
    kept = mx_util.values(x, 8)
    s = torch.sigmoid(torch.from_numpy(kept)).numpy()
    want = f64(kept, act)[1]
    terms = np.abs(want)  # of a slope that is a sum: the terms' magnitudes
    if act == 3:
        terms = 0.5 * torch.special.erfc(-torch.from_numpy(kept) / 2 ** 0.5).numpy() + 0.4 * np.abs(kept) * np.exp(-kept ** 2 / 2)
    if act == 4:
        terms = s + np.abs(kept) * s * torch.sigmoid(-torch.from_numpy(kept)).numpy()
    for got, ref, size, at in ((y, f64(x, act)[0], None, x), (dx, want, terms, kept)):
        size = np.abs(ref) if size is None else size
        least = (2.0 ** -25 if t == "f16" else 0) + 2.0 ** -126 * (np.abs(at) + 1)
        err = np.abs(got.double().cpu().numpy() - ref)
        tol = eps / 2 * np.abs(ref) + 2.0 ** -14 * size * (1 + eps) + least
        assert (err <= tol).all(), f"worst {np.max(err / tol)}, at {np.argmax(err / tol)}"


# ---- how much a long sum may lose ---------------------------------------------------------------------------------------------
# The tensor cores truncate the running sum to fp32.  The worst case: 1 first, then instructions whose products add up to 3/4 of the
# sum's unit in the last place, 2^-23, all of which the truncation drops.  A chain of n instructions loses 3/4 n units that way; the chains
# after it hold multiples of 3/4 unit of their own and lose nothing, and n being a multiple of 4 they are added exactly.
UNIT = 2.0 ** -23


def ones(lib, m, n, fmt):
    """A packed m x n matrix of ones."""
    x = torch.ones(n, m, dtype=torch.bfloat16, device=DEV)
    return quantized(lib, x, m, n, m, "bf16", fmt)


def lost(out, want):
    """Least and most of what is missing from `want`, in units of 2^-23."""
    return (want - float(out.max())) / UNIT, (want - float(out.min())) / UNIT


@pytest.mark.parametrize("O,T,K", [(128, 16, 131072), (128, 48, 131072), (128, 100, 131072), (200, 250, 131072), (4096, 2304, 16384)])
def test_long_sums_of_the_product(lib, O, T, K):
    """64 products an instruction; 32 instructions to a chain, 64 where a tile is 256 wide (more than 128 tokens)."""
    w = torch.full((K, O), 0.75 * UNIT / 64, device=DEV)  # O x K
    w[0] = 1.0
    w[1:32] = 0.0  # they share a scale with the 1
    wc, ws = quantized(lib, w, O, K, O, "f32", lib.MXFP4, True)
    xc, xs = ones(lib, K, T, lib.MXFP4)
    y = torch.zeros(T, O, device=DEV)
    lib.mx_times(wc.data_ptr(), ws.data_ptr(), xc.data_ptr(), xs.data_ptr(), 0, y.data_ptr(), lib.F32, O, O, T, K, stream())
    lib.mx_check(stream())
    least, most = lost(y, 1.0 + (K - 32) * 0.75 * UNIT / 64)
    assert least >= 0 and most <= 0.75 * (32 if T <= 128 else 64)


def test_sums_for_fp16_results(lib):
    """A chain for an fp16 result has 128 instructions at most, and loses 96 of the 8192 units of 2^-23 that fp16's step at 1 has.  The
    sums here lie 150 or more units above the middle between two fp16 values, those of a chain four times as long would lie below it."""
    tie, small = 1.0 + 2.0 ** -11, 0.75 * UNIT
    step = 2.0 ** -10

    # dx: 16 products an instruction (and as many for the second plane of an fp16 dy, which is 0).  Splits take an eighth each.
    for t, O in (("f16", 8 * 8192), ("bf16", 8 * 16384)):
        I, T = 128, 64
        w = torch.full((O, I), small / 16, device=DEV)
        w[:16] = 0.0
        w[0], w[1] = 1.0, 2.0 ** -11
        wc, ws = quantized(lib, w, I, O, I, "f32", lib.MXFP4)
        dy = torch.ones(T, O, dtype=TYPES[t], device=DEV)
        dy[:, O // 8:] = 0.0  # one CTA's part
        want = tie + (O // 8 - 16) * small / 16
        assert want - tie > 150 * UNIT
        dx = torch.zeros(T, I, dtype=torch.float16, device=DEV)
        lib.mx_input_grad(dy.data_ptr(), code(lib, t), O, wc.data_ptr(), ws.data_ptr(), lib.MXFP4, dx.data_ptr(), lib.F16, I, O, I, T, stream())
        lib.mx_check(stream())
        assert bool((dx == 1.0 + step).all())

    O, T, K = 128, 16, 8 * 65536  # 64 products an instruction
    w = torch.full((K, O), small / 64, device=DEV)
    w[:64] = 0.0
    w[0], w[32] = 1.0, 2.0 ** -11
    wc, ws = quantized(lib, w, O, K, O, "f32", lib.MXFP4, True)
    x = torch.ones(T, K, device=DEV)
    x[:, K // 8:] = 0.0
    xc, xs = quantized(lib, x, K, T, K, "f32", lib.MXFP4)
    y = torch.zeros(T, O, dtype=torch.float16, device=DEV)
    lib.mx_times(wc.data_ptr(), ws.data_ptr(), xc.data_ptr(), xs.data_ptr(), 0, y.data_ptr(), lib.F16, O, O, T, K, stream())
    lib.mx_check(stream())
    assert bool((y == 1.0 + step).all())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_results_and_alignment(lib, t):
    """Everything but the gradients of a bf16 dy has the same bits at every alignment; those agree within what their sums may lose."""
    rng = np.random.default_rng(31)
    O, I, T = 2304, 700, 1100
    _, near, dy = dense(rng, T, O, t, 0, 0, 1e-2)
    _, far, _ = place(torch.from_numpy(dy), t, 3, 1)
    (xc, xs), x = packed(rng, T, I, mx_util.INT8)
    (wc, ws), w = packed(rng, O, I, mx_util.FP4, 0.05)
    results = []
    for d, ld, pad, offset in ((near, O, 0, 0), (far, O + 3, 3, 1)):
        flat, dw = room(I, O, "f32", 0, offset)
        lib.mx_weight_grad(d.data_ptr(), code(lib, t), ld, xc.data_ptr(), xs.data_ptr(), 8, dw.data_ptr(), O, I, T, False, stream())
        flat2, dx = room(T, I, t, pad, offset)
        lib.mx_input_grad(d.data_ptr(), code(lib, t), ld, wc.data_ptr(), ws.data_ptr(), 4, dx.data_ptr(), code(lib, t), I + pad, O, I, T, stream())
        codes, scales = run_quantize(lib, d, O, T, t, ld, 8, False)
        turned, turnedScales = run_quantize(lib, d, O, T, t, ld, 4, True)
        flat3, back = room(T, O, t, pad, offset)
        lib.mx_unquantize(codes.data_ptr(), scales.data_ptr(), back.data_ptr(), code(lib, t), O + pad, O, T, 8, stream())
        flat4, y = room(T, O, t, pad, offset)
        x4 = to_dev(*mx_util.pack(x, 4))
        lib.mx_times(wc.data_ptr(), ws.data_ptr(), x4[0].data_ptr(), x4[1].data_ptr(), 0, y.data_ptr(), code(lib, t), O + pad, O, T, I, stream())
        torch.cuda.synchronize()
        results.append([codes, scales, turned, turnedScales, back.clone(), y.clone(), dw.clone(), dx.clone()])
    for k, (a, b) in enumerate(zip(*results)):
        if t != "bf16" or k < 6:
            assert torch.equal(a, b), k
    for dw, dx in ((r[6], r[7]) for r in results):
        planes = {"bf16": 1, "f16": 2, "f32": 3}[t]
        check(dw, x.T @ dy, np.abs(x).T @ np.abs(dy), planes * T / 16, "f32", "weight gradient")
        check(dx, dy @ w, np.abs(dy) @ np.abs(w), planes * O / 16, t, "input gradient")


def test_a_wait_that_runs_out_is_reported(lib):
    """A bounded wait on a barrier that nothing completes, with a limit of 20 ms: the kernel ends, the next check says so, once."""
    lib.mx_check(stream())
    lib.mx_wait_selftest(20_000_000, stream())
    with pytest.raises(lib.QaggError) as e:
        lib.mx_check(stream())
    assert "error -5" in str(e.value)
    lib.mx_check(stream())
    # the report is the device's: a check of any stream brings it, after that stream's work
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    lib.mx_wait_selftest(1_000_000, a.cuda_stream)
    a.synchronize()
    with pytest.raises(lib.QaggError):
        lib.mx_check(b.cuda_stream)
    lib.mx_check(a.cuda_stream)


def test_checks_from_several_threads_report_once(lib):
    """Eight threads check at the same time: one of them gets the report."""
    import threading
    for _ in range(10):
        lib.mx_wait_selftest(1000, stream())
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(8)], []

        def look(s):
            torch.cuda.set_device(0)
            try:
                lib.mx_check(s.cuda_stream)
            except lib.QaggError as e:
                got.append(str(e))

        threads = [threading.Thread(target=look, args=(s,)) for s in streams]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert len(got) == 1 and "error -5" in got[0], got
    lib.mx_check(stream())


def test_check_beside_a_capture(lib):
    """While a stream is being captured another one can be checked; the captured one is refused, and the capture goes on."""
    x = torch.randn(64, 128, device=DEV)
    codes = torch.zeros(lib.mx_code_bytes(128, 64, 8), dtype=torch.uint8, device=DEV)
    scales = torch.zeros(lib.mx_scale_bytes(128, 64), dtype=torch.uint8, device=DEV)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        lib.mx_check(other.cuda_stream)
        with pytest.raises(lib.QaggError) as e:
            lib.mx_check(stream())
        assert "error -4" in str(e.value)
        lib.mx_quantize(x.data_ptr(), lib.F32, 128, codes.data_ptr(), scales.data_ptr(), 128, 64, lib.MXINT8, False, stream())
    graph.replay()
    torch.cuda.synchronize()
    want = mx_util.pack(x.double().cpu().numpy(), mx_util.INT8)
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])


@pytest.mark.parametrize("t,O,I,T,chain", [("bf16", 128, 128, 32768, 32), ("bf16", 2304, 2304, 8192, 32), ("bf16", 1280, 2304, 16384, 64), ("bf16", 2303, 4096, 8192, 32),
                                           ("f32", 2304, 4096, 4096, 32), ("f32", 130, 128, 8192, 32), ("f16", 2304, 4096, 4096, 32)])
def test_long_sums_of_the_weight_gradient(lib, t, O, I, T, chain):
    """16 products an instruction, split and whole, by single CTAs and by pairs (64 instructions where dy is bf16), with and without loaders."""
    small = 0.75 * UNIT / 16
    up = 2.0 ** 14 if t == "f16" else 1.0  # fp16 holds no 2^-28: all values larger
    dy = torch.full((T, O), small * up, dtype=TYPES[t], device=DEV)
    dy[0] = up
    xc, xs = ones(lib, I, T, lib.MXINT8)
    dw = torch.zeros(I, O, device=DEV)
    lib.mx_weight_grad(dy.data_ptr(), code(lib, t), O, xc.data_ptr(), xs.data_ptr(), lib.MXINT8, dw.data_ptr(), O, I, T, False, stream())
    lib.mx_check(stream())
    least, most = lost(dw / up, 1.0 + (T - 1) * small)
    # the first instruction has 15 small values: a sixteenth of 3/4 unit that the total lacks
    assert least >= -0.5 and most <= 0.75 * chain + 0.5


@pytest.mark.parametrize("t,O,I,T,chain", [("bf16", 32768, 128, 64, 32), ("bf16", 8192, 1280, 2304, 32), ("bf16", 8192, 2048, 2048, 64), ("f32", 4096, 2304, 4096, 32),
                                           ("f16", 4096, 2304, 4096, 32)])
def test_long_sums_of_the_input_gradient(lib, t, O, I, T, chain):
    small = 0.75 * UNIT / 16
    up = 2.0 ** 14 if t == "f16" else 1.0
    dy = torch.full((T, O), small * up, dtype=TYPES[t], device=DEV)
    dy[:, 0] = up
    wc, ws = ones(lib, I, O, lib.MXFP4)
    dx = torch.zeros(T, I, device=DEV)
    lib.mx_input_grad(dy.data_ptr(), code(lib, t), O, wc.data_ptr(), ws.data_ptr(), lib.MXFP4, dx.data_ptr(), lib.F32, I, O, I, T, stream())
    lib.mx_check(stream())
    least, most = lost(dx / up, 1.0 + (O - 1) * small)
    assert least >= -0.5 and most <= 0.75 * chain + 0.5


@pytest.mark.parametrize("weight", [True, False])
@pytest.mark.parametrize("t,D", [("f32", (2304, 4096, 4096)), ("f32", (200, 130, 2048)), ("f16", (2304, 4096, 4096)), ("f16", (200, 130, 2048))])
def test_every_plane_of_dy_counts(lib, t, D, weight):
    """Values of one sign with all significant bits set.  fp32: the last of three bf16 terms is 2^-16 of the value, fp16: the second of two is
    7 * 2^-11; the sum's own error is below both: chains of 24 (fp16: 32) instructions, each off by a unit of the sum so far, half the
    chain's sum on average (16.5 units), and at most 96 chains, each addition off by half a unit of the sum so far (24 units)."""
    v = 2.0 - 2.0 ** -23 if t == "f32" else 2.0 - 2.0 ** -10
    A, B, C = D  # results A x B, contraction C
    dy = torch.full((C, A) if weight else (B, C), v, dtype=TYPES[t], device=DEV)
    out = torch.zeros((B, A), device=DEV)
    if weight:
        xc, xs = ones(lib, B, C, lib.MXINT8)
        lib.mx_weight_grad(dy.data_ptr(), code(lib, t), A, xc.data_ptr(), xs.data_ptr(), lib.MXINT8, out.data_ptr(), A, B, C, False, stream())
    else:
        wc, ws = ones(lib, A, C, lib.MXFP4)
        lib.mx_input_grad(dy.data_ptr(), code(lib, t), C, wc.data_ptr(), ws.data_ptr(), lib.MXFP4, out.data_ptr(), lib.F32, A, C, A, B, stream())
    lib.mx_check(stream())
    want = v * C
    worst = max(abs(float(out.max()) - want), abs(float(out.min()) - want))
    assert worst <= 41 * UNIT * want  # 4.9e-6; without the last plane 1.5e-5 (fp16: 1.7e-3)
    assert worst < 2.0 ** -17 * want


@pytest.mark.parametrize("O,I,T,t", [(2304, 4096, 8192, "f32"), (1280, 2304, 16384, "bf16"), (128, 128, 32768, "bf16"), (130, 140, 32768, "f16")])
def test_sums_of_one_sign(lib, O, I, T, t):
    """Random values of one sign: what a chain of n (64 at most) truncating instructions loses, a unit of the sum so far each, is on average
    half of n units of the chain's sum; the additions of m chains, half a unit of the sum so far, a quarter of m units at most."""
    g = torch.Generator(device=DEV).manual_seed(3)
    dy = (torch.rand(T, O, device=DEV, generator=g) + 0.5).to(TYPES[t])
    x = torch.rand(T, I, device=DEV, generator=g) + 0.5
    xc, xs = quantized(lib, x, I, T, I, "f32", lib.MXINT8)
    values = torch.zeros(T, I, device=DEV)
    lib.mx_unquantize(xc.data_ptr(), xs.data_ptr(), values.data_ptr(), lib.F32, I, I, T, lib.MXINT8, stream())
    dw = torch.zeros(I, O, device=DEV)
    lib.mx_weight_grad(dy.data_ptr(), code(lib, t), O, xc.data_ptr(), xs.data_ptr(), lib.MXINT8, dw.data_ptr(), O, I, T, False, stream())
    rows = torch.arange(0, I, max(1, I // 64), device=DEV)
    want = values[:, rows].double().t() @ dy.double()
    planes = {"bf16": 1, "f16": 2, "f32": 3}[t]
    pair = t == "bf16" and O == 1280
    n = 64 if pair else 32 // (4 * planes) * 4 * planes
    m = T * planes / 16 / n
    assert float((dw[rows].double() / want - 1).abs().max()) <= (n / 2 + 2 + m / 4) * UNIT


@pytest.mark.parametrize("t,t2", [("f32", "f16"), ("f32", "bf16"), ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("fmt", [mx_util.FP4, mx_util.INT8])
@pytest.mark.parametrize("O,I,T,pad,offset", [(132, 512, 256, 0, 0), (257, 129, 300, 7, 1), (520, 2304, 4096, 0, 0)])
def test_input_grad_of_another_type(lib, O, I, T, pad, offset, fmt, t, t2):
    """dx of a 16-bit type that is not dy's."""
    rng = np.random.default_rng(O + I + T)
    _, d, dy = dense(rng, T, O, t, pad, offset, 1e-2)
    (wc, ws), w = packed(rng, O, I, fmt, 0.05)
    flat, dx = room(T, I, t2, pad, offset)
    lib.mx_input_grad(d.data_ptr(), code(lib, t), O + pad, wc.data_ptr(), ws.data_ptr(), fmt, dx.data_ptr(), code(lib, t2), I + pad, O, I, T, stream())
    lib.mx_check(stream())
    check(dx, dy @ w, np.abs(dy) @ np.abs(w), {"bf16": 1, "f16": 2, "f32": 3}[t] * O / 16, t2, "input gradient")
    untouched(flat, dx, pad, offset)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("O,T,K", [(130, 40, 40000), (200, 130, 20000), (4096, 2304, 8448)])
def test_times_with_several_chains(lib, O, T, K, t):
    """Contractions that hand the accumulator over within a tile, at every width: 64, 128 and 256."""
    rng = np.random.default_rng(K)
    (wc, ws), w = packed(rng, O, K, mx_util.FP4, 0.05)
    (xc, xs), x = packed(rng, T, K, mx_util.FP4)
    y = torch.zeros(T, O, dtype=TYPES[t], device=DEV)
    lib.mx_times(wc.data_ptr(), ws.data_ptr(), xc.data_ptr(), xs.data_ptr(), 0, y.data_ptr(), code(lib, t), O, O, T, K, stream())
    lib.mx_check(stream())
    check(y, x @ w.T, np.abs(x) @ np.abs(w).T, K / 16, t, "times")


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("O,T,K,pad", [(9304, 1, 1100, 0), (7105, 1, 64, 3), (9304, 2, 2048, 0), (7200, 2, 429, 5), (7111, 4, 96, 0)])
def test_times_of_few_tokens_and_many_outputs(lib, O, T, K, pad, t):
    """Two rows a warp, 32 apart: the last ones beyond the matrix too."""
    rng = np.random.default_rng(O + K)
    (wc, ws), w = packed(rng, O, K, mx_util.FP4, 0.05)
    (xc, xs), x = packed(rng, T, K, mx_util.FP4)
    bias = rng.standard_normal(O).astype(np.float32)
    bd = torch.from_numpy(bias).to(DEV)
    flat, y = room(T, O, t, pad)
    lib.mx_times(wc.data_ptr(), ws.data_ptr(), xc.data_ptr(), xs.data_ptr(), bd.data_ptr(), y.data_ptr(), code(lib, t), O + pad, O, T, K, stream())
    check(y, x @ w.T + bias, np.abs(x) @ np.abs(w).T + np.abs(bias), K / 16, t, "times")
    untouched(flat, y, pad, 0)


@pytest.mark.parametrize("weight", [True, False])
@pytest.mark.parametrize("A,B", [(130, 40), (2304, 4096)])
def test_small_planes_are_added_first(lib, A, B, weight):
    """64 values 1 + 3 * 2^-23, in bf16 terms 1 and 3 * 2^-23.  The small ones first: 3 * 2^-17, then four times 16, all of it exact in 24 bits.
    The large ones first make 64, whose unit is 2^-17: each of four instructions with 3/4 of it is lost."""
    C = 64
    dy = torch.full((C, A) if weight else (B, C), 1.0 + 3 * UNIT, device=DEV)
    out = torch.zeros((B, A), device=DEV)
    if weight:
        xc, xs = ones(lib, B, C, lib.MXINT8)
        lib.mx_weight_grad(dy.data_ptr(), lib.F32, A, xc.data_ptr(), xs.data_ptr(), lib.MXINT8, out.data_ptr(), A, B, C, False, stream())
    else:
        wc, ws = ones(lib, A, C, lib.MXFP4)
        lib.mx_input_grad(dy.data_ptr(), lib.F32, C, wc.data_ptr(), ws.data_ptr(), lib.MXFP4, out.data_ptr(), lib.F32, A, C, A, B, stream())
    lib.mx_check(stream())
    assert bool((out == 64.0 + 3 * 2.0 ** -17).all())


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_fp16_results_with_several_chains(lib, t):
    """Chains for fp16 results end within these contractions: pairs with one accumulator (bf16 dy, the product) and loaders with two."""
    O, I, T = 4200, 2048, 2100
    rng = np.random.default_rng(17)
    _, d, dy = dense(rng, T, O, t, 0, 0, 1e-2)
    (wc, ws), w = packed(rng, O, I, mx_util.FP4, 0.05)
    dx = torch.zeros(T, I, dtype=torch.float16, device=DEV)
    lib.mx_input_grad(d.data_ptr(), code(lib, t), O, wc.data_ptr(), ws.data_ptr(), 4, dx.data_ptr(), lib.F16, I, O, I, T, stream())
    lib.mx_check(stream())
    check(dx, dy @ w, np.abs(dy) @ np.abs(w), {"bf16": 1, "f16": 2, "f32": 3}[t] * O / 16, "f16", "input gradient")


def test_product_for_fp16_with_several_chains(lib):
    O, T, K = 2304, 4096, 16640
    g = torch.Generator(device=DEV).manual_seed(5)
    w, x = torch.randn(K, O, device=DEV, generator=g) * 0.05, torch.randn(T, K, device=DEV, generator=g)
    wq, xq = quantized(lib, w, O, K, O, "f32", lib.MXFP4, True), quantized(lib, x, K, T, K, "f32", lib.MXFP4)
    wv, xv = torch.zeros(O, K, device=DEV), torch.zeros(T, K, device=DEV)
    lib.mx_unquantize(wq[0].data_ptr(), wq[1].data_ptr(), wv.data_ptr(), lib.F32, K, K, O, lib.MXFP4, stream())
    lib.mx_unquantize(xq[0].data_ptr(), xq[1].data_ptr(), xv.data_ptr(), lib.F32, K, K, T, lib.MXFP4, stream())
    y = torch.zeros(T, O, dtype=torch.float16, device=DEV)
    lib.mx_times(wq[0].data_ptr(), wq[1].data_ptr(), xq[0].data_ptr(), xq[1].data_ptr(), 0, y.data_ptr(), lib.F16, O, O, T, K, stream())
    lib.mx_check(stream())
    rows = torch.arange(0, T, 37, device=DEV)
    want, mags = xv[rows].double() @ wv.double().t(), xv[rows].abs().double() @ wv.abs().double().t()
    check(y[rows], want.cpu().numpy(), mags.cpu().numpy(), K / 16, "f16", "times")
