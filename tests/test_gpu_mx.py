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
@pytest.mark.parametrize("O,I,T", [(2048, 1100, 2100), (2049, 1100, 2100)])
def test_more_tiles_than_sms(lib, O, I, T, t):
    """Several tiles per CTA, with and without 16-byte columns of dy."""
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
