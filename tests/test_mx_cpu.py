"""Microscaled matrices without a device: sizes, refusals, and the restatement in mx_util against values worked out by hand."""
import numpy as np
import pytest

import mx_util


@pytest.fixture(scope="module")
def lib():
    from cntk_b200 import build
    build.build()
    from cntk_b200 import lib as L
    return L


def test_restatement_by_hand():
    x = np.zeros((1, 33))
    x[0, :8] = [6.0, 5.0, 0.25, -0.75, 3.5, 1.2, -6.9, 0.0]
    # largest 6.9: floor(log2) = 2, X = 0.  5 lies between 4 and 6: tie, even code 6 (4).  0.25: tie, 0.  -0.75: tie, -1.  3.5: tie, 4
    assert mx_util.values(x, mx_util.FP4)[0, :8].tolist() == [6, 4, 0, -1, 4, 1, -6, 0]
    x[0, 32] = 1.9921875  # 127.5 / 64: a tie between 127 and 128, which is not held
    assert mx_util.values(x, mx_util.INT8)[0, 32] == 127 / 64
    codes, scales = mx_util.pack(x, mx_util.FP4)
    assert codes[0] == 0x67 and codes.size == 32 and scales.size == 512
    assert scales[0] == 127 and scales[1] == 125 and not scales[2:].any()


def test_tiles_of_scales():
    s = np.arange(130 * 5, dtype=np.int64).reshape(130, 5) % 251
    t = mx_util.tile(s.astype(np.uint8))
    assert t.size == 2 * 2 * 512
    for j, b in ((0, 0), (31, 3), (32, 0), (127, 4), (128, 1), (129, 4)):
        at = (j // 128 * 2 + b // 4) * 512 + j % 32 * 16 + j % 128 // 32 * 4 + b % 4
        assert t[at] == s[j, b]


def test_sizes(lib):
    for m in (0, 1, 31, 32, 33, 128, 129, 429, 9304):
        for n in (0, 1, 7, 128, 129):
            x = np.zeros((n, m))
            for fmt in (lib.MXFP4, lib.MXINT8):
                codes, scales = mx_util.pack(x, fmt)
                assert lib.mx_code_bytes(m, n, fmt) == codes.size
                assert lib.mx_scale_bytes(m, n) == scales.size


def test_refusals(lib):
    """Every bad argument is refused before anything is launched (there is no device here to launch on)."""
    p = 4096  # a pointer that is never read

    def refused(f, *a, word=""):
        with pytest.raises(lib.QaggError) as e:
            f(*a)
        assert "error -1" in str(e.value) and word in str(e.value), str(e.value)

    refused(lib.mx_code_bytes, 8, 8, 5)
    refused(lib.mx_code_bytes, -1, 8, lib.MXFP4)
    refused(lib.mx_scale_bytes, 8, -1)
    q = lib.mx_quantize
    refused(q, p, 7, 64, p, p, 64, 8, lib.MXFP4, word="type")
    refused(q, p, lib.F32, 64, p, p, 64, 8, 6, word="format")
    refused(q, p, lib.F32, 63, p, p, 64, 8, lib.MXFP4, word="ld")
    refused(q, p, lib.F32, 64, p, p, -1, 8, lib.MXFP4, word="negative")
    refused(q, p, lib.F32, 1 << 30, p, p, 1 << 30, 8, lib.MXFP4, word="large")
    refused(q, p, lib.F32, 64, p, p, 64, 65535 * 128 + 1, lib.MXFP4, word="large")
    refused(q, p, lib.F32, 65535 * 128 + 1, p, p, 65535 * 128 + 1, 8, lib.MXFP4, True, word="large")
    refused(q, 0, lib.F32, 64, p, p, 64, 8, lib.MXFP4, word="null")
    refused(q, p, lib.F32, 64, 0, p, 64, 8, lib.MXFP4, word="null")
    refused(q, p, lib.F32, 64, p, 0, 64, 8, lib.MXFP4, word="null")
    refused(q, p + 2, lib.F32, 64, p, p, 64, 8, lib.MXFP4, word="aligned")
    refused(q, p + 1, lib.BF16, 64, p, p, 64, 8, lib.MXFP4, word="aligned")
    refused(q, p, lib.F32, 64, p + 8, p, 64, 8, lib.MXFP4, word="aligned")
    refused(q, p, lib.F32, 64, p, p + 4, 64, 8, lib.MXFP4, word="aligned")
    u = lib.mx_unquantize
    refused(u, p, p, p, 3, 64, 64, 8, lib.MXFP4, word="type")
    refused(u, p, p, p, lib.F32, 10, 64, 8, lib.MXFP4, word="ld")
    refused(u, 0, p, p, lib.F32, 64, 64, 8, lib.MXFP4, word="null")
    refused(u, p, p, p + 2, lib.F32, 64, 64, 8, lib.MXFP4, word="aligned")
    t = lib.mx_times
    refused(t, p, p, p, p, 0, p, 9, 64, 64, 8, 64, word="type")
    refused(t, p, p, p, p, 0, p, lib.F32, 63, 64, 8, 64, word="ld")
    refused(t, p, p, p, p, 0, p, lib.F32, 64, 64, 8, -1, word="negative")
    refused(t, 0, p, p, p, 0, p, lib.F32, 64, 64, 8, 64, word="null")
    refused(t, p, p, p, p, 0, 0, lib.F32, 64, 64, 8, 64, word="null")
    refused(t, p, p, p, p, p + 2, p, lib.F32, 64, 64, 8, 64, word="aligned")
    refused(t, p, p, p + 1, p, 0, p, lib.F32, 64, 64, 8, 64, word="aligned")
    w = lib.mx_weight_grad
    refused(w, p, 5, 64, p, p, lib.MXINT8, p, 64, 32, 8, word="type")
    refused(w, p, lib.BF16, 64, p, p, 1, p, 64, 32, 8, word="format")
    refused(w, p, lib.BF16, 63, p, p, lib.MXINT8, p, 64, 32, 8, word="ld")
    refused(w, 0, lib.BF16, 64, p, p, lib.MXINT8, p, 64, 32, 8, word="null")
    refused(w, p, lib.BF16, 64, p, p, lib.MXINT8, 0, 64, 32, 8, word="null")
    refused(w, p, lib.BF16, 64, p, p, lib.MXINT8, p + 2, 64, 32, 8, word="aligned")
    refused(w, p, lib.BF16, 65535 * 64 + 1, p, p, lib.MXINT8, p, 65535 * 64 + 1, 32, 8, word="large")
    g = lib.mx_input_grad
    refused(g, p, lib.BF16, 64, p, p, lib.MXFP4, p, 4, 32, 64, 32, 8, word="type")
    refused(g, p, lib.BF16, 64, p, p, lib.MXFP4, p, lib.BF16, 31, 64, 32, 8, word="ld")
    refused(g, p, lib.BF16, 64, p, p + 3, lib.MXFP4, p, lib.BF16, 32, 64, 32, 8, word="aligned")
    f = lib.mx_act_forward
    refused(f, p, lib.BF16, 64, 5, p, 64, p, p, 64, 8, word="function")
    refused(f, p, lib.BF16, 64, -1, p, 64, p, p, 64, 8, word="function")
    refused(f, p, lib.BF16, 63, 0, p, 64, p, p, 64, 8, word="ld")
    refused(f, p, lib.BF16, 64, 0, p, 64, 0, p, 64, 8, word="null")
    refused(f, p, lib.BF16, 64, 0, p + 1, 64, p, p, 64, 8, word="aligned")
    b = lib.mx_act_backward
    refused(b, p, lib.BF16, 64, p, p, 0, 0, 64, 64, 8, word="null")
    refused(b, p, lib.BF16, 64, p, p, 9, p, 64, 64, 8, word="function")


def test_empty_matrices_need_nothing(lib):
    lib.mx_quantize(0, lib.F32, 0, 0, 0, 0, 5, lib.MXFP4)
    lib.mx_quantize(0, lib.F32, 5, 0, 0, 5, 0, lib.MXINT8, True)
    lib.mx_unquantize(0, 0, 0, lib.BF16, 5, 5, 0, lib.MXFP4)
    lib.mx_times(0, 0, 0, 0, 0, 0, lib.F32, 64, 64, 0, 8)
    lib.mx_weight_grad(0, lib.BF16, 64, 0, 0, lib.MXINT8, 0, 64, 0, 8)
    lib.mx_weight_grad(0, lib.BF16, 64, 0, 0, lib.MXINT8, 0, 64, 32, 0, True)  # adding nothing
    lib.mx_input_grad(0, lib.BF16, 64, 0, 0, lib.MXFP4, 0, lib.BF16, 32, 64, 32, 0)
    lib.mx_act_forward(0, lib.F32, 0, 0, 0, 0, 0, 0, 0, 3)
    lib.mx_act_backward(0, lib.F32, 9, 0, 0, 0, 0, 9, 9, 0)


def test_no_cpu_fallback(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    for call in (lambda: lib.mx_quantize(4096, lib.F32, 64, 4096, 4096, 64, 8, lib.MXFP4),
                 lambda: lib.mx_times(4096, 4096, 4096, 4096, 0, 4096, lib.F32, 64, 64, 8, 64),
                 lambda: lib.mx_weight_grad(4096, lib.BF16, 64, 4096, 4096, lib.MXINT8, 4096, 64, 32, 8)):
        with pytest.raises(lib.QaggError) as e:
            call()
        assert "qagg error -2" in str(e.value)


def test_roles_of_the_gradient_products(tmp_path):
    """Barrier counts, registers and tensor memory of the four ways to divide a CTA, compiled for the host."""
    import os
    import subprocess
    exe = str(tmp_path / "mx_groups_check")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "mx_groups_check.cpp")
    res = subprocess.run(["g++", "-std=c++17", "-O0", src, "-o", exe], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "groups ok" in run.stdout, (run.returncode, run.stdout)


def test_wait_selftest_refuses_long_limits(lib):
    for limit in (0, -1, 10 ** 9 + 1):
        with pytest.raises(lib.QaggError) as e:
            lib.mx_wait_selftest(limit)
        assert "error -1" in str(e.value)


def test_in_place_layers_need_one_ld(lib):
    """y over x and dx over dy with another distance between columns would overwrite columns that are still to be read."""
    p = 4096
    for call in (lambda: lib.mx_act_forward(p, lib.F32, 64, lib.ACT_RELU, p, 72, p, p, 64, 8), lambda: lib.mx_act_backward(p, lib.F32, 72, p, p, lib.ACT_RELU, p, 64, 64, 8)):
        with pytest.raises(lib.QaggError) as e:
            call()
        assert "error -1" in str(e.value) and "in place" in str(e.value)


def test_sizes_beyond_the_limits_are_refused(lib):
    """A matrix that no call takes has no size: the products would not fit 64 bits."""
    for m, n in ((1 << 62, 8), ((1 << 63) - 1, 1), (1 << 40, 1 << 40), (1 << 30, 1), (1, 65535 * 128 + 1), (1, 1 << 62)):
        for call in (lambda: lib.mx_code_bytes(m, n, lib.MXINT8), lambda: lib.mx_scale_bytes(m, n)):
            with pytest.raises(lib.QaggError) as e:
                call()
            assert "error -1" in str(e.value)
    assert lib.mx_code_bytes((1 << 30) - 1, 65535 * 128, lib.MXINT8) == (1 << 30) * 65535 * 128
