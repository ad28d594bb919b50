"""Rows operators (include/speech_hip.h, speech_rows_*) without a device: every refusal of the C ABI comes before a device is touched,
the sizes of the work array, the ctypes structures, and the statement that the GPU tests hold the kernels to."""
import ctypes as C

import numpy as np
import pytest

import rows_ref as R
from speech_amd import _lib, api

P = 1 << 20                                                   # a device address that no call here gets to use


def _drop(p=0.1):
    return C.byref(_lib.SpeechDrop(p, 1, None, None))


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=9), "unknown dtype 9"),
    (dict(drop=None), "null drop"),
    (dict(drop=1.0), "p (probability of dropping) must be in [0 1)"),
    (dict(drop=-0.1), "p (probability of dropping) must be in [0 1)"),
    (dict(drop=float("nan")), "p (probability of dropping) must be in [0 1)"),
    (dict(cols=1 << 31), "at most 2^30"),
    (dict(X=None), "null device pointer X"),
    (dict(Y=None), "null device pointer Y"),
    (dict(ldx=7), "row stride of X is 7, below its 8 columns"),
    (dict(ldy=7), "row stride of Y is 7, below its 8 columns"),
    (dict(X=P + 2), "X is not aligned"),
    (dict(Y=P + 16), "Y overlaps X without being X"),
    (dict(Y=P, ldy=9), "Y overlaps X without being X"),
])
def test_dropout_refuses(kw, msg, capfd):
    a = dict(dtype=0, rows=4, cols=8, X=P, ldx=8, Y=P + 4096, ldy=8, drop=0.1)
    a.update(kw)
    d = None if a["drop"] is None else _drop(a["drop"])
    assert _lib.load().speech_rows_dropout(0, a["dtype"], a["rows"], a["cols"], a["X"], max(a["ldx"], 0), a["Y"], a["ldy"], d, None) == 1
    assert "error in speech_rows_dropout: " in capfd.readouterr().err and msg in _lib.last_error()


def test_empty_calls_succeed_without_a_device():
    lib = _lib.load()
    assert lib.speech_rows_dropout(0, 0, 0, 8, None, 8, None, 8, _drop(), None) == 0
    assert lib.speech_rows_dropout(0, 0, 5, 0, None, 0, None, 0, _drop(), None) == 0
    assert lib.speech_rows_rms_norm(0, C.byref(_lib.SpeechNorm(cols=4, eps=1e-6, Y=P)), None) == 0
    assert lib.speech_rows_rms_norm_backward(0, C.byref(_lib.SpeechNormGrad(cols=4, dH=P)), None) == 0
    assert lib.speech_rows_quantize(0, 0, 0, 8, None, 8, None, 16, None, 4, 0, None) == 0
    assert lib.speech_rows_quantize(0, 0, 8, 0, None, 8, None, 16, None, 4, 1, None) == 0
    assert lib.speech_rows_product(0, 3, 0, 8, 8, None, 16, None, 4, None, 16, None, 4, None, None, 8, None, 0, None) == 0
    assert lib.speech_rows_product(0, 3, 8, 0, 8, None, 16, None, 4, None, 16, None, 4, None, None, 8, None, 0, None) == 0


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=1), "unknown dtype 1"),
    (dict(cols=0), "cols must be positive"),
    (dict(eps=0.0), "eps must be positive"),
    (dict(eps=float("nan")), "eps must be positive"),
    (dict(eps=1e-60), "eps must be positive"),
    (dict(eps=float("inf")), "eps must be positive"),
    (dict(Y=None), "no output"),
    (dict(X=None), "null device pointer X"),
    (dict(ldx=255), "row stride of X is 255, below its 256 columns"),
    (dict(R=P + (1 << 20), ldr=3), "row stride of R"),
    (dict(H=P + (1 << 20), ldh=3), "row stride of H"),
    (dict(ldy=3), "row stride of Y"),
    (dict(Y=P + (1 << 21) + 1), "Y is not aligned"),
    (dict(weight=P + 1), "weight is not aligned"),
    (dict(weight=P + 2, weight_f32=1), "weight is not aligned"),
    (dict(Q=P + (3 << 20), ldq=256, S=None, lds=4), "null device pointer Q"),
    (dict(Q=P + (3 << 20) + 8, ldq=256, S=P + (4 << 20), lds=4), "8-bit rows of Q must start on 16 bytes"),
    (dict(Q=P + (3 << 20), ldq=264, S=P + (4 << 20), lds=4), "8-bit rows of Q must start on 16 bytes"),
    (dict(Q=P + (3 << 20), ldq=240, S=P + (4 << 20), lds=4), "8-bit rows of Q must start on 16 bytes"),
    (dict(Q=P + (3 << 20), ldq=256, S=P + (4 << 20), lds=2), "rows of scales of Q must start on 4 bytes"),
    (dict(Q=P + (3 << 20), ldq=256, S=P + (4 << 20) + 1, lds=4), "rows of scales of Q must start on 4 bytes"),
    (dict(H=P + 64), "H overlaps X or R without being it"),
    (dict(Y=P + 64), "Y overlaps X or R without being it"),
    (dict(H=P + (1 << 21)), "Y overlaps H"),
    (dict(H=P, Y=P), "Y overlaps H"),
    (dict(drop=1.5), "p (probability of dropping)"),
])
def test_norm_refuses(kw, msg, capfd):
    a = dict(dtype=_lib.BF16, rows=4, cols=256, eps=1e-6, X=P, ldx=256, Y=P + (1 << 21), ldy=256, ldh=256, ldr=256)
    a.update(kw)
    drop = a.pop("drop", None)
    if drop is not None:
        a["drop"] = C.pointer(_lib.SpeechDrop(drop, 1, None, None))
    assert _lib.load().speech_rows_rms_norm(0, C.byref(_lib.SpeechNorm(**a)), None) == 1
    assert "error in speech_rows_rms_norm: " in capfd.readouterr().err and msg in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=7), "unknown dtype 7"),
    (dict(cols=0), "cols must be positive"),
    (dict(dH=None), "no output"),
    (dict(dY=None), "null device pointer dY"),
    (dict(H=None), "null device pointer H"),
    (dict(rstd=None), "null device pointer rstd"),
    (dict(lddy=9), "row stride of dY"),
    (dict(ldh=9), "row stride of H"),
    (dict(dR=P + (5 << 20), lddr=9), "row stride of dR"),
    (dict(lddh=9), "row stride of dH"),
    (dict(dX=P + (5 << 20), lddx=9), "row stride of dX"),
    (dict(dW=P + (5 << 20)), "dW needs a work array of 4000 bytes"),
    (dict(dW=P + (5 << 20), work=P + (6 << 20), work_bytes=3999), "dW needs a work array of 4000 bytes"),
    (dict(dW=P + (5 << 20), work=P + (6 << 20) + 4, work_bytes=4000), "dW needs a work array of 4000 bytes"),
    (dict(dH=P + 4), "dH overlaps dY or dR without being it"),
    (dict(dX=P + 4), "dX overlaps dY or dR without being it"),
    (dict(dX=P + (2 << 20)), "dX overlaps dH"),
    (dict(dH=P + (1 << 20)), "dH or dX overlaps H"),
])
def test_norm_backward_refuses(kw, msg, capfd):
    a = dict(dtype=0, rows=10, cols=100, dY=P, lddy=100, H=P + (1 << 20), ldh=100, rstd=P + (7 << 20), dH=P + (2 << 20), lddh=100, lddx=100, lddr=100)
    a.update(kw)
    assert _lib.load().speech_rows_rms_norm_backward(0, C.byref(_lib.SpeechNormGrad(**a)), None) == 1
    assert "error in speech_rows_rms_norm_backward: " in capfd.readouterr().err and msg in _lib.last_error(), _lib.last_error()


def test_work_sizes(capfd):
    assert api.rms_norm_work(10, 100) == 4000
    assert api.rms_norm_work(10 ** 6, 1000) == 1024 * 1000 * 4
    assert api.rms_norm_work(0, 10) == 0
    assert _lib.load().speech_rows_rms_norm_work(1, 1, None) == 1
    with pytest.raises(api.SpeechError):
        api.rms_norm_work(1, 1 << 31)
    capfd.readouterr()


def test_product_work_sizes(capfd):
    assert api.product_work(2048, 1024, 4096) == 0 and api.product_work(1, 512, 1 << 20) == 0 and api.product_work(8192, 8192, 1 << 16) == 0
    assert api.product_work(0, 10, 1 << 20) == 0
    n = api.product_work(512, 720, 31936)
    assert n > 0 and n % (512 * 720 * 4) == 0 and n // (512 * 720 * 4) <= 31
    assert _lib.load().speech_rows_product_work(1, 1, 1, None) == 1
    with pytest.raises(api.SpeechError):
        api.product_work(1, 1, 1 << 31)
    capfd.readouterr()


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=1), "unknown dtype 1"),
    (dict(X=None), "null device pointer X"),
    (dict(ldx=63), "row stride of X is 63"),
    (dict(Q=None), "null device pointer Q"),
    (dict(S=None), "null device pointer Q"),
    (dict(ldq=63), "must start on 16 bytes"),
    (dict(lds=3), "must start on 4 bytes"),
    (dict(transpose=1, rows=200), "must start on 16 bytes, 200 columns apart"),
    (dict(transpose=1, rows=2000, ldq=2000), "must start on 4 bytes, 16 scales apart"),
])
def test_quantize_refuses(kw, msg, capfd):
    a = dict(dtype=0, rows=3, cols=64, X=P, ldx=64, Q=P + (1 << 20), ldq=64, S=P + (2 << 20), lds=4, transpose=0)
    a.update(kw)
    assert _lib.load().speech_rows_quantize(0, a["dtype"], a["rows"], a["cols"], a["X"], a["ldx"], a["Q"], a["ldq"], a["S"], a["lds"], a["transpose"], None) == 1
    assert "error in speech_rows_quantize: " in capfd.readouterr().err and msg in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=1), "the result has 16 bits"),
    (dict(dtype=0), "the result has 16 bits"),
    (dict(A=None), "null device pointer A"),
    (dict(SB=None), "null device pointer B"),
    (dict(lda=24), "8-bit rows of A must start on 16 bytes"),
    (dict(B=P + 8), "8-bit rows of B must start on 16 bytes"),
    (dict(ldsa=1), "rows of scales of A must start on 4 bytes"),
    (dict(Y=None), "null device pointer Y"),
    (dict(ldy=19), "row stride of Y is 19"),
    (dict(bias=P + 2), "bias is not aligned"),
    (dict(k=1 << 31), "at most 2^30"),
    (dict(rows=1 << 30, cols=1 << 30, ldy=1 << 30), "matrix too large"),
    (dict(work=P + 8), "work must start on 16 bytes"),
])
def test_product_refuses(kw, msg, capfd):
    a = dict(dtype=2, rows=10, cols=20, k=30, A=P, lda=32, SA=P + 4096, ldsa=4, B=P + 8192, ldb=32, SB=P + 16384, ldsb=4, bias=None, Y=P + 32768, ldy=20,
             work=None, work_bytes=0)
    a.update(kw)
    args = [a[n] for n in "dtype rows cols k A lda SA ldsa B ldb SB ldsb bias Y ldy work work_bytes".split()]
    assert _lib.load().speech_rows_product(0, *args, None) == 1
    assert "error in speech_rows_product: " in capfd.readouterr().err and msg in _lib.last_error(), _lib.last_error()


def test_row_keys_refuses_a_null_batch(capfd):
    assert _lib.load().speech_batch_row_keys(None, 1, 0, P, None) == 1
    assert "null batch" in capfd.readouterr().err


def test_python_refuses_host_tensors_and_types():
    import torch
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="must be on cuda"):
        api.dropout(x, x, 0.1, 1)
    with pytest.raises(ValueError, match="must have dtype"):
        api.rms_norm(x.double())
    with pytest.raises(ValueError, match="must have dtype"):
        api.quantize(x.int(), x, x)
    q, s = api.held(5, 200, device="cpu")
    assert q.shape == (5, 200) and q.stride(0) == 208 and s.shape == (5, 2) and s.stride(0) == 4
    assert api.held(5, 720, device="cpu")[0].stride(0) == 768


def test_statement_of_the_mask():
    """a fair coin of the stated weight in every row and column, other masks for other seeds and keys, the same one for the same"""
    for p in (0.1, 0.5, 0.9):
        m = R.kept(p, 7, np.arange(4000), 500)
        n = m.size
        assert abs(m.mean() - (1 - p)) < 5 * np.sqrt(p * (1 - p) / n)
        assert np.abs(m.mean(0) - (1 - p)).max() < 6 * np.sqrt(p * (1 - p) / 4000)
        assert np.abs(m.mean(1) - (1 - p)).max() < 6 * np.sqrt(p * (1 - p) / 500)
    a, b = R.kept(0.5, 7, np.arange(200), 300), R.kept(0.5, 8, np.arange(200), 300)
    assert abs((a == b).mean() - 0.5) < 5 * 0.5 / np.sqrt(a.size)
    assert abs((a[1:] == a[:-1]).mean() - 0.5) < 5 * 0.5 / np.sqrt(a.size) and abs((a[:, 1:] == a[:, :-1]).mean() - 0.5) < 5 * 0.5 / np.sqrt(a.size)
    assert np.array_equal(R.kept(0.5, 7, np.arange(50, 200), 300), a[50:])
    assert R.kept(0.0, 1, [3], 100).all()


def test_statement_of_the_8_bit_form():
    """the table and the rounding against torch's e4m3 type, the scale rule at its borders"""
    import torch
    v = R.e4m3_values()
    t = torch.arange(256, dtype=torch.int64).to(torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(v[np.isfinite(v)], t[np.isfinite(t)]) and np.array_equal(np.isnan(v), np.isnan(t))
    x = np.random.default_rng(1).standard_normal(4000) * 2.0 ** np.random.default_rng(2).integers(-12, 7, 4000)
    x = np.concatenate([x, v[np.isfinite(v)], (v[1:126] + v[2:127]) / 2, [448.0, -448.0, 2.0 ** -10, 3 * 2.0 ** -11]]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    assert np.array_equal(R.to_e4m3(x.astype(np.float64)), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    for top, e in ((448.0, 127), (np.nextafter(448.0, 500), 128), (224.0, 126), (1.75, 119), (1.0, 119), (2.0 ** -140, 0), (0.0, 0), (3.4e38, 247)):
        assert R.exponents(np.array([[top, 0.0]]))[0, 0] == e, top
    assert R.exponents(np.array([[np.inf, np.nan, 448.0]]))[0, 0] == 127
