"""Rows operators (include/speech_hip.h, speech_rows_*) on the device against their statement in 64 bits (rows_ref.py).

Tolerances count roundings: u = half a step of the type relative to the value (f32 2^-24, f16 2^-11, bf16 2^-8, e4m3 2^-4), F = 2^-24 for each
operation in 32-bit floats.  A sum of n terms of which a thread adds `seq` one after another and the rest as a tree or in
few partial sums is off by at most (seq + 24) F times the sum of the magnitudes: 24 covers the tree over at most 1024 threads (10),
the roundings of each term (at most 4) and of the partial sums' own additions (at most 10)."""
import ctypes as C

import numpy as np
import pytest

import rows_ref as R

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f64": 2.0 ** -53}
# the smallest normal numbers (5 exponent bits: 2^-14, 8: 2^-126, 11: 2^-1022): below them steps no longer shrink, half a step is TINY U
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -14, "bf16": 2.0 ** -126, "f64": 2.0 ** -1022}


def _t():
    import torch
    return torch


def _type(name):
    return {"f32": _t().float32, "f16": _t().float16, "bf16": _t().bfloat16, "f64": _t().float64}[name]


class Canvas:
    """a rows x cols matrix inside a larger one filled with a sentinel, at an odd place and with a row stride of its own"""

    def __init__(self, rows, cols, dtype, pad=0, lead=0, fill=3.0, data=None):
        torch = _t()
        self.rows, self.cols, self.ld, self.lead = rows, cols, cols + pad, lead
        self.flat = torch.full((lead + rows * self.ld + 64,), fill, dtype=dtype, device="cuda")
        self.fill = fill
        self.m = self.flat[lead:lead + rows * self.ld].view(rows, self.ld)[:, :cols]
        if data is not None:
            self.m.copy_(data)

    def untouched(self):
        """every element outside the matrix still holds the sentinel"""
        f = self.flat.clone()
        f[self.lead:self.lead + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = self.fill
        return bool((f == self.fill).all())


def _normal(rows, cols, seed, scale=1.0):
    x = np.random.default_rng(seed).standard_normal((rows, cols)) * scale
    if rows > 3:
        x[rows // 2] = 0.0                                    # a silent frame
    return x


def _np(t):
    return t.detach().double().cpu().numpy()


def _near(got, want, bound, what):
    """|got - want| <= bound everywhere"""
    off = np.abs(got - want) - bound
    assert np.isfinite(got).all() and (off <= 0).all(), "%s: worst %.3g over at %s" % (what, off.max(), np.unravel_index(np.argmax(off), off.shape))


SIZES = [(1, 1), (1, 13), (5, 23), (98, 80), (3, 128), (7, 129), (33, 257), (2, 511), (9, 512), (4, 1000), (5, 1024), (3, 2049), (2, 4097), (3, 8200), (2, 16385), (2, 33000), (1, 40001),
         (1000, 150), (400, 380), (300, 1000), (290, 1219), (270, 1536), (270, 2047), (265, 2305), (260, 4100), (260, 6001), (3, 12000), (2, 20000)]


# ---- dropout ----

@pytest.mark.parametrize("dt", ["f32", "f64", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (98, 80), (41, 257), (2, 5000), (1000, 13)])
def test_dropout(rows, cols, dt):
    torch = _t()
    from speech_amd import api
    x = Canvas(rows, cols, _type(dt), pad=3, lead=1, data=torch.from_numpy(_normal(rows, cols, 1)))
    x.m[0, 0] = float("nan")
    for p, keyed in ((0.3, True), (0.5, False), (0.0, False), (0.999, True)):
        y = Canvas(rows, cols, _type(dt), pad=5, lead=3)
        keys = torch.arange(rows, device="cuda") * 7919 + (5 << 32) if keyed else None
        api.dropout(x.m, y.m, p, 99, keys=keys)
        torch.cuda.synchronize()
        mask = R.kept(p, 99, keys.cpu().numpy() if keyed else np.arange(rows), cols)
        got, want = _np(y.m), R.dropped(_np(x.m), p, mask)
        assert np.array_equal(np.isnan(got), np.isnan(want))             # a dropped NaN is 0
        assert np.array_equal(got == 0, want == 0)
        ok = ~np.isnan(want)
        op = 2.0 ** -53 if dt == "f64" else F                             # the factor's and the product's rounding
        _near(got[ok], want[ok], (U[dt] + 2 * op) * np.abs(want[ok]) + TINY[dt] * U[dt], "dropout")
        assert y.untouched()
    # in place, and the same call on a gradient uses the same mask
    z = x.m.clone()
    api.dropout(z, z, 0.3, 99)
    g = torch.ones_like(z)
    api.dropout(g, g, 0.3, 99)
    torch.cuda.synchronize()
    assert torch.equal((g != 0).cpu(), torch.from_numpy(R.kept(0.3, 99, np.arange(rows), cols)))
    assert torch.equal(torch.isnan(z) | (z != 0), (g != 0) & ((x.m != 0) | torch.isnan(x.m)))


def test_dropout_long_offsets_and_strided_rows():
    """an element offset past 2^32 and a row stride past 2^31: rows are addressed in 64 bits"""
    torch = _t()
    from speech_amd import api
    ld = (1 << 31) + 40
    flat = torch.zeros(2 * ld + 1000, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((3, 900), (ld, 1))
    x.copy_(torch.arange(2700, device="cuda").view(3, 900) % 250 + 1)
    y = torch.empty(3, 900, dtype=torch.bfloat16, device="cuda")
    api.dropout(x, y, 0.5, 3)
    torch.cuda.synchronize()
    mask = R.kept(0.5, 3, np.arange(3), 900)
    assert np.array_equal(_np(y), np.where(mask, 2.0 * _np(x), 0.0))


def test_dropout_step_counter_in_a_replayed_graph():
    """*step is read when the kernel runs: every replay of a graph that also advances it draws the mask of seed + step"""
    torch = _t()
    from speech_amd import api
    x = torch.ones(50, 333, device="cuda")
    y = torch.zeros_like(x)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    api.dropout(x, y, 0.4, 11, step=step)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.dropout(x, y, 0.4, 11, step=step, stream=torch.cuda.current_stream().cuda_stream)
        step.add_(1)
    step.fill_(5)
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(_np(y) != 0, R.kept(0.4, 11 + 5 + k, np.arange(50), 333))
        z = torch.zeros_like(x)                                           # eager work between the replays
        api.dropout(x, z, 0.4, 11 + 5 + k)
        torch.cuda.synchronize()
        assert torch.equal(y, z)
    assert int(step) == 9


@pytest.mark.parametrize("n,offset", [(1, 0), (3, 0), (3, 2), (200, 150)])
def test_row_keys_of_a_batch_and_of_its_shards(n, offset):
    torch = _t()
    from speech_amd import api
    plan = api.Plan("fbank", B=80)
    lens = [16000, 400, 4321, 30000, 560, 401, 8000] + [700] * 1100       # more utterances than one round of the scan
    b = api.Batch(plan, lens)
    for ids in (None, [3 * i + 1 for i in range(len(lens))]):
        b.set_ids(ids)
        rows, tot = b.subsample_rows(n, offset)
        keys = torch.full((tot + 5,), -1, dtype=torch.int64, device="cuda")
        b.row_keys(keys, n, offset)
        torch.cuda.synchronize()
        want = np.concatenate([((ids[u] if ids else u) << 32) + offset + n * np.arange(rows[u]) for u in range(len(lens))]).astype(np.int64)
        assert np.array_equal(keys.cpu().numpy(), np.concatenate([want, [-1] * 5]))
    # a shard of the corpus, under the corpus' numbers: the same keys, hence the same masks
    part = [3, 0, 5]
    s = api.Batch(plan, [lens[i] for i in part])
    s.set_ids(part)
    b.set_ids(None)
    rows, tot = b.subsample_rows(n, offset)
    ka, kb = torch.empty(tot, dtype=torch.int64, device="cuda"), torch.empty(max(1, s.subsample_rows(n, offset)[1]), dtype=torch.int64, device="cuda")
    b.row_keys(ka, n, offset)
    s.row_keys(kb, n, offset)
    torch.cuda.synchronize()
    at = np.concatenate([[0], np.cumsum(rows)])
    assert np.array_equal(kb.cpu().numpy()[:s.subsample_rows(n, offset)[1]], np.concatenate([ka.cpu().numpy()[at[u]:at[u + 1]] for u in part]))
    with pytest.raises(api.SpeechError):
        b.row_keys(ka, 3, 3)


# ---- RMS norm ----

def _norm_want(x, r, w, eps, mask, p, dt):
    h = R.dropped(x, p, mask) + r
    return h


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_rms_norm(rows, cols, dt):
    torch = _t()
    from speech_amd import api
    ty = _type(dt)
    seq = max(32, -(-cols // 256) + 8)
    x = Canvas(rows, cols, ty, pad=1, lead=1, data=torch.from_numpy(_normal(rows, cols, 2, 3.0)))
    r = Canvas(rows, cols, ty, pad=2, lead=2, data=torch.from_numpy(_normal(rows, cols, 3)))
    w32 = torch.from_numpy(1 + 0.1 * np.random.default_rng(4).standard_normal(cols)).float().cuda()
    keys = torch.arange(rows, device="cuda") + (9 << 32)
    mask = R.kept(0.2, 5, keys.cpu().numpy(), cols)
    for residual, p, weight, eps in ((True, 0.2, w32.to(ty), 1e-6), (False, 0.0, None, 1e-3), (True, 0.0, w32, 1e-6), (False, 0.2, w32, 1e-5)):
        h, y = Canvas(rows, cols, ty, pad=3, lead=3), Canvas(rows, cols, ty, pad=7, lead=1)
        rstd = torch.full((rows + 3,), 3.0, device="cuda")
        q, s = api.held(rows + 1, cols)
        q.view(torch.uint8).fill_(0x55)
        s.fill_(0x33)
        api.rms_norm(x.m, weight, eps, residual=r.m if residual else None, H=h.m, Y=y.m, Q=q[:rows], S=s[:rows], rstd=rstd[:rows], p=p, seed=5, keys=keys)
        torch.cuda.synchronize()
        xd, rr = R.dropped(_np(x.m), p, mask), (_np(r.m) if residual else np.zeros((rows, cols)))
        got_h = _np(h.m)
        _near(got_h, xd + rr, U[dt] * np.abs(xd + rr) + 3 * F * (np.abs(xd) + np.abs(rr)) + TINY[dt] * U[dt], "H")
        want_r = 1.0 / np.sqrt((got_h ** 2).mean(1) + eps)                # from the H it left: what the backward pass will use
        rel = (seq + 24) * F
        _near(_np(rstd[:rows]), want_r, rel * want_r, "rstd")
        want = got_h * want_r[:, None] * (_np(weight) if weight is not None else 1.0)
        _near(_np(y.m), want, (U[dt] + rel + 3 * F) * np.abs(want) + TINY[dt] * U[dt], "Y")
        # 8-bit output: the scale is the rule's for the largest value (either side of a border that is nearer than the error), the
        # values are within half a step of the type, 2^-10 of the scale below its normal range
        e = s[:rows].cpu().numpy()
        lo, hi = R.exponents(want * (1 - rel - 4 * F)), R.exponents(want * (1 + rel + 4 * F))
        assert ((e >= lo) & (e <= hi)).all()
        sc = R.spread(e, cols)
        back = R.e4m3_values()[q[:rows].view(torch.uint8).cpu().numpy()] * sc
        _near(back, want, np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * sc) + (rel + 4 * F) * np.abs(want), "Q")
        assert h.untouched() and y.untouched() and bool((rstd[rows:] == 3).all())
        full_q, full_s = torch.as_strided(q.view(torch.uint8), (rows + 1, q.stride(0)), (q.stride(0), 1)), torch.as_strided(s, (rows + 1, s.stride(0)), (s.stride(0), 1))
        assert bool((full_q[rows:, :cols] == 0x55).all()) and bool((full_s[rows:, :s.shape[1]] == 0x33).all())      # the row behind the last
        assert bool((full_q[:, cols:] == 0).all()) and bool((full_s[:, s.shape[1]:] == 0).all())    # what pads a row, as held left it


@pytest.mark.parametrize("dt,cols", [("f32", 300), ("bf16", 1024), ("f16", 20000), ("bf16", 40000), ("f32", 17000)])
def test_rms_norm_in_place(dt, cols):
    """H over X or the residual, Y over the other one: the same bits as apart from them"""
    torch = _t()
    from speech_amd import api
    ty = _type(dt)
    x, r = (torch.from_numpy(_normal(9, cols, k)).to(ty).cuda() for k in (5, 6))
    h, y = torch.empty_like(x), torch.empty_like(x)
    api.rms_norm(x, residual=r, H=h, Y=y, p=0.1, seed=3)
    for hx in (True, False):
        a, b = x.clone(), r.clone()
        api.rms_norm(a, residual=b, H=a if hx else b, Y=b if hx else a, p=0.1, seed=3)
        torch.cuda.synchronize()
        assert torch.equal(a if hx else b, h) and torch.equal(b if hx else a, y)
    a = x.clone()
    api.rms_norm(a, residual=r, Y=a, p=0.1, seed=3)                       # no H: the row is not read again
    torch.cuda.synchronize()
    assert torch.equal(a, y)
    with pytest.raises(api.SpeechError):
        api.rms_norm(x, H=h, Y=h)


@pytest.mark.parametrize("cols", [40, 100, 300, 1024, 5000, 20000, 33000])
def test_rms_norm_of_what_is_no_number_and_of_silence(cols):
    torch = _t()
    from speech_amd import api
    x = torch.from_numpy(_normal(6, cols, 7)).float().cuda()
    x[1] = 0.0
    x[2, 3] = float("nan")
    x[4, cols - 1] = float("inf")
    y = torch.empty_like(x)
    rstd = torch.empty(6, device="cuda")
    q, s = api.held(6, cols)
    api.rms_norm(x, eps=1e-6, Y=y, Q=q, S=s, rstd=rstd)
    torch.cuda.synchronize()
    yn = _np(y)
    assert np.isfinite(yn[[0, 1, 3, 5]]).all() and (yn[1] == 0).all() and abs(float(rstd[1]) - 1e3) < 1e-3
    assert np.isnan(yn[2]).all()
    assert np.isnan(yn[4, cols - 1]) and (yn[4, :cols - 1] == 0).all()
    qv = q.view(torch.uint8).cpu().numpy()
    assert (qv[1] & 127 == 0).all() and (s[1] == 0).all() and (qv[2] & 127 == 127).all() and (s[2] == 0).all()
    assert qv[4, cols - 1] & 127 == 127 and (qv[4, :cols - 1] & 127 == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", SIZES + [(5000, 40), (3000, 700)])
def test_rms_norm_backward(rows, cols, dt):
    torch = _t()
    from speech_amd import api
    ty = _type(dt)
    seq = max(32, -(-cols // 256) + 8)
    h = Canvas(rows, cols, ty, pad=1, lead=1, data=torch.from_numpy(_normal(rows, cols, 8, 2.0)))
    dy = Canvas(rows, cols, ty, pad=2, lead=2, data=torch.from_numpy(_normal(rows, cols, 9, 0.1)))
    dr = Canvas(rows, cols, ty, pad=3, lead=1, data=torch.from_numpy(_normal(rows, cols, 10, 0.1)))
    w32 = torch.from_numpy(1 + 0.1 * np.random.default_rng(4).standard_normal(cols)).float().cuda()
    H, rstd64 = _np(h.m), 1.0 / np.sqrt((_np(h.m) ** 2).mean(1) + 1e-6)
    rstd = torch.from_numpy(rstd64).float().cuda()
    rs = _np(rstd)[:, None]
    mask = R.kept(0.3, 6, np.arange(rows), cols)
    work = torch.empty(api.rms_norm_work(rows, cols), dtype=torch.uint8, device="cuda")
    for weight, use_r, p in ((w32.to(ty), True, 0.3), (w32, False, 0.0), (None, True, 0.0)):
        dh, dx = Canvas(rows, cols, ty, pad=5, lead=1), Canvas(rows, cols, ty, pad=4, lead=2)
        dw = torch.full((cols + 2,), 3.0, device="cuda")
        api.rms_norm_backward(dy.m, h.m, weight, rstd, dh.m, dR=dr.m if use_r else None, dX=dx.m, dW=dw[:cols], work=work, p=p, seed=6)
        torch.cuda.synchronize()
        w, D = (_np(weight) if weight is not None else np.ones(cols)), _np(dy.m)
        g = D * w
        add = _np(dr.m) if use_r else np.zeros_like(D)
        mean, absm = (g * H).mean(1, keepdims=True), np.abs(g * H).mean(1, keepdims=True)
        want = rs * g - H * rs ** 3 * mean + add
        err = 5 * F * (np.abs(rs * g) + np.abs(add)) + np.abs(H) * rs ** 3 * absm * (seq + 32) * F
        _near(_np(dh.m), want, err + U[dt] * (np.abs(want) + err) + TINY[dt] * U[dt], "dH")
        wx = R.dropped(want, p, mask)
        ex = err / (1 - p) + 2 * F * np.abs(wx)
        _near(_np(dx.m), wx, ex + U[dt] * (np.abs(wx) + ex) + TINY[dt] * U[dt], "dX")
        terms = D * H * rs
        # a thread adds at most rows / 64 + 1 rows (the widest rows: 64 groups), the reduction at most 128 partial sums in turn
        _near(_np(dw[:cols]), terms.sum(0), (rows / 64 + 1 + 128 + 24) * F * np.abs(terms).sum(0), "dW")
        assert dh.untouched() and dx.untouched() and bool((dw[cols:] == 3).all())
        # the same bits again, and with outputs in place of inputs
        again = torch.empty(cols, device="cuda")
        a, b = dy.m.clone(), dr.m.clone()
        if use_r:
            api.rms_norm_backward(a, h.m, weight, rstd, a, dR=b, dX=b, dW=again, work=work, p=p, seed=6)
        else:
            api.rms_norm_backward(a, h.m, weight, rstd, b, dX=a, dW=again, work=work, p=p, seed=6)
        torch.cuda.synchronize()
        assert torch.equal(again, dw[:cols]) and torch.equal(a if use_r else b, dh.m) and torch.equal(b if use_r else a, dx.m)


def test_rms_norm_backward_of_no_rows_and_without_outputs():
    torch = _t()
    from speech_amd import api
    z = torch.zeros(0, 70, device="cuda")
    dw = torch.ones(70, device="cuda")
    api.rms_norm_backward(z, z, None, torch.zeros(0, device="cuda"), z.clone(), dW=dw)
    torch.cuda.synchronize()
    assert bool((dw == 0).all())
    h = torch.randn(4, 70, device="cuda")
    with pytest.raises(api.SpeechError):
        api.rms_norm_backward(h, h, None, torch.ones(4, device="cuda"))
    with pytest.raises(api.SpeechError, match="work"):
        api.rms_norm_backward(h, h, None, torch.ones(4, device="cuda"), dW=dw)


def test_rms_norm_gradients_against_differences():
    """the whole of forward + backward against central differences of the 64-bit statement: residual, dropped input and weight"""
    torch = _t()
    from speech_amd import api
    rows, cols, p, eps = 3, 37, 0.25, 1e-2
    rng = np.random.default_rng(12)
    x, r, w, dy = rng.standard_normal((rows, cols)), rng.standard_normal((rows, cols)), 1 + 0.1 * rng.standard_normal(cols), rng.standard_normal((rows, cols))
    x, r, w, dy = (v.astype(np.float32).astype(np.float64) for v in (x, r, w, dy))
    mask = R.kept(p, 77, np.arange(rows), cols)

    def loss(x, r, w):
        h = R.dropped(x, p, mask) + r
        return float((dy * h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * w).sum() + 0.5 * (h * r0).sum())

    r0 = rng.standard_normal((rows, cols)).astype(np.float32).astype(np.float64)     # the stream's own use of h, with gradient r0 / 2

    def differences(k):
        args = [x, r, w]
        out = np.zeros_like(args[k])
        for i in np.ndindex(out.shape):
            hi, lo = args[k].copy(), args[k].copy()
            hi[i] += 1e-5
            lo[i] -= 1e-5
            out[i] = (loss(*(args[:k] + [hi] + args[k + 1:])) - loss(*(args[:k] + [lo] + args[k + 1:]))) / 2e-5
        return out

    c = lambda v: torch.from_numpy(v).float().cuda()  # noqa: E731
    X, RR, W, DY = c(x), c(r), c(w), c(dy)
    H, Y, rstd = torch.empty_like(X), torch.empty_like(X), torch.empty(rows, device="cuda")
    api.rms_norm(X, W, eps, residual=RR, H=H, Y=Y, rstd=rstd, p=p, seed=77)
    dH, dX, dW = torch.empty_like(X), torch.empty_like(X), torch.empty(cols, device="cuda")
    work = torch.empty(api.rms_norm_work(rows, cols), dtype=torch.uint8, device="cuda")
    api.rms_norm_backward(DY, H, W, rstd, dH, dR=c(r0 / 2), dX=dX, dW=dW, work=work, p=p, seed=77)
    torch.cuda.synchronize()
    # the difference's own error: third derivatives (order 1) times 1e-10 / 6, and 64-bit rounding of a loss of order 100 over 2e-5, about 1e-9;
    # the kernels' 32-bit roundings of gradients of order 1: 64 F or so
    for got, k in ((dX, 0), (dH, 1), (dW, 2)):
        d = differences(k)
        _near(_np(got), d, 64 * F * (np.abs(d) + 4) + 1e-8, "gradient %d" % k)


# ---- the 8-bit form ----

@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 15), (5, 128), (4, 200), (130, 257), (17, 4096), (300, 33), (128, 64), (1, 1000), (1000, 1)])
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize(rows, cols, dt, transpose):
    """bit for bit: a power-of-two scale makes the rounding exact"""
    torch = _t()
    from speech_amd import api
    v = _normal(rows, cols, 13) * 2.0 ** np.random.default_rng(14).integers(-6, 6, (rows, 1))
    if rows * cols > 100:
        v[0, 0], v[rows - 1, cols - 1], v[0, min(cols - 1, 5)] = np.nan, np.inf, -np.inf
    x = Canvas(rows, cols, _type(dt), pad=3, lead=1, data=torch.from_numpy(v))
    r, c = (cols, rows) if transpose else (rows, cols)
    q, s = api.held(r + 1, c)
    q.view(torch.uint8).fill_(0x55)
    s.fill_(0x33)
    api.quantize(x.m, q[:r], s[:r], transpose=transpose)
    torch.cuda.synchronize()
    xs = _np(x.m).T if transpose else _np(x.m)
    wq, we = R.quantized(xs)
    gq = q.view(torch.uint8).cpu().numpy()
    assert np.array_equal(s[:r].cpu().numpy(), we)
    assert np.array_equal(np.where(gq[:r] & 127 == 127, 127, gq[:r]), wq)
    assert (gq[r:] == 0x55).all() and bool((s[r:] == 0x33).all())
    assert bool((torch.as_strided(q.view(torch.uint8), (r, q.stride(0)), (q.stride(0), 1))[:, c:] == 0).all())


def test_quantize_extremes():
    """every finite f32 magnitude class: the largest, the smallest scale, subnormals, borders between two scales"""
    torch = _t()
    from speech_amd import api
    tops = np.array([3.4028234e38, 448.0, np.nextafter(np.float32(448), np.float32(500)), 224.0, 1.75, 2.0 ** -118, 2.0 ** -119, 2.0 ** -126, 2.0 ** -140, 1e-45, 0.0], np.float32)
    v = np.zeros((len(tops), 130), np.float32)
    v[:, 0], v[:, 1], v[:, 129] = tops, -tops / 3, tops / 5
    q, s = api.held(*v.shape)
    api.quantize(torch.from_numpy(v).cuda(), q, s)
    torch.cuda.synchronize()
    wq, we = R.quantized(v.astype(np.float64))
    assert np.array_equal(s.cpu().numpy(), we)
    assert np.array_equal(q.view(torch.uint8).cpu().numpy() & 127, wq & 127)


def _unit(va, vb):
    """what the matrix unit may lose: it adds the products of 8 consecutive columns at a resolution of 2^-13 of the largest one's power
    of two, so each of the 7 others is off by less than 2^-13 of the largest: 7 2^-13 times the sum over groups of their largest
    magnitude (below, group by group; the largest is at most the product of the factors' largest)"""
    torch = _t()
    g = -(-va.shape[1] // 8)
    pa, pb = (torch.nn.functional.pad(torch.from_numpy(np.abs(v)).cuda(), (0, g * 8 - v.shape[1])) for v in (va, vb))
    out = torch.zeros(len(va), len(vb), dtype=torch.float64, device="cuda")
    for i in range(g):
        top = torch.zeros_like(out)
        for j in range(8 * i, 8 * i + 8):
            torch.maximum(top, pa[:, j, None] * pb[None, :, j], out=top)
        out += top
    return 7 * 2.0 ** -13 * out.cpu().numpy()


PRODUCTS = [(1, 1, 1), (1, 16, 128), (1, 512, 2048), (2, 100, 130), (5, 33, 400), (16, 64, 1000), (17, 17, 17), (32, 257, 720), (98, 80, 257), (63, 130, 3000), (64, 512, 512),
            (130, 200, 385), (255, 256, 256), (257, 300, 129), (513, 129, 640), (998, 512, 720), (1, 4096, 33), (700, 1, 500), (3, 5, 0), (300, 1000, 1),
            (1100, 1030, 900), (2048, 2560, 512), (4200, 2100, 300), (2817, 3333, 1152), (33000, 300, 128), (520, 1030, 2064), (300, 1024, 1936), (17, 5000, 1100), (2050, 1000, 1500),
            (4096, 4096, 512), (4300, 3900, 500), (4100, 4000, 1100), (9000, 4200, 640),
            (2000, 1990, 100), (1300, 1100, 1), (1000, 1010, 300), (900, 1024, 384), (4096, 3900, 1040), (3900, 4000, 768), (7900, 4000, 500), (9300, 4200, 640),
            (98, 2048, 2000), (300, 2048, 500), (500, 600, 1700),
            (1100, 1030, 4500), (2048, 1024, 4224), (1990, 1000, 4097), (1025, 1029, 8191)]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rows,cols,k", PRODUCTS)
def test_product(rows, cols, k, dt):
    _product(rows, cols, k, dt)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rows,cols,k", [(17, 1, 8192), (40, 257, 20000), (130, 140, 9001), (257, 512, 8192), (100, 1999, 8200), (520, 700, 17000), (2000, 1990, 16400)])
def test_product_in_parts(rows, cols, k, dt):
    torch = _t()
    from speech_amd import api
    need = api.product_work(rows, cols, k)
    assert need > 0
    work = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    qa, sa, qb, sb, z = _product(rows, cols, k, dt, work[:need])
    assert bool((work[need:] == 0xA5).all()) and not bool((work[:need] == 0xA5).all())
    whole, short, own, other = (torch.empty_like(z) for _ in range(4))
    before = work.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    api.product(qa, sa, qb, sb, whole, work=work[:0])
    api.product(qa, sa, qb, sb, short, work=work[:need - 16])                  # too little: computed whole, nothing left in it
    api.product(qa, sa, qb, sb, own)                                           # room of its own on torch's current stream, none on another
    api.product(qa, sa, qb, sb, other, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(whole, short) and torch.equal(work, before)
    assert torch.equal(own, z) and torch.equal(other, whole)


def _product(rows, cols, k, dt, work=None):
    torch = _t()
    from speech_amd import api
    rng = np.random.default_rng(15 + k)
    scale = 2.0 ** rng.integers(-4, 4, (rows, 1)) if dt != "f16" else 1.0
    a, b = rng.standard_normal((rows, k)) * scale, rng.standard_normal((cols, k)) / max(1, k) ** 0.5
    if rows > 2:
        a[1] = 0.0
    bias = rng.standard_normal(cols).astype(np.float32)

    def put(v):
        qv, ev = R.quantized(v) if v.size else (np.zeros(v.shape, np.uint8), np.zeros((len(v), 0), np.uint8))
        q, s = api.held(*v.shape)
        if v.size:
            torch.as_strided(q.view(torch.uint8), (len(v), q.stride(0)), (q.stride(0), 1)).fill_(0x7F)      # NaN where rows are padded
            torch.as_strided(s, (len(v), s.stride(0)), (s.stride(0), 1)).fill_(0xFF)
        q.view(torch.uint8).copy_(torch.from_numpy(qv))
        s.copy_(torch.from_numpy(ev))
        return q, s, R.stands_for(qv, ev)

    (qa, sa, va), (qb, sb, vb) = put(a), put(b)
    y = Canvas(rows, cols, _type(dt), pad=3, lead=1)
    z = torch.empty(rows, cols, dtype=_type(dt), device="cuda")
    api.product(qa, sa, qb, sb, y.m, bias=torch.from_numpy(bias).cuda(), work=work)
    api.product(qa, sa, qb, sb, z, work=work)
    torch.cuda.synchronize()
    unit = _unit(va, vb)
    for got, add in ((_np(y.m), bias.astype(np.float64)), (_np(z), 0.0)):
        want = va @ vb.T + add
        # 128 products inside the matrix unit, then one addition for each k-step, for each partial sum (of waves at most 16, of parts one for
        # eight k-steps: never more than 64 and the k-steps that they save), and the bias
        err = (128 + -(-k // 128) + 64 + 1) * F * (np.abs(va) @ np.abs(vb).T + np.abs(add)) + unit
        _near(got, want, err + U[dt] * (np.abs(want) + err) + TINY[dt] * U[dt], "product")
    assert y.untouched()
    return qa, sa, qb, sb, z


def test_product_places_every_element():
    """one at a time: A and B with a single one in each row and column give a permutation, exactly"""
    torch = _t()
    from speech_amd import api
    n = 384
    rng = np.random.default_rng(16)
    pa, pb = rng.permutation(n), rng.permutation(n)
    a, b = np.zeros((n, n)), np.zeros((n, n))
    va = 1.0 + (np.arange(n) % 8) / 8.0
    a[np.arange(n), pa] = va
    b[np.arange(n), pb] = 2.0 ** (np.arange(n) % 5)
    qa, sa = api.held(n, n)
    qb, sb = api.held(n, n)
    api.quantize(torch.from_numpy(a).float().cuda(), qa, sa)
    api.quantize(torch.from_numpy(b).float().cuda(), qb, sb)
    for rows in (n, 7, 100):
        y = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
        api.product(qa[:rows], sa[:rows], qb, sb, y)
        torch.cuda.synchronize()
        assert np.array_equal(_np(y), a[:rows] @ b.T)


def test_product_keeps_nan_in_its_row_and_column():
    torch = _t()
    from speech_amd import api
    for rows, cols, k in ((20, 40, 300), (600, 700, 300)):
        a, b = np.ones((rows, k)), np.ones((cols, k))
        a[3, 7], b[5, 299] = np.nan, np.inf
        qa, sa = api.held(rows, k)
        qb, sb = api.held(cols, k)
        api.quantize(torch.from_numpy(a).float().cuda(), qa, sa)
        api.quantize(torch.from_numpy(b).float().cuda(), qb, sb)
        y = torch.empty(rows, cols, device="cuda", dtype=torch.float16)
        api.product(qa, sa, qb, sb, y)
        torch.cuda.synchronize()
        want = np.full((rows, cols), float(k))
        want[3], want[:, 5] = np.nan, np.nan
        assert np.array_equal(_np(y), want, equal_nan=True)


@pytest.mark.parametrize("rows,cols,k", [(20, 40, 300), (600, 700, 300), (1000, 1030, 640), (4096, 4096, 640), (40, 200, 8200)])
def test_product_of_extreme_scales(rows, cols, k):
    """255 is NaN for its rows and columns only; the largest and the smallest scales meet in a finite product"""
    torch = _t()
    from speech_amd import api
    qa, sa = api.held(rows, k)
    qb, sb = api.held(cols, k)
    qa.copy_(torch.ones(rows, k, device="cuda"))
    qb.copy_(torch.ones(cols, k, device="cuda"))
    sa.fill_(127)
    sb.fill_(127)
    sa[5, 1], sb[7, 0] = 255, 255
    sa[3], sb[9] = 254, 0                                                      # 2^127 and 2^-127
    y = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
    need = api.product_work(rows, cols, k)
    api.product(qa, sa, qb, sb, y, work=torch.empty(need, dtype=torch.uint8, device="cuda") if need else None)
    torch.cuda.synchronize()
    bad = torch.isnan(y)
    assert bool(bad[5].all()) and bool(bad[:, 7].all()) and int(bad.sum()) == rows + cols - 1
    one = torch.tensor(float(k)).bfloat16().item()
    assert y[3, 9].item() == one and y[0, 0].item() == one and y[rows - 1, cols - 1].item() == one
    assert torch.isinf(y[3, 0]).item() and y[0, 9].item() == torch.tensor(k * 2.0 ** -127).bfloat16().item()


def test_long_offsets():
    """matrices of more than 2^31 elements: the last rows and columns, bit for bit what the same calls on them alone give"""
    torch = _t()
    from speech_amd import api
    rows, cols, n, last = 2200000, 1024, 256, 300
    X = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    w = torch.linspace(0.5, 1.5, cols, device="cuda")
    q, s = api.held(rows, cols)
    rstd = torch.empty(rows, device="cuda")
    api.rms_norm(X, w, Q=q, S=s, rstd=rstd)
    tail = X[-last:].clone()
    qt, st = api.held(last, cols)
    rt = torch.empty(last, device="cuda")
    api.rms_norm(tail, w, Q=qt, S=st, rstd=rt)
    torch.cuda.synchronize()
    eq = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))  # noqa: E731
    assert eq(q[-last:], qt) and eq(s[-last:], st) and torch.equal(rstd[-last:], rt)
    api.quantize(X, q, s)
    api.quantize(tail, qt, st)
    torch.cuda.synchronize()
    assert eq(q[-last:], qt) and eq(s[-last:], st)

    qb, sb = api.held(n, cols)
    api.quantize(X[:n], qb, sb)
    y = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
    api.product(q, s, qb, sb, y)
    torch.cuda.synchronize()
    va, vb = (R.stands_for(a.view(torch.uint8).cpu().numpy(), b.cpu().numpy()) for a, b in ((qt, st), (qb, sb)))
    want = va @ vb.T
    err = (128 + 8 + 64) * F * (np.abs(va) @ np.abs(vb).T) + _unit(va, vb)
    _near(_np(y[-last:]), want, err + U["bf16"] * (np.abs(want) + err), "last rows")
    del y, q, s

    work = torch.empty(api.rms_norm_work(rows, cols), dtype=torch.uint8, device="cuda")
    dH, dt = torch.empty_like(X), torch.empty_like(tail)
    api.rms_norm_backward(X, X, w, rstd, dH, dW=torch.empty(cols, device="cuda"), work=work)
    api.rms_norm_backward(tail, tail, w, rt, dt)
    torch.cuda.synchronize()
    assert torch.equal(dH[-last:], dt)
    del dH

    q, s = api.held(cols, rows)
    api.quantize(X, q, s, transpose=True)
    part = X[:, -64:].contiguous()
    qt, st = api.held(64, rows)
    api.quantize(part, qt, st, transpose=True)
    torch.cuda.synchronize()
    assert eq(q[-64:], qt) and eq(s[-64:], st)


def test_product_in_parts_in_replayed_graphs():
    """two graphs with a work array each, replayed in turn with eager calls between"""
    torch = _t()
    from speech_amd import api
    rows, cols, k = 96, 200, 8200
    gen = torch.Generator("cuda").manual_seed(4)
    X = [torch.empty(r, k, device="cuda").normal_(generator=gen) for r in (rows, cols)]
    (qa, sa), (qb, sb) = api.held(rows, k), api.held(cols, k)
    work = [torch.empty(api.product_work(rows, cols, k), dtype=torch.uint8, device="cuda") for _ in range(3)]
    out = [torch.zeros(rows, cols, device="cuda", dtype=torch.float16) for _ in range(3)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            st = torch.cuda.current_stream().cuda_stream
            if i == 0:
                api.quantize(X[0], qa, sa, stream=st)
                api.quantize(X[1], qb, sb, stream=st)
            api.product(qa, sa, qb, sb, out[i], work=None if i else work[i], stream=st)   # the second takes its room from the graph's pool
    for _ in range(4):
        X[0].normal_(generator=gen)
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        api.product(qa, sa, qb, sb, out[2], work=work[2])
        torch.cuda.synchronize()
        assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[2]) and bool(out[2].any())
        for o in out:
            o.zero_()


def test_product_gradients_against_the_formula():
    """dX = q(dY) q(W^T)^T and dW = q(dY^T) q(X^T)^T: within the 8-bit rounding (2^-4 of each factor; below a block's
    normal range 2^-10 of its scale, that is 2^-18 of the block's largest value) of dY W and dY^T X, and the result's own"""
    torch = _t()
    from speech_amd import api
    M, N, K = 200, 96, 160
    rng = np.random.default_rng(17)
    x, w, dy = (rng.standard_normal(s) for s in ((M, K), (N, K), (M, N)))
    c = lambda v: torch.from_numpy(v).float().cuda()  # noqa: E731

    def h(v, r, k, t):
        q, s = api.held(r, k)
        api.quantize(c(v), q, s, transpose=t)
        return q, s

    dX, dW = torch.empty(M, K, device="cuda", dtype=torch.bfloat16), torch.empty(N, K, device="cuda", dtype=torch.bfloat16)
    api.product(*h(dy, M, N, False), *h(w, K, N, True), dX)
    api.product(*h(dy, N, M, True), *h(x, K, M, True), dW)
    torch.cuda.synchronize()
    for got, l, r in ((dX, dy, w), (dW, dy.T, x)):
        want, mag = l @ r, np.abs(l) @ np.abs(r)
        low = 2.0 ** -17 * l.shape[1] * np.abs(l).max() * np.abs(r).max()
        _near(_np(got), want, (2 * 2.0 ** -4 + 2.0 ** -8) * mag * 1.01 + low + 2.0 ** -8 * np.abs(want) + _unit(l, r.T) * 1.2, "gradient")
        assert np.abs(_np(got) - want).mean() < 0.05 * np.abs(want).mean()


# ---- together, as a front end uses them ----

def _front_end():
    torch = _t()
    import signals
    from speech_amd import api
    plan = api.Plan("fbank", B=80)
    lens = [16000, 4000, 30000, 401, 12345]
    b = api.Batch(plan, lens)
    X = torch.from_numpy(np.concatenate([signals.utterance(n, 700 + i) for i, n in enumerate(lens)])).cuda()
    Y = torch.zeros(b.total_out, device="cuda")
    rows = b.subsample_rows(3, 0)[1]
    D = 80 * 3
    Z = torch.zeros(rows * D, device="cuda")
    keys = torch.zeros(rows, dtype=torch.int64, device="cuda")
    W = torch.from_numpy(np.random.default_rng(20).standard_normal((192, D)) / D ** 0.5).float().cuda()
    qw, sw = api.held(192, D)
    api.quantize(W, qw, sw)
    b.row_keys(keys, 3, 0)
    q, s = api.held(rows, D)
    out = torch.zeros(rows, 192, dtype=torch.bfloat16, device="cuda")
    bias = torch.linspace(-1, 1, 192, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    b.run(X, Y)
    b.cmvn(Y, norm_vars=True)                                  # a first call of everything outside a capture
    b.splice_subsample(Y, Z, 1, 1, 3, 0)
    torch.cuda.synchronize()

    def go(stream):
        b.run(X, Y, stream=stream)
        b.cmvn(Y, norm_vars=True, stream=stream)
        b.splice_subsample(Y, Z, 1, 1, 3, 0, stream=stream)
        z = Z.view(rows, D)
        api.dropout(z, z, 0.1, 42, step=step, keys=keys, stream=stream)
        api.rms_norm(z, None, 1e-5, Q=q, S=s, stream=stream)
        api.product(q, s, qw, sw, out, bias=bias, stream=stream)

    return dict(plan=plan, b=b, X=X, Y=Y, Z=Z, keys=keys, q=q, s=s, qw=qw, sw=sw, out=out, bias=bias, step=step, go=go, rows=rows, D=D, lens=lens)


def test_front_end_from_audio_to_the_first_layer():
    """audio -> fbank -> cmvn -> splice + subsample -> dropout -> norm in 8 bits -> product, each step against its statement from what the
    step before left"""
    torch = _t()
    f = _front_end()
    f["go"](None)
    torch.cuda.synchronize()
    z = _np(f["Z"]).reshape(f["rows"], f["D"])
    mask = R.kept(0.1, 42, f["keys"].cpu().numpy(), f["D"])
    assert np.array_equal(z == 0, ~mask | (z == 0)) and abs((z == 0).mean() - 0.1) < 0.01
    rstd = 1 / np.sqrt((z ** 2).mean(1, keepdims=True) + 1e-5)
    want = z * rstd
    e = f["s"].cpu().numpy()
    back = R.stands_for(f["q"].view(torch.uint8).cpu().numpy(), e)
    _near(back, want, np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * R.spread(e, f["D"])) + 60 * F * np.abs(want), "norm")
    w = R.stands_for(f["qw"].view(torch.uint8).cpu().numpy(), f["sw"].cpu().numpy())
    y, mag = back @ w.T + _np(f["bias"]), np.abs(back) @ np.abs(w).T + 1
    _near(_np(f["out"]), y, 2.0 ** -8 * np.abs(y) + 260 * F * mag + 1.01 * _unit(back, w), "product")


def test_front_end_in_a_replayed_graph_on_a_side_stream():
    """the same chain captured once and replayed on new audio, a new mask each time, eager work between the replays"""
    torch = _t()
    import signals
    f = _front_end()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            f["go"](torch.cuda.current_stream().cuda_stream)
            f["step"].add_(1)
    f["step"].zero_()
    torch.cuda.synchronize()
    for k in range(3):
        f["X"].copy_(torch.from_numpy(np.concatenate([signals.utterance(n, 800 + 10 * k + i) for i, n in enumerate(f["lens"])])))
        graph.replay()
        torch.cuda.synchronize()
        got = f["out"].clone()
        assert int(f["step"]) == k + 1
        f["step"].fill_(k)
        f["go"](None)
        torch.cuda.synchronize()
        assert torch.equal(f["out"], got) and bool(torch.isfinite(got).all()) and float(got.float().abs().max()) > 0
        f["step"].fill_(k + 1)
        torch.cuda.synchronize()


def test_training_step_of_a_layer_in_a_replayed_graph():
    """norm forward, product, both products' gradients, norm backward: one graph, replayed, against the same calls made eagerly"""
    torch = _t()
    from speech_amd import api
    rows, D, N = 300, 200, 160
    g = torch.Generator(device="cuda").manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    x, r, w, dy, dr = n(rows, D), n(rows, D), n(N, D), n(rows, N), n(rows, D)
    wt = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).bfloat16()
    e = lambda *s, t=torch.bfloat16: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
    o = dict(H=e(rows, D), Y=e(rows, D), rstd=e(rows, t=torch.float32), out=e(rows, N), dYn=e(rows, D), dW=e(N, D), dH=e(rows, D), dX=e(rows, D),
             dwt=e(D, t=torch.float32), work=e(api.rms_norm_work(rows, D), t=torch.uint8))
    held = [api.held(*s) for s in ((rows, D), (N, D), (D, N), (rows, N), (N, rows), (D, rows))]

    def go(stream):
        (q, s), (qw, sw), (qwt, swt), (qy, sy), (qyt, syt), (qxt, sxt) = held
        api.rms_norm(x, wt, residual=r, H=o["H"], Y=o["Y"], Q=q, S=s, rstd=o["rstd"], p=0.1, seed=9, stream=stream)
        api.quantize(w, qw, sw, stream=stream)
        api.quantize(w, qwt, swt, transpose=True, stream=stream)
        api.product(q, s, qw, sw, o["out"], stream=stream)
        api.quantize(dy, qy, sy, stream=stream)
        api.quantize(dy, qyt, syt, transpose=True, stream=stream)
        api.quantize(o["Y"], qxt, sxt, transpose=True, stream=stream)
        api.product(qy, sy, qwt, swt, o["dYn"], stream=stream)
        api.product(qyt, syt, qxt, sxt, o["dW"], stream=stream)
        api.rms_norm_backward(o["dYn"], o["H"], wt, o["rstd"], o["dH"], dR=dr, dX=o["dX"], dW=o["dwt"], work=o["work"], p=0.1, seed=9, stream=stream)

    go(None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(torch.cuda.current_stream().cuda_stream)
    for k in range(3):
        x.copy_(n(rows, D))
        dy.copy_(n(rows, N))
        graph.replay()
        torch.cuda.synchronize()
        got = {k: v.clone() for k, v in o.items() if k != "work"}
        for v in o.values():
            v.zero_()
        go(None)
        torch.cuda.synchronize()
        for k, v in got.items():
            assert torch.equal(v, o[k]) and bool(torch.isfinite(v).all()), k
    # the layer's gradient against the products in 64 bits, within the 8-bit roundings
    want = _np(dy).T @ _np(o["Y"])
    assert np.abs(_np(o["dW"]) - want).mean() < 0.05 * np.abs(want).mean()


def test_two_streams_at_once_and_another_current_device_stream():
    """calls on two streams with their own outputs and work arrays do not touch each other"""
    torch = _t()
    from speech_amd import api
    rows, cols = 4000, 512
    x = torch.randn(rows, cols, device="cuda")
    y = [torch.empty_like(x) for _ in range(3)]
    dw = [torch.empty(cols, device="cuda") for _ in range(3)]
    rstd = torch.rsqrt(x.square().mean(1) + 1e-6)
    work = [torch.empty(api.rms_norm_work(rows, cols), dtype=torch.uint8, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for k, st in ((0, a), (1, b)):
            api.rms_norm_backward(x, x, None, rstd, y[k], dW=dw[k], work=work[k], stream=st.cuda_stream)
    torch.cuda.synchronize()
    api.rms_norm_backward(x, x, None, rstd, y[2], dW=dw[2], work=work[2])
    torch.cuda.synchronize()
    for k in (0, 1):
        assert torch.equal(y[k], y[2]) and torch.equal(dw[k], dw[2])


def test_python_refuses_what_would_fault():
    torch = _t()
    from speech_amd import api
    x = torch.zeros(8, 64, device="cuda")
    q, s = api.held(8, 64)
    for call in (lambda: api.dropout(x, x[:4], 0.1, 1), lambda: api.dropout(x, x.bfloat16(), 0.1, 1), lambda: api.dropout(x.t(), x.t(), 0.1, 1),
                 lambda: api.dropout(x, x, 0.1, 1, keys=torch.zeros(7, dtype=torch.int64, device="cuda")),
                 lambda: api.dropout(x, x, 0.1, 1, keys=torch.zeros(8, dtype=torch.int32, device="cuda")),
                 lambda: api.dropout(x, x, 0.1, 1, keys=torch.zeros(8, dtype=torch.int64)),
                 lambda: api.rms_norm(x, torch.ones(63, device="cuda"), Y=x), lambda: api.rms_norm(x, Q=q), lambda: api.rms_norm(x, Q=q[:4], S=s[:4]),
                 lambda: api.rms_norm(x, Y=x, rstd=torch.zeros(4, device="cuda")), lambda: api.rms_norm(x[:1].expand(8, 64), Y=x),
                 lambda: api.quantize(x, torch.zeros(8, 70, dtype=torch.uint8, device="cuda")[:, :64], s),
                 lambda: api.quantize(x[:, :50], torch.zeros(400, dtype=torch.uint8, device="cuda").view(8, 50), s),
                 lambda: api.product(q, s, q, s, torch.zeros(8, 9, device="cuda")), lambda: api.product(q[:, :32], s, q, s, torch.zeros(8, 8, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(api.SpeechError):
        api.rms_norm(x)
    torch.cuda.synchronize()
