"""The int8 operators on the GPU against their definitions in 64 bits.

Tolerances. A row's scale and elements come from f32 arithmetic whose relative
error r is bounded below for each operator; an element is off the exact
quotient y / scale by half a step of rounding plus r times the quotient (at most
127), so |q - y / scale| <= 0.5 + 127 r. The matrix product is exact up to the
sum; then f32 rounds three times (four with a bias) and the output type once.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DT = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}
F24 = 2.0 ** -24


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


class Rows:
    """rows x cols inside a larger buffer: `shift` elements before it, `pad`
    between rows, and a pattern around the rows that a call has to leave alone."""

    def __init__(self, rows, cols, dtype, pad=0, shift=0, fill=None):
        self.ld = cols + pad
        self.buf = torch.empty(shift + rows * self.ld + 64, dtype=dtype, device="cuda")
        self.buf.view(torch.uint8).fill_(0x5A)
        self.t = self.buf[shift:shift + rows * self.ld].view(rows, self.ld)[:, :cols]
        if fill is not None:
            self.t.copy_(fill)
        self.ptr = self.t.data_ptr() if rows and cols else self.buf.data_ptr()
        self.cols = cols
        self.rows = rows
        self.shift = shift

    def untouched_around(self):
        b = self.buf.clone()
        b[self.shift:self.shift + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = 0
        want = torch.empty_like(self.buf)
        want.view(torch.uint8).fill_(0x5A)
        want[self.shift:self.shift + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = 0
        return torch.equal(b.view(torch.uint8), want.view(torch.uint8))


def _ok(gpu, rc):
    assert rc == 0, gpu.last_error()


def _check_int8(q, scale, y, r, extra=0.0):
    """q, scale against f64 rows y; r relative, extra absolute (in y's units) error."""
    y = y.double()
    s = y.abs().amax(dim=1) / 127
    # a scale below 2^-126 is a multiple of 2^-149, so it is off by up to half of
    # that, 2^-150, whatever its own size: a row of 1e-38 has scale 7.87e-41
    assert torch.all((scale.double() - s).abs() <= s * (r + F24) + extra / 127 + 2.0 ** -150), (scale, s)
    nz = s > 0
    assert torch.all(q[~nz] == 0)
    t = y[nz] / s[nz, None]
    tol = 0.5 + 127 * r + extra / s[nz, None] * 2
    d = (q[nz].double() - t).abs()
    assert torch.all(d <= tol), float((d - tol).max())
    assert q.abs().max() <= 127 if q.numel() else True


# ---------------------------------------------------------------- norm

def _norm(gpu, type, x, resid, out, w, eps, rows, cols, q, scale):
    return gpu.lib().llamini_rms_norm_i8_device(
        type, x.ptr, x.ld, resid.ptr if resid else None, resid.ld if resid else 0, out.ptr if out else None,
        out.ld if out else 0, w.data_ptr(), eps, rows, cols, q.ptr, q.ld, scale.data_ptr(), _stream())


def _norm_r(cols):
    # the sum of squares: at most cols / 32 additions in a row in one thread and
    # 32 more across threads, halved by the root; then a handful of roundings
    return (cols / 32 + 32) / 2 * F24 + 8 * F24


NORM_SHAPES = [(1, 1), (1, 2048), (3, 31), (5, 64), (7, 897), (333, 896), (64, 4096), (9, 4097), (2, 8192), (3, 11008),
               (2, 20000), (1, 131071), (1000, 8), (257, 768), (40, 16384), (33, 1000)]


@pytest.mark.parametrize("type", [0, 1, 30])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("resid,pad,shift", [(False, 0, 0), (True, 16, 0), (True, 3, 1), (False, 8, 8)])
def test_norm(gpu, type, rows, cols, resid, pad, shift):
    g = _gen(rows * 131 + cols + type)
    x = Rows(rows, cols, DT[type], pad, shift, _rand(g, rows, cols))
    r = Rows(rows, cols, DT[type], pad + (16 if pad else 0), shift, _rand(g, rows, cols, scale=3)) if resid else None
    out = Rows(rows, cols, DT[type], pad, shift) if resid else None
    w = 1 + _rand(g, cols, scale=0.05)
    q = Rows(rows, cols, torch.int8, (-cols) % 16 if not shift else pad, 0 if not shift else 5)
    scale = torch.full((rows + 3,), 7.0, device="cuda")
    _ok(gpu, _norm(gpu, type, x, r, out, w, 1e-5, rows, cols, q, scale))
    torch.cuda.synchronize()
    h = x.t.double() + (r.t.double() if resid else 0)
    y = h / (h.square().mean(dim=1, keepdim=True) + float(np.float32(1e-5))).sqrt() * w.double()
    _check_int8(q.t, scale[:rows], y, _norm_r(cols))
    assert q.untouched_around() and torch.all(scale[rows:] == 7)
    if resid:
        half = torch.finfo(DT[type]).eps / 2 + F24
        assert torch.all((out.t.double() - h).abs() <= h.abs() * half + 2.0 ** -25)
        assert out.untouched_around()


@pytest.mark.parametrize("type", [0, 1, 30])
@pytest.mark.parametrize("rows,cols", [(5, 64), (3, 896), (4, 4096), (2, 777), (2, 30000)])
@pytest.mark.parametrize("over", ["x", "resid"])
def test_norm_sum_in_place(gpu, type, rows, cols, over):
    """The sum stored over one of its inputs gives what a separate buffer gives."""
    g = _gen(cols)
    x0, r0 = _rand(g, rows, cols), _rand(g, rows, cols)
    w = 1 + _rand(g, cols, scale=0.05)
    got = []
    for place in (None, over):
        x, r = Rows(rows, cols, DT[type], fill=x0), Rows(rows, cols, DT[type], fill=r0)
        out = {None: Rows(rows, cols, DT[type]), "x": x, "resid": r}[place]
        q, scale = Rows(rows, cols, torch.int8), torch.empty(rows, device="cuda")
        _ok(gpu, _norm(gpu, type, x, r, out, w, 1e-6, rows, cols, q, scale))
        got.append((out.t.clone(), q.t.clone(), scale))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("type", [0, 1, 30])
@pytest.mark.parametrize("cols", [64, 100, 4096])
def test_norm_sum_without_a_residual_and_of_a_row_with_itself(gpu, type, cols):
    g = _gen(cols)
    x = Rows(40, cols, DT[type], fill=_rand(g, 40, cols))
    w = torch.ones(cols, device="cuda")
    q, scale = Rows(40, cols, torch.int8, (-cols) % 16), torch.empty(40, device="cuda")
    out = Rows(40, cols, DT[type])
    _ok(gpu, _norm(gpu, type, x, None, out, w, 1e-5, 40, cols, q, scale))
    assert torch.equal(out.t, x.t)
    _ok(gpu, _norm(gpu, type, x, x, out, w, 1e-5, 40, cols, q, scale))
    assert torch.equal(out.t, x.t + x.t)           # doubling is exact
    h = 2 * x.t.double()
    _check_int8(q.t, scale, h / (h.square().mean(1, True) + float(np.float32(1e-5))).sqrt(), _norm_r(cols))


@pytest.mark.parametrize("cols", [5, 896, 2048, 11008, 40000])
def test_norm_rows_of_zeros_and_of_what_is_not_finite(gpu, cols):
    x = torch.ones(6, cols, device="cuda")
    x[0] = 0
    x[1, cols // 2] = float("nan")
    x[2, cols - 1] = float("inf")
    x[3, 0] = float("-inf")
    x[4] = 1e-30                                   # the mean of squares is below eps
    xr = Rows(6, cols, torch.float32, fill=x)
    q, scale = Rows(6, cols, torch.int8), torch.empty(6, device="cuda")
    w = torch.ones(cols, device="cuda")
    _ok(gpu, _norm(gpu, 0, xr, None, None, w, 1e-5, 6, cols, q, scale))
    s = scale.tolist()
    assert s[0] == 0 and torch.all(q.t[0] == 0)
    for i in (1, 2, 3):
        assert np.isnan(s[i]) and torch.all(q.t[i] == 0)
    _check_int8(q.t[4:], scale[4:], x[4:].double() / (x[4:].double().square().mean(1, True) + float(np.float32(1e-5))).sqrt(),
                _norm_r(cols))


# ---------------------------------------------------------------- gated activation

def _act64(x, act):
    if act == 0:
        return x * torch.sigmoid(x)
    if act == 1:
        return x * torch.sigmoid(2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3))
    return x


def _glu(gpu, type, gate, up, act, rows, cols, q, scale):
    return gpu.lib().llamini_glu_i8_device(type, gate.ptr, gate.ld, up.ptr if up else None, up.ld if up else 0, act,
                                           rows, cols, q.ptr, q.ld, scale.data_ptr(), _stream())


@pytest.mark.parametrize("type", [0, 1, 30])
@pytest.mark.parametrize("act,with_up", [(0, True), (1, True), (1, False), (2, False), (2, True), (0, False)])
@pytest.mark.parametrize("rows,cols,pad,shift", [(1, 1, 0, 0), (1, 11008, 0, 0), (7, 333, 3, 1), (64, 5632, 0, 0), (5, 4864, 16, 0),
                                                 (3, 16400, 0, 8), (2, 40000, 1, 0), (300, 64, 0, 0), (1, 131071, 0, 0)])
def test_glu(gpu, type, act, with_up, rows, cols, pad, shift):
    g = _gen(rows + cols + act)
    gate = Rows(rows, cols, DT[type], pad, shift, _rand(g, rows, cols, scale=3))
    up = Rows(rows, cols, DT[type], pad, shift, _rand(g, rows, cols)) if with_up else None
    q = Rows(rows, cols, torch.int8, pad if shift else (-cols) % 16, 3 if shift else 0)
    scale = torch.full((rows + 2,), 7.0, device="cuda")
    _ok(gpu, _glu(gpu, type, gate, up, act, rows, cols, q, scale))
    torch.cuda.synchronize()
    x, u = gate.t.double(), up.t.double() if with_up else torch.ones(1, 1, device="cuda", dtype=torch.double)
    y = _act64(x, act) * u
    # exp and tanh within 2 ulp, the sums with 1 and the products: relative 16
    # roundings; 1 + tanh cancels, which leaves 2^-22 of |x u| as it stands
    # (and the argument of tanh is itself off by 4 roundings: z (1 - tanh^2) < 0.45)
    extra = ((x * u).abs() * 2.0 ** -22).amax(dim=1, keepdim=True) if act == 1 else 0.0
    if act == 1:
        s = y.abs().amax(dim=1) / 127
        assert torch.all((scale[:rows].double() - s).abs() <= s * 20 * F24 + extra[:, 0] / 127)
        assert torch.all((q.t.double() - y / s[:, None]).abs() <= 0.5 + 127 * 20 * F24 + 2 * extra / s[:, None])
    else:
        _check_int8(q.t, scale[:rows], y, 20 * F24)
    assert q.untouched_around() and torch.all(scale[rows:] == 7)


def test_glu_gate_and_up_side_by_side(gpu):
    g = _gen(3)
    rows, cols = 50, 4864
    both = _rand(g, rows, 2 * cols).to(torch.bfloat16)
    q, scale = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    L = gpu.lib()
    _ok(gpu, L.llamini_glu_i8_device(30, both.data_ptr(), 2 * cols, both.data_ptr() + 2 * cols, 2 * cols, 0, rows, cols,
                                     q.data_ptr(), cols, scale.data_ptr(), _stream()))
    y = _act64(both[:, :cols].double(), 0) * both[:, cols:].double()
    _check_int8(q, scale, y, 20 * F24)


@pytest.mark.parametrize("cols", [3, 512, 11008, 50000])
def test_glu_extreme_rows(gpu, cols):
    x = torch.ones(8, cols, device="cuda")
    x[0] = 0
    x[1, cols // 2] = float("nan")
    x[2, cols - 1] = float("inf")
    x[3] *= 1e-38
    x[4] *= 2e-43                                  # subnormal, the scale rounds
    x[5] *= 1e-45                                  # the scale rounds to zero
    x[6] *= 3e38
    x[7, 0] = -127.0
    gate = Rows(8, cols, torch.float32, fill=x)
    q, scale = Rows(8, cols, torch.int8), torch.empty(8, device="cuda")
    _ok(gpu, _glu(gpu, 0, gate, None, 2, 8, cols, q, scale))
    s = scale.double()
    assert s[0] == 0 and torch.all(q.t[0] == 0)
    for i in (1, 2):
        assert np.isnan(float(s[i])) and torch.all(q.t[i] == 0)
    for i in (3, 6, 7):
        _check_int8(q.t[i:i + 1], scale[i:i + 1], x[i:i + 1].double(), 4 * F24)
    # a scale that is a multiple of 2^-149 is up to 2^-150 off max / 127, which 127
    # steps of it multiply: |q s - x| <= s / 2 + 127 * 2^-150
    assert s[4] > 0 and torch.all((q.t[4].double() * s[4] - x[4].double()).abs() <= s[4] / 2 + 127 * 2.0 ** -150)
    assert s[5] == 0 and torch.all(q.t[5] == 0)


def test_ties_go_to_even(gpu):
    """Rows of max 127 have scale 1: halves are ties."""
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5, 3.4999998, 0.49999997]], device="cuda")
    gate = Rows(1, 11, torch.float32, fill=x)
    q, scale = Rows(1, 11, torch.int8), torch.empty(1, device="cuda")
    _ok(gpu, _glu(gpu, 0, gate, None, 2, 1, 11, q, scale))
    assert float(scale[0]) == 1.0
    assert q.t[0].tolist() == [127, 0, 2, 2, 0, -2, -2, 126, -126, 3, 0]


# ---------------------------------------------------------------- weights

def _weights_call(gpu, t, raw, rows, cols, q, scale):
    return gpu.lib().llamini_weights_i8_device(t, raw, rows, cols, q.ptr, q.ld, scale.data_ptr(), _stream())


def _want_weights(w):
    """Exact: the f32 scale and reciprocal, then the product of two f32 numbers
    in 64 bits, which holds it whole."""
    top = w.abs().amax(dim=1).double()
    s = (top / 127).float()
    inv = torch.where(top > 0, 127 / top, torch.zeros_like(top)).float().double()
    return torch.round(w.double() * inv[:, None]).to(torch.int8), s


@pytest.mark.parametrize("t", [0, 1, 2, 3, 6, 8, 12, 13, 14])
@pytest.mark.parametrize("rows,blocks", [(1, 1), (3, 2), (37, 7), (130, 8), (5, 43), (2, 200)])
def test_weights_exact(gpu, orc, synth, t, rows, blocks):
    cols = 256 * blocks
    if t in (0, 1):
        cols -= 3 if blocks % 2 else 0             # F32 and F16 rows of any length
    elif t < 12 and blocks % 2:
        cols -= 96                                 # not a multiple of 256
    rng = np.random.default_rng(t * 100 + blocks)
    if t == 0:
        raw = rng.standard_normal(rows * cols).astype(np.float32).view(np.uint8)
    elif t == 1:
        raw = rng.standard_normal(rows * cols).astype(np.float16).view(np.uint8)
    else:
        raw = synth.random_blocks(rng, t, rows * cols)
    w = torch.from_numpy(orc.dequant(t, raw, rows * cols).reshape(rows, cols)).cuda()
    want_q, want_s = _want_weights(w)
    for shift in (0, 4 if t == 0 else 2):          # block rows at any alignment of their fields
        d = torch.empty(raw.size + shift, dtype=torch.uint8, device="cuda")
        d[shift:].copy_(torch.from_numpy(raw))
        q = Rows(rows, cols, torch.int8, (-cols) % 16 if not shift else 5, shift)
        scale = torch.full((rows + 2,), 7.0, device="cuda")
        _ok(gpu, _weights_call(gpu, t, d.data_ptr() + shift, rows, cols, q, scale))
        assert torch.equal(scale[:rows], want_s)
        assert torch.equal(q.t, want_q)
        assert q.untouched_around() and torch.all(scale[rows:] == 7)


@pytest.mark.parametrize("t,cols", [(0, 131071), (1, 131071), (8, 131040), (14, 130816), (12, 130816)])
def test_weights_longest_rows(gpu, orc, synth, t, cols):
    rng = np.random.default_rng(cols)
    if t == 0:
        raw = rng.standard_normal(2 * cols).astype(np.float32).view(np.uint8)
    elif t == 1:
        raw = rng.standard_normal(2 * cols).astype(np.float16).view(np.uint8)
    else:
        raw = synth.random_blocks(rng, t, 2 * cols)
    w = torch.from_numpy(orc.dequant(t, raw, 2 * cols).reshape(2, cols)).cuda()
    want_q, want_s = _want_weights(w)
    d = torch.from_numpy(raw.copy()).cuda()
    q, scale = Rows(2, cols, torch.int8), torch.empty(2, device="cuda")
    _ok(gpu, _weights_call(gpu, t, d.data_ptr(), 2, cols, q, scale))
    assert torch.equal(scale, want_s) and torch.equal(q.t, want_q)


@pytest.mark.parametrize("t", [2, 3, 6, 8, 12, 13, 14])
def test_weights_special_scales(gpu, orc, golden, t):
    """The golden blocks hold zero, subnormal, infinite and NaN scales: one row
    each, so that finite rows are exact and the others get a NaN scale."""
    raw = golden["dequant"]["raw_%d" % t]
    w = torch.from_numpy(golden["dequant"]["out_%d" % t].copy())
    be, bb = {2: (32, 18), 3: (32, 20), 6: (32, 22), 8: (32, 34), 12: (256, 144), 13: (256, 176), 14: (256, 210)}[t]
    rows = w.numel() // be
    w = w.view(rows, be).cuda()
    d = torch.from_numpy(raw[:rows * bb].copy()).cuda()
    q, scale = Rows(rows, be, torch.int8), torch.empty(rows, device="cuda")
    _ok(gpu, _weights_call(gpu, t, d.data_ptr(), rows, be, q, scale))
    fine = torch.isfinite(w).all(dim=1)
    assert torch.isnan(scale[~fine]).all() and torch.all(q.t[~fine] == 0)
    want_q, want_s = _want_weights(w[fine])
    assert torch.equal(scale[fine], want_s)
    normal = want_s > 1.2e-38                      # below, q is w / scale and scales are subnormal: as in test_glu_extreme_rows
    assert torch.equal(q.t[fine][normal], want_q[normal])
    rest, s = q.t[fine][~normal].double(), want_s[~normal].double()
    assert torch.all((rest * s[:, None] - w[fine][~normal].double()).abs() <= s[:, None] / 2 + 127 * 2.0 ** -150)


# ---------------------------------------------------------------- matrix product

def _gemm(gpu, a, sa, w, sw, bias, type, out, m, n, k):
    return gpu.lib().llamini_gemm_i8_device(a.ptr, a.ld, sa.data_ptr(), m, w.ptr, w.ld, sw.data_ptr(), n, k,
                                            bias.data_ptr() if bias is not None else None, type, out.ptr, out.ld, _stream())


def _ints(g, rows, cols, low=-127):
    return torch.randint(low, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int8)


def _check_gemm(out, type, a, sa, w, sw, bias):
    p = a.double() @ w.double().t() * sa.double()[:, None] * sw.double()[None, :]
    want = p + bias.double() if bias is not None else p
    eps = torch.finfo(DT[type]).eps / 2 if type != 0 else 0.0
    tol = p.abs() * 4 * F24 + want.abs() * (2 * F24 + eps) + (2.0 ** -25 if type == 1 else 1e-37)
    d = (out.double() - want).abs()
    assert torch.all(d <= tol), float((d / want.abs().clamp_min(1e-30)).max())


def _run_gemm(gpu, m, n, k, type, bias, pad_a=None, pad_w=None, pad_o=0, shift_a=0, shift_w=0, shift_o=0, low=-127, seed=0):
    g = _gen(m * 7 + n * 3 + k + seed)
    a = Rows(m, k, torch.int8, (-k) % 16 if pad_a is None else pad_a, shift_a, _ints(g, m, k, low))
    w = Rows(n, k, torch.int8, (-k) % 16 if pad_w is None else pad_w, shift_w, _ints(g, n, k, low))
    sa = torch.rand(m, generator=g, device="cuda") * 0.01 + 0.001
    sw = torch.rand(n, generator=g, device="cuda") * 0.001 + 0.0001
    b = _rand(g, n) if bias else None
    out = Rows(m, n, DT[type], pad_o, shift_o)
    _ok(gpu, _gemm(gpu, a, sa, w, sw, b, type, out, m, n, k))
    torch.cuda.synchronize()
    _check_gemm(out.t, type, a.t, sa, w.t, sw, b)
    assert out.untouched_around()


SHAPES = [(1, 1, 1), (1, 2560, 2048), (2, 64, 32), (3, 130, 100), (5, 4096, 11008), (8, 129, 512), (15, 257, 4096), (16, 256, 128),
          (17, 1000, 897), (31, 896, 4864), (32, 2048, 2048), (33, 33, 33), (64, 5632, 2048), (65, 127, 300), (100, 896, 896),
          (128, 128, 128), (129, 1152, 896), (200, 2304, 768), (255, 255, 255), (256, 4096, 512), (257, 515, 1024),
          (333, 1152, 896), (500, 4864, 896), (512, 512, 127), (1000, 2000, 64), (1023, 3200, 2048), (1024, 1024, 1024),
          (2000, 896, 640), (4100, 300, 256), (1, 32000, 64), (40, 32001, 80), (300, 17, 5000), (4096, 64, 128)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("type,bias", [(0, False), (0, True), (1, True), (30, False), (30, True)])
def test_gemm(gpu, m, n, k, type, bias):
    _run_gemm(gpu, m, n, k, type, bias)


@pytest.mark.parametrize("m,n,k", [(1, 300, 333), (64, 200, 1000), (70, 129, 129), (300, 513, 777), (513, 260, 64)])
@pytest.mark.parametrize("type", [0, 1, 30])
@pytest.mark.parametrize("layout", [dict(pad_a=0, pad_w=0), dict(pad_a=3), dict(pad_w=5), dict(shift_a=1), dict(shift_w=7),
                                    dict(pad_o=1, shift_o=1), dict(pad_o=5), dict(pad_o=8, shift_o=8), dict(shift_a=16, shift_w=32),
                                    dict(pad_a=64, pad_w=160, pad_o=64)])
def test_gemm_pitches_and_alignments(gpu, m, n, k, type, layout):
    layout = dict(layout)
    for key in ("pad_a", "pad_w"):                 # whole pitches where the case is not about them
        if layout.get(key, 0) % 16 == 0 and key in layout and layout[key]:
            layout[key] += (-k) % 16
    _run_gemm(gpu, m, n, k, type, True, **layout)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("n,k", [(1, 1), (9, 15), (77, 16), (130, 17), (9001, 35), (40, 1000), (33, 2047), (200, 4095), (3, 5001)])
@pytest.mark.parametrize("layout", [dict(), dict(pad_a=0, pad_w=0), dict(pad_a=1, pad_w=2, shift_a=3, shift_w=1),
                                    dict(shift_w=2, pad_w=4), dict(pad_a=13, pad_w=29, shift_w=5)])
def test_gemm_few_tokens_at_any_address(gpu, m, n, k, layout):
    _run_gemm(gpu, m, n, k, 0, True, **layout)


# more than eight tokens where TMA cannot read: eight a CTA while there are few tiles
# of 64 x 64 and the rows are short, else the tiles
@pytest.mark.parametrize("m,n,k", [(9, 77, 33), (16, 260, 1000), (17, 1, 1), (65, 500, 2047), (130, 300, 5631), (8193, 5, 3),
                                   (9, 130, 6001), (64, 64, 5700), (70, 33, 12289), (700, 1100, 333), (130, 9001, 65),
                                   (833, 641, 64), (1000, 600, 63)])
@pytest.mark.parametrize("layout", [dict(pad_a=0, pad_w=0), dict(pad_a=1, pad_w=2, shift_a=3, shift_w=1), dict(shift_w=2, pad_o=5)])
@pytest.mark.parametrize("type", [0, 30])
def test_gemm_more_tokens_at_any_address(gpu, m, n, k, layout, type):
    _run_gemm(gpu, m, n, k, type, True, **layout)


@pytest.mark.parametrize("m,n", [(1, 40), (20, 40), (130, 300)])
def test_gemm_longest_sums(gpu, m, n):
    """131071 columns of -128 x -128, the largest sum: 2147467264."""
    k = 131071
    a = Rows(m, k, torch.int8, 1, fill=torch.full((m, k), -128, dtype=torch.int8, device="cuda"))
    w = Rows(n, k, torch.int8, 1, fill=torch.full((n, k), -128, dtype=torch.int8, device="cuda"))
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    out = Rows(m, n, torch.float32)
    _ok(gpu, _gemm(gpu, a, one_m, w, one_n, None, 0, out, m, n, k))
    assert torch.all(out.t == 2147467264.0)        # 131071 * 2^14 is an f32 number: 17 bits
    w.t.fill_(127)
    _ok(gpu, _gemm(gpu, a, one_m, w, one_n, None, 0, out, m, n, k))
    assert torch.all(out.t == float(np.float32(-131071 * 128 * 127)))


@pytest.mark.parametrize("m", [1, 64, 300])
def test_gemm_scales_that_are_zero_or_not_finite(gpu, m):
    n, k = 200, 256
    g = _gen(m)
    a, w = Rows(m, k, torch.int8, fill=_ints(g, m, k)), Rows(n, k, torch.int8, fill=_ints(g, n, k))
    sa, sw = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    sw[3], sw[5], sa[0] = 0.0, float("nan"), 2.0
    if m > 1:
        sa[1] = float("nan")
    out = Rows(m, n, torch.float32)
    _ok(gpu, _gemm(gpu, a, sa, w, sw, None, 0, out, m, n, k))
    want = (a.t.double() @ w.t.double().t()).float() * sa[:, None] * sw[None, :]
    assert torch.equal(torch.isnan(out.t), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(out.t), torch.nan_to_num(want))


def test_gemm_output_past_the_range_of_f16(gpu):
    a = Rows(3, 64, torch.int8, fill=torch.full((3, 64), 127, dtype=torch.int8, device="cuda"))
    w = Rows(40, 64, torch.int8, fill=torch.full((40, 64), 127, dtype=torch.int8, device="cuda"))
    one3, one40 = torch.ones(3, device="cuda"), torch.ones(40, device="cuda")
    out = Rows(3, 40, torch.float16)
    _ok(gpu, _gemm(gpu, a, one3, w, one40, None, 1, out, 3, 40, 64))
    assert torch.all(torch.isinf(out.t))


def test_gemm_pitches_past_32_bits(gpu):
    """Rows 2.2 GB apart: offsets of rows pass 32 bits."""
    k, n, far = 64, 3, 2_200_000_000 // 16 * 16
    buf = torch.zeros(2 * far + 64, dtype=torch.int8, device="cuda")
    g = _gen(1)
    rows = _ints(g, n, k)
    for i in range(n):
        buf[i * far:i * far + k] = rows[i]
    sa = torch.ones(n, device="cuda")
    out = torch.empty(n, n, device="cuda")
    L = gpu.lib()
    for ld_a, a in ((k, rows), (far, buf)):
        for ld_w, w in ((k, rows), (far, buf)):
            out.fill_(0)
            _ok(gpu, L.llamini_gemm_i8_device(a.data_ptr(), ld_a, sa.data_ptr(), n, w.data_ptr(), ld_w, sa.data_ptr(), n, k,
                                              None, 0, out.data_ptr(), n, _stream()))
            assert torch.equal(out.double(), rows.double() @ rows.double().t())


@pytest.mark.parametrize("type", [0, 1, 30])
@pytest.mark.parametrize("n,k", [(300, 512), (896, 4864), (2048, 100)])
def test_gemm_outputs_do_not_depend_on_the_batch(gpu, type, n, k):
    """A token alone, in batches of every kernel and tile, and from rows of an
    odd pitch: the same bits."""
    g = _gen(n)
    m = 1200
    a, w = Rows(m, k, torch.int8, (-k) % 16, fill=_ints(g, m, k)), Rows(n, k, torch.int8, (-k) % 16, fill=_ints(g, n, k))
    sa, sw, b = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda"), _rand(g, n, scale=100.0)
    whole = Rows(m, n, DT[type])
    _ok(gpu, _gemm(gpu, a, sa, w, sw, b, type, whole, m, n, k))
    for rows in (1, 2, 3, 7, 16, 31, 64, 100, 200, 500):
        for layout in (a, Rows(rows, k, torch.int8, 3, 1, a.t[:rows])):
            out = Rows(rows, n, DT[type], pad=5 if rows % 2 else 0)
            _ok(gpu, _gemm(gpu, layout, sa, w, sw, b, type, out, rows, n, k))
            assert torch.equal(out.t, whole.t[:rows])


# ---------------------------------------------------------------- large and far

@pytest.mark.parametrize("m,n,k", [(70001, 64, 64), (70001, 130, 48), (66000, 9, 33), (2, 140000, 64), (40, 140001, 64),
                                   (300, 70000, 96)])
def test_gemm_many_rows_or_channels(gpu, m, n, k):
    _run_gemm(gpu, m, n, k, 0, True)


@pytest.mark.parametrize("type", [0, 30])
@pytest.mark.parametrize("cols", [8, 17, 300])
def test_row_operators_many_rows(gpu, type, cols):
    rows = 70001
    g = _gen(cols)
    x, r = Rows(rows, cols, DT[type], fill=_rand(g, rows, cols)), Rows(rows, cols, DT[type], fill=_rand(g, rows, cols))
    w = 1 + _rand(g, cols, scale=0.05)
    q, scale = Rows(rows, cols, torch.int8, (-cols) % 16), torch.empty(rows, device="cuda")
    _ok(gpu, _norm(gpu, type, x, r, None, w, 1e-5, rows, cols, q, scale))
    h = x.t.double() + r.t.double()
    _check_int8(q.t, scale, h / (h.square().mean(1, True) + float(np.float32(1e-5))).sqrt() * w.double(), _norm_r(cols))
    _ok(gpu, _glu(gpu, type, x, r, 0, rows, cols, q, scale))
    _check_int8(q.t, scale, _act64(x.t.double(), 0) * r.t.double(), 20 * F24)
    assert q.untouched_around()


@pytest.mark.parametrize("cols", [64, 67, 4096])
def test_pitches_past_32_bits(gpu, cols):
    """Three rows 2.2 GB apart, of inputs and of int8 rows: offsets of rows
    pass 32 bits in elements and in bytes."""
    rows, far = 3, 2_200_000_000 // 64 * 64
    g = _gen(cols)
    buf = torch.empty(2 * far + 65536, dtype=torch.uint8, device="cuda")
    x = _rand(g, rows, cols).half()
    w = torch.ones(cols, device="cuda")
    L = gpu.lib()
    near_q, near_s = torch.empty(rows, 4096, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    far_s = torch.empty(rows, device="cuda")
    xf = buf.view(torch.float16)
    for i in range(rows):
        xf[i * far // 2:i * far // 2 + cols] = x[i]
    at_q = buf.data_ptr() + 32768
    for run in (lambda p, ld, q, ldq, s: L.llamini_rms_norm_i8_device(1, p, ld, None, 0, None, 0, w.data_ptr(), 1e-5, rows, cols,
                                                                      q, ldq, s.data_ptr(), _stream()),
                lambda p, ld, q, ldq, s: L.llamini_glu_i8_device(1, p, ld, None, 0, 0, rows, cols, q, ldq, s.data_ptr(), _stream())):
        _ok(gpu, run(x.data_ptr(), cols, near_q.data_ptr(), 4096, near_s))
        _ok(gpu, run(buf.data_ptr(), far // 2, at_q, far, far_s))
        assert torch.equal(near_s, far_s)
        for i in range(rows):
            assert torch.equal(buf[i * far + 32768:i * far + 32768 + cols].view(torch.int8), near_q[i, :cols])
    # outputs of a product that far apart
    a = _ints(g, rows, 64)
    ones = torch.ones(cols, device="cuda")
    b = _ints(g, cols, 64)
    near = torch.empty(rows, cols, device="cuda")
    _ok(gpu, L.llamini_gemm_i8_device(a.data_ptr(), 64, ones.data_ptr(), rows, b.data_ptr(), 64, ones.data_ptr(), cols, 64, None, 0,
                                      near.data_ptr(), cols, _stream()))
    _ok(gpu, L.llamini_gemm_i8_device(a.data_ptr(), 64, ones.data_ptr(), rows, b.data_ptr(), 64, ones.data_ptr(), cols, 64, None, 0,
                                      buf.data_ptr(), far // 4, _stream()))
    f = buf.view(torch.float32)
    for i in range(rows):
        assert torch.equal(f[i * far // 4:i * far // 4 + cols], near[i])


# ---------------------------------------------------------------- together

def _feed_forward(gpu, x, resid, w, gate_up, s_gu, down, s_d, act, type):
    """One layer's feed-forward half as a caller runs it: norm with the
    residual's addition, gate|up in one product, the gated activation, down."""
    L, st = gpu.lib(), _stream()
    rows, dim = x.shape
    ffn = gate_up.shape[0] // 2
    e = dict(device="cuda")
    h = torch.empty_like(x)
    q1, s1 = torch.empty(rows, dim, dtype=torch.int8, **e), torch.empty(rows, **e)
    gu = torch.empty(rows, 2 * ffn, dtype=x.dtype, **e)
    q2, s2 = torch.empty(rows, ffn, dtype=torch.int8, **e), torch.empty(rows, **e)
    y = torch.empty(rows, dim, dtype=x.dtype, **e)

    def run():
        st = _stream()
        _ok(gpu, L.llamini_rms_norm_i8_device(type, x.data_ptr(), dim, resid.data_ptr(), dim, h.data_ptr(), dim, w.data_ptr(),
                                              1e-5, rows, dim, q1.data_ptr(), dim, s1.data_ptr(), st))
        _ok(gpu, L.llamini_gemm_i8_device(q1.data_ptr(), dim, s1.data_ptr(), rows, gate_up.data_ptr(), dim, s_gu.data_ptr(),
                                          2 * ffn, dim, None, type, gu.data_ptr(), 2 * ffn, st))
        _ok(gpu, L.llamini_glu_i8_device(type, gu.data_ptr(), 2 * ffn, gu.data_ptr() + ffn * gu.element_size(), 2 * ffn, act,
                                         rows, ffn, q2.data_ptr(), ffn, s2.data_ptr(), st))
        _ok(gpu, L.llamini_gemm_i8_device(q2.data_ptr(), ffn, s2.data_ptr(), rows, down.data_ptr(), ffn, s_d.data_ptr(),
                                          dim, ffn, None, type, y.data_ptr(), dim, st))
    return run, h, y, (q1, s1, gu, q2, s2)


def _ffn_weights(gpu, orc, synth, dim, ffn, t_gu=12, t_down=14):
    rng = np.random.default_rng(dim + ffn)
    out = []
    for t, n, k in ((t_gu, 2 * ffn, dim), (t_down, dim, ffn)):
        raw = synth.random_blocks(rng, t, n * k)
        d = torch.from_numpy(raw.copy()).cuda()
        q, s = torch.empty(n, k, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
        _ok(gpu, gpu.lib().llamini_weights_i8_device(t, d.data_ptr(), n, k, q.data_ptr(), k, s.data_ptr(), _stream()))
        torch.cuda.synchronize()
        out += [q, s, torch.from_numpy(orc.dequant(t, raw, n * k).reshape(n, k)).cuda()]
    return out


@pytest.mark.parametrize("rows", [1, 5, 64, 200, 700])
@pytest.mark.parametrize("type,act", [(0, 0), (30, 0), (1, 1)])
def test_feed_forward_from_gguf_blocks(gpu, orc, synth, rows, type, act):
    """Q4_K gate|up and Q6_K down become int8 once; the run of the four
    operators is, step by step, each operator's own definition, and the whole
    is the f32 feed-forward within what 8 bits leave of it."""
    dim, ffn = 512, 1024
    gu_q, gu_s, gu_w, d_q, d_s, d_w = _ffn_weights(gpu, orc, synth, dim, ffn)
    gu_s, gu_w = gu_s * 0.05, gu_w * 0.05          # keeps gate in the activation's curved range
    g = _gen(rows)
    x, r = _rand(g, rows, dim).to(DT[type]), _rand(g, rows, dim).to(DT[type])
    w = 1 + _rand(g, dim, scale=0.05)
    run, h, y, (q1, s1, gu, q2, s2) = _feed_forward(gpu, x, r, w, gu_q, gu_s, d_q, d_s, act, type)
    run()
    torch.cuda.synchronize()
    _check_gemm(gu, type, q1, s1, gu_q, gu_s, None)
    _check_gemm(y, type, q2, s2, d_q, d_s, None)
    h64 = x.double() + r.double()
    n64 = h64 / (h64.square().mean(1, True) + 1e-5).sqrt() * w.double()
    gate, up = (n64 @ gu_w.double().t()).chunk(2, dim=1)
    want = (_act64(gate, act) * up) @ d_w.double().t()
    # every int8 value is within half of max / 127 of what it stands for; on
    # rows of a few standard deviations at most that is 1 - 2 % of their
    # norm, four such roundings, and quadratic terms: within a tenth
    err = (y.double() - want).norm() / want.norm()
    assert err < 0.1, float(err)


def test_captured_run_replays_on_new_inputs(gpu, orc, synth):
    """The run captured into a CUDA graph and replayed on other inputs equals
    the eager one, while another captured run of the same weights is alive."""
    dim, ffn, rows = 512, 1024, 33
    gu_q, gu_s, _, d_q, d_s, _ = _ffn_weights(gpu, orc, synth, dim, ffn)
    g = _gen(5)
    w = torch.ones(dim, device="cuda")
    graphs, kept = [], []                          # a captured run goes on using its buffers
    for k in range(2):
        x, r = _rand(g, rows, dim).bfloat16(), _rand(g, rows, dim).bfloat16()
        run, h, y, _ = _feed_forward(gpu, x, r, w, gu_q, gu_s, d_q, d_s, 0, 30)
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append((graph, x, r, h, y))
        kept.append(run)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    fresh = [(_rand(g, rows, dim).bfloat16(), _rand(g, rows, dim).bfloat16()) for _ in range(2)]
    for (graph, x, r, h, y), (nx, nr), st in zip(graphs, fresh, streams):
        x.copy_(nx)
        r.copy_(nr)
    torch.cuda.synchronize()
    for _ in range(20):                            # both at once
        for (graph, *_), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for (graph, x, r, h, y), (nx, nr) in zip(graphs, fresh):
        run, h2, y2, _ = _feed_forward(gpu, nx, nr, w, gu_q, gu_s, d_q, d_s, 0, 30)
        run()
        torch.cuda.synchronize()
        assert torch.equal(h, h2) and torch.equal(y, y2)


def test_calls_on_two_streams_at_once(gpu):
    """Products without anything shared between calls: two streams, many calls
    in flight, each result that of the call alone."""
    g = _gen(9)
    jobs = []
    for m, n, k in ((1, 4096, 4096), (16, 2048, 5632), (200, 1000, 900), (512, 1024, 512)):
        kp = (k + 15) // 16 * 16
        a, w = _ints(g, m, kp), _ints(g, n, kp)
        sa, sw = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
        jobs.append((m, n, k, kp, a, w, sa, sw))
    L = gpu.lib()

    def call(j, out, st):
        m, n, k, kp, a, w, sa, sw = j
        _ok(gpu, L.llamini_gemm_i8_device(a.data_ptr(), kp, sa.data_ptr(), m, w.data_ptr(), kp, sw.data_ptr(), n, k, None, 0,
                                          out.data_ptr(), n, st))
    want = [torch.empty(j[0], j[1], device="cuda") for j in jobs]
    for j, o in zip(jobs, want):
        call(j, o, _stream())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(o) for o in want] for _ in streams]
    for _ in range(10):
        for st, os_ in zip(streams, outs):
            for j, o in zip(jobs, os_):
                call(j, o, st.cuda_stream)
    torch.cuda.synchronize()
    for os_ in outs:
        for o, wo in zip(os_, want):
            assert torch.equal(o, wo)


def test_weights_are_ready_for_the_product_behind_them(gpu, synth):
    """Weights and product back to back on one stream, without a wait between
    them, each time with other weights in the same buffers."""
    n, k = 2048, 2048
    rng = np.random.default_rng(3)
    raws = [torch.from_numpy(synth.random_blocks(rng, 8, n * k).copy()).cuda() for _ in range(3)]
    q, s = torch.empty(n, k, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    L, st = gpu.lib(), _stream()
    for m in (1, 16, 700):
        a, sa = _ints(_gen(m), m, k), torch.ones(m, device="cuda")
        want, outs = [], []
        for wait in (True, False):
            for raw in raws * 3:
                out = torch.empty(m, n, device="cuda")
                _ok(gpu, L.llamini_weights_i8_device(8, raw.data_ptr(), n, k, q.data_ptr(), k, s.data_ptr(), st))
                if wait:
                    torch.cuda.synchronize()
                _ok(gpu, L.llamini_gemm_i8_device(a.data_ptr(), k, sa.data_ptr(), m, q.data_ptr(), k, s.data_ptr(), n, k, None, 0,
                                                  out.data_ptr(), n, st))
                (want if wait else outs).append(out)
        torch.cuda.synchronize()
        for x, y in zip(want, outs):
            assert torch.equal(x, y)


def test_calls_from_two_host_threads(gpu):
    """Each thread on a stream of its own, the same products at once."""
    import threading
    g = _gen(4)
    shapes = [(1, 512, 1024), (20, 900, 640), (300, 512, 384), (5, 100, 77)]
    jobs = []
    for m, n, k in shapes:
        kp = (k + 15) // 16 * 16
        jobs.append((m, n, k, kp, _ints(g, m, kp), _ints(g, n, kp), torch.rand(m, generator=g, device="cuda"),
                     torch.rand(n, generator=g, device="cuda")))
    L = gpu.lib()
    outs = [[torch.empty(j[0], j[1], device="cuda") for j in jobs] for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    failed = []

    def work(t):
        for _ in range(30):
            for (m, n, k, kp, a, w, sa, sw), o in zip(jobs, outs[t]):
                if L.llamini_gemm_i8_device(a.data_ptr(), kp, sa.data_ptr(), m, w.data_ptr(), kp, sw.data_ptr(), n, k, None, 0,
                                            o.data_ptr(), n, streams[t].cuda_stream) != 0:
                    failed.append(gpu.last_error())
    threads = [threading.Thread(target=work, args=(t,)) for t in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed[0]
    for (m, n, k, kp, a, w, sa, sw), x, y, z in zip(jobs, *outs):
        _check_gemm(x, 0, a[:, :k], sa, w[:, :k], sw, None)
        assert torch.equal(x, y) and torch.equal(x, z)


def test_no_wait_has_run_out(gpu):
    """After every product above: no kernel has given up a wait."""
    assert gpu.lib().llamini_i8_status(_stream()) == 0, gpu.last_error()


def test_host_memory_is_refused(gpu):
    h = np.zeros(4096, np.int8)
    d = torch.zeros(4096, dtype=torch.int8, device="cuda")
    s = torch.zeros(64, device="cuda")
    L = gpu.lib()
    for a, w in ((h.ctypes.data, d.data_ptr()), (d.data_ptr(), h.ctypes.data)):
        assert L.llamini_gemm_i8_device(a, 64, s.data_ptr(), 4, w, 64, s.data_ptr(), 4, 64, None, 0, s.data_ptr(), 4, None) == -1
        assert "not memory of the current device" in gpu.last_error()
    assert L.llamini_glu_i8_device(0, h.ctypes.data, 16, None, 0, 2, 1, 16, d.data_ptr(), 16, s.data_ptr(), None) == -1
    L.llamini_clear_error()
