"""The int8 operators where they could go wrong: ends of kernels, long walks,
lengths at the edge of a launch's limits and values at the edge of a type's range.
Definitions and tolerances as in test_gpu_i8.py."""
from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import conftest  # noqa: E402
import test_gpu_i8 as base  # noqa: E402

pytestmark = pytest.mark.gpu

DT, F24, Rows = base.DT, base.F24, base.Rows


def _product(gpu, m, n, k, type, seed):
    """A product's arguments with its output; call() runs it on a stream."""
    g = base._gen(seed)
    a = Rows(m, k, torch.int8, (-k) % 16, 0, base._ints(g, m, k))
    w = Rows(n, k, torch.int8, (-k) % 16, 0, base._ints(g, n, k))
    sa = torch.rand(m, generator=g, device="cuda") * 0.01 + 0.001
    sw = torch.rand(n, generator=g, device="cuda") * 0.001 + 0.0001
    b = base._rand(g, n)

    def call(out, stream):
        return gpu.lib().llamini_gemm_i8_device(a.ptr, a.ld, sa.data_ptr(), m, w.ptr, w.ld, sw.data_ptr(), n, k, b.data_ptr(),
                                                type, out.ptr, out.ld, stream)
    return a, w, sa, sw, b, call


# several tiles a pair of CTAs and several slabs of columns a tile, so that stages and
# accumulators wrap from tile to tile; with and without halved last tiles; 16-byte and
# odd output pitches
@pytest.mark.parametrize("m,n,k,pad", [(2048, 4232, 2000, 8), (4096, 2568, 700, 0), (1000, 8000, 1152, 0), (2300, 2570, 900, 5),
                                       (300, 32001, 640, 0)])
@pytest.mark.parametrize("type", [0, 30])
def test_products_of_several_tiles_a_pair(gpu, m, n, k, pad, type):
    a, w, sa, sw, b, call = _product(gpu, m, n, k, type, m + n)
    out = Rows(m, n, DT[type], pad)
    base._ok(gpu, call(out, base._stream()))
    torch.cuda.synchronize()
    base._check_gemm(out.t, type, a.t, sa, w.t, sw, b)
    assert out.untouched_around()


def test_products_of_every_kernel_behind_one_another(gpu):
    """CTAs of one product take the shared memory that those of another have just
    left, on two streams: the same bits each time, so that nothing of a kernel that has
    ended arrives in the next one's barriers or stages."""
    shapes = [(600, 2304, 300), (32, 2048, 2048), (1024, 1024, 130), (3, 1000, 512), (2048, 4226, 260), (100, 896, 896)]
    jobs = [_product(gpu, m, n, k, 30, i) + (m, n) for i, (m, n, k) in enumerate(shapes)]
    want = []
    for a, w, sa, sw, b, call, m, n in jobs:
        out = Rows(m, n, torch.bfloat16)
        base._ok(gpu, call(out, base._stream()))
        torch.cuda.synchronize()
        base._check_gemm(out.t, 30, a.t, sa, w.t, sw, b)
        want.append(out.t.clone())
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[[Rows(j[6], j[7], torch.bfloat16) for j in jobs] for _ in range(8)] for _ in streams]
    torch.cuda.synchronize()
    for r in range(8):
        for s, st in enumerate(streams):
            for i in range(len(jobs)):
                i = (i + 2 * s) % len(jobs)
                base._ok(gpu, jobs[i][5](outs[s][r][i], st.cuda_stream))
    torch.cuda.synchronize()
    for per in outs:
        for row in per:
            for o, x in zip(row, want):
                assert torch.equal(o.t, x)


@pytest.mark.parametrize("type", [0, 1, 30])
@pytest.mark.parametrize("cut", range(1, 9))
@pytest.mark.parametrize("m,n,k", [(513, 2600, 260), (1024, 4224, 130)])
def test_product_leaves_the_end_of_a_unit_alone(gpu, m, n, k, cut, type):
    """Rows in pitches of whole 16-byte units that end inside a unit: what lies
    behind a row's last channel stays as it was."""
    n -= cut
    a, w, sa, sw, b, call = _product(gpu, m, n, k, type, cut)
    out = Rows(m, n, DT[type], cut)
    base._ok(gpu, call(out, base._stream()))
    torch.cuda.synchronize()
    base._check_gemm(out.t, type, a.t, sa, w.t, sw, b)
    assert out.untouched_around()


@pytest.mark.parametrize("m,n,k", [(64, 5632, 11008), (16, 2560, 8192), (1024, 4096, 4096)])
def test_products_while_copies_hold_them_up(gpu, m, n, k):
    """Stages arrive late and unevenly beside a stream of copies, so that the waits
    inside the kernels really wait: the same bits as in a quiet run, and none runs out."""
    a, w, sa, sw, b, call = _product(gpu, m, n, k, 30, m)
    quiet = Rows(m, n, torch.bfloat16)
    base._ok(gpu, call(quiet, base._stream()))
    torch.cuda.synchronize()
    base._check_gemm(quiet.t, 30, a.t, sa, w.t, sw, b)
    src, dst = (torch.zeros(256 << 20, dtype=torch.uint8, device="cuda") for _ in range(2))
    copies, products = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [Rows(m, n, torch.bfloat16) for _ in range(10)]
    torch.cuda.synchronize()
    for out in outs:
        with torch.cuda.stream(copies):
            dst.copy_(src, non_blocking=True)
        base._ok(gpu, call(out, products.cuda_stream))
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out.t, quiet.t)
    base._ok(gpu, gpu.lib().llamini_i8_status(base._stream()))


# one CTA a tile, clusters of two, four and eight CTAs a tile, pairs with fewer slabs
# than stages, with more, and with several tiles a pair
@pytest.mark.parametrize("m,n,k", [(16, 4000, 128), (128, 20000, 700), (64, 9000, 2000), (40, 2560, 4096), (16, 896, 4096),
                                   (512, 2304, 300), (600, 4224, 2000), (2048, 8000, 640)])
@pytest.mark.parametrize("type", [0, 30])
def test_product_whose_waits_run_out(gpu, m, n, k, type):
    """A kernel that gives up: its outputs are NaN, the status says so once, nothing
    outside the outputs is written, and the next call finds everything in order."""
    a, w, sa, sw, b, call = _product(gpu, m, n, k, type, n)
    L, st = gpu.lib(), base._stream()
    base._ok(gpu, L.llamini_i8_status(st))
    out = Rows(m, n, DT[type], 1)
    try:
        base._ok(gpu, L.llamini_set_i8_wait_ns(0))
        for _ in range(3):
            base._ok(gpu, call(out, st))
        base._ok(gpu, L.llamini_set_i8_wait_ns(2_000_000_000))
        assert L.llamini_i8_status(st) == -1
        assert "wait inside a kernel ran out" in gpu.last_error()
        L.llamini_clear_error()
        base._ok(gpu, L.llamini_i8_status(st))
    finally:
        L.llamini_set_i8_wait_ns(2_000_000_000)
        L.llamini_i8_status(st)
        L.llamini_clear_error()
    assert torch.isnan(out.t).all() and out.untouched_around()
    for _ in range(3):
        base._ok(gpu, call(out, st))
    torch.cuda.synchronize()
    base._check_gemm(out.t, type, a.t, sa, w.t, sw, b)
    base._ok(gpu, L.llamini_i8_status(st))


def test_status_of_one_stream_leaves_the_other_its_report(gpu):
    """Each stream's status call reports a wait that ran out once, whichever
    stream's product it was and whoever asked before."""
    a, w, sa, sw, b, call = _product(gpu, 64, 2304, 2048, 0, 5)
    L = gpu.lib()
    streams = [torch.cuda.Stream() for _ in range(2)]
    handles = [s.cuda_stream for s in streams] + [None]
    out = Rows(64, 2304, torch.float32)
    try:
        for h in handles:
            L.llamini_i8_status(h)                 # whatever came before this test
            L.llamini_clear_error()
            base._ok(gpu, L.llamini_i8_status(h))
        torch.cuda.synchronize()
        for ran_on in handles:
            base._ok(gpu, L.llamini_set_i8_wait_ns(0))
            base._ok(gpu, call(out, ran_on))
            base._ok(gpu, L.llamini_set_i8_wait_ns(2_000_000_000))
            torch.cuda.synchronize()
            assert [L.llamini_i8_status(h) for h in handles] == [-1, -1, -1]
            L.llamini_clear_error()
            assert [L.llamini_i8_status(h) for h in handles] == [0, 0, 0]
    finally:
        L.llamini_set_i8_wait_ns(2_000_000_000)
        for h in handles:
            L.llamini_i8_status(h)
        L.llamini_clear_error()


def test_status_of_a_stream_in_capture_is_refused(gpu):
    """The refusal leaves the capture whole."""
    a, w, sa, sw, b, call = _product(gpu, 64, 300, 512, 0, 6)
    L = gpu.lib()
    want, out = Rows(64, 300, torch.float32), Rows(64, 300, torch.float32)
    base._ok(gpu, call(want, base._stream()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert L.llamini_i8_status(base._stream()) == -1
        assert "being captured" in gpu.last_error()
        L.llamini_clear_error()
        base._ok(gpu, call(out, base._stream()))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.t, want.t)
    base._ok(gpu, L.llamini_i8_status(base._stream()))


@pytest.mark.parametrize("m", [1, 5, 20, 600])
@pytest.mark.parametrize("k", [3, 7, 8, 19, 20, 35, 67, 71, 72, 131])
@pytest.mark.parametrize("shift", range(4))
def test_rows_that_end_with_the_last_word(gpu, m, k, shift):
    """Rows at every alignment whose last whole vector or word ends where the row does,
    or a byte or two before: the last row is the last of its buffer."""
    n = 650
    a, w, sa, sw, b, call = _product(gpu, m, n, k, 0, k)
    out = Rows(m, n, torch.float32)
    tight = [torch.empty(shift + x.rows * k, dtype=torch.int8, device="cuda") for x in (a, w)]
    for t, x in zip(tight, (a, w)):
        t[shift:].view(x.rows, k).copy_(x.t)
    base._ok(gpu, gpu.lib().llamini_gemm_i8_device(tight[0].data_ptr() + shift, k, sa.data_ptr(), m, tight[1].data_ptr() + shift, k,
                                                   sw.data_ptr(), n, k, b.data_ptr(), 0, out.ptr, out.ld, base._stream()))
    torch.cuda.synchronize()
    base._check_gemm(out.t, 0, a.t, sa, w.t, sw, b)


# ---------------------------------------------------------------- weights

BLOCK = {2: (32, 18), 3: (32, 20), 6: (32, 22), 8: (32, 34), 12: (256, 144), 13: (256, 176), 14: (256, 210)}
# the longest rows whose dynamic shared memory alone stays within a CTA's default 48 KB
# while static and dynamic together do not, and rows on either side
DEFAULT_SMEM, SLACK, STATIC = 48 * 1024, 64, 256


def _edge_lengths(t):
    be, bb = BLOCK[t]
    last = (DEFAULT_SMEM - SLACK) // bb            # blocks of a row
    first = (DEFAULT_SMEM - SLACK - STATIC) // bb + 1
    return [n * be for n in sorted({first - 1, first, last, last + 1})]


def _check_weights(gpu, orc, synth, t, rows, cols, pad=0, shift=0):
    raw = synth.random_blocks(np.random.default_rng(t + cols), t, rows * cols)
    w = torch.from_numpy(orc.dequant(t, raw, rows * cols).reshape(rows, cols)).cuda()
    want_q, want_s = base._want_weights(w)
    d = torch.empty(raw.size + shift, dtype=torch.uint8, device="cuda")
    d[shift:].copy_(torch.from_numpy(raw))
    q = Rows(rows, cols, torch.int8, pad)
    scale = torch.full((rows + 2,), 7.0, device="cuda")
    base._ok(gpu, base._weights_call(gpu, t, d.data_ptr() + shift, rows, cols, q, scale))
    torch.cuda.synchronize()
    assert torch.equal(scale[:rows], want_s) and torch.all(scale[rows:] == 7), (t, cols)
    assert torch.equal(q.t, want_q) and q.untouched_around(), (t, cols)


def weights_at_the_edge_of_shared_memory(gpu, orc, synth):
    for t in BLOCK:
        for cols in _edge_lengths(t):              # rising: no call finds a limit raised by a longer one
            _check_weights(gpu, orc, synth, t, 2, cols)


def test_weights_at_the_edge_of_shared_memory(gpu, orc):
    """Rows that need a little more shared memory than a launch gets unasked, in a
    process whose first calls they are."""
    code = ("import sys; sys.path[:0] = %r\n"
            "import conftest, oracle, tiny, test_gpu_i8_edges as t\n"
            "t.weights_at_the_edge_of_shared_memory(conftest._load_pkg(), oracle, tiny.synthetic())\n"
            % [os.path.dirname(__file__), conftest.GOLDEN, os.path.join(conftest.ROOT, "oracle")])
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("t", sorted(BLOCK))
@pytest.mark.parametrize("cols,pad,shift", [(98304, 0, 0), (130816, 3, 2), (106752, 16, 14)])
def test_weights_in_several_segments(gpu, orc, synth, t, cols, pad, shift):
    _check_weights(gpu, orc, synth, t, 3, cols, pad, shift)


# ---------------------------------------------------------------- gated activation

# gates in [low, high) times an `up` of this size: products of f32's range from gates far
# below zero, down to where 1 + exp(-gate) leaves that range
FAR = [(0, -12.0, -9.0, 1.0), (0, -88.5, -80.0, 1.0), (0, -88.5, -87.0, 1e30), (0, -88.5, -87.5, 1e37), (0, -70.0, -60.0, 1e-3),
       (1, -8.0, -7.0, 1.0), (1, -10.2, -9.9, 1e36), (1, -9.5, -6.0, 1e3)]


def _far_call(gpu, type, act, gate, up, rows, cols, pad):
    gr, ur = Rows(rows, cols, DT[type], pad, fill=gate), Rows(rows, cols, DT[type], pad, fill=up)
    q, scale = Rows(rows, cols, torch.int8, pad if pad else (-cols) % 16), torch.empty(rows, device="cuda")
    base._ok(gpu, base._glu(gpu, type, gr, ur, act, rows, cols, q, scale))
    torch.cuda.synchronize()
    return gr.t, ur.t, q, scale


@pytest.mark.parametrize("type", [0, 30])
@pytest.mark.parametrize("act,low,high,size", FAR)
@pytest.mark.parametrize("rows,cols,pad", [(4, 64, 0), (1100, 64, 0), (1100, 100, 1), (3, 4864, 0), (3, 777, 1), (2, 40000, 1)])
def test_glu_of_gates_far_below_zero(gpu, type, act, low, high, size, rows, cols, pad):
    g = base._gen(cols + rows)
    gate = torch.rand(rows, cols, generator=g, device="cuda") * (high - low) + low
    up = base._rand(g, rows, cols).sign() * (0.5 + torch.rand(rows, cols, generator=g, device="cuda")) * size
    x, u, q, scale = _far_call(gpu, type, act, gate, up, rows, cols, pad)
    x = x.double()
    z = x if act == 0 else 2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)
    y = x * torch.sigmoid(z) * u.double()
    # zero where 1 + exp(-z) is past f32's largest number, z = -88.72; within z's own error
    # of that (six roundings of 89: 3.2e-5) either
    limit = -float(np.log(np.finfo(np.float32).max))
    y = torch.where((z < limit) & ((z - limit).abs() > 1e-4) | ((z - limit).abs() <= 1e-4) & (q.t == 0), 0.0, y)
    # the argument: |z| 2^-23 (SiLU), |z| 2^-22 (GELU); the squares of two approximations
    # of 2^-22; eight roundings of products and sums
    r = ((2 if act == 0 else 4) * float(z.abs().max()) + 4 * 4 + 8) * F24
    base._check_int8(q.t, scale, y, r)
    assert q.untouched_around()


@pytest.mark.parametrize("type", [0, 30])
@pytest.mark.parametrize("cols,pad", [(64, 0), (777, 1), (4864, 0), (40000, 1)])
def test_glu_of_gates_whose_sigmoid_is_zero(gpu, type, cols, pad):
    """Below -89 SiLU is zero in f32, as in ffn_glu: such gates count for nothing
    beside others, and a row of them is a row of zeros."""
    g = base._gen(cols)
    gate = torch.rand(4, cols, generator=g, device="cuda") * -100 - 90
    gate[2, cols // 2], gate[3, 0] = -20.0, 1.0
    up = base._rand(g, 4, cols) * 1e6
    x, u, q, scale = _far_call(gpu, type, 0, gate, up, 4, cols, pad)
    host = [t.float().contiguous().cpu().numpy() for t in (x, u)]
    for i in range(4):
        out = np.empty(cols, np.float32)
        gpu.lib().ffn_glu(gpu.ptr(out), gpu.ptr(host[0][i]), gpu.ptr(host[1][i]), cols, 0)
        assert np.count_nonzero(out) == (0 if i < 2 else 1)
    assert torch.all(scale[:2] == 0) and torch.all(q.t[:2] == 0)
    for i, at in ((2, cols // 2), (3, 0)):
        assert q.t[i].count_nonzero() == 1 and abs(int(q.t[i, at])) == 127
        want = x[i, at].double() * torch.sigmoid(x[i, at].double()) * u[i, at].double()
        assert abs(float(scale[i].double() * 127 / want.abs()) - 1) < 80 * F24      # |z| of 20


# ---------------------------------------------------------------- norm

# sizes of a row's values and eps: sums of squares below, at and past f32's largest number,
# and means past the least that the norm takes
SIZES = [(1e20, 1e-5), (3e37, 1e-5), (1e18, 1e-5), (1e15, 1e-6), (1e-16, 0.0), (1e-21, 0.0), (1e-37, 0.0), (1e-18, 1e-35), (1e-30, 1e-30),
         (1.0, 0.0)]


def _range_of(h, eps):
    """Rows whose mean of squares f32 holds, and those that it does not (the sums of
    no row here lie so close to a limit that the order of its additions decides)."""
    ss = h.square().sum(dim=1)
    mean = ss / h.shape[1] + eps
    top, least = float(np.finfo(np.float32).max), 2.0 ** -120
    assert torch.all((ss / top - 1).abs() > 1e-3) and torch.all((mean / least - 1).abs() > 1e-3)
    fine = (ss < top) & (mean > least)
    return fine, ~fine


@pytest.mark.parametrize("type", [0, 30])
@pytest.mark.parametrize("size,eps", SIZES)
@pytest.mark.parametrize("rows,cols,pad,resid", [(3, 64, 0, False), (1100, 64, 0, True), (1100, 100, 1, True), (3, 4096, 0, True), (5, 777, 1, False),
                                                 (2, 11008, 0, True), (3, 12000, 1, True), (1100, 8192, 0, True), (2, 40000, 0, False)])
def test_norm_of_rows_of_any_size(gpu, type, size, eps, rows, cols, pad, resid):
    """Large and tiny rows, some with a part of ordinary size, beside an ordinary
    one: right, or where a mean leaves f32's range a scale of NaN."""
    g = base._gen(cols + rows)
    x0 = base._rand(g, rows, cols).clamp_(-5, 5) * size
    x0[0] = base._rand(g, cols)                    # an ordinary row
    x0[1, 1:cols // 2] = 0.0
    if size > 1:
        x0[-1, cols // 2:] = 1.0
    x = Rows(rows, cols, DT[type], pad, fill=x0)
    r = Rows(rows, cols, DT[type], pad, fill=base._rand(g, rows, cols) * size / 4) if resid else None
    out = Rows(rows, cols, DT[type], pad) if resid else None
    w = 1 + base._rand(g, cols, scale=0.05)
    q, scale = Rows(rows, cols, torch.int8, pad if pad else (-cols) % 16), torch.empty(rows, device="cuda")
    base._ok(gpu, base._norm(gpu, type, x, r, out, w, eps, rows, cols, q, scale))
    torch.cuda.synchronize()
    h = x.t.double() + (r.t.double() if resid else 0)
    eps = float(np.float32(eps))
    fine, lost = _range_of(h, eps)
    assert torch.isnan(scale[lost]).all() and torch.all(q.t[lost] == 0)
    y = h / (h.square().mean(dim=1, keepdim=True) + eps).sqrt() * w.double()
    # a square is off by up to 2^-150 beside means of 2^-120 and more
    base._check_int8(q.t[fine], scale[fine], y[fine], base._norm_r(cols) + 2.0 ** -30)
    assert q.untouched_around()
    if resid:
        half = torch.finfo(DT[type]).eps / 2 + F24
        assert torch.all((out.t.double() - h).abs() <= h.abs() * half + 2.0 ** -149)


@pytest.mark.parametrize("type", [0, 30])
@pytest.mark.parametrize("rows,cols", [(40, 64), (2000, 100), (300, 2048), (1100, 4096), (700, 20000)])
def test_norm_of_large_rows_among_others(gpu, type, rows, cols):
    """Every third row is too large: CTAs and warps that walk over rows go from one
    kind to the other, and the ordinary rows keep the bits that they have alone."""
    g = base._gen(rows)
    x0 = base._rand(g, rows, cols)
    plain = Rows(rows, cols, DT[type], fill=x0)
    x0[::3] *= 1e25
    x0[::6, : cols // 3] = 2.0
    mixed = Rows(rows, cols, DT[type], fill=x0)
    w = 1 + base._rand(g, cols, scale=0.05)
    got = []
    for x in (plain, mixed):
        q, scale = Rows(rows, cols, torch.int8, (-cols) % 16), torch.empty(rows, device="cuda")
        base._ok(gpu, base._norm(gpu, type, x, None, None, w, 1e-5, rows, cols, q, scale))
        got.append((q.t, scale))
    others = torch.arange(rows, device="cuda") % 3 != 0
    assert torch.equal(got[0][0][others], got[1][0][others]) and torch.equal(got[0][1][others], got[1][1][others])
    assert torch.isnan(got[1][1][~others]).all() and torch.all(got[1][0][~others] == 0)
    h = plain.t.double()
    base._check_int8(*got[0], h / (h.square().mean(1, True) + float(np.float32(1e-5))).sqrt() * w.double(), base._norm_r(cols))


# ---------------------------------------------------------------- long walks
#
# More rows than CTAs run at once, so that each CTA goes through several: buffers and
# halves of shared memory that alternate, the next row's loads under way.

@pytest.mark.parametrize("t,rows,cols", [(2, 4096, 2048), (3, 9000, 256), (6, 4096, 2048), (8, 4096, 2048), (8, 20000, 96), (8, 700, 20480),
                                         (12, 9000, 768), (12, 700, 20480), (13, 4096, 2048), (14, 4096, 2048), (14, 2000, 5632)])
def test_weights_of_many_rows(gpu, orc, synth, t, rows, cols):
    _check_weights(gpu, orc, synth, t, rows, cols)


# vectors a thread: 1, 2, 3, 4, 6, 8 of eight elements and of four; then one element at a time
WALKS = [(1200, 2048), (1000, 4096), (1100, 4096), (700, 11008), (700, 14336), (500, 20480), (400, 30000), (1200, 5632), (1200, 7168),
         (3000, 500), (700, 3001), (500, 12001)]


@pytest.mark.parametrize("type", [0, 1, 30])
@pytest.mark.parametrize("rows,cols", WALKS)
@pytest.mark.parametrize("resid", [False, True])
def test_norm_of_many_rows(gpu, type, rows, cols, resid):
    g = base._gen(rows + cols)
    pad = (-cols) % 8 if cols % 8 == 4 else 0
    x = Rows(rows, cols, DT[type], pad, fill=base._rand(g, rows, cols))
    r0 = base._rand(g, rows, cols, scale=3)
    r = Rows(rows, cols, DT[type], pad, fill=r0) if resid else None
    w = 1 + base._rand(g, cols, scale=0.05)
    q, scale = Rows(rows, cols, torch.int8, pad), torch.empty(rows, device="cuda")
    h = x.t.double() + (r.t.double() if resid else 0)
    base._ok(gpu, base._norm(gpu, type, x, r, r, w, 1e-5, rows, cols, q, scale))      # the sum over the residual
    torch.cuda.synchronize()
    y = h / (h.square().mean(dim=1, keepdim=True) + float(np.float32(1e-5))).sqrt() * w.double()
    base._check_int8(q.t, scale, y, base._norm_r(cols))
    assert q.untouched_around()
    if resid:
        half = torch.finfo(DT[type]).eps / 2 + F24
        assert torch.all((r.t.double() - h).abs() <= h.abs() * half + 2.0 ** -25) and r.untouched_around()


@pytest.mark.parametrize("type", [0, 1, 30])
@pytest.mark.parametrize("rows,cols", WALKS + [(1500, 9000), (2000, 11008)])
@pytest.mark.parametrize("act,with_up", [(0, True), (2, False)])
def test_glu_of_many_rows(gpu, type, rows, cols, act, with_up):
    g = base._gen(rows + cols)
    pad = (-cols) % 8 if cols % 8 == 4 else 0
    gate = Rows(rows, cols, DT[type], pad, fill=base._rand(g, rows, cols, scale=3))
    up = Rows(rows, cols, DT[type], pad, fill=base._rand(g, rows, cols)) if with_up else None
    q, scale = Rows(rows, cols, torch.int8, pad), torch.empty(rows, device="cuda")
    base._ok(gpu, base._glu(gpu, type, gate, up, act, rows, cols, q, scale))
    torch.cuda.synchronize()
    y = base._act64(gate.t.double(), act) * (up.t.double() if with_up else 1.0)
    # SiLU of gates down to 3 x 6: argument 18 x 2^-23, approximations 2 x 2 x 2^-22, roundings
    base._check_int8(q.t, scale, y, (36 + 16 + 8) * F24 if act == 0 else 4 * F24)
    assert q.untouched_around()


# ---------------------------------------------------------------- first calls

def first_calls_in_a_capture(gpu, synth):
    """Each operator and product kernel for the first time in its process, inside a
    capture; the replay, and the same calls made directly."""
    L = gpu.lib()
    e = dict(device="cuda")
    n, k = 1024, 768
    raws = [torch.from_numpy(synth.random_blocks(np.random.default_rng(t), t, n * k).copy()).cuda() for t in (8, 12)]
    wide = torch.from_numpy(synth.random_blocks(np.random.default_rng(9), 8, 2 * 98304).copy()).cuda()
    x = base._rand(base._gen(1), 900, k).bfloat16()
    w = torch.ones(k, **e)
    other = torch.cuda.Stream()

    def run(st):
        outs = []
        for raw, t in zip(raws, (8, 12)):
            q, s = torch.zeros(n, k, dtype=torch.int8, **e), torch.zeros(n, **e)
            base._ok(gpu, L.llamini_weights_i8_device(t, raw.data_ptr(), n, k, q.data_ptr(), k, s.data_ptr(), st))
            outs += [q, s]
        q, s = torch.zeros(2, 98304, dtype=torch.int8, **e), torch.zeros(2, **e)
        base._ok(gpu, L.llamini_weights_i8_device(8, wide.data_ptr(), 2, 98304, q.data_ptr(), 98304, s.data_ptr(), st))
        outs += [q, s]
        for m in (1, 40, 900):
            a, sa = torch.zeros(m, k, dtype=torch.int8, **e), torch.zeros(m, **e)
            h, sh = torch.zeros(m, n // 2, dtype=torch.int8, **e), torch.zeros(m, **e)
            y = torch.zeros(m, n, dtype=torch.bfloat16, **e)
            base._ok(gpu, L.llamini_rms_norm_i8_device(30, x.data_ptr(), k, None, 0, None, 0, w.data_ptr(), 1e-5, m, k, a.data_ptr(), k,
                                                       sa.data_ptr(), st))
            base._ok(gpu, L.llamini_gemm_i8_device(a.data_ptr(), k, sa.data_ptr(), m, outs[0].data_ptr(), k, outs[1].data_ptr(), n, k, None,
                                                   30, y.data_ptr(), n, st))
            base._ok(gpu, L.llamini_glu_i8_device(30, y.data_ptr(), n, y.data_ptr() + n, n, 0, m, n // 2, h.data_ptr(), n // 2,
                                                  sh.data_ptr(), st))
            outs += [a, sa, y, h, sh]
        return outs
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(base._stream())
        base._ok(gpu, L.llamini_i8_status(other.cuda_stream))      # of a stream that is not captured
    graph.replay()
    torch.cuda.synchronize()
    direct = run(base._stream())
    torch.cuda.synchronize()
    assert all(torch.equal(c, d) for c, d in zip(captured, direct))
    assert all(c.float().abs().sum() > 0 for c in captured)


def test_first_calls_in_a_capture(gpu):
    code = ("import sys; sys.path[:0] = %r\n"
            "import conftest, tiny, test_gpu_i8_edges as t\n"
            "t.first_calls_in_a_capture(conftest._load_pkg(), tiny.synthetic())\n"
            % [os.path.dirname(__file__), conftest.GOLDEN, os.path.join(conftest.ROOT, "oracle")])
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


# ---------------------------------------------------------------- refusals

def test_refusals_name_the_array(gpu):
    """One host array among device arrays: the message says which."""
    L, d = gpu.lib(), torch.zeros(8192, device="cuda").data_ptr()
    h = np.zeros(8192, np.float32)

    def each(call, names):
        for at, name in enumerate(names):
            args = [d] * len(names)
            args[at] = h.ctypes.data
            L.llamini_clear_error()
            assert call(*args) == -1
            assert ": %s is not memory of the current device" % name in gpu.last_error()
        L.llamini_clear_error()
    each(lambda b, q, s: L.llamini_weights_i8_device(8, b, 4, 64, q, 64, s, None), ["blocks", "q", "scale"])
    each(lambda x, r, o, w, q, s: L.llamini_rms_norm_i8_device(0, x, 64, r, 64, o, 64, w, 1e-5, 4, 64, q, 64, s, None),
         ["x", "resid", "sum", "w", "q", "scale"])
    each(lambda g, u, q, s: L.llamini_glu_i8_device(0, g, 64, u, 64, 0, 4, 64, q, 64, s, None), ["gate", "up", "q", "scale"])
    each(lambda a, sa, w, sw, b, o: L.llamini_gemm_i8_device(a, 64, sa, 4, w, 64, sw, 8, 64, b, 0, o, 8, None),
         ["a", "a_scale", "w", "w_scale", "bias", "out"])
