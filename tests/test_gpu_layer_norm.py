"""Layer normalisation and its gradient through the C ABI, against the formulas in fp64.

Tolerances count roundings.  With u = 2^-24 (2^-53 for f64 rows) and sums whose longest chain of additions has k steps, a sum
of terms t is off by at most k u sum |t|; a deviation x - mean by e_d = k u (|x| + mean |x|), and the statistics r, mean(a),
mean(a h) follow.  The store adds half a step of the stored type."""
import numpy as np
import pytest
import torch

from dali_b200.capi import BF16, DaliB200Error, F32, F64

pytestmark = pytest.mark.gpu

TORCH = {F32: torch.float32, F64: torch.float64, BF16: torch.bfloat16}
U = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -24}                 # of the arithmetic
HALF_STEP = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -8}          # of the stored type
EPS = 1e-5


def chain(n):
    """More additions than any thread makes one after another in a sum of n terms, and the folds behind it."""
    return 64 + n // 128


def matrix(rng, rows, cols, dtype, stride=None, offset=0, spread=2.0):
    """A [rows, cols] matrix inside a larger buffer: (buffer, view)."""
    stride = cols if stride is None else stride
    buf = torch.full((offset + rows * stride + 7,), 77.0, device="cuda", dtype=TORCH[dtype])
    view = torch.as_strided(buf, (rows, cols), (stride, 1), offset)
    view.copy_(torch.from_numpy(rng.standard_normal((rows, cols)) * spread + rng.standard_normal((rows, 1))).cuda())
    return buf, view


class Formula:
    """Value and error bound of layer_norm and its gradient in fp64."""

    def __init__(self, x, gamma, beta, dtype, eps=EPS):
        x = x.double()
        n = x.shape[1]
        self.u, self.n, self.k = U[dtype], n, chain(n)
        self.gamma = torch.ones(n, device="cuda", dtype=torch.float64) if gamma is None else gamma.double()
        self.beta = torch.zeros(n, device="cuda", dtype=torch.float64) if beta is None else beta.double()
        mean = x.mean(1, keepdim=True)
        d = x - mean
        self.r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
        self.h = d * self.r
        e_d = self.k * self.u * (x.abs() + x.abs().mean(1, keepdim=True))
        # r: half the relative error of var + eps, which is that of the squares (2 e_d / |d|, averaged) and of their sum
        e_var = (2 * d.abs() * e_d + e_d * e_d).mean(1, keepdim=True) + self.k * self.u * (d * d).mean(1, keepdim=True)
        e_r = self.r * (0.5 * e_var * self.r * self.r + 4 * self.u)
        self.e_r = e_r
        self.e_h = self.r * e_d + d.abs() * e_r + 2 * self.u * self.h.abs()

    def y(self):
        y = self.h * self.gamma + self.beta
        return y, self.e_h * self.gamma.abs() + 2 * self.u * ((self.h * self.gamma).abs() + self.beta.abs())

    def grads(self, dy, rows):
        dy, h, r, ku = dy.double(), self.h, self.r, self.k * self.u
        a = dy * self.gamma
        c1, c2 = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
        e_c1 = (ku + 2 * self.u) * a.abs().mean(1, keepdim=True)
        e_c2 = (a.abs() * self.e_h).mean(1, keepdim=True) + (ku + 4 * self.u) * (a * h).abs().mean(1, keepdim=True)
        inner = a - c1 - h * c2
        e_inner = 2 * self.u * a.abs() + e_c1 + self.e_h * c2.abs() + h.abs() * e_c2 + 4 * self.u * (a.abs() + c1.abs() + (h * c2).abs())
        dx, e_dx = r * inner, r * e_inner + self.e_r * inner.abs()
        kr = (64 + rows) * self.u                          # every row added after the other
        dg, e_dg = (dy * h).sum(0), (dy.abs() * self.e_h).sum(0) + kr * (dy * h).abs().sum(0)
        db, e_db = dy.sum(0), kr * dy.abs().sum(0)
        return (dx, e_dx), (dg, e_dg), (db, e_db)


def agree(got, want, bound, stored):
    want_stored_error = HALF_STEP[stored] * want.abs() * (1 + 2.0 ** -7)
    off = (got.double() - want).abs() - bound - want_stored_error
    worst = off.max().item() if off.numel() else 0.0
    assert not torch.isnan(off).any() and worst <= 1e-300 + 0.0, "off by %g more than the bound" % worst


TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F64, F64)]
SHAPES = [(1, 1), (1, 1024), (3, 31), (2, 33), (37, 257), (300, 64), (5, 1000), (7, 1537), (9, 2056), (2, 4096), (3, 8192), (2, 20001),
          (2, 32768), (1, 32776), (2, 70000)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(lib, shape, types):
    (rows, cols), (dt, wt) = shape, types
    rng = np.random.default_rng(rows * 1000003 + cols)
    _, x = matrix(rng, rows, cols, dt)
    gamma = torch.from_numpy(1 + 0.3 * rng.standard_normal(cols)).cuda().to(TORCH[wt])
    beta = torch.from_numpy(0.3 * rng.standard_normal(cols)).cuda().to(TORCH[wt])
    for g, b in ((gamma, beta), (gamma, None), (None, beta), (None, None)):
        out = torch.empty(rows, cols, device="cuda", dtype=TORCH[dt])
        lib.layer_norm(dt, wt, rows, cols, x, g, b, out, eps=EPS)
        agree(out, *Formula(x, g, b, dt).y(), dt)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(lib, shape, types):
    (rows, cols), (dt, wt) = shape, types
    rng = np.random.default_rng(rows * 1000033 + cols)
    _, x = matrix(rng, rows, cols, dt)
    _, dy = matrix(rng, rows, cols, dt, spread=1.0)
    gamma = torch.from_numpy(1 + 0.3 * rng.standard_normal(cols)).cuda().to(TORCH[wt])
    for g in (gamma, None):
        dx = torch.empty(rows, cols, device="cuda", dtype=TORCH[dt])
        dg, db = (torch.empty(cols, device="cuda", dtype=TORCH[wt]) for _ in range(2))
        lib.layer_norm_backward(dt, wt, rows, cols, dy, x, g, dx, dg, db, eps=EPS)
        want = Formula(x, g, None, dt).grads(dy, rows)
        agree(dx, *want[0], dt)
        agree(dg, *want[1], wt)
        agree(db, *want[2], wt)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", [(3, 9001), (2, 12000), (3, 16384), (2, 16383), (1200, 100), (2500, 8), (900, 520), (450, 2047), (301, 4100)])
def test_long_rows_and_many_rows(lib, shape, types):
    """Rows that 8 or 16 warps share, and more rows than a grid takes at once, on the 16-byte grid and off it."""
    test_forward(lib, shape, types)
    test_backward(lib, shape, types)


@pytest.mark.parametrize("types", TYPES[:3])
@pytest.mark.parametrize("cols", [300, 301, 640, 703, 760, 761, 1152, 1201, 1275, 1500, 1505, 2400, 2497, 2990, 5000, 5003, 6000, 6007])
def test_rows_by_any_number_of_warps(lib, cols, types):
    """Widths that a number of warps which is no power of two covers, on the grid and off it; rows that end inside a CTA's groups,
    and matrices that lie unlike one another."""
    dt, wt = types
    rng = np.random.default_rng(cols)
    for rows, shift in ((1, 0), (13, 0), (13, 1), (1501, 0)):
        _, x = matrix(rng, rows, cols, dt)
        _, dy = matrix(rng, rows, cols, dt, offset=shift, spread=1.0)
        gamma = torch.from_numpy(1 + 0.3 * rng.standard_normal(cols)).cuda().to(TORCH[wt])
        beta = torch.from_numpy(0.3 * rng.standard_normal(cols)).cuda().to(TORCH[wt])
        bo, out = matrix(rng, rows, cols, dt, offset=shift)
        bo.fill_(77.0)
        lib.layer_norm(dt, wt, rows, cols, x, gamma, beta, out, eps=EPS)
        agree(out, *Formula(x, gamma, beta, dt).y(), dt)
        bx, dx = matrix(rng, rows, cols, dt)
        bx.fill_(77.0)
        dg, db = (torch.empty(cols, device="cuda", dtype=TORCH[wt]) for _ in range(2))
        lib.layer_norm_backward(dt, wt, rows, cols, dy, x, gamma, dx, dg, db, eps=EPS)
        want = Formula(x, gamma, None, dt).grads(dy, rows)
        agree(dx, *want[0], dt)
        agree(dg, *want[1], wt)
        agree(db, *want[2], wt)
        assert (bo[:shift] == 77.0).all() and (bo[shift + rows * cols:] == 77.0).all() and (bx[rows * cols:] == 77.0).all()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows,cols", [(6, 1000), (150, 1024), (5, 513), (700, 96), (3, 33000)])
def test_strides_offsets_and_writing_over_an_input(lib, rows, cols, types):
    dt, wt = types
    rng = np.random.default_rng(cols)
    for stride, offset in ((cols + 8, 8), (cols + 1, 1), (cols + 3, 0)):
        bx, x = matrix(rng, rows, cols, dt, stride, offset)
        bdy, dy = matrix(rng, rows, cols, dt, stride + 2, offset)
        gamma = torch.from_numpy(1 + 0.3 * rng.standard_normal(cols)).cuda().to(TORCH[wt])
        f = Formula(x, gamma, None, dt)
        bo, out = matrix(rng, rows, cols, dt, stride + 4, offset + 1)
        lib.layer_norm(dt, wt, rows, cols, x, gamma, None, out, eps=EPS, x_row_stride=stride, out_row_stride=stride + 4)
        agree(out, *f.y(), dt)
        out.fill_(77.0)
        assert (bo == 77.0).all()                                       # nothing beside the rows
        want = f.grads(dy, rows)
        dg, db = (torch.empty(cols, device="cuda", dtype=TORCH[wt]) for _ in range(2))
        lib.layer_norm_backward(dt, wt, rows, cols, dy, x, gamma, out, dg, db, eps=EPS, dy_row_stride=stride + 2, x_row_stride=stride,
                                dx_row_stride=stride + 4)
        for got, w, t in zip((out, dg, db), want, (dt, wt, wt)):
            agree(got, *w, t)
        ref = out.clone()
        out.fill_(77.0)
        assert (bo == 77.0).all()
        # over dy, then (dy lost) over x: the same bits
        dy2, x2 = bdy.clone(), bx.clone()
        vdy, vx = torch.as_strided(dy2, (rows, cols), (stride + 2, 1), offset), torch.as_strided(x2, (rows, cols), (stride, 1), offset)
        g2, b2 = torch.empty_like(dg), torch.empty_like(db)
        lib.layer_norm_backward(dt, wt, rows, cols, vdy, x, gamma, vdy, g2, b2, eps=EPS, dy_row_stride=stride + 2, x_row_stride=stride,
                                dx_row_stride=stride + 2)
        agree(vdy, *want[0], dt)
        agree(g2, *want[1], wt)
        lib.layer_norm_backward(dt, wt, rows, cols, dy, vx, gamma, vx, g2, b2, eps=EPS, dy_row_stride=stride + 2, x_row_stride=stride,
                                dx_row_stride=stride)
        agree(vx, *want[0], dt)
        agree(b2, *want[2], wt)
        vx.fill_(77.0)
        assert (x2 == 77.0).all()
        lib.layer_norm(dt, wt, rows, cols, x, gamma, None, x, eps=EPS, x_row_stride=stride, out_row_stride=stride)
        agree(x, *f.y(), dt)
        assert ref.shape == (rows, cols)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("cols", [100, 1024, 5000, 40000])
def test_each_gradient_alone(lib, cols, types):
    dt, wt = types
    rng = np.random.default_rng(cols)
    rows = 20
    _, x = matrix(rng, rows, cols, dt)
    _, dy = matrix(rng, rows, cols, dt)
    gamma = torch.from_numpy(1 + 0.3 * rng.standard_normal(cols)).cuda().to(TORCH[wt])
    want = Formula(x, gamma, None, dt).grads(dy, rows)
    for which in range(1, 7):
        dx = torch.empty(rows, cols, device="cuda", dtype=TORCH[dt]) if which & 1 else None
        dg = torch.empty(cols, device="cuda", dtype=TORCH[wt]) if which & 2 else None
        db = torch.empty(cols, device="cuda", dtype=TORCH[wt]) if which & 4 else None
        lib.layer_norm_backward(dt, wt, rows, cols, dy, x, gamma, dx, dg, db, eps=EPS)
        for got, w, t in zip((dx, dg, db), want, (dt, wt, wt)):
            if got is not None:
                agree(got, *w, t)


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("cols", [40, 1024, 1537, 40000])
def test_rows_that_do_not_vary_and_rows_that_are_not_numbers(lib, cols, dt):
    rng = np.random.default_rng(cols)
    rows = 8
    _, x = matrix(rng, rows, cols, dt)
    x[1] = 3.0                      # no variance: h = 0
    x[2] = 0.0
    x[4, cols // 2] = float("nan")
    x[5, cols - 1] = float("inf")
    x[6] = 1e4 + 8 * torch.randn(cols, device="cuda", dtype=torch.float64).to(TORCH[dt])      # far from zero: deviations have to be taken from the mean
    beta = torch.from_numpy(rng.standard_normal(cols)).cuda().to(TORCH[dt])
    out = torch.empty_like(x)
    lib.layer_norm(dt, dt, rows, cols, x, None, beta, out, eps=EPS)
    assert torch.equal(out[1], beta) and torch.equal(out[2], beta)
    assert torch.isnan(out[4]).all()
    assert torch.isnan(out[5]).all()
    sound = [0, 3, 6, 7]
    agree(out[sound], *Formula(x[sound], None, beta, dt).y(), dt)
    # a NaN in one row stays out of the other rows' dx
    dy = torch.randn(rows, cols, device="cuda", dtype=torch.float64).to(TORCH[dt])
    dx = torch.empty_like(x)
    lib.layer_norm_backward(dt, dt, rows, cols, dy, x, None, dx, None, None, eps=EPS)
    agree(dx[sound], *Formula(x[sound], None, None, dt).grads(dy[sound], rows)[0], dt)
    assert torch.isnan(dx[4]).all()


def test_gradient_against_differences(lib):
    """d/dt of sum(dy * layer_norm(x + t v)) by central differences in fp64: their error is t^2 f'''/6 + 2^-53 |f| / t, both
    below 1e-8 of the scale for t = 1e-5."""
    rng = np.random.default_rng(5)
    rows, cols = 6, 77
    x, dy, v = (torch.from_numpy(rng.standard_normal((rows, cols))).cuda() for _ in range(3))
    gamma, beta, vg, vb = (torch.from_numpy(rng.standard_normal(cols)).cuda() for _ in range(4))

    def f(x, gamma, beta):
        out = torch.empty_like(x)
        lib.layer_norm(F64, F64, rows, cols, x, gamma, beta, out, eps=EPS)
        return (out * dy).sum().item()
    dx, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
    lib.layer_norm_backward(F64, F64, rows, cols, dy, x, gamma, dx, dg, db, eps=EPS)
    t = 1e-5
    for got, plus, minus in (((dx * v).sum(), f(x + t * v, gamma, beta), f(x - t * v, gamma, beta)),
                             ((dg * vg).sum(), f(x, gamma + t * vg, beta), f(x, gamma - t * vg, beta)),
                             ((db * vb).sum(), f(x, gamma, beta + t * vb), f(x, gamma, beta - t * vb))):
        assert abs(got.item() - (plus - minus) / (2 * t)) < 1e-6 * (1 + abs(got.item()))


@pytest.mark.parametrize("rows,cols,dt", [(1000, 1024, F32), (3000, 1000, BF16), (77, 5003, F32), (4000, 130, BF16)])
def test_the_same_call_gives_the_same_bits(lib, rows, cols, dt):
    rng = np.random.default_rng(1)
    _, x = matrix(rng, rows, cols, dt)
    _, dy = matrix(rng, rows, cols, dt)
    seen = []
    for _ in range(3):
        dx, dg, db = torch.empty_like(x), torch.empty(cols, device="cuda", dtype=TORCH[dt]), torch.empty(cols, device="cuda", dtype=TORCH[dt])
        lib.layer_norm_backward(dt, dt, rows, cols, dy, x, None, dx, dg, db)
        seen.append((dx, dg, db))
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


def test_no_rows_and_no_columns(lib):
    x = torch.empty(0, device="cuda")
    g = torch.ones(8, device="cuda")
    dg, db = torch.full((8,), 5.0, device="cuda"), torch.full((8,), 5.0, device="cuda")
    lib.layer_norm(F32, F32, 0, 8, x, g, g, x)
    lib.layer_norm_backward(F32, F32, 0, 8, x, x, g, x, dg, db)
    assert (dg == 0).all() and (db == 0).all()
    lib.layer_norm(F32, F32, 4, 0, x, None, None, x)
    lib.layer_norm_backward(F32, F32, 4, 0, x, x, None, x, None, None)


def test_streams_and_graphs(lib):
    """On another stream than the default one; captured with a workspace of its own and replayed over new values, two graphs
    with a workspace each; refused without one."""
    rng = np.random.default_rng(3)
    rows, cols = 300, 1024
    _, x = matrix(rng, rows, cols, F32)
    _, dy = matrix(rng, rows, cols, F32)
    gamma = torch.ones(cols, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    work = [torch.empty(lib.layer_norm_backward_workspace(F32, rows, cols), device="cuda", dtype=torch.uint8) for _ in range(2)]
    outs = [(torch.empty_like(x), torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)) for _ in range(2)]

    def both(i, stream, workspace):
        y, dx, dg, db = outs[i]
        lib.layer_norm(F32, F32, rows, cols, x, gamma, None, y, eps=EPS, stream=stream)
        lib.layer_norm_backward(F32, F32, rows, cols, dy, x, gamma, dx, dg, db, eps=EPS, workspace=workspace, stream=stream)

    def right(i):
        f = Formula(x, gamma, None, F32)
        y, dx, dg, db = outs[i]
        agree(y, *f.y(), F32)
        for got, w in zip((dx, dg, db), f.grads(dy, rows)):
            agree(got, *w, F32)
    with torch.cuda.stream(s):
        both(0, s.cuda_stream, None)
    s.synchronize()
    right(0)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            both(i, torch.cuda.current_stream().cuda_stream, work[i])
        graphs.append(g)
    x.mul_(-1.5)
    for _ in range(3):
        for o in outs:
            for t in o:
                t.fill_(0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        right(0)
        right(1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(DaliB200Error, match="workspace"):
            both(0, torch.cuda.current_stream().cuda_stream, None)
    del graphs, g


def test_matrices_whose_rows_do_not_lie_alike(lib):
    """x, dy and dx each start elsewhere in a 16-byte packet, and their strides differ by odd numbers."""
    rng = np.random.default_rng(12)
    for dt in (F32, BF16, F64):
        for rows, cols in ((40, 100), (9, 2050), (3, 9000)):
            _, x = matrix(rng, rows, cols, dt, cols + 1, 1)
            _, dy = matrix(rng, rows, cols, dt, cols + 4, 2)
            _, dx = matrix(rng, rows, cols, dt, cols + 7, 3)
            dg, db = (torch.empty(cols, device="cuda", dtype=TORCH[dt]) for _ in range(2))
            f = Formula(x, None, None, dt)
            want = f.grads(dy, rows)
            lib.layer_norm_backward(dt, dt, rows, cols, dy, x, None, dx, dg, db, eps=EPS, dy_row_stride=cols + 4, x_row_stride=cols + 1,
                                    dx_row_stride=cols + 7)
            for got, w in zip((dx, dg, db), want):
                agree(got, *w, dt)
            lib.layer_norm(dt, dt, rows, cols, x, None, None, dx, eps=EPS, x_row_stride=cols + 1, out_row_stride=cols + 7)
            agree(dx, *f.y(), dt)


def test_weights_off_the_grid(lib):
    rng = np.random.default_rng(13)
    for dt, wt in TYPES:
        for cols in (256, 1000, 4096, 8192, 20000):
            _, x = matrix(rng, 5, cols, dt)
            _, dy = matrix(rng, 5, cols, dt)
            both = torch.from_numpy(1 + 0.3 * rng.standard_normal(2 * cols + 3)).cuda().to(TORCH[wt])
            gamma, beta = both[1:1 + cols], both[cols + 3:2 * cols + 3]
            grads = torch.full((2 * cols + 3,), 7.0, device="cuda", dtype=TORCH[wt])
            out = torch.empty_like(x)
            lib.layer_norm(dt, wt, 5, cols, x, gamma, beta, out, eps=EPS)
            f = Formula(x, gamma, beta, dt)
            agree(out, *f.y(), dt)
            lib.layer_norm_backward(dt, wt, 5, cols, dy, x, gamma, out, grads[1:1 + cols], grads[cols + 3:2 * cols + 3], eps=EPS)
            want = f.grads(dy, 5)
            for got, w, t in zip((out, grads[1:1 + cols], grads[cols + 3:2 * cols + 3]), want, (dt, wt, wt)):
                agree(got, *w, t)
            assert grads[0] == 7 and (grads[1 + cols:cols + 3] == 7).all()


def test_threads_that_share_a_stream_and_the_library_space(lib):
    """Four host threads, two of them on one stream, all of them without a workspace of their own."""
    import threading
    rng = np.random.default_rng(14)
    shapes = [(700, 1024), (60, 4096), (900, 300), (33, 9000)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    work = []
    for rows, cols in shapes:
        _, x = matrix(rng, rows, cols, F32)
        _, dy = matrix(rng, rows, cols, F32)
        work.append((rows, cols, x, dy, [torch.empty(cols, device="cuda") for _ in range(2)]))
    torch.cuda.synchronize()
    wrong = []

    def loop(k):
        rows, cols, x, dy, (dg, db) = work[k]
        first = None
        for _ in range(30):
            lib.layer_norm_backward(F32, F32, rows, cols, dy, x, None, None, dg, db, stream=streams[k // 2].cuda_stream)
            lib.sync(stream=streams[k // 2].cuda_stream)
            now = (dg.cpu(), db.cpu())
            if first is None:
                first = now
            elif not all(torch.equal(a, b) for a, b in zip(first, now)):
                wrong.append(k)
    threads = [threading.Thread(target=loop, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for rows, cols, x, dy, (dg, db) in work:
        want = Formula(x, None, None, F32).grads(dy, rows)
        agree(dg, *want[1], F32)
        agree(db, *want[2], F32)


def test_a_workspace_that_is_too_small_is_refused(lib):
    x = torch.zeros(4, 100, device="cuda")
    small = torch.empty(lib.layer_norm_backward_workspace(F32, 4, 100) - 1, device="cuda", dtype=torch.uint8)
    with pytest.raises(DaliB200Error, match="workspace"):
        lib.layer_norm_backward(F32, F32, 4, 100, x, x, None, torch.empty_like(x), torch.empty(100, device="cuda"), None, workspace=small)


def test_offsets_past_32_bits(lib):
    """Rows whose elements lie more than 2^31 elements into the buffer."""
    stride = (1 << 30) + 5
    buf = torch.zeros(2 * stride + 64 + 5, device="cuda", dtype=torch.bfloat16)
    x = torch.as_strided(buf, (3, 64), (stride, 1))
    x.copy_(torch.from_numpy(np.random.default_rng(0).standard_normal((3, 64))).cuda())
    out = torch.empty(3, 64, device="cuda", dtype=torch.bfloat16)
    lib.layer_norm(BF16, BF16, 3, 64, x, None, None, out, eps=EPS, x_row_stride=stride)
    agree(out, *Formula(x, None, None, BF16).y(), BF16)


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("cols", [100, 1024, 40000])
def test_the_gradient_of_the_rows_alone_needs_no_workspace(lib, cols, dt):
    """In a captured graph, on the per-thread default stream, with a workspace of no size, over an argument: the bits of a call that
    has all gradients."""
    rows, rng = 70, np.random.default_rng(cols)
    x, dy = matrix(rng, rows, cols, dt)[1], matrix(rng, rows, cols, dt, spread=1.0)[1]
    want, dx, dg, db = (torch.empty(n, cols, device="cuda", dtype=TORCH[dt]) for n in (rows, rows, 1, 1))
    lib.layer_norm_backward(dt, dt, rows, cols, dy, x, None, want, dg, db, eps=EPS)
    agree(want, *Formula(x, None, None, dt).grads(dy, rows)[0], dt)

    def right():
        torch.cuda.synchronize()
        assert torch.equal(dx, want)
        dx.zero_()
        torch.cuda.synchronize()

    alone = (dt, dt, rows, cols, dy, x, None, dx, None, None)
    right_over = dx.copy_(dy)
    lib.layer_norm_backward(dt, dt, rows, cols, right_over, x, None, dx, None, None, eps=EPS)
    right()
    lib.layer_norm_backward(*alone, eps=EPS, workspace=torch.empty(0, device="cuda"))
    right()
    lib.layer_norm_backward(*alone, eps=EPS, stream=2)
    right()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lib.layer_norm_backward(*alone, eps=EPS, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
        right()
    del graph


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", [(700, 16392), (331, 16401), (620, 20000), (301, 33001)])
def test_many_rows_wider_than_a_gradient_holds(lib, shape, types):
    """More rows than CTAs, of widths beyond what the gradient keeps in registers (and for the last ones, the forward pass too)."""
    test_forward(lib, shape, types)
    test_backward(lib, shape, types)
