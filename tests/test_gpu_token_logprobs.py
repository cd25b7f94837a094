"""Token log probabilities, entropies and alternatives, and their gradient, through the C ABI against the formulas in fp64.

Tolerances count roundings, u = 2^-24 (2^-53 for f64): a difference d = z - m is off by u |d|, and exp(d) by a relative
4 u (1 + |d|) (the argument's rounding and scaling, the function's own error of 2 steps); sums of k steps add k u.  Relative to the
sum, with E[.] the mean under p: lse is off by u |lse| + u (k + 4 + 4 E|d|); H = log s - u/s by the errors of both terms."""
import numpy as np
import pytest
import torch

from dali_b200.capi import BF16, DaliB200Error, F32, F64

pytestmark = pytest.mark.gpu

TORCH = {F32: torch.float32, F64: torch.float64, BF16: torch.bfloat16}
U = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -24}
HALF_STEP = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -8}
INF = float("inf")


def acc(dt):
    return torch.float64 if dt == F64 else torch.float32


def logits_of(rng, rows, vocab, dt, stride=None, offset=0, masked=0.0, spread=3.0):
    stride = vocab if stride is None else stride
    buf = torch.full((offset + rows * stride + 9,), 50.0, device="cuda", dtype=TORCH[dt])
    z = torch.as_strided(buf, (rows, vocab), (stride, 1), offset)
    v = rng.standard_normal((rows, vocab)) * spread
    if masked:
        v[rng.random((rows, vocab)) < masked] = -np.inf
    z.copy_(torch.from_numpy(v).cuda())
    return buf, z


class Formula:
    def __init__(self, z, dt):
        z = z.double()
        self.z, self.u = z, U[dt]
        self.k = 64 + z.shape[1] // 128
        m = z.max(1, keepdim=True).values
        empty = m == -INF
        d = torch.where(empty, -INF, z - torch.where(empty, 0.0, m))
        e = torch.where(empty, 0.0, torch.exp(d))
        s = e.sum(1, keepdim=True)
        self.empty = empty[:, 0]
        self.lse = torch.where(self.empty, -INF, (m + torch.log(s))[:, 0])
        self.p = torch.where(empty, 0.0, e / torch.where(empty, 1.0, s))
        d0 = torch.where(self.p > 0, d, 0.0)
        ls = torch.log(torch.where(empty, 1.0, s))[:, 0]
        mean_d = (self.p * d0.abs()).sum(1)
        mean_d2 = (self.p * d0 * d0).sum(1)
        self.entropy = ls + mean_d
        self.e_lse = self.u * torch.where(self.empty, 0.0, self.lse.abs()) + self.u * (self.k + 4 + 4 * mean_d)
        self.e_entropy = self.u * ((self.k + 4 + 4 * mean_d) * (1 + mean_d) + (self.k + 8) * mean_d + 4 * (mean_d + mean_d2) + 2 * ls)

    def logprob(self, tokens):
        t = tokens.long()
        v = self.z.shape[1]
        given = self.z.gather(1, t.clamp(0, v - 1)[:, None])[:, 0]
        lp = torch.where(self.empty, -INF, given - self.lse)
        return torch.where(t < 0, 0.0, torch.where(t >= v, float("nan"), lp))

    def e_logprob(self, lp):
        return self.e_lse + self.u * torch.where(torch.isfinite(lp), lp.abs(), 0.0)

    def top(self, k):
        values, index = torch.sort(torch.where(torch.isnan(self.z), -INF, self.z), dim=1, descending=True, stable=True)
        return torch.where(self.empty[:, None], -INF, values[:, :k] - self.lse[:, None]), index[:, :k]


def agree(got, want, bound):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    infinite = torch.isinf(want)
    assert torch.equal(got[infinite], want[infinite])
    fine = torch.isfinite(want)
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or (not torch.isnan(off).any() and off.max().item() <= 0), "off by %g more than the bound" % off.max().item()


def forward(lib, dt, z, tokens, top, stride=None, stream=None, only=None):
    rows, vocab = z.shape
    logprob, entropy, lse = (torch.full((rows,), 9.0, device="cuda", dtype=acc(dt)) for _ in range(3))
    tl = torch.full((rows, top), 9.0, device="cuda", dtype=acc(dt))
    tt = torch.full((rows, top), -9, device="cuda", dtype=torch.int32)
    lib.token_logprobs(dt, rows, vocab, z, tokens, logprob, entropy, lse, top=top, top_logprobs=tl if top else None,
                       top_tokens=tt if top else None, row_stride=stride, stream=stream)
    return logprob, entropy, lse, tl, tt


def check_forward(lib, dt, z, tokens, top, stride=None):
    logprob, entropy, lse, tl, tt = forward(lib, dt, z, tokens, top, stride)
    f = Formula(z, dt)
    want = f.logprob(tokens)
    agree(lse, f.lse, f.e_lse)
    agree(entropy, f.entropy, f.e_entropy)
    agree(logprob, want, f.e_logprob(want))
    if top:
        values, index = f.top(top)
        assert torch.equal(tt.long(), index)
        agree(tl, values, f.e_lse[:, None] + f.u * torch.where(torch.isfinite(values), values.abs(), 0.0))
    return logprob, entropy, lse


VOCABS = [1, 2, 5, 31, 32, 33, 100, 255, 1000, 1024, 4097, 10007, 32768, 50001, 131072, 260001]


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
def test_forward(lib, vocab, dt, top):
    rng = np.random.default_rng(vocab)
    top = min(top, vocab)
    for rows in (1, 3, 40) if vocab < 60000 else (1, 5):
        _, z = logits_of(rng, rows, vocab, dt)
        tokens = torch.from_numpy(rng.integers(-1, vocab, rows).astype(np.int32)).cuda()
        check_forward(lib, dt, z, tokens, top)


@pytest.mark.parametrize("dt", [F32, BF16, F64])
def test_many_rows(lib, dt):
    rng = np.random.default_rng(8)
    for rows, vocab in ((700, 1000), (2000, 127), (330, 4096)):
        _, z = logits_of(rng, rows, vocab, dt, masked=0.3)
        tokens = torch.from_numpy(rng.integers(-1, vocab, rows).astype(np.int32)).cuda()
        check_forward(lib, dt, z, tokens, 7)


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("vocab", [7, 40, 1000, 4099, 33000, 131072])
def test_masks(lib, vocab, dt):
    """-infinity in places, in all places but one, in all; the type's lowest value in all; lowest beside -infinity."""
    rng = np.random.default_rng(vocab)
    rows, low = 9, torch.finfo(TORCH[dt]).min
    _, z = logits_of(rng, rows, vocab, dt, masked=0.5)
    z[:, vocab // 2] = 1.0
    z[1] = -INF
    z[2] = -INF
    z[2, vocab - 1] = -3.0
    z[3] = -INF
    z[3, 0] = 5.0
    z[4] = low
    z[5] = low
    z[5, 3] = 0.0
    z[6] = -INF
    z[6, vocab // 3] = low
    z[6, vocab // 3 + 1] = low
    z[7, :] = low
    z[7, ::2] = -INF
    tokens = torch.tensor([vocab // 2, 0, vocab - 1, 1, 2, 3, vocab // 3, 1, -1], dtype=torch.int32, device="cuda")
    logprob, entropy, lse = check_forward(lib, dt, z, tokens, min(6, vocab))
    assert lse[1] == -INF and logprob[1] == -INF and entropy[1] == 0
    assert logprob[2] == 0 and entropy[2] == 0 and logprob[3] == -INF
    assert abs(entropy[4].item() - np.log(vocab)) < 1e-5                # uniform
    assert logprob[8] == 0


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("vocab", [33, 1000, 70001])
def test_ties_go_to_the_lowest_index(lib, vocab, dt):
    rng = np.random.default_rng(vocab)
    rows = 6
    z = torch.zeros(rows, vocab, device="cuda", dtype=TORCH[dt])
    z[1] = torch.from_numpy(rng.integers(0, 3, vocab).astype(np.float64)).cuda()
    z[2, 1::2] = -0.0                                                   # equal to +0
    z[3] = torch.from_numpy(rng.integers(-1, 2, vocab).astype(np.float64)).cuda()
    z[3, -5:] = 7.0
    z[4] = torch.arange(vocab, device="cuda", dtype=torch.float64).div(8, rounding_mode="floor").to(TORCH[dt])   # neighbours together
    z[5] = -torch.arange(vocab, device="cuda", dtype=torch.float64).to(TORCH[dt])
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    for top in (1, 9, 32):
        check_forward(lib, dt, z, tokens, top)


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("vocab", [50, 3001, 90000])
def test_rows_that_are_not_numbers(lib, vocab, dt):
    rng = np.random.default_rng(vocab)
    _, z = logits_of(rng, 6, vocab, dt)
    z[1, vocab // 2] = float("nan")
    z[2] = float("nan")
    z[3, 5] = INF
    z[4, 7] = float("nan")
    z[4, :7] = -INF
    tokens = torch.from_numpy(rng.integers(0, vocab, 6).astype(np.int32)).cuda()
    tokens[5] = vocab                                                   # no such token
    logprob, entropy, lse, tl, tt = forward(lib, dt, z, tokens, 4)
    sound = [0, 5]
    f = Formula(z[sound], dt)
    agree(lse[sound], f.lse, f.e_lse)
    agree(entropy[sound], f.entropy, f.e_entropy)
    for r in (1, 2, 3, 4):
        assert torch.isnan(torch.stack([logprob[r], entropy[r], lse[r]])).all() and torch.isnan(tl[r]).all()
    assert torch.isnan(logprob[5]) and not torch.isnan(logprob[0])
    want = torch.sort(torch.where(torch.isnan(z[1].double()), -INF, z[1].double()), descending=True, stable=True).indices[:4]
    assert torch.equal(tt[1].long(), want)
    assert (tt >= 0).all() and (tt < vocab).all()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 40000), (400, 40000), (1300, 4096), (3, 1500)])
@pytest.mark.parametrize("top", [1, 5, 32])
def test_the_largest_entries_lie_together(lib, rows, vocab, top, dt):
    """More large entries in the packets of a few threads than any other thread's largest: the alternatives are then sorted, not
    counted.  Which threads those are depends on the team: every 16th packet of a row is large, the first 40, or the last 40."""
    rng = np.random.default_rng(vocab + top)
    _, z = logits_of(rng, rows, vocab, dt)
    per = 16 // z.element_size()
    packet = torch.arange(vocab, device="cuda") // per
    for far in (packet % 256 < 4, packet % 32 == 0, packet < 40, packet >= (vocab - 1) // per - 40):
        y = torch.where(far, z + 40, z)
        if rows == 1300:
            y = y[:1200]
        tokens = torch.zeros(y.shape[0], dtype=torch.int32, device="cuda")
        check_forward(lib, dt, y.contiguous(), tokens, top)


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("rows,vocab", [(2, 40), (2, 3000), (400, 3000), (1, 70000), (1500, 2048)])
def test_fewer_numbers_than_alternatives(lib, rows, vocab, dt):
    """Rows of NaN with 3 numbers, of -infinity with 3 numbers, of both: numbers first, then -infinity, then NaN, each by index."""
    rng = np.random.default_rng(vocab)
    for kind in range(3):
        z = torch.full((rows, vocab), (float("nan"), -INF, float("nan"))[kind], device="cuda", dtype=TORCH[dt])
        if kind == 2:
            z[:, vocab // 2:] = -INF
        at = torch.from_numpy(np.stack([rng.permutation(vocab)[:3] for _ in range(rows)])).cuda()
        z.scatter_(1, at, torch.tensor([1.0, 2.0, 2.0], device="cuda", dtype=TORCH[dt]).expand(rows, 3).contiguous())
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        _, _, lse, tl, tt = forward(lib, dt, z, tokens, 10)
        rank = torch.where(torch.isnan(z), -2.0, torch.where(torch.isinf(z), -1.0, z.double()))
        want = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :10]
        assert torch.equal(tt.long(), want)
        if kind == 1:
            check_forward(lib, dt, z, tokens, 10)
        else:
            assert torch.isnan(lse).all() and torch.isnan(tl).all()


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("vocab", [64, 777, 20000, 66001])
def test_strides_and_offsets(lib, vocab, dt):
    rng = np.random.default_rng(vocab)
    for stride, offset in ((vocab + 8, 8), (vocab + 1, 3), (vocab + 2, 1)):
        buf, z = logits_of(rng, 5, vocab, dt, stride, offset, masked=0.1)
        tokens = torch.from_numpy(rng.integers(0, vocab, 5).astype(np.int32)).cuda()
        check_forward(lib, dt, z, tokens, 8, stride)
        check_backward(lib, dt, z, tokens, stride, stride + 5, offset + 2)


def test_results_that_are_not_asked_for(lib):
    rng = np.random.default_rng(4)
    _, z = logits_of(rng, 4, 500, F32)
    tokens = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    all_ = forward(lib, F32, z, tokens, 3)
    for i in range(3):
        out = [None, None, None]
        out[i] = torch.empty(4, device="cuda")
        lib.token_logprobs(F32, 4, 500, z, tokens if i == 0 else None, *out)
        assert torch.equal(out[i], all_[i])
    tl, tt = torch.empty(4, 3, device="cuda"), torch.empty(4, 3, device="cuda", dtype=torch.int32)
    lib.token_logprobs(F32, 4, 500, z, None, None, None, None, top=3, top_logprobs=tl, top_tokens=tt)
    assert torch.equal(tl, all_[3]) and torch.equal(tt, all_[4])


def backward_of(f, tokens, g, w):
    """dlogits and how far off it may be: p is off by a relative e_p = 4u(1 + |log p|) + e_lse."""
    z, p, u = f.z, f.p, f.u
    rows, vocab = z.shape
    t = tokens.long()
    g = torch.zeros(rows, device="cuda", dtype=torch.float64) if g is None else torch.where(t < 0, 0.0, g.double())
    w = torch.zeros_like(g) if w is None else w.double()
    lp = torch.where(p > 0, z - f.lse[:, None], 0.0)
    one = torch.zeros_like(z)
    ok = (t >= 0) & (t < vocab)
    one[ok] = one[ok].scatter(1, t[ok][:, None], 1.0)
    core = g[:, None] + w[:, None] * (lp + f.entropy[:, None])
    want = g[:, None] * one - p * core
    e_lse = f.u * f.lse.abs().clamp(max=1e300)[:, None] + 2 * u
    e_p = 4 * u * (1 + lp.abs()) + e_lse
    bound = p * (core.abs() * e_p + w.abs()[:, None] * (e_lse + 4 * u * (lp.abs() + f.entropy[:, None]))) + 4 * u * (want.abs() + p * core.abs() + g.abs()[:, None] * one)
    return want, bound


def check_backward(lib, dt, z, tokens, stride=None, out_stride=None, out_offset=0, entropy=True, logprob=True):
    rows, vocab = z.shape
    f = Formula(z, dt)
    lse, ent = f.lse.to(acc(dt)), f.entropy.to(acc(dt))
    g = torch.randn(rows, device="cuda", dtype=torch.float64).to(acc(dt)) if logprob else None
    w = torch.randn(rows, device="cuda", dtype=torch.float64).to(acc(dt)) if entropy else None
    out_stride = vocab if out_stride is None else out_stride
    buf = torch.full((out_offset + rows * out_stride + 9,), 50.0, device="cuda", dtype=TORCH[dt])
    dz = torch.as_strided(buf, (rows, vocab), (out_stride, 1), out_offset)
    lib.token_logprobs_backward(dt, rows, vocab, z, tokens if logprob else None, lse, ent if entropy else None, g, w, dz, row_stride=stride,
                                dlogits_row_stride=out_stride)
    want, bound = backward_of(f, tokens, g, w)
    want[f.empty] = 0
    agree(dz, want, torch.where(torch.isfinite(bound), bound, 0.0) + HALF_STEP[dt] * want.abs() * (1 + 2.0 ** -7) + torch.finfo(TORCH[dt]).tiny)
    got = dz.clone()
    dz.fill_(50.0)
    assert (buf == 50.0).all()
    return got, lse, ent, g, w


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("vocab", VOCABS)
def test_backward(lib, vocab, dt):
    rng = np.random.default_rng(vocab + 1)
    for rows in (1, 17) if vocab < 60000 else (1, 3):
        for masked in (0.0, 0.4):
            _, z = logits_of(rng, rows, vocab, dt, masked=masked)
            tokens = torch.from_numpy(rng.integers(0, vocab, rows).astype(np.int32)).cuda()
            z.scatter_(1, tokens.long()[:, None], 0.5)
            if rows > 3:
                tokens[::3] = -1
                z[5] = -INF
                z[5, tokens[5].clamp(min=0)] = 1.0
            for entropy, logprob in ((True, True), (False, True), (True, False)):
                check_backward(lib, dt, z, tokens, entropy=entropy, logprob=logprob)


@pytest.mark.parametrize("dt", [F32, BF16, F64])
def test_backward_over_the_logits(lib, dt):
    rng = np.random.default_rng(6)
    for vocab in (1000, 4097):
        _, z = logits_of(rng, 12, vocab, dt)
        tokens = torch.from_numpy(rng.integers(0, vocab, 12).astype(np.int32)).cuda()
        got, lse, ent, g, w = check_backward(lib, dt, z, tokens)
        lib.token_logprobs_backward(dt, 12, vocab, z, tokens, lse, ent, g, w, z)
        assert torch.equal(z, got)


def test_backward_of_rows_that_say_nothing(lib):
    rng = np.random.default_rng(7)
    _, z = logits_of(rng, 5, 900, F32)
    z[0, 3] = float("nan")
    z[1] = -INF
    z[2, 5] = float("nan")
    tokens = torch.tensor([-1, 4, 1, 900, 7], dtype=torch.int32, device="cuda")
    lse = torch.logsumexp(z, 1)
    g = torch.ones(5, device="cuda")
    dz = torch.full_like(z, 3.0)
    lib.token_logprobs_backward(F32, 5, 900, z, tokens, lse, None, g, None, dz)
    assert (dz[0] == 0).all()                     # no token, no gradient, whatever the logits hold
    assert (dz[1] == 0).all()                     # nothing can be drawn
    assert torch.isnan(dz[2]).all() and torch.isnan(dz[3]).all()
    assert torch.isfinite(dz[4]).all()


def test_gradient_against_differences(lib):
    """d/dt of sum(g logprob + w H)(z + t v) by central differences in fp64 (error t^2 and 2^-53 / t, t = 1e-5)."""
    rng = np.random.default_rng(9)
    rows, vocab = 5, 301
    z, v = (torch.from_numpy(rng.standard_normal((rows, vocab))).cuda() for _ in range(2))
    g, w = (torch.from_numpy(rng.standard_normal(rows)).cuda() for _ in range(2))
    tokens = torch.tensor([0, 300, 7, -1, 150], dtype=torch.int32, device="cuda")

    def f(z):
        logprob, entropy, lse, _, _ = forward(lib, F64, z, tokens, 0)
        return (g * logprob + w * entropy).sum().item(), lse, entropy
    _, lse, ent = f(z)
    dz = torch.empty_like(z)
    lib.token_logprobs_backward(F64, rows, vocab, z, tokens, lse, ent, g, w, dz)
    t = 1e-5
    assert abs((dz * v).sum().item() - (f(z + t * v)[0] - f(z - t * v)[0]) / (2 * t)) < 1e-7


@pytest.mark.parametrize("dt", [F32, BF16])
def test_the_same_call_gives_the_same_bits(lib, dt):
    rng = np.random.default_rng(10)
    for rows, vocab in ((1, 131072), (600, 5000), (3, 60001)):
        _, z = logits_of(rng, rows, vocab, dt)
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        first = forward(lib, dt, z, tokens, 20)
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(first, forward(lib, dt, z, tokens, 20)))


def test_streams_and_graphs(lib):
    rng = np.random.default_rng(11)
    rows, vocab = 4, 40000
    _, z = logits_of(rng, rows, vocab, BF16)
    tokens = torch.tensor([5, 6, 7, 8], dtype=torch.int32, device="cuda")
    f32 = dict(device="cuda", dtype=torch.float32)
    logprob, entropy, lse, tl = torch.empty(rows, **f32), torch.empty(rows, **f32), torch.empty(rows, **f32), torch.empty(rows, 5, **f32)
    tt = torch.empty(rows, 5, device="cuda", dtype=torch.int32)
    dz, g = torch.empty_like(z), torch.ones(rows, **f32)

    def both(stream):
        lib.token_logprobs(BF16, rows, vocab, z, tokens, logprob, entropy, lse, top=5, top_logprobs=tl, top_tokens=tt, stream=stream)
        lib.token_logprobs_backward(BF16, rows, vocab, z, tokens, lse, entropy, g, g, dz, stream=stream)

    def right():
        f = Formula(z, BF16)
        want = f.logprob(tokens)
        agree(logprob, want, f.e_logprob(want))
        assert torch.equal(tt.long(), f.top(5)[1])
        want, bound = backward_of(f, tokens, g, g)
        # (the forward pass's own lse and entropy came in: their errors count too)
        bound = bound + f.p * 4 * (f.e_lse + f.e_entropy)[:, None] * (1 + (f.z - f.lse[:, None]).abs())
        agree(dz, want, bound + HALF_STEP[BF16] * want.abs() * (1 + 2.0 ** -7) + torch.finfo(torch.bfloat16).tiny)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both(s.cuda_stream)
    s.synchronize()
    right()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(torch.cuda.current_stream().cuda_stream)
    z.copy_(z.flip(0))
    tokens.add_(100)
    for _ in range(3):
        tt.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        right()
    del graph


def test_offsets_past_32_bits(lib):
    stride = (1 << 30) + 3
    buf = torch.zeros(2 * stride + 1000, device="cuda", dtype=torch.bfloat16)
    z = torch.as_strided(buf, (3, 1000), (stride, 1))
    z.copy_(torch.from_numpy(np.random.default_rng(0).standard_normal((3, 1000))).cuda())
    tokens = torch.tensor([3, 4, 999], dtype=torch.int32, device="cuda")
    check_forward(lib, BF16, z, tokens, 3, stride)


def test_the_largest_vocabulary(lib):
    """2^31 - 1 entries a row, where a step past the row's end no longer fits an int: the kernels that go entry by entry (the
    gradient of rows that lie unlike one another, f64 rows) end with the row and leave what lies in front of it and behind it."""
    vocab = (1 << 31) - 1
    token, lse = torch.tensor([vocab - 1], dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda")
    z = torch.zeros(vocab, device="cuda", dtype=torch.bfloat16)
    buf = torch.full((vocab + 18,), 5.0, device="cuda", dtype=torch.bfloat16)
    dz = buf[9:9 + vocab]
    assert (z.data_ptr() - dz.data_ptr()) % 16
    lib.token_logprobs_backward(BF16, 1, vocab, z, token, lse, None, torch.zeros(1, device="cuda"), None, dz)
    assert (buf[:9] == 5.0).all() and (buf[9 + vocab:] == 5.0).all()
    assert not dz.view(torch.int16).any()
    del z, buf, dz
    z = torch.full((vocab,), -INF, device="cuda", dtype=torch.float64)
    z[-1] = 2.0
    z[5] = 1.0
    logprob, entropy, lse, tl, tt = forward(lib, F64, z[None], token, 1)
    want = 2.0 + np.log1p(np.exp(-1.0))
    assert abs(lse.item() - want) < 1e-14 and abs(logprob.item() - (2.0 - want)) < 1e-14 and tt.item() == vocab - 1


@pytest.mark.parametrize("dt", [F32, BF16, F64])
@pytest.mark.parametrize("rows,vocab", [(1, 100), (9, 4099), (1300, 1000), (3, 131072), (400, 30001)])
def test_what_all_entries_have_in_common_costs_no_digits(lib, rows, vocab, dt):
    """Rows far from 0: log probabilities and entropies are those of the row less its largest entry (which no rounding touches:
    both are multiples of the same step, a few bits apart), with the error of such a row; lse is off by half a step of itself."""
    rng = np.random.default_rng(rows + vocab)
    for common in {F32: (1e3, -1e4, 3e5), BF16: (200.0, -1e3), F64: (1e6, -1e12)}[dt]:
        z = torch.from_numpy(common + 3.0 * rng.standard_normal((rows, vocab))).cuda().to(TORCH[dt])
        tokens = torch.from_numpy(rng.integers(-1, vocab, rows).astype(np.int32)).cuda()
        logprob, entropy, lse, tl, tt = forward(lib, dt, z, tokens, 8)
        m = z.double().max(1, keepdim=True).values
        f = Formula(z.double() - m, dt)
        want = f.logprob(tokens)
        agree(logprob, want, f.e_logprob(want))
        agree(entropy, f.entropy, f.e_entropy)
        agree(lse, m[:, 0] + f.lse, f.e_lse + f.u * (m[:, 0] + f.lse).abs())
        values, index = f.top(8)
        assert torch.equal(tt.long(), index)
        agree(tl, values, f.e_lse[:, None] + f.u * values.abs())
