"""The operators of a token model through the Array / op:: front end on the GPU: alone, over views and bf16 arrays, together as a
training step, and over shards of the rows."""
import numpy as np
import pytest

from dali_b200.array import Array, DTYPE_BF16, DTYPE_DOUBLE, from_bf16_bits, lazy_stats, op, to_bf16_bits

pytestmark = pytest.mark.gpu
EPS = 1e-5


def norm(x, g, b):
    d = x - x.mean(-1, keepdims=True)
    return d / np.sqrt((d * d).mean(-1, keepdims=True) + EPS) * g + b


def logprobs(z, t):
    m = z.max(-1, keepdims=True)
    lse = m + np.log(np.exp(z - m).sum(-1, keepdims=True))
    p = np.exp(z - lse)
    return np.take_along_axis(z - lse, t[..., None], -1)[..., 0], -(p * (z - lse)).sum(-1), lse[..., 0]


def test_results_against_the_formulas():
    """fp32 over well-scaled values: 1e-5 is more than 100 roundings of 2^-24 of values up to 10."""
    rng = np.random.default_rng(0)
    x, dy = (rng.standard_normal((3, 4, 70)).astype(np.float32) for _ in range(2))
    g, b = (rng.standard_normal(70).astype(np.float32) for _ in range(2))
    y = op.layer_norm(Array(x), Array(g), Array(b))
    np.testing.assert_allclose(y.numpy(), norm(x.astype(np.float64), g, b), rtol=0, atol=1e-5)
    z, t = 2 * dy, rng.integers(0, 70, (3, 4)).astype(np.int32)
    lp, h, lse, tl, tt = op.token_logprobs(Array(z), Array(t), top=5)
    wlp, wh, wlse = logprobs(z.astype(np.float64), t)
    order = np.argsort(-z.astype(np.float64), -1, kind="stable")[..., :5]
    np.testing.assert_array_equal(tt.numpy(), order)
    for got, want in ((lp, wlp), (h, wh), (lse, wlse), (tl, np.take_along_axis(z.astype(np.float64), order, -1) - wlse[..., None])):
        np.testing.assert_allclose(got.numpy(), want, rtol=0, atol=1e-5)
    n = op.global_norm([Array(x), Array(g)]).item()
    assert abs(n - np.sqrt((x.astype(np.float64) ** 2).sum() + (g.astype(np.float64) ** 2).sum())) < 1e-5 * n
    # a row without a batch axis
    np.testing.assert_allclose(op.layer_norm(Array(x[0, 0])).numpy(), norm(x[0, 0].astype(np.float64), 1, 0), rtol=0, atol=1e-5)


def test_views_assignments_and_lazy_arguments():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((12, 40)).astype(np.float32)
    a = Array(x)
    for view, ref in ((a[2:9], x[2:9]), (a[:, 3:30], x[:, 3:30]), (a[::2], x[::2]), (a[:, ::2], x[:, ::2]), (a.T, x.T), (a[::-1], x[::-1]),
                      (a[3], x[3]), (a.reshape((4, 3, 40)), x.reshape(4, 3, 40)), (op.tanh(a), np.tanh(x)),
                      (a[0:1].broadcast_to_shape((5, 40)), np.broadcast_to(x[0:1], (5, 40)))):
        y = op.layer_norm(view)
        np.testing.assert_allclose(y.numpy(), norm(ref.astype(np.float64), 1, 0), rtol=0, atol=2e-5)
    want = norm(x.astype(np.float64), 1, 0)
    np.testing.assert_allclose(op.layer_norm(a).T.numpy(), want.T, rtol=0, atol=2e-5)
    np.testing.assert_allclose((op.layer_norm(a)[2] * 3.0 + 1.0).numpy(), want[2] * 3 + 1, rtol=0, atol=1e-4)
    d = Array(np.ones((12, 40), np.float32))
    d += op.layer_norm(a)
    np.testing.assert_allclose(d.numpy(), 1 + want, rtol=0, atol=2e-5)
    d[0:12].assign(op.layer_norm(a))
    np.testing.assert_allclose(d.numpy(), want, rtol=0, atol=2e-5)
    a.assign(op.layer_norm(a))                                        # over its own argument
    np.testing.assert_allclose(a.numpy(), want, rtol=0, atol=2e-5)
    # the same lazy value read twice, and a result taken after its argument has changed in place
    b = Array(x)
    y = op.layer_norm(b)
    z = y + y
    np.testing.assert_allclose(z.numpy(), 2 * want, rtol=0, atol=4e-5)
    np.testing.assert_allclose(y.numpy(), want, rtol=0, atol=2e-5)


def test_one_kernel_for_all_results():
    rng = np.random.default_rng(2)
    x, dy = (Array(rng.standard_normal((9, 33)).astype(np.float32)) for _ in range(2))
    before = lazy_stats()["kernels"]
    dx, dg, db = op.layer_norm_backward(dy, x)
    first = [a.numpy() for a in (db, dx, dg)]
    assert lazy_stats()["kernels"] == before + 1
    dx, dg, db = op.layer_norm_backward(dy, x)
    del dg, db                                                        # not wanted: not computed
    np.testing.assert_array_equal(dx.numpy(), first[1])
    dx *= 2.0                                                         # a result is an array of its own
    np.testing.assert_array_equal(dx.numpy(), 2 * first[1])
    _, _, _, tl, tt = op.token_logprobs(x, top=3)
    del tl
    np.testing.assert_array_equal(tt.numpy(), np.argsort(-x.numpy(), -1, kind="stable")[:, :3])


def test_bf16_arrays():
    """bf16 rows, fp32 weights: one rounding of 2^-8 at the store beside fp32's."""
    rng = np.random.default_rng(3)
    x = from_bf16_bits(to_bf16_bits(rng.standard_normal((6, 100))))
    g = rng.standard_normal(100).astype(np.float32)
    y = op.layer_norm(Array(x, DTYPE_BF16), Array(g))
    assert y.dtype == DTYPE_BF16
    want = norm(x.astype(np.float64), g, 0)
    got = from_bf16_bits(y.numpy())
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) * 1.01 + 1e-5).all()
    t = rng.integers(0, 100, 6).astype(np.int32)
    lp, h, lse, _, _ = op.token_logprobs(Array(x, DTYPE_BF16), Array(t))
    for a, w in zip((lp, h, lse), logprobs(x.astype(np.float64), t)):
        np.testing.assert_allclose(a.numpy(), w, rtol=0, atol=1e-5)
    # straight into the tensor-core product: rows that stay bf16
    w = Array(np.eye(100, 104, dtype=np.float32), DTYPE_BF16)
    xa = Array(np.tile(x[:, :96], (1, 1)), DTYPE_BF16)
    p = op.dot(op.layer_norm(xa), Array(np.eye(96, 104, dtype=np.float32), DTYPE_BF16)).numpy()
    np.testing.assert_array_equal(p[:, :96], from_bf16_bits(op.layer_norm(xa).numpy()))
    assert w.shape == (100, 104)


class Step:
    """Embedding rows -> layer norm -> product with the output matrix -> log probabilities of the targets and entropies, and the way
    back, with the front end's own operators."""

    def __init__(self, rng, tokens=40, width=48, vocab=65, dtype=np.float64):
        self.ids = rng.integers(0, vocab, tokens).astype(np.int32)
        self.targets = rng.integers(0, vocab, tokens).astype(np.int32)
        self.targets[3] = -1
        self.bonus = 0.05
        self.params = {"table": rng.standard_normal((vocab, width)), "gamma": 1 + 0.1 * rng.standard_normal(width),
                       "beta": 0.1 * rng.standard_normal(width), "out": rng.standard_normal((width, vocab)) / np.sqrt(width)}
        self.params = {k: v.astype(dtype) for k, v in self.params.items()}

    def loss(self, params):
        p = {k: Array(v) for k, v in params.items()}
        x = op.gather(p["table"], Array(self.ids))
        z = op.dot(op.layer_norm(x, p["gamma"], p["beta"], EPS), p["out"])
        lp, h, _, _, _ = op.token_logprobs(z, Array(self.targets))
        return (-op.sum(lp) - self.bonus * op.sum(h)).item()

    def gradients(self):
        p = {k: Array(v) for k, v in self.params.items()}
        one = np.ones(len(self.ids), self.params["table"].dtype)
        x = op.gather(p["table"], Array(self.ids))
        x.eval()
        y = op.layer_norm(x, p["gamma"], p["beta"], EPS)
        z = op.dot(y, p["out"])
        lp, h, lse, _, _ = op.token_logprobs(z, Array(self.targets))
        dz = op.token_logprobs_backward(z, Array(self.targets), lse, h, Array(-one), Array(-self.bonus * one))
        dout = op.dot(y.T, dz)
        dx, dg, db = op.layer_norm_backward(op.dot(dz, p["out"].T), x, p["gamma"], EPS)
        dtable = Array(np.zeros_like(self.params["table"]))
        self.scatter(dtable, dx)
        return {"table": dtable, "gamma": dg, "beta": db, "out": dout}

    def scatter(self, dtable, dx):
        """Rows that name a token more than once are added one after another."""
        d = dx.numpy()
        total = np.zeros_like(self.params["table"])
        np.add.at(total, self.ids, d)
        dtable.assign(Array(total))


def test_a_training_step_against_differences():
    """Every parameter's gradient along a random direction, central differences of the loss in fp64: t = 1e-5 leaves an error of
    about t^2 and 2^-53 |loss| / t = 1e-9."""
    rng = np.random.default_rng(4)
    step = Step(rng)
    grads = step.gradients()
    t = 1e-5
    for name, value in step.params.items():
        v = rng.standard_normal(value.shape)
        plus, minus = ({**step.params, name: value + s * t * v} for s in (1, -1))
        want = (step.loss(plus) - step.loss(minus)) / (2 * t)
        got = (grads[name].numpy() * v).sum()
        assert abs(got - want) < 1e-6 * (1 + abs(want)), (name, got, want)


def test_clipped_updates_go_downhill():
    """The whole step in fp32 with clipping: the gradients agree with those of fp64 to 1e-4 of their norm (products of 48 and sums of
    65 terms in fp32, 2^-24 each, through two products), the clipped list has the norm asked for, and a small step along it does what
    its gradient says."""
    wide, narrow = Step(np.random.default_rng(5)), Step(np.random.default_rng(5), dtype=np.float32)
    exact = {k: g.numpy() for k, g in wide.gradients().items()}
    grads = narrow.gradients()
    total = np.sqrt(sum((g ** 2).sum() for g in exact.values()))
    names = sorted(grads)
    clipped, norm = op.clip_by_global_norm([grads[k] for k in names], 0.5)
    assert abs(norm.item() / total - 1) < 1e-4
    clipped = {k: c.numpy() for k, c in zip(names, clipped)}
    for k in names:
        assert np.linalg.norm(clipped[k] * (total / 0.5) - exact[k]) < 1e-4 * total
    got = np.sqrt(sum((c.astype(np.float64) ** 2).sum() for c in clipped.values()))
    assert abs(got / 0.5 - 1) < 1e-5
    step = 1e-3
    moved = {k: wide.params[k] - step * clipped[k] for k in names}
    slope = -sum((clipped[k] * exact[k]).sum() for k in names)
    assert abs((wide.loss(moved) - wide.loss(wide.params)) / step - slope) < 0.02 * abs(slope)


def test_shards_of_the_rows(lib):
    """Two ranks' rows on one GPU: the host transport's all-reduce adds what the other rank, given the other half of the rows, would
    send (its partial results are computed here beforehand, without shards)."""
    rng = np.random.default_rng(6)
    x, dy = (rng.standard_normal((10, 24)) for _ in range(2))
    g = rng.standard_normal(24)
    mine, theirs = slice(0, 5), slice(5, 10)
    odx, odg, odb = op.layer_norm_backward(Array(dy[theirs]), Array(x[theirs]), Array(g))
    others = [odg.numpy(), odb.numpy(), np.array([(x[theirs] ** 2).sum()])]
    wdx, wdg, wdb = [a.numpy() for a in op.layer_norm_backward(Array(dy), Array(x), Array(g))]
    queue = list(others)

    def allreduce(buf, n, dtype, op_code):
        import ctypes
        assert dtype == 1 and op_code == 0
        a = np.ctypeslib.as_array(ctypes.cast(buf, ctypes.POINTER(ctypes.c_double)), (n,))
        a += queue.pop(0)

    lib.comm_init_host(2, 0, allreduce, lambda *a: None)
    try:
        xs, dys = Array(x[mine]).set_shard(0, 0, 10), Array(dy[mine]).set_shard(0, 0, 10)
        dx, dg, db = op.layer_norm_backward(dys, xs, Array(g))
        np.testing.assert_allclose(dg.numpy(), wdg, rtol=0, atol=1e-13)
        np.testing.assert_allclose(db.numpy(), wdb, rtol=0, atol=1e-13)
        np.testing.assert_allclose(dx.numpy(), wdx[mine], rtol=0, atol=1e-13)
        clipped, norm = op.clip_by_global_norm([xs, Array(g)], 1.0)
        want = np.sqrt((x ** 2).sum() + (g ** 2).sum())
        assert abs(norm.item() / want - 1) < 1e-14
        np.testing.assert_allclose(clipped[0].numpy(), x[mine] / want, rtol=1e-13, atol=0)
        assert not queue
    finally:
        lib.comm_destroy()


def test_lists_whose_results_are_not_all_wanted():
    rng = np.random.default_rng(7)
    a = [rng.standard_normal(n) for n in (5, 1000, 70)]
    want = np.sqrt(sum((x ** 2).sum() for x in a))
    clipped, norm = op.clip_by_global_norm([Array(x) for x in a], 0.5)
    del clipped[1]
    np.testing.assert_allclose(clipped[1].numpy(), a[2] * 0.5 / want, rtol=1e-14)
    assert abs(norm.item() / want - 1) < 1e-14
    np.testing.assert_allclose(clipped[0].numpy(), a[0] * 0.5 / want, rtol=1e-14)
    clipped, norm = op.clip_by_global_norm([Array(x) for x in a] + [Array(a[1].reshape(10, 100)).T], 1e9)
    np.testing.assert_array_equal(clipped[3].numpy(), a[1].reshape(10, 100).T)
    assert op.global_norm([]).item() == 0 and op.clip_by_global_norm([], 1.0)[1].item() == 0
    assert norm.dtype == DTYPE_DOUBLE


def test_shards_of_rows_without_tokens(lib):
    """Nothing of token_logprobs crosses ranks: what a shard's rows give is what those rows give alone, with and without
    tokens, whichever of the results are held."""
    rng = np.random.default_rng(8)
    z = rng.standard_normal((5, 33)).astype(np.float32)
    t = rng.integers(0, 33, 5).astype(np.int32)
    want = [a.numpy() for a in op.token_logprobs(Array(z), Array(t), top=3)]

    def nothing(*args):
        raise AssertionError("no collective step is due")

    lib.comm_init_host(2, 0, nothing, nothing)
    try:
        shard = lambda a: Array(a).set_shard(0, 0, 10)                 # noqa: E731
        lp, h, lse, tl, tt = op.token_logprobs(shard(z))
        assert lp is None and tl is None and tt is None
        np.testing.assert_array_equal(lse.numpy(), want[2])
        np.testing.assert_array_equal(h.numpy(), want[1])
        for tokens in (None, shard(t)):
            got = op.token_logprobs(shard(z), tokens, top=3)
            for g, w in zip(got, want):
                assert (g is None) == (tokens is None and w is want[0])
                if g is not None:
                    np.testing.assert_array_equal(g.numpy(), w)
        _, _, _, _, tt = op.token_logprobs(shard(z), top=2)
        np.testing.assert_array_equal(tt.numpy(), want[4][:, :2])
    finally:
        lib.comm_destroy()


def test_a_norm_that_fp32_cannot_hold_scales_nothing(lib):
    """All of a list, a part of it, and a shard of it (the other rank's rows hold zeros): the same answer."""
    x, y = np.full((9, 10), 1e38, np.float32), np.full(10, 1e38, np.float32)
    clipped, norm = op.clip_by_global_norm([Array(x), Array(y)], 1.0)
    assert norm.item() == np.inf
    np.testing.assert_array_equal(clipped[0].numpy(), x)
    np.testing.assert_array_equal(clipped[1].numpy(), y)
    clipped, norm = op.clip_by_global_norm([Array(x), Array(y)], 1.0)
    del clipped[0]
    np.testing.assert_array_equal(clipped[0].numpy(), y)
    assert norm.item() == np.inf
    lib.comm_init_host(2, 0, lambda buf, n, dtype, op_code: None, lambda *a: None)
    try:
        clipped, norm = op.clip_by_global_norm([Array(x).set_shard(0, 0, 18), Array(y)], 1.0)
        np.testing.assert_array_equal(clipped[0].numpy(), x)
        np.testing.assert_array_equal(clipped[1].numpy(), y)
        assert norm.item() == np.inf
    finally:
        lib.comm_destroy()
    clipped, norm = op.clip_by_global_norm([Array(x.astype(np.float64)), Array(y)], 1e38)
    assert norm.dtype == DTYPE_DOUBLE and abs(norm.item() / np.float64(np.sqrt(100 * np.float64(np.float32(1e38)) ** 2)) - 1) < 1e-14
    np.testing.assert_allclose(clipped[0].numpy(), np.full((9, 10), 1e37), rtol=1e-6)


def test_results_of_a_call_belong_to_one_state_of_its_arguments():
    """The first result asked for runs the call on the arguments of that moment, and its siblings keep to them when an argument
    changes in place; a call that has not run reads what is there."""
    rng = np.random.default_rng(9)
    x, dy, g = (rng.standard_normal(s) for s in ((6, 40), (6, 40), 40))
    want = [a.numpy() for a in op.layer_norm_backward(Array(dy), Array(x), Array(g))]
    moved = [a.numpy() for a in op.layer_norm_backward(Array(dy), Array(3 * x), Array(g))]
    ax, ag = Array(x), Array(g)
    dx, dg, db = op.layer_norm_backward(Array(dy), ax, ag)
    np.testing.assert_array_equal(dg.numpy(), want[1])
    ag -= dg * 0.1                                                    # a solver's step between two gradients of its layer
    ax *= 3.0
    np.testing.assert_array_equal(dx.numpy(), want[0])
    np.testing.assert_array_equal(db.numpy(), want[2])
    np.testing.assert_allclose(ag.numpy(), g - 0.1 * want[1], rtol=0, atol=1e-15)
    bx = Array(x)
    dx, dg, db = op.layer_norm_backward(Array(dy), bx, Array(g))
    bx *= 3.0
    for got, w in zip((dg, dx, db), (moved[1], moved[0], moved[2])):
        np.testing.assert_array_equal(got.numpy(), w)
