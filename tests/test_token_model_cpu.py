"""The operators of a token model in the Array / op:: front end, without a GPU: shapes, types, refusals, laziness (dry run), and
what a shard of the rows ends in."""
import ctypes
import os
import sys

import numpy as np
import pytest
import torch.distributed as dist
import torch.multiprocessing as mp

import dali_b200
from dali_b200 import DaliB200Error
from dali_b200.array import Array, DTYPE_BF16, DTYPE_DOUBLE, DTYPE_FLOAT, DTYPE_INT32, last_variant, lazy_stats, op, set_dry_run

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def dry(tmp_path):
    dali_b200.load_library().cache_set_dir(str(tmp_path))
    set_dry_run(True)
    yield
    set_dry_run(False)


def f32(*shape):
    return Array(np.zeros(shape, np.float32))


def f64(*shape):
    return Array(np.zeros(shape, np.float64))


def bf16(*shape):
    return Array(np.zeros(shape, np.float32), DTYPE_BF16)


def i32(*shape):
    return Array(np.zeros(shape, np.int32))


def launched(arr):
    before = lazy_stats()
    arr.eval()
    after = lazy_stats()
    return {k: after[k] - before[k] for k in after}


def test_shapes_and_types():
    y = op.layer_norm(f32(2, 3, 5), f32(5), f32(5))
    assert y.shape == (2, 3, 5) and y.dtype == DTYPE_FLOAT and not y.is_buffer()
    assert op.layer_norm(bf16(3, 5)).dtype == DTYPE_BF16                       # rows keep their type
    assert op.layer_norm(bf16(3, 5), f32(5)).dtype == DTYPE_BF16
    assert op.layer_norm(f32(3, 5), f64(5)).dtype == DTYPE_DOUBLE and op.layer_norm(f64(3, 5), f32(5)).dtype == DTYPE_DOUBLE
    dx, dg, db = op.layer_norm_backward(f32(3, 5), bf16(3, 5), bf16(5))
    assert dx.dtype == DTYPE_FLOAT and dg.dtype == DTYPE_FLOAT                 # widened, never narrowed
    dx, dg, db = op.layer_norm_backward(bf16(3, 5), bf16(3, 5), f32(5))
    assert dx.dtype == DTYPE_BF16 and dg.dtype == db.dtype == DTYPE_FLOAT and dx.shape == (3, 5) and dg.shape == db.shape == (5,)
    lp, h, lse, tl, tt = op.token_logprobs(bf16(2, 3, 50), i32(2, 3), top=4)
    assert lp.shape == h.shape == lse.shape == (2, 3) and tl.shape == tt.shape == (2, 3, 4)
    assert lp.dtype == tl.dtype == DTYPE_FLOAT and tt.dtype == DTYPE_INT32
    lp, h, lse, tl, tt = op.token_logprobs(f64(50))
    assert lp is None and tl is None and tt is None and h.shape == () and h.dtype == DTYPE_DOUBLE
    dz = op.token_logprobs_backward(bf16(3, 50), i32(3), f32(3), f32(3), f32(3), f32(3))
    assert dz.shape == (3, 50) and dz.dtype == DTYPE_BF16
    assert op.token_logprobs_backward(f32(3, 50), i32(3), f64(3), None, f64(3)).dtype == DTYPE_DOUBLE
    assert op.global_norm([f32(3), bf16(4, 5)]).dtype == DTYPE_FLOAT and op.global_norm([f32(3), f64(4)]).dtype == DTYPE_DOUBLE
    clipped, norm = op.clip_by_global_norm([f32(3), bf16(4, 5)], 1.0)
    assert [c.shape for c in clipped] == [(3,), (4, 5)] and [c.dtype for c in clipped] == [DTYPE_FLOAT, DTYPE_BF16] and norm.shape == ()


@pytest.mark.parametrize("text,call", [
    ("float, double or bfloat16", lambda: op.layer_norm(i32(3, 5))),
    ("last axis", lambda: op.layer_norm(Array(1.0, DTYPE_FLOAT))),
    ("gamma must be a vector", lambda: op.layer_norm(f32(3, 5), f32(4))),
    ("beta must be a vector", lambda: op.layer_norm(f32(3, 5), f32(5), f32(1, 5))),
    ("eps", lambda: op.layer_norm(f32(3, 5), eps=-1.0)),
    ("dy must have x's shape", lambda: op.layer_norm_backward(f32(3, 4), f32(3, 5))),
    ("tokens must be integers", lambda: op.token_logprobs(f32(3, 5), f32(3))),
    ("one value per row", lambda: op.token_logprobs(f32(3, 5), i32(4))),
    ("top must lie", lambda: op.token_logprobs(f32(3, 5), top=6)),
    ("top must lie", lambda: op.token_logprobs(f32(3, 50), top=33)),
    ("vocabulary is empty", lambda: op.token_logprobs(f32(3, 0))),
    ("neither", lambda: op.token_logprobs_backward(f32(3, 5), i32(3), f32(3), None, None)),
    ("needs tokens", lambda: op.token_logprobs_backward(f32(3, 5), None, f32(3), None, f32(3))),
    ("needs entropy", lambda: op.token_logprobs_backward(f32(3, 5), i32(3), f32(3), None, None, f32(3))),
    ("one value per row", lambda: op.token_logprobs_backward(f32(3, 5), i32(3), f32(3), None, f32(2))),
    ("float, double or bfloat16", lambda: op.global_norm([f32(3), i32(3)])),
    ("max_norm", lambda: op.clip_by_global_norm([f32(3)], 0.0)),
    ("max_norm", lambda: op.clip_by_global_norm([f32(3)], float("nan"))),
])
def test_refusals(text, call):
    with pytest.raises(DaliB200Error) as e:
        call()
    assert text in str(e.value), str(e.value)


def test_what_runs():
    x, g = f32(4, 6), f32(6)
    y = op.layer_norm(op.tanh(x), g)
    assert launched(y) == {"kernels": 2, "gemms": 0, "temporaries": 0}         # the fused producer, then the operator
    assert last_variant() == "layer_norm" and y.is_buffer()
    z = op.layer_norm(x, g) * 2.0                                              # not fused with what consumes it
    assert launched(z) == {"kernels": 2, "gemms": 0, "temporaries": 1}
    # one kernel, whichever of the results is asked for first
    dx, dg, db = op.layer_norm_backward(f32(4, 6), x, g)
    assert launched(dg) == {"kernels": 1, "gemms": 0, "temporaries": 0}
    assert not dx.is_buffer()
    assert launched(dx)["kernels"] == 0 and launched(db)["kernels"] == 0 and dx.is_buffer()
    # an expression that is handed to several consumers is evaluated once
    lp, h, lse, _, _ = op.token_logprobs(f32(3, 9), i32(3))
    loss = op.sum(lp) + op.sum(h)
    assert launched(loss)["kernels"] <= 4
    clipped, norm = op.clip_by_global_norm([f32(4), f32(5)], 1.0)
    assert launched(clipped[1])["kernels"] == 1 and launched(norm)["kernels"] == 0 and launched(clipped[0])["kernels"] == 0


def test_views_and_assignments_of_results():
    x = f32(4, 6)
    y = op.layer_norm(x)
    assert y[1].shape == (6,) and y.T.shape == (6, 4) and y.reshape([24]).shape == (24,)
    launched(y.T)
    d = f32(4, 6)
    d += op.layer_norm(x)
    d.assign(op.layer_norm(d))
    assert d.shape == (4, 6)


def _worker(rank, world, port, out):
    sys.path.insert(0, ROOT)
    import dali_b200 as db
    from dali_b200 import comm
    from dali_b200.array import Array, collectives, op, set_dry_run
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    lib = db.load_library()
    comm.init_host_from_torch(lib)
    set_dry_run(True)
    x = Array.scatter_rows(np.zeros((7, 5), np.float32))
    g = Array(np.zeros(5, np.float32))
    mark = x.shard
    said = []

    def took(a):
        before = collectives()[0]
        a.eval()
        n, what = collectives()
        said.append("%d:%s" % (n - before, what if n > before else "-"))
    y = op.layer_norm(x, g)
    assert y.shard == mark
    took(y)
    dx, dg, dbeta = op.layer_norm_backward(x, x, g)
    assert dx.shard == mark and dg.shard[0] == dbeta.shard[0] == -1
    took(dg)
    took(dx)
    t = Array.scatter_rows(np.zeros(7, np.int32))
    lp, h, lse, tl, tt = op.token_logprobs(x, t, 2)
    assert lp.shard == h.shard == mark and tl.shard == mark
    took(op.sum(lp))
    assert op.token_logprobs_backward(x, t, lse, h, lp).shard == mark
    took(op.global_norm([x, g]))
    took(op.global_norm([g]))
    for bad in (lambda: op.layer_norm(Array(np.zeros((4, 5), np.float32)).set_shard(1, 0, 10)), lambda: op.layer_norm(x, Array(np.zeros(5, np.float32)).set_shard(0, 0, 10)),
                lambda: op.layer_norm_backward(Array(np.zeros(x.shape, np.float32)), x, g)):
        try:
            bad()
            said.append("accepted")
        except db.DaliB200Error as e:
            said.append("shard" in str(e))
    set_dry_run(False)
    np.save(os.path.join(out, "said%d.npy" % rank), np.array([str(s) for s in said]))
    lib.comm_destroy()
    dist.destroy_process_group()


def test_shards_of_rows(tmp_path):
    port = 31500 + (os.getpid() % 2000)
    mp.spawn(_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    for rank in range(2):
        said = list(np.load(os.path.join(str(tmp_path), "said%d.npy" % rank)))
        assert said[0] == "0:-" and said[1].startswith("2:allreduce sum 5") and said[2] == "0:-"
        assert said[3].startswith("1:allreduce sum 1")
        assert said[4].startswith("1:allreduce sum 1 f64") and said[5] == "0:-"
        assert said[6:] == ["True", "True", "True"]


@pytest.mark.parametrize("text,call", [
    ("layer_norm needs x", lambda: op.layer_norm(None)),
    ("layer_norm_backward needs dy", lambda: op.layer_norm_backward(None, f32(3, 5))),
    ("layer_norm_backward needs x", lambda: op.layer_norm_backward(f32(3, 5), None)),
    ("token_logprobs needs logits", lambda: op.token_logprobs(None)),
    ("token_logprobs_backward needs lse", lambda: op.token_logprobs_backward(f32(3, 5), i32(3), None, None, f32(3))),
    ("token_logprobs_backward needs logits", lambda: op.token_logprobs_backward(None, i32(3), f32(3), None, f32(3))),
])
def test_arguments_that_may_not_be_left_out(text, call):
    with pytest.raises(DaliB200Error) as e:
        call()
    assert text in str(e.value), str(e.value)


def test_null_handles_and_results_in_c():
    lib = dali_b200.load_library()
    c, error = lib.c, lib.last_error
    handle, eps, one = ctypes.c_void_p, ctypes.c_double(1e-5), ctypes.c_double(1.0)
    x, y = f32(3, 5), f32(4)
    two = (handle * 2)(x._h, y._h)
    # refused: a list with a hole, no list, a negative number of arrays
    assert c.dali_op_global_norm((handle * 2)(x._h, None), 2, ctypes.byref(handle())) != 0 and "global_norm needs array 1" in error()
    assert c.dali_op_global_norm(None, 2, ctypes.byref(handle())) != 0 and "global_norm needs a list" in error()
    assert c.dali_op_clip_by_global_norm(two, -1, one, two, None) != 0 and "clip_by_global_norm needs a list" in error()
    # not wanted: no result, or some of them
    assert c.dali_op_layer_norm(x._h, None, None, eps, None) == 0
    assert c.dali_op_layer_norm_backward(x._h, x._h, None, eps, None, None, None) == 0
    assert c.dali_op_token_logprobs(x._h, None, 0, None, None, None, None, None) == 0
    assert c.dali_op_token_logprobs_backward(x._h, i32(3)._h, f32(3)._h, None, f32(3)._h, None, None) == 0
    assert c.dali_op_global_norm(two, 2, None) == 0
    assert c.dali_op_clip_by_global_norm(two, 2, one, None, None) == 0
    norm = handle()
    assert c.dali_op_clip_by_global_norm(two, 2, one, None, ctypes.byref(norm)) == 0
    assert Array(_handle=norm).shape == ()
    clipped = (handle * 2)()
    assert c.dali_op_clip_by_global_norm(two, 2, one, clipped, None) == 0
    assert [Array(_handle=handle(h)).shape for h in clipped] == [(3, 5), (4,)]
    assert c.dali_op_global_norm(None, 0, ctypes.byref(norm)) == 0 and Array(_handle=norm).shape == ()
