"""What the operators of a token model refuse, without a GPU: every argument is looked at before a device is.  The calls name a
device that no machine has, so that one which is not refused for its arguments is refused for that."""
import pytest

import dali_b200
from dali_b200.capi import BF16, DaliB200Error, F32, F64, I32

A, B, C, D = 1 << 20, 2 << 20, 3 << 20, 4 << 20          # addresses that nobody reads


@pytest.fixture(scope="module")
def lib():
    return dali_b200.load_library()


def refused(text, f, *args, **kw):
    with pytest.raises(DaliB200Error) as e:
        f(*args, device=-1, **kw)
    assert text in str(e.value), str(e.value)


def accepted(f, *args, **kw):
    """Refused for the device alone."""
    with pytest.raises(DaliB200Error) as e:
        f(*args, device=-1, **kw)
    assert "device index out of range" in str(e.value), str(e.value)


class Space:
    """A workspace at an address that nobody reads."""

    def __init__(self, at, size):
        self.at, self.size = at, size

    def data_ptr(self):
        return self.at

    def numel(self):
        return self.size

    def element_size(self):
        return 1


def test_layer_norm(lib):
    f = lib.layer_norm
    accepted(f, F32, F32, 4, 100, A, B, C, D)
    accepted(f, BF16, F32, 4, 100, A, None, None, A)
    accepted(f, F64, F64, 1, 100, A, None, None, D, x_row_stride=0)
    accepted(f, F32, F32, 0, 100, None, None, None, None)
    refused("dtype must be", f, I32, I32, 4, 100, A, B, C, D)
    refused("weights have the rows' type", f, F32, BF16, 4, 100, A, B, C, D)
    refused("weights have the rows' type", f, F64, F32, 4, 100, A, B, C, D)
    refused("negative size", f, F32, F32, -1, 100, A, B, C, D)
    refused("eps", f, F32, F32, 4, 100, A, B, C, D, eps=-1e-5)
    refused("eps", f, F32, F32, 4, 100, A, B, C, D, eps=float("nan"))
    refused("x is a null pointer", f, F32, F32, 4, 100, None, B, C, D)
    refused("out is a null pointer", f, F32, F32, 4, 100, A, B, C, None)
    refused("x is not aligned", f, F32, F32, 4, 100, A + 2, B, C, D)
    refused("gamma is not aligned", f, F32, F32, 4, 100, A, B + 1, C, D)
    refused("row stride of x", f, F32, F32, 4, 100, A, B, C, D, x_row_stride=99)
    refused("row stride of out", f, F32, F32, 4, 100, A, B, C, D, out_row_stride=-100)
    refused("overlaps x", f, F32, F32, 4, 100, A, B, C, A + 400)
    refused("overlaps x", f, F32, F32, 4, 100, A, B, C, A, x_row_stride=100, out_row_stride=104)
    accepted(f, F32, F32, 4, 100, A, None, None, A + 400, x_row_stride=200, out_row_stride=200)      # two halves of one matrix
    accepted(f, F32, F32, 4, 100, A + 400, None, None, A, x_row_stride=200, out_row_stride=200)
    refused("overlaps x", f, F32, F32, 4, 100, A, None, None, A + 396, x_row_stride=200, out_row_stride=200)
    refused("overlaps the weights", f, F32, F32, 4, 100, A, D + 400, C, D)


def test_layer_norm_backward(lib):
    f = lib.layer_norm_backward
    accepted(f, F32, F32, 4, 100, A, B, None, C, D, D + 400)
    accepted(f, F32, F32, 4, 100, A, B, None, A, D, None)
    accepted(f, F32, F32, 4, 100, A, B, None, B, None, None)
    refused("no gradient", f, F32, F32, 4, 100, A, B, None, None, None, None)
    refused("overlaps dbeta", f, F32, F32, 4, 100, A, B, None, C, D, D + 396)
    refused("overlaps the weight", f, F32, F32, 4, 100, A, B, D, C, D, None)
    refused("dx overlaps dy", f, F32, F32, 4, 100, A, B, None, A + 4, D, None)
    refused("dx overlaps x", f, F32, F32, 4, 100, A, B, None, B + 400, D, None)
    refused("overlaps dy or x", f, F32, F32, 4, 100, A, B, None, C, A + 800, None)
    refused("dx overlaps a weight", f, F32, F32, 4, 100, A, B, None, C, C + 400, None)
    refused("dy is a null pointer", f, F32, F32, 4, 100, None, B, None, C, D, None)
    need = lib.layer_norm_backward_workspace(F32, 4, 100)
    for at, name in ((A + 1584, "dy"), (B, "x"), (C - need + 16, "dx"), (D + 384, "a weight"), (D + 784, "a weight")):
        refused("the workspace overlaps " + name, f, F32, F32, 4, 100, A, B, None, C, D, D + 400, workspace=Space(at, need))
    accepted(f, F32, F32, 4, 100, A, B, None, C, D, D + 400, workspace=Space(A + 1600, need))
    assert lib.layer_norm_backward_workspace(F32, 0, 100) == 0
    assert lib.layer_norm_backward_workspace(F32, 4, 100) > 0


def test_token_logprobs(lib):
    f = lib.token_logprobs
    accepted(f, F32, 4, 100, A, B, C, C + 64, C + 128)
    accepted(f, BF16, 4, 100, A, None, None, C, None)
    accepted(f, F32, 4, 100, A, B, C, None, None, top=32, top_logprobs=D, top_tokens=D + 4096)
    accepted(f, F32, 0, 100, None, None, C, C, C)
    refused("dtype must be", f, I32, 4, 100, A, B, C, C + 64, C + 128)
    refused("vocab", f, F32, 4, 0, A, B, C, C + 64, C + 128)
    refused("below 2^31", f, F32, 1, 1 << 31, A, B, C, C + 64, C + 128)
    refused("top must lie", f, F32, 4, 100, A, B, C, None, None, top=33, top_logprobs=D, top_tokens=D + 4096)
    refused("top must lie", f, F32, 4, 10, A, B, C, None, None, top=11, top_logprobs=D, top_tokens=D + 4096)
    refused("top must lie", f, F32, 4, 10, A, B, C, None, None, top=-1)
    refused("need top_logprobs", f, F32, 4, 100, A, B, C, None, None, top=3)
    refused("no result", f, F32, 4, 100, A, B, None, None, None)
    refused("logprob needs tokens", f, F32, 4, 100, A, None, C, None, None)
    refused("logits is a null pointer", f, F32, 4, 100, None, B, C, None, None)
    refused("row stride", f, F32, 4, 100, A, B, C, None, None, row_stride=50)
    refused("entropy overlaps logprob", f, F32, 4, 100, A, B, C, C + 12, None)
    refused("logprob overlaps logits", f, F32, 4, 100, A, B, A + 1596, None, None)
    refused("lse overlaps tokens", f, F32, 4, 100, A, B, C, None, B + 8)
    refused("lse is not aligned", f, F64, 4, 100, A, B, C, None, C + 68)


def test_token_logprobs_backward(lib):
    f = lib.token_logprobs_backward
    accepted(f, F32, 4, 100, A, B, C, C + 64, C + 128, C + 192, D)
    accepted(f, F32, 4, 100, A, B, C, None, C + 128, None, A)
    accepted(f, F32, 4, 100, A, None, C, C + 64, None, C + 192, D)
    refused("lse is a null pointer", f, F32, 4, 100, A, B, None, C, C, None, D)
    refused("neither", f, F32, 4, 100, A, B, C, C + 64, None, None, D)
    refused("needs tokens", f, F32, 4, 100, A, None, C, None, C + 64, None, D)
    refused("needs entropy", f, F32, 4, 100, A, B, C, None, C + 64, C + 128, D)
    refused("overlaps logits", f, F32, 4, 100, A, B, C, None, C + 64, None, A + 4)
    refused("dlogits overlaps lse", f, F32, 4, 100, A, B, D + 16, None, C + 64, None, D)
    refused("dlogits is a null pointer", f, F32, 4, 100, A, B, C, None, C + 64, None, None)


def test_lists(lib):
    ok = ([F32, BF16], [100, 50], [A, B])
    accepted(lib.sum_squares, *ok, C)
    accepted(lib.global_norm, *ok, C)
    accepted(lib.global_norm, [], [], [], C)
    accepted(lib.clip_by_global_norm, *ok, [A, D], 1.0, C)
    accepted(lib.scale_to_norm, *ok, [A, B], C, 1.0)
    accepted(lib.global_norm, [F32, F32], [100, 100], [A, A], C)                       # read twice, written nowhere
    accepted(lib.clip_by_global_norm, [F32, F32], [0, 10], [None, A], [None, A], 1.0, C)
    refused("dtype must be", lib.global_norm, [I32], [10], [A], C)
    refused("out of range", lib.global_norm, [F32], [-1], [A], C)
    refused("null pointer", lib.global_norm, [F32], [10], [None], C)
    refused("not aligned", lib.global_norm, [F32], [10], [A + 2], C)
    refused("norm is f32 or f64", lib.global_norm, *ok, C, norm_dtype=BF16)
    refused("norm is a null pointer", lib.global_norm, *ok, None)
    refused("norm overlaps tensor 1", lib.global_norm, *ok, B + 96)
    refused("norm is not aligned", lib.sum_squares, *ok, C + 4)
    for bad in (0.0, -1.0, float("nan")):
        refused("max_norm", lib.clip_by_global_norm, *ok, [A, B], bad, C)
        refused("max_norm", lib.scale_to_norm, *ok, [A, B], C, bad)
    # the same tensor twice, and tensors that share elements, where one of them is written
    need = lib.global_norm_workspace(1)
    refused("the workspace overlaps tensor 0", lib.global_norm, [F32], [100], [A], C, workspace=Space(A + 384, need))
    refused("the workspace overlaps the result", lib.global_norm, [F32], [100], [A], C, workspace=Space(C, need))
    refused("the workspace overlaps tensor 0", lib.clip_by_global_norm, [F32], [100], [A], [B], 1.0, C, workspace=Space(B - need + 16, need))
    accepted(lib.clip_by_global_norm, [F32], [100], [A], [B], 1.0, C, workspace=Space(D, need))
    refused("overlaps another", lib.clip_by_global_norm, [F32, F32], [100, 100], [A, A], [A, A], 1.0, C)
    refused("overlaps another", lib.clip_by_global_norm, [F32, F32], [100, 100], [A, A], [A, D], 1.0, C)
    refused("overlaps another", lib.clip_by_global_norm, [F32, F32], [100, 100], [A, B], [D, D + 396], 1.0, C)
    refused("overlaps another", lib.clip_by_global_norm, [F32], [100], [A], [A + 4], 1.0, C)
    accepted(lib.clip_by_global_norm, [F32, F32], [100, 100], [A, A], [B, D], 1.0, C)
    with pytest.raises(ValueError):
        lib.global_norm([F32], [1, 2], [A, B], C, device=-1)


def test_a_workspace_that_is_not_needed_is_not_looked_at(lib):
    """The gradient of the rows alone hands nothing from launch to launch."""
    f = lib.layer_norm_backward
    need = lib.layer_norm_backward_workspace(F32, 4, 100)
    accepted(f, F32, F32, 4, 100, A, B, None, C, None, None, workspace=Space(A, need))
    refused("the workspace overlaps dy", f, F32, F32, 4, 100, A, B, None, C, D, None, workspace=Space(A, need))
    refused("the workspace overlaps dy", f, F32, F32, 4, 100, A, B, None, C, None, D, workspace=Space(A, need))
