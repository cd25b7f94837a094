"""The global norm of a list of tensors and clipping to it, through the C ABI, against fp64.

The squares are summed in fp64: the norm is off by half a step of its type (plus n 2^-53).  The factor is rounded to fp32 and the
product to the tensor's type: 2^-24 twice and half a step."""
import ctypes

import numpy as np
import pytest
import torch

from dali_b200.capi import BF16, DaliB200Error, F32, F64

pytestmark = pytest.mark.gpu

TORCH = {F32: torch.float32, F64: torch.float64, BF16: torch.bfloat16}
HALF_STEP = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -8}


def tensors_of(rng, spec):
    return [torch.from_numpy(rng.standard_normal(n)).cuda().to(TORCH[dt]) for n, dt in spec]


def norm_of(tensors):
    return float(np.sqrt(sum(float((t.double() ** 2).sum()) for t in tensors)))


def call(lib, spec, tensors, outs, limit, **kw):
    norm = torch.full((), -1.0, device="cuda", dtype=torch.float32)
    lib.clip_by_global_norm([d for _, d in spec], [n for n, _ in spec], tensors, outs, limit, norm, **kw)
    return norm


def check(spec, before, outs, limit, norm):
    want = norm_of(before)
    assert abs(norm.item() - want) <= want * (2.0 ** -24 + 1e-12)
    f = min(1.0, limit / want) if want > 0 else 1.0
    for (n, dt), b, o in zip(spec, before, outs):
        w = b.double() * f
        if f == 1.0:
            assert torch.equal(o, b)
        else:
            off = (o.double() - w).abs() - w.abs() * (HALF_STEP[dt] + (2 * 2.0 ** -24 if dt != F64 else 2.0 ** -50)) * 1.01 - torch.finfo(TORCH[dt]).tiny
            assert off.numel() == 0 or off.max().item() <= 0


SPECS = [
    [(1, F32)],
    [(1, BF16)],
    [(5, F32), (0, F32), (1000, BF16), (3, F64), (0, BF16), (1025, F32)],
    [(16384, F32), (16385, F32), (16383, BF16), (40000, BF16)],
    [(1000003, BF16)],
    [(3000001, F32), (7, F32)],
    [(100 + 13 * i, (F32, BF16, F64)[i % 3]) for i in range(97)],
    [(1 + i % 5, BF16) for i in range(400)],
]


@pytest.mark.parametrize("limit", [0.25, 1e30])
@pytest.mark.parametrize("spec", SPECS, ids=[str(i) for i in range(len(SPECS))])
def test_clip(lib, spec, limit):
    rng = np.random.default_rng(len(spec))
    tensors = tensors_of(rng, spec)
    outs = [torch.full_like(t, 5.0) for t in tensors]
    norm = call(lib, spec, tensors, outs, limit)
    check(spec, tensors, outs, limit, norm)
    # in place, and some of the list in place: the same bits
    mine = [t.clone() for t in tensors]
    call(lib, spec, mine, mine, limit)
    assert all(torch.equal(a, b) for a, b in zip(mine, outs))
    mine = [t.clone() for t in tensors]
    mixed = [m if i % 2 else torch.empty_like(m) for i, m in enumerate(mine)]
    call(lib, spec, mine, mixed, limit)
    assert all(torch.equal(a, b) for a, b in zip(mixed, outs))


def test_norm_and_sum_of_squares_alone(lib):
    rng = np.random.default_rng(0)
    for spec in SPECS:
        tensors = tensors_of(rng, spec)
        want = norm_of(tensors)
        d, n = [x for _, x in spec], [x for x, _ in spec]
        for dt in (F32, F64):
            norm = torch.full((), -1.0, device="cuda", dtype=TORCH[dt])
            lib.global_norm(d, n, tensors, norm, norm_dtype=dt)
            assert abs(norm.item() - want) <= want * (HALF_STEP[dt] + 1e-12)
        s = torch.full((), -1.0, device="cuda", dtype=torch.float64)
        lib.sum_squares(d, n, tensors, s)
        assert abs(s.item() - want * want) <= 1e-12 * want * want
        outs = [torch.empty_like(t) for t in tensors]
        lib.scale_to_norm(d, n, tensors, outs, s, 0.5)
        norm = torch.tensor(want, device="cuda")
        check(spec, tensors, outs, 0.5, norm)


def test_an_empty_list(lib):
    norm = torch.full((), -1.0, device="cuda")
    lib.clip_by_global_norm([], [], [], [], 1.0, norm)
    assert norm.item() == 0
    norm.fill_(-1)
    lib.global_norm([F32], [0], [torch.empty(0, device="cuda")], norm)
    assert norm.item() == 0


def test_zeros_stay_zeros(lib):
    t = torch.zeros(100000, device="cuda")
    norm = call(lib, [(100000, F32)], [t], [t], 1.0)
    assert norm.item() == 0 and (t == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_norm_that_is_not_finite_scales_nothing(lib, bad):
    t = [torch.full((70000,), 3.0, device="cuda"), torch.full((50,), 2.0, device="cuda", dtype=torch.bfloat16)]
    t[0][69999] = bad
    outs = [torch.empty_like(x) for x in t]
    norm = call(lib, [(70000, F32), (50, BF16)], t, outs, 1.0)
    assert not np.isfinite(norm.item())
    assert torch.equal(outs[0].nan_to_num(7.5), t[0].nan_to_num(7.5)) and torch.equal(outs[1], t[1])


def test_large_and_small_values_neither_overflow_nor_vanish(lib):
    """Squares that fp32 cannot hold."""
    for scale in (1e30, 1e-30):
        t = torch.full((4096,), scale, device="cuda")
        out = torch.empty_like(t)
        norm = call(lib, [(4096, F32)], [t], [out], scale)
        assert abs(norm.item() / (64 * scale) - 1) < 1e-6
        assert abs(out[17].item() / (scale / 64) - 1) < 1e-6


@pytest.mark.parametrize("dt", [F32, BF16, F64])
def test_offsets_from_the_16_byte_grid(lib, dt):
    rng = np.random.default_rng(2)
    for shift_in in range(0, 9, 3):
        for shift_out in range(0, 9, 3):
            n = 50021
            a = torch.from_numpy(rng.standard_normal(n + 20)).cuda().to(TORCH[dt])
            b = torch.full_like(a, 5.0)
            t, o = a[shift_in:shift_in + n], b[shift_out:shift_out + n]
            norm = call(lib, [(n, dt)], [t], [o], 0.125)
            check([(n, dt)], [t], [o], 0.125, norm)
            assert (b[:shift_out] == 5.0).all() and (b[shift_out + n:] == 5.0).all()


def test_the_same_call_gives_the_same_bits(lib):
    rng = np.random.default_rng(3)
    spec = [(300007, F32), (1000, BF16), (5000000, BF16)]
    t = tensors_of(rng, spec)
    seen = []
    for _ in range(3):
        outs = [torch.empty_like(x) for x in t]
        norm = call(lib, spec, t, outs, 1.0)
        seen.append([norm] + outs)
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


def test_threads_that_share_a_stream_and_the_library_space(lib):
    import threading
    rng = np.random.default_rng(9)
    specs = [[(300001, F32), (5, BF16)], [(4000000, BF16)], [(1000 + i, F32) for i in range(150)], [(70, F64)]]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    tensors = [tensors_of(rng, s) for s in specs]
    want = [norm_of(t) for t in tensors]
    norms = [torch.zeros((), device="cuda") for _ in specs]
    torch.cuda.synchronize()
    wrong = []

    def loop(k):
        d, n = [x for _, x in specs[k]], [x for x, _ in specs[k]]
        for _ in range(30):
            lib.global_norm(d, n, tensors[k], norms[k], stream=streams[k // 2].cuda_stream)
            lib.sync(stream=streams[k // 2].cuda_stream)
            if abs(norms[k].item() - want[k]) > want[k] * (2.0 ** -24 + 1e-12):
                wrong.append((k, norms[k].item(), want[k]))
    threads = [threading.Thread(target=loop, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_streams_and_graphs(lib):
    rng = np.random.default_rng(4)
    spec = [(100003, F32), (77, BF16)] * 60
    t = tensors_of(rng, spec)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = [[torch.empty_like(x) for x in t] for _ in range(2)]
    d, n = [x for _, x in spec], [x for x, _ in spec]
    with torch.cuda.stream(s):
        norm = call(lib, spec, t, outs[0], 1.0, stream=s.cuda_stream)
    s.synchronize()
    check(spec, t, outs[0], 1.0, norm)
    graphs, norms = [], [torch.zeros((), device="cuda") for _ in range(2)]
    work = [torch.empty(lib.global_norm_workspace(len(spec)), device="cuda", dtype=torch.uint8) for _ in range(2)]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lib.clip_by_global_norm(d, n, t, outs[i], 1.0 + i, norms[i], workspace=work[i], stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for x in t:
        x.mul_(2)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i in range(2):
            check(spec, t, outs[i], 1.0 + i, norms[i])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(DaliB200Error, match="workspace"):
            lib.global_norm(d, n, t, norms[0], stream=torch.cuda.current_stream().cuda_stream)
    del graphs, g


def test_a_stream_that_lies_where_another_one_lay(lib):
    """Kernels of a destroyed stream may still be using what it was given: a new stream gets space of its own, whatever its address."""
    rt = torch.cuda.cudart()
    big, small = torch.full((1 << 26,), 0.5, device="cuda"), torch.full((1 << 10,), 2.0, device="cuda")
    torch.cuda.synchronize()
    norms = torch.zeros(8, 2, device="cuda")
    torch.cuda.synchronize()
    for i in range(8):
        for j, t in enumerate((big, small)):
            handle = ctypes.c_void_p()
            assert int(rt.cudaStreamCreate(ctypes.addressof(handle))) == 0
            lib.global_norm([F32], [t.numel()], [t], norms[i, j:], stream=handle.value)
            assert int(rt.cudaStreamDestroy(handle.value)) == 0
    torch.cuda.synchronize()
    assert (norms[:, 0] == 4096.0).all() and (norms[:, 1] == 64.0).all()


def test_more_than_2_to_the_31_elements(lib):
    n = (1 << 31) + 12345
    t = torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16)
    t[-1] = 300.0
    norm = call(lib, [(n, BF16)], [t], [t], 1.0)
    want = float(np.sqrt((n - 1) * 0.25 + 90000.0))
    assert abs(norm.item() - want) <= want * 2.0 ** -23
    f = torch.tensor([300.0 * np.float32(1.0 / want)], dtype=torch.float32).to(torch.bfloat16).item()
    assert t[-1].item() == f and t[0].item() == torch.tensor([0.5 / want], dtype=torch.float32).to(torch.bfloat16).item()


@pytest.mark.parametrize("dt,value", [(F32, 1e38), (BF16, 2.0 ** 126), (F64, 1e38), (F64, 1e150)])
def test_a_norm_that_its_type_cannot_hold_scales_nothing(lib, dt, value):
    """100 elements whose norm, 10 times an element, lies beyond fp32's range and inside fp64's: reported in fp32 it is infinity,
    and nothing is scaled; reported in fp64 it is a number, and the list is scaled to it."""
    spec = [(90, dt), (10, dt)]
    t = [torch.full((n,), value, device="cuda", dtype=TORCH[dt]) for n, _ in spec]
    outs = [torch.full_like(x, 5.0) for x in t]
    norm = call(lib, spec, t, outs, 2.0)
    assert norm.item() == float("inf") and all(torch.equal(o, x) for o, x in zip(outs, t))
    mine = [x.clone() for x in t]
    assert call(lib, spec, mine, mine, 2.0).item() == float("inf") and all(torch.equal(o, x) for o, x in zip(mine, t))
    norm = torch.zeros((), device="cuda", dtype=torch.float64)
    lib.clip_by_global_norm([dt, dt], [90, 10], t, outs, value, norm, norm_dtype=F64)
    assert abs(norm.item() / (10 * t[0][0].item()) - 1) < 1e-14           # (of the elements as they are stored)
    for o in outs:            # a tenth of value: the factor and the product rounded to fp32, the result to its type
        off = (HALF_STEP[dt] + (2 * 2.0 ** -24 if dt != F64 else 2.0 ** -50)) * 1.01
        assert ((o.double() / (value / 10) - 1).abs() <= off).all()


def test_a_norm_next_to_the_end_of_fp32(lib):
    """The largest norm that rounds to a number of fp32 still scales (to 16: the factor is no subnormal number)."""
    top = torch.finfo(torch.float32).max
    t = torch.tensor([top, 0.0], device="cuda")
    out = torch.empty_like(t)
    norm = call(lib, [(2, F32)], [t], [out], 16.0)
    assert norm.item() == top and abs(out[0].item() / 16 - 1) <= 3 * 2.0 ** -24 * 1.01
    t[1] = top / 2
    norm = call(lib, [(2, F32)], [t], [out], 16.0)
    assert norm.item() == float("inf") and torch.equal(out, t)


def test_space_of_many_streams_is_bounded(lib):
    """Nothing tells the library that a stream is gone: what it keeps for them stays within 512 MB, and a stream whose space went
    gets another one."""
    rt = torch.cuda.cudart()
    handles = [ctypes.c_void_p() for _ in range(200)]
    assert all(int(rt.cudaStreamCreate(ctypes.addressof(h))) == 0 for h in handles)
    t = torch.arange(1, 3, device="cuda", dtype=torch.float32)
    norms = torch.zeros(2, len(handles), device="cuda")
    lib.global_norm([F32], [2], [t], norms)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for again in range(2):
        for i, h in enumerate(handles):
            lib.global_norm([F32], [2], [t], norms[again, i:], stream=h.value)
    torch.cuda.synchronize()
    taken = free - torch.cuda.mem_get_info()[0]
    assert all(int(rt.cudaStreamDestroy(h.value)) == 0 for h in handles)
    assert (norms == torch.tensor(5.0).sqrt().item()).all()
    assert taken <= (512 + 64) << 20, taken
