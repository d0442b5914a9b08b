"""Gradient norm and clipping against 64-bit NumPy.

The squares are added in fp64, so the norm is off by its rounding to fp32 (2^-24) and the coefficient
by at most 2^-24 more; a clipped value carries the coefficient's rounding, the product's and, for
16-bit types, the type's half step.
"""
import ctypes as C

import numpy as np
import pytest

import novann_b200 as nb
from novann_b200 import _lib, functional as F
from novann_b200.device import DeviceBuffer, Stream
from novann_b200.module import Parameters
from novann_b200.train import MLPTrainStep
from oracle import oracle_np as o

pytestmark = pytest.mark.gpu
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f64": 2.0 ** -53}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "f64": 8}
NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "f64": np.float64}


def to_type(x, dtype):
    return o.f32_to_bf16_bits(x.astype(np.float32)) if dtype == "bf16" else x.astype(NP[dtype])


def wide(a):
    return (o.bf16_bits_to_f32(a) if a.dtype == np.uint16 else a).astype(np.float64)


def run(gpu, arrays, dtypes, max_norm, in_place, offset=0, stream=None):
    bufs = []
    for a, dt in zip(arrays, dtypes):
        b = DeviceBuffer(a.nbytes + 16, gpu)
        b.upload(a, offset=offset * BYTES[dt])
        bufs.append(b)
    outs = bufs if in_place else [DeviceBuffer(a.nbytes + 16, gpu) for a in arrays]
    norm, ws = DeviceBuffer(8, gpu), DeviceBuffer(F.grad_norm_workspace_bytes(), gpu)
    view = [_shift(b, offset * BYTES[dt]) for b, dt in zip(bufs, dtypes)]
    out = None if in_place else [_shift(b, offset * BYTES[dt]) for b, dt in zip(outs, dtypes)]
    F.clip_grads_device(norm, view, [a.size for a in arrays], dtypes, max_norm, ws, out=out, stream=stream)
    got = []
    for b, a, dt in zip(outs, arrays, dtypes):
        x = np.empty(a.shape, a.dtype)
        b.download(x, offset=offset * BYTES[dt])
        got.append(x)
    return norm.to_numpy(np.float32, (2,)), got


def _shift(buf, by):
    from novann_b200.device import DeviceView
    return DeviceView(buf.ptr + by, buf.nbytes - by, buf.device)


def check(arrays, dtypes, max_norm, head, got):
    want = np.sqrt(sum(np.sum(wide(a) ** 2) for a in arrays))
    assert abs(head[0] - want) <= want * 2.0 ** -23
    coef = 1.0 if want <= max_norm else max_norm / want
    assert abs(head[1] - coef) <= coef * 2.0 ** -23
    for a, g, dt in zip(arrays, got, dtypes):
        w = wide(a) * coef
        # 2^-14 * 2^-11 (2^-25): half a step of fp16 below its normal range
        tol = np.abs(w) * (HALF[dt] + 2.0 ** -23) + (2.0 ** -25 if dt == "f16" else 0.0)
        assert np.all(np.abs(wide(g) - w) <= tol)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "f64"])
@pytest.mark.parametrize("counts", [[1], [4095], [4096], [4097], [8191, 8192, 8193], [16384, 16385], [1, 2, 3, 70000], [0, 5, 0], [12345] * 5])
def test_clip_one_type(gpu, in_place, dtype, counts):
    rng = np.random.default_rng(sum(counts))
    arrays = [to_type(rng.standard_normal(n), dtype) for n in counts]
    for max_norm in (0.25, 1e9):
        head, got = run(gpu, arrays, [dtype] * len(counts), max_norm, in_place)
        check(arrays, [dtype] * len(counts), max_norm, head, got)
        if max_norm == 1e9:
            assert all(np.array_equal(a, g) for a, g in zip(arrays, got))


@pytest.mark.parametrize("offset", [0, 1])
def test_clip_mixed_types_and_many_tensors(gpu, offset):
    rng = np.random.default_rng(11)
    dtypes = [["f32", "f16", "bf16", "f64"][i % 4] for i in range(1203)]      # more than one list of tensors
    arrays = [to_type(rng.standard_normal(int(n)) * 0.1, dt) for n, dt in zip(rng.integers(0, 300, 1203), dtypes)]
    arrays[7] = to_type(rng.standard_normal(50001), dtypes[7])
    head, got = run(gpu, arrays, dtypes, 3.0, False, offset)
    check(arrays, dtypes, 3.0, head, got)
    head2, got2 = run(gpu, arrays, dtypes, 3.0, True, offset)
    assert np.array_equal(head.view(np.uint32), head2.view(np.uint32))
    assert all(np.array_equal(a, b) for a, b in zip(got, got2))


def test_large_and_small_values_neither_overflow_nor_vanish(gpu):
    for size in (1e30, 1e-30):
        a = np.full(1000, size, np.float32)
        head, got = run(gpu, [a], ["f32"], size, False)
        assert abs(head[0] / (np.sqrt(1000) * size) - 1) < 1e-6
        assert np.allclose(np.linalg.norm(got[0].astype(np.float64)), size, rtol=1e-6)


def test_nan_inf_zero_and_empty(gpu):
    a = np.ones(100, np.float32)
    a[3] = np.nan
    head, got = run(gpu, [a, np.ones(5, np.float32)], ["f32", "f32"], 1.0, True)
    assert np.isnan(head).all() and np.isnan(got[0]).all() and np.isnan(got[1]).all()
    a[3] = np.inf
    head, got = run(gpu, [a], ["f32"], 1.0, True)
    assert np.isinf(head[0]) and head[1] == 0 and np.isnan(got[0][3]) and not got[0][:3].any()
    head, got = run(gpu, [np.zeros(9, np.float32)], ["f32"], 1.0, False)
    assert head[0] == 0 and head[1] == 1 and not got[0].any()
    norm, ws = DeviceBuffer(8, gpu), DeviceBuffer(F.grad_norm_workspace_bytes(), gpu)
    F.clip_grads_device(norm, [], [], "f32", 1.0, ws)
    assert np.array_equal(norm.to_numpy(np.float32, (2,)), [0, 1])


def test_norm_only_leaves_gradients(gpu):
    rng = np.random.default_rng(2)
    a = [rng.standard_normal(n).astype(np.float32) for n in (300000, 17)]
    bufs = [DeviceBuffer.from_numpy(x, gpu) for x in a]
    norm, ws = DeviceBuffer(8, gpu), DeviceBuffer(F.grad_norm_workspace_bytes(), gpu)
    F.grad_norm_device(norm, bufs, [x.size for x in a], "f32", ws, max_norm=10.0)
    check(a, ["f32"] * 2, 10.0, norm.to_numpy(np.float32, (2,)), [x * np.float32(10 / np.sqrt(sum(
        np.sum(y.astype(np.float64) ** 2) for y in a))) for x in a])
    assert all(np.array_equal(b.to_numpy(np.float32, x.shape), x) for b, x in zip(bufs, a))


def test_sgd_clips_like_the_definition(gpu):
    rng = np.random.default_rng(4)
    params = [Parameters(rng.standard_normal(s).astype(np.float32)) for s in ((5, 7), (1, 7))]
    grads = [rng.standard_normal(p.data.shape).astype(np.float32) * 10 for p in params]
    before = [p.data.copy() for p in params]
    for p, g in zip(params, grads):
        p.grad = g.copy()
    nb.SGD(params + params[:1], lr=0.0, max_grad_norm=1.0, device=gpu).step()     # a tied parameter counts once
    norm = np.sqrt(sum(np.sum(g.astype(np.float64) ** 2) for g in grads))
    for p, g, b in zip(params, grads, before):
        assert np.allclose(p.grad, g / norm, rtol=2.0 ** -21, atol=0)
        assert np.array_equal(p.data, b)
    nb.SGD(params, lr=0.5, max_grad_norm=100.0, device=gpu).step()
    for p, g, b in zip(params, grads, before):
        assert np.allclose(p.data, b - 0.5 * g / norm, rtol=0, atol=2.0 ** -21 * np.abs(b).max() * 2)


def test_mlp_step_clips_eager_and_replayed(gpu):
    rng = np.random.default_rng(6)
    dims = [20, 16, 10]
    params = []
    for fi, fo in zip(dims[:-1], dims[1:]):
        params += [rng.standard_normal((fo, fi)).astype(np.float32), np.zeros((1, fo), np.float32)]
    x, y = rng.random((32, 20)).astype(np.float32), rng.integers(0, 10, 32).astype(np.int32)
    free = MLPTrainStep(params, 32, 0.1, device=gpu)
    free.step(x, y)
    raw = free.grads()
    norm = np.sqrt(sum(np.sum(g.astype(np.float64) ** 2) for g in raw))
    limit = float(norm) / 3
    cut = MLPTrainStep(params, 32, 0.1, device=gpu, max_grad_norm=limit)
    cut.step(x, y)
    assert abs(cut.grad_norm() / norm - 1) <= 2.0 ** -23
    for p, q, r, g in zip(params, cut.params(), raw, cut.grads()):
        assert np.allclose(g, r / 3, rtol=2.0 ** -21, atol=0)
        assert np.array_equal(q, p.reshape(q.shape) - np.float32(0.1) * g.reshape(q.shape))
    again = MLPTrainStep(params, 32, 0.1, device=gpu, max_grad_norm=limit)
    again.step(x, y)
    again.capture()
    again.step(x, y)
    cut.step(x, y)
    assert all(np.array_equal(a, b) for a, b in zip(again.params(), cut.params()))
    assert again.grad_norm() == cut.grad_norm()


def test_on_a_side_stream_and_twice_the_same(gpu):
    rng = np.random.default_rng(8)
    a = [rng.standard_normal(1 << 20).astype(np.float32)]
    st = Stream(gpu)
    first = None
    for _ in range(3):
        b = DeviceBuffer.from_numpy(a[0], gpu)
        norm, ws = DeviceBuffer(8, gpu), DeviceBuffer(F.grad_norm_workspace_bytes(), gpu)
        F.clip_grads_device(norm, [b], [a[0].size], "f32", 0.5, ws, stream=st)
        st.sync()
        out = b.to_numpy(np.float32, a[0].shape)
        first = out if first is None else first
        assert np.array_equal(first, out)
    check(a, ["f32"], 0.5, norm.to_numpy(np.float32, (2,)), [out])
