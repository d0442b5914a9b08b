"""Embedding lookup and its gradient against 64-bit NumPy.

Lookup: one fp32 product rounded once to the table's type, so it equals NumPy's product bit for bit.
Gradient: a sum of n fp32 terms in any order is off by at most n * 2^-24 times the sum of their
magnitudes, the product with the scale by 2^-24 of itself once more.
"""
import numpy as np
import pytest

import novann_b200 as nb
from novann_b200 import _lib, functional as F
from novann_b200.device import DeviceBuffer, Stream, device_sync
from oracle import oracle_np as o

pytestmark = pytest.mark.gpu
NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def to_type(x, dtype):
    return o.f32_to_bf16_bits(x) if dtype == "bf16" else x.astype(NP[dtype])


def wide(a):
    return o.bf16_bits_to_f32(a) if a.dtype == np.uint16 else a.astype(np.float32)


def skewed_ids(rng, n, v):
    return np.minimum(np.exp(rng.random(n) * np.log(v + 1)) - 1, v - 1).astype(np.int32)


def want_grad(dout, ids, v, scale, pad=None):
    g = np.zeros((v, dout.shape[1]))
    mag = np.zeros_like(g)
    keep = np.ones(len(ids), bool) if pad is None else ids != pad
    x = wide(dout).astype(np.float64)
    np.add.at(g, ids[keep], x[keep])
    np.add.at(mag, ids[keep], np.abs(x[keep]))
    n = np.bincount(ids[keep], minlength=v)[:, None]
    return g * scale, (n * mag * abs(scale) + np.abs(g * scale)) * 2.0 ** -24


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,v,d", [(1, 1, 1), (1, 7, 64), (17, 1000, 64), (33, 5, 3), (100, 50, 1001), (65, 40, 2048),
                                   (20000, 300, 8), (9001, 17, 130), (40000, 9, 520)])
def test_lookup(gpu, dtype, t, v, d):
    rng = np.random.default_rng(t * 31 + d)
    table = to_type(rng.standard_normal((v, d)).astype(np.float32), dtype)
    ids = rng.integers(0, v, t)
    out = F.embedding_host(table, ids, scale=1.7, device=gpu)
    prod = wide(table)[ids] * np.float32(1.7)
    assert np.array_equal(out, to_type(prod, dtype))


def test_lookup_misaligned_rows_and_shapes(gpu):
    rng = np.random.default_rng(0)
    table = rng.standard_normal((11, 16)).astype(np.float16)
    ids = rng.integers(0, 11, (3, 5))
    assert F.embedding_host(table, ids, device=gpu).shape == (3, 5, 16)
    assert F.embedding_host(table, np.zeros((0, 4), np.int64), device=gpu).shape == (0, 4, 16)
    # buffers that start on an element, not on a packet
    d_t, d_i = DeviceBuffer(table.nbytes + 2, gpu), DeviceBuffer.from_numpy(ids.astype(np.int32), gpu)
    d_t.upload(table, offset=2)
    d_o = DeviceBuffer(15 * 16 * 2 + 2, gpu)
    L = _lib.lib()
    _lib.check(L.nvq_embedding_fwd(d_o.at(2), d_t.at(2), _lib.F16, d_i.at(0), 15, 11, 16, 1.0, gpu, None))
    got = np.empty((15, 16), np.float16)
    d_o.download(got, offset=2)
    assert np.array_equal(got, table[ids.ravel()])


def test_ids_out_of_range_are_reported_and_give_zeros(gpu):
    table = np.ones((4, 8), np.float32)
    ids = np.array([0, 4, -1, 3], np.int32)
    d_t, d_i, d_o = DeviceBuffer.from_numpy(table, gpu), DeviceBuffer.from_numpy(ids, gpu), DeviceBuffer(128, gpu)
    F.embedding_device(d_o, d_t, "f32", d_i, 4, 4, 8)
    device_sync(gpu)
    with pytest.raises(_lib.NvqError, match="71"):
        F.check_device_errors(gpu)
    F.check_device_errors(gpu)
    assert np.array_equal(d_o.to_numpy(np.float32, (4, 8)).sum(1), [8, 0, 0, 8])
    d_g, ws = DeviceBuffer(128, gpu), DeviceBuffer(F.embedding_bwd_workspace_bytes(4, 4, 8), gpu)
    F.embedding_bwd_device(d_g, d_t, "f32", d_i, 4, 4, 8, ws)
    device_sync(gpu)
    with pytest.raises(_lib.NvqError, match="71"):
        F.check_device_errors(gpu)
    assert np.array_equal(d_g.to_numpy(np.float32, (4, 8)).sum(1), [8, 0, 0, 8])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,v,d", [(1, 1, 1), (1, 9, 5), (31, 3, 64), (32, 1, 8), (33, 1, 8), (64, 2, 12), (1000, 7, 40),
                                   (1024, 600, 33), (512, 3, 100), (513, 3, 100), (512, 300000, 7), (500, 400, 261), (1025, 511, 130), (4095, 512, 260), (4096, 200000, 9), (4097, 3, 30), (2000, 130, 1025), (20000, 70000, 4),
                                   (5000, 300, 1001), (131072, 1000, 2), (131073, 5, 3)])
def test_table_gradient(gpu, dtype, t, v, d):
    rng = np.random.default_rng(t * 7 + d)
    dout = to_type(rng.standard_normal((t, d)).astype(np.float32), dtype)
    ids = skewed_ids(rng, t, v)
    pad = int(ids[t // 2]) if t % 2 == 0 and v > 1 else None
    got = F.embedding_bwd_host(dout, ids, v, scale=0.37, padding_id=pad, device=gpu)
    want, tol = want_grad(dout, ids, v, float(np.float32(0.37)), pad)
    assert np.all(np.abs(got - want) <= tol)
    again = F.embedding_bwd_host(dout, ids, v, scale=0.37, padding_id=pad, device=gpu)
    assert np.array_equal(got.view(np.uint32), again.view(np.uint32))


@pytest.mark.parametrize("t", [500, 3000, 10000])
@pytest.mark.parametrize("case", ["one id", "sorted", "all padding", "last id"])
def test_table_gradient_extremes(gpu, case, t):
    v, d = 257, 72
    rng = np.random.default_rng(3)
    dout = rng.standard_normal((t, d)).astype(np.float32)
    ids = {"one id": np.full(t, 200), "sorted": np.sort(rng.integers(0, v, t)), "all padding": np.full(t, 5),
           "last id": np.where(np.arange(t) % 2, v - 1, 0)}[case].astype(np.int32)
    pad = 5 if case == "all padding" else None
    got = F.embedding_bwd_host(dout, ids, v, padding_id=pad, device=gpu)
    want, tol = want_grad(dout, ids, v, 1.0, pad)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("d", [3, 72, 261])
@pytest.mark.parametrize("first", [0, 31])
def test_runs_of_every_length_from_every_place(gpu, first, d):
    """Ids with 1, 2, ... 300 tokens: runs of the sorted tokens that begin and end anywhere, and some that cover whole
    blocks of them."""
    lengths = np.concatenate([np.ones(first, int), np.arange(1, 301)])
    rng = np.random.default_rng(first + d)
    ids = rng.permutation(np.repeat(np.arange(len(lengths)), lengths)).astype(np.int32)
    dout = rng.standard_normal((ids.size, d)).astype(np.float32)
    got = F.embedding_bwd_host(dout, ids, len(lengths) + 2, device=gpu)
    want, tol = want_grad(dout, ids, len(lengths) + 2, 1.0, None)
    assert np.all(np.abs(got - want) <= tol)


def test_padding_rows_may_hold_anything_and_infinities_stay_in_their_row(gpu):
    dout = np.ones((6, 16), np.float32)
    ids = np.array([0, 3, 1, 3, 2, 1], np.int32)
    dout[[1, 3]] = np.nan                    # padded tokens
    dout[4] = np.inf
    got = F.embedding_bwd_host(dout, ids, 5, padding_id=3, device=gpu)
    assert np.array_equal(got[:, 0], [1, 2, np.inf, 0, 0])


def test_accumulates_onto_a_table_gradient(gpu):
    rng = np.random.default_rng(5)
    t, v, d = 140000, 40, 12                  # two sorted parts
    dout, ids = rng.standard_normal((t, d)).astype(np.float32), rng.integers(0, v - 1, t).astype(np.int32)
    start = rng.standard_normal((v, d)).astype(np.float32)
    d_g, d_o = DeviceBuffer.from_numpy(start, gpu), DeviceBuffer.from_numpy(dout, gpu)
    d_i, ws = DeviceBuffer.from_numpy(ids, gpu), DeviceBuffer(F.embedding_bwd_workspace_bytes(t, v, d), gpu)
    F.embedding_bwd_device(d_g, d_o, "f32", d_i, t, v, d, ws, accumulate=True)
    got = d_g.to_numpy(np.float32, (v, d))
    want, tol = want_grad(dout, ids, v, 1.0)
    assert np.all(np.abs(got - (want + start)) <= tol + (np.abs(start) + np.abs(want + start)) * 2.0 ** -23)
    assert np.array_equal(got[v - 1], start[v - 1])       # a row without tokens is left as it was


def test_gradient_is_the_derivative_of_the_lookup(gpu):
    rng = np.random.default_rng(7)
    table, ids = rng.standard_normal((6, 5)).astype(np.float32), rng.integers(0, 6, 20)
    w = rng.standard_normal((20, 5)).astype(np.float32)
    g = F.embedding_bwd_host(w, ids, 6, scale=2.0, device=gpu)
    for v, c in [(0, 0), (3, 4), (5, 2)]:
        hi, lo = table.copy(), table.copy()
        hi[v, c] += 0.5
        lo[v, c] -= 0.5
        f = [np.sum(F.embedding_host(x, ids, 2.0, gpu).astype(np.float64) * w) for x in (hi, lo)]
        # linear in the table: the difference is the derivative up to the rounding of its operands
        assert abs((f[0] - f[1]) - g[v, c]) <= 20 * 2.0 ** -22 * np.abs(w).max() * 8


def test_layer_and_captured_replay(gpu):
    rng = np.random.default_rng(9)
    emb = nb.Embedding(50, 24, scale=3.0, padding_id=0, device=gpu)
    ids = rng.integers(0, 50, (4, 7))
    assert np.array_equal(emb(ids), emb.weight.data[ids] * np.float32(3))
    g = rng.standard_normal((4, 7, 24)).astype(np.float32)
    assert emb.backward(g) is None
    want, tol = want_grad(g.reshape(28, 24), ids.ravel().astype(np.int32), 50, 3.0, 0)
    assert np.all(np.abs(emb.weight.grad - want) <= tol) and not emb.weight.grad[0].any()
    with pytest.raises(IndexError):
        emb(np.array([50]))
    # two captured graphs on one workspace, replayed in turn with other ids
    t, v, d = 3000, 50, 24
    st = Stream(gpu)
    d_i, d_o = DeviceBuffer(t * 4, gpu), DeviceBuffer(t * d * 4, gpu)
    tabs = [DeviceBuffer(v * d * 4, gpu) for _ in range(2)]
    ws = DeviceBuffer(F.embedding_bwd_workspace_bytes(t, v, d), gpu)
    import ctypes as C
    graphs = []
    for i, tab in enumerate(tabs):
        _lib.check(_lib.lib().nvq_graph_begin_capture(gpu, C.c_void_p(st.ptr)))
        F.embedding_bwd_device(tab, d_o, "f32", d_i, t, v, d, ws, scale=i + 1.0, stream=st)
        h = C.c_void_p()
        _lib.check(_lib.lib().nvq_graph_end_capture(gpu, C.c_void_p(st.ptr), C.byref(h)))
        graphs.append(h)
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        ids, g = skewed_ids(rng, t, v), rng.standard_normal((t, d)).astype(np.float32)
        d_i.upload(ids, st)
        d_o.upload(g, st)
        for h in graphs:
            _lib.check(_lib.lib().nvq_graph_launch(gpu, h, C.c_void_p(st.ptr)))
        st.sync()
        for i, tab in enumerate(tabs):
            want, tol = want_grad(g, ids, v, i + 1.0)
            assert np.all(np.abs(tab.to_numpy(np.float32, (v, d)) - want) <= tol)
    for h in graphs:
        _lib.lib().nvq_graph_destroy(gpu, h)
