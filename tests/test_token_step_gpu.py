"""The token-model operators together, as a training step uses them: lookup, loss head, both gradients into
one tied table, clipping, SGD - device resident, captured and replayed - and the layers on host arrays.

The bounds follow the gradients': a value of g is off by the operands' half step (2^-8 for bf16), the sums'
roundings by n * 2^-23 of the magnitudes that were added; the norm is off by at most the norm of all errors.
"""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

import novann_b200 as nb
from novann_b200 import _lib, functional as F, quant
from novann_b200.device import DeviceBuffer, Stream
from oracle import oracle_np as o

pytestmark = pytest.mark.gpu
H = 2.0 ** -8


def bf16(x):
    return o.bf16_bits_to_f32(o.f32_to_bf16_bits(x.astype(np.float32))).astype(np.float64)


def tied_gradient(table, ids, labels, scale, pad):
    """Gradient of the mean loss by the tied table (through lookup and head) and its bound."""
    v, k = table.shape
    e = bf16(table)
    x = bf16((e[ids] * scale).astype(np.float32))
    z = x @ e.T
    z -= z.max(1, keepdims=True)
    p = np.exp(z) / np.exp(z).sum(1, keepdims=True)
    live = labels != -100
    g = p * live[:, None]
    g[np.arange(len(ids))[live], labels[live]] -= 1.0
    g /= max(1, live.sum())
    # 2^-12 of a probability: logits of at most 32, each off by (k + 2) * 2^-23 * 32 with k = 64
    dg = np.abs(g) * H + p * 2.0 ** -12 / max(1, live.sum())
    dx, ddx = g @ e, dg @ np.abs(e) + v * 2.0 ** -23 * (np.abs(g) @ np.abs(e))
    dw, ddw = g.T @ x, dg.T @ np.abs(x) + len(ids) * 2.0 ** -23 * (np.abs(g).T @ np.abs(x))
    keep = ids != pad
    for t in np.flatnonzero(keep):
        dw[ids[t]] += scale * dx[t]
        ddw[ids[t]] += abs(scale) * (ddx[t] + len(ids) * 2.0 ** -23 * np.abs(dx[t]))
    return dw, ddw


def sgd_step(table, ids, labels, scale, pad, lr, limit):
    g, dg = tied_gradient(table, ids, labels, scale, pad)
    norm, off = np.linalg.norm(g), np.linalg.norm(dg)
    coef = min(1.0, limit / norm)
    cut = g * coef
    tol = dg * coef + np.abs(cut) * (off / norm + 2.0 ** -21)
    return table - lr * cut, lr * tol + np.abs(table) * 2.0 ** -23, norm, off


def test_device_step_eager_and_captured(gpu):
    t, v, k, scale, pad, lr, limit = 300, 700, 64, 4.0, 3, 0.5, 0.25
    rng = np.random.default_rng(0)
    table = (rng.standard_normal((v, k)) / np.sqrt(k)).astype(np.float32)
    st = Stream(gpu)
    master, grad = DeviceBuffer.from_numpy(table, gpu), DeviceBuffer(v * k * 4, gpu)
    low, x = DeviceBuffer(v * k * 2, gpu), DeviceBuffer(t * k * 2, gpu)
    d_ids, d_labels, dx = DeviceBuffer(t * 4, gpu), DeviceBuffer(t * 4, gpu), DeviceBuffer(t * k * 4, gpu)
    head, stats, norm = DeviceBuffer(8, gpu), DeviceBuffer(t * 8, gpu), DeviceBuffer(8, gpu)
    ws = DeviceBuffer(max(F.linear_ce_workspace_bytes(t, v, k), F.embedding_bwd_workspace_bytes(t, v, k),
                          F.grad_norm_workspace_bytes()), gpu)

    def step():
        quant.cast_device(low, "bf16", master, "f32", v * k, stream=st)
        F.embedding_device(x, low, "bf16", d_ids, t, v, k, scale=scale, stream=st)
        F.linear_ce_device(head, stats, x, low, "bf16", d_labels, t, v, k, ws, stream=st)
        F.linear_ce_bwd_device(dx, grad, x, low, "bf16", d_labels, stats, head, t, v, k, ws, stream=st)
        F.embedding_bwd_device(grad, dx, "f32", d_ids, t, v, k, ws, scale=scale, padding_id=pad, accumulate=True, stream=st)
        F.clip_grads_device(norm, [grad], [v * k], "f32", limit, ws, stream=st)
        _lib.check(_lib.lib().nvq_sgd_step_f32(master.at(0), grad.at(0), v * k, lr, 1.0, gpu, C.c_void_p(st.ptr)))

    graph = None
    for i in range(3):
        ids = rng.integers(0, v, t).astype(np.int32)
        ids[-40:] = pad
        labels = rng.integers(0, v, t).astype(np.int32)
        labels[-40:] = -100
        d_ids.upload(ids, st)
        d_labels.upload(labels, st)
        st.sync()
        before = master.to_numpy(np.float32, (v, k))
        if graph is None:
            step()
        else:
            _lib.check(_lib.lib().nvq_graph_launch(gpu, graph, C.c_void_p(st.ptr)))
        st.sync()
        F.check_device_errors(gpu)
        want, tol, n, off = sgd_step(before.astype(np.float64), ids, labels, scale, pad, lr, limit)
        assert np.all(np.abs(master.to_numpy(np.float32, (v, k)) - want) <= tol)
        got = norm.to_numpy(np.float32, (2,))
        assert abs(got[0] - n) <= off + n * 2.0 ** -23 and got[1] < 1
        if graph is None:
            _lib.check(_lib.lib().nvq_graph_begin_capture(gpu, C.c_void_p(st.ptr)))
            step()
            graph = C.c_void_p()
            _lib.check(_lib.lib().nvq_graph_end_capture(gpu, C.c_void_p(st.ptr), C.byref(graph)))
    _lib.lib().nvq_graph_destroy(gpu, graph)


def test_layers_on_host_arrays(gpu):
    rng = np.random.default_rng(1)
    t, v, k = 50, 90, 32
    emb = nb.Embedding(v, k, scale=2.0, padding_id=0, device=gpu)
    mid = nb.Sequential(nb.Linear(k, k, device=gpu), nb.ReLU(device=gpu))
    head = nb.LinearCrossEntropyLoss(k, v, device=gpu)
    for p in emb.parameters() + mid.parameters() + head.parameters():
        p.data = (rng.standard_normal(p.data.shape) / 4).astype(np.float32)
    params = emb.parameters() + mid.parameters() + head.parameters()
    opt = nb.SGD(params, 0.1, max_grad_norm=0.5, device=gpu)
    ids, labels = rng.integers(0, v, (5, 10)), rng.integers(0, v, t)
    x = emb(ids)
    loss, dx = head(mid(x.reshape(t, k)), labels)
    assert emb.backward(mid.backward(dx).reshape(5, 10, k)) is None
    # the same in 64 bits
    e, w1, b1, w2, b2 = (p.data.astype(np.float64) for p in params)
    xe = e[ids.ravel()] * 2.0
    pre = xe @ w1.T + b1
    h, w2b = bf16(np.maximum(pre, 0.0)), bf16(w2)
    z = h @ w2b.T + b2
    z -= z.max(1, keepdims=True)
    p = np.exp(z) / np.exp(z).sum(1, keepdims=True)
    g = p.copy()
    g[np.arange(t), labels] -= 1
    want = -np.log(p[np.arange(t), labels]).mean()
    # h may be rounded to the neighbouring bf16 value where its fp32 sum differs from the 64-bit one
    assert abs(loss - want) <= 2.0 ** -8 * np.abs(h @ w2b.T).max()
    g /= t
    dh = (g @ w2b) * (pre > 0)
    de = np.zeros_like(e)
    np.add.at(de, ids.ravel(), 2.0 * (dh @ w1))
    de[0] = 0
    # every factor carries at most 2^-7 (h and the weight rounded, g rounded), the sums of magnitudes bound the rest
    tol = np.zeros_like(e)
    np.add.at(tol, ids.ravel(), 2.0 * (((np.abs(g) + 2 * p / t) @ np.abs(w2b)) @ np.abs(w1)))
    assert np.all(np.abs(emb.weight.grad - de) <= tol * 2.0 ** -6)
    before = [q.data.copy() for q in params]
    grads = [q.grad.astype(np.float64) for q in params]
    opt.step()
    norm = np.sqrt(sum((q ** 2).sum() for q in grads))
    coef = min(1.0, 0.5 / norm)
    for q, b, gr in zip(params, before, grads):
        assert np.all(np.abs(q.data - (b - 0.1 * coef * gr)) <= (np.abs(b) + np.abs(gr)) * 2.0 ** -22)


def test_offsets_past_32_bits(gpu):
    """A table of 2.3 G elements, and a piece of the logits' gradient of 2.5 G."""
    v, d, t = 1_100_000, 2048, 64
    rng = np.random.default_rng(2)
    ids = np.concatenate([[0, v - 1, v - 1, v // 2], rng.integers(0, v, t - 4)]).astype(np.int32)
    rows = rng.standard_normal((v % 7 + 3, d)).astype(np.float32)
    table = DeviceBuffer(v * d * 4, gpu)
    table.zero()
    table.upload(rows[0], offset=(v - 1) * d * 4)
    d_ids, out = DeviceBuffer.from_numpy(ids, gpu), DeviceBuffer(t * d * 4 + 4, gpu)
    out.upload(np.array([7.0], np.float32), offset=t * d * 4)
    F.embedding_device(out, table, "f32", d_ids, t, v, d)
    got = out.to_numpy(np.float32, (t * d + 1,))
    assert got[-1] == 7.0                         # what lies behind the last row is left as it was
    got = got[:-1].reshape(t, d)
    assert np.array_equal(got[1], rows[0]) and np.array_equal(got[2], rows[0]) and not got[3].any()
    dout = rng.standard_normal((t, d)).astype(np.float32)
    ws = DeviceBuffer(F.embedding_bwd_workspace_bytes(t, v, d), gpu)
    F.embedding_bwd_device(table, DeviceBuffer.from_numpy(dout, gpu), "f32", d_ids, t, v, d, ws)
    for row in (0, v // 2, v - 1, v - 2):
        g = np.empty(d, np.float32)
        table.download(g, offset=row * d * 4)
        want = dout[ids == row].astype(np.float64).sum(0)
        assert np.all(np.abs(g - want) <= 2.0 ** -22 * np.abs(dout[ids == row]).sum(0))
    table.free()

    m, v, k, last = 300_000, 8200, 8, 200         # 2.46 G values of g; only the last rows count
    x = o.f32_to_bf16_bits(rng.standard_normal((m, k)).astype(np.float32))
    w = o.f32_to_bf16_bits(rng.standard_normal((v, k)).astype(np.float32))
    labels = np.full(m, -100)
    labels[-last:] = rng.integers(0, v, last)
    loss, row, dx, dw, _ = F.linear_ce_host(x, w, labels, device=gpu)
    xs, ws_ = o.bf16_bits_to_f32(x[-last:]).astype(np.float64), o.bf16_bits_to_f32(w).astype(np.float64)
    z = xs @ ws_.T
    z -= z.max(1, keepdims=True)
    p = np.exp(z) / np.exp(z).sum(1, keepdims=True)
    y = labels[-last:]
    # logits of at most 32, so rows of at most 64: 2^-22 of that
    assert abs(loss + np.log(p[np.arange(last), y]).mean()) <= 64 * 2.0 ** -22
    g = p.copy()
    g[np.arange(last), y] -= 1
    g /= last
    assert not dx[:-last].any() and not row[:-last].any()
    tol = H * (np.abs(g) @ np.abs(ws_)) + 2.0 ** -12 * (p / last) @ np.abs(ws_)
    assert np.all(np.abs(dx[-last:] - g @ ws_) <= tol)
    tol = H * (np.abs(g).T @ np.abs(xs)) + 2.0 ** -12 * (p / last).T @ np.abs(xs)
    assert np.all(np.abs(dw - g.T @ xs) <= tol)


FIRST_CALLS = """
import ctypes as C
import numpy as np
from novann_b200 import _lib, functional as F
from novann_b200.device import DeviceBuffer, Stream
gpu, (t, v, d) = int({gpu}), (1000, 300, 64)
rng = np.random.default_rng(0)
ids = DeviceBuffer.from_numpy(rng.integers(0, v, t).astype(np.int32), gpu)
table = DeviceBuffer.from_numpy(rng.standard_normal((v, d)).astype(np.float16), gpu)
out, dx, dw, dtable = (DeviceBuffer(n, gpu) for n in (t * d * 2, t * d * 4, v * d * 4, v * d * 4))
loss, stats, norm = DeviceBuffer(8, gpu), DeviceBuffer(t * 8, gpu), DeviceBuffer(8, gpu)
ws = DeviceBuffer(max(F.embedding_bwd_workspace_bytes(t, v, d), F.linear_ce_workspace_bytes(t, v, d),
                      F.grad_norm_workspace_bytes()), gpu)
st = Stream(gpu)
def step():
    F.embedding_device(out, table, "f16", ids, t, v, d, stream=st)
    F.linear_ce_device(loss, stats, out, table, "f16", ids, t, v, d, ws, stream=st)
    F.linear_ce_bwd_device(dx, dw, out, table, "f16", ids, stats, loss, t, v, d, ws, stream=st)
    F.embedding_bwd_device(dtable, dx, "f32", ids, t, v, d, ws, stream=st)
    F.clip_grads_device(norm, [dw, dtable], [v * d] * 2, "f32", 1e-3, ws, stream=st)
def results():
    st.sync()
    return [b.to_numpy(np.uint32, (b.nbytes // 4,)) for b in (out, loss, dw, dtable, norm)]
exe = C.c_void_p()
_lib.check(_lib.lib().nvq_graph_begin_capture(gpu, C.c_void_p(st.ptr)))
step()
_lib.check(_lib.lib().nvq_graph_end_capture(gpu, C.c_void_p(st.ptr), C.byref(exe)))
_lib.check(_lib.lib().nvq_graph_launch(gpu, exe, C.c_void_p(st.ptr)))
first = results()
step()
assert all(a.any() and np.array_equal(a, b) for a, b in zip(first, results()))
print("same bits")
"""


def test_the_first_calls_of_a_process_may_be_captured(gpu):
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS.replace("{gpu}", str(gpu))], capture_output=True, text=True,
                         timeout=300, cwd=Path(__file__).resolve().parents[1])
    assert run.returncode == 0 and "same bits" in run.stdout, run.stderr
