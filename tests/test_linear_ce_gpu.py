"""Linear + softmax cross entropy against 64-bit NumPy.

What the bounds count.  A logit is an fp32 sum of K products that are exact in fp32: off by at most
d = (K + 2) * 2^-23 times the sum of the products' magnitudes (2^-23, since the tensor core may truncate
where it adds).  lse is off by d at its worst logit, by the 2^-22 of each exp2, by V * 2^-24 of the sum and
by the rounding of a value of that size.  A value of g is off by 2 d (logit and lse) and 2^-21 relative to
the probability, and then by the operands' half step h (2^-8 for bf16, 2^-11 for f16) relative to itself.
"""
import ctypes as C

import numpy as np
import pytest

import novann_b200 as nb
from novann_b200 import _lib, functional as F
from novann_b200.device import DeviceBuffer, DeviceView, Stream, device_sync
from oracle import oracle_np as o

pytestmark = pytest.mark.gpu
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def to_type(x, dtype):
    return o.f32_to_bf16_bits(x.astype(np.float32)) if dtype == "bf16" else x.astype(np.float16)


def wide(a):
    return (o.bf16_bits_to_f32(a) if a.dtype == np.uint16 else a).astype(np.float64)


def inputs(m, v, k, dtype, seed, spread=2.0, bias=True, ignore=True):
    rng = np.random.default_rng(seed)
    w = rng.standard_normal((v, k)) * spread / np.sqrt(k)
    labels = rng.integers(0, v, m)
    x = rng.standard_normal((m, k))
    x[::2] += 4.0 * w[labels[::2]] / np.linalg.norm(w[labels[::2]], axis=1, keepdims=True)
    if ignore and m > 2:
        labels[rng.random(m) < 0.2] = -100
    b = (rng.standard_normal(v) * 0.3).astype(np.float32) if bias else None
    return to_type(x, dtype), to_type(w, dtype), labels, b


def reference(x, w, labels, b, mean=True, grad_scale=1.0, ignore=-100):
    """Values and the error bounds of the module's docstring."""
    x, w = wide(x), wide(w)
    m, k = x.shape
    v = w.shape[0]
    z = x @ w.T + (0.0 if b is None else b.astype(np.float64))
    with np.errstate(invalid="ignore", over="ignore"):
        mag = np.abs(x) @ np.abs(w).T
        if b is not None:
            mag = mag + np.where(np.isfinite(b), np.abs(b), 0.0)
        d = (k + 2) * 2.0 ** -23 * mag.max(axis=1)
        top = z.max(axis=1)
        lse = top + np.log(np.exp(z - top[:, None]).sum(axis=1))
    live = labels != ignore
    at = np.where(live, labels, 0)
    row = np.where(live, lse - z[np.arange(m), at], 0.0)
    count = max(1, live.sum()) if mean else 1
    p = np.exp(z - lse[:, None])
    g = p.copy()
    g[np.arange(m), at] -= 1.0
    s = grad_scale / count
    g *= live[:, None] * s
    dl = d + 2.0 ** -22 + v * 2.0 ** -24 + (np.abs(lse) + np.abs(top)) * 2.0 ** -22
    return dict(z=z, lse=lse, row=row, loss=row.sum() / count, g=g, dx=g @ w, dw=g.T @ x, db=g.sum(0), x=x, w=w, p=p,
                dl=dl, s=s, live=live, d_row=live * (dl + d + np.abs(z[np.arange(m), at]) * 2.0 ** -23), count=count)


def check_grads(r, dx, dw, db, dtype, out="f32"):
    h = HALF[dtype]
    floor = 2.0 ** -39 if dtype == "f16" else 2.0 ** -126        # half a step of the type's smallest values
    dg_fp32 = r["live"][:, None] * r["p"] * abs(r["s"]) * (2 * r["dl"][:, None] + 2.0 ** -21) + np.abs(r["g"]) * 2.0 ** -22
    # fp32 has no normal value below 2^-126: a smaller probability becomes 0, off by less than 2^-126 (e^-260 = 1e-113 of
    # a logit 260 below the largest, where 64 bits still hold it)
    dg_fp32 = dg_fp32 + abs(r["s"]) * 2.0 ** -126
    dg = dg_fp32 + np.abs(r["g"]) * h + abs(r["s"]) * floor
    m, v = r["g"].shape
    k = r["x"].shape[1]
    small = 2.0 ** -25 if out == "f16" else 0.0
    ho = HALF[out]
    ag, ax, aw = np.abs(r["g"]), np.abs(r["x"]), np.abs(r["w"])
    tol = dg @ aw + (v + 2) * 2.0 ** -23 * (ag @ aw)
    assert np.all(np.abs(dx - r["dx"]) <= tol + (np.abs(r["dx"]) + tol) * ho + small)
    tol = dg.T @ ax + (m + 2) * 2.0 ** -23 * (ag.T @ ax)
    assert np.all(np.abs(dw - r["dw"]) <= tol + (np.abs(r["dw"]) + tol) * ho + small)
    if db is not None:
        tol = dg_fp32.sum(0) + (m + 2) * 2.0 ** -23 * ag.sum(0)
        assert np.all(np.abs(db - r["db"]) <= tol + np.abs(r["db"]) * 2.0 ** -23)


SHAPES = [(1, 1, 8), (1, 2, 8), (2, 1, 16), (3, 5, 24), (7, 129, 64), (128, 10, 128), (129, 127, 72), (255, 257, 136),
          (256, 256, 64), (257, 385, 200), (300, 1001, 512), (513, 640, 1032), (64, 5000, 40), (1, 9000, 8),
          (1500, 33, 64), (40, 300, 2056)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,v,k", SHAPES)
def test_loss_and_gradients(gpu, dtype, m, v, k):
    x, w, labels, b = inputs(m, v, k, dtype, m + v + k, bias=(m + v) % 2 == 0)
    r = reference(x, w, labels, b, grad_scale=3.0)
    loss, row, dx, dw, db = F.linear_ce_host(x, w, labels, b, grad_scale=3.0, device=gpu)
    assert np.all(np.abs(row - r["row"]) <= r["d_row"])
    assert abs(loss - r["loss"]) <= r["d_row"].sum() / r["count"] + abs(r["loss"]) * 2.0 ** -22
    check_grads(r, dx, dw, db, dtype)
    again = F.linear_ce_host(x, w, labels, b, grad_scale=3.0, device=gpu)
    assert all(np.array_equal(p, q) for p, q in zip((loss, row, dx, dw), again[:4]))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_several_pieces_of_the_vocabulary(gpu, dtype):
    """64 Mi values per piece: 8300 rows take the vocabulary in pieces of 8192 at most."""
    m, v, k = 8300, 8200, 16
    x, w, labels, b = inputs(m, v, k, dtype, 5)
    r = reference(x, w, labels, b)
    loss, row, dx, dw, db = F.linear_ce_host(x, w, labels, b, device=gpu)
    assert np.all(np.abs(row - r["row"]) <= r["d_row"])
    check_grads(r, dx, dw, db, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("want", ["dx", "dw", "db", "all"])
def test_gradients_in_the_operands_type_and_one_at_a_time(gpu, dtype, want):
    m, v, k = 140, 300, 88                      # rows of 176 bytes: not a multiple of 32
    x, w, labels, b = inputs(m, v, k, dtype, 1)
    r = reference(x, w, labels, b, mean=False, grad_scale=0.5)
    bx, bw = DeviceBuffer.from_numpy(x, gpu), DeviceBuffer.from_numpy(w, gpu)
    bl, bb = DeviceBuffer.from_numpy(labels.astype(np.int32), gpu), DeviceBuffer.from_numpy(b, gpu)
    ws = DeviceBuffer(F.linear_ce_workspace_bytes(m, v, k), gpu)
    head, stats = DeviceBuffer(8, gpu), DeviceBuffer(m * 8, gpu)
    F.linear_ce_device(head, stats, bx, bw, dtype, bl, m, v, k, ws, bias=bb, reduction="sum")
    out = {n: DeviceBuffer(s, gpu) if want in (n, "all") else None
           for n, s in (("dx", m * k * 2), ("dw", v * k * 2), ("db", v * 4))}
    F.linear_ce_bwd_device(out["dx"], out["dw"], bx, bw, dtype, bl, stats, head, m, v, k, ws, bias=bb, db=out["db"],
                           grad_dtype=dtype, grad_scale=0.5, reduction="sum")
    device_sync(gpu)
    F.check_device_errors(gpu)
    t = np.uint16 if dtype == "bf16" else np.float16
    got = {"dx": r["dx"], "dw": r["dw"], "db": r["db"]}
    for n, s in (("dx", (m, k)), ("dw", (v, k))):
        if out[n] is not None:
            got[n] = wide(out[n].to_numpy(t, s))
    if out["db"] is not None:
        got["db"] = out["db"].to_numpy(np.float32, (v,))
    check_grads(r, got["dx"], got["dw"], got["db"], dtype, out=dtype)
    n, live = head.to_numpy(np.float32, (2,))
    assert live == r["live"].sum() and abs(n - r["row"].sum()) <= r["d_row"].sum() + abs(n) * 2.0 ** -22


def test_no_row_counts_and_no_rows(gpu):
    x, w, labels, b = inputs(40, 50, 16, "bf16", 2)
    labels[:] = -100
    loss, row, dx, dw, db = F.linear_ce_host(x, w, labels, b, device=gpu)
    assert loss == 0 and not row.any() and not dx.any() and not dw.any() and not db.any()
    loss, row, dx, dw, db = F.linear_ce_host(x[:0], w, labels[:0], b, device=gpu)
    assert loss == 0 and row.size == 0 and dx.shape == (0, 16) and not dw.any() and not db.any()


def test_ignored_rows_may_hold_anything(gpu):
    x, w, labels, b = inputs(40, 50, 16, "f16", 3, ignore=False)
    clean = F.linear_ce_host(x[1:], w, labels[1:], b, device=gpu)
    x[0] = np.inf
    labels[0] = 7                               # any label may be the one that is ignored
    keep = labels[1:] != 7
    clean = F.linear_ce_host(x[1:][keep], w, labels[1:][keep], b, device=gpu)
    labels[1:][~keep] = 7
    loss, row, dx, _, db = F.linear_ce_host(x, w, labels, b, ignore_index=7, device=gpu)
    assert abs(loss - clean[0]) <= abs(loss) * 2.0 ** -22 and row[0] == 0 and not dx[0].any()
    assert np.allclose(db, clean[4], rtol=0, atol=2.0 ** -20)


@pytest.mark.parametrize("low", [-np.inf, np.finfo(np.float32).min, -1e30])
def test_entries_masked_by_the_bias(gpu, low):
    m, v, k = 70, 700, 32
    x, w, labels, b = inputs(m, v, k, "bf16", 4)
    out = np.zeros(v, bool)
    out[:300] = True                            # a whole 256-entry tile and part of the next
    out[650:] = True
    labels[labels >= 0] = 300 + labels[labels >= 0] % 350
    b[out] = low
    loss, row, dx, dw, db = F.linear_ce_host(x, w, labels, b, device=gpu)
    r = reference(x, w[300:650], np.where(labels >= 0, labels - 300, -100), b[300:650])
    assert np.all(np.abs(row - r["row"]) <= r["d_row"])
    check_grads(r, dx, dw[300:650], db[300:650], "bf16")
    assert not dw[out].any() and not db[out].any()


def test_every_entry_masked_alike_and_a_masked_label(gpu):
    x, w, labels, b = inputs(5, 300, 16, "f16", 6, ignore=False)
    low = np.finfo(np.float32).min
    loss, row, dx, dw, db = F.linear_ce_host(x, w, labels, np.full(300, low, np.float32), device=gpu)
    # the logits all round to the lowest value: a uniform distribution
    assert np.all(np.isfinite(dx)) and np.all(np.isfinite(db)) and abs(db.sum()) < 1e-4
    loss, row, dx, dw, db = F.linear_ce_host(x, w, labels, np.full(300, -np.inf, np.float32), device=gpu)
    assert np.all(np.isinf(row)) and not dx.any() and not dw.any() and not db.any()       # nothing left
    b[labels[0]] = -np.inf
    keep = labels != labels[0]
    loss, row, dx, dw, db = F.linear_ce_host(x, w, labels, b, device=gpu)
    assert np.isinf(row[0]) and np.all(np.isfinite(row[keep])) and np.all(np.isfinite(dx))


def test_large_and_equal_logits(gpu):
    m, v, k = 33, 400, 64
    x, w, labels, b = inputs(m, v, k, "bf16", 7, spread=200.0)          # logits of several hundreds
    r = reference(x, w, labels, b)
    loss, row, dx, dw, db = F.linear_ce_host(x, w, labels, b, device=gpu)
    assert np.all(np.abs(row - r["row"]) <= r["d_row"])
    check_grads(r, dx, dw, db, "bf16")
    zero = np.zeros_like(w)
    row = F.linear_ce_host(x, zero, labels, None, grad=False, device=gpu)[1]
    assert np.all(np.abs(row[labels >= 0] - np.log(v)) <= 8 * 2.0 ** -22)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_probabilities_of_a_row_sum_to_one(gpu, dtype):
    """Both passes sum a logit alike, so the gradients of the biases sum to 0 up to what follows the logits: exp2 and
    its argument's rounding (2^-21 of each probability) and fp32 sums over the entries and rows, however long K is."""
    m, v, k = 300, 41, 4096
    x, w, labels, b = inputs(m, v, k, dtype, 12)
    db = F.linear_ce_host(x, w, labels, b, device=gpu)[4].astype(np.float64)
    assert abs(db.sum()) <= 2.0 ** -21 + v * 2.0 ** -24 + m * 2.0 ** -24 * np.abs(db).sum()


def test_labels_out_of_range_are_reported(gpu):
    x, w, labels, _ = inputs(4, 20, 16, "bf16", 8, ignore=False)
    labels[1], labels[2] = 20, -1
    bx, bw = DeviceBuffer.from_numpy(x, gpu), DeviceBuffer.from_numpy(w, gpu)
    bl = DeviceBuffer.from_numpy(labels.astype(np.int32), gpu)
    ws = DeviceBuffer(F.linear_ce_workspace_bytes(4, 20, 16), gpu)
    head, stats, rows, dx = (DeviceBuffer(n, gpu) for n in (8, 32, 16, 4 * 16 * 4))
    F.linear_ce_device(head, stats, bx, bw, "bf16", bl, 4, 20, 16, ws, row_loss=rows)
    F.linear_ce_bwd_device(dx, None, bx, bw, "bf16", bl, stats, head, 4, 20, 16, ws)
    device_sync(gpu)
    with pytest.raises(_lib.NvqError, match="85"):
        F.check_device_errors(gpu)
    assert head.to_numpy(np.float32, (2,))[1] == 2
    got = rows.to_numpy(np.float32, (4,))
    assert got[1] == 0 and got[2] == 0 and got[0] > 0
    d = dx.to_numpy(np.float32, (4, 16))
    assert not d[1:3].any() and d[0].any() and d[3].any()


def test_gradient_against_differences(gpu):
    m, v, k = 6, 40, 16
    x, w, labels, b = inputs(m, v, k, "f16", 9, ignore=False)
    _, _, dx, dw, db = F.linear_ce_host(x, w, labels, b, device=gpu)
    e = 2.0 ** -4

    def loss(xx, ww, bb):
        return float(F.linear_ce_host(xx, ww, labels, bb, grad=False, device=gpu)[0])
    for name, at, g in (("x", (1, 3), dx), ("w", (int(labels[0]), 5), dw), ("w", (7, 0), dw), ("b", (int(labels[2]),), db)):
        args = {"x": x, "w": w, "b": b}
        both, step = [], []
        for sign in (1, -1):
            a = {n: t.copy() for n, t in args.items()}
            a[name][at] += a[name].dtype.type(sign * e)
            step.append(float(a[name][at]))
            both.append(loss(a["x"], a["w"], a["b"]))
        got = (both[0] - both[1]) / (step[0] - step[1])
        # third derivative of lse along one input is below 1 * |other operand|^3: e^2 / 6 of 4^3, and 2^-20 of the
        # loss over the step
        assert abs(got - g[at]) <= e * e / 6 * 64 / m + 5 * 2.0 ** -20 / e + abs(g[at]) * 2.0 ** -9


def test_head_class_and_modes(gpu):
    rng = np.random.default_rng(10)
    head = nb.LinearCrossEntropyLoss(24, 50, device=gpu)
    head.weight.data = rng.standard_normal((50, 24)).astype(np.float32)
    x, y = rng.standard_normal((30, 24)).astype(np.float32), rng.integers(0, 50, 30)
    loss, dx = head(x, y)
    r = reference(to_type(x, "bf16"), to_type(head.weight.data, "bf16"), y, head.bias.data.reshape(-1))
    assert abs(loss - r["loss"]) <= r["d_row"].mean() + abs(r["loss"]) * 2.0 ** -22
    check_grads(r, dx, head.weight.grad, head.bias.grad.reshape(-1), "bf16")
    head.eval()
    assert head(x, y) == (loss, None)
    with pytest.raises(RuntimeError):
        head.backward()


@pytest.mark.parametrize("dtype,grad", [("bf16", "bf16"), ("f16", "f32")])
def test_buffers_on_16_byte_boundaries_and_nothing_behind_them(gpu, dtype, grad):
    m, v, k = 130, 140, 64
    size = 4 if grad == "f32" else 2
    x, w, labels, _ = inputs(m, v, k, dtype, 11, bias=False)
    r = reference(x, w, labels, None)
    bx, bw = DeviceBuffer(x.nbytes + 16, gpu), DeviceBuffer(w.nbytes + 16, gpu)
    bx.upload(x, offset=16)
    bw.upload(w, offset=16)
    bl = DeviceBuffer.from_numpy(labels.astype(np.int32), gpu)
    ws = DeviceBuffer(F.linear_ce_workspace_bytes(m, v, k), gpu)
    head, stats = DeviceBuffer(8, gpu), DeviceBuffer(m * 8, gpu)
    view = lambda b: DeviceView(b.ptr + 16, b.nbytes - 16, gpu)  # noqa: E731
    dx, dw = DeviceBuffer(16 + m * k * size + 16, gpu), DeviceBuffer(16 + v * k * size + 16, gpu)
    for b in (dx, dw):
        b.upload(np.full(b.nbytes, 0x5A, np.uint8))
    F.linear_ce_device(head, stats, view(bx), view(bw), dtype, bl, m, v, k, ws)
    F.linear_ce_bwd_device(view(dx), view(dw), view(bx), view(bw), dtype, bl, stats, head, m, v, k, ws, grad_dtype=grad)
    device_sync(gpu)
    F.check_device_errors(gpu)
    t = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[grad]
    got = []
    for b, n in ((dx, m), (dw, v)):
        raw = b.to_numpy(np.uint8, (b.nbytes,))
        assert np.all(raw[:16] == 0x5A) and np.all(raw[-16:] == 0x5A)
        got.append(wide(raw[16:-16].view(t).reshape(n, k)))
    check_grads(r, got[0], got[1], None, dtype, out=grad)


def test_captured_graphs_share_a_workspace(gpu):
    m, v, k = 200, 600, 64
    st = Stream(gpu)
    ws = DeviceBuffer(F.linear_ce_workspace_bytes(m, v, k), gpu)
    bx, bw, bl = DeviceBuffer(m * k * 2, gpu), DeviceBuffer(v * k * 2, gpu), DeviceBuffer(m * 4, gpu)
    sets = [[DeviceBuffer(n, gpu) for n in (8, m * 8, m * k * 4, v * k * 4)] for _ in range(2)]

    def launch(i):
        head, stats, dx, dw = sets[i]
        F.linear_ce_device(head, stats, bx, bw, "bf16", bl, m, v, k, ws, stream=st)
        F.linear_ce_bwd_device(dx, dw, bx, bw, "bf16", bl, stats, head, m, v, k, ws, grad_scale=i + 1.0, stream=st)
    graphs = []
    for i in range(2):
        _lib.check(_lib.lib().nvq_graph_begin_capture(gpu, C.c_void_p(st.ptr)))
        launch(i)
        h = C.c_void_p()
        _lib.check(_lib.lib().nvq_graph_end_capture(gpu, C.c_void_p(st.ptr), C.byref(h)))
        graphs.append(h)
    for seed in (1, 2):
        x, w, labels, _ = inputs(m, v, k, "bf16", seed)
        for b, a in ((bx, x), (bw, w), (bl, labels.astype(np.int32))):
            b.upload(a, st)
        for h in graphs:
            _lib.check(_lib.lib().nvq_graph_launch(gpu, h, C.c_void_p(st.ptr)))
        st.sync()
        F.check_device_errors(gpu)
        for i in range(2):
            r = reference(x, w, labels, None, grad_scale=i + 1.0)
            check_grads(r, sets[i][2].to_numpy(np.float32, (m, k)), sets[i][3].to_numpy(np.float32, (v, k)), None, "bf16")
    for h in graphs:
        _lib.lib().nvq_graph_destroy(gpu, h)
