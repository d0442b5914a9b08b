"""What the token-model operators refuse, before anything reaches a GPU."""
import ctypes as C

import numpy as np
import pytest

import novann_b200 as nb
from novann_b200 import _lib, functional as F
from novann_b200.device import DeviceView
from novann_b200.module import Parameters

P = C.c_void_p(256)       # an aligned address that is never followed
ODD = C.c_void_p(257)


def refused(status, *words):
    assert status == _lib.ERR_INVALID
    msg = _lib.lib().nvq_last_error().decode()
    assert all(w in msg for w in words), msg


def test_embedding_refusals():
    f = _lib.lib().nvq_embedding_fwd
    refused(f(P, P, _lib.E4M3, P, 4, 4, 4, 1.0, 0, None), "type")
    refused(f(P, P, _lib.F32, P, 4, 0, 4, 1.0, 0, None), "V and D")
    refused(f(P, P, _lib.F32, P, 4, 4, 0, 1.0, 0, None), "V and D")
    refused(f(P, P, _lib.F32, P, 1 << 31, 4, 4, 1.0, 0, None), "T below")
    refused(f(None, P, _lib.F32, P, 4, 4, 4, 1.0, 0, None), "null")
    refused(f(P, ODD, _lib.F16, P, 4, 4, 4, 1.0, 0, None), "misaligned")
    assert f(None, None, _lib.F32, None, 0, 4, 4, 1.0, 0, None) == _lib.OK       # no tokens
    g = _lib.lib().nvq_embedding_bwd
    need = F.embedding_bwd_workspace_bytes(100, 10, 8)
    refused(g(P, P, _lib.F64, P, 100, 10, 8, 1.0, -1, 0, P, need, 0, None), "type")
    refused(g(P, P, _lib.F32, P, 100, 10, 8, 1.0, -1, 0, P, need - 1, 0, None), "workspace", str(need))
    refused(g(P, P, _lib.F32, P, 100, 10, 8, 1.0, -1, 0, None, need, 0, None), "workspace")
    refused(g(ODD, P, _lib.F32, P, 100, 10, 8, 1.0, -1, 0, P, need, 0, None), "table gradient")
    refused(g(P, None, _lib.F32, P, 100, 10, 8, 1.0, -1, 0, P, need, 0, None), "null")
    refused(g(P, P, _lib.F32, P, 100, 10, (1 << 22) + 1, 1.0, -1, 0, P, 1 << 62, 0, None), "D in")
    refused(g(P, P, _lib.F32, P, 100, 10, (1 << 21) + 1, 1.0, -1, 0, P, 1 << 62, 0, None), "D in")


def test_embedding_host_refusals():
    table = np.zeros((4, 8), np.float32)
    for bad in (np.array([4]), np.array([-1])):
        with pytest.raises(IndexError):
            F.embedding_host(table, bad)
        with pytest.raises(IndexError):
            F.embedding_bwd_host(np.zeros((1, 8), np.float32), bad, 4)
    with pytest.raises(TypeError):
        F.embedding_host(table, np.array([1.0]))
    with pytest.raises(TypeError):
        F.embedding_host(table.astype(np.int32), np.array([1]))
    with pytest.raises(ValueError, match="shape"):
        F.embedding_bwd_host(np.zeros((2, 8), np.float32), np.array([1]), 4)
    with pytest.raises(ValueError, match="hold"):
        F.embedding_device(DeviceView(256, 8), DeviceView(256, 128), "f32", DeviceView(256, 4), 1, 4, 8)
    with pytest.raises(ValueError, match="dtype"):
        F.embedding_device(DeviceView(256, 8), DeviceView(256, 128), "e4m3", DeviceView(256, 4), 1, 4, 8)
    with pytest.raises(ValueError, match="padding_id"):
        nb.Embedding(4, 8, padding_id=4)
    emb = nb.Embedding(4, 8)
    assert [p.name for p in emb.parameters()] == ["embedding weight"] and emb.weight.data.shape == (4, 8)
    with pytest.raises(RuntimeError):
        emb.backward(np.zeros((1, 8), np.float32))


def test_clip_refusals():
    ptrs, counts, types = (C.c_void_p * 1)(256), (C.c_size_t * 1)(4), (C.c_int32 * 1)(_lib.F32)
    need = F.grad_norm_workspace_bytes()
    f = _lib.lib().nvq_clip_grads
    refused(f(None, None, ptrs, counts, types, 1, 1.0, P, need, 0, None), "output")
    for bad in (0.0, -1.0, float("nan")):
        refused(f(P, None, ptrs, counts, types, 1, bad, P, need, 0, None), "max_norm")
    refused(f(P, None, ptrs, counts, types, 1, 1.0, P, need - 1, 0, None), "workspace")
    refused(f(P, None, None, counts, types, 1, 1.0, P, need, 0, None), "null")
    refused(f(P, None, ptrs, counts, (C.c_int32 * 1)(_lib.E4M3), 1, 1.0, P, need, 0, None), "type")
    refused(f(P, None, (C.c_void_p * 1)(258), counts, types, 1, 1.0, P, need, 0, None), "misaligned")
    refused(f(P, (C.c_void_p * 1)(None), ptrs, counts, types, 1, 1.0, P, need, 0, None), "output 0")
    v = DeviceView(256, 16)
    with pytest.raises(ValueError, match="twice"):
        F.clip_grads_device(v, [v, v], [4, 4], "f32", 1.0, v)
    with pytest.raises(ValueError, match="does not hold"):
        F.clip_grads_device(v, [v], [5], "f32", 1.0, v)
    with pytest.raises(ValueError, match="one length"):
        F.grad_norm_device(v, [v], [4, 4], "f32", v)
    with pytest.raises(ValueError, match="dtype"):
        F.grad_norm_device(v, [v], [4], "e4m3", v)


def test_optimiser_and_step_refusals():
    p = Parameters(np.zeros(3, np.float32))
    with pytest.raises(ValueError, match="max_grad_norm"):
        nb.SGD([p], 0.1, max_grad_norm=-1.0)
    with pytest.raises(NotImplementedError):
        nb.SGD([p], 0.1, momentum=0.9, max_grad_norm=1.0)
    with pytest.raises(ValueError, match="max_norm"):
        F.clip_grad_norm([p], 0.0)
    p.grad = np.zeros(3, np.int32)
    with pytest.raises(TypeError):
        F.clip_grad_norm([p], 1.0)
    from novann_b200.train import MLPTrainStep
    with pytest.raises(ValueError, match="max_grad_norm"):
        MLPTrainStep([], 4, 0.1, max_grad_norm=0.0)
    with pytest.raises(ValueError, match="peer"):
        MLPTrainStep([], 4, 0.1, peer=object(), max_grad_norm=1.0)


def test_linear_ce_refusals():
    L = _lib.lib()
    need = F.linear_ce_workspace_bytes(100, 50, 16)

    def fwd(dtype=_lib.BF16, m=100, v=50, k=16, x=P, w=P, labels=P, loss=P, stats=P, red=1, ws=P, nbytes=need):
        return L.nvq_linear_ce_fwd(loss, None, stats, x, w, dtype, None, labels, m, v, k, -100, red, ws, nbytes, 0, None)

    def bwd(dtype=_lib.BF16, grad=_lib.F32, dx=P, dw=P, stats=P, loss=P, ws=P, nbytes=need, k=16):
        return L.nvq_linear_ce_bwd(dx, dw, grad, None, P, P, dtype, None, P, stats, loss, 1.0, 100, 50, k, -100, 1, ws,
                                   nbytes, 0, None)
    refused(fwd(dtype=_lib.F32), "type")
    refused(fwd(k=12), "multiple of 8")
    refused(fwd(v=0), "V in")
    refused(fwd(red=2), "reduction")
    refused(fwd(x=None), "aligned")
    refused(fwd(w=C.c_void_p(264)), "aligned")
    refused(fwd(labels=None), "labels")
    refused(fwd(stats=None), "output")
    refused(fwd(loss=None), "output")
    refused(fwd(nbytes=16), "workspace")
    refused(fwd(ws=C.c_void_p(128)), "workspace")
    refused(bwd(grad=_lib.F16), "gradients")
    refused(bwd(dx=C.c_void_p(264)), "aligned")
    refused(bwd(stats=None), "statistics")
    refused(bwd(nbytes=need - 1), "workspace", str(need))
    refused(bwd(k=4), "multiple of 8")
    v = DeviceView(256, 64)
    with pytest.raises(ValueError, match="reduction"):
        F.linear_ce_device(v, v, v, v, "bf16", v, 1, 1, 8, v, reduction="none")
    with pytest.raises(ValueError, match="hold"):
        F.linear_ce_device(v, v, v, v, "bf16", v, 1, 5, 8, v)
    with pytest.raises(ValueError, match="grad_dtype"):
        F.linear_ce_bwd_device(v, v, v, v, "bf16", v, v, v, 1, 1, 8, v, grad_dtype="f16")
    x, w = np.zeros((2, 16), np.float16), np.zeros((5, 16), np.float16)
    with pytest.raises(IndexError):
        F.linear_ce_host(x, w, np.array([0, 5]))
    with pytest.raises(ValueError, match="labels"):
        F.linear_ce_host(x, w, np.array([0]))
    with pytest.raises(TypeError):
        F.linear_ce_host(x, w.view(np.uint16), np.array([0, 1]))
    with pytest.raises(ValueError, match="features"):
        F.linear_ce_host(x, w[:, :8], np.array([0, 1]))
    with pytest.raises(ValueError, match="multiple of 8"):
        nb.LinearCrossEntropyLoss(12, 5)
    with pytest.raises(ValueError, match="dtype"):
        nb.LinearCrossEntropyLoss(16, 5, dtype="f32")
    head = nb.LinearCrossEntropyLoss(16, 5, bias=False)
    assert len(head.parameters()) == 1
    with pytest.raises(RuntimeError):
        head.backward()
