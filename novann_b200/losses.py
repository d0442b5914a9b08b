"""``CrossEntropyLoss`` with the reference's contract (``novann/losses/loss_functions.py:8-75``),
computed on the GPU: ``loss, grad = loss_fn(logits, labels)``; and ``LinearCrossEntropyLoss``, the last
Linear and the loss in one for vocabularies whose logits would not fit."""
from __future__ import annotations

import numpy as np

from . import functional as F
from .module import Module, Parameters


class CrossEntropyLoss:
    def __init__(self, device: int = 0) -> None:
        self.device = device
        self.N = 0
        self._loss = None
        self._grad = None

    def forward(self, logits: np.ndarray, targets: np.ndarray) -> np.float32:
        if targets.ndim != 1:
            targets = np.argmax(targets, axis=1)   # one-hot rows -> class indices
        self.N = logits.shape[0]
        self._loss, self._grad = F.softmax_ce_host(logits, targets, self.device)
        return np.float32(self._loss)

    def backward(self) -> np.ndarray:
        if self._grad is None:
            raise RuntimeError("forward must be called before backward")
        return self._grad

    def __call__(self, logits: np.ndarray, targets: np.ndarray):
        return self.forward(logits, targets), self.backward()


class LinearCrossEntropyLoss(Module):
    """A ``Linear(in_features, num_classes)`` and the mean softmax cross entropy of its output, without
    the (rows, num_classes) logits: ``loss, grad = head(x, labels)`` with x (rows, in_features) float,
    grad the gradient of x; the gradients of ``weight`` and ``bias`` are assigned as ``Linear.backward``
    does.  x and the weight are rounded to bf16 (``dtype="f16"``: fp16) for the tensor cores, sums are
    fp32.  Rows labelled ``ignore_index`` count for nothing.  The value is the ordinary negative log
    likelihood (``CrossEntropyLoss`` reports the reference's, which applies softmax twice)."""

    def __init__(self, in_features: int, num_classes: int, bias: bool = True, ignore_index: int = -100,
                 reduction: str = "mean", dtype: str = "bf16", init=None, device: int = 0) -> None:
        super().__init__()
        if in_features % 8:
            raise ValueError(f"in_features ({in_features}) must be a multiple of 8")
        if dtype not in ("bf16", "f16"):
            raise ValueError(f"dtype must be 'bf16' or 'f16', not {dtype!r}")
        F._reduction(reduction)
        from .layers import small_normal
        self.in_features, self.num_classes = int(in_features), int(num_classes)
        self.ignore_index, self.reduction, self.dtype, self.device = ignore_index, reduction, dtype, device
        self.weight = Parameters(np.asarray((init or small_normal)((num_classes, in_features)), np.float32))
        self.weight.name = "linear weight"
        self.bias = None
        if bias:
            self.bias = Parameters(np.zeros((1, num_classes), np.float32))
            self.bias.name = "linear bias"
        self._grad = None

    def forward(self, x: np.ndarray, targets: np.ndarray) -> np.float32:
        from . import quant
        from .layers import _as_f32
        low = np.float16 if self.dtype == "f16" else "bf16"
        xq = quant.cast(_as_f32(x, self.device), low, device=self.device)
        wq = quant.cast(self.weight.data, low, device=self.device)
        b = None if self.bias is None else self.bias.data
        out = F.linear_ce_host(xq, wq, targets, b, self.ignore_index, self.reduction, grad=self._training,
                               device=self.device)
        if self._training:
            self._grad, self.weight.grad = out[2], out[3]
            if self.bias is not None:
                self.bias.grad = out[4].reshape(self.bias.data.shape)
        else:
            self._grad = None
        return out[0]

    def backward(self) -> np.ndarray:
        if self._grad is None:
            raise RuntimeError("forward in training mode must be called before backward")
        return self._grad

    def __call__(self, x: np.ndarray, targets: np.ndarray):
        loss = self.forward(x, targets)
        return loss, self._grad

    def parameters(self):
        return [self.weight] + ([self.bias] if self.bias is not None else [])
