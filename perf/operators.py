"""Workloads of the token-model operators: embedding lookup and its gradient, the linear layer
fused with softmax cross entropy, and the global gradient norm with clipping.

``run`` computes each in its plain form (elementary torch operations in 32 bits, rounded once at
the end) or, with ``own`` set, through ``novann_b200.functional``.  ``exact`` gives the same
outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}

# Parameter counts of the network of this repository's training benchmark (784-256-128-10).
MLP_TENSORS = "200704,256,32768,128,1280,10"


def _blocks(layers, width, hidden, vocab):
    """Element counts of a decoder's tensors: per layer four width x width projections, three
    width x hidden ones and two norm weights, then an embedding table and a last norm weight."""
    one = [width * width] * 4 + [width * hidden] * 3 + [width] * 2
    return ",".join(str(n) for n in one * layers + [vocab * width, width])


def listed():
    return [
        # one short prompt through a small fp32 table: the call's own latency
        {"name": "embedding_short", "op": "embedding", "dtype": "f32", "tokens": 17, "vocab": 1000, "width": 64,
         "scale": 8.0, "pad": False},
        # a training batch of 32 sequences of 2048 tokens through a wide bf16 table
        {"name": "embedding_batch", "op": "embedding", "dtype": "bf16", "tokens": 65536, "vocab": 128000,
         "width": 4096, "scale": 64.0, "pad": True},
        # gradient of a small fp32 table with an odd width, one padded micro-batch
        {"name": "embedding_grad_odd", "op": "embedding_grad", "dtype": "f32", "tokens": 4095, "vocab": 8191,
         "width": 1001, "scale": 1.0, "pad": True},
        # gradient of a large table from a bf16 training batch
        {"name": "embedding_grad_batch", "op": "embedding_grad", "dtype": "bf16", "tokens": 65536, "vocab": 50001,
         "width": 2048, "scale": 45.25, "pad": True},
        # the ten-class head of this repository's training benchmark, its batch of 128
        {"name": "head_ten_classes", "op": "linear_ce_grad", "dtype": "bf16", "rows": 128, "vocab": 10, "width": 128,
         "bias": True},
        # scoring a few rows against a small vocabulary
        {"name": "head_score_few", "op": "linear_ce", "dtype": "f16", "rows": 7, "vocab": 1001, "width": 512,
         "bias": True},
        # evaluation of a ragged batch: loss of every row, no gradient
        {"name": "head_score_batch", "op": "linear_ce", "dtype": "bf16", "rows": 4095, "vocab": 50001, "width": 2048,
         "bias": False},
        # a training step of a small model's head
        {"name": "head_step", "op": "linear_ce_grad", "dtype": "f16", "rows": 2048, "vocab": 32000, "width": 1024,
         "bias": True},
        # a training step of a large model's head
        {"name": "head_step_large", "op": "linear_ce_grad", "dtype": "bf16", "rows": 8192, "vocab": 128000,
         "width": 4096, "bias": False},
        # the six tensors of this repository's training benchmark, clipped
        {"name": "clip_mlp", "op": "clip", "dtype": "f32", "counts": MLP_TENSORS, "cut": 0.5},
        # the norm alone (as a run logs it every step) of a bf16 model's gradients
        {"name": "norm_bf16", "op": "norm", "dtype": "bf16", "counts": _blocks(12, 1024, 4096, 32000), "cut": 1.0},
        # all fp32 gradients of a larger model, clipped
        {"name": "clip_large", "op": "clip", "dtype": "f32", "counts": _blocks(16, 1408, 5632, 50001), "cut": 0.1},
    ]


def _log_size(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["embedding", "embedding_grad", "linear_ce", "linear_ce_grad", "clip", "norm"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op.startswith("embedding"):
        while True:
            case = {"op": op, "dtype": dtype, "tokens": _log_size(rng, 1, 65536), "vocab": _log_size(rng, 2, 128000),
                    "width": _log_size(rng, 8, 4096), "scale": rng.choice([1.0, 8.0, 45.25]), "pad": rng.random() < 0.5}
            most = 65536 * 2048 * 2 + 50001 * 2048 * 4 if op == "embedding_grad" else 2 * 65536 * 4096 * 2
            if work(case)["bytes"] <= most:
                return case
    if op.startswith("linear_ce"):
        return {"op": op, "dtype": rng.choice(["f16", "bf16"]), "rows": _log_size(rng, 1, 8192),
                "vocab": _log_size(rng, 2, 128000), "width": 8 * _log_size(rng, 4, 512), "bias": rng.random() < 0.5}
    counts = [_log_size(rng, 1, 1 << 22) for _ in range(_log_size(rng, 1, 96))]
    return {"op": op, "dtype": dtype, "counts": ",".join(str(n) for n in counts), "cut": rng.choice([0.1, 0.5, 2.0])}


def _counts(case):
    return [int(n) for n in case["counts"].split(",")]


def _ids(n, vocab, rng):
    """Token ids whose frequency falls with the id as 1 / id, the most frequent first."""
    u = torch.rand(n, generator=rng, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp_(0, vocab - 1).to(torch.int32)


def prepare(case, seed):
    rng = torch.Generator(device="cuda")
    rng.manual_seed(seed)
    op, dtype = case["op"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=rng, device="cuda", dtype=torch.float32)

    state = dict(case)
    if op.startswith("embedding"):
        t, v, d = case["tokens"], case["vocab"], case["width"]
        state["ids"] = _ids(t, v, rng)
        state["pad_id"] = v - 1 if case["pad"] else None
        if case["pad"]:      # the last tenth of the batch is padding
            state["ids"][t - t // 10:] = v - 1
        if op == "embedding":
            state["table"] = (normal(v, d) / math.sqrt(d)).to(dtype)
            state["out"] = torch.empty(t, d, device="cuda", dtype=dtype)
        else:
            state["dout"] = (normal(t, d) * 1e-2).to(dtype)
            state["dtable"] = torch.empty(v, d, device="cuda", dtype=torch.float32)
    elif op.startswith("linear_ce"):
        m, v, k = case["rows"], case["vocab"], case["width"]
        w = normal(v, k)
        labels = _ids(m, v, rng)
        x = normal(m, k)
        # every second row already leans towards its label, as rows of a trained model do
        x[::2] += 4.0 * torch.nn.functional.normalize(w[labels[::2].long()], dim=1)
        state["x"], state["w"] = x.to(dtype), (w * (2.0 / math.sqrt(k))).to(dtype)
        state["bias"] = normal(v) * 0.1 if case["bias"] else None
        # training in fp16 scales the loss, so that small gradients stay above the type's range
        state["loss_scale"] = 1024.0 if case["dtype"] == "f16" else 1.0
        ignored = torch.rand(m, generator=rng, device="cuda") < 0.1      # padding and prompt rows
        ignored[0] = False
        state["labels"] = torch.where(ignored, torch.full_like(labels, -100), labels)
    else:
        counts = _counts(case)
        # one gradient buffer, every tensor starting on a multiple of 16 elements; the tensors'
        # magnitudes differ by up to a factor of a hundred
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + (n + 15) // 16 * 16)
        flat = torch.zeros(starts[-1], device="cuda", dtype=dtype)
        spread = torch.rand(len(counts), generator=rng, device="cuda").cpu().tolist()
        state["grads"] = []
        for n, s, u in zip(counts, starts, spread):
            flat[s:s + n] = (normal(n) * 10.0 ** (-2.0 - 2.0 * u)).to(dtype)
            state["grads"].append(flat[s:s + n])
        # the clipped gradients go to a second buffer of the same layout
        state["out"] = torch.zeros_like(flat)
        state["parts"] = [state["out"][s:s + n] for n, s in zip(counts, starts)]
        # the limit as a share of the norm that such gradients have (above 1: nothing is cut)
        state["max_norm"] = case["cut"] * math.sqrt(sum(n * 10.0 ** (-4.0 - 4.0 * u) for n, u in zip(counts, spread)))
    return state


# ------------------------------------------------------------------ plain forms, 32 bits
def _embedding(s):
    s["out"].copy_(s["table"][s["ids"].long()].float() * s["scale"])
    return s["out"]


def _embedding_grad(s):
    g = s["dout"].float() * s["scale"]
    if s["pad_id"] is not None:
        g = g * (s["ids"] != s["pad_id"]).float()[:, None]
    return s["dtable"].zero_().index_add_(0, s["ids"].long(), g)


def _linear_ce(s, grad):
    x, w, labels = s["x"].float(), s["w"].float(), s["labels"].long()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"]
    valid = labels != -100
    at = torch.where(valid, labels, torch.zeros_like(labels))[:, None]
    top = z.max(dim=1, keepdim=True).values
    lse = top + (z - top).exp().sum(dim=1, keepdim=True).log()
    row = ((lse - z.gather(1, at))[:, 0]) * valid
    count = valid.sum().clamp(min=1).float()
    out = {"loss": row.sum() / count, "rows": row}
    if not grad:
        return out
    g = (z - lse).exp()
    g.scatter_add_(1, at, torch.full_like(lse, -1.0))
    g = g * (valid[:, None] * (s["loss_scale"] / count))
    out["dx"] = (g @ w).to(s["x"].dtype)
    out["dw"] = (g.t() @ x).to(s["w"].dtype)
    if s["bias"] is not None:
        out["db"] = g.sum(dim=0)
    return out


def _norm(s):
    return torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()


def _clip(s):
    norm = _norm(s)
    coef = (s["max_norm"] / norm).clamp(max=1.0)
    [part.copy_(g.float() * coef) for g, part in zip(s["grads"], s["parts"])]
    return {"norm": norm, "grads": s["out"]}


# ------------------------------------------------------------------ the framework's calls
def _view(t):
    from novann_b200.device import DeviceView
    return DeviceView(t.data_ptr(), t.numel() * t.element_size(), t.device.index)


def _space(nbytes):
    return torch.empty(max(1, nbytes), device="cuda", dtype=torch.uint8)


def _run_own(s):
    from novann_b200 import functional as F
    op, dtype = s["op"], s["dtype"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "embedding":
        F.embedding_device(_view(s["out"]), _view(s["table"]), dtype, _view(s["ids"]), s["tokens"], s["vocab"],
                           s["width"], scale=s["scale"], stream=stream)
        return s["out"]
    if op == "embedding_grad":
        t, v, d = s["tokens"], s["vocab"], s["width"]
        space = _space(F.embedding_bwd_workspace_bytes(t, v, d))
        F.embedding_bwd_device(_view(s["dtable"]), _view(s["dout"]), dtype, _view(s["ids"]), t, v, d, _view(space),
                               scale=s["scale"], padding_id=s["pad_id"], stream=stream)
        return s["dtable"]
    if op in ("linear_ce", "linear_ce_grad"):
        m, v, k = s["rows"], s["vocab"], s["width"]
        back = op == "linear_ce_grad"
        bias = None if s["bias"] is None else _view(s["bias"])
        space = _view(_hold := _space(F.linear_ce_workspace_bytes(m, v, k, backward=back)))
        head = torch.empty(2, device="cuda")
        stats, rows = torch.empty(2, m, device="cuda"), torch.empty(m, device="cuda")
        x, w, labels = _view(s["x"]), _view(s["w"]), _view(s["labels"])
        F.linear_ce_device(_view(head), _view(stats), x, w, dtype, labels, m, v, k, space, bias=bias,
                           row_loss=_view(rows), stream=stream)
        out = {"loss": head[0], "rows": rows}
        if back:
            out["dx"], out["dw"] = torch.empty_like(s["x"]), torch.empty_like(s["w"])
            if bias is not None:
                out["db"] = torch.empty(v, device="cuda")
            F.linear_ce_bwd_device(_view(out["dx"]), _view(out["dw"]), x, w, dtype, labels, _view(stats), _view(head),
                                   m, v, k, space, bias=bias, db=None if bias is None else _view(out["db"]),
                                   grad_dtype=dtype, grad_scale=s["loss_scale"], stream=stream)
        return out
    grads = [_view(g) for g in s["grads"]]
    head = torch.empty(2, device="cuda")
    space = _space(F.grad_norm_workspace_bytes())
    counts = [g.numel() for g in s["grads"]]
    if op == "norm":
        F.grad_norm_device(_view(head), grads, counts, dtype, _view(space), stream=stream)
        return head[0]
    F.clip_grads_device(_view(head), grads, counts, dtype, s["max_norm"], _view(space),
                        out=[_view(g) for g in s["parts"]], stream=stream)
    return {"norm": head[0], "grads": s["out"]}


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "embedding":
        return _embedding(state)
    if op == "embedding_grad":
        return _embedding_grad(state)
    if op == "norm":
        return _norm(state)
    if op == "clip":
        return _clip(state)
    return _linear_ce(state, op == "linear_ce_grad")


def work(case):
    op, size = case["op"], SIZES[case["dtype"]]
    if op == "embedding":       # the distinct rows that are read are at most the table's
        t, v, d = case["tokens"], case["vocab"], case["width"]
        return {"bytes": t * 4 + min(t, v) * d * size + t * d * size, "flops": t * d}
    if op == "embedding_grad":
        t, v, d = case["tokens"], case["vocab"], case["width"]
        return {"bytes": t * 4 + t * d * size + v * d * 4, "flops": 2 * t * d}
    if op.startswith("linear_ce"):
        m, v, k = case["rows"], case["vocab"], case["width"]
        bias = v * 4 if case["bias"] else 0
        if op == "linear_ce":
            return {"bytes": (m + v) * k * size + bias + m * 8, "flops": 2 * m * v * k}
        return {"bytes": 2 * (m + v) * k * size + 2 * bias + m * 8, "flops": 6 * m * v * k}
    n = sum(_counts(case))
    return {"bytes": n * size * (2 if op == "clip" else 1) + 4, "flops": (3 if op == "clip" else 2) * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embedding":
        return s["table"].double()[s["ids"].long()] * case["scale"]
    if op == "embedding_grad":
        keep = torch.ones(case["tokens"], dtype=torch.bool, device="cuda")
        if s["pad_id"] is not None:
            keep = s["ids"] != s["pad_id"]
        out = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
        order = torch.nonzero(keep)[:, 0]
        for part in order.split(8192):
            out.index_add_(0, s["ids"][part].long(), s["dout"][part].double())
        return out * case["scale"]
    if op in ("linear_ce", "linear_ce_grad"):
        m, v = case["rows"], case["vocab"]
        w = s["w"].double()
        count = max(1, int((s["labels"] >= 0).sum()))
        rows, dx = [], []
        dw, db = torch.zeros_like(w), torch.zeros(v, dtype=torch.float64, device="cuda")
        for i in range(0, m, 2048):      # rows are independent: a few at a time
            x, y = s["x"][i:i + 2048].double(), s["labels"][i:i + 2048].long()
            z = torch.mm(x, w.t())
            if s["bias"] is not None:
                z += s["bias"].double()
            live = (y >= 0).double()
            logp = torch.log_softmax(z, dim=1)
            hot = torch.nn.functional.one_hot(y.clamp(min=0), v) if m * v < 1 << 22 else None
            picked = (logp * hot).sum(1) if hot is not None else logp[torch.arange(len(y), device="cuda"), y.clamp(min=0)]
            rows.append(-picked * live)
            if op == "linear_ce_grad":
                p = logp.exp_()
                p[torch.arange(len(y), device="cuda"), y.clamp(min=0)] -= 1.0
                p *= (live * (s["loss_scale"] / count))[:, None]
                dx.append(torch.mm(p, w))
                dw += torch.mm(p.t(), x)
                db += p.sum(0)
        rows = torch.cat(rows)
        out = {"loss": rows.sum() / count, "rows": rows}
        if op == "linear_ce_grad":
            out["dx"], out["dw"] = torch.cat(dx), dw
            if s["bias"] is not None:
                out["db"] = db
        return out
    total = 0.0
    for g in s["grads"]:
        total += float(torch.linalg.vector_norm(g.double())) ** 2
    norm = torch.tensor(math.sqrt(total), dtype=torch.float64, device="cuda")
    if op == "norm":
        return norm
    coef = 1.0 if float(norm) <= s["max_norm"] else s["max_norm"] / float(norm)
    grads = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for g, part in zip(s["grads"], s["parts"]):
        start = part.storage_offset()
        grads[start:start + g.numel()] = g.double() * coef
    return {"norm": norm, "grads": grads}
