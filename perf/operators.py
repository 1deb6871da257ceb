"""The linear operators of the ``pulsar_cuda`` op surface, as measured cases.

Three operators: the plan that groups the router's assignments by expert
(``moe_group_rows``), the ragged products of the experts over such a plan
(``grouped_linear_forward`` / ``_backward``) and the dense product with its epilogue
(``fused_linear_forward`` / ``_backward``: bias, activation, residual). A training case runs an
operator forward and backward and returns every gradient; a serving case runs it forward.

The plain form is elementary torch in 32 bits, ``exact`` the definition in 64.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# relu is left out: its derivative steps at 0, so that a sum's last bit decides a gradient
ACTS = ("none", "silu", "gelu", "gelu_tanh", "sigmoid", "swiglu")
MAX_FLOPS = 4.5e11  # of a drawn case; the largest listed ones have 4.1e11 and 5.5e11


# --------------------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------------------

def listed():
    return [
        # The plan of one decoded token: launch latency.
        dict(name="group_1x4_e16", kind="group", tokens=1, top_k=4, experts=16, padded=0),
        # The plan of a training micro-batch of 8 x 2048 tokens, some of them padding.
        dict(name="group_16384x4_e16", kind="group", tokens=16384, top_k=4, experts=16,
             padded=311),
        # One decoded token through its 4 experts' gate/up products: weights streamed once.
        dict(name="experts_decode_1_bf16", kind="experts", tokens=1, top_k=4, experts=16,
             d_in=1024, d_out=1024, act="swiglu", bias=False, w_order="io", gather=True,
             dtype="bf16", train=False),
        # A serving batch of 256 sequences, a token each: about 64 rows an expert.
        dict(name="experts_decode_256_bf16", kind="experts", tokens=256, top_k=4, experts=16,
             d_in=1024, d_out=1024, act="swiglu", bias=False, w_order="io", gather=True,
             dtype="bf16", train=False),
        # The down product of a prompt of odd length, weights stored [out, in].
        dict(name="experts_down_517_bf16", kind="experts", tokens=517, top_k=4, experts=16,
             d_in=512, d_out=1024, act="none", bias=False, w_order="oi", gather=False,
             dtype="bf16", train=False),
        # The gate/up products of a training micro-batch of 8 x 2048 tokens, both ways.
        dict(name="experts_train_16384_bf16", kind="experts", tokens=16384, top_k=4, experts=16,
             d_in=1024, d_out=1024, act="swiglu", bias=False, w_order="io", gather=True,
             dtype="bf16", train=True),
        # fp32 training of a short ragged batch (parity runs).
        dict(name="experts_train_2331_fp32", kind="experts", tokens=2331, top_k=4, experts=16,
             d_in=1024, d_out=1024, act="swiglu", bias=False, w_order="io", gather=True,
             dtype="fp32", train=True),
        # The attention output projection of 16 decoded tokens onto the residual stream.
        dict(name="linear_decode_16_bf16", kind="linear", rows=16, d_in=1024, d_out=1024,
             act="none", bias=False, residual=True, dtype="bf16", train=False),
        # Odd sizes throughout: nothing is a multiple of a vector or a tile.
        dict(name="linear_odd_517_bf16", kind="linear", rows=517, d_in=1023, d_out=777,
             act="gelu", bias=True, residual=False, dtype="bf16", train=False),
        # The shared expert's gate/up product of a training micro-batch, both ways.
        dict(name="linear_train_16384_bf16", kind="linear", rows=16384, d_in=1024, d_out=2048,
             act="swiglu", bias=False, residual=False, dtype="bf16", train=True),
        # fp32 training of a short batch with bias and activation.
        dict(name="linear_train_2331_fp32", kind="linear", rows=2331, d_in=1024, d_out=1024,
             act="silu", bias=True, residual=True, dtype="fp32", train=True),
        # A wide feed-forward product over a long prefill: the largest.
        dict(name="linear_16384x2048x8192_bf16", kind="linear", rows=16384, d_in=2048,
             d_out=8192, act="gelu_tanh", bias=True, residual=False, dtype="bf16", train=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _width(rng, lo, hi):
    """A width: half the time a multiple of 64 as models have, else any (odd ones among them)."""
    n = _log_int(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["group", "experts", "experts", "experts", "linear", "linear"])
    if kind == "group":
        experts = _log_int(rng, 2, 256)
        tokens = _log_int(rng, 1, 16384)
        return dict(kind=kind, tokens=tokens, top_k=rng.randint(1, min(8, experts)),
                    experts=experts, padded=rng.randint(0, tokens // 8))
    while True:
        act = rng.choice(ACTS)
        case = dict(kind=kind, d_in=_width(rng, 16, 4096), d_out=_width(rng, 16, 4096), act=act,
                    bias=rng.random() < 0.5, dtype="bf16" if rng.random() < 0.75 else "fp32",
                    train=rng.random() < 0.5)
        if act == "swiglu":
            case["d_out"] += case["d_out"] % 2
        if kind == "experts":
            experts = _log_int(rng, 2, 64)
            case.update(tokens=_log_int(rng, 1, 16384), top_k=rng.randint(1, min(8, experts)),
                        experts=experts, w_order=rng.choice(["io", "oi"]),
                        gather=rng.random() < 0.6)
        else:
            case.update(rows=_log_int(rng, 1, 32768), residual=rng.random() < 0.5)
        w = work(case)
        if w["flops"] <= MAX_FLOPS * (1.0 if case["dtype"] == "bf16" else 0.1) \
                and w["bytes"] <= 1.0e9:
            return case


# --------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------

def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _topk_idx(g, tokens, top_k, experts):
    """Distinct experts of each token; some experts are more popular, as a trained router's."""
    score = torch.randn(tokens, experts, generator=g, device=DEV)
    score += 0.5 * torch.randn(experts, generator=g, device=DEV)
    return score.topk(top_k, dim=1).indices.contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "group":
        idx = _topk_idx(g, case["tokens"], case["top_k"], case["experts"])
        if case["padded"]:  # padding tokens route nowhere
            idx[torch.randperm(case["tokens"], generator=g, device=DEV)[:case["padded"]]] = -1
        return dict(case=case, idx=idx)
    dt, I, O = DTYPES[case["dtype"]], case["d_in"], case["d_out"]
    y_cols = O // 2 if case["act"] == "swiglu" else O
    s = dict(case=case)
    if case["kind"] == "experts":
        E = case["experts"]
        idx = _topk_idx(g, case["tokens"], case["top_k"], E)
        flat = idx.reshape(-1)
        order = torch.argsort(flat, stable=True)
        counts = torch.bincount(flat, minlength=E)
        offsets = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
        offsets[1:] = counts.cumsum(0)
        M = flat.numel()
        s["offsets"] = offsets
        s["bounds"] = offsets.tolist()  # what a plain program slices by
        s["rows"] = (order // case["top_k"]).to(torch.int32) if case["gather"] else None
        s["x"] = _randn(g, case["tokens"] if case["gather"] else M, I, dtype=dt)
        w = _randn(g, E, O, I, std=I ** -0.5, dtype=dt) if case["w_order"] == "oi" else \
            _randn(g, E, I, O, std=I ** -0.5, dtype=dt)
        s["w"] = w.transpose(1, 2) if case["w_order"] == "oi" else w
        s["bias"] = _randn(g, E, O, std=0.1, dtype=dt) if case["bias"] else None
    else:
        M = case["rows"]
        s["x"] = _randn(g, M, I, dtype=dt)
        s["w"] = _randn(g, O, I, std=I ** -0.5, dtype=dt)
        s["bias"] = _randn(g, O, std=0.1, dtype=dt) if case["bias"] else None
        s["residual"] = _randn(g, M, y_cols, dtype=dt) if case["residual"] else None
    if case["train"]:
        s["dy"] = _randn(g, M, y_cols, dtype=dt)
    return s


# --------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    _pkg = os.path.join(os.getcwd(), "pulsar-300m_amd")
    if _pkg not in sys.path:
        sys.path.insert(0, _pkg)
    import pulsar_cuda as pc

    case = s["case"]
    if case["kind"] == "group":
        offsets, rows, slots = pc.moe_group_rows(s["idx"], case["experts"])
        return dict(offsets=offsets, rows=rows, slots=slots)
    act, train = case["act"], case["train"]
    if case["kind"] == "experts":
        y = pc.grouped_linear_forward(s["x"], s["w"], s["offsets"], rows=s["rows"],
                                      bias=s["bias"], activation=act, save_pre=train)
        if not train:
            return dict(y=y)
        y, pre = y
        dx, dw, db = pc.grouped_linear_backward(s["dy"], s["x"], s["w"], s["offsets"],
                                                rows=s["rows"], pre=pre, activation=act,
                                                bias=case["bias"])
    else:
        y = pc.fused_linear_forward(s["x"], s["w"], bias=s["bias"], activation=act,
                                    residual=s["residual"], save_pre=train)
        if not train:
            return dict(y=y)
        y, pre = y
        dx, dw, db = pc.fused_linear_backward(s["dy"], s["x"], s["w"], pre=pre, activation=act,
                                              bias=case["bias"])
    out = dict(y=y, pre=pre, dx=dx, dw=dw)
    if case["bias"]:
        out["db"] = db
    return out


def _act(act, pre):
    if act == "none":
        return pre
    if act == "silu":
        return pre / (1 + torch.exp(-pre))
    if act == "gelu":
        return 0.5 * pre * (1 + torch.erf(pre * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * pre * (1 + torch.tanh(math.sqrt(2 / math.pi) * (pre + 0.044715 * pre ** 3)))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-pre))
    g, u = pre.chunk(2, dim=-1)
    return g / (1 + torch.exp(-g)) * u


def _act_grad(act, pre, dy):
    """The gradient of act at pre, times dy."""
    if act == "none":
        return dy
    if act == "swiglu":
        g, u = pre.chunk(2, dim=-1)
        sg = 1 / (1 + torch.exp(-g))
        return torch.cat([dy * u * sg * (1 + g * (1 - sg)), dy * g * sg], dim=-1)
    if act == "gelu":
        return dy * (0.5 * (1 + torch.erf(pre * math.sqrt(0.5)))
                     + pre * torch.exp(-0.5 * pre * pre) / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (pre + 0.044715 * pre ** 3))
        return dy * (0.5 * (1 + t) + 0.5 * pre * (1 - t * t) * c * (1 + 3 * 0.044715 * pre * pre))
    sg = 1 / (1 + torch.exp(-pre))
    return dy * sg * (1 - sg) if act == "sigmoid" else dy * sg * (1 + pre * (1 - sg))


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "group":
        flat = s["idx"].reshape(-1)
        E, K = case["experts"], case["top_k"]
        key = torch.where((flat >= 0) & (flat < E), flat, E)
        order = torch.argsort(key, stable=True)
        counts = torch.zeros(E + 1, dtype=torch.int64, device=DEV)
        counts.scatter_add_(0, key, torch.ones_like(key))
        offsets = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
        offsets[1:] = counts[:E].cumsum(0)
        pos = torch.arange(flat.numel(), device=DEV)
        rank = torch.empty_like(flat)
        rank[order] = pos
        rows = torch.where(pos < offsets[E], order // K, -1).to(torch.int32)
        slots = torch.where(key < E, rank, -1).to(torch.int32).view_as(s["idx"])
        return dict(offsets=offsets, rows=rows, slots=slots)
    dt, act, train = DTYPES[case["dtype"]], case["act"], case["train"]
    x, w = s["x"].float(), s["w"].float()
    if case["kind"] == "experts":
        if s["rows"] is not None:
            x = x[s["rows"]]
        spans = list(zip(s["bounds"][:-1], s["bounds"][1:]))
        pre = torch.cat([x[a:b] @ w[e] for e, (a, b) in enumerate(spans)])
        if case["bias"]:
            pre = torch.cat([pre[a:b] + s["bias"][e].float() for e, (a, b) in enumerate(spans)])
    else:
        pre = x @ w.t()
        if case["bias"]:
            pre = pre + s["bias"].float()
    y = _act(act, pre)
    if case["kind"] == "linear" and case["residual"]:
        y = y + s["residual"].float()
    if not train:
        return dict(y=y.to(dt))
    d = _act_grad(act, pre, s["dy"].float())
    out = dict(y=y.to(dt), pre=pre.to(dt))
    if case["kind"] == "experts":
        out["dx"] = torch.cat([d[a:b] @ w[e].t() for e, (a, b) in enumerate(spans)]).to(dt)
        out["dw"] = torch.stack([x[a:b].t() @ d[a:b] for a, b in spans]).to(dt)
        if case["bias"]:
            out["db"] = torch.stack([d[a:b].sum(0) for a, b in spans]).to(dt)
    else:
        out["dx"] = (d @ w).to(dt)
        out["dw"] = (d.t() @ x).to(dt)
        if case["bias"]:
            out["db"] = d.sum(0).to(dt)
    return out


# --------------------------------------------------------------------------------------
# Work and exact results
# --------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "group":
        m = case["tokens"] * case["top_k"]
        return dict(bytes=8 * m + 4 * m + 4 * m + 4 * (case["experts"] + 1), flops=0)
    es, I, O = (2 if case["dtype"] == "bf16" else 4), case["d_in"], case["d_out"]
    yc = O // 2 if case["act"] == "swiglu" else O
    if case["kind"] == "experts":
        m, E = case["tokens"] * case["top_k"], case["experts"]
        # experts that some token takes, of evenly routed tokens
        used = E * (1 - (1 - case["top_k"] / E) ** case["tokens"])
        x_rows = case["tokens"] if case["gather"] else m
        index = 4 * (E + 1) + (4 * m if case["gather"] else 0)
        bias, groups = (es * E * O if case["bias"] else 0), E
    else:
        m = x_rows = case["rows"]
        used, index, groups = 1, 0, 1
        bias = (es * O if case["bias"] else 0) + (es * m * yc if case["residual"] else 0)
    fwd = es * (x_rows * I + used * I * O + m * yc) + index + bias
    if not case["train"]:
        return dict(bytes=int(fwd), flops=2 * m * I * O)
    # backward, each input of the pass read once: dy in; pre, dx, dw, db out
    bwd = es * (m * yc + m * O + m * I + groups * I * O) + (es * groups * O if case["bias"] else 0)
    return dict(bytes=int(fwd + bwd), flops=6 * m * I * O)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "group":
        idx = s["idx"].cpu().numpy()
        E, (N, K) = case["experts"], s["idx"].shape
        lists = [[] for _ in range(E)]
        for i, e in enumerate(idx.reshape(-1).tolist()):
            if 0 <= e < E:
                lists[e].append(i)
        flat = np.array([i for e in lists for i in e], dtype=np.int64)
        offsets = np.cumsum([0] + [len(e) for e in lists]).astype(np.int32)
        rows = np.full(N * K, -1, dtype=np.int32)
        rows[:len(flat)] = flat // K
        slots = np.full(N * K, -1, dtype=np.int32)
        slots[flat] = np.arange(len(flat))
        return dict(offsets=torch.from_numpy(offsets).to(DEV), rows=torch.from_numpy(rows).to(DEV),
                    slots=torch.from_numpy(slots).view(N, K).to(DEV))
    x, w, act = s["x"].double(), s["w"].double(), case["act"]
    if case["kind"] == "linear":
        groups = [(0, case["rows"])]
        w = w.t()[None]
        bias = None if s["bias"] is None else s["bias"].double()[None]
    else:
        groups = list(zip(s["bounds"], s["bounds"][1:]))
        if s["rows"] is not None:
            x = x.index_select(0, s["rows"].long())
        bias = None if s["bias"] is None else s["bias"].double()
    pre = x.new_empty(x.shape[0], case["d_out"])
    for e, (a, b) in enumerate(groups):
        pre[a:b] = torch.mm(x[a:b], w[e])
        if bias is not None:
            pre[a:b] += bias[e]
    # the activation and its derivative, by name
    f = {"none": lambda t: t, "silu": lambda t: t * torch.sigmoid(t), "sigmoid": torch.sigmoid,
         "gelu": lambda t: t * torch.special.ndtr(t),
         "gelu_tanh": lambda t: t * torch.sigmoid(math.sqrt(8 / math.pi) * t
                                                  * (1 + 0.044715 * t * t)),
         "swiglu": lambda t: t[:, :t.shape[1] // 2] * torch.sigmoid(t[:, :t.shape[1] // 2])
         * t[:, t.shape[1] // 2:]}[act]
    leaf = pre.detach().requires_grad_(case["train"])
    y = f(leaf)
    out = dict(y=y.detach())
    if case["kind"] == "linear" and case["residual"]:
        out["y"] = out["y"] + s["residual"].double()
    if not case["train"]:
        return out
    (d,) = torch.autograd.grad(y, leaf, s["dy"].double())
    dx, dw = torch.empty_like(x), torch.zeros_like(w, memory_format=torch.contiguous_format)
    for e, (a, b) in enumerate(groups):
        dx[a:b] = torch.mm(d[a:b], w[e].t())
        dw[e] = torch.mm(x[a:b].t(), d[a:b])
    out.update(pre=pre, dx=dx, dw=dw[0].t().contiguous() if case["kind"] == "linear" else dw)
    if case["bias"]:
        db = torch.stack([d[a:b].sum(0) for a, b in groups])
        out["db"] = db[0] if case["kind"] == "linear" else db
    return out
