"""Cases that measure the operators of a language-model student: embedding and its gradient, the gated Linear pair forward
and backward, the distillation loss with its gradient.

Inputs are torch tensors on the GPU.  With `own` false, run() computes an operator in elementary torch operations; with
`own` true it calls the framework's C entry points on the same memory.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f64": torch.float64}
ITEM = {"f32": 4, "f64": 8, "i32": 4, "i64": 8}
ACTIVATIONS = ("silu", "gelu", "sigmoid")  # not relu: its derivative jumps at 0, where a last bit decides a whole gradient


def listed():
    return [
        # a generation step of a small batch: one token a sequence
        dict(name="embed_step", op="embed", dtype="f32", index="i64", count=8, vocab=32000, dim=1024),
        # the prompt tokens of a large batch in one call, a vocabulary that is not a round number
        dict(name="embed_prompts", op="embed", dtype="f32", index="i32", count=65536, vocab=100003, dim=2048),
        # gradient of a training batch: 16 sequences of 512 tokens, word frequencies falling as 1 / rank
        dict(name="embed_grad", op="embed_grad", dtype="f32", index="i64", count=8192, vocab=32000, dim=1024),
        # a small vocabulary, every token many times over; rows that are no whole vectors
        dict(name="embed_grad_odd", op="embed_grad", dtype="f64", index="i32", count=4001, vocab=997, dim=333),
        # one token through the gated pair while generating
        dict(name="gated_token", op="gated", dtype="f32", rows=1, inner=1024, hidden=4096, act="silu", bias=False, grad=False),
        # the 784-feature, 1024-wide, batch-1024 layer of the framework's MLP as a gated layer, training
        dict(name="gated_mlp", op="gated", dtype="f32", rows=1024, inner=784, hidden=1024, act="silu", bias=True, grad=True),
        # a training batch through a four times wider gated pair
        dict(name="gated_wide", op="gated", dtype="f32", rows=4096, inner=1024, hidden=4096, act="gelu", bias=False, grad=True),
        # double precision, ragged in every direction
        dict(name="gated_f64", op="gated", dtype="f64", rows=777, inner=500, hidden=1001, act="sigmoid", bias=True, grad=True),
        # the MLP's ten outputs at batch 1024
        dict(name="distill_classes", op="distill", dtype="f32", index="i32", rows=1024, vocab=10, top=4, temperature=2.0),
        # a training batch over a 32000-word vocabulary
        dict(name="distill_words", op="distill", dtype="f32", index="i64", rows=2048, vocab=32000, top=64, temperature=2.0),
        # the largest: 4096 positions over 131072 words
        dict(name="distill_large", op="distill", dtype="f32", index="i64", rows=4096, vocab=131072, top=128, temperature=1.5),
        # few positions over a long vocabulary, rows that begin off a vector's boundary
        dict(name="distill_few", op="distill", dtype="f64", index="i32", rows=7, vocab=100003, top=33, temperature=1.0),
    ]


def _distinct(count, vocab):
    """How many different tokens `count` draws of prepare()'s distribution are expected to hold."""
    p = np.diff(np.log1p(np.arange(vocab + 1, dtype=np.float64))) / math.log1p(vocab)
    return int(round(float(np.sum(-np.expm1(count * np.log1p(-np.minimum(p, 1 - 1e-15)))))))


def _log(rng, low, high):
    """A whole number, even in its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """A case of the listed ones' ranges.  Sizes that make it dearer than the dearest of them are cut down row by row."""
    op = rng.choice(("embed", "embed_grad", "gated", "gated", "distill", "distill"))
    dtype = rng.choice(("f32", "f32", "f64"))
    index = rng.choice(("i32", "i64"))
    if op in ("embed", "embed_grad"):
        case = dict(op=op, dtype=dtype, index=index, count=_log(rng, 1, 65536), vocab=_log(rng, 10, 131072), dim=_log(rng, 8, 2048))
        if rng.random() < 0.5:
            case["dim"] = max(8, case["dim"] // 8 * 8)
        while work(case)["bytes"] > 1.5e9:
            case["count"], case["vocab"] = case["count"] // 2 + 1, case["vocab"] // 2 + 10
        return case
    if op == "gated":
        case = dict(op=op, dtype=dtype, rows=_log(rng, 1, 4096), inner=_log(rng, 16, 2048), hidden=_log(rng, 16, 8192),
                    act=rng.choice(ACTIVATIONS), bias=rng.random() < 0.5, grad=rng.random() < 0.6)
        if rng.random() < 0.5:
            case["inner"], case["hidden"] = (case["inner"] + 15) // 16 * 16, (case["hidden"] + 15) // 16 * 16
        while work(case)["flops"] > (2e11 if dtype == "f32" else 1e11):
            case["rows"] = case["rows"] // 2 + 1
        return case
    case = dict(op=op, dtype=dtype, index=index, rows=_log(rng, 1, 4096), vocab=_log(rng, 10, 131072), temperature=rng.choice((1.0, 1.5, 2.0, 4.0)))
    if rng.random() < 0.5:
        case["vocab"] = (case["vocab"] + 7) // 8 * 8
    case["top"] = min(case["vocab"], _log(rng, 1, 256))
    while work(case)["bytes"] > 4e9:
        case["rows"] = case["rows"] // 2 + 1
    return case


def work(case):
    op, e = case["op"], ITEM[case["dtype"]]
    if op == "embed":
        # the indices, every row that is looked up once, the result
        return {"bytes": case["count"] * ITEM[case["index"]] + (_distinct(case["count"], case["vocab"]) + case["count"]) * case["dim"] * e,
                "flops": case["count"] * case["dim"]}
    if op == "embed_grad":
        return {"bytes": case["count"] * ITEM[case["index"]] + (case["count"] + case["vocab"]) * case["dim"] * e,
                "flops": case["count"] * case["dim"]}
    if op == "gated":
        r, i, h = case["rows"], case["inner"], case["hidden"]
        moved = r * i + 2 * i * h + r * h + (2 * h if case["bias"] else 0)
        if case["grad"]:
            moved += r * h + r * i + 2 * i * h + (2 * h if case["bias"] else 0)
        return {"bytes": moved * e, "flops": (12 if case["grad"] else 4) * r * i * h}
    r, v, k = case["rows"], case["vocab"], case["top"]
    return {"bytes": 2 * r * v * e + r * k * (e + ITEM[case["index"]]) + r * e + e, "flops": 5 * r * v}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=dt)  # noqa: E731
    if op in ("embed", "embed_grad"):
        count, vocab, dim = case["count"], case["vocab"], case["dim"]
        # rank falls off as in text: P(rank <= r) = log(1 + r) / log(1 + vocab), the ranks shuffled over the vocabulary
        u = torch.rand(count, generator=gen, device="cuda", dtype=torch.float64)
        rank = (torch.exp(u * math.log1p(vocab)) - 1).long().clamp_(0, vocab - 1)
        ids = torch.randperm(vocab, generator=gen, device="cuda")[rank]
        state = dict(case=case, index=ids.to(torch.int32) if case["index"] == "i32" else ids, scale=math.sqrt(dim))
        if op == "embed":
            state["table"] = normal(vocab, dim) * 0.02
        else:
            state["dy"] = normal(count, dim) * 0.01
        return state
    if op == "gated":
        r, i, h = case["rows"], case["inner"], case["hidden"]
        state = dict(case=case, x=normal(r, i), wg=normal(i, h) * i ** -0.5, wu=normal(i, h) * i ** -0.5, bg=None, bu=None)
        if case["bias"]:
            state["bg"], state["bu"] = normal(h) * 0.1, normal(h) * 0.1
        if case["grad"]:
            state["dh"] = normal(r, h) * 0.01
        return state
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    z = normal(rows, vocab) * 2
    # the teacher's largest logits: distinct words, a little more likely under the student too, falling off
    first = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
    step = torch.arange(top, device="cuda") * max(1, vocab // top)
    ids = (first + step) % vocab
    teacher = normal(rows, top) + 6 - 0.05 * torch.arange(top, device="cuda", dtype=dt)
    z.scatter_add_(1, ids, 0.5 * teacher)
    weight = (torch.rand(rows, generator=gen, device="cuda") < 0.9).to(dt) / rows  # padding positions weigh nothing
    weight[0] = 1 / rows
    return dict(case=case, z=z, ids=ids.to(torch.int32) if case["index"] == "i32" else ids, teacher=teacher, weight=weight)


# ---- the framework's calls: its C entry points, on the tensors' memory and torch's current stream ------------------------


def _ok(status, capi):
    if status:
        raise RuntimeError(capi.last_error())


def _at(t):
    return None if t is None else t.data_ptr()


def _view(capi, t):
    v = capi.View2()
    v.data = t.data_ptr()
    v.stride[0], v.stride[1] = t.stride()
    return v


def _scratch(capi, query, *args):
    need = ctypes.c_size_t()
    _ok(query(*args, ctypes.byref(need)), capi)
    return torch.empty(max(need.value, 1), device="cuda", dtype=torch.uint8), need.value


def _run_own(s):
    from tinytensor_amd import _capi as capi

    lib, case = capi.lib, s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    code = capi.F32 if dt is torch.float32 else capi.F64
    new = lambda *shape: torch.empty(shape, device="cuda", dtype=dt)  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    if op == "embed":
        index, table = s["index"], s["table"]
        count, vocab, dim = case["count"], case["vocab"], case["dim"]
        out = new(count, dim)
        _ok(lib.ttamd_embedding_forward(0, code, capi.I32 if index.dtype is torch.int32 else capi.I64, count, vocab, dim, _at(index),
                                        _at(table), dim, 1, s["scale"], _at(out), stream), capi)
        return out
    if op == "embed_grad":
        index, count, vocab, dim = s["index"], case["count"], case["vocab"], case["dim"]
        icode = capi.I32 if index.dtype is torch.int32 else capi.I64
        out = new(vocab, dim)
        ws, size = _scratch(capi, lib.ttamd_embedding_backward_workspace, code, count, vocab, dim)
        _ok(lib.ttamd_embedding_backward(0, code, icode, count, vocab, dim, _at(s["dy"]), _at(index), s["scale"], 0, _at(out), _at(ws), size,
                                         stream), capi)
        return out
    if op == "gated":
        r, i, h, act, grad = case["rows"], case["inner"], case["hidden"], capi.ACT[case["act"]], case["grad"]
        x, wg, wu = (_view(capi, s[n]) for n in ("x", "wg", "wu"))
        x, wg, wu = ctypes.byref(x), ctypes.byref(wg), ctypes.byref(wu)
        out, gate, up = new(r, h), new(r, h) if grad else None, new(r, h) if grad else None
        ws, size = _scratch(capi, lib.ttamd_gated_linear_workspace, code, r, i, h, 0)
        _ok(lib.ttamd_gated_linear_forward(0, code, act, r, i, h, x, wg, wu, _at(s["bg"]), _at(s["bu"]), _at(out), _at(gate), _at(up),
                                           _at(ws), size, stream), capi)
        if not grad:
            return out
        dx, dwg, dwu = new(r, i), new(i, h), new(i, h)
        dbg, dbu = (new(h), new(h)) if case["bias"] else (None, None)
        ws, size = _scratch(capi, lib.ttamd_gated_linear_workspace, code, r, i, h, 1)
        _ok(lib.ttamd_gated_linear_backward(0, code, act, r, i, h, _at(s["dh"]), x, wg, wu, _at(gate), _at(up), _at(dx), _at(dwg), _at(dwu),
                                            _at(dbg), _at(dbu), _at(ws), size, stream), capi)
        return [out, dx, dwg, dwu] + ([dbg, dbu] if case["bias"] else [])
    z, ids, rows, vocab, top = s["z"], s["ids"], case["rows"], case["vocab"], case["top"]
    loss, dz = new(1), new(rows, vocab)
    ws, size = _scratch(capi, lib.ttamd_distill_loss_workspace, code, rows, vocab, top)
    _ok(lib.ttamd_distill_loss(0, code, capi.I32 if ids.dtype is torch.int32 else capi.I64, rows, vocab, top, _at(z), vocab, _at(ids),
                               _at(s["teacher"]), _at(s["weight"]), case["temperature"], _at(loss), _at(dz), _at(ws), size, stream), capi)
    return [loss, dz]


# ---- the plain forms -----------------------------------------------------------------------------------------------------


def _activate(g, act):
    """act(g) and its derivative."""
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    sig = 1 / (1 + torch.exp(-g))
    if act == "sigmoid":
        return sig, sig * (1 - sig)
    return g * sig, sig * (1 + g * (1 - sig))


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "embed":
        return s["table"][s["index"]] * s["scale"]
    if op == "embed_grad":
        total = torch.zeros((case["vocab"], case["dim"]), device="cuda", dtype=s["dy"].dtype)
        return total.index_add_(0, s["index"], s["dy"]).mul_(s["scale"])
    if op == "gated":
        x, wg, wu = s["x"], s["wg"], s["wu"]
        g, u = x @ wg, x @ wu
        if case["bias"]:
            g, u = g + s["bg"], u + s["bu"]
        a, da = _activate(g, case["act"])
        h = a * u
        if not case["grad"]:
            return h
        dg, du = s["dh"] * u * da, s["dh"] * a
        dx = dg @ wg.t() + du @ wu.t()
        out = [h, dx, x.t() @ dg, x.t() @ du]
        return out + [dg.sum(0), du.sum(0)] if case["bias"] else out
    t, ids = case["temperature"], s["ids"].long()
    weight = s["weight"][:, None]
    zt = (s["z"] - s["z"].amax(1, keepdim=True)) / t
    e = torch.exp(zt)
    total = e.sum(1, keepdim=True)
    tt_ = (s["teacher"] - s["teacher"].amax(1, keepdim=True)) / t
    pe = torch.exp(tt_)
    psum = pe.sum(1, keepdim=True)
    p = pe / psum
    log_p, log_q = tt_ - torch.log(psum), zt.gather(1, ids) - torch.log(total)
    row = (t * t) * (p * (log_p - log_q)).sum(1)
    loss = (s["weight"].double() * row.double()).sum().to(s["z"].dtype).reshape(1)
    dz = e * (weight * t / total)
    dz.scatter_add_(1, ids, -(weight * t) * p)
    return [loss, dz]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = {n: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for n, v in s.items()}
    if op == "embed":
        return torch.index_select(d["table"], 0, d["index"].long()).mul_(d["scale"])
    if op == "embed_grad":
        # rows sorted by token, each token's run added up by itself
        order = torch.argsort(d["index"].long(), stable=True)
        lengths = torch.bincount(d["index"].long(), minlength=case["vocab"])
        return torch.segment_reduce(d["dy"][order], "sum", lengths=lengths, initial=0.0).mul_(d["scale"])
    if op == "gated":
        x = d["x"].clone().requires_grad_(True)
        ws = [d[n].clone().requires_grad_(True) for n in ("wg", "wu")]
        bs = [d[n].clone().requires_grad_(True) for n in ("bg", "bu")] if case["bias"] else [None, None]
        pre = [x.mm(w) if b is None else torch.addmm(b, x, w) for w, b in zip(ws, bs)]
        act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid}[case["act"]]
        h = act(pre[0]) * pre[1]
        if not case["grad"]:
            return h.detach()
        leaves = [x] + ws + (bs if case["bias"] else [])
        return [h.detach()] + list(torch.autograd.grad(h, leaves, d["dh"]))
    t, ids = case["temperature"], d["ids"].long()
    p = torch.softmax(d["teacher"] / t, 1)
    log_q = torch.log_softmax(d["z"] / t, 1)
    row = t * t * (torch.xlogy(p, p) - p * log_q.gather(1, ids)).sum(1)
    dz = log_q.exp_()
    for j in range(ids.shape[1]):
        dz[torch.arange(case["rows"], device="cuda"), ids[:, j]] -= p[:, j]
    return [(d["weight"] * row).sum().reshape(1), dz.mul_(d["weight"][:, None] * t)]
