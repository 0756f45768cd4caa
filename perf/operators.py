"""Operators of microscaled 4-bit floating point and of expert layers: what a
program that uses them has them do, in plain torch and on the package's kernels.

A case is a dict of plain values; `kind` picks the operator, the rest gives its
sizes and types.

  pack      a tensor quantized to blocks of 32 E2M1 codes with one E8M0 scale
            each (mxfp4_quantize), and read back (dequantize)
  product   the product of two packed tensors, a @ b^T (mxfp4_matmul)
  linear    float activations through a weight: packed on the way, multiplied
            (mxfp4_linear); with `train` the weight is a float parameter and
            the gradients of both are taken
  experts   rows sorted by expert through each expert's own weight
            (expert_linear): packed weights and rows fetched by the plan when
            serving; with `train` float weights and both gradients
  dispatch  tokens sorted by expert and copied in that order (expert_sort,
            expert_gather), with `train` the gradient of the tokens
  combine   each token's expert rows weighted and added (expert_combine), with
            `train` the gradients of rows and weights

`run` computes the plain form (32-bit torch operations) or, where `own` is
true, calls the package.
"""
import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # activations of a decode batch, packed and read back: one launch each way
        {"name": "pack-tokens", "kind": "pack", "rows": 16, "cols": 4096, "src": "bf16"},
        # a large weight, an odd number of rows, packed for storage and read back
        {"name": "pack-weight", "kind": "pack", "rows": 16383, "cols": 8192, "src": "bf16"},
        # packed operands of a middle size, ragged rows and columns, an odd number of blocks
        {"name": "product-ragged", "kind": "product", "m": 1500, "n": 1800, "k": 2080, "out": "fp32"},
        # the large prefill product
        {"name": "product-8192", "kind": "product", "m": 8192, "n": 8192, "k": 8192, "out": "bf16"},
        # a decode step's projection for a batch of 16
        {"name": "linear-decode", "kind": "linear", "m": 16, "n": 8192, "k": 8192, "src": "bf16", "train": False},
        # one training step of a layer: forward, gradient of the tokens and of the weight
        {"name": "linear-train", "kind": "linear", "m": 4000, "n": 4096, "k": 4096, "src": "bf16", "train": True},
        # a decode step of an expert layer: few tokens, most experts with one or two of them or none
        {"name": "experts-decode", "kind": "experts", "tokens": 8, "top": 4, "experts": 32, "n": 4096, "k": 4096,
         "src": "bf16", "dropped": 0.0, "train": False},
        # prefill through an expert layer, uneven segments
        {"name": "experts-prefill", "kind": "experts", "tokens": 4000, "top": 4, "experts": 32, "n": 4096, "k": 2048,
         "src": "bf16", "dropped": 0.0, "train": False},
        # the order of a decode batch's tokens: latency of the sort and the copy
        {"name": "dispatch-decode", "kind": "dispatch", "tokens": 16, "top": 4, "experts": 64, "cols": 4096,
         "src": "bf16", "dropped": 0.0, "train": False},
        # a training batch over many experts, an eighth of the picks on another device's experts
        {"name": "dispatch-train", "kind": "dispatch", "tokens": 8192, "top": 8, "experts": 128, "cols": 2048,
         "src": "bf16", "dropped": 0.125, "train": True},
        # a decode batch's expert rows added
        {"name": "combine-decode", "kind": "combine", "tokens": 16, "top": 4, "experts": 64, "cols": 4096,
         "src": "bf16", "dropped": 0.0, "train": False},
        # the same of a training batch, with both gradients
        {"name": "combine-train", "kind": "combine", "tokens": 8000, "top": 4, "experts": 64, "cols": 4096,
         "src": "bf16", "dropped": 0.0, "train": True},
    ]


def _log(rng, lo, hi, step=1):
    """A size from lo to hi, even over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    kind = rng.choice(["pack", "product", "product", "linear", "linear", "experts", "experts", "dispatch", "combine"])
    src = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    step = rng.choice([1, 8, 128])
    if kind == "pack":
        cols = _log(rng, 32, 8192, rng.choice([1, 32, 128]))
        return {"kind": kind, "rows": _log(rng, 1, max(2, (1 << 27) // cols), 1), "cols": cols, "src": src}
    if kind == "product":
        return {"kind": kind, "m": _log(rng, 1, 8192, step), "n": _log(rng, 64, 8192, step),
                "k": _log(rng, 64, 8192, rng.choice([1, 32, 128])), "out": src}
    if kind == "linear":
        train = rng.random() < 0.4
        return {"kind": kind, "m": _log(rng, 16 if train else 1, 4000), "n": _log(rng, 128, 8192, step),
                "k": _log(rng, 128, 8192, rng.choice([8, 32, 128])), "src": src, "train": train}
    top = rng.choice([1, 2, 4, 8])
    if kind == "experts":
        train = rng.random() < 0.3
        return {"kind": kind, "tokens": _log(rng, 16 if train else 1, 2000), "top": top,
                "experts": rng.choice([8, 16, 32]), "n": _log(rng, 256, 4096, rng.choice([8, 128])),
                "k": _log(rng, 256, 4096, rng.choice([8, 32, 128])), "src": src,
                "dropped": rng.choice([0.0, 0.0, 0.5]), "train": train}
    return {"kind": kind, "tokens": _log(rng, 1, 8192), "top": top, "experts": rng.choice([8, 32, 64, 128, 256]),
            "cols": _log(rng, 256, 4096, rng.choice([1, 8, 128])), "src": src, "dropped": rng.choice([0.0, 0.0, 0.25]),
            "train": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _activations(g, shape, src):
    """Normal activations with a few large ones, as they meet a packed layer."""
    x = torch.randn(shape, generator=g, device=DEV)
    x[torch.rand(shape, generator=g, device=DEV) < 1e-3] *= 20.0
    return x.to(TYPES[src])


def _weights(g, shape, src):
    w = 0.02 * torch.randn(shape, generator=g, device=DEV)
    w[torch.rand(shape, generator=g, device=DEV) < 1e-3] *= 10.0
    return w.to(TYPES[src])


def _picks(g, case):
    """Each token's experts, unevenly liked, and their weights; -1: an expert that is not held here."""
    t, k, e = case["tokens"], case["top"], case["experts"]
    logits = torch.randn(t, e, generator=g, device=DEV) + 0.7 * torch.randn(e, generator=g, device=DEV)
    top = logits.topk(k, dim=1)
    ids = top.indices.masked_fill(torch.rand(t, k, generator=g, device=DEV) < case["dropped"], -1)
    return ids, top.values.softmax(1)


def _sorted(ids, e):
    """Picks in order of their experts (those without one last), each pick's place there, the experts' first places."""
    key = torch.where((ids < 0) | (ids >= e), e, ids).reshape(-1)
    order = key.sort(stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    place = torch.where(key < e, place, -1).view(ids.shape)
    first = (key[:, None] < torch.arange(e + 1, device=key.device)).sum(0)
    live = torch.arange(order.numel(), device=order.device) < first[-1]
    return torch.where(live, order, -1).int(), place.int(), first.int()


def _inputs(case, seed):
    """The tensors of a case, in the order that its state and its exact values take them."""
    g = _gen(seed)
    kind = case["kind"]
    if kind == "pack":
        return [_activations(g, (case["rows"], case["cols"]), case["src"])]
    if kind == "product":
        return [_activations(g, (case["m"], case["k"]), "fp32"), _weights(g, (case["n"], case["k"]), "fp32")]
    if kind == "linear":
        t = [_activations(g, (case["m"], case["k"]), case["src"]), _weights(g, (case["n"], case["k"]), case["src"])]
        return t + ([_activations(g, (case["m"], case["n"]), case["src"])] if case["train"] else [])
    ids, gates = _picks(g, case)
    r = ids.numel()
    if kind == "experts":
        rows = r if case["train"] else case["tokens"]
        t = [ids, _activations(g, (rows, case["k"]), case["src"]),
             _weights(g, (case["experts"], case["n"], case["k"]), case["src"])]
        return t + ([_activations(g, (r, case["n"]), case["src"])] if case["train"] else [])
    if kind == "dispatch":
        t = [ids, _activations(g, (case["tokens"], case["cols"]), case["src"])]
        return t + ([_activations(g, (r, case["cols"]), case["src"])] if case["train"] else [])
    t = [ids, gates, _activations(g, (r, case["cols"]), case["src"])]
    return t + ([_activations(g, (case["tokens"], case["cols"]), case["src"])] if case["train"] else [])


def prepare(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "pack":
        s["x"] = t[0]
    elif kind == "product":
        s["a"], s["b"] = _pack(t[0]), _pack(t[1])
    elif kind == "linear":
        s["x"] = t[0].requires_grad_(case["train"])
        s["w"] = t[1].requires_grad_(True) if case["train"] else _pack(t[1])
        s["dy"] = t[2] if case["train"] else None
    elif kind == "experts":
        s["plan"] = _sorted(t[0], case["experts"])
        s["x"] = t[1].requires_grad_(case["train"])
        s["w"] = t[2].requires_grad_(True) if case["train"] else _pack(t[2])
        s["dy"] = t[3] if case["train"] else None
    elif kind == "dispatch":
        s["ids"], s["x"], s["dy"] = t[0], t[1].requires_grad_(case["train"]), t[2] if case["train"] else None
    else:
        s["plan"] = _sorted(t[0], case["experts"])
        s["gates"], s["h"] = t[1].requires_grad_(case["train"]), t[2].requires_grad_(case["train"])
        s["dy"] = t[3] if case["train"] else None
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import qtpytorch_amd as qa

    case = s["case"]
    kind = case["kind"]
    train = case.get("train", False)
    if kind == "pack":
        q = qa.mxfp4_quantize(s["x"])
        return q.scales, q.dequantize(s["x"].dtype)
    if kind == "product":
        return qa.mxfp4_matmul(_held(qa, s["a"]), _held(qa, s["b"]), out_dtype=TYPES[case["out"]])
    if kind == "linear":
        y = qa.mxfp4_linear(s["x"], s["w"] if train else _held(qa, s["w"]))
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])) if train else y
    if kind == "experts":
        plan = qa.expert_plan(*s["plan"])
        y = qa.expert_linear(s["x"], s["w"] if train else _held(qa, s["w"]), plan, gather=not train)
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])) if train else y
    if kind == "dispatch":
        plan = qa.expert_sort(s["ids"], case["experts"])
        y = qa.expert_gather(s["x"], plan)
        out = (plan.order, plan.place, plan.offsets, y.detach())
        return (*out, *torch.autograd.grad(y, s["x"], s["dy"])) if train else out
    y = qa.expert_combine(s["h"], qa.expert_plan(*s["plan"]), s["gates"])
    return (y.detach(), *torch.autograd.grad(y, (s["h"], s["gates"]), s["dy"])) if train else y


def _held(qa, packed):
    codes, scales, cols = packed
    return qa.mxfp4_tensor(codes, scales, (*codes.shape[:-1], cols))


# ---------------------------------------------------------------- the plain forms
def _pack(x):
    """Codes (two a byte, the low half first), scale exponents + 127 and the columns of x, blocks of 32 along the last one."""
    cols = x.shape[-1]
    v = F.pad(x.detach().float(), (0, -cols % 32)).unflatten(-1, (-1, 32))
    top = v.abs().amax(-1)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    e = torch.where(top == 0, -127, e)
    whole = torch.isfinite(top)
    a = torch.ldexp(v.abs(), -e[..., None])
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = ((code + 8 * torch.signbit(v).to(torch.uint8)) * whole[..., None]).to(torch.uint8).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), torch.where(whole, e + 127, 255).to(torch.uint8), cols


def _unpack(packed):
    """The values of packed codes, in 32 bits."""
    codes, scales, cols = packed
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat([grid, -grid])
    v = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).flatten(-2).unflatten(-1, (-1, 32))
    v = torch.ldexp(v, scales[..., None].int() - 127)
    return torch.where(scales[..., None] == 255, math.nan, v).flatten(-2)[..., :cols]


def _slots(plan, e):
    """For rows sorted by expert: those in use, their places in [e, most rows of an expert], that number."""
    order, _, first = plan
    row = torch.arange(order.numel(), device=order.device)
    live = row < first[-1]
    expert = torch.searchsorted(first[1:].contiguous(), row.int(), right=True).clamp(max=e - 1)
    most = max(1, int((first[1:] - first[:-1]).max()))
    return live, (expert * most + row - first[expert])[live], most


def _spread(x, at, e, most):
    out = x.new_zeros(e * most, x.shape[1])
    out[at] = x
    return out.view(e, most, x.shape[1])


def _collect(y, live, at):
    out = y.new_zeros(live.numel(), y.shape[-1])
    out[live] = y.flatten(0, 1)[at]
    return out


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    train = case.get("train", False)
    if kind == "pack":
        q = _pack(s["x"])
        return q[1], _unpack(q).to(s["x"].dtype)
    if kind == "product":
        return (_unpack(s["a"]) @ _unpack(s["b"]).t()).to(TYPES[case["out"]])
    if kind == "linear":
        x = s["x"].detach()
        xq, wq = _unpack(_pack(x)), _unpack(_pack(s["w"]) if train else s["w"])
        y = (xq @ wq.t()).to(x.dtype)
        if not train:
            return y
        dy = s["dy"].float()
        return y, (dy @ wq).to(x.dtype), (dy.t() @ xq).to(s["w"].dtype)
    if kind == "experts":
        order = s["plan"][0]
        e = case["experts"]
        x = s["x"].detach()
        live, at, most = _slots(s["plan"], e)
        xq = _unpack(_pack(x))
        rows = xq[live] if train else xq[order[live] // case["top"]]
        xs = _spread(rows, at, e, most)
        wq = _unpack(_pack(s["w"]) if train else s["w"])
        y = _collect(torch.bmm(xs, wq.transpose(1, 2).contiguous()), live, at).to(x.dtype)
        if not train:
            return y
        dy = _spread(s["dy"].float()[live], at, e, most)
        dx = _collect(torch.bmm(dy, wq), live, at).to(x.dtype)
        return y, dx, torch.bmm(dy.transpose(1, 2).contiguous(), xs).to(s["w"].dtype)
    if kind == "dispatch":
        plan = _sorted(s["ids"], case["experts"])
        order, place, _ = plan
        x = s["x"].detach()
        y = torch.where(order[:, None] >= 0, x.float()[order.clamp(min=0) // case["top"]], 0.0).to(x.dtype)
        if not train:
            return (*plan, y)
        dx = torch.where(place[..., None] >= 0, s["dy"].float()[place.clamp(min=0)], 0.0).sum(1)
        return (*plan, y, dx.to(x.dtype))
    order, place, _ = s["plan"]
    gates, h = s["gates"].detach(), s["h"].detach()
    rows = torch.where(place[..., None] >= 0, h.float()[place.clamp(min=0)], 0.0)
    y = (gates[..., None] * rows).sum(1).to(h.dtype)
    if not train:
        return y
    dy = s["dy"].float()
    live, pick = order[:, None] >= 0, order.clamp(min=0)
    dh = torch.where(live, gates.reshape(-1)[pick][:, None] * dy[pick // case["top"]], 0.0)
    return y, dh.to(h.dtype), (rows * dy[:, None]).sum(-1)


# ---------------------------------------------------------------- what a pass cannot do without
def _packed_bytes(rows, cols):
    return rows * -(-cols // 32) * 17


def work(case):
    kind = case["kind"]
    train = case.get("train", False)
    if kind == "pack":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * BYTES[case["src"]] + _packed_bytes(case["rows"], case["cols"]), "flops": 0}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _packed_bytes(m + n, k) + m * n * BYTES[case["out"]], "flops": 2 * m * n * k}
    b = BYTES[case["src"]]
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        if train:  # x, w and dy read, y and both gradients written
            return {"bytes": 2 * (m * k + n * k + m * n) * b, "flops": 6 * m * n * k}
        return {"bytes": m * k * b + _packed_bytes(n, k) + m * n * b, "flops": 2 * m * n * k}
    e = case["experts"]
    r = case["tokens"] * case["top"]
    live = r * (1 - case["dropped"])  # as expected of the draw
    if kind == "experts":
        n, k = case["n"], case["k"]
        busy = e * (1 - (1 - 1 / e) ** live)
        if train:
            return {"bytes": (2 * r * k + 2 * r * n + (busy + e) * n * k) * b + 8 * r, "flops": 6 * live * n * k}
        return {"bytes": case["tokens"] * k * b + busy * _packed_bytes(n, k) + r * n * b + 4 * r,
                "flops": 2 * live * n * k}
    t, c = case["tokens"], case["cols"]
    if kind == "dispatch":
        rows = t * c + r * c + (live * c + t * c if train else 0)
        return {"bytes": rows * b + 8 * r + 8 * r + 4 * e, "flops": live * c if train else 0}
    # combine: rows, gates and places read, tokens written; the gradients read dy and write both
    rows = live * c + t * c + (t * c + r * c if train else 0)
    return {"bytes": rows * b + 8 * r + (8 * r if train else 0), "flops": (6 if train else 2) * live * c}


# ---------------------------------------------------------------- the same values in 64 bits
def _values64(x):
    """Scale bytes and values of x after packing, by the definition: scale 2^(floor(log2 of the block's largest) - 2),
    the nearest of the grid's values (the one with an even code where two are), at most 6."""
    cols = x.shape[-1]
    v = F.pad(x.detach().double(), (0, -cols % 32)).unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140)))
    e = torch.where(2.0 ** e > top, e - 1, e)
    e = torch.where(2.0 ** (e + 1) <= top, e + 1, e) - 2
    e = torch.where(top > 0, e.clamp(min=-127), -127.0)
    a = v.abs() * 2.0 ** -e
    # spacing of the grid at a: 1/2 below 2, 1 below 4, 2 above; round() takes ties to even multiples, as even codes are
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = ((a / step).round() * step).clamp(max=6.0)
    return (e[..., 0] + 127).to(torch.uint8), (torch.copysign(a, v) * 2.0 ** e).flatten(-2)[..., :cols]


def _by_expert(order, first):
    first = first.tolist()
    return [(i, first[i], first[i + 1]) for i in range(len(first) - 1) if first[i + 1] > first[i]]


def exact(case, seed):
    kind = case["kind"]
    train = case.get("train", False)
    t = _inputs(case, seed)
    if kind == "pack":
        return _values64(t[0])
    if kind == "product":
        return _values64(t[0])[1] @ _values64(t[1])[1].t().contiguous()
    if kind == "linear":
        xq, wq = _values64(t[0])[1], _values64(t[1])[1]
        y = xq @ wq.t().contiguous()
        return (y, t[2].double() @ wq, t[2].double().t().contiguous() @ xq) if train else y
    if kind == "experts":
        order, _, first = _sorted(t[0], case["experts"])
        xq = _values64(t[1])[1]
        y = torch.zeros(order.numel(), case["n"], dtype=torch.float64, device=DEV)
        dx = torch.zeros(order.numel(), case["k"], dtype=torch.float64, device=DEV) if train else None
        dw = torch.zeros(t[2].shape, dtype=torch.float64, device=DEV) if train else None
        for i, lo, hi in _by_expert(order, first):
            w = _values64(t[2][i])[1]
            rows = xq[lo:hi] if train else xq[(order[lo:hi] // case["top"]).long()]
            y[lo:hi] = rows @ w.t().contiguous()
            if train:
                dy = t[3][lo:hi].double()
                dx[lo:hi] = dy @ w
                dw[i] = dy.t().contiguous() @ rows
        return (y, dx, dw) if train else y
    order, place, first = _sorted(t[0], case["experts"])
    n, k, top = order.numel(), case["cols"], case["top"]
    live = int(first[-1])
    pick = order[:live].long()
    token = pick // top
    if kind == "dispatch":
        y = torch.zeros(n, k, dtype=torch.float64, device=DEV)
        y[:live] = t[1].double()[token]
        if not train:
            return None, None, None, y
        dx = torch.zeros(case["tokens"], k, dtype=torch.float64, device=DEV).index_add_(0, token, t[2][:live].double())
        return None, None, None, y, dx
    gates, h = t[1].double().reshape(-1), t[2][:live].double()
    y = torch.zeros(case["tokens"], k, dtype=torch.float64, device=DEV).index_add_(0, token, h * gates[pick, None])
    if not train:
        return y
    dy = t[3].double()[token]
    dh = torch.zeros(n, k, dtype=torch.float64, device=DEV)
    dh[:live] = dy * gates[pick, None]
    dg = torch.zeros(n, dtype=torch.float64, device=DEV)
    dg[pick] = (dy * h).sum(1)
    return y, dh, dg.view(t[1].shape)
