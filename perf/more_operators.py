"""Operators of serving from a paged 8-bit key-value cache, and of rotary
positions: what a program that uses them has them do, in plain torch and on
the package's kernels.

A case is a dict of plain values; `kind` picks the operator, the rest gives its
sizes and types.

  rotary  heads of tokens rotated by their positions, on one axis or on three
          (rotary); with `train` the gradient too
  append  new tokens' keys and values of a batch of sequences, keys and queries
          rotated, packed into pages (kv_pages.append), and read back (read)
  attend  attention of new tokens over their sequences' pages (kv_pages.attend):
          one token, a prompt's chunk, or a tree of drafted tokens
  keep    the accepted path of a tree of drafted tokens moved behind the context
          (kv_pages.keep), and read back

Pages are codes int8 [pages, 2, heads, page, D] (keys, values) and scales
float32 [pages, 2, heads, page]; a batch is the sequences' pages [B, pages],
the tokens that each holds [B], and the first of each one's new tokens [B + 1].

`run` computes the plain form (32-bit torch operations, angles and codes in 64)
or, where `own` is true, calls the package.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # queries of a decode batch rotated: latency of one call
        {"name": "rotary-decode", "kind": "rotary", "tokens": 16, "heads": 32, "dim": 128, "rotated": 128, "axes": 1,
         "interleaved": False, "far": 100000, "src": "bf16", "train": False},
        # a training batch of video and text: three axes, forward and gradient
        {"name": "rotary-train", "kind": "rotary", "tokens": 8190, "heads": 32, "dim": 128, "rotated": 128, "axes": 3,
         "interleaved": False, "far": 0, "src": "bf16", "train": True},
        # a decode batch's step: one token of each sequence into the cache
        {"name": "append-decode", "kind": "append", "seqs": 16, "new": 1, "ctx": 4000, "idle": 0.0, "heads": 8,
         "group": 4, "dim": 128, "page": 16, "axes": 1, "interleaved": False, "src": "bf16"},
        # prompts of several lengths, rotated pair by pair, in 32 bits
        {"name": "append-ragged", "kind": "append", "seqs": 9, "new": 300, "ctx": 1000, "idle": 0.2, "heads": 4,
         "group": 1, "dim": 64, "page": 32, "axes": 1, "interleaved": True, "src": "fp32"},
        # a long prompt of images and text (three axes) into an empty cache
        {"name": "append-prompt", "kind": "append", "seqs": 2, "new": 6000, "ctx": 0, "idle": 0.0, "heads": 8,
         "group": 4, "dim": 128, "page": 64, "axes": 3, "interleaved": False, "src": "bf16"},
        # one sequence, one token, a short context: latency
        {"name": "attend-one", "kind": "attend", "seqs": 1, "new": 1, "ctx": 1000, "idle": 0.0, "heads": 8, "group": 4,
         "dim": 128, "page": 16, "tree": False, "src": "bf16"},
        # a decode batch of uneven contexts
        {"name": "attend-decode", "kind": "attend", "seqs": 64, "new": 1, "ctx": 8192, "idle": 0.0, "heads": 8,
         "group": 4, "dim": 128, "page": 16, "tree": False, "src": "bf16"},
        # few sequences with very long contexts
        {"name": "attend-long", "kind": "attend", "seqs": 2, "new": 1, "ctx": 130003, "idle": 0.0, "heads": 8,
         "group": 8, "dim": 128, "page": 64, "tree": False, "src": "bf16"},
        # trees of drafted tokens over a batch's contexts
        {"name": "attend-tree", "kind": "attend", "seqs": 12, "new": 50, "ctx": 5000, "idle": 0.1, "heads": 8,
         "group": 4, "dim": 128, "page": 32, "tree": True, "src": "fp16"},
        # chunks of two prompts behind what is held of them
        {"name": "attend-chunk", "kind": "attend", "seqs": 2, "new": 2000, "ctx": 6000, "idle": 0.0, "heads": 8,
         "group": 4, "dim": 128, "page": 64, "tree": False, "src": "bf16"},
        # accepted paths of a batch's trees: latency of the move
        {"name": "keep-decode", "kind": "keep", "seqs": 16, "new": 48, "path": 6, "ctx": 2000, "heads": 8, "dim": 128,
         "page": 16},
        # long paths of many sequences
        {"name": "keep-batch", "kind": "keep", "seqs": 250, "new": 64, "path": 16, "ctx": 500, "heads": 16, "dim": 128,
         "page": 32},
    ]


def _log(rng, lo, hi, step=1):
    """A size from lo to hi, even over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "append", "append", "attend", "attend", "attend", "attend", "attend", "keep"])
    src = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64, 128])
    axes = rng.choice([1, 1, 2, 3])
    if kind == "rotary":
        dim = rng.choice([64, 72, 80, 96, 128, 128, 256])
        heads = _log(rng, 1, 64)
        return {"kind": kind, "tokens": _log(rng, 1, min(8190, (1 << 24) // (heads * dim))), "heads": heads, "dim": dim,
                "rotated": rng.choice([dim, dim, dim // 2]), "axes": axes, "interleaved": rng.random() < 0.3,
                "far": rng.choice([0, 1000, 1000000]), "src": src, "train": rng.random() < 0.5}
    heads, group = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([1, 2, 3, 4, 4, 6, 8, 16])
    if kind == "append":
        seqs = _log(rng, 1, 200)
        most = max(1, min(6000, (1 << 24) // (seqs * heads * (group + 2) * dim)))
        return {"kind": kind, "seqs": seqs, "new": rng.choice([1, _log(rng, 1, most)]), "ctx": rng.choice([0, 3000]),
                "idle": rng.choice([0.0, 0.3]), "heads": heads, "group": group, "dim": dim, "page": page, "axes": axes,
                "interleaved": rng.random() < 0.3, "src": src}
    if kind == "keep":
        new = _log(rng, 2, 128)
        return {"kind": kind, "seqs": _log(rng, 1, 250), "new": new, "path": _log(rng, 1, max(1, min(16, new // 2))),
                "ctx": _log(rng, 1, 1000), "heads": heads, "dim": dim, "page": page}
    # keys, and pairs of a query head and a key, bounded: the plain form holds a score for each pair
    tree = rng.random() < 0.4
    one = not tree and rng.random() < 0.55
    seqs = _log(rng, 1, 64)
    new = 1 if one else _log(rng, 2, 128) if tree else _log(rng, 2, 2000)
    keys = (1 << 28) // (seqs * heads * dim)
    pairs = (1 << 28) // (seqs * heads * group * new)
    most = max(new + 16, min(keys, pairs, 130000))
    while seqs * heads * group * new * (most + new) > 1 << 28 and new > 1:
        new = new // 2
        most = max(new + 16, most // 2)
    return {"kind": kind, "seqs": seqs, "new": new, "ctx": rng.choice([0, 1, 1, 1]) and _log(rng, 1, most),
            "idle": rng.choice([0.0, 0.0, 0.3]), "heads": heads, "group": group, "dim": dim, "page": page, "tree": tree,
            "src": src}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _sizes(case):
    """Tokens held and new tokens of each sequence: of the case alone, so that all its states have the same shapes.
    The first has both at their largest; an idle sequence (finished, its place not yet given away) has no new token."""
    r = random.Random("sizes %d %d %d" % (case["seqs"], case["new"], case["ctx"]))
    ctx, new = [], []
    for b in range(case["seqs"]):
        idle = b > 0 and r.random() < case.get("idle", 0.0)
        ctx.append(case["ctx"] if b == 0 else int(case["ctx"] * r.uniform(0.05, 1.0)))
        n = case["new"] if b == 0 or case["kind"] == "keep" else max(1, int(case["new"] * r.uniform(0.4, 1.0)))
        new.append(0 if idle else n)
    return ctx, new


def _tokens(case):
    return sum(_sizes(case)[1])


def _batch(g, case):
    """The sequences' pages in a shuffled pool, the tokens they hold, the first of each one's new tokens."""
    ctx, new = _sizes(case)
    p = case["page"]
    pages = [-(-(c + n) // p) for c, n in zip(ctx, new)]
    width, pool = max(1, max(pages)), sum(pages) + 3
    order = torch.randperm(pool, generator=g, device=DEV)
    need = torch.tensor(pages, device=DEV)
    at = torch.arange(width, device=DEV)
    first = need.cumsum(0) - need
    table = torch.where(at < need[:, None], order[(first[:, None] + at).clamp(max=pool - 1)], -1).int()
    lengths = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    offsets = torch.tensor([0] + new, device=DEV).cumsum(0).int()
    return table, lengths, offsets, pool


def _pool(g, case, pool, held):
    """Pages as they lie in memory; where nothing is held yet they are what their memory held before, here NaN.
    A sequence's first token is often attended and has small values."""
    shape = (pool, 2, case["heads"], case["page"])
    codes = torch.empty(*shape, case["dim"], device=DEV, dtype=torch.int8)
    for i in range(0, pool, 4096):  # the random values of a few pages at a time
        part = codes[i:i + 4096]
        part.copy_((40 * torch.randn(part.shape, generator=g, device=DEV)).round_().clamp_(-127, 127))
    scales = (torch.rand(shape, generator=g, device=DEV) + 0.5) / 40
    if held is not None:
        table, total = held
        b, s = _positions(total)
        page, off = _places(case, table, b, s)
        live = torch.zeros(pool, 1, 1, case["page"], dtype=torch.bool, device=DEV)
        live[page, 0, 0, off] = True
        scales = torch.where(live, scales, math.nan)
        start = table[:, 0][total > 0].long()
        scales[start, 1, :, 0] *= 0.05
    return codes, scales


def _positions(counts):
    """(sequence, index in it) of each of counts[b] things of sequences b, one sequence after the other."""
    counts = counts.long()
    b = torch.repeat_interleave(torch.arange(counts.numel(), device=counts.device), counts)
    return b, torch.arange(b.numel(), device=b.device) - (counts.cumsum(0) - counts)[b]


def _places(case, table, b, s):
    return table[b, s // case["page"]].long(), s % case["page"]


def _table(case, rotated):
    """Radians per position and the axis of each pair; the axes share the pairs out, a quarter to the first of three."""
    pairs, axes = rotated // 2, case["axes"]
    i = torch.arange(pairs, dtype=torch.float64, device=DEV)
    freqs = 1e6 ** (-i / max(1, pairs))
    first = pairs // 4 if axes == 3 else pairs // axes
    axis = (i >= first).int() if axes > 1 else i.int() * 0
    return freqs, axis + (i >= first + (pairs - first) // 2).int() if axes == 3 else axis


def _axes(g, case, base):
    """Positions [tokens, axes]: text advances all axes, an image its rows and columns."""
    n = base.numel()
    p = base.long()[:, None].repeat(1, case["axes"])
    if case["axes"] > 1:
        image = torch.rand(n, 1, generator=g, device=DEV) < 0.5
        p = torch.where(image, p // 2 + torch.randint(0, 60, p.shape, generator=g, device=DEV), p)
    return p


def _values(g, shape, src):
    """Normal activations with a few large ones."""
    x = torch.randn(shape, generator=g, device=DEV)
    x[..., :2] *= 6.0
    return x.to(TYPES[src])


def _inputs(case, seed):
    """The tensors of a case by name."""
    g = _gen(seed)
    kind = case["kind"]
    if kind == "rotary":
        t = {}
        t["freqs"], t["axis"] = _table(case, case["rotated"])
        n = case["tokens"]
        start = torch.randint(case["far"], case["far"] + 5, (1,), generator=g, device=DEV)
        t["pos"] = _axes(g, case, start + torch.arange(n, device=DEV))
        t["x"] = _values(g, (n, case["heads"], case["dim"]), case["src"])
        t["dy"] = _values(g, (n, case["heads"], case["dim"]), case["src"]) if case["train"] else None
        return t
    table, lengths, offsets, pool = _batch(g, case)
    t = {"table": table, "lengths": lengths, "offsets": offsets}
    n = _tokens(case)
    h, d = case["heads"], case["dim"]
    if kind == "keep":
        t["codes"], t["scales"] = _pool(g, case, pool, (table, lengths + case["new"]))
        # the root, then one drafted token of each further level
        last, lo = case["path"], min(case["path"], case["new"] - 1)
        path = lo + torch.rand(case["seqs"], case["new"] - lo, generator=g, device=DEV).argsort(1)[:, :last]
        path = path.sort(1).values
        path = torch.cat([path, path.new_full((case["seqs"], last - path.shape[1]), -1)], 1)
        path[:, 0] = 0
        few = torch.randint(1, last + 1, (case["seqs"], 1), generator=g, device=DEV)
        t["path"] = torch.where(torch.arange(last, device=DEV) < few, path, -1).int()
        return t
    if kind == "append":
        t["codes"], t["scales"] = _pool(g, case, pool, None)
        t["freqs"], t["axis"] = _table(case, d)
        b, i = _positions(offsets.diff())
        t["pos"] = _axes(g, case, lengths[b] + i)
        t["k"], t["v"] = _values(g, (n, h, d), case["src"]), _values(g, (n, h, d), case["src"])
        t["q"] = _values(g, (n, h * case["group"], d), case["src"])
        return t
    t["codes"], t["scales"] = _pool(g, case, pool, (table, lengths + offsets.diff()))
    q = 1.5 * torch.randn(n, h * case["group"], d, generator=g, device=DEV)
    t["q"] = q.to(TYPES[case["src"]])
    t["mask"] = _tree(seed, case, offsets) if case["tree"] else None
    return t


def _tree(seed, case, offsets):
    """Words of bits [tokens, words]: a drafted token sees itself and the tokens on its way from the root."""
    r = random.Random(int(seed))
    words = -(-case["new"] // 64)
    rows = []
    for n in offsets.diff().tolist():
        seen = []
        for i in range(n):
            up = seen[r.randrange(max(0, i - 8), i)] if i else 0
            seen.append(up | 1 << i)
        rows += [[_signed(m >> 64 * w & (1 << 64) - 1) for w in range(words)] for m in seen]
    return torch.tensor(rows, dtype=torch.int64, device=DEV).view(-1, words)


def _signed(word):
    return word - (1 << 64) if word >> 63 else word


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "rotary":
        s["x"].requires_grad_(case["train"])
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import qtpytorch_amd as qa

    case = s["case"]
    kind = case["kind"]
    if kind == "rotary":
        table = qa.rotary_table(s["freqs"], s["axis"], interleaved=case["interleaved"])
        y = qa.rotary(s["x"], s["pos"], table)
        return (y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]) if case["train"] else y
    pages = qa.kv_pages(s["codes"], s["scales"])
    batch = qa.kv_batch(s["table"], s["lengths"], s["offsets"])
    if kind == "append":
        table = qa.rotary_table(s["freqs"], s["axis"], interleaved=case["interleaved"])
        q = pages.append(s["k"], s["v"], batch, rotary=table, positions=s["pos"], q=s["q"])
        return (q, *pages.read(batch, s["k"].shape[0]))
    if kind == "attend":
        return pages.attend(s["q"], batch, mask=s["mask"])
    pages.keep(batch, s["path"])
    n = case["path"]
    first = torch.arange(0, case["seqs"] * n + 1, n, dtype=torch.int32, device=s["path"].device)
    return pages.read(qa.kv_batch(s["table"], s["lengths"], first), case["seqs"] * n)


# ---------------------------------------------------------------- the plain forms
def _rotate(x, pos, freqs, axis, interleaved, back=False, wide=False):
    """x [tokens, heads, D] rotated, in 32 bits (64 where wide); angles in 64."""
    a = pos.double()[:, axis.long()] * freqs
    kind = torch.float64 if wide else torch.float32
    c, s = a.cos().to(kind)[:, None], (-a.sin() if back else a.sin()).to(kind)[:, None]
    r = 2 * freqs.numel()
    x = x.detach().to(kind)
    u, w = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    both = (u * c - w * s, w * c + u * s)
    y = torch.stack(both, -1).flatten(-2) if interleaved else torch.cat(both, -1)
    return torch.cat([y, x[..., r:]], -1)


def _pack(x):
    """Codes and scales of rows of 64-bit values."""
    scale = x.abs().amax(-1, keepdim=True).clamp(min=1e-12) / 127
    return (x / scale).round().clamp(-127, 127).to(torch.int8), scale[..., 0].float()


def _read(s, counts, at, src):
    """Keys and values of the counts[b] positions from at[b] on."""
    b, i = _positions(counts)
    page, off = _places(s["case"], s["table"], b, at.long()[b] + i)
    both = s["codes"][page, :, :, off].float() * s["scales"][page, :, :, off, None]
    return both[:, 0].to(src), both[:, 1].to(src)


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "rotary":
        how = (s["pos"], s["freqs"], s["axis"], case["interleaved"])
        y = _rotate(s["x"], *how).to(s["x"].dtype)
        return (y, _rotate(s["dy"], *how, back=True).to(s["x"].dtype)) if case["train"] else y
    if kind == "append":
        how = (s["pos"], s["freqs"], s["axis"], case["interleaved"])
        b, i = _positions(s["offsets"].diff())
        page, off = _places(case, s["table"], b, s["lengths"].long()[b] + i)
        for which, x in ((0, _rotate(s["k"], *how, wide=True)), (1, s["v"].double())):
            s["codes"][page, which, :, off], s["scales"][page, which, :, off] = _pack(x)
        return (_rotate(s["q"], *how).to(s["q"].dtype), *_read(s, s["offsets"].diff(), s["lengths"], torch.bfloat16))
    if kind == "attend":
        return _attend_plain(s)
    path = s["path"].long()
    at = s["lengths"].long()[:, None]
    b, j = (path >= 0).nonzero(as_tuple=True)
    from_page, from_off = _places(case, s["table"], b, (at + path)[b, j])
    to_page, to_off = _places(case, s["table"], b, at[b, 0] + j)
    codes, scales = s["codes"][from_page, :, :, from_off], s["scales"][from_page, :, :, from_off]
    s["codes"][to_page, :, :, to_off], s["scales"][to_page, :, :, to_off] = codes, scales
    return _read(s, torch.full_like(s["lengths"], case["path"]), s["lengths"], torch.bfloat16)


def _attend_plain(s):
    case = s["case"]
    heads, group, d = case["heads"], case["group"], case["dim"]
    held, new = s["lengths"].long()[:, None], s["offsets"].diff().long()
    most, wide = case["new"], case["ctx"] + case["new"]  # the first sequence has the most of both
    key = torch.arange(wide, device=DEV)
    b = torch.arange(case["seqs"], device=DEV)[:, None]
    page, off = _places(case, s["table"], b, key.expand(case["seqs"], wide))
    live = key < held + new[:, None]
    page = torch.where(live, page, 0)
    both = s["codes"][page, :, :, off].float() * torch.where(live[..., None, None], s["scales"][page, :, :, off],
                                                             0.0)[..., None]
    k, v = both[:, :, 0].permute(0, 2, 1, 3).contiguous(), both[:, :, 1].permute(0, 2, 1, 3).contiguous()
    i = torch.arange(most, device=DEV)
    row = (s["offsets"][:-1, None].long() + i).clamp(max=s["q"].shape[0] - 1)  # [B, most]
    q = s["q"].float()[row].view(-1, most, heads, group, d).permute(0, 2, 1, 3, 4).reshape(-1, heads, most * group, d)
    score = q @ k.transpose(2, 3).contiguous() / math.sqrt(d)
    j = (key - held)[:, None]  # [B, 1, keys]
    if s["mask"] is None:
        seen = j <= i[:, None]
    else:
        words = s["mask"][row]  # [B, most, words]
        at = j.clamp(0, 64 * words.shape[-1] - 1).expand(-1, most, -1)
        seen = (j < 0) | (words.gather(2, at // 64) >> at % 64 & 1).bool()
    seen = (seen & live[:, None])[:, None, :, None]
    score = torch.where(seen, score.view(-1, heads, most, group, wide), -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True)).view(-1, heads, most * group, wide)
    o = (p @ v / p.sum(-1, keepdim=True)).view(-1, heads, most, group, d).permute(0, 2, 1, 3, 4)
    at, i = _positions(new)
    return o[at, i].reshape(-1, heads * group, d).to(s["q"].dtype)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "rotary":
        n = case["tokens"] * case["heads"] * case["dim"]
        times = 2 if case["train"] else 1
        return {"bytes": times * (2 * n * BYTES[case["src"]] + 8 * case["tokens"] * case["axes"]),
                "flops": times * 3 * n * case["rotated"] // case["dim"]}
    ctx, new = _sizes(case)
    n, h, d = sum(new), case["heads"], case["dim"]
    if kind == "append":
        b = BYTES[case["src"]]
        rows, heads = 2 * n * h, n * h * case["group"]
        # keys, values and queries read, codes, scales and queries written; codes and scales read, values written
        return {"bytes": (rows + 2 * heads) * d * b + 2 * rows * (d + 4) + rows * d * 2, "flops": (rows + heads) * 3 * d}
    if kind == "keep":
        moved = case["seqs"] * case["path"] * 2 * h
        return {"bytes": 2 * moved * (d + 4) + moved * (d + 4) + moved * d * 2, "flops": 0}
    keys = sum(c + k for c, k in zip(ctx, new) if k)
    pairs = sum(k * c + k * (k + 1) // 2 for c, k in zip(ctx, new))
    q = n * h * case["group"] * d * BYTES[case["src"]]
    return {"bytes": keys * 2 * h * (d + 4) + 2 * q, "flops": 4 * d * h * case["group"] * pairs}


# ---------------------------------------------------------------- the same values in 64 bits
def _turned64(x, t, case, sign=1.0):
    """Each pair as a complex number times e^(i angle)."""
    x = x.detach().double()
    out = x.clone()
    r = 2 * t["freqs"].numel()
    at = torch.arange(r // 2, device=x.device)
    one, two = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + r // 2)
    angle = sign * t["pos"].double().index_select(1, t["axis"].long()) * t["freqs"]
    z = torch.complex(x[..., one], x[..., two]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    out[..., one], out[..., two] = z.real, z.imag
    return out


def _coded64(x):
    step = x.abs().amax(-1, keepdim=True).clamp(min=1e-12) / 127.0
    return (x / step).round() * step


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        y = _turned64(t["x"], t, case)
        return (y, _turned64(t["dy"], t, case, -1.0)) if case["train"] else y
    if kind == "append":
        return _turned64(t["q"], t, case), _coded64(_turned64(t["k"], t, case)), _coded64(t["v"].double())
    ctx, new = _sizes(case)
    p, h, d = case["page"], case["heads"], case["dim"]

    def rows(b, n):
        """Keys and values [2, heads, n, D] of sequence b's first n positions."""
        pages = t["table"][b, :-(-n // p)].long()
        both = t["codes"][pages].double() * t["scales"][pages].double()[..., None]
        return both.permute(1, 2, 0, 3, 4).reshape(2, h, -1, d)[:, :, :n]

    if kind == "keep":
        out = torch.zeros(2, case["seqs"], case["path"], h, d, dtype=torch.float64, device=DEV)
        for b, path in enumerate(t["path"].tolist()):
            both = rows(b, ctx[b] + new[b])
            at = [ctx[b] + (j if at < 0 else at) for j, at in enumerate(path)]
            out[:, b] = both[:, :, at].transpose(1, 2)
        return out[0].reshape(-1, h, d), out[1].reshape(-1, h, d)
    out, at = [], 0
    for b in range(case["seqs"]):
        n = new[b]
        if not n:
            continue
        k, v = rows(b, ctx[b] + n)
        q = t["q"][at:at + n].double().view(n, h, case["group"], d)
        if t["mask"] is None:
            seen = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        else:
            bit = torch.arange(64, device=DEV)
            seen = (t["mask"][at:at + n, :, None] >> bit & 1).flatten(1)[:, :n].bool()
        seen = torch.cat([torch.ones(n, ctx[b], dtype=torch.bool, device=DEV), seen], 1)
        for i in range(0, n, 256):  # a part of the rows at a time
            part = q[i:i + 256].permute(1, 2, 0, 3).reshape(h, -1, d)
            score = torch.bmm(part, k.transpose(1, 2).contiguous()) * d ** -0.5
            score = score.view(h, case["group"], -1, ctx[b] + n).masked_fill(~seen[i:i + 256], -math.inf)
            o = torch.bmm(score.softmax(-1).view(h, -1, ctx[b] + n), v)
            out.append(o.view(h, case["group"], -1, d).permute(2, 0, 1, 3).reshape(-1, h * case["group"], d))
        at += n
    return torch.cat(out)
