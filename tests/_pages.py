"""Plain 64-bit implementation of rotary positions and of a paged 8-bit
key-value cache, on the CPU: what the GPU tests compare with."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rotate(x, pos, freqs, axis, interleaved, sign=1.0):
    """x [tokens, heads, D] and positions [tokens, axes] in float64; also |u| + |w| of each element's pair."""
    x = x.double()
    n = freqs.numel()
    angle = sign * pos.double()[:, axis.long()] * freqs  # [tokens, pairs]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    i = torch.arange(n)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    y, size = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def rotation_error(want, size, dtype):
    """Angle to 2^-26 of a turn and its sine to 2^-22, three roundings in float32, one to dtype."""
    return 2.0 ** -21 * size + want.abs() * HALF[dtype] + LEAST[dtype]


def near(got, want, error):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    bad = ((got - want).abs() > error) & ~nan
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / error)[bad].max()), bad.nonzero()[:4].tolist())


class Batch:
    """Sequences with `held` positions and `new` tokens each, their pages shuffled; `front` and `back` rows of padding."""

    def __init__(self, held, new, page, seed=0, spare=2, front=0, back=0, width=None):
        self.held, self.new, self.page = list(held), list(new), page
        need = [-(-(h + n) // page) for h, n in zip(self.held, self.new)]
        self.width = max([1] + need) if width is None else width
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=gen(seed)).tolist()
        self.table = torch.full((len(need), self.width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                page = order.pop()
                if i < self.width:
                    self.table[b, i] = page
        first = [front]
        for n in self.new:
            first.append(first[-1] + n)
        self.first, self.tokens = first, first[-1] + back

    def gpu(self):
        import qtpytorch_amd as qa
        return qa.kv_batch(self.table.cuda(), torch.tensor(self.held, dtype=torch.int32).cuda(),
                           torch.tensor(self.first, dtype=torch.int32).cuda())

    def place(self, b, at):
        """(page, position in it) or None."""
        run = at // self.page
        page = int(self.table[b, run]) if 0 <= at and run < self.width else -1
        return (page, at % self.page) if 0 <= page < self.pages else None


def pool(batch, heads, dim, seed=0, poison=True):
    """Codes and scales, NaN scales where no position of a sequence lies."""
    g = gen(seed + 100)
    shape = (batch.pages, 2, heads, batch.page)
    codes = (40 * torch.randn(*shape, dim, generator=g)).round().clamp(-127, 127).to(torch.int8)
    scales = (torch.rand(shape, generator=g) + 0.5) / 40
    if poison:
        live = torch.zeros(batch.pages, batch.page, dtype=torch.bool)
        for b, (h, n) in enumerate(zip(batch.held, batch.new)):
            for at in range(h + n):
                if batch.place(b, at):
                    live[batch.place(b, at)] = True
        scales = torch.where(live[:, None, None], scales, math.nan)
    return codes, scales


def rows(batch, codes, scales, b, count):
    """Keys and values [2, heads, count, D] of sequence b's positions in float64, and which are there."""
    out = torch.zeros(2, codes.shape[2], count, codes.shape[4], dtype=torch.float64)
    there = torch.zeros(count, dtype=torch.bool)
    for at in range(count):
        p = batch.place(b, at)
        if p:
            out[:, :, at] = codes[p[0], :, :, p[1]].double() * scales[p[0], :, :, p[1], None].double()
            there[at] = True
    return out, there


def seen(batch, b, mask):
    """[new, held + new]: which positions each new token of sequence b sees, before pages that are not there."""
    h, n = batch.held[b], batch.new[b]
    out = torch.zeros(n, h + n, dtype=torch.bool)
    out[:, :h] = True
    for i in range(n):
        for j in range(n):
            if mask is None:
                out[i, h + j] = j <= i
            else:
                word = int(mask[batch.first[b] + i, j // 64]) if j // 64 < mask.shape[1] else 0
                out[i, h + j] = bool(word >> (j % 64) & 1)
    return out


def attend(batch, codes, scales, q, mask=None, scale=None):
    """Results [tokens, q_heads, D] in float64 and how far a kernel that rounds as documented may be off."""
    T, Hq, D = q.shape
    H = codes.shape[2]
    scale = D ** -0.5 if scale is None else scale
    dtype = q.dtype
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    error = torch.zeros(T, Hq, D, dtype=torch.float64)
    q_step = 0.5 / (8323072 if dtype == torch.float32 else 32512)  # of a row's largest element
    p_step = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11
    for b in range(len(batch.held)):
        n = batch.new[b]
        if not n:
            continue
        (k, v), there = rows(batch, codes, scales, b, batch.held[b] + n)
        see = seen(batch, b, mask) & there
        for hq in range(Hq):
            kk, vv = k[hq // (Hq // H)], v[hq // (Hq // H)]
            x = q[batch.first[b]:batch.first[b] + n, hq].double()
            s = torch.where(see, scale * (x @ kk.t()), -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(torch.isinf(top), 0.0, top)), 0.0)
            total = p.sum(1, keepdim=True)
            vz = torch.where(see[..., None], vv[None], 0.0)  # [n, keys, D]
            o = (p[..., None] * vz).sum(1) / total
            o = torch.where(total == 0, 0.0, o)
            # scores: the query's integers, float32 products (log2 units, so relative to the score) and the exponential's
            # argument; probabilities rounded; small ones in float16's subnormal steps, 2^-34 of the largest value
            ds = scale * q_step * x.abs().amax(1, keepdim=True) * kk.abs().sum(1) + 2.0 ** -21 * (s.abs() + 1)
            ds = torch.where(see, ds, 0.0).amax(1, keepdim=True)
            mean = torch.where(total == 0, 0.0, (p[..., None] * vz.abs()).sum(1) / total)
            least = see.sum(1, keepdim=True) * 2.0 ** -34 * vz.abs().amax((1, 2))[:, None] if vz.shape[1] else 0.0
            err = mean * (2 * torch.expm1(2 * ds) + p_step + 2.0 ** -20) + least + o.abs() * HALF[dtype] + LEAST[dtype]
            at = slice(batch.first[b], batch.first[b] + n)
            out[at, hq], error[at, hq] = o, err
    return out, error
