"""Plain 64-bit implementation of the microscaled 4-bit format and of expert
routing, on the CPU: what the GPU tests compare with."""
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def pack(x):
    """(codes uint8 [..., 16 * KB], scales uint8 [..., KB]) of x, by the definition in 64 bits."""
    cols = x.shape[-1]
    kb = -(-cols // 32)
    v = torch.zeros(*x.shape[:-1], kb * 32, dtype=torch.float64)
    v[..., :cols] = x.double()
    v = v.view(*x.shape[:-1], kb, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(top)
    exp = torch.frexp(torch.where(bad, 1.0, top))[1].double() - 1 - 2
    exp = torch.where(top == 0, torch.tensor(-127.0, dtype=torch.float64), exp).clamp(min=-127)
    a = v.abs() / torch.exp2(exp)[..., None]
    dist = (a[..., None] - GRID).abs()
    best = dist.min(-1, keepdim=True).values
    near = dist == best  # two grid values at a tie: the even code
    first = near.to(torch.uint8).argmax(-1)
    both = near.sum(-1) == 2
    code = torch.where(both & (first % 2 == 1), first + 1, first)
    code = code + 8 * torch.signbit(v).long()
    code = torch.where(bad[..., None], 0, code).flatten(-2).to(torch.uint8)
    scales = torch.where(bad, 255.0, exp + 127).to(torch.uint8)
    return code[..., ::2] | (code[..., 1::2] << 4), scales


def unpack(codes, scales, cols):
    """The values in float64."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = torch.where(c >= 8, -GRID[c & 7], GRID[c & 7]).unflatten(-1, (-1, 32))
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.tensor(float("nan"), dtype=torch.float64), s)
    return (v * s[..., None]).flatten(-2)[..., :cols]


def rounded(x):
    """Values of x after packing, float64."""
    return unpack(*pack(x.detach().cpu()), x.shape[-1])


def plan(ids, n_experts):
    """order, place, offsets of expert ids [tokens, top], lists by a loop."""
    flat = ids.reshape(-1).tolist()
    order, offsets = [], [0]
    for e in range(n_experts):
        order += [i for i, v in enumerate(flat) if v == e]
        offsets.append(len(order))
    place = [-1] * len(flat)
    for at, i in enumerate(order):
        place[i] = at
    order += [-1] * (len(flat) - len(order))
    return (torch.tensor(order, dtype=torch.int32), torch.tensor(place, dtype=torch.int32).view(ids.shape),
            torch.tensor(offsets, dtype=torch.int32))


def limit(dtype, ref, mass, terms):
    """Largest error a sum of `terms` exact products may have: float32
    additions (each within 2^-23 of the sum of magnitudes `mass`, twice
    rounding to nearest, for accumulators that truncate), then one rounding to dtype."""
    half_ulp = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    tiny = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[dtype]
    return terms * 2.0 ** -23 * mass + half_ulp * ref.abs() + tiny


def assert_close(got, ref, mass, terms):
    got64 = got.detach().cpu().double()
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got64), nan), "NaNs are not where the formula has them"
    err = (got64 - ref).abs()[~nan]
    room = limit(got.dtype, ref, mass, terms)[~nan]
    assert err.numel() == 0 or bool((err <= room).all()), \
        f"error {float((err - room).max()):.3g} above the bound (largest error {float(err.max()):.3g})"
