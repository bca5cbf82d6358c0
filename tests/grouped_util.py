"""Plain 64-bit forms of the grouped and 4-bit operators, and the bounds their outputs are held to.

Bound on a product's element.  The operands' products are exact in fp32 (11 + 11 or 8 + 8 bits, 4-bit
elements times powers of two), so the error comes from the K additions in fp32: each loses at most
one unit in the last place (2^-23, if it truncates) of a partial sum that never exceeds
S = sum |a_k| |b_k|.  One rounding to the output type follows: half a step, eps / 2 relative, and for
float16 at most half the subnormal spacing 2^-25 absolutely.  Together
    |got - want| <= K 2^-23 S + (eps / 2) (|want| + K 2^-23 S) + tiny.
"""
import torch

TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def assert_product(got, want, mag, K, what=""):
    """got: the kernel's output; want and mag: the product and the product of magnitudes in 64 bits."""
    assert got.shape == want.shape, what
    acc = max(K, 1) * 2.0 ** -23 * mag
    tol = acc + torch.finfo(got.dtype).eps / 2 * (want.abs() + acc) + TINY[got.dtype]
    excess = ((got.double() - want).abs() - tol)
    bad = ~(excess <= 0)
    assert not bad.any(), "%s: %d of %d outside, worst excess %g, first at %s" % (
        what, int(bad.sum()), bad.numel(), float(excess.max()), bad.nonzero()[0].tolist())


def clamped(offsets, T):
    """The row ranges of the groups as the operators define them."""
    o = [int(v) for v in offsets]
    out = []
    for a, b in zip(o, o[1:]):
        s = min(max(a, 0), T)
        out.append((s, min(max(b, s), T)))
    return out


def grouped(x, w, offsets):
    """(product, product of magnitudes, rows that some group owns)"""
    x, w = x.double(), w.double()
    T, N = x.shape[0], w.shape[1]
    y, m = (torch.zeros(T, N, dtype=torch.float64, device=x.device) for _ in range(2))
    own = torch.zeros(T, dtype=torch.bool, device=x.device)
    for e, (s, t) in enumerate(clamped(offsets, T)):
        y[s:t], m[s:t] = x[s:t] @ w[e].T, x[s:t].abs() @ w[e].abs().T
        own[s:t] = True
    return y, m, own


def grouped_dw(dy, x, offsets, E):
    dy, x = dy.double(), x.double()
    y, m = (torch.zeros(E, dy.shape[1], x.shape[1], dtype=torch.float64, device=x.device) for _ in range(2))
    for e, (s, t) in enumerate(clamped(offsets, dy.shape[0])):
        y[e], m[e] = dy[s:t].T @ x[s:t], dy[s:t].abs().T @ x[s:t].abs()
    return y, m


def scale_index(rows, K, offsets=None):
    """Place of every scale byte of a (rows, K) matrix, (rows, K/32); -1 for rows of no group."""
    kt = -(-K // 128)
    at = torch.full((rows, K // 32), -1, dtype=torch.int64)
    ranges = [(0, rows)] if offsets is None else clamped(offsets, rows)
    for g, (s, t) in enumerate(ranges):
        for r in range(s, t):
            local = r - s
            tile = (s // 128 + g if offsets is not None else 0) + local // 128
            for b in range(K // 32):
                at[r, b] = (tile * kt + b // 4) * 512 + (local % 32) * 16 + (local % 128) // 32 * 4 + b % 4
    return at


GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantise(x):
    """(rows, K) -> (scale bytes, element codes, values in 64 bits), by the definition: the nearest element,
    on a tie the one with the even code."""
    rows, K = x.shape
    v = x.double().cpu().reshape(rows, K // 32, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(top)
    _, e = torch.frexp(torch.where(bad, 1.0, top))
    s = torch.where(top > 0, e - 3, -127).clamp(min=-127)
    y = torch.where(bad[..., None], 0.0, v) / torch.exp2(s.double())[..., None]
    grid = torch.tensor(GRID, dtype=torch.float64)
    d = (y.abs()[..., None] - grid).abs()
    near = d == d.amin(-1, keepdim=True)
    idx = torch.arange(8)
    # among the nearest (one, or two on a tie) the even code
    code = torch.where(near, torch.where(idx % 2 == 0, idx, idx + 100), 1000).amin(-1) % 100
    values = torch.copysign(grid[code], y) * torch.exp2(s.double())[..., None]
    values = torch.where(bad[..., None], torch.nan, values)
    code = code + 8 * torch.signbit(y).long()
    byte = torch.where(bad, 255, s + 127).to(torch.uint8)
    return byte, code.reshape(rows, K).to(torch.uint8), values.reshape(rows, K)


def unpack(codes):
    """Packed bytes (..., K/2) -> element codes (..., K)."""
    return torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)


def offsets_of(counts, lead=0):
    """Row ranges of groups of these sizes behind `lead` rows of no group."""
    o = [lead]
    for c in counts:
        o.append(o[-1] + c)
    return o
