"""The operators of a mixture of experts and of 4-bit inference that heron_b200.kernels offers, as
cases to be timed and compared.

Operators (``op`` of a case):

  grouped      y[r] = w[e(r)] @ x[r]: matrix products grouped by expert over ragged runs of rows
  grouped_bwd  its gradients: dx[r] = w[e(r)]^T @ dy[r] and dw[e] = sum over e's rows of dy[r] x[r]^T
  quant        a matrix to microscaled 4-bit floating point (blocks of 32 along a row, E2M1 elements,
               one power-of-two scale in E8M0 per block) and read back as values
  mx           product of two such matrices, C = A @ B^T; with ``quantise`` the activations arrive in 16
               bits and are quantised within the pass (a linear layer with 4-bit weights)
  grouped_mx   the grouped product with 4-bit weights; the activations are quantised within the pass

``own`` selects the framework's kernels; otherwise ``run`` computes the plain form with elementary
torch operations in 32 bits.
"""
import math
import random

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decoding step of a small batch: four tokens, four or fewer experts hit; weights dominate
        dict(name="grouped_decode_4", op="grouped", T=4, E=16, K=2048, N=1024, dtype="bf16", routing=1),
        # odd sizes, several experts without a row, K not a multiple of a tile
        dict(name="grouped_ragged_odd", op="grouped", T=1003, E=24, K=712, N=1001, dtype="f16", routing=2),
        # a prompt's rows over 32 experts
        dict(name="grouped_prefill", op="grouped", T=8192, E=32, K=2048, N=2048, dtype="bf16", routing=3),
        # a training step's gradients of one expert layer
        dict(name="grouped_bwd_train", op="grouped_bwd", T=8192, E=16, K=1024, N=2048, dtype="bf16", routing=4),
        # a small odd one: most runs end inside a tile
        dict(name="grouped_bwd_odd", op="grouped_bwd", T=777, E=20, K=520, N=328, dtype="f16", routing=5),
        # activations of a long prompt, quantised and read back
        dict(name="quant_prompt", op="quant", M=8192, K=4096, dtype="bf16"),
        # few rows in 32 bits, K not a multiple of the scales' tile
        dict(name="quant_few_rows", op="quant", M=33, K=1056, dtype="f32"),
        # the square product of the GEMM benchmark, both operands in 4 bits
        dict(name="mx_square", op="mx", M=4096, K=4096, N=4096, dtype="bf16", quantise=False),
        # one token through a linear layer with 4-bit weights
        dict(name="mx_one_token", op="mx", M=1, K=4096, N=4096, dtype="bf16", quantise=True),
        # sixteen tokens through 4-bit experts
        dict(name="grouped_mx_decode", op="grouped_mx", T=16, E=32, K=2048, N=2048, dtype="bf16", routing=6),
        # a prompt through 4-bit experts, odd row count
        dict(name="grouped_mx_prefill", op="grouped_mx", T=6001, E=32, K=2048, N=2048, dtype="bf16", routing=7),
    ]


def _log(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return max(lo, min(hi // step * step, v))


def draw(rng):
    op = rng.choice(["grouped", "grouped", "grouped_bwd", "quant", "mx", "mx", "grouped_mx"])
    if op == "quant":
        return dict(op=op, M=_log(rng, 1, 8192), K=_log(rng, 32, 4096, 32), dtype=rng.choice(["bf16", "f16", "f32"]))
    if op == "mx":
        return dict(op=op, M=_log(rng, 1, 4096), K=_log(rng, 64, 4096, 32), N=_log(rng, 64, 4096),
                    dtype=rng.choice(["bf16", "f16"]), quantise=rng.random() < 0.6)
    E = _log(rng, 1, 48)
    step = 32 if op == "grouped_mx" else 8
    K, N = _log(rng, 64, 2048, step), _log(rng, 64, 2048, 8 if op == "grouped_bwd" else 1)
    T = _log(rng, 1, 4096 if op == "grouped_bwd" else 8192)
    return dict(op=op, T=T, E=E, K=K, N=N, dtype=rng.choice(["bf16", "f16"]), routing=rng.randrange(1 << 20))


def _counts(case):
    """Rows per expert, a skewed draw; its multiset belongs to the case, its order to the seed."""
    rng = random.Random(case["routing"])
    p = [math.exp(0.5 * rng.gauss(0, 1)) for _ in range(case["E"])]
    n = [0] * case["E"]
    for e in rng.choices(range(case["E"]), weights=p, k=case["T"]):
        n[e] += 1
    return n


# ---- the 4-bit format -----------------------------------------------------------------------
# A block of 32 values along a row: scale 2^s with s = floor(log2(largest magnitude)) - 2, at least
# -127; elements round(x / 2^s) to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to the even code,
# larger ones to 6).  A block with a value that is not finite has the scale code 255 and reads back
# as NaN.  Two elements to a byte, the even one in the low half.  The scales lie in tiles of
# 128 rows x 4 blocks: byte (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4 of tile (r / 128, b / 4).
def _scale_at(tile_row, local, blocks, kt):
    """Place of the scales of rows (tile row, row within it) and all blocks, (rows, blocks)."""
    b = torch.arange(blocks, device=local.device)
    return ((tile_row * kt)[:, None] + b // 4) * 512 + ((local % 32) * 16 + local // 32 * 4)[:, None] + b % 4


def _rows_at(M, device):
    r = torch.arange(M, device=device)
    return r // 128, r % 128


def _group_rows_at(offsets, T):
    """The same for rows grouped by expert: group g's tiles start at tile row offsets[g] / 128 + g."""
    r = torch.arange(T, device=offsets.device)
    g = torch.searchsorted(offsets[1:].contiguous(), r.to(offsets.dtype), right=True)
    first = offsets.long()[g]
    return first // 128 + g + (r - first) // 128, (r - first) % 128


def _plain_quantise(x):
    """(M, K) -> element codes (M, K) and scale codes (M, K/32)."""
    M, K = x.shape
    v = x.float().reshape(M, K // 32, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(top)
    _, e = torch.frexp(torch.where(bad, 1.0, top))
    s = torch.where(top > 0, e - 3, -127).clamp(-127, 127)
    y = torch.ldexp(torch.where(bad[..., None], 0.0, v), -s[..., None])
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * torch.signbit(y).int()
    return code.reshape(M, K).to(torch.uint8), torch.where(bad, 255, s + 127).to(torch.uint8)


def _plain_values(code, scale):
    """Codes (..., K) and scale codes (..., K/32) -> the values they stand for, in 32 bits."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    s = torch.where(scale == 255, math.nan, torch.exp2(scale.float() - 127))
    v = table[code.int()].reshape(*scale.shape, 32) * s[..., None]
    return v.reshape(code.shape)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], packed.shape[-1] * 2)


def _pack(code, scale):
    """Codes (B, M, K) and scale codes (B, M, K/32) -> the layout that the operators take."""
    B, M, K = code.shape
    mt, kt = -(-M // 128), -(-K // 128)
    at = _scale_at(*_rows_at(M, code.device), K // 32, kt)
    out = torch.zeros(B, mt * kt * 512, dtype=torch.uint8, device=code.device)
    out[:, at.reshape(-1)] = scale.reshape(B, -1)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), out


def _plain_unpacked(packed, scales, M, K):
    """The values of a packed operand: (B, M, K/2) and (B, bytes) -> (B, M, K) in 32 bits."""
    at = _scale_at(*_rows_at(M, packed.device), K // 32, -(-K // 128))
    return _plain_values(_unpack(packed), scales[:, at])


# ---- inputs ------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def activations(M, K):  # channels of different strength, as a layer's inputs have
        return (randn(M, K) * torch.exp(0.5 * randn(K))).to(dt)

    op, s = case["op"], dict(case=case, dt=dt)
    K = case["K"]
    if op == "quant":
        s["x"] = activations(case["M"], K)
        return s
    if op == "mx":
        M, N = case["M"], case["N"]
        w, ws = _pack(*(t[None] for t in _plain_quantise(randn(N, K) / math.sqrt(K))))
        s["w"], s["ws"] = w[0], ws[0]
        s["x"] = activations(M, K)
        if not case["quantise"]:
            x, xs = _pack(*(t[None] for t in _plain_quantise(s["x"])))
            s["x"], s["xs"] = x[0], xs[0]
        return s
    T, E, N = case["T"], case["E"], case["N"]
    n = _counts(case)
    random.Random(seed).shuffle(n)
    ends = [0]
    for c in n:
        ends.append(ends[-1] + c)
    s["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    s["longest"] = max(n)
    if op == "grouped_mx":
        wq = [_plain_quantise(randn(N, K) / math.sqrt(K)) for _ in range(E)]
        s["w"], s["ws"] = _pack(torch.stack([c for c, _ in wq]), torch.stack([c for _, c in wq]))
        s["x"] = activations(T, K)
        return s
    s["w"] = torch.empty(E, N, K, dtype=dt, device="cuda")
    for e in range(E):
        s["w"][e] = randn(N, K) / math.sqrt(K)
    s["x"] = activations(T, K)
    if op == "grouped_bwd":
        s["dy"] = randn(T, N).to(dt)
    return s


# ---- one pass ------------------------------------------------------------------------------------
def _places(s):
    """Expert of each row and the row's place in its run."""
    off = s["offsets"].long()
    r = torch.arange(s["case"]["T"], device=off.device)
    e = torch.searchsorted(off[1:].contiguous(), r, right=True)
    return e, r - off[e]


def _padded(rows, s, e, at):
    """Rows in order -> (E, longest run, columns) with zeros behind each run."""
    p = torch.zeros(s["case"]["E"], s["longest"], rows.shape[1], device=rows.device)
    p[e, at] = rows.float()
    return p


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "quant":
        return {"values": _plain_values(*_plain_quantise(s["x"])).to(torch.bfloat16)}
    if op == "mx":
        M, K, N = case["M"], case["K"], case["N"]
        w = _plain_unpacked(s["w"][None], s["ws"][None], N, K)[0]
        if case["quantise"]:
            x = _plain_values(*_plain_quantise(s["x"]))
        else:
            x = _plain_unpacked(s["x"][None], s["xs"][None], M, K)[0]
        return {"y": (x @ w.T).to(s["dt"])}
    e, at = _places(s)
    if op == "grouped_mx":
        w = _plain_unpacked(s["w"], s["ws"], case["N"], case["K"])
        x = _plain_values(*_plain_quantise(s["x"]))
        return {"y": (_padded(x, s, e, at) @ w.transpose(1, 2))[e, at].to(s["dt"])}
    w = s["w"].float()
    if op == "grouped":
        return {"y": (_padded(s["x"], s, e, at) @ w.transpose(1, 2))[e, at].to(s["dt"])}
    dy = _padded(s["dy"], s, e, at)
    dx = (dy @ w)[e, at]
    dw = dy.transpose(1, 2) @ _padded(s["x"], s, e, at)
    return {"dx": dx.to(s["dt"]), "dw": dw.to(s["dt"])}


def _own(s):
    from heron_b200 import kernels as K
    case, op, dt = s["case"], s["case"]["op"], s["dt"]
    if op == "quant":
        codes, scales = K.quantize_mxfp4(s["x"])
        return {"values": K.dequantize_mxfp4(codes, scales, out_dtype=torch.bfloat16)}
    if op == "mx":
        x, xs = K.quantize_mxfp4(s["x"]) if case["quantise"] else (s["x"], s["xs"])
        return {"y": K.gemm_mxfp4(x, xs, s["w"], s["ws"], out_dtype=dt)}
    if op == "grouped_mx":
        x, xs = K.quantize_mxfp4(s["x"], offsets=s["offsets"])
        return {"y": K.grouped_gemm_mxfp4(x, xs, s["w"], s["ws"], s["offsets"], out_dtype=dt)}
    if op == "grouped":
        return {"y": K.grouped_gemm(s["x"], s["w"], s["offsets"], out_dtype=dt)}
    return {"dx": K.grouped_gemm_dx(s["dy"], s["w"], s["offsets"], out_dtype=dt),
            "dw": K.grouped_gemm_dw(s["dy"], s["x"], s["offsets"], out_dtype=dt)}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    op, K = case["op"], case["K"]
    es = 4 if case["dtype"] == "f32" else 2
    q = 0.5 + 1 / 32  # bytes of one 4-bit element and its share of a scale
    if op == "quant":  # the values once in, the quantised form out and in again, the values out
        n = case["M"] * K
        return {"bytes": n * (es + 2 * q + 2), "flops": 0}
    if op == "mx":
        M, N = case["M"], case["N"]
        return {"bytes": M * K * (es if case["quantise"] else q) + N * K * q + M * N * es, "flops": 2 * M * N * K}
    T, N = case["T"], case["N"]
    hit = sum(c > 0 for c in _counts(case))
    if op == "grouped_mx":
        return {"bytes": T * K * es + hit * N * K * q + T * N * es, "flops": 2 * T * N * K}
    if op == "grouped":
        return {"bytes": (T * K + hit * N * K + T * N) * es, "flops": 2 * T * N * K}
    # dx: dy and w in, dx out; dw: dy (again the same bytes) and x in, dw out, of every expert
    return {"bytes": (T * N + hit * N * K + T * K + T * K + case["E"] * N * K) * es, "flops": 4 * T * N * K}


# ---- the definition in 64 bits -------------------------------------------------------------------
def _exact_quantised(x):
    """The values that a matrix has after quantisation, from the definition: the nearest element by
    distance, the even code on a tie."""
    v = x.double()
    out = torch.empty_like(v)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=v.device)
    step = max(1, (1 << 22) // v.shape[1])
    for r in range(0, v.shape[0], step):
        b = v[r:r + step].reshape(-1, 32)
        top = b.abs().max(1, keepdim=True).values
        # (64 bits hold the logarithm of a 16- or 32-bit number next to a power of two exactly enough)
        s = torch.floor(torch.log2(top)) - 2
        s = torch.where(torch.exp2(s + 2) > top, s - 1, torch.where(torch.exp2(s + 3) <= top, s + 1, s))
        unit = torch.exp2(torch.clamp(s, min=-127.0))
        d = ((b / unit).abs()[..., None] - grid).abs()
        d = d + torch.tensor([0, 1, 0, 1, 0, 1, 0, 1], dtype=torch.float64, device=v.device) * 1e-9
        out[r:r + step] = (torch.sign(b) * grid[d.argmin(-1)] * unit).reshape(-1, v.shape[1])
    return out


def _exact_unpacked(packed, scales, M, K):
    """(M, K/2) bytes and tiled scales -> values in 64 bits, tile by tile of the layout."""
    kt = -(-K // 128)
    tiles = scales.reshape(-1, kt, 32, 4, 4)  # tile row, tile column, row % 32, row / 32, block
    s = tiles.permute(0, 3, 2, 1, 4).reshape(-1, kt * 4)[:M, :K // 32].double()
    low, high = packed.long() % 16, packed.long() // 16
    n = torch.stack((low, high), 2).reshape(M, K)
    m = n % 8
    mag = torch.where(m < 2, m * 0.5, (1 + (m % 2) * 0.5) * 2.0 ** (m // 2 - 1).double())
    return torch.where(n >= 8, -mag, mag) * torch.exp2(s - 127).repeat_interleave(32, 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        return {"values": _exact_quantised(s["x"])}
    if op == "mx":
        w = _exact_unpacked(s["w"], s["ws"], case["N"], case["K"])
        x = _exact_quantised(s["x"]) if case["quantise"] else _exact_unpacked(s["x"], s["xs"], case["M"], case["K"])
        return {"y": x @ w.T}
    ends = s["offsets"].tolist()
    T, E, K, N = case["T"], case["E"], case["K"], case["N"]
    x = _exact_quantised(s["x"]) if op == "grouped_mx" else s["x"].double()
    if op != "grouped_bwd":
        y = torch.zeros(T, N, dtype=torch.float64, device="cuda")
        for e in range(E):
            w = _exact_unpacked(s["w"][e], s["ws"][e], N, K) if op == "grouped_mx" else s["w"][e].double()
            y[ends[e]:ends[e + 1]] = x[ends[e]:ends[e + 1]] @ w.T
        return {"y": y}
    dx = torch.zeros(T, K, dtype=torch.float64, device="cuda")
    dw = torch.zeros(E, N, K, dtype=torch.float64, device="cuda")
    for e in range(E):
        rows = slice(ends[e], ends[e + 1])
        dx[rows] = s["dy"][rows].double() @ s["w"][e].double()
        dw[e] = s["dy"][rows].double().T @ x[rows]
    return {"dx": dx, "dw": dw}
