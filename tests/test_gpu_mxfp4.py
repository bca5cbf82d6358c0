"""MXFP4 quantisation, the way back and the products, against the definition in 64 bits."""
import pytest
import torch

from grouped_util import (assert_product, grouped, grouped_dw, offsets_of, quantise, scale_index,
                          unpack)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(hb_lib):
    assert torch.cuda.is_available(), "GPU tests need a B200"
    from heron_b200 import kernels
    assert hb_lib.hb_sm_count() > 0, "libheron_b200.so found no sm_100 device"
    return kernels


@pytest.fixture(autouse=True)
def _status_clean(hb_lib):
    yield
    from heron_b200 import _lib
    assert _lib.last_status() == 0, "a bounded device-side wait ran out"


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def check_quantised(K, x, offsets=None, off=None):
    codes, scales = K.quantize_mxfp4(x, offsets=offsets)
    byte, code, values = quantise(x)
    at = scale_index(*x.shape, off)
    own = at[:, 0] >= 0
    assert torch.equal(unpack(codes.cpu())[own], code[own])
    assert torch.equal(scales.cpu()[at[own]], byte[own])
    for od in (torch.float32, torch.bfloat16):
        out = torch.full(x.shape, 7.0, dtype=od, device="cuda")
        K.dequantize_mxfp4(codes, scales, offsets=offsets, out=out)
        assert torch.equal(torch.nan_to_num(out[own.cuda()].double().cpu(), nan=99.0),
                           torch.nan_to_num(values[own], nan=99.0))
        assert (out[~own.cuda()] == 7.0).all()
    return codes, scales, values.cuda()


@pytest.mark.parametrize("rows,k", [(1, 32), (3, 64), (33, 96), (128, 128), (129, 160), (300, 544), (2, 4096)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_quantise(K, rows, k, dtype):
    check_quantised(K, randn(rows + k, rows, k, dtype=dtype, scale=3.0))


def test_every_border(K):
    """All ties and their neighbours at every sign, over scales from the smallest to the largest."""
    mids = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0])
    near = torch.cat([mids, torch.nextafter(mids, torch.tensor(9.0)), torch.nextafter(mids, torch.tensor(0.0))])
    near = torch.cat([near, -near])  # 96 values
    rows = []
    for e in (-149, -140, -130, -127, -126, -125, -64, -3, 0, 5, 64, 124, 125):
        v = near.double() * 2.0 ** e
        v = torch.cat([v, torch.full((3,), 4.0 * 2.0 ** e, dtype=torch.float64)])[:96]
        # each block of 32 gets a 4 so that its scale is 2^e where that is in range
        v = v.reshape(3, 32).clone()
        v[:, 31] = 4.0 * 2.0 ** e
        rows.append(v.reshape(96).float())
    rows += [torch.zeros(96), torch.full((96,), 3.4e38), torch.full((96,), -1e-45)]
    check_quantised(K, torch.stack(rows).cuda())
    check_quantised(K, torch.stack(rows).bfloat16().cuda())
    check_quantised(K, torch.stack(rows[6:9]).half().cuda())


def test_values_that_are_not_finite(K):
    x = randn(1, 5, 96)
    x[0, 3], x[1, 40], x[2, 95], x[4, 0] = torch.inf, -torch.inf, torch.nan, torch.nan
    check_quantised(K, x)
    check_quantised(K, x.bfloat16())


def test_pad_bytes_are_zero(K):
    x = randn(1, 40, 160)
    scales = torch.full((K.mxfp4_scale_bytes(40, 160),), 255, dtype=torch.uint8, device="cuda")
    K.quantize_mxfp4(x, scales=scales)
    s = scales.cpu().reshape(2, 32, 4, 4)  # tile column, row % 32, row / 32, block
    assert (s[1, :, 0, 1:] == 0).all() and (s[1, :8, 1, 1:] == 0).all()
    assert (s[1, 8:, 1, :] == 255).all()  # rows the matrix has not


@pytest.mark.parametrize("counts,lead,tail", [([0, 5, 130, 0, 1], 3, 4), ([0, 0], 2, 2), ([300], 0, 0), ([128, 128, 1], 0, 1)])
def test_quantise_by_groups(K, counts, lead, tail):
    off = offsets_of(counts, lead)
    x = randn(2, off[-1] + tail, 160, dtype=torch.bfloat16)
    check_quantised(K, x, torch.tensor(off, dtype=torch.int32, device="cuda"), off)


@pytest.mark.parametrize("E", [31, 33, 64, 100, 1024])
def test_quantise_by_many_groups(K, E):
    g = torch.Generator().manual_seed(E)
    counts = (torch.randint(0, 5, (E,), generator=g) * (torch.rand(E, generator=g) < 0.6)).tolist()
    counts[E // 2] = 150
    off = offsets_of(counts, 2)
    x = randn(E, off[-1] + 1, 64, dtype=torch.bfloat16)
    check_quantised(K, x, torch.tensor(off, dtype=torch.int32, device="cuda"), off)


def test_quantise_a_batch(K):
    x = randn(3, 3, 130, 96, dtype=torch.float16)
    codes, scales = K.quantize_mxfp4(x)
    back = K.dequantize_mxfp4(codes, scales)
    for i in range(3):
        c, s, v = check_quantised(K, x[i])
        assert torch.equal(codes[i], c) and torch.equal(back[i].double(), v)
        assert torch.equal(scales[i, scale_index(130, 96).cuda()], s[scale_index(130, 96).cuda()])


def test_float16_values_round_and_overflow(K):
    x = torch.tensor([[6.0 * 2.0 ** 20] * 16 + [0.0] * 16, [6.0 * 2.0 ** -26] * 32], device="cuda")
    codes, scales = K.quantize_mxfp4(x)
    v = K.dequantize_mxfp4(codes, scales, out_dtype=torch.float16)
    assert torch.isinf(v[0, :16]).all() and (v[0, 16:] == 0).all()
    assert torch.equal(v[1], x[1].half())


def product(K, M, N, k, seed, out_dtype, knobs=None, xdtype=torch.bfloat16):
    a, b = randn(seed, M, k, dtype=xdtype), randn(seed + 1, N, k, dtype=xdtype, scale=k ** -0.5)
    ac, asc = K.quantize_mxfp4(a)
    bc, bsc = K.quantize_mxfp4(b)
    av, bv = K.dequantize_mxfp4(ac, asc), K.dequantize_mxfp4(bc, bsc)
    out = K.gemm_mxfp4(ac, asc, bc, bsc, out_dtype=out_dtype, knobs=knobs)
    want, mag, _ = grouped(av, bv[None], [0, M])
    assert_product(out, want, mag, k, "%d x %d x %d" % (M, N, k))


@pytest.mark.parametrize("M,N,k", [(1, 128, 256), (1, 1, 32), (16, 128, 64), (5, 100, 96), (64, 128, 128), (65, 130, 160),
                                   (128, 256, 512), (129, 257, 544), (200, 128, 288), (333, 500, 1056), (640, 384, 2048)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_product(K, M, N, k, out_dtype):
    product(K, M, N, k, M + N + k, out_dtype)


@pytest.mark.parametrize("knobs", [dict(tile_n=64), dict(tile_n=128), dict(tile_n=192), dict(tile_n=256),
                                   dict(stages=1), dict(acc_stages=1), dict(max_ctas=2), dict(tile_n=192, max_ctas=1),
                                   dict(tile_n=128, cta_group=2), dict(tile_n=192, cta_group=2), dict(tile_n=256, cta_group=2),
                                   dict(tile_n=192, cta_group=2, stages=1), dict(tile_n=192, cta_group=2, max_ctas=2)])
def test_product_knobs(K, knobs):
    product(K, 700, 300, 800, 11, torch.float32, knobs)
    product(K, 130, 200, 160, 12, torch.float32, knobs)


@pytest.mark.parametrize("split", [2, 4, 8])
@pytest.mark.parametrize("M,N,k", [(1, 1, 32), (3, 200, 1056), (64, 130, 2048), (130, 300, 800)])
def test_a_reduction_over_a_cluster(K, split, M, N, k):
    for od in (torch.float32, torch.bfloat16):
        product(K, M, N, k, split, od, dict(tile_n=64, split_k=split))
        product(K, M, N, k, split, od, dict(tile_n=64, split_k=split, max_ctas=split, stages=2))


def test_product_of_single_elements(K):
    """One non-zero element a row: every (row, k) place of codes and scales meets its partner and no other."""
    k = 512
    a, b = torch.zeros(256, k, device="cuda"), torch.zeros(256, k, device="cuda")
    i = torch.arange(256, device="cuda")
    a[i, (i * 37 + 5) % k] = 2.0 ** (i % 9 - 4).float() * 1.5
    b[i, (i * 53 + 7) % k] = 2.0 ** (i % 7 - 3).float() * 3.0
    out = K.gemm_mxfp4(*K.quantize_mxfp4(a), *K.quantize_mxfp4(b))
    assert torch.equal(out.double(), a.double() @ b.double().T)


@pytest.mark.parametrize("M", [1, 3, 8, 13, 40])
@pytest.mark.parametrize("k", [32, 96, 1024])
def test_sums_of_blocks_are_exact(K, M, k):
    """With scales of 1 every sum of products is a multiple of 1/4 below 2^24 quarters: no bit may be lost."""
    g = torch.Generator(device="cuda").manual_seed(M * k)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda")

    def operand(rows):
        v = grid[torch.randint(0, 8, (rows, k), generator=g, device="cuda")]
        v = v * (torch.randint(0, 4, (rows, k), generator=g, device="cuda") * 2 - 1).clamp(-1, 1)
        v[0] = 6.0  # the largest sum there is
        v[:, ::32] = 4.0  # (sets the block's scale to 1)
        return v
    a, b = operand(M), operand(150)
    out = K.gemm_mxfp4(*K.quantize_mxfp4(a), *K.quantize_mxfp4(b))
    assert torch.equal(out.double(), a.double() @ b.double().T)


def test_nan_scale_makes_its_row_nan(K):
    a, b = randn(1, 20, 128), randn(2, 40, 128)
    a[3, 70], b[9, 1] = torch.nan, torch.inf
    out = K.gemm_mxfp4(*K.quantize_mxfp4(a), *K.quantize_mxfp4(b))
    assert torch.isnan(out[3]).all() and torch.isnan(out[:, 9]).all()
    out[3], out[:, 9] = 0, 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("counts,lead,tail", [([0, 5, 130, 0, 1], 3, 4), ([0, 0], 2, 2), ([300, 0, 513], 0, 0),
                                              ([128, 128, 1], 0, 1), ([1], 0, 0), ([64, 65, 192, 193], 1, 0)])
@pytest.mark.parametrize("k,n", [(96, 100), (512, 256)])
def test_grouped_product(K, counts, lead, tail, k, n):
    off = offsets_of(counts, lead)
    T, E = off[-1] + tail, len(counts)
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    x, w = randn(4, T, k, dtype=torch.bfloat16), randn(5, E, n, k, dtype=torch.bfloat16)
    x[:lead], x[off[-1]:] = torch.nan, torch.nan
    xc, xs = K.quantize_mxfp4(x, offsets=offsets)
    wc, ws = K.quantize_mxfp4(w)
    xv = torch.zeros(T, k, device="cuda")
    K.dequantize_mxfp4(xc, xs, offsets=offsets, out=xv)
    wv = K.dequantize_mxfp4(wc, ws)
    want, mag, own = grouped(xv, wv, off)
    for knobs in (None, dict(tile_n=64), dict(tile_n=192), dict(tile_n=256), dict(tile_n=192, cta_group=2),
                  dict(tile_n=256, cta_group=2)):
        out = torch.full((T, n), 7.0, device="cuda")
        K.grouped_gemm_mxfp4(xc, xs, wc, ws, offsets, out=out, knobs=knobs)
        assert_product(out[own], want[own], mag[own], k, str(knobs))
        assert (out[~own] == 7.0).all()


def test_offsets_are_clamped(K):
    x, w = randn(6, 40, 64), randn(7, 3, 32, 64)
    wc, ws = K.quantize_mxfp4(w)
    wv = K.dequantize_mxfp4(wc, ws)
    off = [-7, 9, 30, 1000]
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    xc, xs = K.quantize_mxfp4(x, offsets=offsets)
    out = K.grouped_gemm_mxfp4(xc, xs, wc, ws, offsets)
    want, mag, _ = grouped(quantise(x)[2].cuda(), wv, off)
    assert_product(out, want, mag, 64)
    # out of order: nothing is read or written out of range
    offsets.copy_(torch.tensor([30, 9, 35, 2], dtype=torch.int32))
    xc, xs = K.quantize_mxfp4(x, offsets=offsets)
    K.grouped_gemm_mxfp4(xc, xs, wc, ws, offsets)
    torch.cuda.synchronize()


def test_no_rows(K):
    w = randn(1, 2, 16, 64)
    wc, ws = K.quantize_mxfp4(w)
    offsets = torch.zeros(3, dtype=torch.int32, device="cuda")
    x = randn(1, 0, 64)
    xc, xs = K.quantize_mxfp4(x, offsets=offsets)
    assert K.grouped_gemm_mxfp4(xc, xs, wc, ws, offsets).shape == (0, 16)
    xc, xs = K.quantize_mxfp4(x)
    assert K.gemm_mxfp4(xc, xs, wc[0], ws[0]).shape == (0, 16)
    assert K.dequantize_mxfp4(xc, xs).shape == (0, 64)


def test_two_streams_at_once(K):
    """No call keeps anything between calls: the same operands on two streams, outputs of their own."""
    x, w = randn(1, 300, 512, dtype=torch.bfloat16), randn(2, 260, 512, dtype=torch.bfloat16)
    wq = K.quantize_mxfp4(w)
    want = K.gemm_mxfp4(*K.quantize_mxfp4(x), *wq)
    got, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(K.gemm_mxfp4(*K.quantize_mxfp4(x), *wq))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_a_silent_producer_ends_in_a_status(K):
    from heron_b200 import _lib
    a, b = K.quantize_mxfp4(randn(1, 64, 256)), K.quantize_mxfp4(randn(2, 128, 256))
    for knobs in (dict(silent_producer=1), dict(silent_producer=1, cta_group=2, tile_n=192),
                  dict(silent_producer=1, tile_n=64, split_k=2)):
        K.gemm_mxfp4(*a, *b, knobs=knobs)
        assert _lib.last_status() == _lib.HB_ERR_TIMEOUT
    want = K.dequantize_mxfp4(*a).double() @ K.dequantize_mxfp4(*b).double().T
    mag = K.dequantize_mxfp4(*a).double().abs() @ K.dequantize_mxfp4(*b).double().abs().T
    assert_product(K.gemm_mxfp4(*a, *b), want, mag, 256)


def test_expert_layer_in_training_and_serving(K):
    """The operators together: forward, gradients, a step on the weights, then the trained experts in 4 bits;
    the whole captured once and replayed with other routing."""
    E, k, n, T = 4, 128, 192, 150
    w = randn(1, E, n, k, dtype=torch.bfloat16, scale=k ** -0.5)
    x, dy = randn(2, T, k, dtype=torch.bfloat16), randn(3, T, n, dtype=torch.bfloat16)
    offsets = torch.tensor([0, 40, 40, 141, 150], dtype=torch.int32, device="cuda")
    w2 = torch.empty_like(w)

    def step():
        y = K.grouped_gemm(x, w, offsets, out_dtype=torch.bfloat16)
        dx = K.grouped_gemm_dx(dy, w, offsets, out_dtype=torch.bfloat16)
        dw = K.grouped_gemm_dw(dy, x, offsets, out_dtype=torch.float32)
        w2.copy_(w - 0.01 * dw)
        xc, xs = K.quantize_mxfp4(x, offsets=offsets)
        wc, ws = K.quantize_mxfp4(w2)
        return y, dx, dw, xc, xs, wc, ws, K.grouped_gemm_mxfp4(xc, xs, wc, ws, offsets, out_dtype=torch.bfloat16)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx, dw, xc, xs, wc, ws, y4 = step()
    for off in ([0, 40, 40, 141, 150], [0, 0, 150, 150, 150], [0, 1, 2, 77, 150]):
        offsets.copy_(torch.tensor(off, dtype=torch.int32))
        graph.replay()
        want, mag, _ = grouped(x, w, off)
        assert_product(y, want, mag, k, "y")
        want, mag, _ = grouped(dy, w.transpose(1, 2), off)
        assert_product(dx, want, mag, n, "dx")
        want, mag = grouped_dw(dy, x, off, E)
        assert_product(dw, want, mag, T, "dw")
        xv, wv = K.dequantize_mxfp4(xc, xs, offsets=offsets), K.dequantize_mxfp4(wc, ws)
        want, mag, _ = grouped(xv, wv, off)
        assert_product(y4, want, mag, k, "y4")
        assert torch.equal(xv.double().cpu(), quantise(x)[2])


def check_product(K, a, b, what):
    """gemm_mxfp4 of two matrices against 64 bits, in 32 and 16 bits out."""
    a, b = K.quantize_mxfp4(a), K.quantize_mxfp4(b)
    av, bv = K.dequantize_mxfp4(*a), K.dequantize_mxfp4(*b)
    want, mag, _ = grouped(av, bv[None], [0, av.shape[0]])
    for od in (torch.float32, torch.bfloat16):
        assert_product(K.gemm_mxfp4(*a, *b, out_dtype=od), want, mag, av.shape[1], "%s %s" % (what, od))


@pytest.mark.parametrize("M", [1, 3, 8, 9, 40])
@pytest.mark.parametrize("k", [96, 1024])
@pytest.mark.parametrize("ea,eb", [(-60, -60), (60, 60), (-70, -48), (-48, -70), (100, -100), (-100, 100), (120, -124),
                                   (-30, -31), (31, 32), (33, 40), (-126, 100)])
def test_product_of_scales_far_from_one(K, M, k, ea, eb):
    """Results from 2^-120 to 2^120, which all output types but fp16 hold: no scale may leave fp32 on the way."""
    a, b = randn(M + k, M, k, scale=2.0 ** ea), randn(7, 40, k, scale=k ** -0.5) * 2.0 ** eb
    check_product(K, a, b, "2^%d x 2^%d" % (ea, eb))


@pytest.mark.parametrize("M", [1, 5, 8, 9])
def test_product_of_blocks_of_mixed_scales(K, M):
    """Every block of 32 with an exponent of its own, some blocks zero."""
    g = torch.Generator(device="cuda").manual_seed(M)

    def operand(seed, rows, k):
        e = torch.randint(-60, 55, (rows, k // 32, 1), generator=g, device="cuda").float()
        z = (torch.rand(rows, k // 32, 1, generator=g, device="cuda") < 0.8).float()
        return (randn(seed, rows, k // 32, 32) * torch.exp2(e) * z).reshape(rows, k)
    for k in (32, 160, 1056):
        check_product(K, operand(1, M, k), operand(2, 50, k), "k %d" % k)


@pytest.mark.parametrize("M", [1, 8, 9])
def test_large_scales_and_small_sums(K, M):
    """Blocks whose scales' product passes 2^128 while the sum of their elements' products is 0 or 1/4."""
    for e, meet, want in ((66, 0.0, 0.0), (110, 0.0, 0.0), (64, 0.5, 2.0 ** 126), (-66, 0.5, 2.0 ** -134)):
        a, b = torch.zeros(M, 64, device="cuda"), torch.zeros(20, 64, device="cuda")
        a[:, 1], b[:, 2] = 4.0, 4.0  # the scales are 2^e
        a[:, 5], b[:, 5] = meet, meet
        a[:, 40], b[:, 50] = 4.0, 4.0
        out = K.gemm_mxfp4(*K.quantize_mxfp4(a * 2.0 ** e), *K.quantize_mxfp4(b * 2.0 ** e))
        assert (out == want).all(), (e, meet, out[0, 0].item())


@pytest.mark.parametrize("M", [1, 5, 8])
def test_nan_scale_of_few_rows(K, M):
    """As test_nan_scale_makes_its_row_nan, in the kernel of few rows."""
    a, b = randn(1, M, 416), randn(2, 40, 416)
    b[9, 1], b[30, 400] = torch.inf, torch.nan
    if M > 1:
        a[3, 170] = torch.nan
    out = K.gemm_mxfp4(*K.quantize_mxfp4(a), *K.quantize_mxfp4(b))
    nan = torch.zeros(M, 40, dtype=torch.bool, device="cuda")
    nan[:, [9, 30]] = True
    nan[3:4] = M > 1
    assert torch.equal(torch.isnan(out), nan) and torch.isfinite(out[~nan]).all()


@pytest.mark.parametrize("k", [64, 416])
def test_overlapping_offsets(K, k):
    """Offsets out of order, groups' tiles of scales apart: rows that one group owns are right."""
    from grouped_util import clamped
    w = randn(7, 3, 40, k)
    wc, ws = K.quantize_mxfp4(w)
    wv = K.dequantize_mxfp4(wc, ws)
    for off in ([0, 6, 2, 8], [0, 5, 1, 8], [3, 7, 0, 6], [2, 8, 3, 8]):
        x = randn(6, 8, k)
        offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
        xc, xs = K.quantize_mxfp4(x, offsets=offsets)
        xv = quantise(x)[2].cuda()
        for knobs in (None, dict(tile_n=64)):
            out = torch.full((8, 40), 7.0, device="cuda")
            K.grouped_gemm_mxfp4(xc, xs, wc, ws, offsets, out=out, knobs=knobs)
            owners = torch.zeros(8, dtype=torch.int64)
            for s, t in clamped(off, 8):
                owners[s:t] += 1
            once = (owners == 1).cuda()
            want, mag, _ = grouped(xv, wv, off)
            assert_product(out[once], want[once], mag[once], k, "%s %s" % (off, knobs))
            assert (out[(owners == 0).cuda()] == 7.0).all()


def grouped_operands(K, counts, lead, tail, k, n):
    off = offsets_of(counts, lead)
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    T = off[-1] + tail
    x, w = randn(4, T, k, dtype=torch.bfloat16), randn(5, len(counts), n, k, dtype=torch.bfloat16)
    xq, wq = K.quantize_mxfp4(x, offsets=offsets), K.quantize_mxfp4(w)
    xv = torch.zeros(T, k, device="cuda")
    K.dequantize_mxfp4(*xq, offsets=offsets, out=xv)
    return off, offsets, xq, wq, grouped(xv, K.dequantize_mxfp4(*wq), off)


@pytest.mark.parametrize("counts", [[1, 2, 3, 2] * 8, [0, 1, 40, 3, 64, 0, 33, 5] * 4, [129] * 6 + [0] * 26])
@pytest.mark.parametrize("k,n", [(416, 2048), (1024, 2000)])
def test_grouped_product_in_several_rounds(K, counts, k, n):
    """More tiles than the CTAs that run at once, the default's choice of tiles."""
    off, offsets, xq, wq, (want, mag, own) = grouped_operands(K, counts, 1, 2, k, n)
    for od in (torch.float32, torch.bfloat16):
        out = torch.full(want.shape, 7.0, dtype=od, device="cuda")
        K.grouped_gemm_mxfp4(*xq, *wq, offsets, out=out)
        assert_product(out[own], want[own], mag[own], k)
        assert (out[~own] == 7.0).all()


@pytest.mark.parametrize("counts,lead,tail", [([3, 0, 1, 4], 0, 0), ([3, 0, 1, 2], 1, 1), ([0, 8], 0, 0), ([9, 0, 0, 1, 17], 3, 0),
                                              ([1] * 20, 130, 0)])
@pytest.mark.parametrize("k,n", [(416, 300), (64, 130), (1056, 17)])
def test_few_rows_of_several_groups(K, counts, lead, tail, k, n):
    """The kernel of few rows with more than one tile of scales to an expert and groups that start inside a tile."""
    off, offsets, xq, wq, (want, mag, own) = grouped_operands(K, counts, lead, tail, k, n)
    for knobs in (None, dict(tile_n=64)):
        out = torch.full(want.shape, 7.0, device="cuda")
        K.grouped_gemm_mxfp4(*xq, *wq, offsets, out=out, knobs=knobs)
        assert_product(out[own], want[own], mag[own], k, str(knobs))
        assert (out[~own] == 7.0).all()


@pytest.mark.parametrize("split", [2, 4, 8])
@pytest.mark.parametrize("counts", [[0, 1, 0, 2, 70], [17, 0, 128, 1, 129, 63], [0, 0]])
@pytest.mark.parametrize("k,n", [(96, 130), (2080, 300)])
def test_grouped_reduction_over_a_cluster(K, split, counts, k, n):
    off, offsets, xq, wq, (want, mag, own) = grouped_operands(K, counts, 2, 3, k, n)
    for extra in (dict(), dict(max_ctas=2 * split), dict(stages=1)):
        out = torch.full(want.shape, 7.0, device="cuda")
        K.grouped_gemm_mxfp4(*xq, *wq, offsets, out=out, knobs=dict(tile_n=64, split_k=split, **extra))
        assert_product(out[own], want[own], mag[own], k, str(extra))
        assert (out[~own] == 7.0).all()
