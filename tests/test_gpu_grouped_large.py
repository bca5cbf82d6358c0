"""The grouped and 4-bit operators at sizes that pass 32 bits or the usual time of a tile."""
import pytest
import torch

from grouped_util import assert_product, offsets_of, quantise, unpack

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
    torch.cuda.empty_cache()
    assert _lib.last_status() == 0, "a bounded device-side wait ran out"


def test_the_longest_reduction(K):
    """2^30 rows in one group: 2^24 blocks into one tile, whose accumulator takes seconds.  Few rows are not zero, so the
    sums are exact."""
    T = 1 << 30
    x, dy = (torch.zeros(T, 8, dtype=torch.float16, device="cuda") for _ in range(2))
    rows = torch.tensor([0, 1, 63, 64, T // 3, T // 2, T - 65, T - 2, T - 1], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for t in (x, dy):
        t[rows] = torch.randint(-8, 9, (9, 8), generator=g, device="cuda").half()
    offsets = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    dw = K.grouped_gemm_dw(dy, x, offsets)
    assert torch.equal(dw[0].double(), dy[rows].double().T @ x[rows].double())


def test_weights_beyond_32_bits(K):
    """More than 2^31 weights: the last expert's lie past what an int holds, in all kernels."""
    E, N, k = 131, 4096, 4104
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.empty(E, N, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    for counts in ([2] + [0] * (E - 2) + [3], [70] + [0] * (E - 2) + [90], [0] * (E - 1) + [300]):
        off = offsets_of(counts)
        x = torch.randn(off[-1], k, generator=g, device="cuda").bfloat16()
        dy = torch.randn(off[-1], N, generator=g, device="cuda").bfloat16()
        offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
        y, dx = K.grouped_gemm(x, w, offsets), K.grouped_gemm_dx(dy, w, offsets)
        for e in (0, E - 1):
            rows = slice(off[e], off[e + 1])
            xe, de, we = x[rows].double(), dy[rows].double(), w[e].double()
            assert_product(y[rows], xe @ we.T, xe.abs() @ we.abs().T, k, "y of %d" % e)
            assert_product(dx[rows], de @ we, de.abs() @ we.abs(), N, "dx of %d" % e)
    dw = K.grouped_gemm_dw(dy, x, offsets, out=w)
    assert_product(dw[E - 1], dy.double().T @ x.double(), dy.double().abs().T @ x.double().abs(), 300, "dw")
    assert not dw[:E - 1].any()


def test_outputs_beyond_32_bits(K):
    T, N, k = (1 << 18) + 5, 8200, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(T, k, generator=g, device="cuda").bfloat16()
    w = torch.randn(2, N, k, generator=g, device="cuda").bfloat16()
    offsets = torch.tensor([0, 1000, T], dtype=torch.int32, device="cuda")
    wt = w.transpose(1, 2).contiguous()
    for out in (K.grouped_gemm(x, w, offsets, out_dtype=torch.bfloat16), K.grouped_gemm_dx(x, wt, offsets, out_dtype=torch.bfloat16)):
        for rows, e in ((slice(0, 500), 0), (slice(T - 500, T), 1), (slice(T // 2, T // 2 + 500), 1)):
            a, b = x[rows].double(), w[e].double()
            assert_product(out[rows], a @ b.T, a.abs() @ b.abs().T, k)
        del out


def test_quantised_values_beyond_32_bits(K):
    """2^31 values and more quantised, read back and multiplied; checked where the offsets are largest."""
    g = torch.Generator(device="cuda").manual_seed(4)
    E, N, k = 66, 4096, 8224
    w = torch.empty(E, N, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    wq = K.quantize_mxfp4(w)
    back = K.dequantize_mxfp4(*wq, out_dtype=torch.bfloat16)
    del w
    w = torch.empty(E, N, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g.manual_seed(4))
    byte, code, values = quantise(w[-1, -40:])
    assert torch.equal(back[-1, -40:].double().cpu(), values) and torch.equal(unpack(wq[0][-1, -40:].cpu()), code)
    rows = w.reshape(E * N, k)
    del w
    rq = K.quantize_mxfp4(rows)
    assert torch.equal(rq[0][-40:].cpu(), wq[0][-1, -40:].cpu())
    assert torch.equal(K.dequantize_mxfp4(*rq, out_dtype=torch.bfloat16)[-40:].double().cpu(), values)
    del rq, rows
    for T in (1, 5, 300):
        x = torch.randn(T, k, generator=g, device="cuda").bfloat16()
        offsets = torch.tensor([0] * E + [T], dtype=torch.int32, device="cuda")
        xq = K.quantize_mxfp4(x, offsets=offsets)
        xv = K.dequantize_mxfp4(*xq, offsets=offsets).double()
        wv = back[-1].double()
        assert_product(K.grouped_gemm_mxfp4(*xq, *wq, offsets), xv @ wv.T, xv.abs() @ wv.abs().T, k, "%d rows" % T)
