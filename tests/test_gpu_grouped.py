"""The products grouped by expert and their gradients, against a plain form in 64 bits."""
import pytest
import torch

from grouped_util import assert_product, grouped, grouped_dw, offsets_of

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


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def make(seed, counts, lead, tail, k, n, dtype):
    """x, w, dy and offsets; rows of no group hold NaN, which must reach nothing."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    off = offsets_of(counts, lead)
    T = off[-1] + tail
    x, dy = randn(g, T, k, dtype=dtype), randn(g, T, n, dtype=dtype)
    for t in (x, dy):
        t[:lead] = torch.nan
        t[off[-1]:] = torch.nan
    w = randn(g, len(counts), n, k, dtype=dtype, scale=k ** -0.5)
    return x, w, dy, off, torch.tensor(off, dtype=torch.int32, device="cuda")


def clean(t):
    return torch.nan_to_num(t, nan=0.0)


COUNTS = {
    "one_row": [1],
    "decode": [0, 1, 0, 0, 2, 1, 0],
    "uneven": [17, 0, 128, 1, 129, 63],
    "all_in_one": [0, 0, 300, 0],
    "one_group": [256],
    "tile_edges": [16, 32, 48, 49, 64, 65],
    "wide": [257, 511, 40],
    "empty": [0, 0, 0],
}


@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("k,n", [(8, 8), (64, 128), (72, 136), (520, 264)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_forward_and_gradients(K, counts, k, n, dtype):
    c = COUNTS[counts]
    x, w, dy, off, offsets = make(k * 1000 + n, c, 3, 5, k, n, dtype)
    T = x.shape[0]
    for od in (torch.float32, dtype):
        out = torch.full((T, n), 7.0, dtype=od, device="cuda")
        assert K.grouped_gemm(x, w, offsets, out=out) is out
        want, mag, own = grouped(clean(x), w, off)
        assert_product(out[own], want[own], mag[own], k, "y")
        assert (out[~own] == 7.0).all(), "rows of no group changed"
        dx = torch.full((T, k), 7.0, dtype=od, device="cuda")
        K.grouped_gemm_dx(dy, w, offsets, out=dx)
        want, mag, own = grouped(clean(dy), w.transpose(1, 2), off)
        assert_product(dx[own], want[own], mag[own], n, "dx")
        assert (dx[~own] == 7.0).all(), "rows of no group changed"
        dw = torch.full((len(c), n, k), 7.0, dtype=od, device="cuda")
        K.grouped_gemm_dw(dy, x, offsets, out=dw)
        want, mag = grouped_dw(clean(dy), clean(x), off, len(c))
        assert_product(dw, want, mag, max(c), "dw")


@pytest.mark.parametrize("n", [1, 7, 127, 1001])
def test_forward_takes_any_output_width(K, n):
    x, w, _, off, offsets = make(n, [5, 0, 70], 0, 0, 64, n, torch.float16)
    for od in (torch.float32, torch.float16, torch.bfloat16):
        want, mag, _ = grouped(x, w, off)
        assert_product(K.grouped_gemm(x, w, offsets, out_dtype=od), want, mag, 64, str(od))


@pytest.mark.parametrize("knobs", [dict(tile_n=64), dict(tile_n=128), dict(tile_n=192), dict(tile_n=256),
                                   dict(tile_n=128, cta_group=2), dict(tile_n=256, cta_group=2), dict(tile_n=192, cta_group=2),
                                   dict(stages=1), dict(acc_stages=1), dict(max_ctas=2), dict(max_ctas=3, stages=2)])
def test_knobs_do_not_change_the_product(K, knobs):
    c = [300, 0, 1, 97, 514]
    x, w, dy, off, offsets = make(5, c, 1, 1, 200, 328, torch.bfloat16)
    own = grouped(clean(x), w, off)[2]
    want, mag, _ = grouped(clean(x), w, off)
    assert_product(K.grouped_gemm(x, w, offsets, knobs=knobs)[own], want[own], mag[own], 200, "y")
    want, mag, _ = grouped(clean(dy), w.transpose(1, 2), off)
    assert_product(K.grouped_gemm_dx(dy, w, offsets, knobs=knobs)[own], want[own], mag[own], 328, "dx")
    if knobs.get("cta_group") != 2:
        want, mag = grouped_dw(clean(dy), clean(x), off, len(c))
        assert_product(K.grouped_gemm_dw(dy, x, offsets, knobs=knobs), want, mag, 514, "dw")


@pytest.mark.parametrize("split", [2, 4, 8])
@pytest.mark.parametrize("counts", ["decode", "uneven", "tile_edges", "empty"])
@pytest.mark.parametrize("k,n", [(8, 40), (520, 264), (1024, 1001)])
def test_a_reduction_over_a_cluster(K, split, counts, k, n):
    c = COUNTS[counts]
    x, w, _, off, offsets = make(split, c, 2, 3, k, n, torch.bfloat16)
    want, mag, own = grouped(clean(x), w, off)
    for od in (torch.float32, torch.bfloat16):
        for extra in (dict(), dict(max_ctas=2 * split), dict(stages=1)):
            out = torch.full((x.shape[0], n), 7.0, dtype=od, device="cuda")
            K.grouped_gemm(x, w, offsets, out=out, knobs=dict(tile_n=64, split_k=split, **extra))
            assert_product(out[own], want[own], mag[own], k, str(extra))
            assert (out[~own] == 7.0).all()


@pytest.mark.parametrize("T,E", [(1, 1), (1, 64), (5, 3), (8, 1), (9, 1), (16, 2), (40, 40), (64, 100)])
@pytest.mark.parametrize("k,n", [(8, 1), (264, 40), (2056, 17), (4096, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_few_rows(K, T, E, k, n, dtype):
    g = torch.Generator().manual_seed(T * E + k)
    c = torch.bincount(torch.randint(0, E, (T,), generator=g), minlength=E).tolist()
    x, w, _, off, offsets = make(T + k, c, 1, 1, k, n, dtype)
    want, mag, own = grouped(clean(x), w, off)
    for od in (torch.float32, dtype):
        out = torch.full((T + 2, n), 7.0, dtype=od, device="cuda")
        K.grouped_gemm(x, w, offsets, out=out)
        assert_product(out[own], want[own], mag[own], k)
        assert (out[~own] == 7.0).all()


def test_an_infinity_stays_in_its_group(K):
    x, w, dy, off, offsets = make(3, [5, 9, 20], 0, 0, 64, 64, torch.float16)
    x[6], dy[6] = torch.inf, torch.nan
    y = K.grouped_gemm(x, w, offsets)
    assert torch.isfinite(y[:6]).all() and torch.isfinite(y[7:]).all() and not torch.isfinite(y[6]).any()
    dw = K.grouped_gemm_dw(dy, x, offsets)
    assert torch.isfinite(dw[0]).all() and torch.isfinite(dw[2]).all() and torch.isnan(dw[1]).all()


def test_many_groups(K):
    g = torch.Generator().manual_seed(1)
    c = torch.randint(0, 3, (1024,), generator=g).tolist()
    x, w, dy, off, offsets = make(9, c, 0, 0, 64, 72, torch.bfloat16)
    want, mag, _ = grouped(x, w, off)
    assert_product(K.grouped_gemm(x, w, offsets), want, mag, 64, "y")
    want, mag = grouped_dw(dy, x, off, 1024)
    assert_product(K.grouped_gemm_dw(dy, x, offsets), want, mag, 2, "dw")


def test_no_rows(K):
    w = torch.ones(3, 16, 8, dtype=torch.float16, device="cuda")
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert K.grouped_gemm(w.new_empty(0, 8), w, offsets).shape == (0, 16)
    assert K.grouped_gemm_dx(w.new_empty(0, 16), w, offsets).shape == (0, 8)
    dw = torch.full((3, 16, 8), 7.0, device="cuda")
    K.grouped_gemm_dw(w.new_empty(0, 16), w.new_empty(0, 8), offsets, out=dw)
    assert (dw == 0).all()
    plan = K.plan_grouped_gemm_dw(w.new_empty(0, 16), w.new_empty(0, 8), offsets, out=dw.fill_(7.0))
    plan.launch()
    assert (dw == 0).all()


@pytest.mark.parametrize("off", [[-5, 4, 8], [0, 4, 1000], [6, 2, 8], [8, 8, 8], [0, 2 ** 31 - 1, 8]])
def test_offsets_are_clamped(K, off):
    """Offsets outside the rows or out of order: rows that one group owns are right, the others untouched."""
    from grouped_util import clamped
    x, w, dy, _, _ = make(4, [8, 0], 0, 0, 64, 64, torch.float16)
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    owners = torch.zeros(8, dtype=torch.int64)
    for s, t in clamped(off, 8):
        owners[s:t] += 1
    once = (owners == 1).cuda()
    out = torch.full((8, 64), 7.0, device="cuda")
    K.grouped_gemm(x, w, offsets, out=out)
    want, mag, _ = grouped(x, w, off)
    assert_product(out[once], want[once], mag[once], 64)
    assert (out[(owners == 0).cuda()] == 7.0).all()
    want, mag = grouped_dw(dy, x, off, 2)
    assert_product(K.grouped_gemm_dw(dy, x, offsets), want, mag, 8)


def test_graph_replay_with_other_offsets_and_streams(K):
    x, w, dy, off, offsets = make(6, [40, 3, 90], 0, 0, 128, 192, torch.bfloat16)
    out = torch.empty(133, 192, device="cuda")
    dw = torch.empty(3, 192, 128, device="cuda")
    plan = K.plan_grouped_gemm(x, w, offsets, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            plan.launch()
            K.grouped_gemm_dw(dy, x, offsets, out=dw)
    torch.cuda.current_stream().wait_stream(side)
    for other in ([0, 40, 43, 133], [0, 0, 133, 133], [0, 65, 66, 133]):
        offsets.copy_(torch.tensor(other, dtype=torch.int32))
        out.fill_(7.0)
        dw.fill_(7.0)
        graph.replay()
        want, mag, _ = grouped(x, w, other)
        assert_product(out, want, mag, 128)
        want, mag = grouped_dw(dy, x, other, 3)
        assert_product(dw, want, mag, 133)
    # two streams at once
    res = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            res.append([K.grouped_gemm(x, w, offsets) for _ in range(4)])
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for r in res:
        for y in r:
            assert torch.equal(y, res[0][0])


def test_gradients_against_differences(K):
    """The directional derivative of sum(c * y) by central differences of the forward operator.  y is linear in
    x and in w, so the difference quotient has no truncation error, only that of two forward passes."""
    x, w, dy, off, offsets = make(8, [20, 0, 44], 0, 0, 64, 128, torch.float16)
    g = torch.Generator(device="cuda").manual_seed(2)
    # a direction and a step that fp16 holds exactly: multiples of 2^-6 on values rounded to 2^-6
    x = (x * 64).round() / 64
    w = (w * 64).round() / 64
    vx = torch.randint(-2, 3, x.shape, generator=g, device="cuda").half() / 64
    vw = torch.randint(-2, 3, w.shape, generator=g, device="cuda").half() / 64
    dx, dw = K.grouped_gemm_dx(dy, w, offsets), K.grouped_gemm_dw(dy, x, offsets)
    up, down = (K.grouped_gemm(x + s * vx, w, offsets).double() for s in (1, -1))
    mag = grouped(x.abs() + vx.abs(), w.abs(), off)[1]
    tol = 64 * 2.0 ** -23 * (2 * mag * dy.double().abs()).sum() + \
        128 * 2.0 ** -23 * (grouped(dy, w.transpose(1, 2), off)[1] * vx.double().abs()).sum() * 2
    assert abs(((up - down) * dy.double()).sum() - 2 * (dx.double() * vx.double()).sum()) <= tol
    up, down = (K.grouped_gemm(x, w + s * vw, offsets).double() for s in (1, -1))
    mag = grouped(x.abs(), w.abs() + vw.abs(), off)[1]
    tol = 64 * 2.0 ** -23 * (2 * mag * dy.double().abs()).sum() + \
        44 * 2.0 ** -23 * (grouped_dw(dy, x, off, 3)[1] * vw.double().abs()).sum() * 2
    assert abs(((up - down) * dy.double()).sum() - 2 * (dw.double() * vw.double()).sum()) <= tol


def test_plans_report_their_knobs(K):
    x, w, dy, _, offsets = make(6, [40, 3, 90], 0, 0, 128, 192, torch.bfloat16)
    for plan in (K.plan_grouped_gemm(x, w, offsets), K.plan_grouped_gemm_dx(dy, w, offsets),
                 K.plan_grouped_gemm_dw(dy, x, offsets)):
        k = plan.knobs()
        assert k["tile_n"] in (64, 128, 192, 256) and k["stages"] >= 1 and k["grid"] >= 1 and k["smem_bytes"] <= 232448
    few = K.plan_grouped_gemm(x[:3].contiguous(), w, offsets)
    assert few.knobs()["tile_n"] == 0  # a kernel without tiles
    for bad in (dict(tile_n=64, split_k=3), dict(tile_n=128, split_k=2), dict(tile_n=64, cta_group=2), dict(tile_n=256, stages=12)):
        from heron_b200._lib import HeronB200Error
        with pytest.raises(HeronB200Error):
            K.plan_grouped_gemm(x, w, offsets, knobs=bad)


def test_a_silent_producer_ends_in_a_status(K):
    """The bounded waits: nothing is loaded, the launch ends by itself and reports it."""
    from heron_b200 import _lib
    x, w, dy, off, offsets = make(6, [40, 3, 90], 0, 0, 128, 192, torch.bfloat16)
    for fn, args in ((K.grouped_gemm, (x, w)), (K.grouped_gemm_dx, (dy, w)), (K.grouped_gemm_dw, (dy, x))):
        fn(*args, offsets, knobs=dict(silent_producer=1))
        assert _lib.last_status() == _lib.HB_ERR_TIMEOUT
    for knobs in (dict(silent_producer=1, cta_group=2, tile_n=128), dict(silent_producer=1, tile_n=64, split_k=4)):
        K.grouped_gemm(x, w, offsets, knobs=knobs)
        assert _lib.last_status() == _lib.HB_ERR_TIMEOUT
    want, mag, _ = grouped(x, w, off)
    assert_product(K.grouped_gemm(x, w, offsets), want, mag, 128)


@pytest.mark.parametrize("knobs", [None, dict(tile_n=64), dict(tile_n=128, cta_group=2)])
def test_overlapping_offsets(K, knobs):
    """Offsets out of order whose ranges overlap: a row that one group owns is right, a row of two groups is one of the
    two results, a row of none is untouched."""
    from grouped_util import clamped
    g = torch.Generator().manual_seed(3)
    cases = [(8, [0, 6, 2, 8]), (8, [0, 5, 1, 8]), (8, [3, 7, 0, 6]), (20, [0, 11, 3, 20]), (40, [30, 9, 35, 2])]
    cases += [(T, torch.randint(-2, T + 3, (E + 1,), generator=g).tolist()) for T, E in ((8, 5), (8, 8), (30, 41), (40, 64))]
    for T, off in cases:
        E = len(off) - 1
        x, w, dy, _, _ = make(T + E, [T] + [0] * (E - 1), 0, 0, 264, 72, torch.bfloat16)
        offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
        for fn, a, b in ((K.grouped_gemm, x, w), (K.grouped_gemm_dx, dy, w.transpose(1, 2))):
            out = torch.full((T, b.shape[1]), 7.0, device="cuda")
            fn(a, w, offsets, out=out, knobs=knobs)
            near = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
            free = torch.ones(T, dtype=torch.bool, device="cuda")
            for e, (s, t) in enumerate(clamped(off, T)):
                want, mag, _ = grouped(a[s:t], b[e][None], [0, t - s])
                k = a.shape[1]
                near[s:t] |= (out[s:t].double() - want).abs() <= k * 2.0 ** -23 * mag
                free[s:t] = False
            assert near[~free].all(), "%s %s: rows %s" % (fn.__name__, off, (~near.all(1) & ~free).nonzero().flatten().tolist())
            assert (out[free] == 7.0).all()


def test_other_threads_run_while_a_launch_waits(K):
    """Launches behind a long kernel fill the stream's queue until one of them has to wait; Python's lock is free
    meanwhile.  (A host function in that queue that needs the lock would otherwise wait for good.)"""
    import threading
    import time
    x, w, dy, _, offsets = make(1, [2, 2], 0, 0, 64, 64, torch.float16)
    out = torch.empty(4, 64, device="cuda")
    codes, scales = K.quantize_mxfp4(x)
    wq = K.quantize_mxfp4(w[0])
    calls = [lambda: K.grouped_gemm(x, w, offsets, out=out), lambda: K.quantize_mxfp4(x, codes=codes, scales=scales),
             lambda: K.dequantize_mxfp4(codes, scales, out=out), lambda: K.gemm_mxfp4(codes, scales, *wq, out=out)]
    for call in calls:
        call()
        torch.cuda.synchronize()
        gaps, stop = [0.0], threading.Event()

        def watch():
            last = time.perf_counter()
            while not stop.is_set():
                time.sleep(0.001)
                now = time.perf_counter()
                gaps.append(now - last)
                last = now
        thread = threading.Thread(target=watch)
        thread.start()
        torch.cuda._sleep(800_000_000)  # 0.4 s
        longest = 0.0
        for _ in range(3000):
            t0 = time.perf_counter()
            call()
            longest = max(longest, time.perf_counter() - t0)
        stop.set()
        thread.join()
        torch.cuda.synchronize()
        assert longest > 0.1, "no launch had to wait: the test shows nothing"
        assert max(gaps) < longest / 2


def test_tensors_that_require_a_gradient(K):
    """Refused where a graph would be expected; in an autograd.Function the operators are its forward and backward."""
    x, w, dy, off, offsets = make(2, [20, 0, 44], 0, 0, 64, 128, torch.float16)
    x.requires_grad_()
    w.requires_grad_()
    for call in (lambda: K.grouped_gemm(x, w, offsets), lambda: K.grouped_gemm(x.detach(), w, offsets),
                 lambda: K.grouped_gemm(x, w.detach(), offsets), lambda: K.grouped_gemm_dx(dy, w, offsets),
                 lambda: K.grouped_gemm_dw(dy, x, offsets),
                 lambda: K.grouped_gemm(x.detach(), w.detach(), offsets, out=torch.empty(64, 128, device="cuda").requires_grad_())):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()

    class Experts(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ctx.save_for_backward(x, w)
            return K.grouped_gemm(x, w, offsets, out_dtype=x.dtype)

        @staticmethod
        def backward(ctx, dy):
            x, w = ctx.saved_tensors
            dy = dy.contiguous()
            return K.grouped_gemm_dx(dy, w, offsets, out_dtype=x.dtype), K.grouped_gemm_dw(dy, x, offsets, out_dtype=w.dtype)
    y = Experts.apply(x, w)
    y.backward(dy)
    want, mag, _ = grouped(x.detach(), w.detach(), off)
    assert_product(y.detach(), want, mag, 64)
    want, mag, _ = grouped(dy, w.detach().transpose(1, 2), off)
    assert_product(x.grad, want, mag, 128)
    want, mag = grouped_dw(dy, x.detach(), off, 3)
    assert_product(w.grad, want, mag, 44)


def test_without_the_front_end(K, monkeypatch):
    """The Python path does the same calls."""
    from heron_b200._lib import HeronB200Error
    x, w, dy, off, offsets = make(2, [20, 0, 44], 0, 0, 64, 128, torch.float16)

    def all_calls():
        xq, wq = K.quantize_mxfp4(x, offsets=offsets), K.quantize_mxfp4(w)
        aq, bq = K.quantize_mxfp4(x), K.quantize_mxfp4(w[0])
        return [K.grouped_gemm(x, w, offsets), K.grouped_gemm_dx(dy, w, offsets), K.grouped_gemm_dw(dy, x, offsets),
                K.grouped_gemm_mxfp4(*xq, *wq, offsets), K.gemm_mxfp4(*aq, *bq), K.dequantize_mxfp4(*wq)]
    want = all_calls()
    front = K._Front()
    for name in front.NAMES:
        setattr(front, name, lambda *args: None)
    monkeypatch.setattr(K, "_fast", front)
    for got, ref in zip(all_calls(), want):
        assert torch.equal(got, ref)
    with pytest.raises(HeronB200Error):
        K.grouped_gemm(x, w.bfloat16(), offsets)


NARROW = {"few": [1, 2, 3, 2] * 10, "uneven": [0, 1, 40, 3, 64, 0, 33, 5] * 5, "long_runs": [0] * 8 + [70] * 32}


@pytest.mark.parametrize("counts", list(NARROW))
@pytest.mark.parametrize("m,r", [(2048, 64), (2040, 200), (2048, 520)])
@pytest.mark.parametrize("od", [torch.float32, torch.bfloat16])
def test_narrow_tiles_in_several_rounds(K, counts, m, r, od):
    """More tiles than two CTAs on every SM take at once: rings and accumulators go round from tile to tile."""
    c = NARROW[counts]
    x, w, _, off, offsets = make(m + r, c, 1, 2, r, m, torch.bfloat16)
    out = torch.full((x.shape[0], m), 7.0, dtype=od, device="cuda")
    plan = K.plan_grouped_gemm(x, w, offsets, out=out)
    if counts != "long_runs":  # (long runs: about 50 rows a group and more take wider tiles)
        assert plan.knobs()["tile_n"] == 64 and plan.knobs()["grid"] > K._lib.load().hb_sm_count()
    plan.launch()
    want, mag, own = grouped(clean(x), w, off)
    assert_product(out[own], want[own], mag[own], r, "y")
    assert (out[~own] == 7.0).all()
    dy, wt = x, w.transpose(1, 2).contiguous()  # (rows of r values, weights (E, r, m): dx has m features)
    out.fill_(7.0)
    K.grouped_gemm_dx(dy, wt, offsets, out=out)
    assert_product(out[own], want[own], mag[own], r, "dx")
    assert (out[~own] == 7.0).all()


@pytest.mark.parametrize("T,E", [(2, 33), (7, 40), (8, 100), (8, 1024)])
@pytest.mark.parametrize("k,n", [(264, 40), (2056, 17)])
def test_few_rows_over_many_groups(K, T, E, k, n):
    """The kernel of few rows with more groups than a warp looks at at once, offsets in order and not."""
    g = torch.Generator().manual_seed(T + E)
    x, w, _, _, _ = make(T + k, [T] + [0] * (E - 1), 0, 0, k, n, torch.bfloat16)
    ordered = torch.randint(0, T + 1, (E + 1,), generator=g).sort().values.tolist()
    for off in (ordered, torch.randint(-2, T + 3, (E + 1,), generator=g).tolist(), [T] * (E - 1) + [1, T], [0] * E + [T]):
        offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
        out = torch.full((T, n), 7.0, device="cuda")
        plan = K.plan_grouped_gemm(x, w, offsets, out=out)
        assert plan.knobs()["tile_n"] == 0  # the kernel without tiles
        plan.launch()
        near = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
        from grouped_util import clamped
        free = torch.ones(T, dtype=torch.bool, device="cuda")
        for e, (s, t) in enumerate(clamped(off, T)):
            if t > s:
                want, mag, _ = grouped(x[s:t], w[e][None], [0, t - s])
                near[s:t] |= (out[s:t].double() - want).abs() <= k * 2.0 ** -23 * mag
                free[s:t] = False
        assert near[~free].all() and (out[free] == 7.0).all()


def test_which_products_stream(K):
    """The rule of hb_plan_group.cuh, both sides of each border."""
    def tiles(T, E, n, k):
        x, w = torch.zeros(T, k, dtype=torch.float16, device="cuda"), torch.zeros(E, n, k, dtype=torch.float16, device="cuda")
        return K.plan_grouped_gemm(x, w, torch.zeros(E + 1, dtype=torch.int32, device="cuda")).knobs()["tile_n"] > 0

    def mx_tiles(T, E, n, k):
        kt = -(-k // 128)
        a, w = (torch.zeros(*s, k // 2, dtype=torch.uint8, device="cuda") for s in ((T,), (E, n)))
        xs = torch.zeros((T // 128 + E) * kt * 512, dtype=torch.uint8, device="cuda")
        ws = torch.zeros(E, -(-n // 128) * kt * 512, dtype=torch.uint8, device="cuda")
        return K.plan_grouped_gemm_mxfp4(a, xs, w, ws, torch.zeros(E + 1, dtype=torch.int32, device="cuda")).knobs()["tile_n"] > 0
    for T, E, n, k, want in ((8, 1, 4096, 4096, False), (8, 1, 4104, 2048, True), (1, 1, 8192, 1024, False), (1, 1, 8192, 1016, True),
                             (1, 1, 8200, 64, True), (16, 1, 2048, 2048, False), (32, 1, 2048, 2048, True), (64, 1, 512, 64, False),
                             (64, 1, 520, 64, True), (65, 1, 64, 64, True), (8, 4, 2048, 2048, False), (8, 4, 1280, 64, False),
                             (8, 4, 1288, 64, True), (9, 4, 64, 64, True), (10, 12, 64, 64, False), (13, 12, 64, 64, True)):
        assert tiles(T, E, n, k) == want, (T, E, n, k)
    for T, E, n, k, want in ((8, 1, 4096, 4096, False), (8, 1, 4128, 64, True), (1, 1, 4096, 4128, True), (9, 1, 64, 64, True),
                             (4, 4, 2048, 1024, False), (4, 4, 2049, 64, True), (2, 2, 2048, 2080, True), (64, 3, 128, 64, False)):
        assert mx_tiles(T, E, n, k) == want, (T, E, n, k)


@pytest.mark.parametrize("tile_n", [128, 192, 256])
def test_pairs_do_not_share_an_sm(K, tile_n):
    """Whatever the stages, two CTAs of pairs need more shared memory than an SM has."""
    from heron_b200 import kernels
    x, w, dy, _, offsets = make(2, [300, 20, 44], 0, 0, 64, 128, torch.float16)
    xq, wq = kernels.quantize_mxfp4(x, offsets=offsets), kernels.quantize_mxfp4(w)
    for stages in (0, 1, 2, 3):
        knobs = dict(tile_n=tile_n, cta_group=2, stages=stages)
        for plan in (K.plan_grouped_gemm(x, w, offsets, knobs=knobs), K.plan_grouped_gemm_dx(dy, w, offsets, knobs=knobs),
                     K.plan_grouped_gemm_mxfp4(*xq, *wq, offsets, knobs=knobs)):
            assert 2 * (plan.knobs()["smem_bytes"] + 1024) > 228 * 1024 and plan.knobs()["smem_bytes"] <= 232448
