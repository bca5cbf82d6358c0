"""Operators called from a thread that has not used the GPU yet (autograd's, a server's worker)."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(hb_lib):
    assert torch.cuda.is_available(), "GPU tests need a B200"
    from heron_b200 import kernels
    assert hb_lib.hb_sm_count() > 0, "libheron_b200.so found no sm_100 device"
    return kernels


def calls(K):
    """Name -> a call on buffers made here, and its output."""
    a, b = torch.randn(256, 256, device="cuda").half(), torch.randn(256, 256, device="cuda").half()
    out = torch.empty(256, 256, device="cuda")
    offsets = torch.tensor([0, 100, 256], dtype=torch.int32, device="cuda")
    w = torch.stack([b, a])
    dw = torch.empty(2, 256, 256, device="cuda")
    aq, bq = K.quantize_mxfp4(a), K.quantize_mxfp4(b)
    ag, wq = K.quantize_mxfp4(a, offsets=offsets), K.quantize_mxfp4(w)
    img, flt = torch.randn(1, 14, 14, 64, device="cuda").half(), torch.randn(3, 3, 64, 64, device="cuda").half()
    conv = torch.empty(1, 14, 14, 64, device="cuda")
    return {
        "gemm": (lambda: K.gemm(a, b, out=out), out),
        "bmm": (lambda: K.bmm(a[None], b[None], out=out[None]), out),
        "conv2d": (lambda: K.conv2d_nhwc(img, flt, padding=1, out=conv), conv),
        "grouped_gemm": (lambda: K.grouped_gemm(a, w, offsets, out=out), out),
        "grouped_gemm, knobs": (lambda: K.grouped_gemm(a, w, offsets, out=out, knobs=dict(tile_n=64)), out),
        "grouped_gemm_dx": (lambda: K.grouped_gemm_dx(a, w, offsets, out=out), out),
        "grouped_gemm_dw": (lambda: K.grouped_gemm_dw(a, b, offsets, out=dw), dw),
        "plan": (lambda: K.plan_grouped_gemm(a, w, offsets, out=out).launch(), out),
        "gemm_mxfp4": (lambda: K.gemm_mxfp4(*aq, *bq, out=out), out),
        "grouped_gemm_mxfp4": (lambda: K.grouped_gemm_mxfp4(*ag, *wq, offsets, out=out), out),
        "quantize_mxfp4": (lambda: K.quantize_mxfp4(a, codes=aq[0], scales=aq[1]), aq[0]),
    }


@pytest.mark.parametrize("name", ["gemm", "bmm", "conv2d", "grouped_gemm", "grouped_gemm, knobs", "grouped_gemm_dx",
                                  "grouped_gemm_dw", "plan", "gemm_mxfp4", "grouped_gemm_mxfp4", "quantize_mxfp4"])
def test_a_thread_of_its_own(K, name):
    call, out = calls(K)[name]
    call()
    torch.cuda.synchronize()
    want = out.clone()
    out.zero_()
    torch.cuda.synchronize()
    failed = []

    def work():
        try:
            call()
        except Exception as e:  # noqa: BLE001  (told to the test's own thread)
            failed.append(e)
    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert not failed, failed[0]
    torch.cuda.synchronize()
    assert torch.equal(out, want)
