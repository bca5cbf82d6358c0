"""Device-tensor front end of the C ABI: torch tensors in, torch tensors out.

torch is used for device memory and streams only; every function here hands raw device pointers
to libheron_b200.so and raises ``HeronB200Error`` on a non-zero status.  Operand conventions are
the reference operators' own: GEMM / batched GEMM take ``B`` as (N, K) (ops/cuda/dense.py:6,
ops/cuda/batch_matmul.py:8), NHWC conv takes an HWIO filter (ops/cuda/conv2d.py:155).
"""
import ctypes
import warnings

import torch

from . import _lib

_TORCH_CODES = {
    torch.float16: _lib.HB_F16,
    torch.float32: _lib.HB_F32,
    torch.int8: _lib.HB_S8,
    torch.uint8: _lib.HB_U8,
    torch.int32: _lib.HB_S32,
}

TORCH_DTYPES = {
    "float16": torch.float16,
    "float32": torch.float32,
    "int8": torch.int8,
    "uint8": torch.uint8,
    "int32": torch.int32,
}


def _code(t):
    try:
        return _TORCH_CODES[t.dtype]
    except KeyError:
        raise _lib.HeronB200Error(_lib.HB_ERR_DTYPE, "dtype %s" % t.dtype)


def _dev(t, name):
    if not t.is_cuda:
        raise ValueError("%s must be a CUDA tensor: the kernels have no CPU path" % name)
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return ctypes.c_void_p(t.data_ptr())


def _out(out, shape, like, name="out"):
    """A caller-supplied output must be exactly what the kernel will write: a wrong size would put
    stores past the end of the buffer."""
    if tuple(out.shape) != tuple(shape):
        raise ValueError("%s has shape %s, the operator writes %s" % (name, tuple(out.shape), tuple(shape)))
    if out.dtype not in _TORCH_CODES:
        raise _lib.HeronB200Error(_lib.HB_ERR_DTYPE, "dtype %s" % out.dtype)
    if out.device != like.device:
        raise ValueError("%s is on %s, the inputs are on %s" % (name, out.device, like.device))
    return out


def _same_device(*tensors):
    """All operands on one device, and that device current: the library launches on the current
    CUDA device, so a tensor elsewhere would hand it a pointer of another GPU."""
    dev = tensors[0].device
    for t in tensors:
        if t.device != dev:
            raise ValueError("operands live on different devices: %s and %s" % (dev, t.device))
    if dev.type == "cuda" and dev.index is not None and dev.index != torch.cuda.current_device():
        raise ValueError("tensors are on cuda:%d but the current device is cuda:%d; wrap the call in "
                         "torch.cuda.device(...)" % (dev.index, torch.cuda.current_device()))


def _bytes_buf(buf, need, like, name):
    if buf.numel() * buf.element_size() < need:
        raise ValueError("%s holds %d bytes, the operator needs %d" % (name, buf.numel() * buf.element_size(), need))
    if buf.device != like.device:
        raise ValueError("%s is on %s, the inputs are on %s" % (name, buf.device, like.device))
    return buf


def _knobs(knobs):
    if knobs is None:
        return None
    if isinstance(knobs, _lib.HbKnobs):
        return ctypes.byref(knobs)
    return ctypes.byref(_lib.HbKnobs.from_dict(knobs))


def _stream(t):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def default_out_dtype(in_dtype):
    return torch.float32 if in_dtype == torch.float16 else torch.int32


def gemm(a, b, out=None, out_dtype=None, knobs=None):
    """out[M,N] = sum_k a[M,k] * b[N,k]."""
    M, K = a.shape
    N, K2 = b.shape
    if K != K2:
        raise ValueError("a is (M,K), b is (N,K): K differs")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or default_out_dtype(a.dtype), device=a.device)
    _same_device(a, b, _out(out, (M, N), a))
    rc = _lib.load().hb_gemm(_dev(a, "a"), _dev(b, "b"), _dev(out, "out"), M, K, N, _code(a),
                             _code(b), _code(out), _knobs(knobs), _stream(a))
    _lib.check(rc, "hb_gemm")
    return out


def bmm(a, b, out=None, out_dtype=None, knobs=None):
    """out[b,M,N] = sum_k a[b,M,k] * b[b,N,k]."""
    B, M, K = a.shape
    B2, N, K2 = b.shape
    if K != K2 or B != B2:
        raise ValueError("a is (B,M,K), b is (B,N,K): shapes differ")
    if out is None:
        out = torch.empty((B, M, N), dtype=out_dtype or default_out_dtype(a.dtype), device=a.device)
    _same_device(a, b, _out(out, (B, M, N), a))
    rc = _lib.load().hb_bmm(_dev(a, "a"), _dev(b, "b"), _dev(out, "out"), B, M, K, N, _code(a),
                            _code(b), _code(out), _knobs(knobs), _stream(a))
    _lib.check(rc, "hb_bmm")
    return out


def _pair(v):
    if isinstance(v, int):
        return v, v
    a, b = v
    return int(a), int(b)


def conv_out_hw(H, W, KH, KW, stride, padding, dilation):
    """Output extent of the reference's NHWC conv (ops/cuda/conv2d.py:165-175)."""
    sh, sw = _pair(stride)
    dh, dw = _pair(dilation)
    HO = (H - ((KH - 1) * dh + 1) + 2 * padding) // sh + 1
    WO = (W - ((KW - 1) * dw + 1) + 2 * padding) // sw + 1
    if HO <= 0 or WO <= 0:
        # the window does not fit the padded image: the library's own answer, before any allocation
        raise _lib.HeronB200Error(_lib.HB_ERR_SHAPE, "conv output extent %d x %d" % (HO, WO))
    return HO, WO


def conv2d_nhwc(x, w, stride=1, padding=0, dilation=1, out=None, out_dtype=None, knobs=None):
    """out[n,y,x,f] = sum pad(x)[n, y*s+ry*d, x*s+rx*d, c] * w[ry,rx,c,f]; w is HWIO."""
    N, H, W, CI = x.shape
    KH, KW, CI2, CO = w.shape
    if CI != CI2:
        raise ValueError("input channels of x and w differ")
    sh, sw = _pair(stride)
    dh, dw = _pair(dilation)
    HO, WO = conv_out_hw(H, W, KH, KW, stride, padding, dilation)
    if out is None:
        out = torch.empty((N, HO, WO, CO), dtype=out_dtype or default_out_dtype(x.dtype),
                          device=x.device)
    _same_device(x, w, _out(out, (N, HO, WO, CO), x))
    rc = _lib.load().hb_conv2d_nhwc(_dev(x, "x"), _dev(w, "w"), _dev(out, "out"), N, H, W, CI, CO,
                                    KH, KW, sh, sw, int(padding), dh, dw, _code(x), _code(w),
                                    _code(out), _knobs(knobs), _stream(x))
    _lib.check(rc, "hb_conv2d_nhwc")
    return out


def conv2d_nhwc_packed(x, w_packed, CO, KH, KW, stride=1, padding=0, dilation=1, sco=64, out=None,
                       scratch=None, knobs=None):
    """The x86 operator's conv: uint8 NHWC input, int8 filter packed (CO/sco,KH,KW,CI/4,sco,4)."""
    N, H, W, CI = x.shape
    sh, sw = _pair(stride)
    dh, dw = _pair(dilation)
    HO, WO = conv_out_hw(H, W, KH, KW, stride, padding, dilation)
    lib = _lib.load()
    need = lib.hb_conv2d_packed_scratch_bytes(CI, CO, KH, KW)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.int8, device=x.device)
    if out is None:
        out = torch.empty((N, HO, WO, CO // sco, sco), dtype=torch.int32, device=x.device)
    _packed_checks(x, w_packed, out, scratch, need, (N, HO, WO, CO // sco, sco), (CO // sco, KH, KW, CI // 4, sco, 4))
    rc = lib.hb_conv2d_nhwc_packed(_dev(x, "x"), _dev(w_packed, "w_packed"), _dev(out, "out"), N, H,
                                   W, CI, CO, KH, KW, sh, sw, int(padding), dh, dw, int(sco),
                                   _dev(scratch, "scratch"), scratch.numel(), _knobs(knobs),
                                   _stream(x))
    _lib.check(rc, "hb_conv2d_nhwc_packed")
    return out


def _packed_checks(x, w_packed, out, scratch, need, out_shape, w_shape):
    n_w = 1
    for d in w_shape:
        n_w *= d
    if w_packed.numel() != n_w or w_packed.element_size() != 1:
        raise ValueError("w_packed holds %d elements, the packed filter %s has %d" % (w_packed.numel(), w_shape, n_w))
    if tuple(out.shape) == out_shape[:3] + (out_shape[3] * out_shape[4],):
        out_shape = tuple(out.shape)  # (N, HO, WO, CO): the same bytes as (N, HO, WO, CO/sco, sco)
    _same_device(x, w_packed, _out(out, out_shape, x), _bytes_buf(scratch, need, x, "scratch"))


def _nchw_common(x, w, stride, padding, out, out_dtype, scratch):
    N, CI, H, W = x.shape
    CO, CI2, KH, KW = w.shape
    if CI != CI2:
        raise ValueError("input channels of x and w differ")
    sh, sw = _pair(stride)
    HO, WO = conv_out_hw(H, W, KH, KW, stride, padding, 1)
    if out is None:
        out = torch.empty((N, CO, HO, WO), dtype=out_dtype or default_out_dtype(x.dtype), device=x.device)
    need = _lib.load().hb_conv2d_nchw_scratch_bytes(N, H, W, CI, CO, KH, KW, sh, sw, int(padding), _code(x),
                                                   _code(out))
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    _same_device(x, w, _out(out, (N, CO, HO, WO), x), _bytes_buf(scratch, need, x, "scratch"))
    return (N, H, W, CI, CO, KH, KW, sh, sw, int(padding)), out, scratch


def conv2d_nchw(x, w, stride=1, padding=0, out=None, out_dtype=None, scratch=None, knobs=None):
    """out[n,c,p,q] = sum pad(x)[n,ci,p*s+kh,q*s+kw] * w[c,ci,kh,kw]; x NCHW, w OIHW, dilation 1."""
    dims, out, scratch = _nchw_common(x, w, stride, padding, out, out_dtype, scratch)
    rc = _lib.load().hb_conv2d_nchw(_dev(x, "x"), _dev(w, "w"), _dev(out, "out"), *dims, _code(x), _code(w),
                                    _code(out), _dev(scratch, "scratch"), scratch.numel(), _knobs(knobs),
                                    _stream(x))
    _lib.check(rc, "hb_conv2d_nchw")
    return out


def plan_conv2d_nchw(x, w, stride=1, padding=0, out=None, out_dtype=None, scratch=None, knobs=None):
    dims, out, scratch = _nchw_common(x, w, stride, padding, out, out_dtype, scratch)
    h = ctypes.c_void_p()
    rc = _lib.load().hb_plan_conv2d_nchw(ctypes.byref(h), _dev(x, "x"), _dev(w, "w"), _dev(out, "out"), *dims,
                                         _code(x), _code(w), _code(out), _dev(scratch, "scratch"),
                                         scratch.numel(), _knobs(knobs))
    _lib.check(rc, "hb_plan_conv2d_nchw")
    return Plan(h, (x, w, scratch), out)


class Plan:
    """A launch-ready kernel bound to fixed buffers (hb_plan): build once, launch many times.

    Keeps references to the tensors it was built on so that their memory outlives the plan.
    """

    def __init__(self, handle, tensors, out):
        self._handle = handle
        self._tensors = tensors
        self.out = out

    def launch(self, stream=None):
        if stream is None:
            stream = torch.cuda.current_stream(self.out.device).cuda_stream
        _lib.check(_lib.load().hb_plan_launch(self._handle, ctypes.c_void_p(stream)), "hb_plan_launch")
        return self.out

    __call__ = launch

    def knobs(self):
        """Resolved knobs plus the persistent grid size and dynamic shared memory of the launch."""
        k = _lib.HbKnobs()
        grid, smem = ctypes.c_int(0), ctypes.c_int(0)
        _lib.check(_lib.load().hb_plan_knobs(self._handle, ctypes.byref(k), ctypes.byref(grid),
                                             ctypes.byref(smem)), "hb_plan_knobs")
        d = k.to_dict()
        d["grid"], d["smem_bytes"] = grid.value, smem.value
        return d

    def set_peer_outputs(self, outs):
        """Every tile the kernel stores to this plan's output also goes to each tensor of `outs`
        (same shape, dtype and layout; typically this rank's slice of the other GPUs' output
        buffers, mapped into this process).  An empty list removes them."""
        outs = list(outs)
        for o in outs:
            if tuple(o.shape) != tuple(self.out.shape) or o.dtype != self.out.dtype or not o.is_contiguous():
                raise ValueError("a peer output must have the plan's output shape, dtype and a dense layout")
        arr = (ctypes.c_void_p * max(len(outs), 1))(*[o.data_ptr() for o in outs])
        _lib.check(_lib.load().hb_plan_set_peer_outputs(self._handle, len(outs), arr), "hb_plan_set_peer_outputs")
        self._peer_outs = outs  # (kept alive with the plan)

    def close(self):
        if self._handle is not None:
            _lib.load().hb_plan_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def plan_gemm(a, b, out=None, out_dtype=None, knobs=None):
    M, K = a.shape
    N, K2 = b.shape
    if K != K2:
        raise ValueError("a is (M,K), b is (N,K): K differs")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or default_out_dtype(a.dtype), device=a.device)
    _same_device(a, b, _out(out, (M, N), a))
    h = ctypes.c_void_p()
    rc = _lib.load().hb_plan_gemm(ctypes.byref(h), _dev(a, "a"), _dev(b, "b"), _dev(out, "out"), M,
                                  K, N, _code(a), _code(b), _code(out), _knobs(knobs))
    _lib.check(rc, "hb_plan_gemm")
    return Plan(h, (a, b), out)


def plan_bmm(a, b, out=None, out_dtype=None, knobs=None):
    B, M, K = a.shape
    B2, N, K2 = b.shape
    if K != K2 or B != B2:
        raise ValueError("a is (B,M,K), b is (B,N,K): shapes differ")
    if out is None:
        out = torch.empty((B, M, N), dtype=out_dtype or default_out_dtype(a.dtype), device=a.device)
    _same_device(a, b, _out(out, (B, M, N), a))
    h = ctypes.c_void_p()
    rc = _lib.load().hb_plan_bmm(ctypes.byref(h), _dev(a, "a"), _dev(b, "b"), _dev(out, "out"), B,
                                 M, K, N, _code(a), _code(b), _code(out), _knobs(knobs))
    _lib.check(rc, "hb_plan_bmm")
    return Plan(h, (a, b), out)


def plan_conv2d_nhwc(x, w, stride=1, padding=0, dilation=1, out=None, out_dtype=None, knobs=None):
    N, H, W, CI = x.shape
    KH, KW, CI2, CO = w.shape
    if CI != CI2:
        raise ValueError("input channels of x and w differ")
    sh, sw = _pair(stride)
    dh, dw = _pair(dilation)
    HO, WO = conv_out_hw(H, W, KH, KW, stride, padding, dilation)
    if out is None:
        out = torch.empty((N, HO, WO, CO), dtype=out_dtype or default_out_dtype(x.dtype),
                          device=x.device)
    _same_device(x, w, _out(out, (N, HO, WO, CO), x))
    h = ctypes.c_void_p()
    rc = _lib.load().hb_plan_conv2d_nhwc(ctypes.byref(h), _dev(x, "x"), _dev(w, "w"),
                                         _dev(out, "out"), N, H, W, CI, CO, KH, KW, sh, sw,
                                         int(padding), dh, dw, _code(x), _code(w), _code(out),
                                         _knobs(knobs))
    _lib.check(rc, "hb_plan_conv2d_nhwc")
    return Plan(h, (x, w), out)


def plan_conv2d_nhwc_packed(x, w_packed, CO, KH, KW, stride=1, padding=0, dilation=1, sco=64,
                            out=None, scratch=None, knobs=None):
    N, H, W, CI = x.shape
    sh, sw = _pair(stride)
    dh, dw = _pair(dilation)
    HO, WO = conv_out_hw(H, W, KH, KW, stride, padding, dilation)
    lib = _lib.load()
    need = lib.hb_conv2d_packed_scratch_bytes(CI, CO, KH, KW)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.int8, device=x.device)
    if out is None:
        out = torch.empty((N, HO, WO, CO // sco, sco), dtype=torch.int32, device=x.device)
    _packed_checks(x, w_packed, out, scratch, need, (N, HO, WO, CO // sco, sco), (CO // sco, KH, KW, CI // 4, sco, 4))
    h = ctypes.c_void_p()
    rc = lib.hb_plan_conv2d_nhwc_packed(ctypes.byref(h), _dev(x, "x"), _dev(w_packed, "w_packed"),
                                        _dev(out, "out"), N, H, W, CI, CO, KH, KW, sh, sw,
                                        int(padding), dh, dw, int(sco), _dev(scratch, "scratch"),
                                        scratch.numel(), _knobs(knobs))
    _lib.check(rc, "hb_plan_conv2d_nhwc_packed")
    return Plan(h, (x, w_packed, scratch), out)


# ---- operators next to the hot path that run on the same kernels ---------------------------
def _gemv_args(a, x, out, out_dtype):
    M, K = a.shape
    if tuple(x.shape) != (1, K):
        raise ValueError("a is (M,K), x is (1,K)")
    if out is None:
        out = torch.empty((M, 8), dtype=out_dtype or default_out_dtype(a.dtype), device=a.device)
    if tuple(out.shape) != (M, 8):
        raise ValueError("out is (M, 8): column 0 holds the product (ops/cuda/gemv.py:7)")
    return M, K, out


def gemv(a, x, out=None, out_dtype=None, knobs=None):
    """out[i,0] = sum_k a[i,k] * x[0,k]; out[i,1..7] = 0 (the reference's 8-row padded form)."""
    M, K, out = _gemv_args(a, x, out, out_dtype)
    rc = _lib.load().hb_gemv(_dev(a, "a"), _dev(x, "x"), _dev(out, "out"), M, K, _code(a), _code(x),
                             _code(out), _knobs(knobs), _stream(a))
    _lib.check(rc, "hb_gemv")
    return out


def plan_gemv(a, x, out=None, out_dtype=None, knobs=None):
    M, K, out = _gemv_args(a, x, out, out_dtype)
    h = ctypes.c_void_p()
    rc = _lib.load().hb_plan_gemv(ctypes.byref(h), _dev(a, "a"), _dev(x, "x"), _dev(out, "out"), M, K,
                                  _code(a), _code(x), _code(out), _knobs(knobs))
    _lib.check(rc, "hb_plan_gemv")
    return Plan(h, (a, x), out)


def conv1d_out_w(W, KW, stride, padding, dilation=1):
    """(W - dilated_KW + 2*pad) // stride + 1 (ops/cuda/conv1d.py:24-25, ops/x86/conv1d_int8.py:53-55)."""
    WO = (W - ((KW - 1) * dilation + 1) + 2 * padding) // stride + 1
    if WO <= 0:
        raise _lib.HeronB200Error(_lib.HB_ERR_SHAPE, "conv1d output extent %d" % WO)
    return WO


def _c1d_ncw_args(x, w, stride, padding, out, out_dtype, scratch):
    N, CI, W = x.shape
    CO, CI2, KW = w.shape
    if CI != CI2:
        raise ValueError("input channels of x and w differ")
    WO = conv1d_out_w(W, KW, int(stride), int(padding))
    if out is None:
        out = torch.empty((N, CO, WO), dtype=out_dtype or default_out_dtype(x.dtype), device=x.device)
    need = _lib.load().hb_conv1d_ncw_scratch_bytes(N, W, CI, CO, KW, int(stride), int(padding), _code(x),
                                                  _code(out))
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    return (N, W, CI, CO, KW, int(stride), int(padding)), out, scratch


def conv1d_ncw(x, w, stride=1, padding=0, out=None, out_dtype=None, scratch=None, knobs=None):
    """out[n,c,q] = sum pad(x)[n,ci,q*s+kw] * w[c,ci,kw]; x (N,CI,W), w (CO,CI,KW), dilation 1."""
    dims, out, scratch = _c1d_ncw_args(x, w, stride, padding, out, out_dtype, scratch)
    rc = _lib.load().hb_conv1d_ncw(_dev(x, "x"), _dev(w, "w"), _dev(out, "out"), *dims, _code(x), _code(w),
                                   _code(out), _dev(scratch, "scratch"), scratch.numel(), _knobs(knobs),
                                   _stream(x))
    _lib.check(rc, "hb_conv1d_ncw")
    return out


def plan_conv1d_ncw(x, w, stride=1, padding=0, out=None, out_dtype=None, scratch=None, knobs=None):
    dims, out, scratch = _c1d_ncw_args(x, w, stride, padding, out, out_dtype, scratch)
    h = ctypes.c_void_p()
    rc = _lib.load().hb_plan_conv1d_ncw(ctypes.byref(h), _dev(x, "x"), _dev(w, "w"), _dev(out, "out"), *dims,
                                        _code(x), _code(w), _code(out), _dev(scratch, "scratch"),
                                        scratch.numel(), _knobs(knobs))
    _lib.check(rc, "hb_plan_conv1d_ncw")
    return Plan(h, (x, w, scratch), out)


def _c1d_packed_args(x, CO, KW, stride, padding, dilation, sco, out, scratch):
    N, W, CI = x.shape
    WO = conv1d_out_w(W, KW, int(stride), int(padding), int(dilation))
    lib = _lib.load()
    if scratch is None:
        scratch = torch.empty(lib.hb_conv2d_packed_scratch_bytes(CI, CO, 1, KW), dtype=torch.int8,
                              device=x.device)
    if out is None:
        out = torch.empty((N, WO, CO // sco, sco), dtype=torch.int32, device=x.device)
    return (N, W, CI, CO, KW, int(stride), int(padding), int(dilation), int(sco)), out, scratch


def conv1d_nwc_packed(x, w_packed, CO, KW, stride=1, padding=0, dilation=1, sco=64, out=None,
                      scratch=None, knobs=None):
    """The x86 1-D conv: uint8 (N,W,CI) input, int8 filter packed (CO/sco, KW, CI/4, sco, 4)."""
    dims, out, scratch = _c1d_packed_args(x, CO, KW, stride, padding, dilation, sco, out, scratch)
    rc = _lib.load().hb_conv1d_nwc_packed(_dev(x, "x"), _dev(w_packed, "w_packed"), _dev(out, "out"), *dims,
                                          _dev(scratch, "scratch"), scratch.numel(), _knobs(knobs),
                                          _stream(x))
    _lib.check(rc, "hb_conv1d_nwc_packed")
    return out


def plan_conv1d_nwc_packed(x, w_packed, CO, KW, stride=1, padding=0, dilation=1, sco=64, out=None,
                           scratch=None, knobs=None):
    dims, out, scratch = _c1d_packed_args(x, CO, KW, stride, padding, dilation, sco, out, scratch)
    h = ctypes.c_void_p()
    rc = _lib.load().hb_plan_conv1d_nwc_packed(ctypes.byref(h), _dev(x, "x"), _dev(w_packed, "w_packed"),
                                               _dev(out, "out"), *dims, _dev(scratch, "scratch"),
                                               scratch.numel(), _knobs(knobs))
    _lib.check(rc, "hb_plan_conv1d_nwc_packed")
    return Plan(h, (x, w_packed, scratch), out)


def _scan_args(a, N, out, out_dtype, scratch):
    M, K = a.shape
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or default_out_dtype(a.dtype), device=a.device)
    if scratch is None:
        scratch = torch.empty(_lib.load().hb_scan_scratch_bytes(N, K, _code(a)), dtype=torch.uint8, device=a.device)
    return M, K, out, scratch


def scan(a, N, out=None, out_dtype=None, scratch=None, knobs=None):
    """out[m,n] = sum of a[m,k] over k < min(n, K): the reference's scan operator, a GEMM with the
    constant matrix B[n,k] = (n <= k) ? 0 : 1 (ops/cuda/scan.py:6-23)."""
    M, K, out, scratch = _scan_args(a, N, out, out_dtype, scratch)
    rc = _lib.load().hb_scan(_dev(a, "a"), _dev(out, "out"), M, N, K, _code(a), _code(out),
                             _dev(scratch, "scratch"), scratch.numel(), _knobs(knobs), _stream(a))
    _lib.check(rc, "hb_scan")
    return out


def plan_scan(a, N, out=None, out_dtype=None, scratch=None, knobs=None):
    M, K, out, scratch = _scan_args(a, N, out, out_dtype, scratch)
    h = ctypes.c_void_p()
    rc = _lib.load().hb_plan_scan(ctypes.byref(h), _dev(a, "a"), _dev(out, "out"), M, N, K, _code(a),
                                  _code(out), _dev(scratch, "scratch"), scratch.numel(), _knobs(knobs))
    _lib.check(rc, "hb_plan_scan")
    return Plan(h, (a, scratch), out)


def _triple(v):
    if isinstance(v, int):
        return v, v, v
    a, b, c = v
    return int(a), int(b), int(c)


def _c3d_args(x, w, stride, padding, out, out_dtype, scratch):
    N, CI, D, H, W = x.shape
    CO, CI2, KD, KH, KW = w.shape
    if CI != CI2:
        raise ValueError("input channels of x and w differ")
    sd, sh, sw = _triple(stride)
    p = int(padding)
    DO, HO, WO = (D - KD + 2 * p) // sd + 1, (H - KH + 2 * p) // sh + 1, (W - KW + 2 * p) // sw + 1
    if DO <= 0 or HO <= 0 or WO <= 0:
        raise _lib.HeronB200Error(_lib.HB_ERR_SHAPE, "conv3d output extent %d x %d x %d" % (DO, HO, WO))
    if out is None:
        out = torch.empty((N, CO, DO, HO, WO), dtype=out_dtype or default_out_dtype(x.dtype), device=x.device)
    dims = (N, D, H, W, CI, CO, KD, KH, KW, sd, sh, sw, p)
    need = _lib.load().hb_conv3d_ncdhw_scratch_bytes(*dims, _code(x), _code(out))
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    return dims, out, scratch


def conv3d_ncdhw(x, w, stride=1, padding=0, out=None, out_dtype=None, scratch=None, knobs=None):
    """out[n,c,d,p,q] = sum pad(x)[n,ci,d*sd+kd,p*sh+kh,q*sw+kw] * w[c,ci,kd,kh,kw]; x NCDHW, w OIDHW,
    dilation 1 (ops/cuda/conv3d.py:9-85)."""
    dims, out, scratch = _c3d_args(x, w, stride, padding, out, out_dtype, scratch)
    rc = _lib.load().hb_conv3d_ncdhw(_dev(x, "x"), _dev(w, "w"), _dev(out, "out"), *dims, _code(x), _code(w),
                                     _code(out), _dev(scratch, "scratch"), scratch.numel(), _knobs(knobs),
                                     _stream(x))
    _lib.check(rc, "hb_conv3d_ncdhw")
    return out


def plan_conv3d_ncdhw(x, w, stride=1, padding=0, out=None, out_dtype=None, scratch=None, knobs=None):
    dims, out, scratch = _c3d_args(x, w, stride, padding, out, out_dtype, scratch)
    h = ctypes.c_void_p()
    rc = _lib.load().hb_plan_conv3d_ncdhw(ctypes.byref(h), _dev(x, "x"), _dev(w, "w"), _dev(out, "out"), *dims,
                                          _code(x), _code(w), _code(out), _dev(scratch, "scratch"),
                                          scratch.numel(), _knobs(knobs))
    _lib.check(rc, "hb_plan_conv3d_ncdhw")
    return Plan(h, (x, w, scratch), out)


# ---- products grouped by expert --------------------------------------------------------------
# (types of these operators and of the 4-bit ones only: the operators above keep refusing bfloat16)
_WIDE_CODES = {torch.float16: _lib.HB_F16, torch.bfloat16: _lib.HB_BF16, torch.float32: _lib.HB_F32}

# The small calls of these operators are bound by the host (a token's product takes the GPU a few
# microseconds).  A call without knobs first goes to the C++ front end (csrc/hb_front.cpp), which checks,
# allocates and launches in one step; what it finds unusual it hands back (None), and the code below
# checks again, names the fault or does the call.  Without the extension it does every call, at some
# 6 us more of the host's time each.
class _Front:
    """The extension module, loaded by the first call (importing this file loads nothing)."""

    NAMES = ("grouped", "quantize", "dequantize", "mx")

    def __getattr__(self, name):
        if name not in self.NAMES:
            raise AttributeError(name)
        _lib.load()
        from . import build
        try:
            from . import _front
            if getattr(_front, "built_for", None) != build.front_key():
                raise ImportError("it is built for another torch")
        except ImportError as e:
            warnings.warn("heron_b200: no C++ front end, calls take longer on the host (run `python -m heron_b200.build`): %s"
                          % e, RuntimeWarning, stacklevel=3)
            _front = None
        for fn in self.NAMES:
            setattr(self, fn, getattr(_front, fn) if _front else lambda *args: None)
        return getattr(self, name)


_fast = _Front()


def _done(result, kind):
    if result.__class__ is int:
        _lib.check(result, kind)
    return result


_raw_stream = torch._C._cuda_getCurrentRawStream


def _wide_code(dtype):
    code = _WIDE_CODES.get(dtype)
    if code is None:
        raise _lib.HeronB200Error(_lib.HB_ERR_DTYPE, "dtype %s" % dtype)
    return code


def _is(t, name, shape, dtype):
    if t.shape != shape:
        raise ValueError("%s has shape %s, the operator takes %s" % (name, tuple(t.shape), tuple(shape)))
    if t.dtype != dtype:
        raise _lib.HeronB200Error(_lib.HB_ERR_DTYPE, "%s has dtype %s, the operator takes %s" % (name, t.dtype, dtype))


def _dims(t, name, n):
    if t.dim() != n:
        raise ValueError("%s has %d dimensions, the operator takes %d" % (name, t.dim(), n))
    return t.shape


def _ptrs(*tensors):
    """(addresses, stream) of an operator's tensors: dense, on one CUDA device, and that one current."""
    dev = tensors[0].get_device()
    ptrs = []
    for t in tensors:
        if t.get_device() != dev or dev < 0:
            if not t.is_cuda:
                raise ValueError("a tensor of shape %s must be a CUDA tensor: the kernels have no CPU path"
                                 % (tuple(t.shape),))
            raise ValueError("operands live on different devices: %s and %s" % (tensors[0].device, t.device))
        if not t.is_contiguous():
            raise ValueError("a tensor of shape %s must be contiguous" % (tuple(t.shape),))
        ptrs.append(t.data_ptr())
    if dev != torch.cuda.current_device():
        _same_device(*tensors)
    return ptrs, _raw_stream(dev)


def _fits(sizes):
    """The library's sizes are ints; a larger one would arrive cut to 32 bits."""
    if max(sizes) > 0x7fffffff:
        raise _lib.HeronB200Error(_lib.HB_ERR_SHAPE, "sizes %s" % (sizes,))


def _no_graph(kind, *tensors):
    """The products are called outside autograd: an output without a graph would end training in silence."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("%s builds no autograd graph, and one of its tensors requires a gradient: call it under "
                         "torch.no_grad() or in an autograd.Function (with its gradient operators), or detach"
                         % kind.replace("hb_", "", 1))


def _groups(offsets, groups=None):
    n = offsets.numel() - 1
    if offsets.dim() != 1 or n < 1 or (groups is not None and n != groups):
        raise ValueError("offsets holds the groups' first rows and the end of the last: %s entries, got shape %s"
                         % ("at least 2" if groups is None else groups + 1, tuple(offsets.shape)))
    if offsets.dtype != torch.int32:
        raise _lib.HeronB200Error(_lib.HB_ERR_DTYPE, "offsets has dtype %s, the operator takes int32" % offsets.dtype)
    return n


def _result(out, shape, like, out_dtype):
    if out is None:
        _wide_code(out_dtype or torch.float32)
        return like.new_empty(shape, dtype=out_dtype or torch.float32)
    _wide_code(out.dtype)
    if out_dtype is not None and out.dtype != out_dtype:
        raise ValueError("out is %s, out_dtype is %s" % (out.dtype, out_dtype))
    if out.shape != shape:
        raise ValueError("out has shape %s, the operator writes %s" % (tuple(out.shape), tuple(shape)))
    return out


def _grouped_args(kind, first, second, offsets, out, out_dtype):
    """(tensors in ABI order, sizes T, K, N, E and types) of one of the three grouped products."""
    _no_graph(kind, first, second, out)
    if kind == "hb_grouped_gemm_dw":
        T, N = _dims(first, "dy", 2)
        T2, K = _dims(second, "x", 2)
        if T != T2:
            raise ValueError("dy is (T,N), x is (T,K): T differs")
        E = _groups(offsets)
        shape = (E, N, K)
    else:
        T, R = _dims(first, "x" if kind == "hb_grouped_gemm" else "dy", 2)
        E, N, K = _dims(second, "w", 3)
        if R != (K if kind == "hb_grouped_gemm" else N):
            raise ValueError("w is (E,N,K): its reduction axis differs from the rows' length %d" % R)
        _groups(offsets, E)
        shape = (T, N if kind == "hb_grouped_gemm" else K)
    if second.dtype != first.dtype:
        raise _lib.HeronB200Error(_lib.HB_ERR_DTYPE, "operands of %s and %s" % (first.dtype, second.dtype))
    out = _result(out, shape, first, out_dtype)
    return (first, second, out, offsets), (T, K, N, E, _wide_code(first.dtype), _WIDE_CODES[out.dtype])


def _run(kind, tensors, sizes, knobs, out):
    _fits(sizes)
    ptrs, stream = _ptrs(*tensors)
    rc = getattr(_lib.load(), kind)(*ptrs, *sizes, _knobs(knobs), stream)
    if rc:
        _lib.check(rc, kind)
    return out


def _plan(kind, tensors, sizes, knobs, out):
    _fits(sizes)
    h = ctypes.c_void_p()
    name = kind.replace("hb_", "hb_plan_", 1)
    _lib.check(getattr(_lib.load(), name)(ctypes.byref(h), *_ptrs(*tensors)[0], *sizes, _knobs(knobs)), name)
    return Plan(h, tensors, out)


def grouped_gemm(x, w, offsets, out=None, out_dtype=None, knobs=None):
    """out[r] = w[e] @ x[r] for the rows r of each group e: x (T,K), w (E,N,K), out (T,N).

    Group e owns rows offsets[e] .. offsets[e+1]-1 (offsets: int32 on the device, E + 1 entries; it is
    read by the kernel, so a captured call may be replayed with other offsets).  float16 or bfloat16
    operands, fp32 accumulation, out float32 (default), float16 or bfloat16.  K % 8 == 0.  Rows of no
    group are left as they are in `out` (arbitrary in a fresh one).

    No autograd graph is built: under torch.enable_grad() tensors that require a gradient are refused, here and
    in the two gradients.  An autograd.Function calls this in its forward and grouped_gemm_dx and
    grouped_gemm_dw in its backward."""
    if knobs is None:
        done = _fast.grouped(0, x, w, offsets, out, out_dtype)
        if done is not None:
            return _done(done, "hb_grouped_gemm")
    tensors, sizes = _grouped_args("hb_grouped_gemm", x, w, offsets, out, out_dtype)
    return _run("hb_grouped_gemm", tensors, sizes, knobs, tensors[2])


def grouped_gemm_dx(dy, w, offsets, out=None, out_dtype=None, knobs=None):
    """Gradient of grouped_gemm's rows: out[r] = w[e]^T @ dy[r]; dy (T,N), out (T,K).  N % 8 == K % 8 == 0."""
    if knobs is None:
        done = _fast.grouped(1, dy, w, offsets, out, out_dtype)
        if done is not None:
            return _done(done, "hb_grouped_gemm_dx")
    tensors, sizes = _grouped_args("hb_grouped_gemm_dx", dy, w, offsets, out, out_dtype)
    return _run("hb_grouped_gemm_dx", tensors, sizes, knobs, tensors[2])


def grouped_gemm_dw(dy, x, offsets, out=None, out_dtype=None, knobs=None):
    """Gradient of grouped_gemm's weights: out[e] = sum of dy[r] x[r]^T over the rows of group e, zeros
    for a group without rows; dy (T,N), x (T,K), out (E,N,K).  N % 8 == K % 8 == 0."""
    if knobs is None:
        done = _fast.grouped(2, dy, x, offsets, out, out_dtype)
        if done is not None:
            return _done(done, "hb_grouped_gemm_dw")
    tensors, sizes = _grouped_args("hb_grouped_gemm_dw", dy, x, offsets, out, out_dtype)
    return _run("hb_grouped_gemm_dw", tensors, sizes, knobs, tensors[2])


def plan_grouped_gemm(x, w, offsets, out=None, out_dtype=None, knobs=None):
    tensors, sizes = _grouped_args("hb_grouped_gemm", x, w, offsets, out, out_dtype)
    return _plan("hb_grouped_gemm", tensors, sizes, knobs, tensors[2])


def plan_grouped_gemm_dx(dy, w, offsets, out=None, out_dtype=None, knobs=None):
    tensors, sizes = _grouped_args("hb_grouped_gemm_dx", dy, w, offsets, out, out_dtype)
    return _plan("hb_grouped_gemm_dx", tensors, sizes, knobs, tensors[2])


def plan_grouped_gemm_dw(dy, x, offsets, out=None, out_dtype=None, knobs=None):
    tensors, sizes = _grouped_args("hb_grouped_gemm_dw", dy, x, offsets, out, out_dtype)
    return _plan("hb_grouped_gemm_dw", tensors, sizes, knobs, tensors[2])


# ---- microscaled 4-bit floating point ----------------------------------------------------------
def mxfp4_scale_bytes(rows, K, groups=0):
    """Bytes of the scale array of a quantised (rows, K) matrix (include/heron_b200.h has the layout);
    `groups`: of one whose rows are grouped by offsets."""
    _fits((rows, K, groups))
    n = _lib.load().hb_mxfp4_scale_bytes(1, rows, K, groups)
    if n == 0 and (rows > 0 or groups > 0 or K <= 0 or K % 32):
        raise _lib.HeronB200Error(_lib.HB_ERR_SHAPE, "mxfp4_scale_bytes")
    return n


def _mx_shape(x, K, offsets, what):
    """(batch, rows, groups, shape of the scales) of a matrix or batch of matrices with K elements a row."""
    n = x.dim()
    if n != 2 and n != 3:
        raise ValueError("%s is (rows, K) or (batch, rows, K)" % what)
    groups = 0
    if offsets is not None:
        if n != 2:
            raise ValueError("rows grouped by offsets are a matrix (rows, K)")
        groups = _groups(offsets)
    rows = x.shape[-2]
    need = mxfp4_scale_bytes(rows, K, groups)
    return (1, rows, groups, (need,)) if n == 2 else (x.shape[0], rows, 0, (x.shape[0], need))


def _run_mx(kind, tensors, offsets, sizes, code):
    _fits(sizes)
    if offsets is None:
        ptrs, stream = _ptrs(*tensors)
        ptrs.append(None)
    else:
        ptrs, stream = _ptrs(*tensors, offsets)
    rc = getattr(_lib.load(), kind)(*ptrs, *sizes, code, stream)
    if rc:
        _lib.check(rc, kind)


def quantize_mxfp4(x, offsets=None, codes=None, scales=None):
    """x (rows, K) or (batch, rows, K), float32, float16 or bfloat16 -> (codes, scales), uint8.

    codes has x's shape with K / 2; scales is (mxfp4_scale_bytes(...),), for a batch (batch, ...).  With
    `offsets` the rows belong to groups, as grouped_gemm_mxfp4 takes them; rows of no group are skipped.
    K % 32 == 0."""
    done = _fast.quantize(x, offsets, codes, scales)
    if done is not None:
        return _done(done, "hb_quantize_mxfp4")
    shape = x.shape
    K = shape[-1] if shape else 0
    code = _wide_code(x.dtype)
    batch, rows, groups, scale_shape = _mx_shape(x, K, offsets, "x")
    code_shape = shape[:-1] + (K // 2,)
    if codes is None:
        codes = x.new_empty(code_shape, dtype=torch.uint8)
    else:
        _is(codes, "codes", code_shape, torch.uint8)
    if scales is None:
        scales = x.new_empty(scale_shape, dtype=torch.uint8)
    else:
        _is(scales, "scales", scale_shape, torch.uint8)
    _run_mx("hb_quantize_mxfp4", (x, codes, scales), offsets, (batch, rows, K, groups), code)
    return codes, scales


def dequantize_mxfp4(codes, scales, offsets=None, out=None, out_dtype=None):
    """The values that quantize_mxfp4's result stands for, float32 (default), bfloat16 or float16.  With `offsets`, those of
    the quantisation, rows of no group are left as they are in `out` (arbitrary in a fresh one)."""
    done = _fast.dequantize(codes, scales, offsets, out, out_dtype)
    if done is not None:
        return _done(done, "hb_dequantize_mxfp4")
    shape = codes.shape
    K = 2 * shape[-1] if shape else 0
    batch, rows, groups, scale_shape = _mx_shape(codes, K, offsets, "codes")
    _is(codes, "codes", shape, torch.uint8)
    _is(scales, "scales", scale_shape, torch.uint8)
    out = _result(out, shape[:-1] + (K,), codes, out_dtype)
    _run_mx("hb_dequantize_mxfp4", (codes, scales, out), offsets, (batch, rows, K, groups), _WIDE_CODES[out.dtype])
    return out


def _mx_args(a, a_scales, b, b_scales, offsets, out, out_dtype):
    """(tensors in ABI order, sizes and type) of a product of quantised matrices."""
    T, half = _dims(a, "a" if offsets is None else "x", 2)
    K = 2 * half
    if offsets is None:
        N, half_b = _dims(b, "b", 2)
        sizes, groups = (T, K, N), 0
    else:
        groups, N, half_b = _dims(b, "w", 3)
        _groups(offsets, groups)
        sizes = (T, K, N, groups)
    if half != half_b:
        raise ValueError("the operands' K differs: %d and %d code bytes a row" % (half, half_b))
    _is(a, "the first operand", a.shape, torch.uint8)
    _is(b, "the second operand", b.shape, torch.uint8)
    _is(a_scales, "the first operand's scales", (mxfp4_scale_bytes(T, K, groups),), torch.uint8)
    need = mxfp4_scale_bytes(N, K)
    _is(b_scales, "the second operand's scales", (groups, need) if groups else (need,), torch.uint8)
    out = _result(out, (T, N), a, out_dtype)
    tensors = (a, a_scales, b, b_scales, out)
    return tensors if offsets is None else tensors + (offsets,), sizes + (_WIDE_CODES[out.dtype],)


def _needs_offsets(offsets):
    if offsets is None:
        raise ValueError("offsets is missing (the product without groups is gemm_mxfp4)")


def gemm_mxfp4(a, a_scales, b, b_scales, out=None, out_dtype=None, knobs=None):
    """out[M,N] = sum_k a[m,k] * b[n,k] over the values that two quantised matrices stand for:
    a (M, K/2) and b (N, K/2) with the scales quantize_mxfp4 gave; out float32 (default), float16 or
    bfloat16, fp32 accumulation."""
    if knobs is None:
        done = _fast.mx(a, a_scales, b, b_scales, None, out, out_dtype)
        if done is not None:
            return _done(done, "hb_gemm_mxfp4")
    tensors, sizes = _mx_args(a, a_scales, b, b_scales, None, out, out_dtype)
    return _run("hb_gemm_mxfp4", tensors, sizes, knobs, tensors[4])


def grouped_gemm_mxfp4(x, x_scales, w, w_scales, offsets, out=None, out_dtype=None, knobs=None):
    """grouped_gemm over quantised operands: x (T, K/2) quantised with the same offsets, w (E, N, K/2)
    quantised as a batch."""
    _needs_offsets(offsets)
    if knobs is None:
        done = _fast.mx(x, x_scales, w, w_scales, offsets, out, out_dtype)
        if done is not None:
            return _done(done, "hb_grouped_gemm_mxfp4")
    tensors, sizes = _mx_args(x, x_scales, w, w_scales, offsets, out, out_dtype)
    return _run("hb_grouped_gemm_mxfp4", tensors, sizes, knobs, tensors[4])


def plan_gemm_mxfp4(a, a_scales, b, b_scales, out=None, out_dtype=None, knobs=None):
    tensors, sizes = _mx_args(a, a_scales, b, b_scales, None, out, out_dtype)
    return _plan("hb_gemm_mxfp4", tensors, sizes, knobs, tensors[4])


def plan_grouped_gemm_mxfp4(x, x_scales, w, w_scales, offsets, out=None, out_dtype=None, knobs=None):
    _needs_offsets(offsets)
    tensors, sizes = _mx_args(x, x_scales, w, w_scales, offsets, out, out_dtype)
    return _plan("hb_grouped_gemm_mxfp4", tensors, sizes, knobs, tensors[4])
