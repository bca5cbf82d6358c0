"""The grouped and 4-bit operators on a machine without a GPU: refusals come before any launch."""
import ctypes

import numpy as np
import pytest
import torch

from grouped_util import GRID, quantise, scale_index


@pytest.fixture(scope="module")
def ptrs():
    buf = np.zeros(1 << 16, dtype=np.uint8)
    base = (buf.ctypes.data + 255) & ~255
    return buf, ctypes.c_void_p(base), ctypes.c_void_p(base + 8), ctypes.c_void_p(base + 2)


def test_grouped_argument_errors(hb_lib, ptrs):
    from heron_b200 import _lib
    _, p, odd, worse = ptrs
    F16, BF16, F32, U8, S32 = _lib.HB_F16, _lib.HB_BF16, _lib.HB_F32, _lib.HB_U8, _lib.HB_S32
    for fn in (hb_lib.hb_grouped_gemm, hb_lib.hb_grouped_gemm_dx, hb_lib.hb_grouped_gemm_dw):
        def call(a=p, b=p, c=p, o=p, T=16, K=64, N=64, E=2, i=BF16, t=F32, knobs=None):
            return fn(a, b, c, o, T, K, N, E, i, t, knobs, None)
        for bad in (dict(T=-1), dict(K=0), dict(N=0), dict(E=0), dict(E=1025), dict(K=60)):
            assert call(**bad) == _lib.HB_ERR_SHAPE, bad
        for bad in (dict(i=U8), dict(i=F32), dict(t=S32), dict(t=99), dict(i=-1)):
            assert call(**bad) == _lib.HB_ERR_DTYPE, bad
        for bad in (dict(a=None), dict(b=None), dict(c=None), dict(o=None), dict(a=odd), dict(b=odd), dict(c=odd),
                    dict(o=worse)):
            assert call(**bad) == _lib.HB_ERR_ALIGN, bad
        if fn is not hb_lib.hb_grouped_gemm:
            assert call(N=60) == _lib.HB_ERR_SHAPE
    # no rows: nothing is looked at, and without a device only the weight gradient has something to do
    assert hb_lib.hb_grouped_gemm(None, p, None, p, 0, 64, 64, 2, F16, F32, None, None) == _lib.HB_OK
    assert hb_lib.hb_grouped_gemm_dw(None, None, None, p, 0, 64, 64, 2, F16, F32, None, None) == _lib.HB_ERR_ALIGN


@pytest.mark.parametrize("bad", [dict(tile_n=-128), dict(tile_n=(1 << 25) - 128), dict(tile_n=96), dict(tile_n=320),
                                 dict(cta_group=3), dict(cta_group=-1), dict(split_k=-1), dict(split_k=9), dict(stages=-1),
                                 dict(stages=13), dict(acc_stages=3), dict(max_ctas=-1)])
def test_knobs_out_of_range(hb_lib, ptrs, bad):
    from heron_b200 import _lib
    _, p, _, _ = ptrs
    k = ctypes.byref(_lib.HbKnobs.from_dict(bad))
    for fn in (hb_lib.hb_grouped_gemm, hb_lib.hb_grouped_gemm_dx, hb_lib.hb_grouped_gemm_dw):
        assert fn(p, p, p, p, 16, 64, 64, 2, _lib.HB_F16, _lib.HB_F32, k, None) == _lib.HB_ERR_KNOB
    assert hb_lib.hb_gemm_mxfp4(p, p, p, p, p, 4, 64, 8, _lib.HB_F32, k, None) == _lib.HB_ERR_KNOB


@pytest.mark.parametrize("n", [2 ** 30 + 32, 2 ** 31 - 32])
def test_sizes_whose_round_up_would_wrap(hb_lib, ptrs, n):
    """Sizes are rounded up to whole tiles in 32 bits: what could wrap is refused."""
    from heron_b200 import _lib
    _, p, _, _ = ptrs
    F16, F32 = _lib.HB_F16, _lib.HB_F32
    for T, K, N in ((n, 64, 64), (16, n, 64), (16, 64, n)):
        for fn in (hb_lib.hb_grouped_gemm, hb_lib.hb_grouped_gemm_dx, hb_lib.hb_grouped_gemm_dw):
            assert fn(p, p, p, p, T, K, N, 2, F16, F32, None, None) == _lib.HB_ERR_SHAPE
        assert hb_lib.hb_gemm_mxfp4(p, p, p, p, p, T, K, N, F32, None, None) == _lib.HB_ERR_SHAPE
        assert hb_lib.hb_grouped_gemm_mxfp4(p, p, p, p, p, p, T, K, N, 2, F32, None, None) == _lib.HB_ERR_SHAPE


def test_the_other_operators_keep_refusing_bfloat16(hb_lib, ptrs):
    from heron_b200 import _lib
    _, p, _, _ = ptrs
    B, F = _lib.HB_BF16, _lib.HB_F32
    assert hb_lib.hb_gemm(p, p, p, 64, 64, 64, B, B, F, None, None) == _lib.HB_ERR_DTYPE
    assert hb_lib.hb_gemm(p, p, p, 64, 64, 64, _lib.HB_F16, _lib.HB_F16, B, None, None) == _lib.HB_ERR_DTYPE
    assert hb_lib.hb_bmm(p, p, p, 2, 64, 64, 64, B, B, B, None, None) == _lib.HB_ERR_DTYPE
    assert hb_lib.hb_gemv(p, p, p, 64, 64, B, B, F, None, None) == _lib.HB_ERR_DTYPE
    assert hb_lib.hb_conv2d_nhwc(p, p, p, 1, 8, 8, 16, 16, 3, 3, 1, 1, 1, 1, 1, B, B, F, None, None) == _lib.HB_ERR_DTYPE


def test_mxfp4_argument_errors(hb_lib, ptrs):
    from heron_b200 import _lib
    _, p, odd, worse = ptrs
    F16, F32, U8 = _lib.HB_F16, _lib.HB_F32, _lib.HB_U8
    for fn in (hb_lib.hb_quantize_mxfp4, hb_lib.hb_dequantize_mxfp4):
        def call(a=p, b=p, c=p, o=None, batch=1, rows=4, K=64, groups=0, t=F16):
            return fn(a, b, c, o, batch, rows, K, groups, t, None)
        for bad in (dict(batch=0), dict(rows=-1), dict(K=0), dict(K=48), dict(groups=-1), dict(groups=1025),
                    dict(batch=2, groups=1, o=p), dict(batch=1 << 20, rows=1 << 20)):
            assert call(**bad) == _lib.HB_ERR_SHAPE, bad
        assert call(t=U8) == _lib.HB_ERR_DTYPE
        for bad in (dict(a=None), dict(b=odd), dict(c=odd), dict(groups=2), dict(o=p), dict(groups=2, o=worse)):
            assert call(**bad) == _lib.HB_ERR_ALIGN, bad
        assert call(a=None, b=None, c=None, rows=0) == _lib.HB_OK

    def gemm(a=p, s=p, b=p, bs=p, c=p, M=4, K=64, N=8, t=F32):
        return hb_lib.hb_gemm_mxfp4(a, s, b, bs, c, M, K, N, t, None, None)

    def group(a=p, s=p, b=p, bs=p, c=p, o=p, M=4, K=64, N=8, E=2, t=F32):
        return hb_lib.hb_grouped_gemm_mxfp4(a, s, b, bs, c, o, M, K, N, E, t, None, None)
    for call in (gemm, group):
        for bad in (dict(M=-1), dict(K=0), dict(K=48), dict(N=0)):
            assert call(**bad) == _lib.HB_ERR_SHAPE, bad
        assert call(t=U8) == _lib.HB_ERR_DTYPE
        for bad in (dict(a=None), dict(s=odd), dict(b=odd), dict(bs=None), dict(c=odd)):
            assert call(**bad) == _lib.HB_ERR_ALIGN, bad
        assert call(M=0) == _lib.HB_OK
    assert group(E=0) == _lib.HB_ERR_SHAPE and group(E=1025) == _lib.HB_ERR_SHAPE
    assert group(o=None) == _lib.HB_ERR_ALIGN and group(o=worse) == _lib.HB_ERR_ALIGN


def test_without_a_device_nothing_is_computed(hb_lib, ptrs):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    from heron_b200 import _lib
    _, p, _, _ = ptrs
    assert hb_lib.hb_grouped_gemm(p, p, p, p, 16, 64, 64, 2, _lib.HB_F16, _lib.HB_F32, None, None) == _lib.HB_ERR_DEVICE
    assert hb_lib.hb_quantize_mxfp4(p, p, p, None, 1, 4, 64, 0, _lib.HB_F16, None) == _lib.HB_ERR_DEVICE
    assert hb_lib.hb_gemm_mxfp4(p, p, p, p, p, 4, 64, 8, _lib.HB_F32, None, None) == _lib.HB_ERR_DEVICE
    h = ctypes.c_void_p()
    assert hb_lib.hb_plan_grouped_gemm(ctypes.byref(h), p, p, p, p, 16, 64, 64, 2, _lib.HB_F16, _lib.HB_F32,
                                       None) == _lib.HB_ERR_DEVICE and not h.value


@pytest.mark.parametrize("rows,K,off", [(1, 32, None), (129, 160, None), (300, 544, None), (5, 64, [0, 0, 3, 5]),
                                        (600, 96, [2, 130, 130, 258, 590]), (8, 32, [6, 2, 8]), (8, 64, [-3, 4, 99])])
def test_scale_layout_fits_and_no_byte_is_used_twice(hb_lib, rows, K, off):
    groups = 0 if off is None else len(off) - 1
    at = scale_index(rows, K, off)
    used = at[at >= 0]
    assert used.max() < hb_lib.hb_mxfp4_scale_bytes(1, rows, K, groups)
    if off is None or sorted(off) == off:
        assert used.unique().numel() == used.numel()


def test_group_tile_rows_never_overlap(hb_lib):
    """Group g starts at tile row offsets[g] / 128 + g: behind every group before it, and within the array."""
    rng = np.random.default_rng(0)
    for _ in range(300):
        counts = rng.integers(0, 400, rng.integers(1, 30)) * (rng.random(1) < 0.9)
        off = np.concatenate([[rng.integers(0, 200)], counts]).cumsum()
        T = int(off[-1] + rng.integers(0, 200))
        free = 0
        for g, n in enumerate(np.diff(off)):
            first = off[g] // 128 + g
            assert first >= free
            free = first + -(-n // 128)
        assert free * 512 <= hb_lib.hb_mxfp4_scale_bytes(1, T, 32, len(counts))


def test_scale_bytes(hb_lib):
    f = hb_lib.hb_mxfp4_scale_bytes
    assert f(1, 1, 32, 0) == 512 and f(1, 128, 128, 0) == 512 and f(1, 129, 160, 0) == 4 * 512
    assert f(3, 129, 160, 0) == 3 * f(1, 129, 160, 0)
    assert f(1, 0, 64, 0) == 0 and f(1, 0, 64, 2) == 2 * 512 and f(1, 128, 64, 2) == 3 * 512
    assert f(0, 4, 64, 0) == 0 and f(1, 4, 48, 0) == 0 and f(2, 4, 64, 1) == 0 and f(1, 4, 64, 1025) == 0
    assert f(1, 2 ** 31 - 1, 2 ** 31 - 32, 0) == 2 ** 24 * 2 ** 24 * 512  # sizes that pass 32 bits


def test_python_refusals(hb_lib):
    from heron_b200 import kernels as K
    from heron_b200._lib import HeronB200Error
    x, w = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(2, 8, 64, dtype=torch.float16)
    off = torch.zeros(3, dtype=torch.int32)
    for bad in [(x[0], w, off), (x, w[0], off), (x[:, :32], w, off), (x, w, off[:2]), (x, w, off.reshape(1, 3))]:
        with pytest.raises(ValueError):
            K.grouped_gemm(*bad)
    with pytest.raises(HeronB200Error):
        K.grouped_gemm(x, w, off.long())
    with pytest.raises(HeronB200Error):
        K.grouped_gemm(x, w.bfloat16(), off)
    with pytest.raises(HeronB200Error):
        K.grouped_gemm(x, w, off, out_dtype=torch.int32)
    for out in (torch.zeros(4, 9), torch.zeros(3, 8)):
        with pytest.raises(ValueError):
            K.grouped_gemm(x, w, off, out=out)
    with pytest.raises(ValueError):
        K.grouped_gemm(x, w, off, out=torch.zeros(4, 8), out_dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        K.grouped_gemm(x, w, off)
    with pytest.raises(ValueError):
        K.grouped_gemm_dw(x, x[:3], off)
    with pytest.raises(ValueError):
        K.grouped_gemm_dx(x, w, off)  # rows of 64, w has N = 8
    for bad in (torch.zeros(64), torch.zeros(1, 1, 1, 64)):
        with pytest.raises(ValueError):
            K.quantize_mxfp4(bad)
    with pytest.raises(HeronB200Error):
        K.quantize_mxfp4(torch.zeros(2, 48))
    with pytest.raises(HeronB200Error):
        K.quantize_mxfp4(torch.zeros(2, 64, dtype=torch.float64))
    with pytest.raises(ValueError):
        K.quantize_mxfp4(torch.zeros(2, 2, 64), offsets=off)
    with pytest.raises(ValueError):
        K.quantize_mxfp4(torch.zeros(2, 64), scales=torch.zeros(100, dtype=torch.uint8))
    c, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    with pytest.raises(ValueError):
        K.gemm_mxfp4(c, s, c[:, :16], s)
    with pytest.raises(ValueError):
        K.gemm_mxfp4(c, s[:256], c, s)
    with pytest.raises(HeronB200Error):
        K.gemm_mxfp4(c.float(), s, c, s)
    with pytest.raises(ValueError):
        K.grouped_gemm_mxfp4(c, s, c, s, None)
    with pytest.raises(ValueError, match="CUDA"):
        K.gemm_mxfp4(c, s, c, s)


def test_sizes_beyond_32_bits_are_refused(hb_lib):
    """Tensors without memory stand in: the refusal comes before any address is looked at."""
    from heron_b200 import kernels as K
    from heron_b200._lib import HeronB200Error
    for n in (2 ** 31, 2 ** 32 + 64):
        x = torch.empty(n, 8, dtype=torch.float16, device="meta")
        w, off = torch.empty(2, 8, 8, dtype=torch.float16, device="meta"), torch.empty(3, dtype=torch.int32, device="meta")
        with pytest.raises(HeronB200Error):
            K.grouped_gemm(x, w, off)
        with pytest.raises(HeronB200Error):
            K.quantize_mxfp4(torch.empty(n, 32, device="meta"))
        with pytest.raises(HeronB200Error):
            K.mxfp4_scale_bytes(n, 32)


def test_the_definition_of_the_format():
    """The oracle itself, on values whose codes are known."""
    x = torch.zeros(1, 32)
    x[0, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.26, -0.74, 0.3, 4.9, 5.1, -5.0, 6.0, -0.0])
    byte, code, values = quantise(x)
    assert byte.item() == 127  # largest magnitude in [4, 8): scale 1
    assert values[0, :16].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -0.5, -0.5, 0.5, 4.0, 6.0, -4.0, 6.0, 0.0]
    assert [GRID[int(c) & 7] for c in code[0, :8]] == values[0, :8].abs().tolist()


def test_tensors_that_require_a_gradient_are_refused(hb_lib):
    """No output without a graph in silence; without grad mode (an autograd.Function's forward) the call goes on to
    the next check."""
    from heron_b200 import kernels as K
    x, w = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(2, 64, 64, dtype=torch.float16)
    off, out = torch.zeros(3, dtype=torch.int32), torch.zeros(4, 64)
    xg, wg, og = (t.clone().requires_grad_() for t in (x, w, out))
    calls = [lambda x, w, out: K.grouped_gemm(x, w, off, out=out), lambda x, w, out: K.grouped_gemm_dx(x, w, off, out=out),
             lambda x, w, out: K.plan_grouped_gemm(x, w, off, out=out), lambda x, w, out: K.plan_grouped_gemm_dx(x, w, off, out=out),
             lambda x, w, out: K.grouped_gemm(x, w, off, out=out, knobs=dict(tile_n=64))]
    for call in calls:
        for bad in ((xg, w, None), (x, wg, None), (x, w, og)):
            with pytest.raises(ValueError, match="requires a gradient"):
                call(*bad)
            with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
                call(*bad)
        with pytest.raises(ValueError, match="CUDA"):
            call(xg.detach(), w, out)
    for fn in (K.grouped_gemm_dw, K.plan_grouped_gemm_dw):
        for a, b in ((xg, x), (x, xg)):
            with pytest.raises(ValueError, match="requires a gradient"):
                fn(a, b, off)


def test_a_call_without_the_front_end_takes_the_python_path(hb_lib, monkeypatch):
    """An extension that is missing, or built for another torch, costs a warning and no call."""
    import sys
    import types
    import heron_b200
    from heron_b200 import kernels as K
    x, w, off = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(2, 8, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int32)

    def never(*args):
        raise AssertionError("called")
    other = types.SimpleNamespace(built_for="another", grouped=never, quantize=never, dequantize=never, mx=never)
    for module in (None, other, types.SimpleNamespace(**dict(vars(other), built_for=None))):
        monkeypatch.setitem(sys.modules, "heron_b200._front", module)
        monkeypatch.setattr(heron_b200, "_front", module, raising=False)
        if module is None:
            monkeypatch.delattr(heron_b200, "_front")
        monkeypatch.setattr(K, "_fast", K._Front())
        with pytest.warns(RuntimeWarning, match="front end"), pytest.raises(ValueError, match="CUDA"):
            K.grouped_gemm(x, w, off)
        with pytest.raises(ValueError, match="CUDA"):
            K.quantize_mxfp4(x)


def test_the_library_builds_without_torch(hb_lib, monkeypatch, capsys):
    import os
    import subprocess
    import sys
    from heron_b200 import build
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == build.TARGET
    assert "front end not built" in capsys.readouterr().err
    # as a command, from nothing but the package's own files
    code = "import sys; sys.modules['torch'] = None; from heron_b200 import build; assert build.build() == build.TARGET"
    root = os.path.dirname(os.path.dirname(os.path.abspath(build.__file__)))
    assert subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True).returncode == 0


def test_the_front_end_follows_torch_and_the_toolkit(hb_lib, monkeypatch, tmp_path):
    import os
    from heron_b200 import build
    assert build.FRONT.endswith(build.sysconfig.get_config_var("EXT_SUFFIX"))
    assert not build.front_is_stale()
    nvcc = tmp_path / "bin" / "nvcc"
    nvcc.parent.mkdir()
    nvcc.write_text("")
    with monkeypatch.context() as m:
        m.setenv("NVCC", str(nvcc))
        assert build.cuda_include() == os.path.realpath(tmp_path / "include")
    commands = []
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "9.9.9")
        m.setattr(build, "_run", lambda cmd, target, verbose: commands.append((cmd, target)))
        assert build.front_is_stale()
        build.build_front()
    assert len(commands) == 1 and commands[0][1] == build.FRONT and any("9.9.9" in c for c in commands[0][0])


def test_scale_bytes_that_pass_64_bits(hb_lib):
    f = hb_lib.hb_mxfp4_scale_bytes
    one = f(1, 2 ** 31 - 1, 2 ** 31 - 32, 0)
    assert f(127, 2 ** 31 - 1, 2 ** 31 - 32, 0) == 127 * one
    assert f(128, 2 ** 31 - 1, 2 ** 31 - 32, 0) == 0 and f(2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 32, 0) == 0


def test_largest_conversions(hb_lib, ptrs):
    """The limits that the header gives are looked at before a device is."""
    from heron_b200 import _lib
    _, p, _, _ = ptrs
    F16 = _lib.HB_F16
    for fn in (hb_lib.hb_quantize_mxfp4, hb_lib.hb_dequantize_mxfp4):
        for batch, rows, k in ((1, 4, 65535 * 1024 + 32), (2, 2 ** 30, 32), (2 ** 27, 1, 32)):
            assert fn(p, p, p, None, batch, rows, k, 0, F16, None) == _lib.HB_ERR_SHAPE
