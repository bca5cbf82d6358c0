"""The grouped and 4-bit operators at sizes that pass 32 bits or the usual time of a tile."""
import pytest
import torch

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
