"""What the paged kernels record about a call, and when it can be read."""
import pytest
import torch

from sunshape_b200 import paged
from sunshape_b200.paged import SunShapePagedCache
from tests.paged_reference import make_paged_codec

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def no_error_left():
    paged.paged_error(DEV)
    yield
    assert paged.paged_error(DEV) is None


def test_error_of_a_call_that_still_waits_on_a_side_stream():
    """``paged_error`` waits for work on streams that the default stream does not wait for."""
    codec, _ = make_paged_codec(64, 8, 2, seed=1)
    cache = SunShapePagedCache.allocate(codec, 4, 2, page_size=16)
    k = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16, device=DEV)
    bad, good = torch.tensor([[4 * 16]], device=DEV), torch.tensor([[3]], device=DEV)
    cache.append(k, k, good)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for clear in (False, True):
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)
            cache.append(k, k, bad)
        assert paged.paged_error(DEV, clear=clear) == "a slot is outside the page pool"
    with torch.cuda.stream(side):                # a clear that came late would lose this one
        cache.append(k, k, bad)
    assert "slot" in paged.paged_error(DEV)
    with torch.cuda.stream(side):
        cache.append(k, k, good)
    assert paged.paged_error(DEV) is None
