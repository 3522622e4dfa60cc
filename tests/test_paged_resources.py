"""CPU: register budgets of the kernels over paged caches.  They are sized to
the register file (the flash kernel's 8-wave form to 256 registers): a spill
costs 10-40% with correct results, so every instantiation has to compile
without scratch."""
import concurrent.futures

import pytest

from hippo_leap_amd import build as hb
from test_kernel_resources import _resources

CHECKED = {"chunk.hip": "chunk_few_kernel", "chunk_tile.hip": "_kernel",
           "rope_chunk.hip": "rope_chunk_kernel", "pages.hip": "pages_copy_kernel"}


@pytest.fixture(scope="module")
def resources():
    try:
        hb.hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    with concurrent.futures.ThreadPoolExecutor(len(CHECKED)) as ex:
        return dict(ex.map(_resources, CHECKED))


@pytest.mark.parametrize("src", sorted(CHECKED))
def test_no_scratch(resources, src):
    seen = 0
    for name, res in resources[src].items():
        if CHECKED[src] not in name:
            continue
        seen += 1
        assert res.get("ScratchSize [bytes/lane]") == "0", (name, res)
    assert seen, f"no checked kernel found in {src}"
