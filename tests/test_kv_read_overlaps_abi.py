"""CPU: kv_read refuses outputs that lie over the cache or the lists that it reads."""
import pytest

import nedo_gpu
from q4_ref import Q4_0
from test_paged_abi import A, batch, cache

AT, FREE = 1 << 30, 1 << 40  # aligned, never read addresses
OUT = 5 * 4 * 128 * 4  # bytes of an output of batch() over cache()
TOKEN = {nedo_gpu.F16: 256, 0: 512, Q4_0: 72}  # bytes of one KV head's 128 channels


def refused(lib, c, b, at):
    for k, v in ((at, FREE), (FREE, at)):
        with pytest.raises(nedo_gpu.NedoGpuError, match="outputs overlap what is read") as e:
            lib.kv_read_dev(c, b, k, v)
        assert e.value.code == nedo_gpu.ERR_ARG


@pytest.mark.parametrize("type_", list(TOKEN))
@pytest.mark.parametrize("which", ["k", "v"])
def test_outputs_over_the_cache_refused(lib, type_, which):
    """Up to the last bytes of the last page."""
    c = cache(type=type_, **{which: AT})
    size = 100 * 4 * 64 * TOKEN[type_]
    for at in (AT, AT + size // 2, AT + size - 16, AT - OUT + 16):
        refused(lib, c, batch(), at)


@pytest.mark.parametrize("name,size", [("q_start", 12), ("kv_len", 8), ("page_table", 80)])
def test_outputs_over_the_lists_refused(lib, name, size):
    for at in (AT - size + 4, AT, AT + OUT - 4):
        refused(lib, cache(), batch(**{name: at}), AT)
    assert A + 100 * 4 * 64 * 512 < AT
