"""GPU: attention over 4-bit caches whose chunks follow from the lengths, at the numbers of sequences where a warp holds
one or two of them to a lane, and where it holds them no more."""
import numpy as np
import pytest

import nedo_gpu
from paged_ref import check_attention
from q4_ref import DeviceQ4, SetupQ4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [31, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("shape,shared,rows", [((4, 1, 32, 32), 3, 1), ((2, 1, 64, 32), 3, 3), ((4, 2, 32, 32), 2, 2)])
def test_many_sequences(lib, cuda, seqs, shape, shared, rows):
    """Lengths of one, of the limit and between, sequences without rows or keys, and rows behind the last sequence."""
    r, page = np.random.default_rng(seqs), shape[3]
    most = 400000 // seqs
    first = shared * page
    kv = [first + int(n) for n in r.integers(1, most, seqs)]
    q = [int(n) for n in r.integers(1, rows + 1, seqs)]
    kv[0], kv[1], kv[seqs // 2], kv[-1] = first + most, first + rows, first + 2 * rows, first + most - 1
    q[0], q[2], q[-1] = rows, 0, 1
    d = DeviceQ4(lib, cuda, SetupQ4(*shape, q=q, kv=kv, shared=shared, tail=2, seed=60))
    need = lib.paged_attention_workspace(d.cache, d.batch, shape[0])
    chunks = need % (d.s.tokens * shape[0] * (shape[2] * 4 + 8))
    assert chunks == (16 if seqs <= 64 else 0)  # their length is in the workspace
    check_attention(d.s, d.attention(), d.s.attention())
    lib.status()
    if seqs <= 64:
        # of lengths out of range only the sequences with them are left out
        d.out.fill_(777.0)
        d.len[seqs - 1] = 1 << 20
        got = d.attention()
        with pytest.raises(nedo_gpu.NedoGpuError):
            lib.status()
        d.s.kv[seqs - 1] = 0
        want = d.s.attention()
        want[2][int(d.s.start[seqs - 1]):] = False
        check_attention(d.s, got, want)
