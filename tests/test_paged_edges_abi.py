"""CPU: plans and refusals of the paged KV-cache entry points at the edges of what they take."""
import pytest

import nedo_gpu

A = 4096  # an aligned, never read address


def cache(**kw):
    d = dict(type=nedo_gpu.F16, kv_heads=1, head_dim=128, page_size=64, num_pages=1000, k=A, v=A, bounds=A)
    return nedo_gpu.KvCache(**{**d, **kw})


def batch(**kw):
    d = dict(seqs=2, tokens=4096, max_q_len=2048, max_kv_len=20000, max_pages=400, shared_pages=0, q_start=A, kv_len=A,
             page_table=A)
    return nedo_gpu.KvBatch(**{**d, **kw})


@pytest.mark.parametrize("type_", [0, nedo_gpu.F16])
@pytest.mark.parametrize("heads", [17, 32, 40])
def test_no_part_for_few_rows_where_every_token_has_many(lib, type_, heads):
    """Two long prompts, every row tile with all of its keys: no chunks to add, and no second part
    for sequences with few rows, because one token already has more."""
    assert lib.paged_attention_workspace(cache(type=type_), batch(), heads) == 0
