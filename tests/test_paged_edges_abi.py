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


@pytest.mark.parametrize("name", ["q_start", "kv_len", "page_table", "blocks"])
@pytest.mark.parametrize("off", [1, 2])
def test_lists_out_of_alignment_are_refused(lib, name, off):
    """A list that the kernels could not read is refused on the host."""
    c, b, q, o = cache(), batch(max_kv_len=640), 1 << 20, 1 << 34
    if name != "blocks":
        b = batch(max_kv_len=640, **{name: A + off})
    at = A + off if name == "blocks" else A
    calls = [lambda: lib.block_select_dev(c, b, 4, q, 8, at), lambda: lib.block_attention_dev(c, b, 4, q, at, 8, o, 0.1, A, 1 << 40)]
    if name != "blocks":
        calls += [lambda: lib.kv_append_dev(c, b, 4, q, 1e4, o), lambda: lib.paged_attention_dev(c, b, 4, q, o, 0.1, 0, A, 1 << 40)]
    for call in calls:
        with pytest.raises(nedo_gpu.NedoGpuError, match="4-byte aligned") as e:
            call()
        assert e.value.code == nedo_gpu.ERR_ARG
