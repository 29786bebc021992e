"""CPU: the paged KV-cache entry points refuse what they cannot honour, before they
touch a GPU, and size their workspaces without one."""
import re

import numpy as np
import pytest

import nedo_gpu
from paged_ref import F16, F32, Setup

A = 4096  # an aligned, never read address


def cache(**kw):
    d = dict(type=F16, kv_heads=4, head_dim=128, page_size=64, num_pages=100, k=A, v=A, bounds=A)
    return nedo_gpu.KvCache(**{**d, **kw})


def batch(**kw):
    d = dict(seqs=2, tokens=5, max_q_len=4, max_kv_len=640, max_pages=10, shared_pages=0, q_start=A, kv_len=A,
             page_table=A)
    return nedo_gpu.KvBatch(**{**d, **kw})


def calls(lib, c, b, heads=12):
    """Every entry point on these descriptors."""
    return (lambda: lib.kv_append_dev(c, b, heads, 1 << 20, 1e4, 1 << 30),
            lambda: lib.paged_attention_workspace(c, b, heads),
            lambda: lib.paged_attention_dev(c, b, heads, 1 << 20, 1 << 30, 0.1, 0, A, 1 << 40),
            lambda: lib.block_select_dev(c, b, heads, 1 << 20, 8, 1 << 30),
            lambda: lib.block_attention_workspace(c, b, heads, 8),
            lambda: lib.block_attention_dev(c, b, heads, 1 << 20, A, 8, 1 << 30, 0.1, A, 1 << 40))


@pytest.mark.parametrize("kw,heads,code,msg", [
    (dict(type=8), 12, nedo_gpu.ERR_TYPE, "KV cache type not supported"),
    (dict(type=30), 12, nedo_gpu.ERR_TYPE, "KV cache type not supported"),
    (dict(kv_heads=0), 12, nedo_gpu.ERR_ARG, "invalid GQA dimensions"),
    (dict(kv_heads=5), 12, nedo_gpu.ERR_ARG, "invalid GQA dimensions"),
    (dict(), 0, nedo_gpu.ERR_ARG, "invalid GQA dimensions"),
    (dict(), 4100, nedo_gpu.ERR_ARG, "more than 4096 heads"),
    (dict(head_dim=0), 12, nedo_gpu.ERR_ARG, "head_dim"),
    (dict(head_dim=100), 12, nedo_gpu.ERR_ARG, "head_dim"),
    (dict(head_dim=264), 12, nedo_gpu.ERR_ARG, "head_dim"),
    (dict(page_size=8), 12, nedo_gpu.ERR_ARG, "page_size"),
    (dict(page_size=48), 12, nedo_gpu.ERR_ARG, "page_size"),
    (dict(page_size=512), 12, nedo_gpu.ERR_ARG, "page_size"),
    (dict(num_pages=0), 12, nedo_gpu.ERR_ARG, "num_pages"),
    (dict(num_pages=1 << 32), 12, nedo_gpu.ERR_ARG, "num_pages"),
    (dict(num_pages=1 << 29), 12, nedo_gpu.ERR_ARG, "num_pages"),
    (dict(k=None), 12, nedo_gpu.ERR_ARG, "null pointer"),
    (dict(v=None), 12, nedo_gpu.ERR_ARG, "null pointer"),
    (dict(k=A + 8), 12, nedo_gpu.ERR_ARG, "16-byte aligned"),
    (dict(v=A + 2), 12, nedo_gpu.ERR_ARG, "16-byte aligned"),
    (dict(bounds=A + 4), 12, nedo_gpu.ERR_ARG, "16-byte aligned"),
])
def test_bad_cache_refused(lib, kw, heads, code, msg):
    for call in calls(lib, cache(**kw), batch(), heads):
        with pytest.raises(nedo_gpu.NedoGpuError, match=re.escape(msg)) as e:
            call()
        assert e.value.code == code


@pytest.mark.parametrize("kw,msg", [
    (dict(max_kv_len=641), "max_kv_len exceeds"),
    (dict(max_kv_len=0xFFFFFFFF, max_pages=0xFFFFFFFF), "batch too large"),
    (dict(tokens=0x80000000), "batch too large"),
    (dict(seqs=1 << 24), "batch too large"),
    (dict(shared_pages=11), "shared_pages exceeds"),
    (dict(q_start=None), "null pointer"),
    (dict(kv_len=None), "null pointer"),
    (dict(page_table=None), "null pointer"),
    (dict(max_q_len=0), "max_q_len"),
])
def test_bad_batch_refused(lib, kw, msg):
    for call in calls(lib, cache(), batch(**kw)):
        with pytest.raises(nedo_gpu.NedoGpuError, match=re.escape(msg)) as e:
            call()
        assert e.value.code == nedo_gpu.ERR_ARG


def refused(msg, call):
    with pytest.raises(nedo_gpu.NedoGpuError, match=re.escape(msg)) as e:
        call()
    assert e.value.code == nedo_gpu.ERR_ARG


def test_bad_buffers_refused(lib):
    c, b, q, o = cache(), batch(), 1 << 20, 1 << 30
    for theta in (-1.0, float("nan"), float("inf")):
        refused("rope_theta", lambda: lib.kv_append_dev(c, b, 12, q, theta, o))
    refused("null pointer", lambda: lib.kv_append_dev(c, b, 12, None, 1e4, o))
    refused("null pointer", lambda: lib.kv_append_dev(c, b, 12, q, 1e4, None))
    refused("aligned", lambda: lib.kv_append_dev(c, b, 12, q + 4, 1e4, o))
    refused("overlap", lambda: lib.kv_append_dev(c, b, 12, q, 1e4, q + 1024))
    refused("null pointer", lambda: lib.paged_attention_dev(c, b, 12, None, o, 0.1, 0, A, 1 << 40))
    refused("null pointer", lambda: lib.paged_attention_dev(c, b, 12, q, None, 0.1, 0, A, 1 << 40))
    refused("aligned", lambda: lib.paged_attention_dev(c, b, 12, q, o + 8, 0.1, 0, A, 1 << 40))
    refused("overlap", lambda: lib.paged_attention_dev(c, b, 12, q, q, 0.1, 0, A, 1 << 40))
    for picks in (0, 1025):
        refused("picks", lambda: lib.block_select_dev(c, b, 12, q, picks, o))
        refused("picks", lambda: lib.block_attention_workspace(c, b, 12, picks))
        refused("picks", lambda: lib.block_attention_dev(c, b, 12, q, A, picks, o, 0.1, A, 1 << 40))
    refused("no key bounds", lambda: lib.block_select_dev(cache(bounds=None), b, 12, q, 8, o))
    refused("null pointer", lambda: lib.block_select_dev(c, b, 12, q, 8, None))
    refused("null pointer", lambda: lib.block_attention_dev(c, b, 12, q, None, 8, o, 0.1, A, 1 << 40))
    many = batch(max_kv_len=16385 * 64, max_pages=16385)
    refused("pages per sequence", lambda: lib.block_select_dev(c, many, 12, q, 8, o))
    large = batch(max_kv_len=65536, max_pages=1024)
    need = lib.paged_attention_workspace(c, large, 12)
    assert need > 0
    refused("workspace", lambda: lib.paged_attention_dev(c, large, 12, q, o, 0.1, 0, A, need - 1))
    refused("workspace", lambda: lib.paged_attention_dev(c, large, 12, q, o, 0.1, 0, None, need))
    refused("aligned", lambda: lib.paged_attention_dev(c, large, 12, q, o, 0.1, 0, A + 8, need))
    assert lib.lib.nedo_gpu_paged_attention_workspace(None, b, 12, 0, None) == nedo_gpu.ERR_ARG
    assert lib.lib.nedo_gpu_kv_append_dev(None, None, 12, None, 1.0, None, None) == nedo_gpu.ERR_ARG


def test_empty_batch_is_a_noop(lib):
    for kw in (dict(seqs=0), dict(tokens=0)):
        b = batch(q_start=None, kv_len=None, page_table=None, **kw)
        lib.kv_append_dev(cache(), b, 12, None, 1e4, None)
        assert lib.paged_attention_workspace(cache(), b, 12) == 0
        lib.paged_attention_dev(cache(), b, 12, None, None, 0.1)
        lib.block_select_dev(cache(), b, 12, None, 8, None)
        lib.block_attention_dev(cache(), b, 12, None, None, 8, None, 0.1)


def test_workspace_covers_what_it_must(lib):
    """Sizes are monotonic enough to plan with: a smaller bound never needs more than a
    workspace for tokens * heads rows of every chunk, and nothing is needed for a batch
    that one work item per row serves."""
    assert lib.paged_attention_workspace(cache(), batch(max_kv_len=64, max_pages=1), 12) == 0
    for kv in (640, 65536, 1 << 20):
        n = lib.paged_attention_workspace(cache(), batch(max_kv_len=kv, max_pages=kv // 64), 12)
        assert n % (12 * 5 * (128 + 2) * 4) == 0
        w = lib.paged_attention_workspace(cache(), batch(max_kv_len=kv, max_pages=kv // 64), 12, 640)
        assert w <= max(n, 64 * 12 * 5 * 130 * 4)


def test_reference_agrees_with_differences():
    """The 64-bit reference of these operators, checked against itself: attention over
    listed pages that cover everything is dense attention, and the selection of all
    pages lists them."""
    s = Setup(F32, 6, 2, 16, 16, q=[1, 3, 2], kv=[40, 3, 0], tail=1, seed=3)
    dense, _, inside = s.attention()
    every = np.full((s.tokens, 2, 4), 0xFFFFFFFF, np.uint32)
    every[:, :, :3] = np.arange(3)
    sparse, _, _ = s.attention(blocks=every)
    np.testing.assert_allclose(dense[inside], sparse[inside], rtol=0, atol=0)
    pick = s.select(4)
    for t, q, p in s.rows():
        n = p // 16 + 1 if p >= 0 else 0
        assert (pick[t, :, :n] == np.arange(n)).all() and (pick[t, :, n:] == 0xFFFFFFFF).all()
    assert not inside[-1] and (dense[[t for t, _, p in s.rows() if p < 0]] == 0).all()
