"""CPU: caches of 4-bit numbers and the verification of drafts -- what their entry points refuse before
they touch a GPU, workspaces sized without one, and the tests' own references."""
import re

import numpy as np
import pytest

import nedo_gpu
from drafts_ref import NONE, verify
from q4_ref import Q4_0, SetupQ4, pack, quantise, unpack, values
from test_paged_abi import A, batch, cache, calls


@pytest.mark.parametrize("hd", [8, 40, 72, 136, 200, 248])
def test_head_sizes_that_are_no_blocks(lib, hd):
    for call in (*calls(lib, cache(type=Q4_0, head_dim=hd), batch()),
                 lambda: lib.kv_read_dev(cache(type=Q4_0, head_dim=hd), batch(), 1 << 20, 1 << 30)):
        with pytest.raises(nedo_gpu.NedoGpuError, match="Q4_0 head_dim not block aligned") as e:
            call()
        assert e.value.code == nedo_gpu.ERR_ALIGN


@pytest.mark.parametrize("type_", [0, 1, Q4_0])
@pytest.mark.parametrize("kw,msg", [(dict(kv_heads=0), "invalid GQA"), (dict(page_size=20), "page_size"), (dict(k=None), "null pointer"),
                                    (dict(v=A + 4), "16-byte aligned")])
def test_read_refuses_bad_caches(lib, type_, kw, msg):
    with pytest.raises(nedo_gpu.NedoGpuError, match=re.escape(msg)):
        lib.kv_read_dev(cache(type=type_, **kw), batch(), 1 << 20, 1 << 30)


@pytest.mark.parametrize("k,v,msg", [(None, 1 << 30, "null pointer"), (1 << 20, None, "null pointer"), ((1 << 20) + 4, 1 << 30, "16-byte"),
                                     (1 << 20, (1 << 30) + 8, "16-byte"), (1 << 20, 1 << 20, "overlap"),
                                     (1 << 20, (1 << 20) + 5 * 4 * 128 * 4 - 16, "overlap")])
def test_read_refuses_bad_buffers(lib, k, v, msg):
    with pytest.raises(nedo_gpu.NedoGpuError, match=msg) as e:
        lib.kv_read_dev(cache(type=Q4_0), batch(), k, v)
    assert e.value.code == nedo_gpu.ERR_ARG


def test_nothing_to_do_is_no_error(lib):
    c = cache(type=Q4_0)
    for b in (batch(seqs=0), batch(tokens=0)):
        lib.kv_append_dev(c, b, 12, None, 1e4, None)
        lib.kv_read_dev(c, b, None, None)
        lib.paged_attention_dev(c, b, 12, None, None, 0.1)
    for kw in (dict(seqs=0), dict(rows=0)):
        assert lib.verify_drafts_workspace(drafts(**kw)) == 0
        lib.verify_drafts_dev(drafts(**kw), 1.0, None, None, None, 0)


def test_attention_workspaces(lib):
    """Sized without a device, and enough for every row's chunks."""
    for hd in (32, 128, 256):
        for seqs, q, kv in ((1, 1, 640), (64, 1, 32768), (2, 2048, 4096)):
            b = batch(seqs=seqs, tokens=seqs * q, max_q_len=q, max_kv_len=kv, max_pages=-(-kv // 64))
            n = lib.paged_attention_workspace(cache(type=Q4_0, head_dim=hd), b, 12)
            assert n % (seqs * q * 12 * (hd * 4 + 8)) in (0, 16)  # chunks of every row, and their length


# --------------------------------------------------------------------- drafts
def drafts(**kw):
    d = dict(seqs=2, rows=5, max_rows=4, vocab=1000, row_start=A, logits=A, draft_ids=A, draft_probs=A, accept_u=A, sample_u=A)
    return nedo_gpu.Drafts(**{**d, **kw})


@pytest.mark.parametrize("kw,msg", [(dict(seqs=1 << 24), "batch too large"), (dict(rows=1 << 31), "batch too large"),
                                    (dict(rows=(1 << 31) - 1, vocab=1 << 20), "batch too large"), (dict(vocab=0), "vocab"),
                                    (dict(vocab=1 << 31), "vocab"), (dict(max_rows=0), "max_rows"), (dict(max_rows=257), "max_rows")])
def test_bad_drafts_refused(lib, kw, msg):
    for call in (lambda d: lib.verify_drafts_workspace(d), lambda d: lib.verify_drafts_dev(d, 1.0, 1 << 20, 1 << 21, A, 1 << 40)):
        with pytest.raises(nedo_gpu.NedoGpuError, match=msg) as e:
            call(drafts(**kw))
        assert e.value.code == nedo_gpu.ERR_ARG


@pytest.mark.parametrize("kw,temperature,msg", [
    (dict(row_start=None), 1.0, "null pointer"), (dict(logits=None), 0.0, "null pointer"), (dict(draft_ids=None), 0.0, "null pointer"),
    (dict(accept_u=None), 1.0, "null pointer"), (dict(sample_u=None), 1.0, "null pointer"), (dict(sample_u=None, max_rows=1), 1.0, "null pointer"),
    (dict(logits=A + 4), 1.0, "16-byte aligned"), (dict(draft_probs=A + 8), 1.0, "16-byte aligned"), (dict(row_start=A + 2), 1.0, "4-byte aligned"),
    (dict(draft_ids=A + 1), 0.0, "4-byte aligned"), (dict(accept_u=A + 2), 1.0, "4-byte aligned"), (dict(sample_u=A + 3), 1.0, "4-byte aligned"),
    (dict(), -1.0, "temperature"), (dict(), float("nan"), "temperature"), (dict(), float("inf"), "temperature"), (dict(), 1e-7, "temperature"),
    (dict(), 1e7, "temperature"), (dict(draft_ids=1 << 21), 0.0, "overlap"), (dict(draft_ids=(1 << 21) + 16), 1.0, "overlap"),
])
def test_bad_calls_refused(lib, kw, temperature, msg):
    with pytest.raises(nedo_gpu.NedoGpuError, match=msg) as e:
        lib.verify_drafts_dev(drafts(**kw), temperature, 1 << 20, 1 << 21, A, 1 << 40)
    assert e.value.code == nedo_gpu.ERR_ARG


@pytest.mark.parametrize("name,size", [("row_start", 12), ("logits", 20000), ("draft_probs", 20000), ("accept_u", 20), ("sample_u", 8)])
def test_results_over_inputs_refused(lib, name, size):
    """What is read, up to its last element; not where the temperature leaves it unread."""
    last = (1 << 21) - size + (16 if size > 20 else 4)  # its last elements under the first of ids
    for at in (1 << 20, 1 << 21, last):
        with pytest.raises(nedo_gpu.NedoGpuError, match="the results overlap") as e:
            lib.verify_drafts_dev(drafts(**{name: at}), 1.0, 1 << 20, 1 << 21, A, 1 << 40)
        assert e.value.code == nedo_gpu.ERR_ARG
    for name in ("draft_probs", "accept_u", "sample_u"):
        with pytest.raises(nedo_gpu.NedoGpuError, match="workspace"):
            lib.verify_drafts_dev(drafts(**{name: 1 << 21}), 0.0, 1 << 20, 1 << 21, A, 0)


def test_bad_outputs_refused(lib):
    need = lib.verify_drafts_workspace(drafts())
    assert need >= 5 * 8
    for accepted, ids, ws, n, msg in ((None, 1 << 21, A, need, "null"), (1 << 20, None, A, need, "null"), (1 << 20, 1 << 21, None, need, "workspace"),
                                      (1 << 20, 1 << 21, A, need - 1, "workspace"), (1 << 20, 1 << 21, A + 8, need, "16-byte"),
                                      ((1 << 20) + 2, 1 << 21, A, need, "4-byte"), (1 << 20, (1 << 21) + 1, A, need, "4-byte")):
        with pytest.raises(nedo_gpu.NedoGpuError, match=msg):
            lib.verify_drafts_dev(drafts(), 1.0, accepted, ids, ws, n)


# ----------------------------------------------------------- the references' own
def test_pages_pack_and_unpack():
    r = np.random.default_rng(0)
    n, d = r.integers(0, 16, (3, 2, 16, 96)).astype(np.uint8), r.standard_normal((3, 2, 16, 3)).astype(np.float16)
    b = pack(n, d)
    assert b.shape == (3, 2, 16 * 3 * 18)
    got = unpack(b, 16, 96)
    assert np.array_equal(got[0], n) and np.array_equal(got[1], d)
    # a word by hand: channels 8 .. 15 of token 5
    word = int.from_bytes(b[1, 1, 5 * 48 + 4:5 * 48 + 8].tobytes(), "little")
    for j in range(8):
        assert word >> (14 + 2 * j if j % 2 else 2 * j) & 15 == n[1, 1, 5, 8 + j]
    assert np.frombuffer(b[1, 1, 16 * 48 + 2 * (2 * 16 + 5):][:2].tobytes(), np.float16)[0] == d[1, 1, 5, 2]


def test_quantiser():
    """Scales of eight bits whose values are fp16 numbers, off by at most half a step (a whole one
    at the far end of the other sign)."""
    x = np.random.default_rng(1).standard_normal((200, 96)) * np.exp2(np.random.default_rng(2).integers(-20, 12, (200, 1)))
    n, d = quantise(x)
    held = np.repeat(d, 32, -1) * (n.astype(np.float64) - 8)
    assert np.array_equal(held, values(n, d).astype(np.float64)) and np.array_equal(d, d.astype(np.float16))
    step = np.repeat(np.abs(d), 32, -1)
    assert (np.abs(x - held) <= step * 1.05).all()
    inside = np.abs(x) <= 7.4 * step
    assert (np.abs(x - held)[inside] <= 0.5 * step[inside]).all()


def test_setup_holds_what_is_packed():
    s = SetupQ4(6, 2, 64, 16, q=[1, 3], kv=[40, 17], seed=3)
    for name in "kv":
        n, d = unpack(pack(getattr(s, name + "n"), getattr(s, name + "d")), 16, 64)
        assert np.array_equal(values(n, d), getattr(s, name), equal_nan=True)


def test_verify_reference_by_hand():
    logits = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.2, 0.7], [0.3, 0.3, 0.4]])).astype(np.float32)
    starts, ids = np.array([0, 3], np.uint32), np.full(3, 9, np.uint32)
    drafts_ = np.array([0, 2, 5], np.uint32)
    run = lambda t, u, v, p=None: verify(logits, starts, drafts_, t, p, np.array(u, np.float32), np.array([v], np.float32), ids)  # noqa: E731
    assert [x.tolist() for x in run(1.0, [0.4, 0.6, 0], 0.5)] == [[2], [0, 2, 1]]
    assert [x.tolist() for x in run(1.0, [0.6, 0.6, 0], 0.51)] == [[0], [2, NONE, NONE]]
    assert [x.tolist() for x in run(1.0, [0.4, 0.8, 0], 0.2)] == [[1], [0, 0, NONE]]
    p = np.array([[0.8, 0.1, 0.1], [0.0, 0.1, 0.9], [0, 0, 1]], np.float32)
    assert [x.tolist() for x in run(1.0, [0.6, 0.7, 0], 0.7, p)] == [[2], [0, 2, 2]]
    assert [x.tolist() for x in run(1.0, [0.7, 0.7, 0], 0.4, p)] == [[0], [1, NONE, NONE]]
    assert [x.tolist() for x in run(0.0, [0, 0, 0], 0.0)] == [[2], [0, 2, 2]]
