"""GPU: verification of drafted tokens where a random number falls next to a border: rows whose sum many
small roundings lean on, and borders of two tokens known to more digits than 64-bit sums carry."""
import numpy as np
import pytest

import nedo_gpu
from drafts_ref import probabilities, verify

pytestmark = pytest.mark.gpu


def call(lib, torch, starts, logits, drafts, accept_u, sample_u, temperature=1.0, probs=None):
    """accepted and ids of the call; `logits` and `probs` on the GPU already."""
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int32) if a.dtype == np.uint32 else a).cuda()  # noqa: E731
    rows, vocab = logits.shape
    lists = [up(x) for x in (starts, drafts, accept_u, sample_u)]
    d = nedo_gpu.Drafts(seqs=len(starts) - 1, rows=rows, max_rows=int(np.diff(starts.astype(np.int64)).max()), vocab=vocab,
                        row_start=lists[0].data_ptr(), logits=logits.data_ptr(), draft_ids=lists[1].data_ptr(),
                        draft_probs=None if probs is None else probs.data_ptr(), accept_u=lists[2].data_ptr(),
                        sample_u=lists[3].data_ptr())
    accepted = torch.full((len(starts) - 1,), 777, dtype=torch.int32, device="cuda")
    ids = torch.full((rows,), 777, dtype=torch.int32, device="cuda")
    need = lib.verify_drafts_workspace(d)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    lib.verify_drafts_dev(d, temperature, accepted.data_ptr(), ids.data_ptr(), ws.data_ptr(), need,
                          torch.cuda.current_stream().cuda_stream)
    lib.status()
    return accepted.cpu().numpy(), ids.cpu().numpy().view(np.uint32)


def leaning(vocab, kind):
    """A row whose sum in 32 bits, number after number, goes astray: weights of 1 at every fourth of the first
    1024 tokens and of some 1.5 2^-23 at all others, each of which a sum of 1 takes as one or as two steps; or
    weights that grow by a part in 2^10 every 4096 tokens, so that every largest one takes over from the last."""
    if kind == "grow":
        return (np.arange(vocab) // 4096 * np.float32(2.0 ** -10)).astype(np.float32)
    row = np.full(vocab, np.log(2.0 ** -23 * (1.49 if kind == "down" else 1.51)), np.float32)
    row[:1024:4] = 0.0
    return row


@pytest.mark.parametrize("kind", ["down", "up", "grow"])
@pytest.mark.parametrize("vocab", [131072, 524288 + 1])
def test_long_sums(lib, cuda, vocab, kind):
    """600 rows, so many that no more than one CTA need take a row: the fate of a draft whose accept_u lies within
    1e-4 of the border, and no nearer than 1e-6, is that of 64 bits (whose sums are off by some 1e-13)."""
    seqs = 300
    row = leaning(vocab, kind)
    token = 0 if kind != "grow" else vocab - 1
    p = probabilities(row, 1.0)[token]
    delta = np.geomspace(1e-6, 1e-4, seqs // 2)
    u = (p * (1.0 + np.concatenate((delta, -delta)))).astype(np.float32)
    starts = (2 * np.arange(seqs + 1)).astype(np.uint32)
    accept_u = np.repeat(u, 2)
    got = call(lib, cuda, starts, cuda.from_numpy(row).cuda().expand(2 * seqs, vocab).contiguous(), np.full(2 * seqs, token, np.uint32),
               accept_u, np.full(seqs, 0.3, np.float32))
    # what follows a draft that stands, and one that does not
    want = verify(np.stack([row] * 4), np.array([0, 2, 4], np.uint32), np.full(4, token, np.uint32), 1.0, None,
                  np.array([0, 0, 0.9999, 0], np.float32), np.full(2, 0.3, np.float32), np.zeros(4, np.uint32))[1].reshape(2, 2)
    stands = u.astype(np.float64) < p
    assert stands.sum() == seqs // 2
    assert np.array_equal(got[0], stands), np.flatnonzero(got[0] != stands)
    assert np.array_equal(got[1].reshape(seqs, 2), np.where(stands[:, None], want[0], want[1]))


def near_border(n, seed):
    """Numbers u and logits -x of a token next to one of logit 0 with 1 / (1 + e^-x) = u (1 + off), off known to
    some 1e-18 and between 1e-13 and 2e-12: of 2^22 random u and their nearest x."""
    r = np.random.default_rng(seed)
    u = (r.integers(1 << 22, (1 << 24) - (1 << 18), 1 << 22) * 2.0 ** -24).astype(np.float32)
    wide = u.astype(np.longdouble)
    x = (-np.log(1 / wide - 1)).astype(np.float32)
    off = 1 / (1 + np.exp(-x.astype(np.longdouble))) / wide - 1
    assert np.finfo(np.longdouble).eps < 2e-19
    at = np.flatnonzero((np.abs(off) > 1e-13) & (np.abs(off) < 2e-12) & (np.abs(x) > 0.01))
    assert len(at) >= n and (off[at[:n]] > 0).any() and (off[at[:n]] < 0).any()
    return u[at[:n]], x[at[:n]], off[at[:n]]


def test_borders_of_two_tokens(lib, cuda):
    """The sampled token, and a draft's fate, where the random number is a part in 10^12 or 10^13 from the border of
    two tokens.  The call's exponential is off by 3e-15, its exponents (up to 4 here) by 2^-53 of themselves, and half a
    dozen 64-bit roundings follow: below 5e-15 together."""
    n = 16
    u, x, off = near_border(n, 5)
    # token 0 weighs 1 / (1 + e^-x) where its logit is x above the other's
    logits = np.zeros((n, 2), np.float32)
    logits[:, 0] = np.maximum(x, 0)
    logits[:, 1] = np.maximum(-x, 0)
    one = np.arange(n + 1, dtype=np.uint32)
    zeros = np.zeros(n, np.uint32)
    got = call(lib, cuda, one, cuda.from_numpy(logits).cuda(), zeros, np.zeros(n, np.float32), u)
    assert np.array_equal(got[1], np.where(off > 0, 0, 1))
    # a draft of token 0 stands where u is below its weight; what follows is the other one, or the second row's
    rows = np.repeat(logits, 2, 0)
    got = call(lib, cuda, 2 * one, cuda.from_numpy(rows).cuda(), np.zeros(2 * n, np.uint32), np.repeat(u, 2), np.zeros(n, np.float32))
    assert np.array_equal(got[0], off > 0)
    assert np.array_equal(got[1][0::2], np.where(off > 0, 0, 1))
    assert np.array_equal(got[1][1::2], np.where(off > 0, 0, 0xFFFFFFFF))
