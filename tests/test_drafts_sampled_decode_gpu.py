"""GPU: decoding at a temperature with drafts that a second model samples, verified by probabilities (the call over
several rows of a sequence), step by step against the 64-bit reference on the same logits; and how the tokens behind
a draft that stands are distributed."""
import numpy as np
import pytest

from drafts_ref import NONE, probabilities, verify
from nedo_gpu import blocks as B
from q4_ref import Q4_0
from test_drafts_borders_gpu import call
from test_drafts_decode_gpu import ROOM, SEQS, VOCAB, Model

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 17, 400, 2, 9], [77], [1, 2, 3, 650, 0, 12, 13, 14, 15, 16, 88, 20, 21, 300, 301, 302, 303]]


@pytest.mark.parametrize("type_", [Q4_0, B.F16])
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("temperature,noise", [(0.7, 0.4), (0.15, 0.4), (0.03, 0.0)])
def test_sampled_drafts_step_by_step(lib, cuda, type_, certain, temperature, noise):
    """A draft model (the same one, its logits disturbed) samples up to four tokens for each sequence, or names its
    likeliest; the target's logits behind all of them decide.  accepted and ids are the reference's, and what the
    target has in its cache goes on from there."""
    r = np.random.default_rng(11)
    target, draft = Model(lib, cuda, type_, seed=4), Model(lib, cuda, Q4_0, seed=4)
    text = [list(p) for p in PROMPTS]
    held = [0] * SEQS  # tokens of the text that the draft model's cache has
    logits, start = target.logits([p[:-1] or p for p in PROMPTS], [0] * SEQS)  # all but the last token
    stood = short = 0
    for step in range(10):
        want = [int(k) for k in r.integers(0, 5, SEQS)]
        drafts, guesses = [[] for _ in text], [[] for _ in text]
        for i in range(max(want)):
            rows = [(t + d)[h:] or [(t + d)[-1]] for t, d, h in zip(text, drafts, held)]
            before = [len(t + d) - len(x) for t, d, x in zip(text, drafts, rows)]
            out, at = draft.logits(rows, before)
            held = [b + len(x) for b, x in zip(before, rows)]
            out = out[at[1:].long() - 1].cpu().numpy() + noise * r.standard_normal((SEQS, VOCAB)).astype(np.float32)
            for s in range(SEQS):
                if i < want[s]:
                    q = probabilities(out[s], temperature).astype(np.float32)
                    guesses[s].append(q)
                    drafts[s].append(int(q.argmax() if certain else r.choice(VOCAB, p=q.astype(np.float64) / q.astype(np.float64).sum())))
        rows = [[t[-1]] + d for t, d in zip(text, drafts)]
        logits, start = target.logits(rows, [len(t) - 1 for t in text])
        starts = start.cpu().numpy().view(np.uint32)
        n = int(starts[-1])
        ids = np.concatenate([np.array(d + [0], np.uint32) for d in drafts])
        probs = None if certain else np.zeros((n, VOCAB), np.float32)
        if not certain:
            for s in range(SEQS):
                for i, q in enumerate(guesses[s]):
                    probs[int(starts[s]) + i] = q
        accept_u, sample_u = r.random(n, np.float32), r.random(SEQS, np.float32)
        got = call(lib, cuda, starts, logits, ids, accept_u, sample_u, temperature, None if certain else cuda.from_numpy(probs).cuda())
        ref = verify(logits.cpu().numpy(), starts, ids, temperature, probs, accept_u, sample_u, np.zeros(n, np.uint32))
        assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])
        for s in range(SEQS):
            a = int(got[0][s])
            new = got[1][int(starts[s]):int(starts[s]) + a + 1].tolist()
            assert NONE not in new and new[:a] == drafts[s][:a]
            held[s] = min(held[s], len(text[s]) + a)  # (what it has behind that is another token's)
            text[s] += new
            stood, short = stood + a, short + (a < len(drafts[s]))
    assert max(len(t) for t in text) <= ROOM
    # both fates come up, but that no token of 700 is likely enough at 0.15 for a disturbed draft that is certain
    assert stood > 0 if noise == 0 else short > 0 and (stood > 0 or certain)


@pytest.mark.parametrize("certain", [False, True])
def test_tokens_behind_a_draft_follow_the_target(lib, cuda, certain):
    """60,000 sequences of two drafts: the first token is distributed as the target's, and among those whose
    first draft stands the second as the target's behind that draft.  Chi-squared over 6 tokens (5 degrees of freedom:
    36 is passed once in 10^6) and over 6 tokens behind each of 6 (30: 82)."""
    n, vocab = 60000, 6
    r = np.random.default_rng(21)
    first, behind = r.standard_normal(vocab).astype(np.float32), r.standard_normal((vocab, vocab)).astype(np.float32)
    guess = np.stack([probabilities(x, 1.0) for x in r.standard_normal((vocab + 1, vocab))]).astype(np.float32)
    u = r.random((n, 2))
    x0 = (u[:, :1] > guess[vocab].cumsum()[None, :-1]).sum(1)
    x1 = (u[:, 1:] > guess[x0].cumsum(1)[:, :-1]).sum(1)
    logits = np.zeros((n, 3, vocab), np.float32)
    logits[:, 0], logits[:, 1], logits[:, 2] = first, behind[x0], r.standard_normal(vocab)
    probs = np.zeros((n, 3, vocab), np.float32)
    probs[:, 0], probs[:, 1] = guess[vocab], guess[x0]
    drafts = np.stack((x0, x1, np.zeros(n, np.int64)), 1).astype(np.uint32).reshape(-1)
    got = call(lib, cuda, (3 * np.arange(n + 1)).astype(np.uint32), cuda.from_numpy(logits).cuda().reshape(-1, vocab), drafts,
               r.random(3 * n, np.float32), r.random(n, np.float32), 1.0,
               None if certain else cuda.from_numpy(probs).cuda().reshape(-1, vocab))
    ids = got[1].reshape(n, 3)
    p = probabilities(first, 1.0)
    seen = np.bincount(ids[:, 0], minlength=vocab)
    assert ((seen - n * p) ** 2 / (n * p)).sum() < 36
    total = 0.0
    for x in range(vocab):
        of_x = ids[(got[0] >= 1) & (x0 == x), 1]
        p = probabilities(behind[x], 1.0) * len(of_x)
        assert p.min() > 5
        total += ((np.bincount(of_x, minlength=vocab) - p) ** 2 / p).sum()
    assert total < 82
