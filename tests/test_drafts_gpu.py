"""GPU: verification of drafted tokens against its 64-bit reference (drafts_ref.py).  What comes out are
whole numbers, and they have to be equal."""
import numpy as np
import pytest

import nedo_gpu
from drafts_ref import NONE, greedy, probabilities, verify

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, rows, vocab, temperature=1.0, probs=False, seed=0, tail=0, spread=2.5, noise=0.5):
        r = self.rng = np.random.default_rng(seed)
        self.rows, self.vocab, self.temperature = list(rows), vocab, temperature
        self.starts = np.concatenate(([0], np.cumsum(rows))).astype(np.uint32)
        n = self.n = int(self.starts[-1]) + tail
        self.logits = (r.standard_normal((n, vocab)) * spread).astype(np.float32)
        guess = self.logits + noise * r.standard_normal((n, vocab)).astype(np.float32)
        self.probs = None
        if probs:
            t = temperature or 1.0
            self.probs = np.stack([probabilities(g, t) for g in guess]).astype(np.float32)
            self.drafts = np.array([int((p / np.maximum(r.exponential(size=vocab), 1e-30)).argmax()) for p in self.probs])
        else:
            self.drafts = guess.argmax(1)
        self.drafts = self.drafts.astype(np.uint32)
        self.accept_u, self.sample_u = r.random(n, np.float32), r.random(len(self.rows), np.float32)

    def want(self):
        return verify(self.logits, self.starts, self.drafts, self.temperature, self.probs, self.accept_u, self.sample_u,
                      np.full(self.n, 777, np.uint32))

    def upload(self, lib, torch):
        up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a).view(np.int32) if a.dtype == np.uint32 else a).cuda()  # noqa: E731
        self.lib, self.torch = lib, torch
        self.dev = {k: up(v) for k, v in dict(row_start=self.starts, logits=self.logits, draft_ids=self.drafts, draft_probs=self.probs,
                                              accept_u=self.accept_u, sample_u=self.sample_u).items()}
        self.desc = nedo_gpu.Drafts(seqs=len(self.rows), rows=self.n, max_rows=max(max(self.rows), 1), vocab=self.vocab,
                                    **{k: None if v is None else v.data_ptr() for k, v in self.dev.items()})
        self.accepted = torch.full((len(self.rows),), 777, dtype=torch.int32, device="cuda")
        self.ids = torch.full((self.n,), 777, dtype=torch.int32, device="cuda")
        self.need = lib.verify_drafts_workspace(self.desc)
        self.ws = torch.full((max(16, self.need),), 0xFF, dtype=torch.uint8, device="cuda")
        return self

    def call(self, stream=None):
        stream = self.torch.cuda.current_stream().cuda_stream if stream is None else stream
        self.lib.verify_drafts_dev(self.desc, self.temperature, self.accepted.data_ptr(), self.ids.data_ptr(),
                                   self.ws.data_ptr(), self.need, stream)

    def run(self, lib, torch):
        self.upload(lib, torch).call()
        return self.got()

    def got(self):
        return tuple(x.cpu().numpy().view(np.uint32) for x in (self.accepted, self.ids))

    def check(self, lib, torch):
        got, want = self.run(lib, torch), self.want()
        assert np.array_equal(got[0], want[0]), (got[0], want[0])
        assert np.array_equal(got[1], want[1]), np.flatnonzero(got[1] != want[1])
        return want


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0, 5.0])
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 257, 1000, 4095, 4096, 4097, 32003])
def test_sizes(lib, cuda, vocab, temperature, probs):
    """Odd vocabularies (rows that begin anywhere within 16 bytes), no rows, one row, many rows."""
    taken = 0
    for seed in range(3):
        c = Case([5, 1, 0, 9, 2, 3, 17], vocab, temperature, probs, seed=seed, tail=2)
        taken += c.check(lib, cuda)[0].sum()
    lib.status()
    if vocab > 2 and temperature == 0.3:
        assert 0 < taken


@pytest.mark.parametrize("rows,vocab,probs", [([5], 128000, True), ([3], 151937, False), ([5] * 40, 20000, True), ([1] * 70, 5000, False),
                                              ([256], 700, False), ([2] * 400, 300, True), ([2], 1 << 20, True)])
def test_batches(lib, cuda, rows, vocab, probs):
    Case(rows, vocab, 0.9, probs, seed=7, noise=0.3).check(lib, cuda)
    Case(rows, vocab, 0.0, probs, seed=8, noise=0.3).check(lib, cuda)
    lib.status()


def test_flat_distributions(lib, cuda):
    """Tokens of 10^-5 of the whole each: sums in 32 bits would miss the border every so often."""
    for seed in range(6):
        Case([2, 3] * 8, 100003, 1.0, True, seed=seed, spread=0.02, noise=0.01).check(lib, cuda)
        Case([1] * 16, 100003, 1.0, False, seed=seed, spread=0.02).check(lib, cuda)


@pytest.mark.parametrize("probs", [False, True])
def test_numbers_at_borders(lib, cuda, probs):
    """Random numbers of 0, of the largest below 1, and next to the border of a draft's acceptance."""
    c = Case([4] * 12, 999, 1.0, probs, seed=3)
    for i in range(48):
        p = probabilities(c.logits[i], 1.0)[c.drafts[i]]
        q = float(c.probs[i, c.drafts[i]]) if probs else 1.0
        u = np.float32(min(p / q, 1.0))
        c.accept_u[i] = [0.0, np.float32(1 - 2.0 ** -24), u, np.nextafter(u, np.float32(0)), np.nextafter(u, np.float32(1))][i % 5]
    c.accept_u = np.minimum(c.accept_u, np.float32(1 - 2.0 ** -24))
    c.sample_u[:3], c.sample_u[3:6] = 0.0, np.float32(1 - 2.0 ** -24)
    c.check(lib, cuda)
    # the border of two tokens exactly: four equal weights
    c = Case([1] * 8, 4, 1.0, seed=4)
    c.logits[:] = 0.0
    c.sample_u[:] = [0.0, 0.25, 0.5, 0.75, np.float32(1 - 2.0 ** -24), 0.249999, 0.499999, 0.9]
    assert c.check(lib, cuda)[1].tolist() == [0, 1, 2, 3, 3, 0, 1, 3]


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("probs", [False, True])
def test_masked_rows(lib, cuda, temperature, probs):
    """Logits of minus infinity, infinity and NaN, rows of nothing else, drafts that are masked."""
    c = Case([4, 4, 4, 4, 4, 3, 1, 1, 2], 5001, temperature, probs, seed=5, noise=0.1)
    c.logits[:, ::3] = -np.inf
    c.logits[1] = -np.inf
    c.logits[5, 100:] = np.nan
    c.logits[9, [7, 4000]] = np.inf
    c.logits[10, 11] = -np.float32(3.4028235e38)
    c.logits[12] = -np.float32(3.4028235e38)
    c.logits[16, 3:] = np.nan
    c.logits[16, :3] = -np.inf
    c.drafts[13], c.drafts[9] = 3, 4000
    c.logits[20] = np.nan
    c.logits[23] = -np.inf
    c.logits[23, 4444] = -1e30
    with np.errstate(invalid="ignore"):
        want = c.check(lib, cuda)
    assert (want[1] == NONE).sum() and want[1][23] == 4444 and want[1][24] != NONE
    lib.status()


def test_greedy_ties(lib, cuda):
    """The first of equal logits; -0 equals 0."""
    c = Case([3, 2, 1], 9000, 0.0, seed=6)
    c.logits[:] = np.minimum(c.logits, 0.0)
    c.logits[0, [8000, 50, 4500]] = 1.0
    c.logits[1, :] = -1.0
    c.logits[1, [77, 4100]] = [-0.0, 0.0]
    c.logits[3] = -2.0
    c.drafts[:2] = [50, 77]
    c.drafts[3] = 1
    accepted, ids = c.run(lib, cuda)
    assert accepted.tolist()[:2] == [2, 0] and ids[:2].tolist() == [50, 77] and ids[3] == 0
    assert ids[5] == greedy(c.logits[5])


def test_draft_probabilities_that_cover_the_target(lib, cuda):
    """Where p - q leaves nothing the token comes from p; probabilities that are negative, NaN or infinite."""
    c = Case([2, 2, 2, 2], 300, 1.0, True, seed=9)
    c.probs[0], c.probs[2] = 1.0, np.inf
    c.probs[4, ::2], c.probs[4, 1::2] = np.nan, -1.0
    c.probs[6, :] = 0.0
    c.accept_u[:] = 0.5
    with np.errstate(invalid="ignore"):
        want = c.check(lib, cuda)
    assert want[0].tolist()[:2] == [0, 0] and want[0][2] == want[0][3] == 1


def test_same_distributions_accept_all(lib, cuda):
    """A draft model that is the target: p / q is 1 but for its rounding."""
    c = Case([9] * 6, 4001, 1.0, True, seed=10, noise=0.0)
    c.accept_u = np.minimum(c.accept_u, 0.999)
    assert (c.check(lib, cuda)[0] == 8).all()


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("probs", [False, True])
def test_drafts_that_are_no_tokens(lib, cuda, temperature, probs):
    c = Case([4, 3], 700, temperature, probs, seed=11, noise=0.0)
    c.accept_u[:] = 0.0
    if not temperature:
        c.drafts = c.logits.argmax(1).astype(np.uint32)
    c.drafts[1], c.drafts[4] = 700, 0xFFFFFFFF
    got = c.run(lib, cuda)
    with pytest.raises(nedo_gpu.NedoGpuError) as e:
        lib.status()
    assert e.value.code == nedo_gpu.ERR_DEVICE
    assert got[0].tolist() == [1, 0]
    want = c.want()
    assert np.array_equal(got[0], want[0])
    if not probs:
        assert np.array_equal(got[1], want[1])
    lib.status()


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("what", ["order", "beyond", "too many"])
def test_rows_out_of_range(lib, cuda, temperature, what):
    """A sequence whose rows leave the batch's bounds is reported and left out."""
    c = Case([2, 3, 2], 700, temperature, seed=12, tail=1).upload(lib, cuda)
    want = c.want()
    if what == "order":
        c.dev["row_start"].copy_(cuda.tensor([0, 5, 2, 7], dtype=cuda.int32))
        c.desc.max_rows = 3
        out = [0, 1, 2]
    elif what == "beyond":
        c.dev["row_start"][3] = 900
        out = [2]
    else:
        c.desc.max_rows = 2
        out = [1]
    c.need = lib.verify_drafts_workspace(c.desc)
    c.call()
    got = c.got()
    with pytest.raises(nedo_gpu.NedoGpuError) as e:
        lib.status()
    assert e.value.code == nedo_gpu.ERR_DEVICE
    for s in range(3):
        rows = slice(int(c.starts[s]), int(c.starts[s + 1]))
        if s in out:
            assert got[0][s] == 777 and (what == "order" or (got[1][rows] == 777).all())
        else:
            assert got[0][s] == want[0][s] and np.array_equal(got[1][rows], want[1][rows])
    assert got[1][-1] == 777
    lib.status()


def test_offsets_beyond_32_bits(lib, cuda):
    """Logits of more than 2^32 elements: the last sequence's rows lie behind them."""
    vocab, rows = 1 << 20, (1 << 12) + 3
    c = Case([3], vocab, 1.0, seed=13)
    logits = cuda.zeros((rows, vocab), device="cuda")
    logits[-3:] = cuda.from_numpy(c.logits).cuda()
    starts = np.zeros(2, np.uint32)
    starts[:] = [rows - 3, rows]
    want = c.want()
    c.upload(lib, cuda)
    pad = lambda x: cuda.cat((cuda.zeros(rows - 3, dtype=x.dtype, device="cuda"), x))  # noqa: E731
    keep = [pad(c.dev["draft_ids"]), pad(c.dev["accept_u"]), cuda.from_numpy(starts.view(np.int32)).cuda()]
    c.ids = cuda.full((rows,), 777, dtype=cuda.int32, device="cuda")
    c.desc.rows, c.desc.logits, c.desc.draft_ids, c.desc.accept_u, c.desc.row_start = rows, logits.data_ptr(), keep[0].data_ptr(), keep[1].data_ptr(), keep[2].data_ptr()
    c.need = lib.verify_drafts_workspace(c.desc)
    c.ws = cuda.empty(c.need, dtype=cuda.uint8, device="cuda")
    for temperature in (1.0, 0.0):
        c.temperature = temperature
        want = c.want()
        c.call()
        assert np.array_equal(c.got()[0], want[0]) and np.array_equal(c.got()[1][-3:], want[1])
        assert (c.got()[1][:-3] == 777).all()


def test_lists_that_are_not_needed(lib, cuda):
    """One row per sequence: a token for each, no drafts; greedy: no random numbers."""
    c = Case([1] * 5, 6007, 0.8, seed=14)
    want = c.want()
    c.upload(lib, cuda)
    c.desc.draft_ids = c.desc.accept_u = None
    c.call()
    assert np.array_equal(c.got()[1], want[1])
    c = Case([3] * 5, 6007, 0.0, seed=15)
    want = c.want()
    c.upload(lib, cuda)
    c.desc.sample_u = c.desc.accept_u = None
    c.call()
    assert np.array_equal(c.got()[1], want[1])


def test_graphs_streams_and_repeats(lib, cuda):
    """Two calls on two streams at once, and a captured call replayed with other logits, give what eager ones give."""
    a, b = Case([5] * 12, 9001, 1.0, True, seed=16), Case([3] * 9, 30011, 0.7, False, seed=17)
    a.upload(lib, cuda), b.upload(lib, cuda)
    want = a.want(), b.want()
    streams = cuda.cuda.Stream(), cuda.cuda.Stream()
    cuda.cuda.synchronize()
    for _ in range(20):
        for c, s in zip((a, b), streams):
            c.call(s.cuda_stream)
    cuda.cuda.synchronize()
    for c, w in zip((a, b), want):
        assert all(np.array_equal(x, y) for x, y in zip(c.got(), w))
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        a.call()
    other = Case([5] * 12, 9001, 1.0, True, seed=18)
    for k, x in (("logits", other.logits), ("draft_probs", other.probs), ("accept_u", other.accept_u), ("sample_u", other.sample_u)):
        a.dev[k].copy_(cuda.from_numpy(x))
    a.dev["draft_ids"].copy_(cuda.from_numpy(other.drafts.view(np.int32)))
    graph.replay()
    assert all(np.array_equal(x, y) for x, y in zip(a.got(), other.want()))
    lib.status()


def test_samples_follow_the_target(lib, cuda):
    """Whatever drafts and their probabilities: the first token of 40,000 sequences is distributed as
    the target's probabilities say (chi-squared over 8 tokens, 7 degrees of freedom: 40 is passed once in 10^6)."""
    n, vocab = 40000, 8
    r = np.random.default_rng(19)
    row = (r.standard_normal(vocab)).astype(np.float32)
    c = Case([2] * n, vocab, 1.0, True, seed=20)
    c.logits[0::2] = row
    p = probabilities(row, 1.0)
    got = c.run(lib, cuda)
    first = np.bincount(got[1][0::2], minlength=vocab)
    assert ((first - n * p) ** 2 / (n * p)).sum() < 40
