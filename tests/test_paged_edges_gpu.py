"""GPU: the paged KV-cache operators at the edges of their types and sizes, against the 64-bit
reference (paged_ref.py)."""
import threading

import numpy as np
import pytest

import nedo_gpu
from paged_ref import F16, F32, U, Device, Setup

pytestmark = pytest.mark.gpu


class Without(Setup):
    """A Setup whose reference leaves out the keys (sequence, position) in `out` for KV head 0."""

    out = frozenset()

    def keys(self, s, kh, positions):
        if kh == 0:
            positions = np.array([p for p in positions if (s, int(p)) not in self.out], np.int64)
        return super().keys(s, kh, positions)


def place(s, seq, pos):
    return int(s.table[seq, pos // s.page]), pos % s.page


def check(got, want, tol, inside):
    """Infinities and NaN where the definition has them, the others within the tolerance."""
    got = got.cpu().numpy().astype(np.float64)
    assert (got[~inside] == 777.0).all()
    got, want, tol = got[inside], want[inside], tol[inside]
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN elsewhere"
    odd = np.isinf(want)
    assert np.array_equal(got[odd], want[odd]), "infinities elsewhere"
    fine = np.isfinite(want)
    err = np.abs(got[fine] - want[fine])
    assert (err <= tol[fine]).all(), f"worst {np.max(err / np.maximum(tol[fine], 1e-300)):.2f} x tolerance"


def every_page(s):
    """A list of all pages of every row's sequence, for block attention."""
    n = s.max_pages
    out = np.full((s.tokens, s.kv_heads, n), 0xFFFFFFFF, np.uint32)
    for t, _, p in s.rows():
        if p >= 0:
            out[t, :, :p // s.page + 1] = np.arange(p // s.page + 1)
    return out


# heads, KV heads, channels: tiles of up to 8 and of 16 rows, of 128 rows up to and above 128 channels
KINDS = [(12, 4, 128), (12, 1, 64), (11, 1, 128), (4, 2, 256), (6, 2, 40)]


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd", KINDS)
@pytest.mark.parametrize("shared", [0, 8])
def test_infinite_values(lib, cuda, type_, heads, kv_heads, hd, shared):
    """An infinite value gives its channel of every row that sees it that infinity, two of
    different signs NaN, wherever its tile lies; no other channel and no other row is touched."""
    q, kv = [1, 70, 9, 1], [3000, 700, 300, 513]
    s = Setup(type_, heads, kv_heads, hd, 32, q=q, kv=kv, shared=shared, tail=2, seed=40)
    for seq, pos, ch, x in ((0, 37, 5, np.inf), (0, 2990, 6, -np.inf), (0, 1500, 5, np.inf), (1, 300, 0, -np.inf),
                            (1, 660, 7, np.inf), (1, 650, 7, -np.inf), (1, 699, 9, np.inf), (2, 299, 3, -np.inf),
                            (3, 512, 2, np.inf), (3, 260, 33, -np.inf), (3, 400, 33, np.inf)):
        page, slot = place(s, seq, pos)
        s.v[page, 0, slot, ch] = x
    d = Device(lib, cuda, s)
    with np.errstate(invalid="ignore"):
        want = s.attention()
    assert np.isinf(want[0]).any() and np.isnan(want[0]).any()
    check(d.attention(), *want)
    d.out.fill_(777.0)
    check(d.block_attention(every_page(s)), *want)
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd", KINDS)
@pytest.mark.parametrize("shared", [0, 8])
def test_infinite_keys(lib, cuda, type_, heads, kv_heads, hd, shared):
    """A key whose score is -infinity has no weight; one whose score is +infinity makes the row
    NaN."""
    q, kv = [1, 70, 9, 1], [3000, 700, 300, 513]
    s = Without(type_, heads, kv_heads, hd, 32, q=q, kv=kv, shared=shared, tail=2, seed=41)
    s.out = frozenset([(0, 37), (0, 2990), (1, 300), (1, 660), (2, 299), (3, 260), (3, 400)])
    if shared:  # the first sequence's key lies in the prefix of all
        s.out |= {(1, 37), (2, 37), (3, 37)}
    s.queries[:, :, 1] = np.abs(s.queries[:, :, 1]) + 0.1  # their scores are -infinity in every row
    s.queries[5:9, 0, 1] *= -1.0                           # but in these: +infinity
    for seq, pos in s.out:
        page, slot = place(s, seq, pos)
        s.k[page, 0, slot, 1] = -np.inf
    d = Device(lib, cuda, s)
    want, tol, inside = s.attention()
    for t, seq, p in s.rows():
        if 5 <= t < 9 and any(x[0] == seq and x[1] <= p for x in s.out):
            want[t, 0] = np.nan
    assert np.isnan(want).any()
    check(d.attention(), want, tol, inside)
    d.out.fill_(777.0)
    check(d.block_attention(every_page(s)), want, tol, inside)
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd", KINDS)
@pytest.mark.parametrize("shared", [0, 8])
def test_infinite_values_of_no_weight(lib, cuda, type_, heads, kv_heads, hd, shared):
    """An infinite value whose weight is below the smallest number still makes its channel no number."""
    q, kv = [1, 70, 9], [3000, 700, 300]
    s = Setup(type_, heads, kv_heads, hd, 32, q=q, kv=kv, shared=shared, seed=48)
    s.queries[..., 0] = 40.0
    s.scale = 1.0
    for seq in range(3):  # the newest key and the first one: scores of 400 above all others
        for pos, x in [(p, 0.0) for p in range(kv[seq] - q[seq], kv[seq])] + [(0, 10.0)]:
            page, slot = place(s, seq, pos)
            s.k[page, :, slot, 0] = x
    for seq, pos in ((0, 2000), (1, 500), (2, 280)):
        page, slot = place(s, seq, pos)
        s.k[page, 0, slot, 0] = -10.0
        s.v[page, 0, slot, 3] = np.inf
    d = Device(lib, cuda, s)
    for got in (d.attention().cpu().numpy(), d.block_attention(every_page(s)).cpu().numpy()):
        g = heads // kv_heads
        assert not np.isfinite(got[:, :g, 3]).any()
        got[:, :g, 3] = 0
        assert np.isfinite(got).all()


@pytest.mark.parametrize("picks", [2, 5, 20])
@pytest.mark.parametrize("query,bound", [(1e-26, 1e-22), (1e-38, 1e-30), (1e-44, 1e-38), (1e-30, 1e-10)])
def test_select_tiny_scores(lib, cuda, picks, query, bound):
    """Scores that are nothing in 32 bits are still told apart in 64."""
    s = Setup(F32, 6, 2, 64, 16, q=[1, 2], kv=[700, 500], seed=42)
    s.queries = (s.queries * query).astype(np.float32)
    s.bounds = (s.bounds * np.float64(bound)).astype(np.float32)
    d = Device(lib, cuda, s)
    assert np.array_equal(d.select(picks).cpu().numpy().view(np.uint32), s.select(picks))


def test_select_from_two_host_threads(lib, cuda):
    """Calls with short and with long sequences from two threads, each on a stream of its own."""
    sets = [Setup(F16, 2, 1, 64, 16, q=[1], kv=[100], seed=43), Setup(F16, 2, 1, 64, 16, q=[1], kv=[100], seed=44)]
    sets[1].kv, sets[1].max_pages = [16384 * 16], 16384
    sets[1].table = sets[1].table[:, np.arange(16384) % 6]
    ds = [Device(lib, cuda, s) for s in sets]
    want = [s.select(4) for s in sets]
    streams = [cuda.cuda.Stream() for _ in ds]
    outs = [cuda.zeros((1, 1, 4), dtype=cuda.int32, device="cuda") for _ in ds]
    cuda.cuda.synchronize()
    errors, go = [], threading.Barrier(2)

    def work(i):
        try:
            go.wait(10)
            for _ in range(3000):
                lib.block_select_dev(ds[i].cache, ds[i].batch, 2, ds[i].q.data_ptr(), 4, outs[i].data_ptr(),
                                     streams[i].cuda_stream)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    cuda.cuda.synchronize()
    assert not errors, errors[0]
    for o, w in zip(outs, want):
        assert np.array_equal(o.cpu().numpy().view(np.uint32), w)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q", [1, 60])
def test_largest_values(lib, cuda, hd, q):
    """Weighted sums that fp32 holds do not leave it on the way."""
    s = Setup(F32, 4, 2, hd, 16, q=[q, 1], kv=[120, 90], seed=47)
    for seq in range(2):
        for pos in range(s.kv[seq]):
            page, slot = place(s, seq, pos)
            s.v[page, :, slot] = np.clip(s.v[page, :, slot], -3, 3) * np.float32(5e35)
    d = Device(lib, cuda, s)
    check(d.attention(), *s.attention())


@pytest.mark.parametrize("hd", [64, 128, 200])
@pytest.mark.parametrize("size", [1e-4, 1e-7, 1e-10, 1e-13, 1e-25])
def test_value_channels_of_different_size(lib, cuda, hd, size):
    """Channels far smaller than their neighbours keep their digits (F32 caches, tiles of many rows)."""
    s = Setup(F32, 4, 2, hd, 32, q=[70, 1, 90], kv=[500, 90, 91], shared=1, seed=45)
    s.v[..., 3] *= np.float32(size)
    s.v[..., 17::8] *= np.float32(size)
    d = Device(lib, cuda, s)
    check(d.attention(), *s.attention())
    check(d.attention(60), *s.attention(60))


@pytest.mark.parametrize("hd", [64, 128, 200])
@pytest.mark.parametrize("size", [1e4, 1e7, 1e10, 1e13, 1e25])
def test_key_channels_of_different_size(lib, cuda, hd, size):
    """A key channel far larger than its neighbours, of queries that are zero there, takes no digits
    from the others."""
    s = Setup(F32, 4, 2, hd, 32, q=[70, 1, 90], kv=[500, 90, 91], shared=1, seed=46)
    s.k[..., 5] *= np.float32(size)
    s.queries[..., 5] = 0
    d = Device(lib, cuda, s)
    check(d.attention(), *s.attention())


@pytest.mark.parametrize("hd,page", [(256, 32), (136, 64)])
@pytest.mark.parametrize("seqs,q,kv", [(74, 32, 100), (37, 32, 130), (3, 50, 700)])
def test_wide_heads_in_tiles_of_either_height(lib, cuda, hd, page, seqs, q, kv):
    """Heads above 128: batches that the plan takes in tiles of 128 rows (the first) and of 64, whole
    and cut by a window, with a padded row and an infinite value in one of them."""
    r = np.random.default_rng(seqs)
    lens = [int(kv - x) for x in r.integers(0, 30, seqs)]
    s = Setup(F16, 8, 2, hd, page, q=[q] * (seqs - 1) + [q - 3], kv=lens[:-1] + [5], tail=2, seed=49)
    page_id, slot = place(s, 1, lens[1] - 20)
    s.v[page_id, 0, slot, 9] = np.inf
    d = Device(lib, cuda, s)
    check(d.attention(), *s.attention())
    d.out.fill_(777.0)
    check(d.attention(40), *s.attention(40))
    lib.status()


@pytest.mark.parametrize("heads,kv_heads,hd", [(12, 4, 128), (12, 4, 64), (8, 2, 256), (12, 1, 128)])
def test_long_sums_are_not_cut(lib, cuda, heads, kv_heads, hd):
    """Single tokens over many keys, all values between 1 and 2.  A tile's sum may be cut by less than
    a step, 2 u of it; what comes after is rounded to nearest, whose errors even out: the mean error
    is above -2 u, however many tiles there are, and below what the weights' rounding leaves, u."""
    s = Setup(F16, heads, kv_heads, hd, 64, q=[1] * 3, kv=[20000, 19000, 15017], seed=60)
    r = np.random.default_rng(61)
    s.v = (1 + r.random(s.v.shape)).astype(np.float16)
    d = Device(lib, cuda, s)
    want = s.attention()[0]
    err = (d.attention().cpu().numpy() - want) / want
    assert -2 * U < err.mean() < U, err.mean() / U


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("what", ["order", "too many rows"])
def test_rows_of_sequences_left_out_stay_as_they_were(lib, cuda, type_, what):
    """Every row of a sequence whose lengths are out of range is left alone, by append and by every
    attention; the others' rows come out right."""
    s = Setup(type_, 6, 2, 64, 32, q=[2, 3, 2], kv=[50, 40, 30], seed=15)
    d = Device(lib, cuda, s)
    want, tol, inside = s.attention()
    if what == "order":  # 5 rows, -3 and 5, of at most 3
        d.start[1], d.start[2] = 5, 2
        inside[:] = False
    else:  # 2 rows, 4 and 1: the last row stands where it stood
        d.start[2] = 6
        inside[2:6] = False
    k = d.k.clone()
    for run in (d.attention, lambda: d.attention(7), lambda: d.block_attention(every_page(s)), lambda: d.append(1e4)):
        d.out.fill_(777.0)
        got = run()
        with pytest.raises(nedo_gpu.NedoGpuError) as e:
            lib.status(d.stream())
        assert e.value.code == nedo_gpu.ERR_DEVICE
        assert (got[cuda.from_numpy(~inside).cuda()] == 777.0).all()
        if run == d.attention:
            check(got, want, tol, inside)
    # append has written the keys of the rows left, and no others
    changed = (d.k != k).any(-1).any(1)
    changed &= ~(cuda.isnan(d.k) & cuda.isnan(k)).any(-1).any(1)
    rows = {place(s, sq, p) for t, sq, p in s.rows() if inside[t]}
    assert {tuple(x) for x in changed.nonzero().tolist()} == rows


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd", KINDS)
@pytest.mark.parametrize("nats", [12.0, 18.0, 22.0])
def test_small_weights_of_large_values(lib, cuda, type_, heads, kv_heads, hd, nats):
    """Keys of far lower score with far larger values: their small weights keep their digits."""
    q, kv = [1, 70, 9, 1], [3000, 700, 300, 513]
    s = Setup(type_, heads, kv_heads, hd, 32, q=q, kv=kv, shared=4, seed=50)
    s.scale = 1.0
    s.queries *= np.float32(0.05)
    s.queries[..., 0] = 1.0
    r = np.random.default_rng(51)
    seen = set()
    for seq in range(4):
        for pos in range(kv[seq]):
            page, slot = place(s, seq, pos)
            if (page, slot) in seen:
                continue
            seen.add((page, slot))
            far = r.random() < 0.3
            s.k[page, :, slot, 0] = -nats if far else 0.0
            s.v[page, :, slot] *= s.v.dtype.type(1e4 if far else 1e4 * np.exp(-nats))
    d = Device(lib, cuda, s)
    want = s.attention()
    check(d.attention(), *want)
    check(d.block_attention(every_page(s)), *want)


@pytest.mark.parametrize("heads,kv_heads,hd", KINDS)
@pytest.mark.parametrize("size", [1e-3, 1e-5, 1e-7])
def test_small_query_channels_of_large_key_channels(lib, cuda, heads, kv_heads, hd, size):
    """A query channel far smaller than its neighbours, which meets a key channel as much larger."""
    q, kv = [1, 70, 9], [3000, 700, 300]
    s = Setup(F16, heads, kv_heads, hd, 32, q=q, kv=kv, seed=52)
    s.queries[..., 4] *= np.float32(size)
    s.k[..., 4] *= np.float16(1e3)
    s.k[..., :4] *= np.float16(1e3 * size)
    s.k[..., 5:] *= np.float16(1e3 * size)
    s.scale = 1.0 / (1e3 * size)
    d = Device(lib, cuda, s)
    check(d.attention(), *s.attention())
