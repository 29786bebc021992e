"""GPU: the paged KV-cache operators against their 64-bit reference (paged_ref.py),
one small case for each way they can go wrong.  Everything in the pages that no
sequence owns is NaN or infinite."""
import numpy as np
import pytest

import nedo_gpu
from paged_ref import F16, F32, U, Device, Setup, check_attention

pytestmark = pytest.mark.gpu

# head groupings and sizes: (heads, kv_heads, head_dim, page_size)
SHAPES = [(12, 4, 128, 64), (12, 12, 128, 64), (8, 8, 64, 16), (8, 1, 128, 32), (5, 1, 96, 16), (16, 1, 64, 128),
          (6, 2, 8, 16), (4, 2, 40, 256), (3, 3, 200, 64), (6, 1, 256, 32), (17, 1, 72, 16), (40, 2, 16, 64)]


def dev(lib, cuda, *a, **kw):
    return Device(lib, cuda, Setup(*a, **kw))


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_single_tokens(lib, cuda, type_, shape):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300]
    d = dev(lib, cuda, type_, *shape, q=[1] * len(kv), kv=kv, seed=1)
    check_attention(d.s, d.attention(), d.s.attention())
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_ragged_prompts(lib, cuda, type_, shape):
    q, kv = [1, 37, 0, 5, 64, 1, 23], [90, 37, 12, 133, 65, 0, 24]
    d = dev(lib, cuda, type_, *shape, q=q, kv=kv, tail=3, seed=2)
    check_attention(d.s, d.attention(), d.s.attention())
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 4000])
def test_window(lib, cuda, type_, window):
    q, kv = [1, 70, 3, 1, 1], [500, 140, 66, 64, 1]
    d = dev(lib, cuda, type_, 6, 2, 64, 32, q=q, kv=kv, seed=3)
    # pages in front of every row's window are not read
    for s in range(d.s.seqs):
        first = max(0, d.s.kv[s] - d.s.q[s] + 1 - window)
        d.table[s, :first // 32] = -1
    check_attention(d.s, d.attention(window), d.s.attention(window))
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
def test_fewer_keys_than_rows(lib, cuda, type_):
    """Rows in front of position 0 are padding: zeros, whatever their queries hold."""
    d = dev(lib, cuda, type_, 12, 4, 128, 64, q=[5, 1, 4, 9], kv=[2, 0, 0, 9], seed=4)
    d.q[[0, 1, 2, 5, 6, 7, 8, 9]] = float("nan")
    out, tol, inside = d.s.attention()
    check_attention(d.s, d.attention(), (out, tol, inside))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("kv", [2049, 5000, 20011])
def test_long_sequences(lib, cuda, type_, kv):
    """Many chunks per row, alone and next to short ones."""
    d = dev(lib, cuda, type_, 6, 2, 64, 64, q=[1], kv=[kv], seed=5)
    check_attention(d.s, d.attention(), d.s.attention())
    d = dev(lib, cuda, type_, 6, 2, 64, 64, q=[1, 1, 2, 1], kv=[3, kv, 1500, 0], seed=6)
    check_attention(d.s, d.attention(), d.s.attention())
    check_attention(d.s, d.attention(1000), d.s.attention(1000))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads,kv_heads", [(6, 2), (2, 2), (16, 2)])
def test_long_prompt(lib, cuda, type_, heads, kv_heads):
    d = dev(lib, cuda, type_, heads, kv_heads, 64, 64, q=[333, 1, 130], kv=[1200, 700, 130], seed=7)
    check_attention(d.s, d.attention(), d.s.attention())
    check_attention(d.s, d.attention(257), d.s.attention(257))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd,page,shared,q,kv", [
    (12, 4, 128, 64, 3, [1] * 9, [193 + 31 * i for i in range(9)]),
    (12, 4, 128, 64, 20, [1] * 40, [1280 + 7 * i for i in range(40)]),      # a sequence that ends with the prefix
    (4, 4, 64, 16, 1, [1, 1], [17, 40]),
    (8, 1, 96, 32, 40, [3, 1, 0, 7], [1300, 1281, 1290, 1400]),
    (6, 2, 40, 16, 5, [1, 2, 1, 1, 30], [60, 3, 0, 200, 100]),              # sequences inside the prefix, a padding slot
    (6, 2, 256, 128, 9, [1] * 3, [1160, 1153, 3000]),
    (2, 2, 64, 64, 33, [1], [2500]),                                        # nobody to share with
])
def test_shared_prefix(lib, cuda, type_, heads, kv_heads, hd, page, shared, q, kv):
    d = dev(lib, cuda, type_, heads, kv_heads, hd, page, q=q, kv=kv, shared=shared, tail=2, seed=8)
    check_attention(d.s, d.attention(), d.s.attention())
    check_attention(d.s, d.attention(77), d.s.attention(77))
    lib.status()
    # the table's first row serves the prefix of all: the others' entries are not read
    d.table[1:, :shared] = -1
    check_attention(d.s, d.attention(), d.s.attention())
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
def test_large_scores(lib, cuda, type_):
    """Scores of some hundreds: the running maximum carries them; one key has all the weight."""
    d = dev(lib, cuda, type_, 6, 2, 64, 32, q=[1, 40], kv=[700, 90], seed=9)
    d.s.scale = 20.0
    check_attention(d.s, d.attention(), d.s.attention())
    d.s.scale = -20.0
    check_attention(d.s, d.attention(), d.s.attention())
    d.s.scale = 0.0  # every key the same weight
    check_attention(d.s, d.attention(), d.s.attention())


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads,kv_heads", [(6, 2), (2, 2), (48, 2)])
def test_very_negative_scores(lib, cuda, type_, heads, kv_heads):
    """Every score far below zero, in rows that see nothing of some chunks: a chunk without weight
    has no say in the row's maximum."""
    d = dev(lib, cuda, type_, heads, kv_heads, 64, 16, q=[1, 30, 1, 1], kv=[900, 2600, 33, 40], shared=64, seed=35)
    d.s.queries = -np.abs(d.s.queries) - 1
    d.q.copy_(cuda.from_numpy(d.s.queries))
    for sq in range(4):
        for i in range(-(-d.s.kv[sq] // 16)):
            d.s.k[d.s.table[sq, i]] = np.abs(d.s.k[d.s.table[sq, i]]) + 1
    d.k.copy_(cuda.from_numpy(d.s.k))
    d.s.scale = 3.0
    check_attention(d.s, d.attention(), d.s.attention())
    check_attention(d.s, d.attention(500), d.s.attention(500))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4, 1e30])
def test_query_sizes(lib, cuda, type_, size):
    """Queries far from 1 (the scale brings the scores back), and rows with one large channel."""
    d = dev(lib, cuda, type_, 6, 2, 64, 32, q=[1, 30], kv=[300, 90], seed=10)
    d.s.queries *= np.float32(size)
    d.s.queries[:, 1, 5] *= 100
    d.q.copy_(cuda.from_numpy(d.s.queries))
    d.s.scale /= size
    if size < 1e-20:
        d.s.scale = 1e29
    check_attention(d.s, d.attention(), d.s.attention())


@pytest.mark.parametrize("type_", [F16, F32])
def test_value_sizes(lib, cuda, type_):
    """Small and large values; in F16 the smallest it holds and nearly the largest."""
    for size in (6e-8, 1e-4, 6e4) if type_ == F16 else (1e-30, 6e-8, 1e30):
        d = dev(lib, cuda, type_, 6, 2, 64, 32, q=[1, 30], kv=[300, 90], seed=11)
        top = np.nanmax(np.abs(np.where(np.isfinite(d.s.v), d.s.v, 0).astype(np.float64)))
        unit = size / top if size > 1 else size
        d.s.v = (d.s.v.astype(np.float64) * unit).astype(d.s.v.dtype)
        d.v.copy_(cuda.from_numpy(d.s.v))
        check_attention(d.s, d.attention(), d.s.attention())


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads,hd,window", [(6, 64, 0), (6, 128, 0), (2, 256, 0), (6, 40, 30)])
def test_keys_and_values_of_very_different_size(lib, cuda, type_, heads, hd, window):
    """Rows that do not see a far larger key or value next to theirs keep all their digits."""
    s = Setup(type_, heads, 2, hd, 16, q=[70, 1, 90], kv=[150, 90, 91], seed=30)
    large, small = (3e3, 1e-4) if type_ == F16 else (1e25, 1e-25)
    for seq, pos, f in ((0, 146, large), (0, 100, small), (1, 88, small), (2, 30, large), (2, 31, small), (2, 88, large)):
        at = s.table[seq, pos // 16], slice(None), pos % 16
        s.v[at] = (s.v[at].astype(np.float64) * f).astype(s.v.dtype)
        s.k[at] = (s.k[at].astype(np.float64) * (f if f < 1 else 1e3)).astype(s.k.dtype)
    d = Device(lib, cuda, s)
    check_attention(s, d.attention(window), s.attention(window))
    lib.status()


@pytest.mark.parametrize("q", [1, 9, 40])
@pytest.mark.parametrize("type_", [F16, F32])
def test_windows_wider_than_any_sequence(lib, cuda, type_, q):
    d = dev(lib, cuda, type_, 6, 2, 64, 16, q=[q, q], kv=[200, 90], seed=31)
    whole = d.attention().clone()
    for window in (200, 201, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1):
        assert cuda.equal(d.attention(window), whole), window


@pytest.mark.parametrize("type_,hd,page", [(F16, 64, 16), (F16, 128, 256), (F32, 64, 32), (F16, 136, 64)])
@pytest.mark.parametrize("seqs", [33, 64, 70])
def test_many_sequences_of_many_lengths(lib, cuda, type_, hd, page, seqs):
    """Row tiles found among many sequences, in order of their keys and not."""
    r = np.random.default_rng(seqs)
    q = r.integers(0, 24, seqs)
    q[3] = 0
    kv = q + r.integers(-3, 200, seqs).clip(-q)
    d = dev(lib, cuda, type_, 6, 2, hd, page, q=[int(x) for x in q], kv=[int(x) for x in kv], tail=2, seed=34)
    for window in (0, 50):
        check_attention(d.s, d.attention(window), d.s.attention(window))
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("q", [1, 40])
def test_nothing_cached_anywhere(lib, cuda, type_, q):
    d = dev(lib, cuda, type_, 6, 2, 64, 16, q=[q, 0, 1], kv=[0, 0, 0], tail=1, seed=32)
    d.batch.max_pages, d.batch.page_table = 0, None
    check_attention(d.s, d.attention(), d.s.attention())
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite(lib, cuda, type_, bad):
    """A value that is not finite reaches the rows that see it, in its channel, and no other row."""
    q, kv = [40, 1, 1], [100, 300, 60]
    d = dev(lib, cuda, type_, 6, 2, 64, 32, q=q, kv=kv, seed=12)
    want = d.s.attention()
    for s, p in ((0, 85), (1, 120)):
        page = int(d.s.table[s, p // 32])
        d.v[page, 1, p % 32, 7] = bad
    got = d.attention().cpu().numpy()
    hit = np.zeros_like(got, bool)
    for t, s, p in d.s.rows():
        if (s == 0 and p >= 85) or s == 1:
            hit[t, 3:, 7] = True
    assert not np.isfinite(got[hit]).any()
    clean = np.where(hit, want[0], got)
    check_attention(d.s, cuda.from_numpy(clean), want)


@pytest.mark.parametrize("type_", [F16, F32])
def test_queries_that_are_not_finite(lib, cuda, type_):
    d = dev(lib, cuda, type_, 6, 2, 64, 32, q=[20, 1, 1], kv=[100, 300, 60], seed=13)
    want = d.s.attention()
    d.q[3, 2, 0] = float("nan")
    d.q[20, 4, 63] = float("nan")
    got = d.attention().cpu().numpy()
    hit = np.zeros_like(got, bool)
    hit[3, 2] = hit[20, 4] = True
    assert np.isnan(got[hit]).all()
    check_attention(d.s, cuda.from_numpy(np.where(hit, want[0], got)), want)


@pytest.mark.parametrize("type_", [F16, F32])
def test_pages_out_of_range(lib, cuda, type_):
    """A page id that is no page is reported, and counts as a page without keys."""
    d = dev(lib, cuda, type_, 6, 2, 64, 32, q=[1, 1], kv=[100, 90], seed=14)
    d.table[0, 1] = d.s.num_pages
    got = d.attention()
    with pytest.raises(nedo_gpu.NedoGpuError) as e:
        lib.status(d.stream())
    assert e.value.code == nedo_gpu.ERR_DEVICE
    blocks = np.full((2, 2, 4), 0xFFFFFFFF, np.uint32)
    blocks[0, :, :3] = [0, 2, 3]
    blocks[1, :, :3] = [0, 1, 2]
    check_attention(d.s, got, d.s.attention(blocks=blocks))
    lib.status()


@pytest.mark.parametrize("what", ["rows", "length", "order", "too many rows"])
def test_lengths_out_of_range(lib, cuda, what):
    """A sequence whose lengths leave the batch's bounds is reported and left out."""
    d = dev(lib, cuda, F16, 6, 2, 64, 32, q=[2, 3, 2], kv=[50, 40, 30], seed=15)
    out, tol, inside = d.s.attention()
    if what == "length":
        d.len[1] = 51
        inside[2:5] = False
    elif what == "rows":
        d.start[3] = 1000
        inside[5:] = False
    elif what == "order":
        d.start[1], d.start[2] = 5, 2  # sequence 1 runs backwards
        inside[:] = False
    else:
        d.start[2] = 6  # sequence 1 has four rows, sequence 2 one
        inside[2:] = False
    got = d.attention().cpu().numpy()
    with pytest.raises(nedo_gpu.NedoGpuError) as e:
        lib.status(d.stream())
    assert e.value.code == nedo_gpu.ERR_DEVICE
    if what != "order":
        keep = inside.copy()
        if what == "too many rows":
            inside[5:] = True  # sequence 2 has kept one row
            got = got[:5]
            assert (got[2:] == 777.0).all()
            return
        check_attention(d.s, cuda.from_numpy(np.where(keep[:, None, None], got, 777.0)), (out, tol, keep))
        assert (got[~keep] == 777.0).all()


def test_offsets_beyond_32_bits(lib, cuda):
    """Pages at both ends of a cache of more than 2^32 elements."""
    s = Setup(F16, 4, 2, 128, 64, q=[1, 7, 1], kv=[200, 130, 64], seed=16)
    d = Device(lib, cuda, s)
    pages = (1 << 32) // (2 * 64 * 128) + 40
    k = cuda.empty((pages, 2, 64, 128), dtype=cuda.float16, device="cuda")
    v = cuda.empty_like(k)
    spread = {int(p): (int(p) if i % 2 else pages - 1 - int(p)) for i, p in
              enumerate(np.unique(s.table[s.table != 0xFFFFFFFF]))}
    for a, b in spread.items():
        k[b], v[b] = d.k[a], d.v[a]
    table = np.vectorize(lambda p: spread.get(int(p), 0xFFFFFFFF))(s.table).astype(np.uint32)
    d.table.copy_(cuda.from_numpy(table.view(np.int32)))
    d.cache.k, d.cache.v, d.cache.num_pages, d.cache.bounds = k.data_ptr(), v.data_ptr(), pages, None
    check_attention(s, d.attention(), s.attention())
    qkv = d.append(10000.0)
    lib.status()
    q, kk, vv, real = s.append(10000.0)
    assert np.abs(qkv.cpu().numpy() - q).max() < 1e-5
    for t, sq, p in s.rows():
        got = k[int(table[sq, p // 64]), :, p % 64].cpu().numpy().astype(np.float64)
        assert (np.abs(got - kk[t]) <= 2.0 ** -11 * np.abs(kk[t]) + 1e-6).all()


# --------------------------------------------------------------------- append
@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("theta", [10000.0, 0.0])
def test_append(lib, cuda, type_, shape, theta):
    """Rotated queries, keys and values where they belong, nothing else touched, bounds exact.

    A rotated channel is x cos - y sin: three fp32 roundings, and sine and cosine are off by
    up to four steps from an angle (|angle| <= pi after the turns are taken off) rounded to
    fp32, pi 2^-24: below 16 u (|x| + |y|); then half a step of the cache's type."""
    q, kv = [1, 70, 0, 5, 1, 3, 1], [90, 137, 12, 5, 0, 2, 64]
    d = dev(lib, cuda, type_, *shape, q=q, kv=kv, tail=2, seed=17)
    s = d.s
    d.out.fill_(777.0)
    got = d.append(theta).cpu().numpy()
    lib.status()
    qq, kk, vv, real = s.append(theta)
    hd, half = s.hd, s.hd // 2
    x = np.abs(s.qkv.astype(np.float64))
    size = lambda a: np.tile(a[..., :half] + a[..., half:], 2)  # noqa: E731
    qt = 16 * U * size(x[:, :s.heads * hd].reshape(-1, s.heads, hd))
    kt = 16 * U * size(x[:, s.heads * hd:(s.heads + s.kv_heads) * hd].reshape(-1, s.kv_heads, hd))
    assert (got[~real] == 777.0).all()
    assert (np.abs(got[real] - qq[real]) <= qt[real]).all()
    want_k, want_v = s.k.copy(), s.v.copy()
    k, v = d.k.cpu().numpy(), d.v.cpu().numpy()
    step = 2.0 ** -11 if type_ == F16 else U
    small = 2.0 ** -25 if type_ == F16 else 0.0  # half the smallest step of fp16
    bounds = s.bounds.copy()
    for t, sq, p in s.rows():
        if p < 0:
            continue
        page, off = int(s.table[sq, p // s.page]), p % s.page
        kg = k[page, :, off].astype(np.float64)
        assert (np.abs(kg - kk[t]) <= kt[t] + step * (np.abs(kk[t]) + kt[t]) + small).all()
        assert np.array_equal(v[page, :, off], vv[t].astype(np.float32).astype(v.dtype))
        if off == 0:
            bounds[page, :, 0], bounds[page, :, 1] = np.inf, -np.inf
        bounds[page, :, 0] = np.minimum(bounds[page, :, 0], k[page, :, off])
        bounds[page, :, 1] = np.maximum(bounds[page, :, 1], k[page, :, off])
        want_k[page, :, off], want_v[page, :, off] = k[page, :, off], v[page, :, off]
    assert np.array_equal(k, want_k, equal_nan=True) and np.array_equal(v, want_v, equal_nan=True)
    assert np.array_equal(d.bounds.cpu().numpy(), bounds)


def test_append_far_positions(lib, cuda):
    """Angles of far positions keep their fraction of a turn (32 bits would lose it)."""
    for theta in (10000.0, 500000.0, 1.0, 1e-3):
        n = 2_000_003
        s = Setup(F32, 2, 1, 64, 16, q=[3], kv=[40], seed=18)
        d = Device(lib, cuda, s)
        pages = -(-n // 16)
        table = cuda.full((1, pages), -1, dtype=cuda.int32, device="cuda")
        table[0, -1] = 0
        d.table, d.batch.page_table, d.batch.max_pages, d.batch.max_kv_len = table, table.data_ptr(), pages, n
        d.len[0] = n
        s.kv[0] = n
        got = d.append(theta).cpu().numpy()
        lib.status()
        # theta = 1e-3 turns the last pair by 800 radians a token: the reference's own angle, p times
        # a frequency rounded to 64 bits, is off by up to p freq 2^-50
        want = s.append(float(np.float32(theta)))[0]
        x = np.abs(s.qkv.astype(np.float64))[:, :128].reshape(3, 2, 64)
        size = np.tile(x[..., :32] + x[..., 32:], 2)
        angle = n * np.maximum(1.0, float(np.float32(theta)) ** (-2.0 * np.arange(32) / 64)) * 2.0 ** -50
        worst = (np.abs(got - want) / (size * np.tile(16 * U + angle, 2))).max()
        assert worst <= 1, (theta, worst)


def test_append_nan_keys_leave_bounds(lib, cuda):
    d = dev(lib, cuda, F16, 2, 1, 16, 16, q=[4], kv=[20], seed=19)
    d.qkv[:, 2 * 16:3 * 16] = cuda.arange(4, device="cuda", dtype=cuda.float32)[:, None]
    d.qkv[1, 2 * 16 + 5] = float("nan")
    d.append(0.0)
    b = d.bounds[int(d.s.table[0, 1]), 0].cpu().numpy()
    assert (b[0] == 0).all() and (b[1] == 3).all()


def test_append_page_out_of_range(lib, cuda):
    d = dev(lib, cuda, F16, 6, 2, 64, 32, q=[1, 2], kv=[33, 40], seed=20)
    k = d.k.clone()
    d.table[0, 1] = -5
    d.append(1e4)
    with pytest.raises(nedo_gpu.NedoGpuError):
        lib.status(d.stream())
    pages = [int(p) for p in d.s.table[1, :2]]
    same = [p for p in range(d.s.num_pages) if p not in pages]
    assert cuda.equal(d.k[same].view(cuda.int16), k[same].view(cuda.int16))
    lib.status()


# -------------------------------------------------------------- page selection
@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("picks", [1, 2, 5, 40])
def test_select(lib, cuda, type_, shape, picks):
    page = shape[3]
    kv = [1, page, page + 1, 3 * page, 12 * page + 3, 0, 39 * page, 41 * page + 1]
    q = [1, 1, 1, 2, 3, 1, 1, 1]
    d = dev(lib, cuda, type_, *shape, q=q, kv=kv, tail=2, seed=21)
    got = d.select(picks).cpu().numpy().view(np.uint32)
    n = int(d.s.start[-1])
    assert np.array_equal(got[:n], d.s.select(picks)[:n])
    assert (got[n:].view(np.int32) == -7).all()
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
def test_select_ties_and_odd_scores(lib, cuda, type_):
    """Equal scores: the lower page; infinite bounds; NaN below every number; -0 equals 0."""
    d = dev(lib, cuda, type_, 4, 2, 64, 16, q=[1, 1], kv=[500, 490], seed=22)
    b = d.bounds
    ids = [int(p) for p in d.s.table[0, :31]]
    for i in range(3, 20):
        b[ids[i]] = b[ids[3]]
    b[ids[25], :, 1, 3] = float("nan")
    b[ids[26], :, 1] = 3e4
    b[ids[27], :, 0] = float("-inf")
    b[ids[28], :, :] = 0.0
    b[ids[29], :, :] = -0.0
    d.s.bounds = b.cpu().numpy()
    for picks in (1, 2, 3, 7, 12, 29, 30, 31, 32):
        assert np.array_equal(d.select(picks).cpu().numpy().view(np.uint32), d.s.select(picks)), picks
    d.q.zero_()
    d.s.queries[:] = 0
    assert np.array_equal(d.select(9).cpu().numpy().view(np.uint32), d.s.select(9))


@pytest.mark.parametrize("pages,picks", [(1500, 100), (5000, 1024), (16384, 33)])
def test_select_many_pages(lib, cuda, pages, picks):
    s = Setup(F16, 3, 1, 64, 16, q=[1, 1], kv=[pages * 16, pages * 11 + 5], seed=23)
    d = Device(lib, cuda, s)
    assert np.array_equal(d.select(picks).cpu().numpy().view(np.uint32), s.select(picks))


@pytest.mark.parametrize("type_,hd", [(F16, 256), (F32, 256), (F32, 128)])
def test_select_most_pages_of_wide_heads(lib, cuda, type_, hd):
    """The most pages that a selection takes, their numbers and the copies in flight in shared
    memory together; equal scores everywhere take the path that scores all pages in 64 bits."""
    s = Setup(type_, 2, 1, hd, 16, q=[1], kv=[90], seed=33)
    s.kv, s.max_pages = [16384 * 16], 16384
    s.table = s.table[:, np.arange(16384) % 6]  # six pages, over and over
    d = Device(lib, cuda, s)
    assert np.array_equal(d.select(40).cpu().numpy().view(np.uint32), s.select(40))


# ------------------------------------------------------ attention over picked pages
def random_blocks(s, picks, rng):
    out = np.full((s.tokens, s.kv_heads, picks), 0xFFFFFFFF, np.uint32)
    for t, sq, p in s.rows():
        for kh in range(s.kv_heads):
            if p >= 0:
                n = min(picks, p // s.page + 1)
                out[t, kh, :n] = np.sort(rng.choice(p // s.page + 1, n, replace=False))
    return out


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("picks", [1, 3, 30])
def test_block_attention(lib, cuda, type_, shape, picks):
    page = shape[3]
    kv = [1, page, page + 1, 3 * page, 12 * page + 3, 0, 29 * page, 31 * page + 1]
    q = [1, 1, 1, 2, 3, 1, 1, 1]
    d = dev(lib, cuda, type_, *shape, q=q, kv=kv, tail=2, seed=24)
    blocks = random_blocks(d.s, picks, np.random.default_rng(picks))
    check_attention(d.s, d.block_attention(blocks), d.s.attention(blocks=blocks))
    lib.status()


@pytest.mark.parametrize("type_", [F16, F32])
def test_block_lists_out_of_order(lib, cuda, type_):
    """Entries not above all before them, beyond the row's page or empty are passed over; an
    empty list gives zeros."""
    d = dev(lib, cuda, type_, 6, 2, 64, 16, q=[1, 1, 1, 1, 1], kv=[200, 200, 200, 200, 200], seed=25)
    rng = np.random.default_rng(5)
    blocks = rng.integers(0, 14, (5, 2, 70)).astype(np.uint32)
    blocks[1, :, :3] = [5, 5, 3]
    blocks[1, :, 3:] = 5
    blocks[2] = 0xFFFFFFFF
    blocks[3, 0] = 99
    blocks[3, 1, :2] = [0x80000001, 12]
    blocks[4, :, 40:] = np.arange(30)
    check_attention(d.s, d.block_attention(blocks), d.s.attention(blocks=blocks))
    lib.status()


def test_many_picks(lib, cuda):
    d = dev(lib, cuda, F16, 6, 2, 64, 16, q=[1, 2], kv=[16 * 1030, 16 * 700 + 3], seed=26)
    blocks = random_blocks(d.s, 1024, np.random.default_rng(7))
    check_attention(d.s, d.block_attention(blocks), d.s.attention(blocks=blocks))


# ---------------------------------------------------------------- used together
@pytest.mark.parametrize("type_", [F16, F32])
def test_selected_pages_are_attended(lib, cuda, type_):
    """append, select and block attention in a row: selecting every page is dense attention."""
    d = dev(lib, cuda, type_, 12, 4, 128, 64, q=[3, 1, 1], kv=[300, 900, 64], seed=27)
    s = d.s
    q = d.append(10000.0)
    d.q.copy_(q)
    s.queries = q.cpu().numpy()
    s.k, s.v, s.bounds = d.k.cpu().numpy(), d.v.cpu().numpy(), d.bounds.cpu().numpy()
    picked = d.select(16).cpu().numpy().view(np.uint32)
    assert np.array_equal(picked, s.select(16))
    dense = d.attention().clone()
    check_attention(s, dense, s.attention())
    check_attention(s, d.block_attention(picked), s.attention())
    few = d.select(4).cpu().numpy().view(np.uint32)
    check_attention(s, d.block_attention(few), s.attention(blocks=few))


def test_decode_steps_match_whole_prompt(lib, cuda):
    """Tokens appended and attended one by one give what the prompt taken in whole gives,
    within the two runs' tolerances."""
    n = 150
    s = Setup(F16, 12, 4, 128, 64, q=[n], kv=[n], seed=28)
    whole = Device(lib, cuda, s)
    whole.q.copy_(whole.append(10000.0))
    s.queries = whole.q.cpu().numpy()
    s.k, s.v = whole.k.cpu().numpy(), whole.v.cpu().numpy()
    want = s.attention()
    check_attention(s, whole.attention(), want)
    one = Device(lib, cuda, s)
    one.qkv = whole.qkv
    one.k.fill_(float("nan"))
    one.v.fill_(float("nan"))
    got = cuda.empty_like(whole.out)
    one.batch.tokens = one.batch.max_q_len = 1
    one.start[1] = 1
    row = cuda.empty((1, s.qkv.shape[1]), device="cuda")
    q1, o1 = cuda.empty((1, 12, 128), device="cuda"), cuda.empty((1, 12, 128), device="cuda")
    need = lib.paged_attention_workspace(one.cache, one.batch, 12)
    ws = one.space(need)
    for p in range(n):
        one.len[0] = p + 1
        row.copy_(whole.qkv[p:p + 1])
        lib.kv_append_dev(one.cache, one.batch, 12, row.data_ptr(), 10000.0, q1.data_ptr(), one.stream())
        lib.paged_attention_dev(one.cache, one.batch, 12, q1.data_ptr(), o1.data_ptr(), s.scale, 0, ws.data_ptr(), need,
                                one.stream())
        got[p] = o1[0]
    lib.status(one.stream())
    live = [int(p) for p in s.table[0]]
    assert cuda.equal(one.k[live[:2]], whole.k[live[:2]])
    check_attention(s, got, want)


def test_batched_layer(lib, cuda):
    """q|k|v of a batch from one matvec_dev, append, attention with a shared prefix and the output
    projection, as a serving loop runs them, on one side stream and without a host wait between,
    against the same steps in 64 bits."""
    from nedo_gpu import blocks as B

    heads, kvh, hd, dim, n = 12, 4, 128, 512, 6
    s = Setup(F16, heads, kvh, hd, 64, q=[1] * n, kv=[130 + 9 * i for i in range(n)], shared=2, seed=29)
    d = Device(lib, cuda, s)
    rows = (heads + 2 * kvh) * hd
    wqkv, wo = B.gen_weight(B.Q8_0, rows, dim, seed=1), B.gen_weight(B.Q8_0, dim, heads * hd, seed=2)
    x = np.random.default_rng(3).standard_normal((n, dim)).astype(np.float32)
    wq, wod, xd = (cuda.from_numpy(a).cuda() for a in (wqkv, wo, x))
    y = cuda.empty((n, dim), device="cuda")
    need = lib.paged_attention_workspace(d.cache, d.batch, heads)
    ws, qout = d.space(need), cuda.empty((n, heads, hd), device="cuda")
    deq = cuda.empty((rows, dim), device="cuda")
    deqo = cuda.empty((dim, heads * hd), device="cuda")
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    st = side.cuda_stream
    lib.matvec_dev(B.Q8_0, rows, dim, wq.data_ptr(), xd.data_ptr(), d.qkv.data_ptr(), n, st)
    lib.kv_append_dev(d.cache, d.batch, heads, d.qkv.data_ptr(), 10000.0, qout.data_ptr(), st)
    lib.paged_attention_dev(d.cache, d.batch, heads, qout.data_ptr(), d.out.data_ptr(), s.scale, 0, ws.data_ptr(), need, st)
    lib.matvec_dev(B.Q8_0, dim, heads * hd, wod.data_ptr(), d.out.data_ptr(), y.data_ptr(), n, st)
    lib.dequant_rows_dev(B.Q8_0, rows, dim, wq.data_ptr(), 0, rows, deq.data_ptr(), st)
    lib.dequant_rows_dev(B.Q8_0, dim, heads * hd, wod.data_ptr(), 0, dim, deqo.data_ptr(), st)
    lib.status(st)
    s.qkv = d.qkv.cpu().numpy()
    wide = x.astype(np.float64) @ deq.cpu().numpy().astype(np.float64).T
    assert (np.abs(s.qkv - wide) <= 1e-4 * (np.abs(x).astype(np.float64) @ np.abs(deq.cpu().numpy()).T)).all()
    qq, kk, vv, _ = s.append(10000.0)
    s.queries = qout.cpu().numpy()
    assert np.abs(s.queries - qq).max() <= 16 * U * 2 * np.abs(s.qkv).max()
    s.k, s.v = d.k.cpu().numpy(), d.v.cpu().numpy()
    want = s.attention()
    check_attention(s, d.out, want)
    o = d.out.cpu().numpy().reshape(n, -1).astype(np.float64)
    wo64 = deqo.cpu().numpy().astype(np.float64)
    assert (np.abs(y.cpu().numpy() - o @ wo64.T) <= 1e-4 * (np.abs(o) @ np.abs(wo64).T)).all()


def test_against_the_decode_pass(lib, cuda):
    """One sequence through append and attention reproduces the attention arithmetic of the decode
    pass: RoPE of src/kernels.cpp:93-105 and the window of src/model.cpp:218-247 in 64 bits."""
    n, window = 90, 32
    s = Setup(F32, 4, 2, 16, 16, q=[1], kv=[n], seed=30)
    d = Device(lib, cuda, s)
    rng = np.random.default_rng(31)
    rows = rng.standard_normal((n, (4 + 4) * 16)).astype(np.float32)
    d.k.zero_()
    d.v.zero_()
    keys, outs, wants = [], [], []
    need = lib.paged_attention_workspace(d.cache, d.batch, 4, window)
    ws = d.space(need)
    for p in range(n):
        d.len[0] = p + 1
        d.qkv.copy_(cuda.from_numpy(rows[p:p + 1]))
        q = cuda.empty((1, 4, 16), device="cuda")
        lib.kv_append_dev(d.cache, d.batch, 4, d.qkv.data_ptr(), 10000.0, q.data_ptr(), d.stream())
        lib.paged_attention_dev(d.cache, d.batch, 4, q.data_ptr(), d.out.data_ptr(), 0.25, window, ws.data_ptr(), need,
                                d.stream())
        outs.append(d.out.cpu().numpy()[0].astype(np.float64))
        x = rows[p].astype(np.float64).reshape(8, 16)
        a = p * 10000.0 ** (-np.arange(8) / 8.0)
        rot = np.concatenate((x[:6, :8] * np.cos(a) - x[:6, 8:] * np.sin(a), x[:6, :8] * np.sin(a) + x[:6, 8:] * np.cos(a)), 1)
        keys.append((rot[4:6], x[6:8]))
        seen = keys[max(0, p - window + 1):]
        o = np.zeros((4, 16))
        for h in range(4):
            k = np.stack([e[0][h // 2] for e in seen])
            v = np.stack([e[1][h // 2] for e in seen])
            w = np.exp(k @ rot[h] * 0.25 - (k @ rot[h] * 0.25).max())
            o[h] = w @ v / w.sum()
        wants.append(o)
    # scores of |q||k| / 4 < 40: weights off by 40 * 40 u, values below 4
    assert np.abs(np.stack(outs) - np.stack(wants)).max() < 40 * 40 * U * 4


# ------------------------------------------------------- graphs, streams, repeats
@pytest.mark.parametrize("type_", [F16, F32])
def test_results_repeat(lib, cuda, type_):
    for kw in (dict(q=[1] * 5, kv=[3000, 40, 900, 1, 2500]), dict(q=[1] * 8, kv=[1100 + i for i in range(8)], shared=17),
               dict(q=[100, 1], kv=[700, 650])):
        d = dev(lib, cuda, type_, 12, 4, 128, 64, seed=32, **kw)
        first = d.attention().clone()
        for _ in range(3):
            d.out.fill_(777.0)
            assert cuda.equal(d.attention(), first)


def test_captured_and_replayed(lib, cuda):
    """One graph of append, select and both attentions serves later lengths; a second graph over the
    same cache with a workspace of its own replays beside it."""
    s = Setup(F16, 12, 4, 128, 64, q=[1, 1, 1], kv=[3000, 70, 2000], seed=33)
    d = Device(lib, cuda, s)
    d.len.copy_(cuda.tensor([2990, 60, 0], dtype=cuda.int32))
    need = lib.paged_attention_workspace(d.cache, d.batch, 12)
    need2 = lib.block_attention_workspace(d.cache, d.batch, 12, 8)
    sides = []
    for _ in range(2):
        ws, ws2 = d.space(need), d.space(need2)
        q, o1, o2 = (cuda.zeros((3, 12, 128), device="cuda") for _ in range(3))
        picked = cuda.zeros((3, 4, 8), dtype=cuda.int32, device="cuda")
        sides.append((ws, ws2, q, o1, o2, picked))

    def step(ws, ws2, q, o1, o2, picked, st):
        lib.kv_append_dev(d.cache, d.batch, 12, d.qkv.data_ptr(), 10000.0, q.data_ptr(), st)
        lib.paged_attention_dev(d.cache, d.batch, 12, q.data_ptr(), o1.data_ptr(), s.scale, 0, ws.data_ptr(), need, st)
        lib.block_select_dev(d.cache, d.batch, 12, q.data_ptr(), 8, picked.data_ptr(), st)
        lib.block_attention_dev(d.cache, d.batch, 12, q.data_ptr(), picked.data_ptr(), 8, o2.data_ptr(), s.scale,
                                ws2.data_ptr(), need2, st)

    graphs = []
    for side in sides:
        g = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(g):
            step(*side, cuda.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for lens in ([2991, 61, 0], [3000, 1, 2000], [64, 70, 65]):
        d.len.copy_(cuda.tensor(lens, dtype=cuda.int32))
        s.kv = lens
        streams = [cuda.cuda.Stream() for _ in graphs]
        for st, g in zip(streams, graphs):
            st.wait_stream(cuda.cuda.current_stream())
            with cuda.cuda.stream(st):
                g.replay()
        cuda.cuda.synchronize()
        lib.status()
        s.k, s.v, s.bounds = d.k.cpu().numpy(), d.v.cpu().numpy(), d.bounds.cpu().numpy()
        for ws, ws2, q, o1, o2, picked in sides:
            s.queries = q.cpu().numpy()
            pick = picked.cpu().numpy().view(np.uint32)
            check_attention(s, o1, s.attention())
            assert np.array_equal(pick, s.select(8))
            check_attention(s, o2, s.attention(blocks=pick))


def test_two_streams_at_once(lib, cuda):
    ds = [dev(lib, cuda, t, 12, 4, 128, 64, q=[1] * 4, kv=[2000, 3000, 50, 900], seed=34 + t) for t in (F16, F32)]
    wants = [d.s.attention() for d in ds]
    streams = [cuda.cuda.Stream() for _ in ds]
    cuda.cuda.synchronize()
    for _ in range(5):
        for d, st in zip(ds, streams):
            with cuda.cuda.stream(st):
                d.attention()
    cuda.cuda.synchronize()
    for d, w in zip(ds, wants):
        check_attention(d.s, d.out, w)
