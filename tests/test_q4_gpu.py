"""GPU: the paged KV-cache operators over caches of 4-bit numbers against their 64-bit reference
(q4_ref.py, paged_ref.py).  Slots that no sequence owns have NaN and infinite scales."""
import numpy as np
import pytest

import nedo_gpu
from paged_ref import F16, F32, U, Device, Setup, check_attention
from q4_ref import Q4_0, DeviceQ4, SetupQ4, quantise, unpack, values
from test_paged_edges_gpu import check

pytestmark = pytest.mark.gpu

# head groupings and sizes: (heads, kv_heads, head_dim, page_size)
SHAPES = [(12, 4, 128, 64), (12, 12, 128, 64), (8, 8, 64, 16), (8, 1, 128, 32), (5, 1, 96, 16), (16, 1, 64, 128),
          (6, 2, 32, 16), (4, 2, 32, 256), (3, 3, 160, 64), (6, 1, 256, 32), (17, 1, 96, 16), (40, 2, 64, 64),
          (7, 1, 224, 16)]


def dev(lib, cuda, *a, **kw):
    return DeviceQ4(lib, cuda, SetupQ4(*a, **kw))


# --------------------------------------------------------------------- append
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("theta", [10000.0, 0.0])
@pytest.mark.parametrize("one", [False, True])
def test_append(lib, cuda, shape, theta, one):
    """Rotated queries, quantised keys and values where they belong, nothing else touched, bounds
    exact.  Numbers and scales are those of 64-bit arithmetic: the angles' 2^-50 would have to
    fall on a border of two steps to be seen.  Queries as over other caches: 16 u (|x| + |y|)."""
    q, kv = ([1] * 7, [90, 137, 1, 65, 0, 17, 64]) if one else ([1, 70, 0, 5, 1, 3, 1], [90, 137, 12, 5, 0, 2, 64])
    d = dev(lib, cuda, *shape, q=q, kv=kv, tail=2, seed=17)
    s, hd, half = d.s, d.s.hd, d.s.hd // 2
    got = d.append(theta).cpu().numpy()
    lib.status()
    qq, kk, vv, real = s.append(theta)
    x = np.abs(s.qkv.astype(np.float64))[:, :s.heads * hd].reshape(-1, s.heads, hd)
    assert (got[~real] == 777.0).all()
    assert (np.abs(got[real] - qq[real]) <= 16 * U * np.tile(x[..., :half] + x[..., half:], 2)[real]).all()
    kn, kd, vn, vd = (a.copy() for a in (s.kn, s.kd, s.vn, s.vd))
    bounds = s.bounds.copy()
    for t, sq, p in s.rows():
        if p < 0:
            continue
        page, off = int(s.table[sq, p // s.page]), p % s.page
        for n, sc, y in ((kn, kd, kk[t]), (vn, vd, vv[t])):
            n[page, :, off], sc[page, :, off] = quantise(y)
        held = values(kn[page, :, off], kd[page, :, off])
        if off == 0:
            bounds[page, :, 0], bounds[page, :, 1] = np.inf, -np.inf
        bounds[page, :, 0], bounds[page, :, 1] = np.minimum(bounds[page, :, 0], held), np.maximum(bounds[page, :, 1], held)
    for buf, n, sc in ((d.k, kn, kd), (d.v, vn, vd)):
        gn, gd = unpack(buf.cpu().numpy(), s.page, hd)
        assert np.array_equal(gn, n) and np.array_equal(gd, sc, equal_nan=True)
    assert np.array_equal(d.bounds.cpu().numpy(), bounds)


@pytest.mark.parametrize("q", [1, 3])
def test_append_numbers_at_borders(lib, cuda, q):
    """Ties of the rounding, both signs at the largest magnitude, blocks of zeros, of the smallest and of
    the largest numbers, of infinities and NaN, for keys (not rotated) and values."""
    kvh, hd = 1, 32
    rng = np.random.default_rng(3)
    blocks = [np.zeros(32), np.full(32, -0.0), np.arange(-8, 24) * 1.0, np.arange(-16, 16) * 0.5, np.arange(-15, 17) * 0.5,
              np.where(np.arange(32) % 2, 4.0, -4.0), np.arange(32) * 2.0 ** -24, np.arange(32) * 2.0 ** -27,
              np.arange(32) * 2.0 ** -29, np.full(32, 1e-45), np.linspace(-1e38, 1e38, 32), np.linspace(-7e4, 3e4, 32),
              np.linspace(0, 65280.0, 32), np.where(np.arange(32) == 5, np.inf, 1.0), np.where(np.arange(32) == 31, -np.inf, 1.0),
              np.where(np.arange(32) == 0, np.nan, 1.0), np.full(32, np.nan)]
    for e in (-30, -14, 0, 9):  # borders of scales and of numbers, and their neighbours
        d = (128 + rng.integers(0, 128)) * 2.0 ** (e - 7)
        x = d * (rng.integers(0, 16, 32) - 8.5)
        x[0] = -8 * d
        x[8:16] = np.nextafter(x[8:16].astype(np.float32), np.float32(np.inf))
        x[16:24] = np.nextafter(x[16:24].astype(np.float32), np.float32(-np.inf))
        blocks += [x, -x, x * 1.001, np.where(np.arange(32) == 0, -8 * (d + d / 256), x), np.where(np.arange(32) == 0, -8 * (d + 3 * d / 256), x)]
    blocks = np.array(blocks).astype(np.float32)
    n = -(-len(blocks) // q)
    blocks = np.concatenate((blocks, blocks))[:n * q]
    s = SetupQ4(1, kvh, hd, 16, [q] * n, [q] * n, seed=5)
    s.qkv[:, 32:64], s.qkv[:, 64:] = blocks, blocks[::-1]
    d = DeviceQ4(lib, cuda, s)
    d.append(0.0)
    lib.status()
    (kn, kd), (vn, vd) = (unpack(x.cpu().numpy(), 16, hd) for x in (d.k, d.v))
    bounds = d.bounds.cpu().numpy()
    for i in range(n):
        page = int(s.table[i, 0])
        for gn, gd, x in ((kn, kd, blocks[i * q:(i + 1) * q]), (vn, vd, blocks[::-1][i * q:(i + 1) * q])):
            wn, wd = quantise(x)
            ok = np.isfinite(x).all(-1)
            assert np.array_equal(gn[page, 0, :q][ok], wn[ok])
            assert np.array_equal(gd[page, 0, :q].astype(np.float64), wd, equal_nan=True)
        held = values(*quantise(blocks[i * q:(i + 1) * q])).astype(np.float64)
        seen = np.where(np.isnan(held), np.inf, held).min(0), np.where(np.isnan(held), -np.inf, held).max(0)
        assert np.array_equal(bounds[page, 0].astype(np.float64), np.stack(seen))


@pytest.mark.parametrize("q", [1, 2])
def test_append_turned_keys_at_borders(lib, cuda, q):
    """Keys whose turn leaves them where they are (position 0, and pairs of zeros), next to and on the borders of
    scales and numbers: what 32 bits leave open has to come out as in 64."""
    rng = np.random.default_rng(4)
    x = []
    for e in (-20, -17, -14, 0, 5):
        for _ in range(8):
            d = (128 + rng.integers(0, 128)) * 2.0 ** (e - 7)
            y = d * (rng.integers(0, 16, 64) - 8.5)
            y[[0, 32]] = -8 * d * np.array([1.0, 1.0 + rng.integers(0, 3) / 512])
            y[5:10] = np.nextafter(y[5:10].astype(np.float32), np.float32(np.inf))
            y[40:50] = np.nextafter(y[40:50].astype(np.float32), np.float32(-np.inf))
            x += [y, -y, np.where(np.arange(64) < 32, y, 0.0)]
    x = np.array(x).astype(np.float32)
    n = len(x)
    s = SetupQ4(2, 1, 64, 16, [q] * n, [q] * n, seed=6)
    s.qkv[0::q, 128:192] = x
    d = DeviceQ4(lib, cuda, s)
    d.append(10000.0)
    lib.status()
    kn, kd = unpack(d.k.cpu().numpy(), 16, 64)
    want = s.append(10000.0)[1]
    for t, sq, p in s.rows():
        wn, wd = quantise(want[t, 0])
        page = int(s.table[sq, 0])
        assert np.array_equal(kn[page, 0, p], wn) and np.array_equal(kd[page, 0, p].astype(np.float64), wd), (t, p)


def test_append_turned_keys_of_any_size(lib, cuda):
    """Keys up to the largest and down to the smallest numbers, infinities and NaN, turned."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((60, 64)) * np.exp2(rng.integers(-140, 127, (60, 1)))
    x[10:20] = rng.choice([-3.4e38, 3.4e38, 1e38, 0.0, 1.0], (10, 64))
    x[20:30, 40] = [np.inf, -np.inf, np.nan, np.inf, 3.4e38, -3.4e38, 1e37, 1.01e37, -0.0, 1e-45]
    s = SetupQ4(2, 1, 64, 16, [60], [60], seed=7)
    s.qkv[:, 128:192] = x
    d = DeviceQ4(lib, cuda, s)
    d.append(10000.0)
    lib.status()
    kn, kd = unpack(d.k.cpu().numpy(), 16, 64)
    with np.errstate(invalid="ignore"):
        want = s.append(10000.0)[1]
    for t, sq, p in s.rows():
        wn, wd = quantise(want[t, 0])
        page, off = int(s.table[sq, p // 16]), p % 16
        assert np.array_equal(kd[page, 0, off].astype(np.float64), wd, equal_nan=True), t
        ok = np.repeat(np.isfinite(wd), 32)
        assert np.array_equal(kn[page, 0, off][ok], wn[ok]), t


def test_append_far_positions(lib, cuda):
    """A page of keys at positions near 2 10^6, turned as the definition turns each."""
    n = 2_000_064
    for theta in (10000.0, 500000.0):
        s = SetupQ4(2, 1, 64, 64, q=[64], kv=[64], seed=18)
        d = DeviceQ4(lib, cuda, s)
        table = cuda.full((1, n // 64), -1, dtype=cuda.int32, device="cuda")
        table[0, -1] = int(s.table[0, 0])
        d.table, d.batch.page_table, d.batch.max_pages, d.batch.max_kv_len = table, table.data_ptr(), n // 64, n
        d.len[0] = n
        s.kv[0] = n
        d.append(theta)
        lib.status()
        want = s.append(theta)[1]
        gn, gd = unpack(d.k.cpu().numpy(), 64, 64)
        wn, wd = quantise(want[:, 0])
        page = int(s.table[0, 0])
        assert np.array_equal(gn[page, 0], wn) and np.array_equal(gd[page, 0].astype(np.float64), wd)


# ----------------------------------------------------------------------- read
@pytest.mark.parametrize("type_", [F16, F32, Q4_0])
@pytest.mark.parametrize("shape", SHAPES)
def test_read(lib, cuda, type_, shape):
    q, kv = [1, 70, 0, 5, 1, 3, 1], [90, 137, 12, 5, 0, 2, 64]
    s = SetupQ4(*shape, q=q, kv=kv, tail=2, seed=6) if type_ == Q4_0 else Setup(type_, *shape, q=q, kv=kv, tail=2, seed=6)
    d = (DeviceQ4 if type_ == Q4_0 else Device)(lib, cuda, s)
    k, v = (x.cpu().numpy() for x in DeviceQ4.read(d))
    lib.status()
    want_k, want_v = np.full_like(k, 777.0), np.full_like(v, 777.0)
    for t, sq, p in s.rows():
        want_k[t] = want_v[t] = 0.0
        if p >= 0:
            page, off = int(s.table[sq, p // s.page]), p % s.page
            want_k[t], want_v[t] = s.k[page, :, off], s.v[page, :, off]
    assert np.array_equal(k, want_k) and np.array_equal(v, want_v)


def test_read_pages_out_of_range(lib, cuda):
    d = dev(lib, cuda, 6, 2, 64, 32, q=[3, 2], kv=[34, 40], seed=7)
    d.table[0, 1] = d.s.num_pages
    k, _ = d.read()
    with pytest.raises(nedo_gpu.NedoGpuError) as e:
        lib.status(d.stream())
    assert e.value.code == nedo_gpu.ERR_DEVICE
    assert (k[1:3] == 0).all() and (k[0] != 0).any() and (k[3] != 0).any()


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("shape", SHAPES)
def test_single_tokens(lib, cuda, shape):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 0]
    d = dev(lib, cuda, *shape, q=[1] * len(kv), kv=kv, tail=1, seed=1)
    check_attention(d.s, d.attention(), d.s.attention())
    lib.status()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("q", [2, 3, 5])
def test_drafted_tokens(lib, cuda, shape, q):
    kv = [q, q + 1, 16, 64, 127, 131, 300, 2, 0]
    d = dev(lib, cuda, *shape, q=[q] * len(kv), kv=kv, seed=2)
    check_attention(d.s, d.attention(), d.s.attention())
    check_attention(d.s, d.attention(33), d.s.attention(33))
    lib.status()


@pytest.mark.parametrize("shape", SHAPES)
def test_ragged_prompts(lib, cuda, shape):
    q, kv = [1, 37, 0, 5, 64, 1, 23, 150], [90, 37, 12, 133, 65, 0, 24, 410]
    d = dev(lib, cuda, *shape, q=q, kv=kv, tail=3, seed=3)
    check_attention(d.s, d.attention(), d.s.attention())
    check_attention(d.s, d.attention(70), d.s.attention(70))
    lib.status()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 4000])
def test_window(lib, cuda, hd, window):
    q, kv = [1, 70, 3, 1, 1], [500, 140, 66, 64, 1]
    d = dev(lib, cuda, 6, 2, hd, 32, q=q, kv=kv, seed=4)
    for s in range(d.s.seqs):  # pages in front of every row's window are not read
        d.table[s, :max(0, d.s.kv[s] - d.s.q[s] + 1 - window) // 32] = -1
    check_attention(d.s, d.attention(window), d.s.attention(window))
    lib.status()


def test_fewer_keys_than_rows(lib, cuda):
    d = dev(lib, cuda, 12, 4, 128, 64, q=[5, 1, 4, 9, 60], kv=[2, 0, 0, 9, 50], seed=5)
    d.q[[0, 1, 2, 5, 6, 7, 8, 9] + list(range(19, 29))] = float("nan")
    check_attention(d.s, d.attention(), d.s.attention())


@pytest.mark.parametrize("kv", [2049, 5000, 20011])
@pytest.mark.parametrize("heads,hd", [(6, 64), (32, 128), (16, 256)])
def test_long_sequences(lib, cuda, kv, heads, hd):
    d = dev(lib, cuda, heads, 2, hd, 64, q=[1], kv=[kv], seed=6)
    check_attention(d.s, d.attention(), d.s.attention())
    d = dev(lib, cuda, heads, 2, hd, 64, q=[1, 1, 2, 1], kv=[3, kv, 1500, 0], seed=7)
    check_attention(d.s, d.attention(), d.s.attention())
    check_attention(d.s, d.attention(1000), d.s.attention(1000))


@pytest.mark.parametrize("heads,kv_heads,hd", [(6, 2, 64), (2, 2, 128), (16, 2, 96), (4, 2, 192)])
def test_long_prompt(lib, cuda, heads, kv_heads, hd):
    d = dev(lib, cuda, heads, kv_heads, hd, 64, q=[333, 1, 130], kv=[1200, 700, 130], seed=8)
    check_attention(d.s, d.attention(), d.s.attention())
    check_attention(d.s, d.attention(257), d.s.attention(257))


@pytest.mark.parametrize("heads,kv_heads,hd,page,shared,q,kv", [
    (12, 4, 128, 64, 3, [1] * 9, [193 + 31 * i for i in range(9)]),
    (12, 4, 128, 64, 20, [1] * 40, [1280 + 7 * i for i in range(40)]),
    (4, 4, 64, 16, 1, [1, 1], [17, 40]),
    (8, 1, 96, 32, 40, [3, 1, 0, 7], [1300, 1281, 1290, 1400]),
    (6, 2, 32, 16, 5, [1, 2, 1, 1, 30], [60, 3, 0, 200, 100]),
    (6, 2, 256, 128, 9, [1] * 9, [1160, 1153, 3000, 1200, 1153, 1400, 1300, 2000, 1153]),
    (2, 2, 64, 64, 33, [1], [2500]),
])
def test_shared_prefix(lib, cuda, heads, kv_heads, hd, page, shared, q, kv):
    d = dev(lib, cuda, heads, kv_heads, hd, page, q=q, kv=kv, shared=shared, tail=2, seed=9)
    check_attention(d.s, d.attention(), d.s.attention())
    check_attention(d.s, d.attention(77), d.s.attention(77))
    lib.status()
    d.table[1:, :shared] = -1
    check_attention(d.s, d.attention(), d.s.attention())
    lib.status()


@pytest.mark.parametrize("hd", [64, 128, 160])
def test_large_scores(lib, cuda, hd):
    d = dev(lib, cuda, 6, 2, hd, 32, q=[1, 4, 40], kv=[700, 90, 90], seed=10)
    for scale in (20.0, -20.0, 0.0):
        d.s.scale = scale
        check_attention(d.s, d.attention(), d.s.attention())


@pytest.mark.parametrize("hd", [64, 128, 160])
@pytest.mark.parametrize("f", [2.0 ** -22, 2.0 ** -14, 1.0 / 3, 20000.0])
def test_sizes_of_scales(lib, cuda, hd, f):
    """Scales of one or two smallest steps, of eleven bits (the values are rounded to fp16), large ones."""
    s = SetupQ4(6, 2, hd, 32, q=[1, 3, 30], kv=[300, 70, 90], seed=11)
    s.scale_values("v", f)
    s.scale_values("k", min(f, 1.0 / 3))
    d = DeviceQ4(lib, cuda, s)
    with np.errstate(invalid="ignore"):
        want = s.attention()
    check(d.attention(), *want)  # (the largest values are infinities)


@pytest.mark.parametrize("hd,heads", [(64, 6), (128, 6), (128, 2), (256, 2), (128, 16)])
@pytest.mark.parametrize("window", [0, 30])
def test_rows_that_do_not_see_odd_blocks(lib, cuda, hd, heads, window):
    """A value block of scale NaN or infinity reaches the rows that see it, in its channels, a key block the
    whole rows, and no other row."""
    q, kv = [40, 1, 3, 2], [100, 300, 60, 200]
    s = SetupQ4(heads, 2, hd, 32, q=q, kv=kv, seed=12)
    plain = s.attention(window)
    odd = {}
    for seq, pos, block, name, x in ((0, 85, 1, "v", np.nan), (1, 290, 0, "v", np.nan), (2, 58, 0, "k", np.nan),
                                     (3, 199, 1, "v", np.inf), (3, 10, 0, "k", np.nan), (0, 99, 1, "k", np.nan)):
        d, n = getattr(s, name + "d"), getattr(s, name + "n")
        at = int(s.table[seq, pos // 32]), 1, pos % 32
        d[at][block] = x
        s.put(name, n, d)
        odd.setdefault(seq, []).append((pos, block, name))
    want, tol, inside = (a.copy() for a in plain)
    group = heads // 2
    hit = np.zeros(want.shape, bool)
    for t, seq, p in s.rows():
        for pos, block, name in odd[seq]:
            if pos <= p and (not window or pos > p - window):
                hit[t, group:, slice(None) if name == "k" else slice(32 * block, 32 * block + 32)] = True
    assert hit.any() and not hit.all()
    got = DeviceQ4(lib, cuda, s).attention(window).cpu().numpy()
    assert not np.isfinite(got[hit]).any()
    check_attention(s, cuda.from_numpy(np.where(hit, want, got)), (want, tol, inside))
    lib.status()


def test_queries_that_are_not_finite(lib, cuda):
    d = dev(lib, cuda, 6, 2, 64, 32, q=[20, 1, 3], kv=[100, 300, 60], seed=13)
    want = d.s.attention()
    hit = np.zeros_like(want[0], bool)
    for t, h in ((3, 2), (20, 4), (22, 5)):
        d.q[t, h, 31] = float("nan")
        hit[t, h] = True
    got = d.attention().cpu().numpy()
    assert np.isnan(got[hit]).all()
    check_attention(d.s, cuda.from_numpy(np.where(hit, want[0], got)), want)


@pytest.mark.parametrize("q", [1, 3, 40])
def test_pages_out_of_range(lib, cuda, q):
    d = dev(lib, cuda, 6, 2, 64, 32, q=[q, q], kv=[100, 90], seed=14)
    d.table[0, 1] = d.s.num_pages
    got = d.attention()
    with pytest.raises(nedo_gpu.NedoGpuError) as e:
        lib.status(d.stream())
    assert e.value.code == nedo_gpu.ERR_DEVICE
    blocks = np.full((2 * q, 2, 4), 0xFFFFFFFF, np.uint32)
    blocks[:q, :, :3] = [0, 2, 3]
    blocks[q:, :, :3] = [0, 1, 2]
    check_attention(d.s, got, d.s.attention(blocks=blocks))
    lib.status()


def test_offsets_beyond_32_bits(lib, cuda):
    """Pages at both ends of a cache of more than 2^32 bytes, written, read back and attended."""
    s = SetupQ4(4, 2, 128, 64, q=[1, 7, 1, 30], kv=[200, 130, 64, 90], seed=16)
    d = DeviceQ4(lib, cuda, s)
    pages = (1 << 32) // d.k[0].numel() + 40
    k = cuda.empty((pages,) + d.k.shape[1:], dtype=cuda.uint8, device="cuda")
    v = cuda.empty_like(k)
    spread = {int(p): (int(p) if i % 2 else pages - 1 - int(p)) for i, p in
              enumerate(np.unique(s.table[s.table != 0xFFFFFFFF]))}
    for a, b in spread.items():
        k[b], v[b] = d.k[a], d.v[a]
    table = np.vectorize(lambda p: spread.get(int(p), 0xFFFFFFFF))(s.table).astype(np.uint32)
    d.table.copy_(cuda.from_numpy(table.view(np.int32)))
    d.cache.k, d.cache.v, d.cache.num_pages, d.cache.bounds = k.data_ptr(), v.data_ptr(), pages, None
    check_attention(s, d.attention(), s.attention())
    d.append(10000.0)
    got = d.read()
    lib.status()
    for x, want in zip(got, s.append(10000.0)[1:3]):
        assert np.array_equal(x.cpu().numpy(), values(*quantise(want)).astype(np.float32))


# -------------------------------------------------- selection, attention over picked pages
def random_blocks(s, picks, rng):
    out = np.full((s.tokens, s.kv_heads, picks), 0xFFFFFFFF, np.uint32)
    for t, _, p in s.rows():
        for kh in range(s.kv_heads):
            if p >= 0:
                n = min(picks, p // s.page + 1)
                out[t, kh, :n] = np.sort(rng.choice(p // s.page + 1, n, replace=False))
    return out


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("picks", [1, 3, 30])
def test_block_attention(lib, cuda, shape, picks):
    page = shape[3]
    kv = [1, page, page + 1, 3 * page, 12 * page + 3, 0, 29 * page, 31 * page + 1]
    d = dev(lib, cuda, *shape, q=[1, 1, 1, 2, 3, 1, 1, 1], kv=kv, tail=2, seed=24)
    blocks = random_blocks(d.s, picks, np.random.default_rng(picks))
    check_attention(d.s, d.block_attention(blocks), d.s.attention(blocks=blocks))
    lib.status()


def test_block_lists_out_of_order(lib, cuda):
    d = dev(lib, cuda, 6, 2, 64, 16, q=[1] * 5, kv=[200] * 5, seed=25)
    blocks = np.random.default_rng(5).integers(0, 14, (5, 2, 70)).astype(np.uint32)
    blocks[1, :, :3] = [5, 5, 3]
    blocks[1, :, 3:] = 5
    blocks[2] = 0xFFFFFFFF
    blocks[3, 0] = 99
    blocks[3, 1, :2] = [0x80000001, 12]
    blocks[4, :, 40:] = np.arange(30)
    check_attention(d.s, d.block_attention(blocks), d.s.attention(blocks=blocks))
    lib.status()


@pytest.mark.parametrize("shape", SHAPES)
def test_append_select_attend(lib, cuda, shape):
    """A prompt, then single tokens, appended; pages selected by the bounds that were kept; dense
    attention and attention over the pages."""
    page = shape[3]
    d = dev(lib, cuda, *shape, q=[2 * page + 3, 5, 40], kv=[4 * page + 3, 5, 41], seed=27)
    d.append(10000.0)
    s = d.held()
    q = d.out.clone()
    d.q.copy_(q)
    s.queries, s.bounds = q.cpu().numpy(), d.bounds.cpu().numpy()
    check_attention(s, d.attention(), s.attention())
    for picks in (2, 9):
        picked = d.select(picks).cpu().numpy().view(np.uint32)
        assert np.array_equal(picked, s.select(picks))
        check_attention(s, d.block_attention(picked), s.attention(blocks=picked))
    lib.status()


def test_decode_steps_match_whole_prompt(lib, cuda):
    """Tokens appended one by one leave the same numbers and scales as the prompt taken in whole."""
    n = 150
    s = SetupQ4(12, 4, 128, 64, q=[n], kv=[n], seed=28)
    whole, one = DeviceQ4(lib, cuda, s), DeviceQ4(lib, cuda, s)
    whole.append(10000.0)
    one.batch.tokens = one.batch.max_q_len = 1
    one.start[1] = 1
    q1 = cuda.empty((1, 12, 128), device="cuda")
    for p in range(n):
        one.len[0] = p + 1
        lib.kv_append_dev(one.cache, one.batch, 12, whole.qkv[p].data_ptr(), 10000.0, q1.data_ptr(), one.stream())
    lib.status()
    assert cuda.equal(one.k, whole.k) and cuda.equal(one.v, whole.v) and cuda.equal(one.bounds, whole.bounds)


# ------------------------------------------------------- graphs, streams, repeats
def test_results_repeat_and_graphs(lib, cuda):
    """Repeated calls, and a captured step replayed with other lengths, give the same bits as eager ones."""
    for kw in (dict(q=[1] * 5, kv=[3000, 40, 900, 1, 2500]), dict(q=[1] * 8, kv=[1100 + i for i in range(8)], shared=17),
               dict(q=[100, 1, 3], kv=[700, 650, 90])):
        d = dev(lib, cuda, 12, 4, 128, 64, seed=32, **kw)
        first = d.attention().clone()
        for _ in range(3):
            assert cuda.equal(d.attention(), first)
    d = dev(lib, cuda, 12, 4, 128, 64, q=[5] * 6, kv=[300, 900, 64, 2000, 5, 17], seed=33)
    need = lib.paged_attention_workspace(d.cache, d.batch, 12)
    ws, qo = d.space(need), cuda.zeros_like(d.q)
    ko, vo = (cuda.zeros((30, 4, 128), device="cuda") for _ in "kv")

    def step():
        lib.kv_append_dev(d.cache, d.batch, 12, d.qkv.data_ptr(), 1e4, qo.data_ptr(), d.stream())
        lib.paged_attention_dev(d.cache, d.batch, 12, qo.data_ptr(), d.out.data_ptr(), d.s.scale, 0, ws.data_ptr(), need, d.stream())
        lib.kv_read_dev(d.cache, d.batch, ko.data_ptr(), vo.data_ptr(), d.stream())

    step()
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        step()
    for lens in ([300, 900, 64, 2000, 5, 17], [299, 5, 64, 1500, 0, 7]):
        d.len.copy_(cuda.tensor(lens, dtype=cuda.int32))
        for x in (d.out, qo, ko, vo):
            x.fill_(777.0)  # (append leaves the queries of padding rows)
        step()
        want = [x.clone() for x in (d.out, qo, ko, vo, d.k, d.v)]
        for x in (d.out, qo, ko, vo):
            x.fill_(777.0)
        graph.replay()
        for a, b in zip((d.out, qo, ko, vo, d.k, d.v), want):
            assert cuda.equal(a, b)
    lib.status()


@pytest.mark.parametrize("shape,q,kv,shared", [
    ((4, 4, 64, 64), [1] * 6, [19001, 300, 12345, 18999, 1, 17000], 0), ((12, 12, 32, 16), [1] * 2, [16500, 6400], 0),
    ((12, 4, 128, 64), [5, 1, 3, 5], [20000, 5, 6400, 17777], 0), ((8, 4, 160, 32), [1, 2, 1], [17000, 300, 16999], 0),
    ((16, 8, 128, 64), [1] * 6, [9000, 1200, 8999, 1281, 5000, 6001], 18),
])
def test_chunks_from_the_lengths(lib, cuda, shape, q, kv, shared):
    """Batches whose chunks the device makes as long as the lengths ask: with other lengths of the same limits, none
    at all, and lengths out of range; eager and replayed."""
    d = dev(lib, cuda, *shape, q=q, kv=kv, seed=35, shared=shared)
    heads, hd = shape[0], shape[2]
    need = lib.paged_attention_workspace(d.cache, d.batch, heads)
    assert need % (d.s.tokens * heads * (hd * 4 + 8)) == 16  # the chunks' length is there
    check_attention(d.s, d.attention(), d.s.attention())
    window = 5000
    check_attention(d.s, d.attention(window), d.s.attention(window))
    ws, out = d.space(need), cuda.empty_like(d.out)

    def step(into):
        lib.paged_attention_dev(d.cache, d.batch, heads, d.q.data_ptr(), into.data_ptr(), d.s.scale, 0, ws.data_ptr(), need, d.stream())

    step(out)
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        step(out)
    first = shared * shape[3]
    for lens in (kv, [first + (n - first) // 2 for n in kv], [min(n, first + 70) for n in kv], [first + n for n in q], [0] * len(kv), kv):
        d.s.kv = list(lens)
        d.len.copy_(cuda.tensor(lens, dtype=cuda.int32))
        want = d.s.attention()
        d.out.fill_(777.0)
        out.fill_(777.0)
        step(d.out)
        check_attention(d.s, d.out, want)
        ws.fill_(255)
        graph.replay()
        assert cuda.equal(out, d.out)
    lib.status()


def test_two_streams_at_once(lib, cuda):
    """Two batches on two streams, each call with a workspace of its own, and two graphs replayed at once."""
    ds = [dev(lib, cuda, 12, 4, 128, 64, q=[1] * 8, kv=[4000 + 31 * i for i in range(8)], seed=41),
          dev(lib, cuda, 8, 2, 160, 32, q=[40, 1, 7], kv=[300, 900, 64], seed=42)]
    want = [d.attention().clone() for d in ds]
    need = [lib.paged_attention_workspace(d.cache, d.batch, d.s.heads) for d in ds]
    ws = [d.space(n) for d, n in zip(ds, need)]
    outs = [[cuda.empty_like(d.out) for _ in range(8)] for d in ds]
    streams = [cuda.cuda.Stream() for _ in ds]

    def call(i, out, stream):
        d = ds[i]
        lib.paged_attention_dev(d.cache, d.batch, d.s.heads, d.q.data_ptr(), out.data_ptr(), d.s.scale, 0, ws[i].data_ptr(), need[i],
                                stream.cuda_stream)

    def check_all():
        cuda.cuda.synchronize()
        for i in range(2):
            for out in outs[i]:
                inside = want[i] != 777.0
                assert cuda.equal(out[inside], want[i][inside])

    cuda.cuda.synchronize()
    for n in range(8):
        for i in range(2):
            call(i, outs[i][n], streams[i])
    check_all()
    graphs = [cuda.cuda.CUDAGraph() for _ in ds]
    for i in range(2):
        with cuda.cuda.graph(graphs[i], stream=streams[i]):
            for n in range(8):
                call(i, outs[i][n], streams[i])
    for x in outs[0] + outs[1]:
        x.zero_()
    cuda.cuda.synchronize()
    for i in range(2):
        with cuda.cuda.stream(streams[i]):
            graphs[i].replay()
    check_all()
    lib.status()
