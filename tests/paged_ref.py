"""The paged KV-cache operators in 64 bits, one query row at a time (numpy), and
small caches and batches to run them on.  Test infrastructure."""
from __future__ import annotations

import math

import numpy as np

F32, F16 = 0, 1
DTYPES = {F32: np.float32, F16: np.float16}
U = 2.0 ** -24  # half a step of fp32, relative


class Setup:
    """A cache and a ragged batch over it: `q` new tokens and `kv` cached tokens per
    sequence, pages dealt out in no order, everything no sequence owns filled with
    NaN and infinities."""

    def __init__(self, type_, heads, kv_heads, hd, page, q, kv, shared=0, tail=0, seed=0, spare=3, same_prefix=True):
        r = self.rng = np.random.default_rng(seed)
        self.type, self.heads, self.kv_heads, self.hd, self.page = type_, heads, kv_heads, hd, page
        self.q, self.kv, self.shared, self.tail = list(q), list(kv), shared, tail
        self.seqs = len(q)
        self.start = np.concatenate(([0], np.cumsum(q))).astype(np.uint32)
        self.tokens = int(self.start[-1]) + tail
        self.max_pages = max(1, shared, max((-(-n // page) for n in kv), default=1))
        count = shared + sum(max(0, -(-n // page) - shared) for n in kv)
        self.num_pages = count + spare
        order = list(r.permutation(self.num_pages)[:count])
        prefix, order = order[:shared], order[shared:]
        self.table = np.full((self.seqs, self.max_pages), 0xFFFFFFFF, np.uint32)
        for s in range(self.seqs):
            self.table[s, :shared] = prefix
            for i in range(shared, -(-self.kv[s] // page)):
                self.table[s, i] = order.pop()
        dt = DTYPES[type_]
        shape = (self.num_pages, kv_heads, page, hd)
        junk = np.array([np.nan, np.inf, -np.inf], dt)
        self.k = junk[r.integers(0, 3, shape)]
        self.v = junk[r.integers(0, 3, shape)]
        for s in range(self.seqs):
            for i in range(-(-self.kv[s] // page)):
                p, n = self.table[s, i], min(page, self.kv[s] - i * page)
                if i < shared:
                    n = page
                if not np.isfinite(self.k[p, :, :n].astype(np.float32)).all():
                    self.k[p, :, :n] = r.standard_normal((kv_heads, n, hd)).astype(dt)
                    self.v[p, :, :n] = r.standard_normal((kv_heads, n, hd)).astype(dt)
        self.queries = r.standard_normal((self.tokens, heads, hd)).astype(np.float32)
        self.qkv = r.standard_normal((self.tokens, (heads + 2 * kv_heads) * hd)).astype(np.float32)
        self.scale = 1.0 / math.sqrt(hd)
        lo, hi = np.full((self.num_pages, kv_heads, hd), 1e4), np.full((self.num_pages, kv_heads, hd), -1e4)
        for s in range(self.seqs):
            for i in range(-(-self.kv[s] // page)):
                p, n = self.table[s, i], min(page, self.kv[s] - i * page)
                lo[p], hi[p] = self.k[p, :, :n].min(1), self.k[p, :, :n].max(1)
        self.bounds = np.stack((lo, hi), 2).astype(dt)

    def rows(self):
        """(row, sequence, position) of every row that belongs to a sequence."""
        for s in range(self.seqs):
            for t in range(int(self.start[s]), int(self.start[s + 1])):
                yield t, s, self.kv[s] - (int(self.start[s + 1]) - t)

    def keys(self, s, kh, positions):
        pages = self.table[s][positions // self.page]
        return (self.k[pages, kh, positions % self.page].astype(np.float64),
                self.v[pages, kh, positions % self.page].astype(np.float64))

    def attention(self, window=0, blocks=None):
        """(out, tolerance, rows that belong to a sequence).

        The tolerance counts fp32 roundings as independent: a dot of hd terms is off
        by about u (sqrt(hd) + 4) S with S = scale sum |q k|, the weights by twice that
        (numerator and normaliser), the weighted sum of n keys by u (sqrt(n) + 16) of
        sum p |v|; twice the total is allowed.  In the weighted sum an F16 value below 2^-14
        counts as 2^-14: the tensor core takes the exponent of a subnormal operand as -14 when it
        lines products up, so what it cuts off is u of p 2^-14, not of p |v| (found with values
        of one or two smallest steps, 2^-24, whose sums were 1e-12 off)."""
        out = np.zeros((self.tokens, self.heads, self.hd))
        tol = np.zeros_like(out)
        inside = np.zeros(self.tokens, bool)
        g = self.heads // self.kv_heads
        for t, s, p in self.rows():
            inside[t] = True
            if p < 0:
                continue
            for kh in range(self.kv_heads):
                pos = np.arange(max(0, p - window + 1) if window else 0, p + 1)
                if blocks is not None:
                    listed, best = [], -1
                    for b in blocks[t, kh]:
                        if b <= p // self.page and int(b) > best:
                            listed.append(int(b))
                        if b <= p // self.page:
                            best = max(best, int(b))
                    pos = pos[np.isin(pos // self.page, listed)]
                if pos.size == 0:
                    continue
                k, v = self.keys(s, kh, pos)
                q = self.queries[t, kh * g:(kh + 1) * g].astype(np.float64)
                sc = q @ k.T * self.scale
                w = np.exp(sc - sc.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                out[t, kh * g:(kh + 1) * g] = w @ v
                big = (np.abs(q) @ np.abs(k).T * abs(self.scale)).max(1, keepdims=True)
                least = 2.0 ** -14 if self.type == F16 else 0.0
                tol[t, kh * g:(kh + 1) * g] = (4 * U * (math.sqrt(self.hd) + 4) * big * (w @ np.abs(v)) +
                                               2 * U * (math.sqrt(pos.size) + 16) * (w @ np.maximum(np.abs(v), least)))
        return out, tol, inside

    def select(self, picks):
        out = np.full((self.tokens, self.kv_heads, picks), 0xFFFFFFFF, np.uint32)
        g = self.heads // self.kv_heads
        for t, s, p in self.rows():
            if p < 0:
                continue
            own = p // self.page
            for kh in range(self.kv_heads):
                q = self.queries[t, kh * g:(kh + 1) * g].astype(np.float64)
                b = self.bounds[self.table[s, :own], kh].astype(np.float64)  # [own, 2, hd]
                with np.errstate(invalid="ignore"):
                    score = b[:, 1] @ np.maximum(q, 0).sum(0) + b[:, 0] @ np.minimum(q, 0).sum(0)
                key = np.where(np.isnan(score), -np.inf, score)
                order = sorted(range(own), key=lambda i: (np.isnan(score[i]), -key[i], i))
                got = sorted(order[:picks - 1] + [own])
                out[t, kh, :len(got)] = got
        return out

    def append(self, theta):
        """(rotated queries, keys [row, kv_heads, hd], values, rows that are tokens), unrounded."""
        hd, half = self.hd, self.hd // 2
        x = self.qkv.astype(np.float64)
        q = x[:, :self.heads * hd].reshape(-1, self.heads, hd).copy()
        k = x[:, self.heads * hd:(self.heads + self.kv_heads) * hd].reshape(-1, self.kv_heads, hd).copy()
        v = x[:, (self.heads + self.kv_heads) * hd:].reshape(-1, self.kv_heads, hd)
        real = np.zeros(self.tokens, bool)
        for t, s, p in self.rows():
            if p < 0:
                continue
            real[t] = True
            if theta:
                a = p * theta ** (-2.0 * np.arange(half) / hd)
                c, sn = np.cos(a), np.sin(a)
                for y in (q, k):
                    u, w = y[t, :, :half].copy(), y[t, :, half:].copy()
                    y[t, :, :half], y[t, :, half:] = u * c - w * sn, u * sn + w * c
        return q, k, v, real


class Device:
    """A Setup's arrays on the GPU and its calls of the library."""

    def __init__(self, lib, torch, s):
        import nedo_gpu

        self.lib, self.torch, self.s = lib, torch, s
        up = lambda a: torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda()  # noqa: E731
        self.k, self.v, self.bounds = up(s.k.copy()), up(s.v.copy()), up(s.bounds.copy())
        self.q, self.qkv = up(s.queries), up(s.qkv)
        self.start, self.len = up(s.start), up(np.asarray(s.kv, np.uint32))
        self.table = up(s.table.copy())
        self.cache = nedo_gpu.KvCache(type=s.type, kv_heads=s.kv_heads, head_dim=s.hd, page_size=s.page,
                                      num_pages=s.num_pages, k=self.k.data_ptr(), v=self.v.data_ptr(),
                                      bounds=self.bounds.data_ptr())
        self.batch = nedo_gpu.KvBatch(seqs=s.seqs, tokens=s.tokens, max_q_len=max(s.q), max_kv_len=max(s.kv),
                                      max_pages=s.max_pages, shared_pages=s.shared, q_start=self.start.data_ptr(),
                                      kv_len=self.len.data_ptr(), page_table=self.table.data_ptr())
        self.out = torch.full((s.tokens, s.heads, s.hd), 777.0, device="cuda")

    def stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    def space(self, n):
        return self.torch.full((max(16, n),), 0xFF, dtype=self.torch.uint8, device="cuda")  # NaN wherever read unwritten

    def attention(self, window=0, scale=None):
        n = self.lib.paged_attention_workspace(self.cache, self.batch, self.s.heads, window)
        self.ws = self.space(n)
        self.lib.paged_attention_dev(self.cache, self.batch, self.s.heads, self.q.data_ptr(), self.out.data_ptr(),
                                     self.s.scale if scale is None else scale, window, self.ws.data_ptr(), n,
                                     self.stream())
        return self.out

    def block_attention(self, blocks):
        picks = blocks.shape[-1]
        self.blocks = self.torch.from_numpy(np.ascontiguousarray(blocks).view(np.int32)).cuda()
        n = self.lib.block_attention_workspace(self.cache, self.batch, self.s.heads, picks)
        self.ws = self.space(n)
        self.lib.block_attention_dev(self.cache, self.batch, self.s.heads, self.q.data_ptr(), self.blocks.data_ptr(),
                                     picks, self.out.data_ptr(), self.s.scale, self.ws.data_ptr(), n, self.stream())
        return self.out

    def select(self, picks):
        self.picked = self.torch.full((self.s.tokens, self.s.kv_heads, picks), -7, dtype=self.torch.int32, device="cuda")
        self.lib.block_select_dev(self.cache, self.batch, self.s.heads, self.q.data_ptr(), picks,
                                  self.picked.data_ptr(), self.stream())
        return self.picked

    def append(self, theta):
        self.lib.kv_append_dev(self.cache, self.batch, self.s.heads, self.qkv.data_ptr(), theta, self.out.data_ptr(),
                               self.stream())
        return self.out


def check_attention(s, got, want, untouched=777.0):
    out, tol, inside = want
    got = got.cpu().numpy().astype(np.float64)
    assert (got[~inside] == untouched).all(), "rows behind the last sequence were written"
    err = np.abs(got[inside] - out[inside])
    bad = ~(err <= tol[inside])
    assert not bad.any(), f"{bad.sum()} outputs off, worst {np.nanmax(err / np.maximum(tol[inside], 1e-300)):.2f} x tolerance"
