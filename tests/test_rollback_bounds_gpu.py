"""GPU: what drafts that did not stand leave in the key bounds of a paged cache, and how a caller has the bounds
as if they had never been appended: the last page's rows read and appended again from its first slot."""
import numpy as np
import pytest

import nedo_gpu
from paged_ref import F16, F32
from q4_ref import Q4_0

pytestmark = pytest.mark.gpu

HEADS, KVH, HD, PAGE, ROOM, SEQS = 6, 2, 64, 16, 8, 3
BYTES = {F32: HD * 4, F16: HD * 2, Q4_0: HD // 32 * 18}


class Cache:
    def __init__(self, lib, torch, type_):
        self.lib, self.torch = lib, torch
        pages = SEQS * ROOM
        self.k, self.v = (torch.full((pages, KVH, PAGE * BYTES[type_]), 0xFF, dtype=torch.uint8, device="cuda") for _ in "kv")
        self.bounds = torch.zeros((pages, KVH, 2, HD), dtype=torch.float32 if type_ == F32 else torch.float16, device="cuda")
        self.table = torch.from_numpy(np.random.default_rng(1).permutation(pages).astype(np.int32).reshape(SEQS, ROOM)).cuda()
        self.desc = nedo_gpu.KvCache(type=type_, kv_heads=KVH, head_dim=HD, page_size=PAGE, num_pages=pages, k=self.k.data_ptr(),
                                     v=self.v.data_ptr(), bounds=self.bounds.data_ptr())

    def stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    def batch(self, n, lens):
        up = lambda x: self.torch.tensor([int(i) for i in x], dtype=self.torch.int32, device="cuda")  # noqa: E731
        self.lists = up(np.concatenate(([0], np.cumsum(n)))), up(lens)
        return nedo_gpu.KvBatch(seqs=SEQS, tokens=int(sum(n)), max_q_len=int(max(n)), max_kv_len=ROOM * PAGE, max_pages=ROOM, shared_pages=0,
                                q_start=self.lists[0].data_ptr(), kv_len=self.lists[1].data_ptr(), page_table=self.table.data_ptr())

    def append(self, rows, lens, theta=10000.0, heads=HEADS):
        """Rows of q|k|v of every sequence (a list of arrays), up to lens tokens cached."""
        qkv = self.torch.cat(rows).contiguous()
        q = self.torch.empty((len(qkv), heads, HD), device="cuda")
        self.lib.kv_append_dev(self.desc, self.batch([len(r) for r in rows], lens), heads, qkv.data_ptr(), theta, q.data_ptr(), self.stream())
        return q

    def read(self, n, lens):
        k, v = (self.torch.full((int(sum(n)), KVH, HD), 777.0, device="cuda") for _ in "kv")
        self.lib.kv_read_dev(self.desc, self.batch(n, lens), k.data_ptr(), v.data_ptr(), self.stream())
        return k, v

    def begin_last_page_anew(self, lens):
        """The bounds of every sequence's last page from the keys that count: its rows read, and appended unturned.
        (A full page holds no rows that do not count.)"""
        n = [x % PAGE for x in lens]
        if not sum(n):
            return
        k, v = self.read(n, lens)
        rows = self.torch.cat((k, k, v), 1).reshape(-1, 3 * KVH * HD).split(n)  # (as many query heads as KV heads, not used)
        self.append(rows, lens, 0.0, KVH)

    def select(self, q, n, lens, picks):
        out = self.torch.full((len(q), KVH, picks), -7, dtype=self.torch.int32, device="cuda")
        self.lib.block_select_dev(self.desc, self.batch(n, lens), HEADS, q.data_ptr(), picks, out.data_ptr(), self.stream())
        return out


@pytest.mark.parametrize("type_", [F32, F16, Q4_0])
@pytest.mark.parametrize("cached", [[37, 16, 60], [41, 95, 7]])
def test_rejected_drafts_and_bounds(lib, cuda, type_, cached):
    """Three steps whose drafts, keys of fifty times the size, do not stand, within a page and over a page's end."""
    g = cuda.Generator(device="cuda").manual_seed(3)
    fresh = lambda n, size=1.0: cuda.randn((n, (HEADS + 2 * KVH) * HD), generator=g, device="cuda") * size  # noqa: E731
    never, kept, anew = (Cache(lib, cuda, type_) for _ in range(3))
    lens, wider = list(cached), False
    prompt = [fresh(n) for n in lens]
    for c in (never, kept, anew):
        c.append(prompt, lens)
    for step in range(3):
        # a step with drafts in two of the caches; only its first row stands
        one = [fresh(1) for _ in lens]
        drafted = [cuda.cat((x, fresh(2 + s + step, 50.0))) for s, x in enumerate(one)]
        after = [x + 1 for x in lens]
        for c in (kept, anew):
            c.append(drafted, [x + len(d) for x, d in zip(lens, drafted)])
        never.append(one, after)
        lens = after
        anew.begin_last_page_anew(lens)
        for c in (kept, anew):  # the rows that count are there, bit for bit
            assert all(cuda.equal(a, b) for a, b in zip(c.read(lens, lens), never.read(lens, lens)))
        for s, x in enumerate(lens):
            for i in range(-(-x // PAGE)):
                p = int(never.table[s, i])
                # the extremes are kept by the drafts, on the page that they went to: bounds, but wider
                assert (kept.bounds[p, :, 0] <= never.bounds[p, :, 0]).all() and (kept.bounds[p, :, 1] >= never.bounds[p, :, 1]).all()
                wider = wider or not cuda.equal(kept.bounds[p], never.bounds[p])
                assert cuda.equal(anew.bounds[p], never.bounds[p])
    assert wider
    lib.status()


@pytest.mark.parametrize("type_", [F32, F16, Q4_0])
def test_pages_selected_after_rejected_drafts(lib, cuda, type_):
    """Pages are picked as if the drafts had never been, once the last page has begun anew after each step."""
    g = cuda.Generator(device="cuda").manual_seed(4)
    fresh = lambda n, size=1.0: cuda.randn((n, (HEADS + 2 * KVH) * HD), generator=g, device="cuda") * size  # noqa: E731
    never, kept, anew = (Cache(lib, cuda, type_) for _ in range(3))
    lens = [40, 50, 61]
    prompt = [fresh(n) for n in lens]
    for c in (never, kept, anew):
        c.append(prompt, lens)
    other = 0
    for step in range(40):
        one = [fresh(1) for _ in lens]
        drafted = [cuda.cat((x, fresh(3, 50.0))) for x in one]
        after = [x + 1 for x in lens]
        for c in (kept, anew):
            c.append(drafted, [x + 4 for x in lens])
        q = never.append(one, after)
        lens = after
        anew.begin_last_page_anew(lens)
        picked = [c.select(q, [1] * SEQS, lens, 3) for c in (never, kept, anew)]
        assert cuda.equal(picked[0], picked[2])
        other += not cuda.equal(picked[0], picked[1])
    assert other
    lib.status()
