"""GPU: the operators of a served batch in a row -- projections, append into a 4-bit cache, attention over
it, the head, verification of drafts -- as a loop that tries several tokens at a time.  What it produces is what
the same model produces one token at a time."""
import numpy as np
import pytest

import nedo_gpu
from drafts_ref import NONE
from nedo_gpu import blocks as B
from q4_ref import Q4_0

pytestmark = pytest.mark.gpu

HEADS, KVH, HD, DIM, VOCAB, PAGE, SEQS, ROOM = 6, 2, 64, 384, 700, 16, 3, 96


class Model:
    """One layer: x = embedding, x + W_o attention(W_qkv x), logits = W_head x; weights Q8_0."""

    def __init__(self, lib, torch, type_, seed):
        self.lib, self.torch = lib, torch
        up = lambda rows, cols, s: torch.from_numpy(B.gen_weight(B.Q8_0, rows, cols, seed=seed + s)).cuda()  # noqa: E731
        self.qkv, self.o, self.head = up((HEADS + 2 * KVH) * HD, DIM, 1), up(DIM, HEADS * HD, 2), up(VOCAB, DIM, 3)
        self.emb = torch.from_numpy(np.random.default_rng(seed).standard_normal((VOCAB, DIM)).astype(np.float32) * 2).cuda()
        pages = SEQS * (ROOM // PAGE)
        size = {Q4_0: PAGE * HD // 32 * 18, B.F16: PAGE * HD * 2}[type_]
        # (NaN scales and numbers wherever nothing has been appended)
        self.k, self.v = (torch.full((pages, KVH, size), 0xFF, dtype=torch.uint8, device="cuda") for _ in "kv")
        order = np.random.default_rng(seed + 9).permutation(pages).astype(np.int32).reshape(SEQS, -1)
        self.table = torch.from_numpy(order).cuda()
        self.cache = nedo_gpu.KvCache(type=type_, kv_heads=KVH, head_dim=HD, page_size=PAGE, num_pages=pages,
                                      k=self.k.data_ptr(), v=self.v.data_ptr(), bounds=None)

    def logits(self, rows, before):
        """Logits of every sequence's new tokens (lists), `before` tokens of it being cached."""
        torch, lib = self.torch, self.lib
        st = torch.cuda.current_stream().cuda_stream
        starts = np.concatenate(([0], np.cumsum([len(r) for r in rows]))).astype(np.int32)
        n = int(starts[-1])
        lens = torch.tensor([b + len(r) for b, r in zip(before, rows)], dtype=torch.int32, device="cuda")
        start = torch.from_numpy(starts).cuda()
        batch = nedo_gpu.KvBatch(seqs=SEQS, tokens=n, max_q_len=max(len(r) for r in rows), max_kv_len=ROOM, max_pages=ROOM // PAGE,
                                 shared_pages=0, q_start=start.data_ptr(), kv_len=lens.data_ptr(), page_table=self.table.data_ptr())
        x = self.emb[torch.tensor(sum(rows, []), device="cuda")].contiguous()
        new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        qkv, q, att, y, out = new(n, (HEADS + 2 * KVH) * HD), new(n, HEADS, HD), new(n, HEADS, HD), new(n, DIM), new(n, VOCAB)
        need = lib.paged_attention_workspace(self.cache, batch, HEADS)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        lib.matvec_dev(B.Q8_0, (HEADS + 2 * KVH) * HD, DIM, self.qkv.data_ptr(), x.data_ptr(), qkv.data_ptr(), n, st)
        lib.kv_append_dev(self.cache, batch, HEADS, qkv.data_ptr(), 10000.0, q.data_ptr(), st)
        lib.paged_attention_dev(self.cache, batch, HEADS, q.data_ptr(), att.data_ptr(), HD ** -0.5, 0, ws.data_ptr(), need, st)
        lib.matvec_dev(B.Q8_0, DIM, HEADS * HD, self.o.data_ptr(), att.data_ptr(), y.data_ptr(), n, st)
        y += x
        lib.matvec_dev(B.Q8_0, VOCAB, DIM, self.head.data_ptr(), y.data_ptr(), out.data_ptr(), n, st)
        return out, start

    def verify(self, logits, start, drafts, temperature, accept_u=None, sample_u=None):
        torch, n = self.torch, logits.shape[0]
        ids = torch.full((n,), -7, dtype=torch.int32, device="cuda")
        accepted = torch.full((SEQS,), -7, dtype=torch.int32, device="cuda")
        rows = (start[1:] - start[:-1]).max().item()
        d = nedo_gpu.Drafts(seqs=SEQS, rows=n, max_rows=rows, vocab=VOCAB, row_start=start.data_ptr(), logits=logits.data_ptr(),
                            draft_ids=drafts.data_ptr(), draft_probs=None, accept_u=None if accept_u is None else accept_u.data_ptr(),
                            sample_u=None if sample_u is None else sample_u.data_ptr())
        need = self.lib.verify_drafts_workspace(d)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        self.lib.verify_drafts_dev(d, temperature, accepted.data_ptr(), ids.data_ptr(), ws.data_ptr(), need,
                                   torch.cuda.current_stream().cuda_stream)
        return accepted.cpu().numpy(), ids.cpu().numpy().view(np.uint32)


@pytest.mark.parametrize("type_", [Q4_0, B.F16])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_drafted_decoding_is_decoding(lib, cuda, type_, temperature):
    prompts = [[5, 17, 400, 2, 9], [77], [1, 2, 3, 650, 0, 12, 13, 14, 15, 16, 88, 20, 21, 300, 301, 302, 303]]
    n = 40
    u = np.random.default_rng(1).random((SEQS, n + 16)).astype(np.float32)  # one number for each place

    def pick(model, logits, start, at, drafts=None):
        """Drafts taken, and the token behind them; without a draft's luck: a draft is taken where the token that
        the place's number draws is the draft."""
        rows = np.diff(start.cpu().numpy())
        d = cuda.full((logits.shape[0],), -1, dtype=cuda.int32, device="cuda")
        if drafts is not None:
            for s in range(SEQS):
                d[int(start[s]):int(start[s]) + len(drafts[s])] = cuda.tensor(drafts[s], dtype=cuda.int32)
        if not temperature:
            accepted, ids = model.verify(logits, start, d, 0.0)
            return [[int(x) for x in ids[int(start[s]):int(start[s]) + int(accepted[s]) + 1]] for s in range(SEQS)]
        # every row as a sequence of its own: sampling without drafts
        out, one = [], cuda.arange(SEQS + 1, dtype=cuda.int32, device="cuda")
        for i in range(int(rows.max())):
            row = cuda.stack([logits[int(start[s]) + min(i, int(rows[s]) - 1)] for s in range(SEQS)])
            v = cuda.from_numpy(np.array([u[s, at[s] + i] for s in range(SEQS)])).cuda()
            accepted, ids = model.verify(row, one, d, temperature, sample_u=v)
            assert (accepted == 0).all()
            out.append(ids)
        got = []
        for s in range(SEQS):
            tokens = []
            for i in range(int(rows[s])):
                tokens.append(int(out[i][s]))
                if drafts is None or i >= len(drafts[s]) or tokens[-1] != drafts[s][i]:
                    break
            got.append(tokens)
        return got

    before = lib.set_exact_batches(True)  # (the same products whatever the batch)
    try:
        # a token at a time
        slow = Model(lib, cuda, type_, seed=4)
        logits, start = slow.logits(prompts, [0] * SEQS)
        last = start[1:].long() - 1
        one = cuda.arange(SEQS + 1, dtype=cuda.int32, device="cuda")
        token = [x[0] for x in pick(slow, logits[last].contiguous(), one, [0] * SEQS)]
        text = [[t] for t in token]
        for i in range(1, n):
            logits, start = slow.logits([[t[-1]] for t in text], [len(p) + i - 1 for p in prompts])
            for s, x in enumerate(pick(slow, logits, start, [i] * SEQS)):
                text[s].append(x[0])
        # with drafts: the tokens to come, some of them wrong
        fast = Model(lib, cuda, type_, seed=4)
        rng = np.random.default_rng(2)
        logits, start = fast.logits(prompts, [0] * SEQS)
        got = [[x[0]] for x in pick(fast, logits[last].contiguous(), one, [0] * SEQS)]
        steps = 0
        while min(len(g) for g in got) < n:
            steps += 1
            rows, drafts = [], []
            for s in range(SEQS):
                k = int(rng.integers(0, 5)) if len(got[s]) < n else 0
                d = [t if rng.random() < 0.8 else (t + 1) % VOCAB for t in text[s][len(got[s]):len(got[s]) + k]]
                drafts.append(d)
                rows.append([got[s][-1] if len(got[s]) <= n else text[s][n - 1]] + d)
            logits, start = fast.logits(rows, [len(prompts[s]) + len(got[s]) - 1 for s in range(SEQS)])
            for s, x in enumerate(pick(fast, logits, start, [len(g) for g in got], drafts)):
                assert NONE not in x
                if len(got[s]) < n:
                    got[s] += x
        lib.status()
    finally:
        lib.set_exact_batches(before)
    assert steps < n - 5
    for s in range(SEQS):
        assert got[s][:n] == text[s][:n]
