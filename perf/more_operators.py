"""Serving many sequences from a 4-bit cache, with drafted tokens, as measured cases.

Entry points of the library (include/nedo_gpu.h) on a paged cache of type Q4_0, and the
sampling step of a batch whose sequences try several tokens at a time:

  append     nedo_gpu_kv_append_dev       q|k|v rows in: rotated queries out, rotated keys and
                                          values quantised into their pages, key bounds per page;
             nedo_gpu_kv_read_dev         the same rows' keys and values as the cache holds them
  attention  nedo_gpu_paged_attention_dev softmax attention of a ragged batch over 4-bit pages
  blocks     nedo_gpu_block_attention_dev attention over selected 4-bit pages only
  verify     nedo_gpu_verify_drafts_dev   drafted tokens against the target's probabilities, from
                                          given random numbers, and the token that follows them

A page of a Q4_0 cache holds, for one KV head, blocks of 32 channels of a token: 4-bit numbers
n in 0..15 for the values d (n - 8), and the blocks' fp16 scales d.  The numbers of all the page's
tokens come first, [page_size][head_dim / 8] words of 32 bits (channel 8 w + j in bits 2 j.. for
even j, 16 + 2 (j - 1).. for odd j), then the scales, [head_dim / 32][page_size].

``run`` computes them in plain torch operations, or through the library where ``own`` is true.
``exact`` is the definition in 64 bits, one sequence at a time.
"""
import math
import os
import sys

import torch

own = False

Q4_0 = 2  # GGUF tensor type code


# --------------------------------------------------------------------- cases
def _case(name, op, heads=12, kv_heads=4, head_dim=128, page=64, seqs=1, q=(1, 1), kv=(512, 512), idle=0, tail=0,
          theta=10000.0, bounds=False, window=0, shared=0, picks=0):
    """One case over the cache: `seqs` sequences of q[0]..q[1] new tokens and kv[0]..kv[1] cached
    tokens (the new ones included), every `idle`-th of them an unused slot of a padded batch (one
    token, nothing cached), `tail` rows behind the last token, the first `shared` pages common to
    all."""
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "seqs": seqs,
         "q_min": q[0], "q_max": q[1], "kv_min": kv[0], "kv_max": kv[1], "idle": idle, "tail": tail, "theta": theta,
         "bounds": bounds, "window": window, "shared": shared, "picks": picks}
    if name:
        c["name"] = name
    return c


def _verify(name, vocab=64000, seqs=1, q=(5, 5), temperature=0.8, probs=True, tail=0):
    """Logits of q[0]..q[1] rows (drafts + 1) for each of `seqs` sequences; `probs`: the drafts
    were drawn from a distribution that comes with them (else they are one model's single guess)."""
    c = {"op": "verify", "vocab": vocab, "seqs": seqs, "q_min": q[0], "q_max": q[1], "temperature": temperature,
         "probs": probs, "tail": tail}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token of one conversation: the call whose latency every generated token pays
        _case("append one token", "append", kv=(513, 513), bounds=True),
        # three prompts of odd lengths in one batch
        _case("append prompts", "append", seqs=3, q=(317, 1025), kv=(1025, 2047), bounds=True),
        # the decode step of one conversation at position 512
        _case("attention one token", "attention", kv=(513, 513)),
        # long conversations served together: the cache is what is read
        _case("attention long batch", "attention", seqs=32, kv=(8191, 32768)),
        # four drafted tokens and the one before them, of each of 16 conversations
        _case("attention drafts", "attention", seqs=16, q=(5, 5), kv=(2005, 16001)),
        # one token of each of 64 conversations behind one long system prompt, some slots unused
        _case("attention shared prefix", "attention", seqs=64, kv=(16384 + 33, 16384 + 701), shared=256, tail=2),
        # a prompt taken in whole, with the sliding window of the model's configuration
        _case("attention prompt", "attention", seqs=2, q=(1711, 2048), kv=(2048, 4096), window=2048),
        # attention over the pages that were selected for one token
        _case("blocks one token", "blocks", kv=(8200, 8200), picks=16),
        # and for a batch, 32 of up to 512 pages each
        _case("blocks batch", "blocks", seqs=64, kv=(16001, 32768), picks=32),
        # four drafts of one conversation, sampled from a draft model's distributions
        _verify("verify one sequence"),
        # two to eight drafts of each of 48 conversations, greedy
        _verify("verify greedy batch", seqs=48, q=(3, 9), temperature=0.0, probs=False, tail=1),
        # four drafts of each of 32 conversations over the large vocabulary
        _verify("verify batch", vocab=128000, seqs=32, q=(5, 5), temperature=1.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))) - 0.5))))


def draw(rng):
    op = rng.choice(("append", "append", "attention", "attention", "attention", "blocks", "verify", "verify"))
    if op == "verify":
        vocab, q = _log(rng, 500, 152000), rng.choice((1, 2, 3, 5, 8, 9))
        seqs = max(1, min(_log(rng, 1, 64), (32 * 5 * 128000) // (vocab * q)))
        return _verify("", vocab=vocab, seqs=seqs, q=(rng.choice((1, q)), q), tail=rng.choice((0, 0, 3)),
                       temperature=rng.choice((0.0, 0.6, 1.0, 1.3)), probs=rng.random() < 0.6)
    kv_heads, group = rng.choice(((4, 3), (12, 1), (2, 4), (1, 8), (3, 2), (8, 4), (2, 16), (1, 5)))
    kw = dict(kv_heads=kv_heads, heads=kv_heads * group, head_dim=rng.choice((128, 128, 64, 96, 32, 256, 160)),
              page=rng.choice((16, 32, 64, 64, 128)), seqs=_log(rng, 1, 64), tail=rng.choice((0, 0, 1, 5)),
              idle=rng.choice((0, 0, 3)))
    width = kv_heads * kw["head_dim"]  # channels of one token's keys
    if op == "append":
        q = _log(rng, 1, 1500)
        kw["seqs"] = min(kw["seqs"], max(1, 2000 // q))
        kw.update(q=(max(1, q // 3), q), kv=(q, q + _log(rng, 1, 900)), theta=rng.choice((10000.0, 500000.0, 0.0)),
                  bounds=rng.random() < 0.5)
        return _case("", "append", **kw)
    if op == "blocks":
        kv, picks = _log(rng, 50, 30000), _log(rng, 1, 64)
        kw["seqs"] = max(1, min(kw["seqs"], (32 * 20000 * 512) // (kv * width),
                                (64 * 32 * 64 * 512) // (picks * kw["page"] * width)))
        if rng.random() < 0.2:
            kw.update(seqs=1, q=(1, _log(rng, 2, 16)))
        kw.update(kv=(max(1, kv // 4), kv), picks=picks)
        return _case("", "blocks", **kw)
    form = rng.choice(("decode", "drafts", "prefix", "prompt"))
    kw["window"] = rng.choice((0, 0, 0, 129, 2048))
    if form == "prompt":
        q = _log(rng, 2, 1500)
        kv = q + rng.choice((0, 1, _log(rng, 1, 2000)))
        kw["seqs"] = max(1, min(kw["seqs"], (2048 * 3000 * 12 * 128) // (q * kv * kw["heads"] * kw["head_dim"])))
        kw.update(q=(max(1, q // 5), q), kv=(q, kv))
    elif form == "prefix":
        shared = _log(rng, 1, 8000 // kw["page"])
        kw.update(shared=shared, q=(1, rng.choice((1, 1, 3))), idle=0)
        kw["kv"] = (shared * kw["page"] + 3, shared * kw["page"] + 3 + _log(rng, 1, 600))
        kw["seqs"] = max(1, min(kw["seqs"], (64 * 16384 * 512) // (kw["kv"][1] * width * kw["q"][1] * group)))
    else:
        kv = _log(rng, 9, 30000)
        q = rng.choice((2, 3, 5, 9)) if form == "drafts" else 1
        kw["seqs"] = max(1, min(kw["seqs"], (32 * 20000 * 512) // (kv * width * q)))
        kw.update(q=(rng.choice((1, q)), q), kv=(max(1, kv // 4), kv))
    return _case("", "attention", **kw)


def _spread(lo, hi, u):
    return lo + min(hi - lo, int((hi - lo + 1) * u))


def _lengths(c):
    """New and cached tokens of every sequence, spread evenly over the case's ranges (the first at the top)."""
    q, kv = [], []
    for i in range(c["seqs"]):
        u, w = (1.0 - i * 0.6180339887498949) % 1.0 or 1.0, (1.0 - i * 0.7548776662466927) % 1.0 or 1.0
        n = _spread(c["q_min"], c["q_max"], u)
        length = 0
        if c["op"] != "verify":
            length = max(_spread(c["kv_min"], c["kv_max"], w), n)
            if c["idle"] and i % c["idle"] == c["idle"] - 1:
                n, length = 1, 0
        q.append(n)
        kv.append(length)
    return q, kv


def work(c):
    """Bytes that have to be read and written once, and the products' operations."""
    q, kv = _lengths(c)
    if c["op"] == "verify":
        rows, vocab = sum(q), c["vocab"]
        drafts = rows - c["seqs"]
        lists = 4 * (c["seqs"] + 1 + drafts + c["seqs"] + rows)  # starts, drafts, counts, ids
        if not c["temperature"]:
            return {"bytes": 4 * rows * vocab + lists, "flops": rows * vocab}
        # the draft's probabilities: one row of a sequence for what is left of the target's, one number of the others
        probs = 4 * (c["seqs"] * vocab + drafts) if c["probs"] else 0
        return {"bytes": 4 * rows * vocab + probs + lists + 4 * rows, "flops": 4 * rows * vocab}
    row = c["kv_heads"] * c["head_dim"] // 32 * 18  # one token's keys
    tokens = sum(n for n, length in zip(q, kv) if length)
    qbytes = 4 * tokens * c["heads"] * c["head_dim"]
    lists = 4 * (2 * c["seqs"] + sum(-(-length // c["page"]) for length in kv))
    if c["op"] == "append":
        kvbytes = 8 * tokens * c["kv_heads"] * c["head_dim"]  # keys and values in 32 bits: in, and read back
        b = 2 * (qbytes + kvbytes) + 4 * tokens * row + lists
        if c["bounds"]:  # fp16, read and written once for each page that gets a key
            b += 8 * c["kv_heads"] * c["head_dim"] * sum(-(-length // c["page"]) - (length - n) // c["page"]
                                                         for n, length in zip(q, kv) if length)
        flops = 3 * tokens * (c["heads"] + c["kv_heads"]) * c["head_dim"] if c["theta"] else 0
        return {"bytes": b, "flops": flops + 8 * tokens * c["kv_heads"] * c["head_dim"]}
    if c["op"] == "attention":
        shared = c["shared"] * c["page"]
        keys, flops, first = 0, 0, shared
        for n, length in zip(q, kv):
            if not length:
                continue
            begin = max(0, length - n + 1 - c["window"]) if c["window"] else 0
            keys += length - max(begin, shared)
            first = min(first, begin)
            seen = sum(min(p + 1, c["window"]) if c["window"] else p + 1 for p in range(length - n, length))
            flops += 4 * c["heads"] * c["head_dim"] * seen
        return {"bytes": 2 * qbytes + 2 * row * (keys + shared - first) + lists, "flops": flops}
    keys = 0
    for n, length in zip(q, kv):
        for p in range(length - n, length):
            if p >= 0:
                keys += min(c["picks"] - 1, p // c["page"]) * c["page"] + p % c["page"] + 1
    read = min(keys, sum(kv)) if max(q) > 1 else keys
    return {"bytes": 2 * qbytes + 2 * row * read + 4 * sum(q) * c["kv_heads"] * c["picks"] + lists,
            "flops": 4 * c["heads"] * c["head_dim"] * keys}


# ----------------------------------------------------------- the 4-bit format
def _quantise(x):
    """Numbers n in 0..15 and scales d of the blocks of 32 along the last axis (64 bits in).

    d takes the block's largest magnitude to n = 0 (a negative one where both signs reach it) in
    eight significant bits and steps of no less than 2^-24, at most 8160; n = floor(x / d + 8.5)
    within 0..15.  A block with a number that is not finite has the scale NaN."""
    x = x.view(*x.shape[:-1], -1, 32)
    low, high = x.amin(-1), x.amax(-1)
    d = torch.where(-low >= high, -low, -high) / 8.0
    step = torch.ldexp(torch.ones_like(d), (torch.frexp(d).exponent - 8).clamp(min=-24))
    d = ((d / step).round() * step).clamp(-8160.0, 8160.0)
    n = torch.floor(x / d.unsqueeze(-1) + 8.5).clamp(0.0, 15.0)
    n = torch.where(d.unsqueeze(-1) != 0, n, torch.full_like(n, 8.0))
    d = torch.where(x.isfinite().all(-1), d, torch.full_like(d, math.nan))
    return n.nan_to_num(8.0).flatten(-2), d


_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)  # channels of a word from its lowest four bits up


def _page_bytes(c):
    return c["page"] * (c["head_dim"] // 32) * 18


def _store(cache, c, where, off, n, d):
    """Numbers n [rows, kv_heads, head_dim] and scales d into slots `off` of pages `where`."""
    page, hd = c["page"], c["head_dim"]
    bits = n.to(torch.uint8).view(*n.shape[:-1], hd // 8, 8)[..., _ORDER].view(*n.shape[:-1], hd // 2, 2)
    split = page * hd // 2
    cache[..., :split].view(-1, c["kv_heads"], page, hd // 2)[where, :, off] = bits[..., 0] | bits[..., 1] << 4
    cache[..., split:].view(torch.float16).view(-1, c["kv_heads"], hd // 32, page)[where, :, :, off] = d.half()


def _numbers(cache, c):
    """n - 8 [pages, kv_heads, page, head_dim] (8 bits) and d [pages, kv_heads, page, head_dim / 32]."""
    page, hd = c["page"], c["head_dim"]
    split = page * hd // 2
    b = cache[..., :split].view(-1, c["kv_heads"], page, hd // 2)
    back = [_ORDER.index(j) for j in range(8)]
    n = torch.stack((b & 15, b >> 4), -1).view(-1, c["kv_heads"], page, hd // 8, 8)[..., back]
    d = cache[..., split:].view(torch.float16).view(-1, c["kv_heads"], hd // 32, page)
    return n.flatten(-2).to(torch.int8) - 8, d.transpose(-1, -2)


def _values(cache, c, dtype=torch.float32):
    """The cache's values [pages, kv_heads, page, head_dim]."""
    n, d = _numbers(cache, c)
    return (n.to(dtype).view(*d.shape, 32) * d.to(dtype).unsqueeze(-1)).flatten(-2)


# -------------------------------------------------------------------- inputs
def _prepare_verify(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, _ = _lengths(c)
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    tokens, vocab = starts[-1] + c["tail"], c["vocab"]
    # a few likely tokens over many unlikely ones
    logits = torch.randn((tokens, vocab), generator=g, device="cuda") * 2.5
    guess = logits + 0.5 * torch.randn((tokens, vocab), generator=g, device="cuda")  # a smaller model's
    probs = None
    if c["probs"]:
        probs = torch.softmax(guess / (c["temperature"] or 1.0), -1)
        noise = torch.rand((tokens, vocab), generator=g, device="cuda").clamp_(min=1e-30)
        drafts = (probs / -noise.log_()).argmax(-1)
    else:
        drafts = torch.where(torch.rand((tokens,), generator=g, device="cuda") < 0.8, logits.argmax(-1), guess.argmax(-1))
    ends = torch.tensor(starts[1:], device="cuda")
    drafts[ends - 1] = -1  # nothing was drafted behind a sequence's last row
    return {"case": c, "tokens": tokens, "max_rows": max(q), "logits": logits, "probs": probs, "drafts": drafts.int(),
            "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "accept_u": torch.rand((tokens,), generator=g, device="cuda"),
            "sample_u": torch.rand((c["seqs"],), generator=g, device="cuda"),
            "accepted": torch.zeros((c["seqs"],), dtype=torch.int32, device="cuda"),
            "ids": torch.full((tokens,), -2, dtype=torch.int32, device="cuda")}


def prepare(c, seed):
    if c["op"] == "verify":
        return _prepare_verify(c, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, kv = _lengths(c)
    kvh, hd, page = c["kv_heads"], c["head_dim"], c["page"]
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    tokens = starts[-1] + c["tail"]
    lens = torch.tensor(kv, dtype=torch.int32, device="cuda")
    max_pages = max(1, -(-max(kv) // page))
    # pages handed out in no order; entries behind a sequence's last page mean nothing
    own_pages = (lens.long() + page - 1) // page
    count = c["shared"] + int(sum(max(0, -(-length // page) - c["shared"]) for length in kv))
    num_pages = count + 2
    order = torch.randperm(num_pages, generator=g, device="cuda")[:count]
    col = torch.arange(max_pages, device="cuda")
    rest = (own_pages - c["shared"]).clamp(min=0)
    at = c["shared"] + (rest.cumsum(0) - rest)[:, None] + col[None, :] - c["shared"]
    at = torch.where(col[None, :] < c["shared"], col[None, :].expand_as(at), at)
    used = col[None, :] < own_pages[:, None]
    table = torch.where(used, order[at.clamp(0, count - 1)] if count else at, torch.full_like(at, -1)).int()
    st = {"case": c, "tokens": tokens, "max_q": max(q), "max_kv": max(kv), "max_pages": max_pages,
          "num_pages": num_pages, "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
          "kv_len": lens, "table": table.contiguous()}
    # keys spread differently in every channel, as projections give them
    lean = 0.5 * torch.randn((1, kvh, 1, hd), generator=g, device="cuda")
    for name in ("k", "v"):
        cache = st[name] = torch.empty((num_pages, kvh, _page_bytes(c)), dtype=torch.uint8, device="cuda")
        some = max(1, (1 << 25) // (kvh * page * hd))
        for p in range(0, num_pages, some):
            x = torch.randn((min(some, num_pages - p), kvh, page, hd), generator=g, device="cuda")
            n, d = _quantise((x + lean if name == "k" else x).double())
            where = torch.arange(p, p + len(x), device="cuda").repeat_interleave(page)
            off = torch.arange(page, device="cuda").repeat(len(x))
            _store(cache, c, where, off, *(y.transpose(1, 2).flatten(0, 1) for y in (n, d)))
    st["bounds"] = None
    if c["op"] == "append":
        st["qkv"] = torch.randn((tokens, (c["heads"] + 2 * kvh) * hd), generator=g, device="cuda")
        st["q_out"] = torch.zeros((tokens, c["heads"], hd), device="cuda")
        st["k_out"], st["v_out"] = (torch.zeros((tokens, kvh, hd), device="cuda") for _ in "kv")
        if c["bounds"]:
            k = _values(st["k"], c).half()
            st["bounds"] = torch.stack((k.amin(2), k.amax(2)), 2)
        return st
    st["q"] = torch.randn((tokens, c["heads"], hd), generator=g, device="cuda")
    if c["op"] == "blocks":  # any visible blocks, the token's own one among them, in ascending order
        st["picked"] = torch.full((tokens, kvh, c["picks"]), -1, dtype=torch.int32, device="cuda")
        seq, pos, live = _positions(st)
        own_block = torch.div(pos, page, rounding_mode="floor")
        score = torch.rand((tokens, kvh, max_pages), generator=g, device="cuda")
        score = torch.where(col == own_block[:, None, None], torch.full_like(score, 2.0), score)
        score = score.masked_fill(col > own_block[:, None, None], -1.0)
        best = score.topk(min(c["picks"], max_pages), -1)
        pick = torch.where(best.values >= 0, best.indices, torch.full_like(best.indices, 1 << 40)).sort(-1).values
        pick = torch.where(pick < (1 << 40), pick, torch.full_like(pick, -1)).int()
        st["picked"][:, :, :pick.shape[-1]] = torch.where(live[:, None, None], pick, torch.full_like(pick, -1))
    st["out"] = torch.zeros((tokens, c["heads"], hd), device="cuda")
    return st


# ---------------------------------------------------------------- plain forms
def _positions(st):
    """Sequence and position of every token row, and whether it is a token (not padding)."""
    t = torch.arange(st["tokens"], device="cuda")
    start, lens = st["q_start"].long(), st["kv_len"].long()
    seq = torch.searchsorted(start[1:].contiguous(), t, right=True)
    inside = seq < lens.numel()
    seq = seq.clamp(max=lens.numel() - 1)
    pos = lens[seq] - start[seq + 1] + t
    return seq, torch.where(inside, pos, torch.full_like(pos, -1)), inside & (pos >= 0)


def _padded(st, most):
    """Token rows as [sequence, place], and which of them are rows of the sequence."""
    start = st["q_start"].long()
    row = start[:-1, None] + torch.arange(most, device="cuda")[None, :]
    real = row < start[1:, None]
    return row.clamp(max=st["tokens"] - 1), real


def _rotate(x, pos, theta):
    """In 64 bits: a number next to a border of two 4-bit steps falls on the same side everywhere."""
    half = x.shape[-1] // 2
    x = x.double()
    if not theta:
        return x
    freq = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 * math.log(theta) / x.shape[-1]))
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos()[:, None, :], angle.sin()[:, None, :]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _plain_append(st, c):
    h, kvh, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    seq, pos, live = _positions(st)
    seq, pos, rows = seq[live], pos[live], st["qkv"][live]
    q, k, v = (x.reshape(len(pos), -1, hd) for x in rows.split((h * hd, kvh * hd, kvh * hd), 1))
    st["q_out"][live] = _rotate(q, pos, c["theta"]).float()
    where, off = st["table"].long()[seq, pos // page], pos % page
    held = {}
    for name, x in (("k", _rotate(k, pos, c["theta"])), ("v", v.double())):
        n, d = _quantise(x)
        _store(st[name], c, where, off, n, d)
        held[name] = ((n.float() - 8.0).view(*d.shape, 32) * d.float().unsqueeze(-1)).flatten(-2)
        st[name + "_out"][live] = held[name]
    if st["bounds"] is not None:
        # a page whose first slot is written begins anew
        low, high = st["bounds"][:, :, 0].float(), st["bounds"][:, :, 1].float()
        low[where[off == 0]], high[where[off == 0]] = math.inf, -math.inf
        low.index_reduce_(0, where, held["k"], "amin")
        high.index_reduce_(0, where, held["k"], "amax")
        st["bounds"].copy_(torch.stack((low, high), 2).half())


def _softmax_product(q, k, v, see, scale):
    """q [..., rows, hd], k and v [..., keys, hd], see [..., rows, keys]; rows that see nothing give zero."""
    s = (q @ k.transpose(-1, -2)) * scale
    s = s.masked_fill(~see, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, (e @ v) / total, torch.zeros((), device="cuda"))


def _plain_attention(st, c):
    h, kvh, hd, page, seqs = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["seqs"]
    group, keys = h // kvh, st["max_pages"] * page
    row, real = _padded(st, st["max_q"])
    lens = st["kv_len"].long()
    pos = lens[:, None] - (st["q_start"][1:] - st["q_start"][:-1]).long()[:, None] + torch.arange(st["max_q"], device="cuda")
    at = st["table"].long().clamp(0)
    j = torch.arange(keys, device="cuda")
    there = (j < lens[:, None])[:, None, :, None]
    k, v = (_values(st[x], c)[at].transpose(1, 2).reshape(seqs, kvh, keys, hd).masked_fill_(~there, 0.0) for x in "kv")
    see = j <= pos[:, :, None]
    if c["window"]:
        see = see & (j > pos[:, :, None] - c["window"])
    see = see[:, None, :, None, :].expand(seqs, 1, st["max_q"], group, keys).reshape(seqs, 1, -1, keys)
    q = st["q"][row].view(seqs, st["max_q"], kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, hd)
    o = _softmax_product(q, k, v, see, 1.0 / math.sqrt(hd))
    o = o.view(seqs, kvh, st["max_q"], group, hd).permute(0, 2, 1, 3, 4).reshape(seqs, st["max_q"], h, hd)
    st["out"][row[real]] = o[real]


def _plain_blocks(st, c):
    h, kvh, hd, page, t = c["heads"], c["kv_heads"], c["head_dim"], c["page"], st["tokens"]
    seq, pos, live = _positions(st)
    pick = st["picked"].long()
    at = st["table"].long()[seq[:, None, None], pick.clamp(0)].clamp(0)
    head = torch.arange(kvh, device="cuda")[None, :, None].expand_as(at)
    j = (pick[..., None] * page + torch.arange(page, device="cuda")).reshape(t, kvh, -1)
    see = (pick[..., None].expand(*pick.shape, page).reshape(t, kvh, -1) >= 0) & (j <= pos[:, None, None])
    k, v = (_values(st[x], c)[at, head].reshape(t, kvh, -1, hd).masked_fill_(~see[..., None], 0.0) for x in "kv")
    q = st["q"].view(t, kvh, h // kvh, hd)
    o = _softmax_product(q, k, v, see[:, :, None, :], 1.0 / math.sqrt(hd))
    inside = torch.arange(t, device="cuda") < st["q_start"][-1]
    st["out"].copy_(torch.where(inside[:, None, None], o.reshape(t, h, hd), st["out"]))


def _plain_verify(st, c):
    """A draft x of row i is taken where u q_i(x) < p_i(x).  The token behind the drafts taken is
    drawn from max(p - q, 0) of the row whose draft was not, or from p of the last row."""
    row, real = _padded(st, st["max_rows"])
    rows = real.sum(1)
    place = torch.arange(st["max_rows"], device="cuda")
    x = torch.where(place < rows[:, None] - 1, st["drafts"][row].long(), torch.full_like(row, -1))
    logits = st["logits"].masked_fill(st["logits"].isnan(), -math.inf).clamp(max=torch.finfo(torch.float32).max)
    most, first = logits.max(-1)
    if not c["temperature"]:
        first = torch.where(most > -math.inf, first, torch.full_like(first, -1))
        taken = (first[row] == x) & (x >= 0)
    else:
        # in 64 bits: u next to the border of two tokens falls on the same side everywhere
        p = ((logits.double() - most.double()[:, None]) / c["temperature"]).exp().nan_to_num(0.0)
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        at_x = row, x.clamp(min=0)
        q = st["probs"][at_x].double().clamp(min=0) if c["probs"] else torch.ones_like(p[at_x])
        taken = (st["accept_u"][row].double() * q < p[at_x]) & (x >= 0)
    count = taken.long().cumprod(1).sum(1)
    end = st["q_start"][:-1].long() + count
    if not c["temperature"]:
        token = first[end]
    else:
        left = p[end]
        short = count < rows - 1  # a draft was not taken
        if c["probs"]:
            rest = (left - st["probs"][end].double().clamp(min=0)).clamp(min=0)
        else:
            rest = left.scatter(1, x.gather(1, count[:, None]).clamp(min=0), 0.0)
        short = short & (rest.sum(1) > 0)
        left = torch.where(short[:, None], rest, left)
        total = left.cumsum(1)
        token = torch.searchsorted(total, st["sample_u"].double()[:, None] * total[:, -1:], right=True)[:, 0]
        last = c["vocab"] - 1 - (left.flip(1) > 0).int().argmax(1)
        token = torch.where(total[:, -1] > 0, torch.minimum(token, last), torch.full_like(token, -1))
    st["accepted"].copy_(count)
    ids = torch.where(place < count[:, None], x, torch.full_like(x, -1))
    ids = torch.where(place == count[:, None], token[:, None], ids)
    st["ids"][row[real]] = ids[real].int()


_PLAIN = {"append": _plain_append, "attention": _plain_attention, "blocks": _plain_blocks, "verify": _plain_verify}


# ------------------------------------------------------------- the library's
def _handle(st, c):
    """The descriptors and the workspace that a program keeps next to its cache."""
    root = os.path.join(os.getcwd(), "nedo.cpp_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import nedo_gpu

    lib = nedo_gpu.load()
    if c["op"] == "verify":
        drafts = nedo_gpu.Drafts(seqs=c["seqs"], rows=st["tokens"], max_rows=st["max_rows"], vocab=c["vocab"],
                                 row_start=st["q_start"].data_ptr(), logits=st["logits"].data_ptr(),
                                 draft_ids=st["drafts"].data_ptr(),
                                 draft_probs=st["probs"].data_ptr() if c["probs"] else None,
                                 accept_u=st["accept_u"].data_ptr(), sample_u=st["sample_u"].data_ptr())
        need = lib.verify_drafts_workspace(drafts)
        first = (drafts,)
    else:
        cache = nedo_gpu.KvCache(type=Q4_0, kv_heads=c["kv_heads"], head_dim=c["head_dim"], page_size=c["page"],
                                 num_pages=st["num_pages"], k=st["k"].data_ptr(), v=st["v"].data_ptr(),
                                 bounds=None if st["bounds"] is None else st["bounds"].data_ptr())
        batch = nedo_gpu.KvBatch(seqs=c["seqs"], tokens=st["tokens"], max_q_len=st["max_q"], max_kv_len=st["max_kv"],
                                 max_pages=st["max_pages"], shared_pages=c["shared"], q_start=st["q_start"].data_ptr(),
                                 kv_len=st["kv_len"].data_ptr(), page_table=st["table"].data_ptr())
        need = 0
        if c["op"] == "attention":
            need = lib.paged_attention_workspace(cache, batch, c["heads"], c["window"])
        elif c["op"] == "blocks":
            need = lib.block_attention_workspace(cache, batch, c["heads"], c["picks"])
        first = (cache, batch)
    space = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    st["handle"] = (lib, first, space, need)
    return st["handle"]


def _own(st, c):
    lib, first, space, need = st.get("handle") or _handle(st, c)
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "verify":
        lib.verify_drafts_dev(*first, c["temperature"], st["accepted"].data_ptr(), st["ids"].data_ptr(),
                              space.data_ptr(), need, stream)
        return
    scale = 1.0 / math.sqrt(c["head_dim"])
    if c["op"] == "append":
        lib.kv_append_dev(*first, c["heads"], st["qkv"].data_ptr(), c["theta"], st["q_out"].data_ptr(), stream)
        lib.kv_read_dev(*first, st["k_out"].data_ptr(), st["v_out"].data_ptr(), stream)
    elif c["op"] == "attention":
        lib.paged_attention_dev(*first, c["heads"], st["q"].data_ptr(), st["out"].data_ptr(), scale, c["window"],
                                space.data_ptr(), need, stream)
    else:
        lib.block_attention_dev(*first, c["heads"], st["q"].data_ptr(), st["picked"].data_ptr(), c["picks"],
                                st["out"].data_ptr(), scale, space.data_ptr(), need, stream)


def run(st):
    c = st["case"]
    if own:
        _own(st, c)
    else:
        _PLAIN[c["op"]](st, c)
    if c["op"] == "append":
        return {"q": st["q_out"], "k": st["k_out"], "v": st["v_out"], "bounds": st["bounds"]}
    return {"accepted": st["accepted"], "ids": st["ids"]} if c["op"] == "verify" else {"out": st["out"]}


# -------------------------------------------------------- the definition in 64 bits
def _held(x):
    """What a block-wise 4-bit cache makes of x [..., head_dim]: the definition, block by block."""
    out = torch.empty_like(x)
    for b in range(0, x.shape[-1], 32):
        y = x[..., b:b + 32]
        size = y.abs().amax(-1, keepdim=True)
        sign = torch.where((y == -size).any(-1, keepdim=True), 1.0, -1.0).double()
        d = size / 8
        unit = torch.pow(2.0, torch.floor(torch.log2(d.clamp(min=1e-300))))
        unit = torch.where(unit > d, unit / 2, torch.where(2 * unit <= d, 2 * unit, unit))
        grain = (unit / 128).clamp(min=2.0 ** -24)
        d = sign * torch.round(d / grain) * grain
        n = (torch.floor(y / d + 0.5)).clamp(-8, 7)
        out[..., b:b + 32] = torch.where(d != 0, n * d.clamp(-8160, 8160), torch.zeros_like(n))
    return out


def exact(c, seed):
    if c["op"] == "verify":  # whole numbers have no value in 64 bits
        return None
    st = prepare(c, seed)
    starts, lens, table = st["q_start"].tolist(), st["kv_len"].tolist(), st["table"].tolist()
    h, kvh, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    group, half = h // kvh, c["head_dim"] // 2

    def spin(x, pos):  # x [n, heads, hd] in 64 bits
        if not c["theta"]:
            return x
        z = torch.complex(x[..., :half], x[..., half:])
        i = torch.arange(half, device="cuda", dtype=torch.float64)
        angle = pos.double()[:, None] * torch.pow(torch.tensor(c["theta"], device="cuda", dtype=torch.float64), -2 * i / hd)
        z = z * torch.polar(torch.ones_like(angle), angle)[:, None, :]
        return torch.cat((z.real, z.imag), -1)

    if c["op"] == "append":
        q, k, v = (st[x + "_out"].double() for x in "qkv")
        low = high = None
        if c["bounds"]:
            low, high = st["bounds"][:, :, 0].double(), st["bounds"][:, :, 1].double()
        for s, length in enumerate(lens):
            n = starts[s + 1] - starts[s]
            if not length or not n:
                continue
            x = st["qkv"][starts[s]:starts[s + 1]].double()
            pos = torch.arange(length - n, length, device="cuda")
            q[starts[s]:starts[s + 1]] = spin(x[:, :h * hd].reshape(n, h, hd), pos)
            kk = _held(spin(x[:, h * hd:(h + kvh) * hd].reshape(n, kvh, hd), pos))
            k[starts[s]:starts[s + 1]] = kk
            v[starts[s]:starts[s + 1]] = _held(x[:, (h + kvh) * hd:].reshape(n, kvh, hd))
            if not c["bounds"]:
                continue
            for b in range((length - n) // page, (length - 1) // page + 1):
                a, z = max(b * page, length - n), min((b + 1) * page, length)
                p, took = table[s][b], slice(a - (length - n), z - (length - n))
                lo, hi = kk[took].amin(0), kk[took].amax(0)
                low[p] = lo if a % page == 0 else torch.minimum(low[p], lo)
                high[p] = hi if a % page == 0 else torch.maximum(high[p], hi)
        return {"q": q, "k": k, "v": v, "bounds": torch.stack((low, high), 2) if c["bounds"] else None}

    out = st["out"].double()
    for s, length in enumerate(lens):
        n = starts[s + 1] - starts[s]
        if not length or not n:
            continue
        pages = torch.tensor(table[s][:-(-length // page)], device="cuda")
        k, v = (_values(st[x][pages], c, torch.float64).transpose(0, 1).reshape(kvh, -1, hd)[:, :length] for x in "kv")
        pos = torch.arange(length - n, length, device="cuda")
        see = torch.arange(length, device="cuda")[None, :] <= pos[:, None]  # [n, length]
        if c["window"]:
            see &= torch.arange(length, device="cuda")[None, :] > pos[:, None] - c["window"]
        see = see[None].expand(kvh, n, length)
        if c["op"] == "blocks":
            pick = st["picked"][starts[s]:starts[s + 1]].long().transpose(0, 1)  # [kvh, n, picks]
            on = torch.zeros((kvh, n, -(-length // page) + 1), dtype=torch.bool, device="cuda")
            on.scatter_(2, torch.where(pick >= 0, pick, torch.full_like(pick, on.shape[2] - 1)), True)
            see = see & on[:, :, :-1].repeat_interleave(page, 2)[:, :, :length]
        for g in range(group):
            q = st["q"][starts[s]:starts[s + 1]].double().view(n, kvh, group, hd)[:, :, g].transpose(0, 1)
            score = torch.baddbmm(torch.zeros((), device="cuda", dtype=torch.float64), q, k.transpose(1, 2)) / math.sqrt(hd)
            score[~see] = -math.inf
            w = torch.softmax(score, -1)
            out[starts[s]:starts[s + 1]].view(n, kvh, group, hd)[:, :, g] = torch.bmm(w, v).transpose(0, 1)
    return {"out": out}
