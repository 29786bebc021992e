"""Paged key/value cache operators of the decode path, as measured cases.

Four entry points of the library (include/nedo_gpu.h) that work on one paged
cache ([pages][kv_heads][page_size][head_dim], F16 or F32):

  append     nedo_gpu_kv_append_dev       q|k|v rows in, rotated queries out, rotated
                                          keys and values into their pages, key bounds
                                          (channel-wise minimum and maximum) per page
  attention  nedo_gpu_paged_attention_dev softmax attention of a ragged batch over its
                                          pages, causal, optionally a sliding window and
                                          a prefix that all sequences share
  select     nedo_gpu_block_select_dev    for each query token and KV head the pages whose
                                          key bounds promise the largest scores
  blocks     nedo_gpu_block_attention_dev attention over the selected pages only

``run`` computes them in plain torch operations, or through the library where
``own`` is true.  ``exact`` is the definition in 64 bits, one sequence at a time.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f16": torch.float16, "f32": torch.float32}
CODES = {"f16": 1, "f32": 0}  # GGUF tensor type codes


# --------------------------------------------------------------------- cases
def _case(name, op, type="f16", heads=12, kv_heads=4, head_dim=128, page=64, seqs=1, q=(1, 1), kv=(512, 512),
          idle=0, tail=0, theta=10000.0, bounds=False, window=0, shared=0, picks=0):
    """One case: `seqs` sequences of q[0]..q[1] new tokens and kv[0]..kv[1] cached
    tokens (the new ones included), every `idle`-th of them an unused slot of a
    padded batch (one token, nothing cached), `tail` rows behind the last token,
    the first `shared` pages common to all."""
    c = {"op": op, "type": type, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
         "seqs": seqs, "q_min": q[0], "q_max": q[1], "kv_min": kv[0], "kv_max": kv[1], "idle": idle, "tail": tail,
         "theta": theta, "bounds": bounds, "window": window, "shared": shared, "picks": picks}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token of one conversation: the call whose latency every generated token pays
        _case("append one token", "append", kv=(513, 513), bounds=True),
        # three prompts of odd lengths in one batch
        _case("append prompts", "append", seqs=3, q=(317, 1025), kv=(1025, 2047), bounds=True),
        # one token of each of 128 conversations into an F32 cache, some slots unused
        _case("append batch f32", "append", type="f32", kv_heads=12, seqs=128, kv=(3, 1021), idle=7, tail=3),
        # the decode pass of one conversation at position 512
        _case("attention one token", "attention", kv=(513, 513)),
        # long conversations served together: the cache is what is read
        _case("attention long batch", "attention", seqs=32, kv=(8191, 32768)),
        # one token of each of 64 conversations behind one long system prompt
        _case("attention shared prefix", "attention", seqs=64, kv=(16384 + 33, 16384 + 701), shared=256),
        # a prompt taken in whole, with the sliding window of the model's configuration
        _case("attention prompt", "attention", seqs=2, q=(1711, 2048), kv=(2048, 4096), window=2048),
        # the F32 cache of the decode pass (every head its own keys), a window, unused slots
        _case("attention batch f32", "attention", type="f32", kv_heads=12, seqs=24, kv=(700, 4096), window=2048,
              idle=9, tail=2),
        # which pages of one long conversation the next token looks at
        _case("select one token", "select", kv=(8200, 8200), picks=16),
        # the same for a batch of long conversations
        _case("select batch", "select", seqs=48, kv=(16001, 65536), picks=32),
        # attention over what was selected, one conversation
        _case("blocks one token", "blocks", kv=(8200, 8200), picks=16),
        # and for a batch, 32 of up to 512 pages each
        _case("blocks batch", "blocks", seqs=64, kv=(16001, 32768), picks=32),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))) - 0.5))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "attention", "select", "blocks"))
    kv_heads, group = rng.choice(((4, 3), (12, 1), (2, 4), (1, 8), (3, 2), (8, 4), (2, 16), (1, 5)))
    kw = dict(type=rng.choice(("f16", "f16", "f32")), kv_heads=kv_heads, heads=kv_heads * group,
              head_dim=rng.choice((128, 128, 64, 96, 40, 256)), page=rng.choice((16, 32, 64, 64, 128)),
              seqs=_log(rng, 1, 64), tail=rng.choice((0, 0, 1, 5)), idle=rng.choice((0, 0, 3)))
    width = kv_heads * kw["head_dim"] * (4 if kw["type"] == "f32" else 2)  # bytes of one token's keys
    if op == "append":
        q = _log(rng, 1, 1500)
        kw["seqs"] = min(kw["seqs"], max(1, 4000 // q))
        kw.update(q=(max(1, q // 3), q), kv=(q, q + _log(rng, 1, 900)), theta=rng.choice((10000.0, 500000.0, 0.0)),
                  bounds=rng.random() < 0.5)
        return _case("", "append", **kw)
    if op == "select":
        kv = _log(rng, 50, 60000)
        kw["seqs"] = max(1, min(kw["seqs"], (48 * 40000 * 4 * 128 * 2) // (kv * width)))
        if rng.random() < 0.2:  # a chunk of a prompt that selects for each of its tokens
            kw.update(seqs=min(kw["seqs"], 2), q=(1, _log(rng, 2, 40)))
            kv = min(kv, 8000)
        kw.update(kv=(max(1, kv // 4), kv), picks=_log(rng, 1, 64))
        return _case("", "select", **kw)
    if op == "blocks":
        kv, picks = _log(rng, 50, 30000), _log(rng, 1, 64)
        kw["seqs"] = max(1, min(kw["seqs"], (32 * 20000 * 4 * 128 * 2) // (kv * width),
                                (64 * 32 * 64 * 4 * 128 * 2) // (picks * kw["page"] * width)))
        if rng.random() < 0.2:
            kw.update(seqs=1, q=(1, _log(rng, 2, 16)))
        kw.update(kv=(max(1, kv // 4), kv), picks=picks)
        return _case("", "blocks", **kw)
    form = rng.choice(("decode", "decode", "prefix", "prompt"))
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
        kw["seqs"] = max(1, min(kw["seqs"], (64 * 16384 * 4 * 128 * 2) // (kw["kv"][1] * width * kw["q"][1] * group)))
    else:
        kv = _log(rng, 1, 30000)
        kw["seqs"] = max(1, min(kw["seqs"], (32 * 20000 * 4 * 128 * 2) // (kv * width)))
        kw.update(q=(1, rng.choice((1, 1, 2))), kv=(max(1, kv // 4), kv))
    return _case("", "attention", **kw)


def _lengths(c):
    """New and cached tokens of every sequence, spread evenly over the case's ranges (the first at the top)."""
    q, kv = [], []
    for i in range(c["seqs"]):
        u, w = (1.0 - i * 0.6180339887498949) % 1.0 or 1.0, (1.0 - i * 0.7548776662466927) % 1.0 or 1.0
        n = c["q_min"] + min(c["q_max"] - c["q_min"], int((c["q_max"] - c["q_min"] + 1) * u))
        length = c["kv_min"] + min(c["kv_max"] - c["kv_min"], int((c["kv_max"] - c["kv_min"] + 1) * w))
        length = max(length, n)
        if c["idle"] and i % c["idle"] == c["idle"] - 1:
            n, length = 1, 0
        q.append(n)
        kv.append(length)
    return q, kv


def _visible(c, pos):
    """Keys that a query at `pos` sees."""
    return 0 if pos < 0 else min(pos + 1, c["window"]) if c["window"] else pos + 1


def work(c):
    """Bytes that have to be read and written once, and the products' operations."""
    q, kv = _lengths(c)
    size = 4 if c["type"] == "f32" else 2
    row = c["kv_heads"] * c["head_dim"] * size  # one token's keys
    tokens = sum(n for n, length in zip(q, kv) if length)
    qbytes = 4 * tokens * c["heads"] * c["head_dim"]
    pages = [-(-length // c["page"]) for length in kv]
    lists = 4 * (2 * c["seqs"] + sum(pages))
    if c["op"] == "append":
        b = 4 * tokens * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"] + qbytes + 2 * tokens * row + lists
        if c["bounds"]:  # read and written once for each page that gets a key
            b += 4 * row * sum(-(-length // c["page"]) - (length - n) // c["page"] for n, length in zip(q, kv) if length)
        return {"bytes": b, "flops": 3 * tokens * (c["heads"] + c["kv_heads"]) * c["head_dim"] if c["theta"] else 0}
    if c["op"] == "attention":
        shared = c["shared"] * c["page"]
        keys, flops, first = 0, 0, shared
        for n, length in zip(q, kv):
            if not length:
                continue
            begin = max(0, length - n + 1 - c["window"]) if c["window"] else 0
            keys += length - max(begin, shared)
            first = min(first, begin)
            flops += 4 * c["heads"] * c["head_dim"] * sum(_visible(c, p) for p in range(length - n, length))
        return {"bytes": 2 * qbytes + 2 * row * (keys + shared - first) + lists, "flops": flops}
    if c["op"] == "select":
        out = 4 * sum(q) * c["kv_heads"] * c["picks"]
        blocks = sum(n * p for n, p in zip(q, pages))
        return {"bytes": qbytes + 2 * row * sum(pages) + lists + out,
                "flops": 4 * blocks * c["kv_heads"] * c["head_dim"]}
    keys = 0
    for n, length in zip(q, kv):
        for p in range(length - n, length):
            if p >= 0:
                full = min(c["picks"] - 1, p // c["page"])
                keys += full * c["page"] + p % c["page"] + 1
    read = min(keys, sum(kv)) if max(q) > 1 else keys
    return {"bytes": 2 * qbytes + 2 * row * read + 4 * sum(q) * c["kv_heads"] * c["picks"] + lists,
            "flops": 4 * c["heads"] * c["head_dim"] * keys}


# -------------------------------------------------------------------- inputs
def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[c["type"]]
    q, kv = _lengths(c)
    seqs, kvh, hd, page = c["seqs"], c["kv_heads"], c["head_dim"], c["page"]
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
    shape = (num_pages, kvh, page, hd)
    # keys spread differently in every channel, as projections give them
    lean = torch.randn((1, kvh, 1, hd), generator=g, device="cuda")
    if c["op"] == "select":  # the bounds are all that it reads
        mid = torch.randn((num_pages, kvh, hd), generator=g, device="cuda") * 0.4 + lean[:, :, 0]
        half = 1.5 + torch.rand((num_pages, kvh, hd), generator=g, device="cuda")
        st["bounds"] = torch.stack((mid - half, mid + half), 2).to(dt)
        st["k"] = st["v"] = torch.zeros((1,), dtype=dt, device="cuda")
    else:
        st["k"] = torch.randn(shape, generator=g, device="cuda", dtype=dt).add_((0.5 * lean).to(dt))
        st["v"] = torch.randn(shape, generator=g, device="cuda", dtype=dt)
        st["bounds"] = None
    width = (c["heads"] + 2 * kvh) * hd
    if c["op"] == "append":
        st["qkv"] = torch.randn((tokens, width), generator=g, device="cuda")
        st["q_out"] = torch.zeros((tokens, c["heads"], hd), device="cuda")
        if c["bounds"]:
            st["bounds"] = torch.stack((st["k"].amin(2), st["k"].amax(2)), 2)
        return st
    st["q"] = torch.randn((tokens, c["heads"], hd), generator=g, device="cuda")
    if c["op"] in ("select", "blocks"):
        st["picked"] = torch.full((tokens, kvh, c["picks"]), -1, dtype=torch.int32, device="cuda")
    if c["op"] == "blocks":  # any visible blocks, the token's own one among them, in ascending order
        seq, pos, live = _positions(st)
        own_block = torch.div(pos, page, rounding_mode="floor")
        score = torch.rand((tokens, kvh, max_pages), generator=g, device="cuda")
        score = torch.where(col == own_block[:, None, None], torch.full_like(score, 2.0), score)
        score = score.masked_fill(col > own_block[:, None, None], -1.0)
        best = score.topk(min(c["picks"], max_pages), -1)
        pick = torch.where(best.values >= 0, best.indices, torch.full_like(best.indices, 1 << 40)).sort(-1).values
        pick = torch.where(pick < (1 << 40), pick, torch.full_like(pick, -1)).int()
        st["picked"][:, :, :pick.shape[-1]] = torch.where(live[:, None, None], pick, torch.full_like(pick, -1))
    if c["op"] in ("attention", "blocks"):
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


def _padded(st):
    """Token rows as [sequence, place], and which of them are tokens of the sequence."""
    start = st["q_start"].long()
    row = start[:-1, None] + torch.arange(st["max_q"], device="cuda")[None, :]
    real = row < start[1:, None]
    return row.clamp(max=st["tokens"] - 1), real


def _rotate(x, pos, theta):
    half = x.shape[-1] // 2
    if not theta:
        return x
    freq = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 * math.log(theta) / x.shape[-1]))
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _plain_append(st, c):
    h, kvh, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    seq, pos, live = _positions(st)
    seq, pos, rows = seq[live], pos[live], st["qkv"][live]
    q, k, v = (x.reshape(len(pos), -1, hd) for x in rows.split((h * hd, kvh * hd, kvh * hd), 1))
    q, k = _rotate(q, pos, c["theta"]), _rotate(k, pos, c["theta"]).to(st["k"].dtype)
    st["q_out"][live] = q
    where, off = st["table"].long()[seq, pos // page], pos % page
    st["k"][where, :, off] = k
    st["v"][where, :, off] = v.to(st["v"].dtype)
    if st["bounds"] is not None:
        # a page whose first slot is written begins anew
        low, high = st["bounds"][:, :, 0].float(), st["bounds"][:, :, 1].float()
        low[where[off == 0]], high[where[off == 0]] = math.inf, -math.inf
        low.index_reduce_(0, where, k.float(), "amin")
        high.index_reduce_(0, where, k.float(), "amax")
        st["bounds"].copy_(torch.stack((low, high), 2).to(st["bounds"].dtype))


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
    row, real = _padded(st)
    lens = st["kv_len"].long()
    pos = lens[:, None] - (st["q_start"][1:] - st["q_start"][:-1]).long()[:, None] + torch.arange(st["max_q"], device="cuda")
    at = st["table"].long().clamp(0)
    j = torch.arange(keys, device="cuda")
    there = (j < lens[:, None])[:, None, :, None]
    k, v = (x[at].transpose(1, 2).reshape(seqs, kvh, keys, hd).float().masked_fill_(~there, 0.0) for x in (st["k"], st["v"]))
    see = j <= pos[:, :, None]
    if c["window"]:
        see = see & (j > pos[:, :, None] - c["window"])
    see = see[:, None, :, None, :].expand(seqs, 1, st["max_q"], group, keys).reshape(seqs, 1, -1, keys)
    q = st["q"][row].view(seqs, st["max_q"], kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, hd)
    o = _softmax_product(q, k, v, see, 1.0 / math.sqrt(hd))
    o = o.view(seqs, kvh, st["max_q"], group, hd).permute(0, 2, 1, 3, 4).reshape(seqs, st["max_q"], h, hd)
    st["out"][row[real]] = o[real]


def _plain_select(st, c):
    kvh, hd, page = c["kv_heads"], c["head_dim"], c["page"]
    row, real = _padded(st)
    q = st["q"][row].double().view(c["seqs"], st["max_q"], kvh, -1, hd)
    up, down = q.clamp(min=0).sum(3).transpose(1, 2), q.clamp(max=0).sum(3).transpose(1, 2)
    b = st["bounds"][st["table"].long().clamp(0)].double().permute(0, 2, 3, 4, 1)  # [seqs, kvh, 2, hd, pages]
    score = (up @ b[:, :, 1] + down @ b[:, :, 0]).transpose(1, 2)  # [seqs, q, kvh, pages]
    pos = st["kv_len"].long()[:, None] - (st["q_start"][1:] - st["q_start"][:-1]).long()[:, None] + torch.arange(st["max_q"], device="cuda")
    last = torch.div(pos, page, rounding_mode="floor")[:, :, None, None]
    n = torch.arange(st["max_pages"], device="cuda")
    score = torch.where(n == last, torch.full_like(score, math.inf), score).masked_fill(n > last, -math.inf)
    first = score.sort(dim=-1, descending=True, stable=True).indices[..., :c["picks"]]
    none = 1 << 40
    first = torch.where(first <= last, first, torch.full_like(first, none)).sort(-1).values
    first = torch.where(first < none, first, torch.full_like(first, -1)).int()
    st["picked"].fill_(-1)
    st["picked"][row[real], :, :first.shape[-1]] = first[real]


def _plain_blocks(st, c):
    h, kvh, hd, page, t = c["heads"], c["kv_heads"], c["head_dim"], c["page"], st["tokens"]
    seq, pos, live = _positions(st)
    pick = st["picked"].long()
    at = st["table"].long()[seq[:, None, None], pick.clamp(0)].clamp(0)
    head = torch.arange(kvh, device="cuda")[None, :, None].expand_as(at)
    j = (pick[..., None] * page + torch.arange(page, device="cuda")).reshape(t, kvh, -1)
    see = (pick[..., None].expand(*pick.shape, page).reshape(t, kvh, -1) >= 0) & (j <= pos[:, None, None])
    k, v = (x[at, head].reshape(t, kvh, -1, hd).float().masked_fill_(~see[..., None], 0.0) for x in (st["k"], st["v"]))
    q = st["q"].view(t, kvh, h // kvh, hd)
    o = _softmax_product(q, k, v, see[:, :, None, :], 1.0 / math.sqrt(hd))
    inside = torch.arange(t, device="cuda") < st["q_start"][-1]
    st["out"].copy_(torch.where(inside[:, None, None], o.reshape(t, h, hd), st["out"]))


_PLAIN = {"append": _plain_append, "attention": _plain_attention, "select": _plain_select, "blocks": _plain_blocks}


# ------------------------------------------------------------- the library's
def _handle(st, c):
    """The descriptors and the workspace that a program keeps next to its cache."""
    root = os.path.join(os.getcwd(), "nedo.cpp_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import nedo_gpu

    lib = nedo_gpu.load()
    cache = nedo_gpu.KvCache(type=CODES[c["type"]], kv_heads=c["kv_heads"], head_dim=c["head_dim"],
                             page_size=c["page"], num_pages=st["num_pages"], k=st["k"].data_ptr(), v=st["v"].data_ptr(),
                             bounds=None if st["bounds"] is None else st["bounds"].data_ptr())
    batch = nedo_gpu.KvBatch(seqs=c["seqs"], tokens=st["tokens"], max_q_len=st["max_q"], max_kv_len=st["max_kv"],
                             max_pages=st["max_pages"], shared_pages=c["shared"], q_start=st["q_start"].data_ptr(),
                             kv_len=st["kv_len"].data_ptr(), page_table=st["table"].data_ptr())
    need = 0
    if c["op"] == "attention":
        need = lib.paged_attention_workspace(cache, batch, c["heads"], c["window"])
    elif c["op"] == "blocks":
        need = lib.block_attention_workspace(cache, batch, c["heads"], c["picks"])
    space = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    st["handle"] = (lib, cache, batch, space, need)
    return st["handle"]


def _own(st, c):
    lib, cache, batch, space, need = st.get("handle") or _handle(st, c)
    stream = torch.cuda.current_stream().cuda_stream
    scale = 1.0 / math.sqrt(c["head_dim"])
    if c["op"] == "append":
        lib.kv_append_dev(cache, batch, c["heads"], st["qkv"].data_ptr(), c["theta"], st["q_out"].data_ptr(), stream)
    elif c["op"] == "attention":
        lib.paged_attention_dev(cache, batch, c["heads"], st["q"].data_ptr(), st["out"].data_ptr(), scale, c["window"],
                                space.data_ptr(), need, stream)
    elif c["op"] == "select":
        lib.block_select_dev(cache, batch, c["heads"], st["q"].data_ptr(), c["picks"], st["picked"].data_ptr(), stream)
    else:
        lib.block_attention_dev(cache, batch, c["heads"], st["q"].data_ptr(), st["picked"].data_ptr(), c["picks"],
                                st["out"].data_ptr(), scale, space.data_ptr(), need, stream)


def run(st):
    c = st["case"]
    if own:
        _own(st, c)
    else:
        _PLAIN[c["op"]](st, c)
    if c["op"] == "append":
        return {"q": st["q_out"], "k": st["k"], "v": st["v"], "bounds": st["bounds"]}
    return {"blocks": st["picked"]} if c["op"] == "select" else {"out": st["out"]}


# -------------------------------------------------------- the definition in 64 bits
def exact(c, seed):
    st = prepare(c, seed)
    starts, lens, table = st["q_start"].tolist(), st["kv_len"].tolist(), st["table"].tolist()
    h, kvh, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    group, half = h // kvh, c["head_dim"] // 2
    if c["op"] == "select":  # whole numbers have no value in 64 bits
        return None

    def spin(x, pos):  # x [n, heads, hd] in 64 bits
        if not c["theta"]:
            return x
        z = torch.complex(x[..., :half], x[..., half:])
        i = torch.arange(half, device="cuda", dtype=torch.float64)
        angle = pos.double()[:, None] * torch.pow(torch.tensor(c["theta"], device="cuda", dtype=torch.float64), -2 * i / hd)
        z = z * torch.polar(torch.ones_like(angle), angle)[:, None, :]
        return torch.cat((z.real, z.imag), -1)

    if c["op"] == "append":
        q, k, v = st["q_out"].double(), st["k"].double(), st["v"].double()
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
            kk = spin(x[:, h * hd:(h + kvh) * hd].reshape(n, kvh, hd), pos)
            vv = x[:, (h + kvh) * hd:].reshape(n, kvh, hd)
            for b in range((length - n) // page, (length - 1) // page + 1):
                a, z = max(b * page, length - n), min((b + 1) * page, length)
                p, took = table[s][b], slice(a - (length - n), z - (length - n))
                k[p, :, a % page:a % page + z - a] = kk[took].transpose(0, 1)
                v[p, :, a % page:a % page + z - a] = vv[took].transpose(0, 1)
                if c["bounds"]:
                    kept = kk[took].to(TYPES[c["type"]]).double()
                    lo, hi = kept.amin(0), kept.amax(0)
                    low[p] = lo if a % page == 0 else torch.minimum(low[p], lo)
                    high[p] = hi if a % page == 0 else torch.maximum(high[p], hi)
        return {"q": q, "k": k, "v": v, "bounds": torch.stack((low, high), 2) if c["bounds"] else None}

    out = st["out"].double()
    for s, length in enumerate(lens):
        n = starts[s + 1] - starts[s]
        if not length or not n:
            continue
        pages = torch.tensor(table[s][:-(-length // page)], device="cuda")
        k, v = (x[pages].transpose(0, 1).reshape(kvh, -1, hd)[:, :length].double() for x in (st["k"], st["v"]))
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
