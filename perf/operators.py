"""Cases of the 8-bit paged KV cache: append, attention (decode, verify, prompt, with the attention mass) and eviction.

The cache holds K and V as e4m3 codes in pages of `page` tokens, one power-of-two scale per (page, KV head) for K and
one for V.  Codes of 16 tokens form a tile of 16 * d bytes whose byte order is the tensor core's operand order (see
`_tile_index`); a page is its K tiles, then its V tiles.  `run` computes either the plain form in elementary torch
operations or, where `own` is set, the calls a user makes of the framework."""

import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
E_MIN, E_MAX = -120, 119          # exponents a scale may take


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one generated token of four sequences of an 8-KV-head model (the smallest write, latency)
        {"name": "append-token", "op": "append", "batch": 4, "kv": 8, "d": 128, "page": 16, "ctx": 32768, "rows": 1,
         "ragged": False, "src": "bf16"},
        # a prompt chunk of four sequences, the last one shorter, starting inside a page
        {"name": "append-prompt", "op": "append", "batch": 4, "kv": 8, "d": 128, "page": 16, "ctx": 8192, "rows": 512,
         "ragged": True, "src": "bf16"},
        # the first tokens of one short sequence of a small model: the smallest attention call
        {"name": "decode-short", "op": "attn", "batch": 1, "kv": 3, "group": 3, "d": 64, "page": 16, "ctx": 37, "T": 1,
         "out": "bf16", "mass": False},
        # plain decoding of four long sequences, Llama-3-8B heads
        {"name": "decode-32k", "op": "attn", "batch": 4, "kv": 8, "group": 4, "d": 128, "page": 16, "ctx": 32768, "T": 1,
         "out": "bf16", "mass": False},
        # one very long sequence: the key axis has to be split
        {"name": "decode-262k", "op": "attn", "batch": 1, "kv": 8, "group": 4, "d": 128, "page": 64, "ctx": 262144, "T": 1,
         "out": "bf16", "mass": False},
        # verification of 8 drafted tokens of 16 sequences of a small model
        {"name": "verify-2k", "op": "attn", "batch": 16, "kv": 3, "group": 3, "d": 64, "page": 16, "ctx": 2048, "T": 9,
         "out": "bf16", "mass": False},
        # decoding with the attention mass that eviction goes by, fp32 output, one query head per KV head
        {"name": "decode-mass", "op": "attn", "batch": 8, "kv": 12, "group": 1, "d": 64, "page": 32, "ctx": 8191, "T": 1,
         "out": "f32", "mass": True},
        # the first prompt chunk of an odd length
        {"name": "prompt-first", "op": "attn", "batch": 2, "kv": 12, "group": 1, "d": 64, "page": 16, "ctx": 301, "T": 301,
         "out": "bf16", "mass": False},
        # a later chunk of a long prompt
        {"name": "prompt-8k", "op": "attn", "batch": 2, "kv": 8, "group": 4, "d": 128, "page": 16, "ctx": 8192, "T": 512,
         "out": "bf16", "mass": False},
        # a short sequence pruned to half
        {"name": "evict-short", "op": "evict", "batch": 1, "kv": 3, "d": 64, "page": 16, "ctx": 301, "budget": 150,
         "sink": 4, "recent": 16},
        # four long sequences pruned to a quarter
        {"name": "evict-32k", "op": "evict", "batch": 4, "kv": 8, "d": 128, "page": 16, "ctx": 32768, "budget": 8192,
         "sink": 4, "recent": 64},
        # one very long sequence pruned to an eighth
        {"name": "evict-262k", "op": "evict", "batch": 1, "kv": 8, "d": 128, "page": 64, "ctx": 262144, "budget": 32768,
         "sink": 4, "recent": 256},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "attn", "evict"])
    d = rng.choice([64, 128])
    page = rng.choice([16, 32, 64])
    batch, kv = _log(rng, 1, 16), rng.randint(1, 12)
    top = min(262144, 536870912 // (2 * d * batch * kv))       # at most 0.5 GB of codes
    ctx = _log(rng, 1, top)
    c = {"op": op, "batch": batch, "kv": kv, "d": d, "page": page, "ctx": ctx}
    if op == "append":
        rows = min(ctx, _log(rng, 1, 512))
        c |= {"rows": rows, "ragged": rng.random() < 0.5, "src": rng.choice(["bf16", "f32"])}
    elif op == "evict":
        c["budget"] = max(1, int(ctx * rng.uniform(0.05, 1.1)))
        c |= {"sink": rng.choice([0, 1, 4]), "recent": rng.choice([0, 1, 16, 64])}
    else:
        group = rng.choice([1, 2, 3, 4, 7, 8])
        c["group"] = group
        if rng.random() < 0.7:                                  # decode and verify: up to 64 query rows a KV head
            c["T"] = min(ctx, _log(rng, 1, 64 // group))
            c |= {"out": rng.choice(["bf16", "f32"]), "mass": rng.random() < 0.4}
        else:                                                   # prompt chunks
            t = _log(rng, 64 // group + 1, 512)
            c["batch"] = batch = min(batch, 4)
            c["ctx"] = ctx = max(t, min(ctx, 250000000 // (batch * kv * group * t)))
            c |= {"T": t, "out": "bf16", "mass": False}
    return c


# ------------------------------------------------------------------ the byte order of a tile
def _tile_index(d):
    """(K, V) tables [16, d]: the byte of element (token, dim) inside a 16-token tile.  A tile is d / 32 blocks of 512
    bytes, 16 bytes a lane; lane 4 g + t of the matrix operand's row g holds columns 2t, 2t+1, 2t+8, 2t+9 of rows g and
    g + 8 (K: rows are tokens and columns dims; V: rows are dims and columns tokens)."""
    tok, dim = torch.arange(16)[:, None], torch.arange(d)[None, :]
    blk, r = dim // 32, dim % 32
    c = r % 16
    k = blk * 512 + ((tok % 8) * 4 + (c % 8) // 2) * 16 + ((r // 16) * 2 + tok // 8) * 4 + (c // 8) * 2 + c % 2
    v = blk * 512 + ((c % 8) * 4 + (tok % 8) // 2) * 16 + ((r // 16) * 2 + c // 8) * 4 + (tok // 8) * 2 + tok % 2
    return k, v


def _page_index(page, d):
    """[2, page, d]: the byte of (K or V, token, dim) inside a page of one head."""
    k, v = _tile_index(d)
    tile = torch.arange(page // 16)[:, None, None] * (16 * d)
    return torch.stack([(tile + k).reshape(page, d), page * d + (tile + v).reshape(page, d)])


# ------------------------------------------------------------------ inputs
def _storage(c, g, n_pages):
    """Random codes and scales in storage order: normal values under a scale of their own per page."""
    d, page, kv = c["d"], c["page"], c["kv"]
    codes = torch.empty((n_pages, kv, 2, page * d), dtype=torch.uint8, device=DEV)
    scale = torch.empty((n_pages, kv, 2), device=DEV)
    step = max(1, (1 << 26) // (kv * 2 * page * d))
    for i in range(0, n_pages, step):
        n = min(step, n_pages - i)
        x = torch.randn((n, kv, 2, page * d), generator=g, device=DEV)
        x *= torch.exp(0.5 * torch.randn((n, kv, 2, 1), generator=g, device=DEV))
        e = torch.ceil(torch.log2(x.abs().amax(-1) / 448.0)).int()
        scale[i:i + n] = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
        codes[i:i + n] = torch.ldexp(x, -e[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, scale


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    host = random.Random(seed)
    batch, kv, d, page, ctx = c["batch"], c["kv"], c["d"], c["page"], c["ctx"]
    pages = -(-ctx // page)
    n_src = batch * pages
    st = {"c": c, "index": _page_index(page, d).to(DEV)}
    if c["op"] == "evict":
        # the pruned copies go to fresh pages at the pool's end
        out_pages = -(-min(ctx, max(c["budget"], c["sink"] + c["recent"])) // page)
        st["codes"], st["scale"] = _storage(c, g, n_src + batch * out_pages)
        st["first_out"] = n_src
        order = torch.randperm(n_src, generator=g, device=DEV).to(torch.int32)
        st["table"] = order.view(batch, 1, pages).contiguous()
        st["out_table"] = (n_src + torch.randperm(batch * out_pages, generator=g, device=DEV)).to(torch.int32).view(
            batch, out_pages).contiguous()
        n = [ctx if b == 0 else host.randint(max(1, ctx - ctx // 8), ctx) for b in range(batch)]
        st["n"] = torch.tensor(n, dtype=torch.int32, device=DEV)
        st["budget"] = torch.full((batch,), c["budget"], dtype=torch.int32, device=DEV)
        # attention mass: a heavy tail, many small values, some never attended
        m = torch.exp(2.0 * torch.randn((batch, kv, pages * page), generator=g, device=DEV))
        m = torch.where(torch.rand(m.shape, generator=g, device=DEV) < 0.05, torch.zeros((), device=DEV), m)
        st["mass"] = m
        st["pos"] = torch.arange(pages * page, dtype=torch.int32, device=DEV).expand(batch, kv, -1).contiguous()
        return st
    # the last page takes writes of rows that are not there (plain form only) and is never in a table
    st["codes"], st["scale"] = _storage(c, g, n_src + 1)
    st["table"] = torch.randperm(n_src, generator=g, device=DEV).to(torch.int32).view(batch, 1, pages).contiguous()
    if c["op"] == "append":
        rows = c["rows"]
        n = [rows if not c["ragged"] or b == 0 else host.randint(0, rows) for b in range(batch)]
        e0 = [ctx - rows - (host.randint(0, min(page, ctx - rows)) if ctx > rows else 0) for _ in range(batch)]
        st["entry0"] = torch.tensor(e0, dtype=torch.int32, device=DEV)
        st["rows"] = torch.tensor(n, dtype=torch.int32, device=DEV)
        dt = torch.bfloat16 if c["src"] == "bf16" else torch.float32
        st["k"] = (2.0 * torch.randn((batch, rows, kv, d), generator=g, device=DEV)).to(dt)
        st["v"] = torch.randn((batch, rows, kv, d), generator=g, device=DEV).to(dt)
        return st
    T, group = c["T"], c["group"]
    n = [ctx if b == 0 else host.randint(max(T, ctx // 2), ctx) for b in range(batch)]
    st["entry0"] = torch.tensor([x - T for x in n], dtype=torch.int32, device=DEV)
    st["q"] = 1.5 * torch.randn((batch, T, kv * group, d), generator=g, device=DEV)
    if c["mass"]:
        st["mass"] = torch.rand((batch, kv, pages * page), generator=g, device=DEV)
    return st


# ------------------------------------------------------------------ the framework's calls
def _cache(st):
    """The user's cache object over the state's storage, made on the first pass and kept."""
    if "cache" not in st:
        package = str(Path(__file__).resolve().parent.parent / "draft-kv_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from draftkv import Q8KVCache
        st["cache"] = Q8KVCache.from_storage(st["codes"], st["scale"], st["table"], block_size=st["c"]["page"])
    return st["cache"]


def _run_own(st):
    c, cache = st["c"], _cache(st)
    if c["op"] == "append":
        cache.write(0, st["k"], st["v"], st["entry0"], n_rows=st["rows"])
        return {"codes": st["codes"][:-1].view(torch.float8_e4m3fn), "scale": st["scale"][:-1]}
    if c["op"] == "attn":
        out = cache.attention(0, st["q"], st["entry0"], mass=st.get("mass"),
                              out_dtype=torch.bfloat16 if c["out"] == "bf16" else torch.float32)
        return {"out": out, "mass": st["mass"]} if c["mass"] else {"out": out}
    kept, mass, pos = cache.evict_rows(0, st["n"], st["budget"], st["out_table"], mass=st["mass"], pos=st["pos"],
                                       sink=c["sink"], recent=c["recent"])
    at = st["first_out"]
    return {"codes": st["codes"][at:].view(torch.float8_e4m3fn), "scale": st["scale"][at:], "kept": kept, "mass": mass,
            "pos": pos}


# ------------------------------------------------------------------ the plain form
def _values(codes):
    return codes.view(torch.float8_e4m3fn).to(torch.float32)


def _exponent(amax):
    """Smallest e with amax 2^-e <= 448 = 0.875 2^9."""
    f, k = torch.frexp(amax)
    e = torch.where(f <= 0.875, k - 9, k - 8)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _pow2(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _encode(x, e):
    """e4m3 codes of x 2^-e (|x| 2^-e <= 448 but for the largest fp32 values), rounded to nearest even."""
    return (x * _pow2(-e)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_append(st):
    c = st["c"]
    batch, kv, d, page, rows = c["batch"], c["kv"], c["d"], c["page"], c["rows"]
    codes, scale, index = st["codes"], st["scale"], st["index"]
    touched = (rows + page - 2) // page + 1                     # pages a run of rows can reach
    e0, n = st["entry0"].long(), st["rows"].long()
    pg = e0[:, None] // page + torch.arange(touched, device=DEV)                        # [B, P]
    ent = pg[..., None] * page + torch.arange(page, device=DEV)                         # [B, P, page]
    old = ent < e0[:, None, None]
    new = ~old & (ent < (e0 + n)[:, None, None])
    live = new.any(-1)
    pages = st["table"][:, 0].long()
    pid = torch.where(live, pages.gather(1, pg.clamp(max=pages.shape[1] - 1)), codes.shape[0] - 1)
    cur = codes[pid]                                                                    # [B, P, kv, 2, page*d]
    row = (ent - e0[:, None, None]).clamp(0, rows - 1)                                  # source row of an entry
    x = torch.stack([st["k"], st["v"]], 3).float()                                      # [B, rows, kv, 2, d]
    x = x[torch.arange(batch, device=DEV)[:, None, None], row]                          # [B, P, page, kv, 2, d]
    x = x.permute(0, 1, 3, 4, 2, 5)                                                     # [B, P, kv, 2, page, d]
    is_new, is_old = new[:, :, None, None, :, None], old[:, :, None, None, :, None]
    e_new = _exponent(torch.where(is_new, x.abs(), 0.0).amax((-1, -2)))                 # [B, P, kv, 2]
    e_old = (torch.frexp(scale[pid])[1] - 1)
    has_old = (old.any(-1) & live)[:, :, None, None]
    e = torch.where(has_old, torch.maximum(e_old, e_new), e_new)
    flat = index.reshape(1, 1, 1, 2, page * d).expand(cur.shape[0], touched, kv, 2, -1)
    flat = flat - torch.tensor([0, page * d], device=DEV)[:, None]                      # byte inside K or V
    was = cur.gather(-1, flat).view(batch, touched, kv, 2, page, d)
    again = _encode(_values(was), (e - e_old)[..., None, None])
    put = torch.where(is_new, _encode(x, e[..., None, None]), torch.where(is_old, again, was))
    cur = cur.scatter(-1, flat, put.reshape(cur.shape))
    codes[pid] = cur
    scale[pid] = torch.where(live[:, :, None, None], _pow2(e), scale[pid])
    return {"codes": codes[:-1].view(torch.float8_e4m3fn), "scale": scale[:-1]}


def _gathered(st, n):
    """K and V of every sequence's first n entries in fp32: 2 x [B, kv, n, d]."""
    c = st["c"]
    page, d, kv, batch = c["page"], c["d"], c["kv"], c["batch"]
    pid = st["table"][:, 0, : -(-n // page)].long()
    x = st["codes"][pid][..., 0, :], st["codes"][pid][..., 1, :]
    s = st["scale"][pid]
    out = []
    for i in (0, 1):
        at = st["index"][i] - i * page * d
        v = _values(x[i])[..., at.reshape(-1)].view(batch, -1, kv, page, d) * s[..., i, None, None]
        out.append(v.transpose(1, 2).reshape(batch, kv, -1, d)[:, :, :n])
    return out


def _plain_attn(st):
    c = st["c"]
    batch, kv, d, T, group, ctx = c["batch"], c["kv"], c["d"], c["T"], c["group"], c["ctx"]
    k, v = _gathered(st, ctx)
    q = st["q"].view(batch, T, kv, group, d).permute(0, 2, 1, 3, 4).reshape(batch, kv, T * group, d)
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / d ** 0.5)
    last = (st["entry0"][:, None] + torch.arange(T, device=DEV)).repeat_interleave(group, 1)     # [B, T*group]
    dead = torch.arange(ctx, device=DEV) > last[:, None, :, None]
    s = s.masked_fill(dead, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, v).view(batch, kv, T, group, d).permute(0, 2, 1, 3, 4).reshape(batch, T, kv * group, d)
    res = {"out": out.to(torch.bfloat16 if c["out"] == "bf16" else torch.float32)}
    if c["mass"]:
        st["mass"][:, :, :ctx] += p.sum(2)
        res["mass"] = st["mass"]
    return res


def _plain_evict(st):
    c = st["c"]
    batch, kv, d, page = c["batch"], c["kv"], c["d"], c["page"]
    sink, recent = c["sink"], c["recent"]
    cap = st["mass"].shape[-1]
    ld = st["out_table"].shape[1] * page
    n = st["n"].long()[:, None, None]
    m = torch.minimum(n, torch.clamp(st["budget"].long()[:, None, None], min=sink + recent))
    j = torch.arange(cap, device=DEV)
    inf = torch.full((), float("inf"), device=DEV)
    key = torch.where((j < sink) | (j >= n - recent), inf, st["mass"])
    key = torch.where(j < n, key, -inf)
    rank = torch.argsort(key, dim=-1, stable=True)              # drop order: ascending (mass, index)
    order = torch.empty_like(rank).scatter_(-1, rank, j.expand_as(rank).contiguous())
    keep = order >= cap - m
    slot = torch.where(keep, keep.long().cumsum(-1) - 1, ld)
    kept = torch.full((batch, kv, ld + 1), -1, dtype=torch.int64, device=DEV)
    kept.scatter_(-1, slot.clamp(max=ld), torch.where(keep, j, -1))
    kept = kept[..., :ld]
    live = kept >= 0
    src = kept.clamp(min=0)
    w = min(ld, cap)
    mass = torch.zeros_like(st["mass"])
    mass[..., :w] = torch.where(live, st["mass"].gather(-1, src), 0.0)[..., :w]
    pos = torch.full_like(st["pos"], -1)
    pos[..., :w] = torch.where(live, st["pos"].gather(-1, src), -1)[..., :w]
    # the kept rows' values, written to the fresh pages as an append would
    pid = st["table"][:, 0].long()
    bb, hh = torch.arange(batch, device=DEV)[:, None, None], torch.arange(kv, device=DEV)[None, :, None]
    at = pid[bb, src // page]                                   # [B, kv, ld]
    out_id = st["out_table"].long().view(batch, 1, -1)          # [B, 1, out pages]
    n_out = out_id.shape[-1]
    for i in (0, 1):
        byte = (st["index"][i] - i * page * d)[src % page]      # [B, kv, ld, d]
        x = _values(st["codes"][at[..., None], hh[..., None], i, byte]) * st["scale"][at, hh, i][..., None]
        x = torch.where(live[..., None], x, 0.0).view(batch, kv, n_out, page, d)
        e = _exponent(x.abs().amax((-1, -2)))
        put = _encode(x, e[..., None, None]).view(batch, kv, n_out, page * d)
        there = live.view(batch, kv, n_out, page)
        flat = (st["index"][i] - i * page * d).reshape(-1)
        was = st["codes"][out_id, hh, i]                        # [B, kv, out pages, page*d]
        mask = there[..., None].expand(-1, -1, -1, -1, d).reshape(batch, kv, n_out, page * d)
        new = was.clone()
        new[..., flat] = torch.where(mask, put, was[..., flat])
        st["codes"][out_id, hh, i] = new
        st["scale"][out_id, hh, i] = torch.where(there.any(-1), _pow2(e), st["scale"][out_id, hh, i])
    first = st["first_out"]
    return {"codes": st["codes"][first:].view(torch.float8_e4m3fn), "scale": st["scale"][first:],
            "kept": kept.to(torch.int32), "mass": mass, "pos": pos}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attn": _plain_attn, "evict": _plain_evict}[state["c"]["op"]](state)


# ------------------------------------------------------------------ the work that cannot be avoided
def work(case):
    c = case
    batch, kv, d, ctx, page = c["batch"], c["kv"], c["d"], c["ctx"], c["page"]
    row = 2 * d                                                 # bytes of one entry's codes (K and V) in one head
    if c["op"] == "append":
        n = batch * c["rows"] * kv
        elem = 2 if c["src"] == "bf16" else 4
        return {"bytes": n * (row * elem + row) + n / page * 8, "flops": 2 * n * row}
    if c["op"] == "evict":
        m = batch * kv * min(ctx, max(c["budget"], c["sink"] + c["recent"]))
        return {"bytes": batch * kv * ctx * 4 + m * (2 * row + 4 + 8 + 8), "flops": m * row}
    T, heads = c["T"], kv * c["group"]
    mean = 0.75 if batch > 1 else 1.0                           # sequences end between half and the whole length
    n = batch * ctx * mean
    pairs = batch * heads * (T * ctx * mean - T * (T - 1) / 2) if ctx * mean > T else batch * heads * T * (T + 1) / 2
    q = batch * T * heads * d
    moved = n * kv * (row + 8 / page) + q * 4 + q * (2 if c["out"] == "bf16" else 4)
    if c["mass"]:
        moved += n * kv * 8
    return {"bytes": moved, "flops": 4 * d * max(pairs, 1)}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_pow2(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e.int())


def _exact_values(codes, scale, index):
    """[pages..., 2, page, d] in 64 bits from the codes' bits: sign, exponent (bias 7), fraction of 3 bits."""
    page, d = index.shape[1:]
    b = codes.reshape(codes.shape[:-2] + (2 * page * d,))[..., index.reshape(-1)].to(torch.int64)
    e, f = (b >> 3) & 15, b & 7
    mag = torch.where(e == 0, f.double() / 8 * 2.0 ** -6, (1 + f.double() / 8) * _exact_pow2((e - 7).double()))
    v = torch.where(b >= 128, -mag, mag).view(codes.shape[:-2] + (2, page, d))
    return v * scale.double()[..., None, None]


def _exact_round(q):
    """Nearest e4m3 value of q (|q| <= 448), ties to even: 3 fraction bits, exponents from -6."""
    mag = q.abs().clamp(min=2.0 ** -40)
    e = torch.floor(torch.log2(mag))
    e = torch.where(_exact_pow2(e) > mag, e - 1, torch.where(_exact_pow2(e + 1) <= mag, e + 1, e)).clamp(min=-6)
    step = _exact_pow2(e - 3)
    return torch.round(q / step) * step


def _exact_exponent(amax):
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448))
    e = torch.where(448 * _exact_pow2(e - 1) >= amax, e - 1, e)
    e = torch.where(448 * _exact_pow2(e) < amax, e + 1, e)
    return torch.where(amax > 0, e, torch.full_like(e, float(E_MIN))).clamp(E_MIN, E_MAX)


def exact(case, seed):
    st = prepare(case, seed)
    c = st["c"]
    batch, kv, d, page = c["batch"], c["kv"], c["d"], c["page"]
    index, table = st["index"], st["table"][:, 0].tolist()
    if c["op"] == "append":
        return _exact_append(st, c, index, table)
    if c["op"] == "evict":
        return _exact_evict(st, c, index, table)
    T, group, ctx = c["T"], c["group"], c["ctx"]
    out = torch.zeros((batch, T, kv * group, d), dtype=torch.float64, device=DEV)
    mass = st["mass"].double() if c["mass"] else None
    e0 = st["entry0"].tolist()
    for b in range(batch):
        n = e0[b] + T
        pid = torch.tensor(table[b][: -(-n // page)], device=DEV)
        for h in range(kv):
            kvv = _exact_values(st["codes"][pid, h], st["scale"][pid, h], index)
            k, v = kvv[:, 0].reshape(-1, d)[:n], kvv[:, 1].reshape(-1, d)[:n]
            q = st["q"][b, :, h * group:(h + 1) * group].double().reshape(T * group, d)
            for r in range(0, T * group, 512):
                qr = q[r:r + 512]
                s = qr @ k.T / np.sqrt(d)
                t = torch.arange(r, r + qr.shape[0], device=DEV) // group
                s[torch.arange(n, device=DEV)[None] > (e0[b] + t)[:, None]] = float("-inf")
                p = torch.softmax(s, -1)
                o = p @ v
                out[b, t, h * group + torch.arange(r, r + qr.shape[0], device=DEV) % group] = o
                if mass is not None:
                    mass[b, h, :n] += p.sum(0)
    return {"out": out, "mass": mass} if c["mass"] else {"out": out}


def _as_codes(st, index, first, last):
    """The pool's codes as values [pages, kv, 2, page, d] in 64 bits (scales left out)."""
    cd = st["codes"][first:last]
    return _exact_values(cd, torch.ones(cd.shape[:-1], device=DEV), index)


def _stored(vals, index):
    """Values [pages, kv, 2, page, d] laid out as the pool stores them."""
    out = torch.empty(vals.shape[:2] + (vals.shape[2] * vals.shape[3] * vals.shape[4],), dtype=torch.float64, device=DEV)
    out[..., index.reshape(-1)] = vals.reshape(out.shape)
    return out.view(vals.shape[:3] + (-1,))


def _exact_append(st, c, index, table):
    batch, kv, page = c["batch"], c["kv"], c["page"]
    touched = [(b, p) for b, (e0, n) in enumerate(zip(st["entry0"].tolist(), st["rows"].tolist())) if n > 0
               for p in range(e0 // page, -(-(e0 + n) // page))]
    if len(touched) > 8192:
        return None
    # untouched codes keep their values, which fp32 holds exactly, as it does what e4m3 rounding gives
    codes = st["codes"][:-1].view(torch.float8_e4m3fn).to(torch.float32)
    scale = st["scale"][:-1].double()
    for b, p in touched:
        pid = table[b][p]
        e0, n = int(st["entry0"][b]), int(st["rows"][b])
        lo = max(e0 - p * page, 0)
        r0 = p * page + lo - e0
        cnt = min(n - r0, page - lo)
        vals = _exact_values(st["codes"][pid:pid + 1], torch.ones((1, kv, 2), device=DEV), index)[0]
        for i, x in ((0, st["k"]), (1, st["v"])):
            x = x[b, r0:r0 + cnt].double()                       # [cnt, kv, d]
            e = _exact_exponent(x.abs().amax((0, 2)))            # [kv]
            if lo:
                eo = torch.round(torch.log2(scale[pid, :, i]))
                e = torch.maximum(e, eo)
                vals[:, i, :lo] = _exact_round(vals[:, i, :lo] * _exact_pow2(eo - e)[:, None, None])
            y = (x * _exact_pow2(-e)[None, :, None]).clamp(-448, 448)
            vals[:, i, lo:lo + cnt] = _exact_round(y).transpose(0, 1)
            scale[pid, :, i] = _exact_pow2(e)
        codes[pid] = _stored(vals[None], index)[0].to(codes.dtype)
    return {"codes": codes, "scale": scale}


def _exact_evict(st, c, index, table):
    batch, kv, d, page = c["batch"], c["kv"], c["d"], c["page"]
    first, ld = st["first_out"], st["out_table"].shape[1] * c["page"]
    cap = st["mass"].shape[-1]
    if batch * kv * ld * d > 1 << 27:
        vals_ok = False
    else:
        vals_ok = True
        out = _as_codes(st, index, first, st["codes"].shape[0])
        scale = st["scale"][first:].double()
    kept = np.full((batch, kv, ld), -1, dtype=np.int32)
    mass = torch.zeros((batch, kv, cap), dtype=torch.float64, device=DEV)
    pos = torch.full((batch, kv, cap), -1, dtype=torch.int32, device=DEV)
    allm = st["mass"].cpu().numpy()
    for b in range(batch):
        n = int(st["n"][b])
        m = min(n, max(int(st["budget"][b]), c["sink"] + c["recent"]))
        pid = torch.tensor(table[b], device=DEV)
        for h in range(kv):
            idx = np.arange(n)
            free = idx[(idx >= c["sink"]) & (idx < n - c["recent"])]
            drop = free[np.lexsort((free, allm[b, h, free]))][: n - m]
            ks = np.setdiff1d(idx, drop)
            kept[b, h, :len(ks)] = ks
            at = torch.from_numpy(ks).to(DEV)
            mass[b, h, :len(ks)] = st["mass"][b, h, at].double()
            pos[b, h, :len(ks)] = st["pos"][b, h, at]
            if not vals_ok:
                continue
            src = pid[at // page]
            rows = _exact_rows(st, index, src, h, at % page)      # [m, 2, d]
            for p in range(-(-len(ks) // page)):
                o = int(st["out_table"][b, p]) - first
                x = rows[p * page:(p + 1) * page]
                for i in (0, 1):
                    e = _exact_exponent(x[:, i].abs().max())
                    out[o, h, i, :len(x)] = _exact_round(x[:, i] * _exact_pow2(-e))
                    scale[o, h, i] = _exact_pow2(e)
    return {"codes": _stored(out, index) if vals_ok else None, "scale": scale if vals_ok else None,
            "kept": torch.from_numpy(kept), "mass": mass, "pos": pos}


def _exact_rows(st, index, src, h, slot):
    """Dequantised rows [m, 2, d] of one head: page src[i], row slot[i]."""
    byte = index[:, slot].transpose(0, 1)                         # [m, 2, d]
    flat = st["codes"][:, h].reshape(st["codes"].shape[0], -1)
    b = flat[src[:, None, None], byte].to(torch.int64)
    e, f = (b >> 3) & 15, b & 7
    mag = torch.where(e == 0, f.double() / 8 * 2.0 ** -6, (1 + f.double() / 8) * _exact_pow2((e - 7).double()))
    return torch.where(b >= 128, -mag, mag) * st["scale"][src, h].double()[..., None]
