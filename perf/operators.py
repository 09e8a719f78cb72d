"""The operators of the packed key/value cache, as cases that can be prepared, run, timed and compared.

A packed cache holds a key or value head of a token as 4-bit codes: every 32 neighbouring numbers x share a zero point z and a
step s, both bfloat16, and the cache's number is z + s n with n in 0 .. 15

    z = the largest bfloat16 <= min x,   s = bfloat16((max x - z) * (1 / 15)),   n = clamp(rint((x - z) * (1 / s)), 0, 15)

(s below the smallest normal float32 counts as 0, and n is 0 then; a token whose key or value has a group with a z or s that is not
finite keeps a NaN key and a value of zeros in that head).  A page of `page` tokens is, per key/value head, the key codes, the
key parameters, the value codes and the value parameters of its tokens (`_code_orders` says which nibble is which number): 40 bytes per
32 numbers of a head where bfloat16 takes 128.

    store     queries and keys rotated, keys and values packed and stored at their slots, and those slots read back as numbers
    single    attention of one new token per request over its packed keys and values: a decode step's
    prompt    the same for portions of prompts of several tokens, with or without earlier tokens in the cache
    copy      pages copied inside the pool in every layer's entry: what forking requests that share a prompt has to move

The head counts are those of the 8b, 3b and 1b presets (32, 24 and 32 query heads, 8 key/value heads, 128, 128 and 64 numbers a head).
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

SHAPES = {"8b": (32, 8, 128), "3b": (24, 8, 128), "1b": (32, 8, 64)}       # query heads, key/value heads, numbers a head
LAYERS = {"8b": 32, "3b": 28, "1b": 16}
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _case(name, op, shape, **fields):
    base = {"op": op, "shape": shape, "dtype": "bfloat16", "page": 16}
    more = {"pairs": 1, "pool": 64, "packed": True} if op == "copy" else \
        {"batch": 1, "prompt": 1, "context": 0, "spread": 0.0, "window": 0}
    return {"name": name, **base, **more, **fields} if name else {**base, **more, **fields}


def listed():
    return [
        # the store of a decode step: eight rows, latency alone
        _case("store-8b-b8", "store", "8b", batch=8, context=8192),
        # of a prompt
        _case("store-8b-2048", "store", "8b", prompt=2048),
        # of an odd prompt in the engine's other type
        _case("store-1b-f32-777", "store", "1b", dtype="float32", prompt=777),
        # one user at a prompt: the least work there is
        _case("single-1b-b1-500", "single", "1b", context=500),
        # eight long conversations: the headline batch
        _case("single-8b-b8-8192", "single", "8b", batch=8, context=8192),
        # a server's batch of uneven contexts, three query heads to a key/value head
        _case("single-3b-b37", "single", "3b", batch=37, context=600, spread=0.7),
        # two long documents
        _case("single-8b-b2-32k", "single", "8b", batch=2, context=32000, spread=0.02, page=32),
        # a whole prompt
        _case("prompt-8b-2048", "prompt", "8b", prompt=2048),
        # a portion of a long prompt, odd lengths
        _case("prompt-3b-511-over-7777", "prompt", "3b", prompt=511, context=7777),
        # short prompts of uneven lengths in the engine's other type
        _case("prompt-1b-f32-ragged", "prompt", "1b", dtype="float32", batch=5, prompt=133, spread=0.8),
        # three more answers to one prompt: the page that every answer goes on writing, in every layer
        _case("copy-8b-3", "copy", "8b", pairs=3),
        # the same for a batch of requests with answers of their own, in a cache of bfloat16 pages
        _case("copy-1b-bf16-96", "copy", "1b", pairs=96, pool=256, packed=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["store", "single", "single", "prompt", "prompt", "copy"])
    shape, page = rng.choice(list(SHAPES)), rng.choice([8, 16, 16, 32, 64])
    if op == "copy":
        packed = rng.random() < 0.5
        return _case("", op, shape, pairs=_log(rng, 1, 96), pool=256, packed=packed, page=16 if not packed else page,
                     dtype=rng.choice(["bfloat16", "float32"]) if not packed and shape == "1b" else "bfloat16")
    f32 = rng.random() < 0.3
    f = {"page": page, "dtype": "float32" if f32 else "bfloat16", "spread": round(rng.uniform(0.0, 0.8), 2)}
    if op == "store":
        f["batch"] = _log(rng, 1, 32)
        f["prompt"] = max(1, _log(rng, 1, 2048 if not f32 else 1024) // f["batch"])
        f["context"] = rng.randint(0, 4000)
    elif op == "single":
        f["batch"] = _log(rng, 1, 64 if not f32 else 16)
        f["context"] = _log(rng, 1, min(32000, (60000 if not f32 else 6000) // f["batch"]))
        f["window"] = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
    else:
        f["batch"] = _log(rng, 1, 8)
        f["prompt"] = max(2, _log(rng, 8, 2048 if not f32 else 400) // f["batch"])
        f["context"] = rng.choice([0, _log(rng, 1, (8000 if not f32 else 600) // f["batch"])])
        f["window"] = rng.choice([0, 0, 0, _log(rng, 16, 1024)])
    return _case("", op, shape, **f)


# ---- what a case consists of -----------------------------------------------------------------------------------------
def _lengths(case):
    """[(tokens in the cache before, new tokens)] of the requests; the lengths belong to the case, not to the seed."""
    rng = random.Random(case["batch"] * 100003 + case["context"] * 31 + case["prompt"])
    out = []
    for _ in range(case["batch"]):
        f = 1.0 + case["spread"] * rng.uniform(-1.0, 1.0)
        new = 1 if case["op"] == "single" or case["prompt"] == 1 else max(1, round(case["prompt"] * f))
        out.append((max(0, round(case["context"] * f)), new))
    return out


def _code_orders(dim):
    """For the nibbles of a key row and of a value row, low nibble of a byte first: the number each one belongs to.  With
    groups = dim / 32: key word j * groups + g (four bytes, j < 4) holds the numbers 32 g + 8 j .. + 7, the even ones in its
    low half, the odd ones in its high half; value half-word c * groups + g (two bytes, c < 8) holds the numbers
    32 g + 8 (c // 2) + (c % 2) + {0, 2, 4, 6}."""
    groups = dim // 32
    j, g, i = torch.meshgrid(torch.arange(4), torch.arange(groups), torch.arange(8), indexing="ij")
    key = 32 * g + 8 * j + 2 * (i % 4) + i // 4
    c, g, i = torch.meshgrid(torch.arange(8), torch.arange(groups), torch.arange(4), indexing="ij")
    value = 32 * g + 8 * (c // 2) + c % 2 + 2 * i
    return key.reshape(-1), value.reshape(-1)


def _floor_bf16(x):
    """The largest bfloat16 that is not above x (float32)."""
    bits = x.view(torch.int32)
    up = (bits < 0) & ((bits & 0xFFFF) != 0)
    return ((bits & -65536) + up.int() * 65536).view(torch.float32)


def _pack(x):
    """Codes (uint8 [..., dim]), steps and zero points (float32 [..., dim / 32]) of the rows of x (float32)."""
    xg = x.unflatten(-1, (-1, 32))
    z = _floor_bf16(xg.amin(-1).contiguous())
    s = ((xg.amax(-1) - z) * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)).bfloat16().float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    r = torch.where(s > 0, torch.ones_like(s) / s, torch.zeros_like(s))
    n = ((xg - z[..., None]) * r[..., None]).round().clamp(0, 15).to(torch.uint8)
    return n.flatten(-2), s, z


def _rows(codes, s, z, order):
    """(code bytes, parameter bytes) of rows: [n, heads, dim / 2] and [n, heads, dim / 8] uint8."""
    n = codes[..., order].unflatten(-1, (-1, 2))
    par = torch.stack([s.bfloat16(), z.bfloat16()], dim=-1).contiguous()
    return n[..., 0] | (n[..., 1] << 4), par.flatten(-2).view(torch.uint8)


def _regions(pages, kv, page, dim):
    """The four byte regions of a layer's pages [pages, bytes], as views [pages, kv, page, bytes]: key codes, key parameters,
    value codes, value parameters."""
    per = pages.view(pages.shape[0], kv, page * (dim // 32) * 40)
    at, out = 0, []
    for width in (dim // 2, dim // 8, dim // 2, dim // 8):
        out.append(per[..., at:at + page * width].unflatten(-1, (page, width)))
        at += page * width
    return out


def _put(pages, slots, key, value, kv, page, dim, orders):
    """Packs key and value rows [n, kv, dim] (float32) into the pages at `slots`."""
    kc, ks, kz = _pack(key)
    vc, vs, vz = _pack(value)
    fine = torch.isfinite(ks).all(-1) & torch.isfinite(kz).all(-1) & torch.isfinite(vs).all(-1) & torch.isfinite(vz).all(-1)
    nan, zero = torch.full_like(ks, math.nan), torch.zeros_like(ks)
    keep = fine[..., None]
    rows = _rows(torch.where(keep, kc, 0), torch.where(keep, ks, nan), torch.where(keep, kz, nan), orders[0]) + \
        _rows(torch.where(keep, vc, 0), torch.where(keep, vs, zero), torch.where(keep, vz, zero), orders[1])
    at, off = slots // page, slots % page
    a, b, c, d = _regions(pages, kv, page, dim)
    a[at, :, off], b[at, :, off], c[at, :, off], d[at, :, off] = rows


def _numbers(codes, par, dim, order):
    """float32 [..., dim] of code and parameter bytes."""
    n = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    x = torch.empty_like(n)
    x[..., order] = n
    sz = par.contiguous().view(torch.bfloat16).float().unflatten(-1, (dim // 32, 2))
    return (x.unflatten(-1, (-1, 32)).float() * sz[..., :1] + sz[..., 1:]).flatten(-2)


def _tables(case, seed, gen, dev):
    """Lengths, page ids (a pool in random order, one spare page at its end), and the index arrays of a step."""
    page, lens = case["page"], _lengths(case)
    need = [-(-(c + n) // page) for c, n in lens]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(int(seed)))
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    new = torch.tensor([n for _, n in lens])
    request = torch.repeat_interleave(torch.arange(len(lens)), new)
    first = torch.cumsum(new, 0) - new
    position = torch.arange(int(new.sum())) - first[request] + torch.tensor([c for c, _ in lens])[request]
    slots = table[request, position // page].long() * page + position % page
    return lens, sum(need) + 1, table.to(dev), request.int().to(dev), position.int().to(dev), slots.int().to(dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    heads, kv, dim = SHAPES[case["shape"]]
    dtype, page, op = DTYPES[case["dtype"]], case["page"], case["op"]
    state = {"op": op, "heads": heads, "kv": kv, "dim": dim, "page": page}
    if op == "copy":
        # a pool of pages for every layer; the pages copied are anywhere in it, none is read and written
        entries, pool = LAYERS[case["shape"]], case["pool"]
        if case["packed"]:
            pages = torch.randint(0, 256, (entries, pool, kv * page * (dim // 32) * 40), generator=gen, device=dev, dtype=torch.uint8)
        else:
            pages = torch.randn(entries, pool, 2, kv, page, dim, generator=gen, device=dev).to(dtype)
        at = random.Random(int(seed)).sample(range(pool), 2 * case["pairs"])
        pairs = list(zip(at[::2], at[1::2]))
        return dict(state, pages=pages, pairs=pairs)
    lens, pool, table, request, position, slots = _tables(case, seed, gen, dev)
    tokens = request.shape[0]
    orders = tuple(o.to(dev) for o in _code_orders(dim))
    pages = torch.zeros(pool, kv * page * (dim // 32) * 40, dtype=torch.uint8, device=dev)
    # keys as projections give them: a few numbers of every head larger than the rest, the same ones for all tokens
    loud = 1.0 + 5.0 * (torch.rand(kv, dim, generator=gen, device=dev) < 0.05)
    state.update(pages=pages, orders=orders, dtype=dtype)
    if op == "store":
        qkv = torch.randn(tokens, heads + 2 * kv, dim, generator=gen, device=dev)
        qkv[:, heads:heads + kv] *= loud
        inv = 10000.0 ** (-torch.arange(0, dim, 2, device=dev, dtype=torch.float64) / dim)
        angle = position.double()[:, None] * inv
        return dict(state, qkv=qkv.flatten(1).to(dtype), cos=angle.cos().float(), sin=angle.sin().float(), slots=slots,
                    q_out=torch.empty(tokens, heads * dim, dtype=dtype, device=dev),
                    numbers=torch.empty(tokens, 2, kv, dim, dtype=torch.float32, device=dev))
    for b, (before, new) in enumerate(lens):        # everything up to the step's last token is in the cache
        p = torch.arange(before + new, device=dev)
        at = table[b].long()[p // page] * page + p % page
        k = torch.randn(before + new, kv, dim, generator=gen, device=dev) * loud
        v = torch.randn(before + new, kv, dim, generator=gen, device=dev)
        _put(pages, at, k.to(dtype).float(), v.to(dtype).float(), kv, page, dim, orders)
    q = torch.randn(tokens, heads * dim, generator=gen, device=dev)
    # queries of requests side by side, padded to the longest: row of every (request, place), and its place back
    new = torch.tensor([n for _, n in lens])
    first = torch.cumsum(new, 0) - new
    places = (first[:, None] + torch.arange(int(new.max()))).clamp(max=tokens - 1).to(dev)
    place_of = (torch.arange(tokens, device=dev) - first.to(dev)[request.long()])
    meta = SimpleNamespace(block_table=table, token_request=request, positions=position, query_lens=[n for _, n in lens],
                           seq_lens_host=[c + n for c, n in lens], attention_plan=None)
    return dict(state, q=q.to(dtype), meta=meta, window=case["window"], places=places, place_of=place_of,
                out=torch.empty(tokens, heads * dim, dtype=dtype, device=dev))


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _plain_store(st):
    heads, kv, dim, page = st["heads"], st["kv"], st["dim"], st["page"]
    x = st["qkv"].float().unflatten(1, (-1, dim))
    rot, v = x[:, :heads + kv], x[:, heads + kv:]
    a, b = rot.chunk(2, dim=-1)
    c, s = st["cos"][:, None], st["sin"][:, None]
    rot = torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(st["dtype"])
    slots = st["slots"].long()
    _put(st["pages"], slots, rot[:, heads:].float(), v, kv, page, dim, st["orders"])
    kc, kp, vc, vp = (r[slots // page, :, slots % page] for r in _regions(st["pages"], kv, page, dim))
    numbers = torch.stack([_numbers(kc, kp, dim, st["orders"][0]), _numbers(vc, vp, dim, st["orders"][1])], dim=1)
    return rot[:, :heads].flatten(1), numbers


def _plain_attend(st):
    heads, kv, dim, page, meta = st["heads"], st["kv"], st["dim"], st["page"], st["meta"]
    table = meta.block_table.long()
    kc, kp, vc, vp = (r[table].transpose(2, 3).flatten(1, 2) for r in _regions(st["pages"], kv, page, dim))     # [B, C, kv, bytes]
    keys = _numbers(kc, kp, dim, st["orders"][0]).transpose(1, 2)                                               # [B, kv, C, dim]
    values = _numbers(vc, vp, dim, st["orders"][1]).transpose(1, 2)
    q = st["q"].float()[st["places"]].unflatten(-1, (kv, heads // kv, dim))                                     # [B, T, kv, group, dim]
    batch, longest = q.shape[:2]
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)                                                                  # [B, kv, group * T, dim]
    scores = (q @ keys.transpose(2, 3)).mul_(1.0 / math.sqrt(dim)).unflatten(2, (-1, longest))
    at, key = meta.positions[st["places"]], torch.arange(keys.shape[2], device=q.device)
    seen = key <= at[..., None]
    if st["window"]:
        seen &= key > at[..., None] - st["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    p /= p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ values).unflatten(2, (-1, longest))                                                  # [B, kv, group, T, dim]
    o = o.permute(0, 3, 1, 2, 4).flatten(2)
    return o[meta.token_request.long(), st["place_of"]].to(st["dtype"])


def _plain_copy(st):
    src, dst = (torch.tensor(x, device=st["pages"].device) for x in zip(*st["pairs"]))
    st["pages"][:, dst] = st["pages"][:, src]
    return st["pages"]


def _kernels():
    from iitj_llm_coopt_b200 import kernels
    return kernels.load()


def run(st):
    op, heads, kv, dim = st["op"], st["heads"], st["kv"], st["dim"]
    if not own:
        return {"store": _plain_store, "single": _plain_attend, "prompt": _plain_attend, "copy": _plain_copy}[op](st)
    k = _kernels()
    if op == "copy":
        return k.copy_pages(st["pages"], st["pairs"])
    if op == "store":
        q = k.rope_store_kv4(st["qkv"], (st["cos"], st["sin"]), st["slots"], st["pages"], heads, kv, dim, dim, q_out=st["q_out"])
        return q, k.kv4_read(st["pages"], st["slots"], st["numbers"], kv, dim)
    return k.attention_kv4(st["q"], st["pages"], st["meta"], st["out"], heads, kv, dim, window=st["window"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    heads, kv, dim = SHAPES[case["shape"]]
    size = 2 if case["dtype"] == "bfloat16" else 4
    packed = kv * (dim // 32) * 40                          # bytes of a token in a layer
    if case["op"] == "copy":
        token = packed if case["packed"] else 2 * kv * dim * size
        return {"bytes": 2 * case["pairs"] * LAYERS[case["shape"]] * case["page"] * token, "flops": 0}
    lens = _lengths(case)
    tokens = sum(n for _, n in lens)
    if case["op"] == "store":
        rows = (2 * heads + 2 * kv) * dim * size            # queries in and out, keys and values in
        return {"bytes": tokens * (rows + dim * 4 + 2 * packed + 2 * kv * dim * 4), "flops": tokens * 6 * (heads + kv) * dim}
    window, pairs, read = case["window"], 0, 0
    for before, new in lens:
        read += min(before + new, window + new - 1) if window else before + new
        pairs += sum(min(before + i + 1, window) if window else before + i + 1 for i in range(new))
    return {"bytes": read * packed + 2 * tokens * heads * dim * size, "flops": 4 * heads * dim * pairs}


# ---- the same from the definition, in 64 bits ------------------------------------------------------------------------
def _unpacked(pages, request_pages, count, which, kv, page, dim):
    """Keys (which 0) or values (1) of the first `count` tokens of a request, float64 [kv, count, dim], bit by bit."""
    raw = pages[request_pages.long()].view(-1, kv, page * dim // 32 * 40)
    groups, base = dim // 32, which * page * dim // 32 * 20
    codes = raw[:, :, base:base + page * dim // 2].reshape(-1, kv, page, dim // 2).to(torch.int64)
    par = raw[:, :, base + page * dim // 2:base + page * dim // 32 * 20].contiguous().view(torch.bfloat16).reshape(-1, kv, page, groups, 2).double()
    x = torch.empty(*codes.shape[:3], dim, dtype=torch.float64, device=pages.device)
    for c in range(dim):
        g, r = c // 32, c % 32
        if which == 0:
            nibble = ((r // 8) * groups + g) * 8 + (r % 8) // 2 + 4 * (r % 2)
        else:
            nibble = ((2 * (r // 8) + r % 2) * groups + g) * 4 + (r % 8) // 2
        n = (codes[..., nibble // 2] >> (4 * (nibble % 2))) & 15
        x[..., c] = par[..., g, 1] + par[..., g, 0] * n.double()
    return x.transpose(1, 2).reshape(-1, kv, dim)[:count].transpose(0, 1)


def exact(case, seed):
    if case["op"] == "copy":
        return None
    st = prepare(case, seed)
    heads, kv, dim, page = st["heads"], st["kv"], st["dim"], st["page"]
    if case["op"] == "store":
        q = st["qkv"][:, :heads * dim].double().view(-1, heads, 2, dim // 2)
        turn = torch.complex(st["cos"].double(), st["sin"].double())[:, None]
        z = torch.complex(q[:, :, 0], q[:, :, 1]) * turn
        return torch.cat([z.real, z.imag], dim=-1).flatten(1), None     # (codes have no value between: they are whole numbers)
    meta, group, at, rows = st["meta"], heads // kv, 0, []
    for b, (new, total) in enumerate(zip(meta.query_lens, meta.seq_lens_host)):
        count = -(-total // page)
        k = _unpacked(st["pages"], meta.block_table[b, :count], total, 0, kv, page, dim)
        v = _unpacked(st["pages"], meta.block_table[b, :count], total, 1, kv, page, dim)
        q = st["q"][at:at + new].double().view(new, kv, group, dim)
        gone = torch.arange(total, device=q.device)[None] - torch.arange(total - new, total, device=q.device)[:, None]     # key minus query
        hidden = (gone > 0) | (gone <= -st["window"]) if st["window"] else gone > 0
        o = []
        for h in range(heads):
            s = (q[:, h // group, h % group] @ k[h // group].T / dim ** 0.5).masked_fill(hidden, -math.inf)
            o.append(torch.softmax(s, dim=-1) @ v[h // group])
        rows.append(torch.stack(o, dim=1).flatten(1))
        at += new
    return torch.cat(rows)
