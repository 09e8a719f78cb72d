"""Inputs of the bound tests of attention over a packed cache: random numbers, pages in random order, NaN wherever no request owns a row."""
from types import SimpleNamespace

import torch

import kv4_plain as P

LENS = [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 255, 300]
# name: seed, tokens of each request, of which queries, query heads, key/value heads, numbers a head, tokens a page, window
CASES = {
    "single 64": (1, LENS, [1] * len(LENS), 4, 2, 64, 16, 0),
    "single 128": (1, LENS, [1] * len(LENS), 6, 2, 128, 4, 0),
    "single, 9 heads a group": (1, LENS, [1] * len(LENS), 9, 1, 64, 8, 0),
    "single, 16 heads a group, pages of 64": (1, LENS, [1] * len(LENS), 16, 1, 128, 64, 0),
    "single, windows of 33": (2, LENS, [1] * len(LENS), 8, 2, 64, 8, 33),
    "single, windows of 7": (3, [300, 40, 9], [1] * 3, 4, 1, 128, 64, 7),
    "single, long 128": (8, [3000, 2600, 70], [1] * 3, 4, 1, 128, 16, 0),
    "single, long 64": (8, [3100, 1900], [1] * 2, 8, 2, 64, 32, 0),
    "single, long, windows of 1000": (9, [3000, 900], [1] * 2, 4, 1, 128, 16, 1000),
    "general, pages of 12": (1, LENS, [1] * len(LENS), 2, 1, 128, 12, 0),
    "general 96": (1, LENS, [1] * len(LENS), 6, 3, 96, 20, 0),
    "prompt 64": (4, [1, 2, 17, 127, 128, 130, 260], [1, 2, 17, 127, 128, 130, 260], 4, 2, 64, 16, 0),
    "prompt 128": (4, [2, 17, 127, 130, 260], [2, 17, 127, 130, 260], 3, 1, 128, 4, 0),
    "prompt, pages of 24": (5, [300, 41, 9, 513, 129, 64], [3, 1, 9, 130, 128, 1], 6, 2, 128, 24, 0),
    "prompt, windows of 5": (6, [300, 41, 513], [290, 41, 130], 4, 2, 64, 16, 5),
    "prompt, windows of 200": (7, [257, 500], [257, 2], 4, 1, 128, 8, 200),
    "prompt, long": (9, [3300, 1500], [40, 129], 4, 1, 64, 16, 0),
}


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def pages(seed, lens, kv, D, page, spoil=True):
    """A table of page ids in random order, and the empty pages."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(seed))
    table = torch.zeros(len(lens), max(need) + 2, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    return table, torch.full((sum(need) + 3, kv * page * (D // 32) * 40), 0xff if spoil else 0, dtype=torch.uint8)


def fill(cache, table, b, page, k, v):
    p = torch.arange(len(k))
    P.store(cache, table[b].long()[p // page] * page + p % page, k, v, page)


def inputs(seed, lens, news, heads, kv, D, page, dtype):
    table, cache = pages(seed, lens, kv, D, page)
    for b, n in enumerate(lens):
        k, v = rnd(n, kv, D, seed=seed * 100 + b), rnd(n, kv, D, seed=seed * 100 + 50 + b)
        k[:, :, ::11] *= 4.0
        fill(cache, table, b, page, k.to(dtype), v.to(dtype))
    return rnd(sum(news), heads * D, seed=seed + 9).to(dtype), cache, table


def attention(K, q, cache, table, lens, news, heads, kv, D, window=0, scale=0.0):
    request = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(news)).int()
    position = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, news)]).int()
    meta = SimpleNamespace(block_table=table.cuda(), token_request=request.cuda(), positions=position.cuda(), query_lens=list(news),
                           seq_lens_host=list(lens))
    out = torch.full((sum(news), heads * D), 7.0, dtype=q.dtype, device="cuda")
    K.attention_kv4(q.cuda(), cache.cuda(), meta, out, heads, kv, D, window=window, scale=scale)
    K.check_health()
    return out.cpu()
