"""The packed key/value cache restated plainly: the format number by number, attention in 64 bits with the error that roundings may
add, and a kernel double for the CPU tests of the engine.

Format (csrc/kv4.cuh): 32 neighbouring numbers share a zero point z (the largest bfloat16 not above their minimum) and a step
s = bfloat16((max - z) / 15); a number is z + s n.  Where each nibble lies is written down here once more, as loops over numbers.
"""
import math

import torch

from torch_kernels import TorchKernels, ref_rope

U16, U32 = 2.0 ** -8, 2.0 ** -24            # half a step of a bfloat16 and of a float32, relative


def floor_bf16(x):
    """The largest bfloat16 that is not above x (float32 -> float32)."""
    r = x.bfloat16()
    down = torch.where(r == 0, torch.full_like(r, -1e-45).float().bfloat16(), r)          # (a step below 0: the smallest negative number)
    bits = r.view(torch.int16).int()
    stepped = torch.where(r.float() > 0, bits - 1, bits + 1)
    below = stepped.to(torch.int16).view(torch.bfloat16)
    below = torch.where(r == 0, torch.tensor(-2.0 ** -133, dtype=torch.float32).bfloat16().expand_as(down), below)
    return torch.where(r.float() > x, below, r).float()


def pack(x):
    """float32 [..., D] -> codes [..., D] (int), s and z [..., D / 32] float32."""
    g = x.float().unflatten(-1, (-1, 32))
    z = floor_bf16(g.amin(-1))
    s = ((g.amax(-1) - z) * torch.tensor(1.0 / 15.0, dtype=torch.float32)).bfloat16().float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    r = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    n = torch.round((g - z[..., None]) * r[..., None]).clamp(0, 15)
    n = torch.where(torch.isnan(n), torch.zeros_like(n), n)
    return n.int().flatten(-2), s, z


def key_place(D, c):
    """(byte, shift) of number c in a key row's codes."""
    G, g, r = D // 32, c // 32, c % 32
    nibble = [0, 2, 4, 6, 1, 3, 5, 7].index(r % 8)
    return 4 * ((r // 8) * G + g) + nibble // 2, 4 * (nibble % 2)


def value_place(D, c):
    G, g, r = D // 32, c // 32, c % 32
    half = (2 * (r // 8) + r % 2) * G + g
    nibble = [0, 2, 4, 6].index(r % 8 - r % 2)
    return 2 * half + nibble // 2, 4 * (nibble % 2)


def offsets(page, D):
    """Byte offsets of the four regions of a head's block, and the block's size."""
    G = D // 32
    return 0, page * 16 * G, page * 20 * G, page * 36 * G, page * 40 * G


def _views(cache, kv, page, D):
    G = D // 32
    b = cache.view(cache.shape[0], kv, page * 40 * G)
    kc, kp, vc, vp, end = offsets(page, D)
    return [b[..., lo:hi].unflatten(-1, (page, -1)) for lo, hi in ((kc, kp), (kp, vc), (vc, vp), (vp, end))]


def store(cache, slots, keys, values, page):
    """Writes keys and values [n, kv, D] (numbers of the engine's type) into a layer's pages (CPU uint8 [pages, bytes])."""
    n, kv, D = keys.shape
    kc, ks, kz = pack(keys)
    vc, vs, vz = pack(values)
    bad = ~(torch.isfinite(keys.float()).all(-1) & torch.isfinite(values.float()).all(-1) & torch.isfinite(ks).all(-1) &
            torch.isfinite(kz).all(-1) & torch.isfinite(vs).all(-1) & torch.isfinite(vz).all(-1))          # [n, kv]
    regions = _views(cache, kv, page, D)
    kept = slots >= 0
    at, off = slots[kept].long() // page, slots[kept].long() % page
    for codes, s, z, place, which in ((kc, ks, kz, key_place, 0), (vc, vs, vz, value_place, 1)):
        row = torch.zeros(n, kv, D // 2, dtype=torch.int32)
        for shift in (0, 4):                       # every byte holds one number at either shift
            numbers_of = [c for c in range(D) if place(D, c)[1] == shift]
            row[..., [place(D, c)[0] for c in numbers_of]] |= codes[..., numbers_of] << shift
        par = torch.stack([s, z], dim=-1)
        row[bad] = 0
        par[bad] = math.nan if which == 0 else 0.0
        regions[2 * which][at, :, off] = row[kept].to(torch.uint8)
        regions[2 * which + 1][at, :, off] = par.bfloat16().flatten(-2).contiguous().view(torch.uint8)[kept]


def numbers(cache, slots, kv, page, D):
    """(z, s n) of keys and of values at `slots`, float64 [n, 2, kv, D] each: the numbers are their sums."""
    regions = _views(cache, kv, page, D)
    slots = slots.long()
    out_z = torch.zeros(len(slots), 2, kv, D, dtype=torch.float64)
    out_sn = torch.zeros_like(out_z)
    for which, place in ((0, key_place), (1, value_place)):
        codes = regions[2 * which][slots // page, :, slots % page]
        par = regions[2 * which + 1][slots // page, :, slots % page].contiguous().view(torch.bfloat16).double().unflatten(-1, (-1, 2))
        places = [place(D, c) for c in range(D)]
        n = (codes[..., [p[0] for p in places]].int() >> torch.tensor([p[1] for p in places], dtype=torch.int32)) & 15
        par = par.repeat_interleave(32, dim=-2)
        out_sn[:, which], out_z[:, which] = par[..., 0] * n, par[..., 1]
    return out_z, out_sn


def attend(q, cache, table, lens, news, heads, kv, page, D, window=0, scale=0.0, unit=U16):
    """(output float64 [T, heads * D], tolerance of the same shape).  q [T, heads * D]; request b holds lens[b] tokens of which the
    last news[b] are queries.

    The tolerance counts roundings: with u half a relative step, A the largest sum scale |q| |k| of the row and M = sum p (|z| + s n):
    keys taken as bfloat16 move a score by at most u A and so a probability by 2 u A (in the sum and in its own term); the
    probability times the step, the value and the result are each rounded once more: 3 u M; float32 sums over D numbers and n keys
    add (2 (D + 8) A + 2 n + 32) 2^-24 M."""
    scale = scale or 1.0 / math.sqrt(D)
    rows, tols = [], []
    at = 0
    for b, (total, new) in enumerate(zip(lens, news)):
        pos = torch.arange(total)
        z, sn = numbers(cache, table[b].long()[pos // page] * page + pos % page, kv, page, D)
        k, v, mag = z[:, 0] + sn[:, 0], z[:, 1] + sn[:, 1], z[:, 1].abs() + sn[:, 1]
        qb = q[at:at + new].double().view(new, heads, D)
        group = heads // kv
        o, t = torch.zeros(new, heads, D, dtype=torch.float64), torch.zeros(new, heads, D, dtype=torch.float64)
        query = torch.arange(total - new, total)
        hidden = pos[None] > query[:, None]
        if window:
            hidden |= pos[None] <= query[:, None] - window
        for h in range(heads):
            kk, vv, mm = k[:, h // group], v[:, h // group], mag[:, h // group]
            s = qb[:, h] @ kk.T * scale
            a = (qb[:, h].abs() @ kk.abs().T * scale).masked_fill(hidden, 0).amax(-1, keepdim=True)
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            # a token that a row does not see must not matter whatever it holds
            seen_v = torch.where(hidden.all(0)[:, None], torch.zeros_like(vv), vv)
            o[:, h], m = p @ seen_v, p @ mm
            small = U32 * (2 * (D + 8) * a + 2 * total + 32)
            t[:, h] = m * (small + (2 * a + 3) * unit if unit == U16 else small)
        rows.append(o.flatten(1))
        tols.append(t.flatten(1))
        at += new
    return torch.cat(rows), torch.cat(tols) + 1e-30


class PackedTorchKernels(TorchKernels):
    """The CPU kernel double with the packed cache and the page copies."""

    def __init__(self):
        self.copied = []

    @staticmethod
    def _page(cache, kv, D):
        return cache.shape[1] // (kv * (D // 32) * 40)

    def rope_store_kv4(self, qkv, tables, slots, cache_layer, heads, kv_heads, head_dim, rotary_dim, q_out=None):
        T = qkv.shape[0]
        x = qkv.float().view(T, -1, head_dim).clone()
        if rotary_dim:
            c, s = tables[0][:, None], tables[1][:, None]
            half = rotary_dim // 2
            a, b = x[:, :heads + kv_heads, :half].clone(), x[:, :heads + kv_heads, half:rotary_dim].clone()
            x[:, :heads + kv_heads, :half] = a * c - b * s
            x[:, :heads + kv_heads, half:rotary_dim] = b * c + a * s
        x = x.to(qkv.dtype)
        if slots is not None:
            store(cache_layer, slots, x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], self._page(cache_layer, kv_heads, head_dim))
        q_out = qkv if q_out is None else q_out
        q_out[:, :heads * head_dim] = x[:, :heads].flatten(1)
        return q_out

    def kv4_read(self, cache_layer, slots, out, kv_heads, head_dim):
        z, sn = numbers(cache_layer, slots, kv_heads, self._page(cache_layer, kv_heads, head_dim), head_dim)
        out.copy_(z + sn)
        return out

    def attention_kv4(self, q, cache_layer, meta, out, heads, kv_heads, head_dim, window=0, scale=0.0):
        page = self._page(cache_layer, kv_heads, head_dim)
        o, _ = attend(q[:, :heads * head_dim], cache_layer, meta.block_table, meta.seq_lens_host, meta.query_lens, heads, kv_heads, page,
                      head_dim, window, scale)
        out.copy_(o)
        return out

    def copy_pages(self, storage, pairs):
        self.copied += list(pairs)
        if pairs:
            src, dst = zip(*pairs)
            storage[:, list(dst)] = storage[:, list(src)]
        return storage
