"""How far bfloat16 attention over a packed cache may be off, from the roundings that its kernels make and not from their worst case.

Every rounding is taken as an error of its own, evenly spread over half a step u to either side (so its mean square is (u x)^2 / 3 at
most), and errors of different keys as independent.  For a query row and head, with p the softmax weights, o = sum p v the result, and
a value v = z + s n, the mean square of an error of number c is then (U = 2^-8, H = 2^-11, half a step of bfloat16 and of float16)

  all kernels      the result's last rounding                  U^2 / 3 o^2
  general          nothing else (float32 throughout)
  single tokens    p as float16                                sum_j p^2 H^2 / 3 (v - o)^2
                   p s as bfloat16, a group at a time          sum_j p^2 U^2 / 3 (s (n - 8))^2
                   p as bfloat16, for the middles and the sum  sum_j p^2 U^2 / 3 (z + 8 s - o)^2
                   the middles z + 8 s as bfloat16             sum_j p^2 U^2 / 3 (z + 8 s)^2
                   scores: sums of (1024 + n) q in float32     sum_j p^2 (2^-14 scale sum_g s_g |q_g|_1)^2 (v - o)^2
                   (each of two sums of 16 products is off by up to 2^-23 1040 |q_g|_1, which is 2^-13 of that; half of it)
  prompt portions  keys as float16                             sum_j p^2 H^2 / 3 scale^2 (sum_d q_d^2 k_d^2) (v - o)^2
                   p and values as float16                     2 sum_j p^2 H^2 / 3 v^2
                  and where float16 is not a matter of half steps relative to the number any more: keys and values lie in it over the
                  power of two of the largest |z| + 15 s among a tile's 128 tokens (2^-67 and 2^-27 at least; the largest becomes
                  2^14 to 2^15), so that s, z and z + s n are off by up to 2^-25 there, 17 2^-25 with fifteen steps, which is
                  17 2^-39 of the tile's largest.  A tile with a token more than 2^22 below that is not worked on in float16 at all.
                  For keys a score moves by up to 17 2^-39 scale |q|_1 of it, for values it adds up as it is.
                  p times a tile's power, over the row's largest such product M, lies in float16 times 2^7: number v_j is off by up
                  to 2^-25 2^-7 2 M |v_j| / (the tile's power).
                  Results below 2^-126 are off by up to 2^-134.

and the error of the row's head, as a vector, is allowed MARGIN times the root of the sum over its numbers.  The half step that a
rounding takes is relative to the power of two below x, so (u x)^2 / 3 is twice the mean on average: three times the root are more than
four standard deviations, and an error that a single rounding makes cannot pass sqrt(3) times its own root at all."""
import math

import torch

import kv4_plain as P

U, H, MARGIN = 2.0 ** -8, 2.0 ** -11, 3.0


def form_of(heads, kv, page, D, news):
    """Which kernels answer: 'prompt' for portions, 'single' or 'general' for single tokens."""
    if D not in (64, 128):
        return "general", "general"
    return "prompt", "single" if 32 % page == 0 or page % 32 == 0 else "general"


def tile_powers(z, s15, seen, least):
    """([n] the largest |z| + 15 s among the tokens of each token's tile that the query tile sees, [n] whether the products work on that
    tile in float16); z, 15 s: [n, D]."""
    own = torch.where(seen, (z.abs() + s15).nan_to_num(nan=0.0).amax(-1), 0.0)
    power, fine = torch.zeros_like(own), torch.ones_like(seen)
    for t in range(0, len(own), 128):
        tile = own[t:t + 128]
        power[t:t + 128] = tile.max().clamp(min=least)
        # (told apart by exponents: a token 2^22 to 2^23 below may count as either, and is off by as much as that)
        fine[t:t + 128] = not bool(((tile > 0) & (tile * 2.0 ** 23 < power[t])).any())
    return power, fine


def attend(q, cache, table, lens, news, heads, kv, page, D, window=0, scale=0.0, wrong=None):
    """(result float64 [T, heads, D], allowed error in norm [T, heads]).  `wrong` plants a mistake: "scale" (10% off), "first" (the first
    32 keys left out), "step" (value steps 6% too large), "window" (a key more), "tile" (keys 64 .. 95 left out)."""
    scale = scale or 1.0 / math.sqrt(D)
    if wrong == "scale":
        scale *= 1.1
    rows, tols, at, group = [], [], 0, heads // kv
    portion, alone = form_of(heads, kv, page, D, news)
    for b, (total, new) in enumerate(zip(lens, news)):
        form = alone if new == 1 else portion
        pos = torch.arange(total)
        z, sn = P.numbers(cache, table[b].long()[pos // page] * page + pos % page, kv, page, D)
        steps = P._views(cache, kv, page, D)[3][table[b].long()[pos // page], :, pos % page]
        vstep = steps.contiguous().view(torch.bfloat16).double().unflatten(-1, (-1, 2))[..., 0].repeat_interleave(32, dim=-1)
        ksteps = P._views(cache, kv, page, D)[1][table[b].long()[pos // page], :, pos % page]
        kstep = ksteps.contiguous().view(torch.bfloat16).double().unflatten(-1, (-1, 2))[..., 0]                       # [n, kv, G]
        sn_max = 15 * torch.stack([kstep.repeat_interleave(32, dim=-1), vstep], dim=1)
        query = torch.arange(total - new, total)
        hidden = pos[None] > query[:, None]
        reach = window + 1 if wrong == "window" else window
        if window:
            hidden = hidden | (pos[None] <= query[:, None] - reach)
        if wrong in ("first", "tile"):
            lo = 0 if wrong == "first" else 64
            gone = (pos >= lo) & (pos < lo + 32)
            if total > lo + 32:
                hidden = hidden | (gone[None] & (query >= lo + 32)[:, None])
        unseen = hidden.all(0)
        o, tol = torch.zeros(new, heads, D, dtype=torch.float64), torch.zeros(new, heads, dtype=torch.float64)
        for h in range(heads):
            g = h // group
            k = z[:, 0, g] + sn[:, 0, g]
            s, n_s = vstep[:, g], sn[:, 1, g] * (1.06 if wrong == "step" else 1.0)
            v, middle = z[:, 1, g] + n_s, z[:, 1, g] + 8 * s
            k, v, middle, s, n_s = (torch.where(unseen[:, None], 0.0, x) for x in (k, v, middle, s, n_s))
            qh = q[at:at + new, h * D:(h + 1) * D].double()
            p = torch.softmax((qh @ k.T * scale).masked_fill(hidden, -math.inf), -1)
            r = o[:, h] = p @ v

            def spread(w, x):                          # sum_c sum_j w_j (x_jc - r_c)^2
                return w @ (x * x).sum(-1) - 2 * ((w @ x) * r).sum(-1) + w.sum(-1) * (r * r).sum(-1)
            p2 = p * p
            var = U * U / 3 * (r * r).sum(-1) + D * 2.0 ** -268
            if form == "single":
                var = var + H * H / 3 * spread(p2, v) + U * U / 3 * (p2 @ ((n_s - 8 * s) ** 2 + middle ** 2).sum(-1) + spread(p2, middle))
                off = 2.0 ** -14 * scale * qh.abs().unflatten(-1, (-1, 32)).sum(-1) @ torch.where(unseen[:, None], 0.0, kstep[:, g]).T
                var = var + spread(p2 * off * off, v)
            elif form == "prompt":
                off = H * H / 3 * scale * scale * ((qh * qh) @ (k * k).T)
                var = var + spread(p2 * off, v) + 2 * H * H / 3 * (p2 @ (v * v).sum(-1))
                for r0 in range(0, new, 128):          # the kernel's query tiles
                    at_rows = slice(r0, min(new, r0 + 128))
                    lo, hi = int(query[r0]), int(query[at_rows][-1])
                    seen = (pos <= hi) & (pos > lo - window if window else True)
                    (kp, k_fine), (vp, v_fine) = (tile_powers(z[:, i, g], sn_max[:, i, g], seen, least) for i, least in ((0, 2.0 ** -67), (1, 2.0 ** -27)))
                    fine = (k_fine & v_fine).double()
                    pr = p[at_rows] * fine
                    moved = (17 * 2.0 ** -39 * scale) * qh[at_rows].abs().sum(-1)[:, None] * kp[None]
                    top = (pr * vp).amax(-1)
                    var[at_rows] += (pr * pr * torch.expm1(moved.clamp(max=1)) ** 2) @ (v * v).sum(-1)
                    var[at_rows] += D * (17 * 2.0 ** -39 * (pr @ vp)) ** 2
                    var[at_rows] += (2.0 ** -31 * top) ** 2 * ((pr > 0).double() @ ((v * v).sum(-1) / vp ** 2))
            tol[:, h] = MARGIN * var.clamp(min=0).sqrt()
        rows.append(o)
        tols.append(tol)
        at += new
    return torch.cat(rows), torch.cat(tols)


def worst(got, want, tol):
    """The largest error of a row and head over what it is allowed."""
    return ((got.double().view_as(want) - want).norm(dim=-1) / tol).max().item()
