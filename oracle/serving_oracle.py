"""Restatements in 64 bits, or in whole numbers, of the operators between a projection and a paged cache: norm with rotation
and its gradients, the plan of a serving step, and attention over pages.  Test infrastructure only; plain loops and CPU
tensors, written from the formulas."""
from __future__ import annotations

import math

import torch


# ---- norm and rotation -------------------------------------------------------------------------------------------
def rope_angles(positions, inv_freq, axes=None):
    """Angles (B | 1, S, 1, pairs) in 64 bits."""
    f = inv_freq.detach().double().cpu()
    pos = positions.detach().cpu()
    if axes is None:
        pos = pos if pos.dim() == 2 else pos[None]
        a = pos.double()[..., None] * f
    else:
        pos = pos if pos.dim() == 3 else pos[:, None]
        a = torch.stack([pos[x].double() * f[i] for i, x in enumerate(axes)], -1)
    return a[:, :, None, :]


def rotate(y, angles, interleaved):
    half = angles.shape[-1]
    out = y.clone()
    for i in range(half):
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = torch.cos(angles[..., i]), torch.sin(angles[..., i])
        out[..., lo] = y[..., lo] * c - y[..., hi] * s
        out[..., hi] = y[..., hi] * c + y[..., lo] * s
    return out


def norm_rope(x, weight=None, angles=None, interleaved=False, eps=1e-6):
    x = x.detach().double().cpu()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.detach().double().cpu()
    return x if angles is None else rotate(x, angles, interleaved)


def norm_rope_grads(x, dout, weight=None, angles=None, interleaved=False, eps=1e-6):
    """(dx, dw, size of the terms of dx, sum of the magnitudes that make up dw): the last two scale a rounding bound.  A
    rotated gradient g_lo c + g_hi s may cancel, and each product carries a rounding of its own and that of its cosine or
    sine: its error is a multiple of 2^-24 (|g_lo| + |g_hi|), which is what counts in the second."""
    x, g = x.detach().double().cpu(), dout.detach().double().cpu()
    mag = g.abs()
    if angles is not None:
        half = angles.shape[-1]
        for i in range(half):
            lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            mag[..., lo] = mag[..., hi] = g[..., lo].abs() + g[..., hi].abs()
        g = rotate(g, -angles, interleaved)
    if weight is None:
        return g, None, g.abs(), None
    w = weight.detach().double().cpu()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    dx = r * (w * g - x * r ** 2 * (w * g * x).mean(-1, keepdim=True))
    size = r * ((w * g).abs() + x.abs() * r ** 2 * (w * g * x).abs().mean(-1, keepdim=True))
    return dx, (g * x * r).flatten(0, -2).sum(0), size, (mag * (x * r).abs()).flatten(0, -2).sum(0)


# ---- the plan of a step ------------------------------------------------------------------------------------------
def plan(table, held, free_pages, free_count, lens, new_lens, page_size, num_tokens, parents=None, max_tree=64):
    """Everything as lists of ints; returns the new state and the step, in plain sequential code."""
    table, held, stack = [list(r) for r in table], list(held), list(free_pages)
    B, width, count = len(table), len(table[0]), free_count
    words = -(-max_tree // 64)
    cu, ok, total = [0], [], 0
    for b in range(B):
        t = max(new_lens[b], 0)
        total += t
        fits = lens[b] >= 0 and new_lens[b] >= 0 and -(-(lens[b] + t) // page_size) <= width and total <= num_tokens
        ok.append(fits and (parents is None or t <= 64 * words))
        cu.append(min(total, num_tokens))
    need = [-(-(lens[b] + new_lens[b]) // page_size) if ok[b] else held[b] for b in range(B)]
    back = [table[b][i] for b in range(B) for i in range(need[b], held[b])]
    stack[count:count + len(back)] = back[::-1]
    count += len(back)
    out_of_pages = False
    for b in range(B):
        more = need[b] - held[b]
        if ok[b] and more > 0:
            if out_of_pages or more > count:
                out_of_pages, ok[b] = True, False
                continue
            for i in range(held[b], need[b]):
                count -= 1
                table[b][i] = stack[count]
        if ok[b]:
            held[b] = need[b]
    slots, positions, masks = [-1] * num_tokens, [0] * num_tokens, [[0] * words for _ in range(num_tokens)]
    for b in range(B):
        if not ok[b]:
            continue
        for t in range(cu[b + 1] - cu[b]):
            n, place = cu[b] + t, lens[b] + t
            slots[n] = table[b][place // page_size] * page_size + place % page_size
            positions[n] = place
            if parents is not None:
                at, depth = t, -1
                while at >= 0:
                    masks[n][at // 64] |= 1 << (at % 64)
                    at, depth = parents[cu[b] + at], depth + 1
                positions[n] = lens[b] + depth
    signed = [[w - (1 << 64) if w >> 63 else w for w in m] for m in masks]
    return dict(table=table, held=held, stack=stack, count=count, slots=slots, positions=positions, cu=cu,
                lens=[lens[b] if ok[b] else -1 for b in range(B)], masks=signed)


# ---- attention over pages ----------------------------------------------------------------------------------------
def paged_attention(q, key_cache, value_cache, table, lens, cu, tree_mask=None, positions=None, slopes=None, q_bias=None,
                    bias_cache=None, scale=None):
    """(o, lse, weight, logit size): o and lse in 64 bits, sum of p |v| per output value and the largest sum of magnitudes
    that makes up a visible logit per row.  Only visible keys are touched."""
    q = q.detach().double().cpu()
    kc, vc = key_cache.detach().double().cpu(), value_cache.detach().double().cpu()
    N, Hq, D = q.shape
    page, Hk = kc.shape[1], kc.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    table, lens, cu = table.tolist(), lens.tolist(), cu.tolist()
    kvh = torch.arange(Hq) // (Hq // Hk)
    o, lse = torch.zeros(N, Hq, D, dtype=torch.float64), torch.full((N, Hq), -math.inf, dtype=torch.float64)
    weight, size = torch.zeros_like(o), torch.zeros(N, Hq, dtype=torch.float64)
    for b in range(len(table)):
        ctx, first, T = lens[b], cu[b], cu[b + 1] - cu[b]
        if ctx < 0:
            continue
        where = [(table[b][j // page], j % page) for j in range(ctx + T)]
        for t in range(T):
            n = first + t
            if tree_mask is not None:
                words = tree_mask[n].reshape(-1).tolist()
                seen = [i for i in range(T) if i < 64 * len(words) and (words[i // 64] >> (i % 64)) & 1]
            else:
                seen = list(range(t + 1))
            keys = list(range(ctx)) + [ctx + i for i in seen]
            if not keys:
                continue
            pg = torch.tensor([where[j][0] for j in keys])
            pl = torch.tensor([where[j][1] for j in keys])
            k, v = kc[pg, pl][:, kvh], vc[pg, pl][:, kvh]  # (keys, Hq, D)
            z, mag = torch.einsum("hd,khd->hk", q[n], k) * scale, torch.einsum("hd,khd->hk", q[n].abs(), k.abs()) * abs(scale)
            if slopes is not None:
                mine = int(positions[n]) if positions is not None else ctx + t
                at = torch.tensor([j if j < ctx or positions is None else int(positions[first + j - ctx]) for j in keys])
                bias = slopes.double().cpu()[:, None] * (at - mine).double()
                z, mag = z + bias, mag + bias.abs()
            if q_bias is not None:
                qb = q_bias.detach().double().cpu()[n].expand(Hq, -1)
                kb = bias_cache.detach().double().cpu()[pg, pl]
                kb = kb[:, kvh] if kb.shape[1] > 1 else kb.expand(-1, Hq, -1)
                z, mag = z + torch.einsum("hr,khr->hk", qb, kb), mag + torch.einsum("hr,khr->hk", qb.abs(), kb.abs())
            p = torch.softmax(z, -1)
            o[n], weight[n] = torch.einsum("hk,khd->hd", p, v), torch.einsum("hk,khd->hd", p, v.abs())
            lse[n], size[n] = torch.logsumexp(z, -1), mag.amax(-1)
    return o, lse, weight, size
