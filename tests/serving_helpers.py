"""Shared by the tests of the operators around a paged cache: inputs, and bounds that follow from the roundings."""
import torch

FP32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(name, got, want, bound):
    """Element by element; what the bound allows follows from the roundings that the kernel makes."""
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, f"{name}: shape {tuple(got.shape)}, not {tuple(want.shape)}"
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} values beyond their bound, the worst by a factor of "
                           f"{float((off / bound.clamp_min(1e-300))[bad].max()):.3g}")


def rounded(want, dtype, size, ops=64):
    """One rounding to `dtype` of a value computed in fp32 by about `ops` roundings of terms of magnitude `size`; half the
    smallest step below fp16's normal numbers."""
    return half_step(dtype) * want.abs() * 1.001 + ops * FP32 * size + torch.finfo(dtype).smallest_normal * half_step(dtype)


def pool_of(lens, new_lens, page, width, seed, spare=3, lost=()):
    """A random distribution of pages: (table, held, stack, count) as lists, for requests that hold the pages of `lens`."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-max(x, 0) // page) for x in lens]
    growth = sum(max(0, -(-(max(a, 0) + max(b, 0)) // page) - h) for a, b, h in zip(lens, new_lens, held))
    total = sum(held) + growth + spare
    perm = torch.randperm(total, generator=g).tolist()
    table, at = [], 0
    for h in held:
        table.append(perm[at:at + h] + [-7] * (width - h))
        at += h
    free = perm[at:]
    return table, held, free + [-9] * (total - len(free)), len(free)


def paged_inputs(lens, new, Hq, Hk, D, page, dtype, seed, R=0, bias_heads=None, order="phd", extra_pages=2):
    """Caches with every unused place NaN, a block table with -1 behind each request's pages, and the step's tokens."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-(max(a, 0) + b) // page) for a, b in zip(lens, new)]
    pool, width = sum(pages) + extra_pages, max(max(pages), 1) + 1
    perm = torch.randperm(pool, generator=g)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n

    def cache(heads, cols):
        c = torch.full((pool, page, heads, cols), float("nan"), dtype=dtype)
        for b, (ctx, t) in enumerate(zip(lens, new)):
            for j in range(max(ctx, 0) + t):
                c[table[b, j // page], j % page] = torch.randn(heads, cols, generator=g).to(dtype)
        if order == "hpd":  # heads outside the places of a page
            return c.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        return c

    N = sum(new)
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
    out = dict(q=torch.randn(N, Hq, D, generator=g).to(dtype), key_cache=cache(Hk, D), value_cache=cache(Hk, D), block_table=table,
               lens=torch.tensor(lens, dtype=torch.int32), cu_tokens=cu)
    if R:
        out["q_bias"] = torch.randn(N, Hq, R, generator=g).to(dtype)
        out["bias_cache"] = cache(bias_heads or Hk, R)
    return out


def tree(new, seed, words=1):
    """Random parents, and the ancestor bits and depths that they mean: (parents, mask (N, words), depth) on the host."""
    g = torch.Generator().manual_seed(seed)
    parents, masks, depths = [], [], []
    for T in new:
        mine, deep = [], []
        for t in range(T):
            up = int(torch.randint(-1, t, (1,), generator=g)) if t else -1
            parents.append(up)
            mine.append((mine[up] if up >= 0 else 0) | 1 << t)
            deep.append(deep[up] + 1 if up >= 0 else 0)
        masks += mine
        depths += deep
    rows = [[(m >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for m in masks]
    rows = [[w - 2 ** 64 if w >> 63 else w for w in r] for r in rows]
    return (torch.tensor(parents, dtype=torch.int32), torch.tensor(rows, dtype=torch.int64).reshape(len(rows), words),
            torch.tensor(depths, dtype=torch.int32))
