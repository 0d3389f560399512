"""The operators between a projection and the attention over a paged cache, as cases that can be timed and compared.

Four operators: norm and rotation of queries and keys (training and inference), the same pass with the keys and values
going into the pages of a cache, the plan of a serving step (block tables, slots, positions and ancestor masks from request
lengths), and attention of one, several or a tree of drafted tokens over the paged cache with the framework's two kinds of
bias.  ``run`` computes them in elementary operations in 32 bits, or, where ``own`` is set, through the package's entry
points.

Values: activations are N(0, 1), norm weights near one, upstream gradients N(0, 1); keys in a cache are what a norm leaves
(unit mean square); slopes are those of ALiBi, factors N(0, 1) with the spread of a unit-variance bias.  Activations are slices
of a fused projection, as layers hold them; pages of a request lie anywhere in the pool.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def _rope(name, B, S, Hq, Hk, D, rot, naxes, interleaved, norm, dtype, train, wtype="same"):
    return _named(name, dict(op="norm_rope", B=B, S=S, Hq=Hq, Hk=Hk, D=D, rot=rot, naxes=naxes, interleaved=interleaved,
                             norm=norm, dtype=dtype, train=train, wtype=wtype))


def _append(name, N, Hq, Hk, D, rot, page, norm, R, dtype):
    return _named(name, dict(op="append", N=N, Hq=Hq, Hk=Hk, D=D, rot=rot, page=page, norm=norm, R=R, dtype=dtype))


def _plan(name, B, T, L, page, tree):
    return _named(name, dict(op="plan", B=B, T=T, L=L, page=page, tree=tree))


def _attend(name, B, T, L, Hq, Hk, D, page, tree, bias, R, dtype):
    return _named(name, dict(op="attend", B=B, T=T, L=L, Hq=Hq, Hk=Hk, D=D, page=page, tree=tree, bias=bias, R=R, dtype=dtype))


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # one image of 16 x 16 patches and a class token in a small vision layer, rotation by row and column: a training
        # step in which the calls themselves are what a user waits for
        _rope("rope_image_train", 2, 257, 6, 6, 64, 64, 2, True, True, "fp16", True),
        # a training step of a language model's layer with grouped heads, fp32 norm weights
        _rope("rope_text_train", 4, 4096, 32, 8, 128, 128, 1, False, True, "bf16", True, "fp32"),
        # a video clip of 21 frames of 30 x 52 patches, rotation by time, height and width, training
        _rope("rope_video_train", 1, 32760, 12, 12, 128, 128, 3, False, True, "bf16", True),
        # a prompt of odd length without norms, a quarter of the head rotated, at a head_dim that is no power of two
        _rope("rope_prompt_partial", 1, 4001, 25, 25, 80, 20, 1, False, False, "fp16", False),
        # one token each of 32 sequences on its way into the cache
        _append("append_decode", 32, 32, 8, 128, 128, 16, True, 0, "bf16"),
        # prompts of several requests, 16384 tokens with some padding, with low-rank key factors beside the keys
        _append("append_prompt", 16384, 32, 8, 128, 128, 64, True, 4, "bf16"),
        # the plan of a decoding step of 64 sequences
        _plan("plan_decode", 64, 1, 4096, 16, False),
        # the plan of a speculative step: 256 requests, trees of up to 64 drafted tokens
        _plan("plan_tree", 256, 64, 8192, 16, True),
        # one token of one sequence with slopes, a short cache: the latency of a single user
        _attend("attend_one", 1, 1, 1000, 32, 8, 128, 16, False, "slopes", 0, "bf16"),
        # a decoding step of 64 ragged sequences with up to 8192 cached tokens, grouped heads
        _attend("attend_decode", 64, 1, 8192, 32, 8, 128, 16, False, "none", 0, "bf16"),
        # trees of up to 60 drafted tokens of 8 requests over caches of up to 6000 tokens, slopes by depth
        _attend("attend_tree", 8, 60, 6000, 32, 8, 128, 32, True, "slopes", 0, "bf16"),
        # small trees in a model with ungrouped heads and low-rank factors in a cache of their own
        _attend("attend_tree_factors", 16, 7, 3001, 16, 16, 64, 64, True, "factors", 8, "fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope", "append", "plan", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "norm_rope":
        Hk = rng.choice([1, 2, 4, 6, 8, 12])
        Hq = Hk * rng.choice([1, 1, 2, 4])
        D = rng.choice([20, 32, 48, 64, 72, 80, 96, 128, 128])
        rot = rng.choice([D, D, D // 4 * 2])
        naxes = rng.choice([1, 1, 2, 3])
        B, S = rng.choice([1, 2, 3]), _log_int(rng, 64, 8192)
        return _rope(None, B, S, Hq, Hk, D, rot, naxes, rng.random() < 0.4, rng.random() < 0.7, dtype, rng.random() < 0.7,
                     rng.choice(["same", "fp32"]))
    if op == "append":
        Hk = rng.choice([1, 2, 4, 8, 16])
        D = rng.choice([32, 64, 80, 96, 128, 128])
        return _append(None, _log_int(rng, 1, 8192), Hk * rng.choice([1, 2, 4]), Hk, D, rng.choice([D, D // 4 * 2]),
                       rng.choice([8, 16, 32, 64]), rng.random() < 0.6, rng.choice([0, 0, 2, 5, 8]), dtype)
    if op == "plan":
        tree = rng.random() < 0.5
        return _plan(None, _log_int(rng, 1, 512), _log_int(rng, 1, 64 if tree else 200), _log_int(rng, 64, 16384),
                     rng.choice([8, 16, 32, 64]), tree)
    G = rng.choice([1, 1, 2, 4, 8])
    Hk = rng.choice([2, 4, 8, 16]) if G < 8 else rng.choice([1, 2, 4])
    L = _log_int(rng, 16, 16384)
    tree = rng.random() < 0.5
    T = _log_int(rng, 2, 64) if tree else rng.choice([1, 1, 2, 4, 17])
    B = max(1, min(_log_int(rng, 1, 64), 2 ** 21 // (L * Hk), 2 ** 26 // (L * Hk * G * T)))
    bias = rng.choice(["none", "slopes", "factors"])
    return _attend(None, B, T, L, Hk * G, Hk, rng.choice([32, 64, 64, 80, 96, 128, 128]), rng.choice([8, 16, 32, 64]),
                   tree, bias, rng.choice([2, 5, 8, 16]) if bias == "factors" else 0, dtype)


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
class _Make:
    def __init__(self, seed):
        self.device = torch.device("cuda")
        self.g = torch.Generator(device=self.device).manual_seed(seed)
        self.host = torch.Generator().manual_seed(seed)
        self.shape = torch.Generator().manual_seed(0)  # the lengths of a case's requests are its own: its sizes are fixed

    def normal(self, shape, dtype, scale=1.0, shift=0.0):
        x = torch.randn(shape, generator=self.g, device=self.device, dtype=torch.float32 if dtype == torch.float32 else dtype)
        return x.mul_(scale).add_(shift) if (scale, shift) != (1.0, 0.0) else x

    def ints(self, lo, hi, n):
        """n host integers in [lo, hi]"""
        return torch.randint(lo, hi + 1, (n,), generator=self.host).tolist()

    def lengths(self, lo, hi, n):
        return torch.randint(lo, hi + 1, (n,), generator=self.shape).tolist()

    def tensor(self, values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device=self.device)

    def inv_freq(self, rot):
        return (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().to(self.device)


def _frequency_axes(rot, naxes):
    """The axis of each rotated pair: equal runs, the first axis with what is left over."""
    each = rot // 2 // naxes
    return [0] * (rot // 2 - each * (naxes - 1)) + [a for a in range(1, naxes) for _ in range(each)]


def _rope_inputs(m, s, case, tokens, dtype):
    D, rot = case["D"], case["rot"]
    s["inv_freq"] = m.inv_freq(rot)
    wtype = torch.float32 if case.get("wtype") == "fp32" else dtype
    for n in ("qw", "kw"):
        s[n] = m.normal((D,), wtype, 0.1, 1.0) if case["norm"] else None


def _prepare_norm_rope(case, m, s):
    B, S, Hq, Hk, D, naxes = (case[n] for n in ("B", "S", "Hq", "Hk", "D", "naxes"))
    dtype = DTYPES[case["dtype"]]
    qkv = m.normal((B, S, (Hq + 2 * Hk) * D), dtype)
    s["q"], s["k"] = qkv[..., : Hq * D].view(B, S, Hq, D), qkv[..., Hq * D : (Hq + Hk) * D].view(B, S, Hk, D)
    _rope_inputs(m, s, case, S, dtype)
    if naxes == 1:
        s["axes"], s["positions"] = None, torch.arange(S, device=m.device) + m.ints(0, 100000, 1)[0]
    else:
        s["axes"] = _frequency_axes(case["rot"], naxes)
        n, w = torch.arange(S, device=m.device), max(1, round(S ** (1.0 / naxes)))
        grid = [n // w ** (naxes - 1), n // w % w] if naxes == 2 else [n // w ** 2, n // w % w, n % w]
        s["positions"] = torch.stack(grid[:naxes])[:, None] + m.tensor(m.ints(0, 64, naxes), torch.int64)[:, None, None]
    s["interleaved"], s["train"] = case["interleaved"], case["train"]
    if case["train"]:
        s["gq"], s["gk"] = m.normal((B, S, Hq, D), dtype), m.normal((B, S, Hk, D), dtype)
        s["leaves"] = []
        for n in ("q", "k", "qw", "kw"):
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_(True)
                s["leaves"].append(s[n])


def _page_tables(m, pages, width):
    """A (B, width) table of distinct pages, -1 behind a request's last one, and the pages that the pool has left."""
    B, total = len(pages), sum(pages)
    pool = total + max(8, total // 8)
    perm = torch.randperm(pool, generator=m.g, device=m.device, dtype=torch.int32)
    n = m.tensor(pages, torch.int64)
    first = torch.cumsum(n, 0) - n
    i = torch.arange(width, device=m.device)
    table = torch.where(i < n[:, None], perm[(first[:, None] + i).clamp_(max=pool - 1)], -1)
    return table.int().contiguous(), perm[total:].clone(), pool


def _prepare_append(case, m, s):
    N, Hq, Hk, D, page, R = (case[n] for n in ("N", "Hq", "Hk", "D", "page", "R"))
    dtype = DTYPES[case["dtype"]]
    qkv = m.normal((N, (Hq + 2 * Hk) * D), dtype)
    s["q"] = qkv[:, : Hq * D].view(N, Hq, D)
    s["k"] = qkv[:, Hq * D : (Hq + Hk) * D].view(N, Hk, D)
    s["v"] = qkv[:, (Hq + Hk) * D :].view(N, Hk, D)
    _rope_inputs(m, s, case, N, dtype)
    pages = -(-N // page) * 5 // 4 + 2
    s["key_cache"], s["value_cache"] = (torch.zeros(pages, page, Hk, D, dtype=dtype, device=m.device) for _ in range(2))
    order = torch.randperm(pages, generator=m.g, device=m.device)
    n = torch.arange(N, device=m.device)
    slots = order[n // page] * page + n % page
    # padding behind the last request, and within a batch that was filled up
    s["slots"] = torch.where((n % 97 == 96) | (n >= N - N // 50), -1, slots)
    s["positions"] = (n % 4099 + m.ints(0, 30000, 1)[0]).int()
    s["k_bias"] = m.normal((N, Hk, R), dtype) if R else None
    s["bias_cache"] = torch.zeros(pages, page, Hk, R, dtype=dtype, device=m.device) if R else None


def _tree_parents(m, lengths):
    """A parent for every drafted token: one of the eight before it, or the context (-1) for the first of a request."""
    N = sum(lengths)
    n = m.tensor(lengths, torch.int64)
    start = torch.cumsum(n, 0) - n
    t = torch.arange(N, device=m.device) - torch.repeat_interleave(start, n, output_size=N)
    back = torch.randint(1, 9, (N,), generator=m.g, device=m.device)
    return torch.clamp(t - back, min=-1).int()


def _prepare_plan(case, m, s):
    B, T, L, page = (case[n] for n in ("B", "T", "L", "page"))
    lens, new = m.lengths(L // 4, L, B), m.lengths((T + 1) // 2, T, B)
    held = [-(-x // page) for x in lens]
    width = max(-(-(a + b) // page) for a, b in zip(lens, new)) + 1
    table, free, _ = _page_tables(m, held, width)
    need = sum(-(-(a + b) // page) for a, b in zip(lens, new)) - sum(held)
    s["table"] = table
    # the pool's free pages: enough for the step and some more, in any order; page numbers above those in use
    s["free_pages"] = torch.cat([free, sum(held) + free.numel() + torch.randperm(need + 16, generator=m.g, device=m.device).int()])
    s["free_count"] = m.tensor([s["free_pages"].numel() - 8])
    s["held"], s["lens"], s["new"], s["zero"] = m.tensor(held), m.tensor(lens), m.tensor(new), m.tensor([0] * B)
    s["page"], s["T"], s["tree"] = page, T, case["tree"]
    # a batch that was filled up with rows of no request
    s["N"] = sum(new) + sum(new) // 16
    s["parents"] = torch.cat([_tree_parents(m, new), torch.full((s["N"] - sum(new),), -1, dtype=torch.int32, device=m.device)]) if case["tree"] else None


def _slopes(H, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device=device)


def _prepare_attend(case, m, s):
    B, T, L, Hq, Hk, D, page, R = (case[n] for n in ("B", "T", "L", "Hq", "Hk", "D", "page", "R"))
    dtype = DTYPES[case["dtype"]]
    lens, new = [L] + m.lengths(L // 4, L, B - 1), m.lengths((T + 1) // 2, T, B)
    pages = [-(-(a + b) // page) for a, b in zip(lens, new)]
    s["table"], _, pool = _page_tables(m, pages, max(pages) + 1)
    N = sum(new)
    s["key_cache"], s["value_cache"] = m.normal((pool, page, Hk, D), dtype), m.normal((pool, page, Hk, D), dtype)
    s["q"] = m.normal((N, Hq, D), dtype)
    s["lens"] = m.tensor(lens)
    s["cu"] = m.tensor([sum(new[:b]) for b in range(B + 1)])
    s["host_lens"], s["host_new"], s["T"], s["L"] = lens, new, max(new), max(a + b for a, b in zip(lens, new))
    s["tree_mask"] = s["positions"] = None
    if case["tree"]:
        s["tree_mask"], depth = _ancestors(_tree_parents(m, new), s["cu"], s["T"])
        token = torch.arange(N, device=m.device)
        s["positions"] = s["lens"][torch.searchsorted(s["cu"][1:].long(), token, right=True)] + depth
    s["slopes"] = _slopes(Hq, m.device) if case["bias"] == "slopes" else None
    s["q_bias"] = s["bias_cache"] = None
    if R:
        s["q_bias"], s["bias_cache"] = m.normal((N, Hq, R), dtype, R ** -0.5), m.normal((pool, page, Hk, R), dtype)
    s["page"], s["scale"] = page, 1.0 / math.sqrt(D)


def prepare(case, seed):
    m, s = _Make(seed), {"op": case["op"]}
    {"norm_rope": _prepare_norm_rope, "append": _prepare_append, "plan": _prepare_plan, "attend": _prepare_attend}[case["op"]](case, m, s)
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _norm_rope(x, positions, inv_freq, weight, axes, interleaved, eps=1e-6):
    """x (B, S, H, D) or (S, H, D); positions (S), or with axes (A, B | 1, S); the result in 32 bits."""
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * weight.float()
    half = inv_freq.numel()
    per_pair = positions[..., None] if axes is None else positions[axes].movedim(0, -1)
    angle = per_pair.double() * inv_freq.double()
    cos, sin = torch.cos(angle).float().unsqueeze(-2), torch.sin(angle).float().unsqueeze(-2)
    turned, rest = y[..., : 2 * half], y[..., 2 * half :]
    if interleaved:
        lo, hi = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([lo * cos - hi * sin, hi * cos + lo * sin], -1).flatten(-2)
    else:
        lo, hi = turned[..., :half], turned[..., half:]
        turned = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    return torch.cat([turned, rest], -1)


def _ancestors(parents, cu, T):
    """Bit j of word (n, j // 64): token j of n's request is n or before it on its path; and the depth of each token.  With A
    the matrix of parents, (1 - A)^-1 = 1 + A + A^2 + ... has a one for every ancestor."""
    N, words = parents.numel(), -(-T // 64)
    token = torch.arange(N, device=parents.device)
    req = torch.searchsorted(cu[1:].long(), token, right=True).clamp(max=cu.numel() - 2)
    t = token - cu.long()[req]
    inside = token < cu[-1]
    A = torch.zeros(cu.numel() - 1, T + 1, T + 1, dtype=torch.float64, device=parents.device)
    # row and column T take what no token owns
    A.index_put_((req, torch.where(inside, t, T), torch.where(inside & (parents >= 0), parents.long(), T)),
                 torch.ones((), dtype=torch.float64, device=parents.device))
    A = A[:, :T, :T]
    one = torch.eye(T, dtype=torch.float64, device=parents.device)
    paths = torch.linalg.solve_triangular(one - A, one.expand_as(A), upper=False, unitriangular=True).round().long()
    paths = torch.where(inside[:, None], paths[req, t.clamp(0, T - 1)], 0)
    depth = (paths.sum(-1) - 1).clamp(min=0).int()
    bits = torch.nn.functional.pad(paths, (0, 64 * words - T)).view(N, words, 64)
    return (bits << torch.arange(64, device=parents.device)).sum(-1), depth


def _plan_plain(s, new):
    """One step: page counts follow the lengths, the stack of free pages follows the page counts."""
    table, held, free, count, lens, page, N = (s[n] for n in ("table", "held", "free_pages", "free_count", "lens", "page", "N"))
    B, width = table.shape
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0, dtype=torch.int32)])
    need = (lens + new + page - 1) // page
    back, more = (held - need).clamp(min=0).long(), (need - held).clamp(min=0).long()
    col = torch.arange(width, device=table.device)
    # pages given back, the first of them on top of the stack
    first = torch.cumsum(back, 0) - back
    top = count.long() + back.sum()
    gone = (col >= need[:, None]) & (col < held[:, None])
    at = torch.where(gone, top - 1 - (first[:, None] + col - need[:, None]), free.numel())
    grown = torch.cat([free, free.new_zeros(1)])
    grown.scatter_(0, at.flatten(), table.flatten())
    free.copy_(grown[:-1])
    # pages taken, from the top down
    first = torch.cumsum(more, 0) - more
    fresh = (col >= held[:, None]) & (col < need[:, None])
    at = torch.where(fresh, top - 1 - (first[:, None] + col - held[:, None]), 0)
    table.copy_(torch.where(fresh, free[at], table))
    held.copy_(need)
    count.copy_(top - more.sum())
    token = torch.arange(N, device=table.device)
    req = torch.searchsorted(cu[1:].long(), token, right=True)
    inside = req < B
    req = req.clamp(max=B - 1)
    pos = lens.long()[req] + token - cu.long()[req]
    slots = torch.where(inside, table[req, (pos // page).clamp(0, width - 1)].long() * page + pos % page, -1)
    mask = None
    if s["parents"] is not None and new is not s["zero"]:
        mask, depth = _ancestors(s["parents"], cu, s["T"])
        pos = lens.long()[req] + depth
    return slots, torch.where(inside, pos, 0).int(), cu, mask


def _attend_plain(s):
    q, cu, lens, T, L, page = s["q"], s["cu"].long(), s["lens"].long(), s["T"], s["L"], s["page"]
    (N, Hq, D), Hk, B = q.shape, s["key_cache"].shape[2], lens.numel()
    G, dev = Hq // Hk, q.device
    new = cu[1:] - cu[:-1]
    t, j = torch.arange(T, device=dev), torch.arange(L, device=dev)
    token = torch.where(t < new[:, None], cu[:-1, None] + t, 0)
    known = j < (lens + new)[:, None]
    slot = torch.where(known, s["table"].long()[:, (j // page).clamp(max=s["table"].shape[1] - 1)] * page + j % page, 0)
    k, v = s["key_cache"].flatten(0, 1)[slot].float(), s["value_cache"].flatten(0, 1)[slot].float()
    rows = q.float()[token].view(B, T, Hk, G, D)
    logits = torch.einsum("btkgd,blkd->bkgtl", rows, k) * s["scale"]
    # (B, T, L): drafted key j - lens on the path of token t, or not after it
    drafted = j - lens[:, None]
    if s["tree_mask"] is not None:
        words = s["tree_mask"][token]
        bit = drafted.clamp(0, 64 * words.shape[-1] - 1)[:, None].expand(B, T, L)
        on_path = (words.gather(2, bit // 64) >> (bit % 64)) & 1 == 1
    else:
        on_path = drafted[:, None] <= t[:, None]
    visible = known[:, None] & ((drafted < 0)[:, None] | on_path)
    if s["slopes"] is not None:
        depth = s["positions"].long()[token] if s["positions"] is not None else lens[:, None] + t
        at = torch.where(drafted < 0, j, depth.gather(1, drafted.clamp(0, T - 1)))
        logits = logits + s["slopes"].view(Hk, G, 1, 1) * (at[:, None] - depth[:, :, None])[:, None, None].float()
    if s["q_bias"] is not None:
        qb, kb = s["q_bias"].float()[token].view(B, T, Hk, G, -1), s["bias_cache"].flatten(0, 1)[slot].float()
        logits = logits + torch.einsum("btkgr,blkr->bkgtl", qb, kb)
    logits = logits.masked_fill(~visible[:, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(logits - top)
    o = torch.einsum("bkgtl,blkd->btkgd", p, v) / p.sum(-1).clamp(min=1e-30).permute(0, 3, 1, 2)[..., None]
    # back to flat tokens
    req = torch.searchsorted(cu[1:], torch.arange(N, device=dev), right=True)
    return o[req, torch.arange(N, device=dev) - cu[req]].reshape(N, Hq, D).to(q.dtype)


def _run_plain(s):
    if s["op"] == "norm_rope":
        rot = (s["positions"], s["inv_freq"])
        more = (s["axes"], s["interleaved"])
        if not s["train"]:
            with torch.no_grad():
                return tuple(_norm_rope(s[n], *rot, s[w], *more).to(s[n].dtype) for n, w in (("q", "qw"), ("k", "kw")))
        q, k = (_norm_rope(s[n], *rot, s[w], *more).to(s[n].dtype) for n, w in (("q", "qw"), ("k", "kw")))
        return (q, k) + torch.autograd.grad((q, k), s["leaves"], (s["gq"], s["gk"]))
    if s["op"] == "append":
        q, k = (_norm_rope(s[n], s["positions"], s["inv_freq"], s[w], None, False).to(s["q"].dtype) for n, w in (("q", "qw"), ("k", "kw")))
        caches = [s[n] for n in ("key_cache", "value_cache", "bias_cache") if s[n] is not None]
        at = s["slots"].clamp(min=0)
        keep = (s["slots"] >= 0)[:, None, None]
        # padding rows write nothing: their place gets what a slot of its own already holds
        spare = torch.where(s["slots"] >= 0, at, at.amax())
        row = torch.where(keep[:, 0, 0], torch.arange(at.numel(), device=at.device), torch.argmax(at))
        _put(caches[0], spare, k[row])
        _put(caches[1], spare, s["v"][row])
        if s["k_bias"] is not None:
            _put(caches[2], spare, s["k_bias"][row])
        return (q, *caches)
    if s["op"] == "plan":
        step = _plan_plain(s, s["new"])
        _plan_plain(s, s["zero"])
        return tuple(x for x in step if x is not None) + (s["table"], s["held"], s["free_pages"], s["free_count"])
    return _attend_plain(s)


def _put(cache, slots, rows):
    cache.flatten(0, 1).index_copy_(0, slots, rows)


def run(state):
    """One pass.  A plan's pass is a step that takes pages and the step that gives them back, so that it can be repeated."""
    s = state
    if not own:
        return _run_plain(s)
    import flashbias_b200 as fb

    if s["op"] == "norm_rope":
        if not s["train"]:
            with torch.no_grad():
                return fb.norm_rope_func(s["q"], s["k"], s["positions"], s["inv_freq"], s["qw"], s["kw"], s["axes"], s["interleaved"])
        q, k = fb.norm_rope_func(s["q"], s["k"], s["positions"], s["inv_freq"], s["qw"], s["kw"], s["axes"], s["interleaved"])
        return (q, k) + torch.autograd.grad((q, k), s["leaves"], (s["gq"], s["gk"]))
    if s["op"] == "append":
        q = fb.paged_append(s["q"], s["k"], s["v"], s["key_cache"], s["value_cache"], s["slots"], s["positions"], s["inv_freq"],
                            s["qw"], s["kw"], k_bias=s["k_bias"], bias_cache=s["bias_cache"])
        return tuple(x for x in (q, s["key_cache"], s["value_cache"], s["bias_cache"]) if x is not None)
    if s["op"] == "plan":
        pool = (s["table"], s["held"], s["free_pages"], s["free_count"])
        step = fb.paged_plan(*pool, s["lens"], s["new"], s["page"], s["N"], parents=s["parents"])
        fb.paged_plan(*pool, s["lens"], s["zero"], s["page"], s["N"])
        return tuple(x for x in (step.slots, step.positions, step.cu_tokens, step.tree_mask) if x is not None) + pool
    return fb.flash_bias_paged_func(s["q"], s["key_cache"], s["value_cache"], s["table"], s["lens"], s["cu"], s["tree_mask"],
                                    s["positions"], s["slopes"], s["q_bias"], s["bias_cache"], s["scale"])


# ---------------------------------------------------------------------------------------------------------------
# the work of a pass, and its results in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    """Bytes: every input read once, every output written once.  Flop: of the products (attention), or of the norm and the
    rotation (about 8 a value forward, 20 backward)."""
    c = case
    if c["op"] == "norm_rope":
        values = c["B"] * c["S"] * (c["Hq"] + c["Hk"]) * c["D"]
        passes = 5 if c["train"] else 2
        return {"bytes": float(2 * values * passes + 8 * c["S"] * c["naxes"]), "flops": float(values * (28 if c["train"] else 8))}
    if c["op"] == "append":
        live = c["N"] - c["N"] // 50
        values = 2 * c["N"] * c["Hq"] * c["D"] + live * c["Hk"] * (4 * c["D"] + 2 * c["R"])
        return {"bytes": float(2 * values + 12 * c["N"]), "flops": float(8 * c["N"] * (c["Hq"] + c["Hk"]) * c["D"])}
    if c["op"] == "plan":
        new = c["B"] * (c["T"] + (c["T"] + 1) // 2) / 2
        pages = new / c["page"] + c["B"] / 2
        return {"bytes": float(new * (12 + (12 if c["tree"] else 0)) + 24 * c["B"] + 16 * pages), "flops": float(10 * new)}
    lens = (c["L"] + (c["B"] - 1) * 0.625 * c["L"]) / c["B"]
    new = (c["T"] + (c["T"] + 1) // 2) / 2
    keys = c["B"] * (lens + new)
    nbytes = 2 * keys * c["Hk"] * (2 * c["D"] + c["R"]) + 2 * c["B"] * new * c["Hq"] * (2 * c["D"] + c["R"])
    return {"bytes": float(nbytes), "flops": float(keys * new * c["Hq"] * (4 * c["D"] + 2 * c["R"]))}


def _exact_norm_rope(x, weight, positions, inv_freq, axes, interleaved, dout=None):
    """In 64 bits, the rotation as a complex product; with dout the gradients of x and weight too, by their formulas."""
    x, half = x.detach().double(), inv_freq.numel()
    r = torch.rsqrt((x ** 2).mean(-1, keepdim=True) + 1e-6) if weight is not None else torch.ones_like(x[..., :1])
    w = weight.detach().double() if weight is not None else torch.ones(x.shape[-1], dtype=torch.float64, device=x.device)
    pos = positions.double()[..., None].expand(*positions.shape, half) if axes is None else positions.double()[list(axes)].movedim(0, -1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), pos * inv_freq.double())[..., None, :]

    def rotate(y, by):
        z = y[..., : 2 * half].unflatten(-1, (half, 2) if interleaved else (2, half))
        z = torch.complex(z[..., 0], z[..., 1]) if interleaved else torch.complex(z[..., 0, :], z[..., 1, :])
        z = z * by
        z = torch.stack([z.real, z.imag], -1 if interleaved else -2).flatten(-2)
        return torch.cat([z, y[..., 2 * half :]], -1)

    out = rotate(x * r * w, turn)
    if dout is None:
        return out
    g = rotate(dout.double(), turn.conj())
    if weight is None:
        return out, g, None
    dx = r * (w * g - x * r ** 2 * (w * g * x).mean(-1, keepdim=True))
    return out, dx, (g * x * r).flatten(0, -2).sum(0)


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers throughout
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        more = (s["positions"], s["inv_freq"], s["axes"], s["interleaved"])
        if not s["train"]:
            return tuple(_exact_norm_rope(s[n], s[w], *more) for n, w in (("q", "qw"), ("k", "kw")))
        q, dq, dqw = _exact_norm_rope(s["q"], s["qw"], *more, s["gq"])
        k, dk, dkw = _exact_norm_rope(s["k"], s["kw"], *more, s["gk"])
        return (q, k, dq, dk) + ((dqw, dkw) if case["norm"] else ())
    if case["op"] == "append":
        more = (s["positions"], s["inv_freq"], None, False)
        live = s["slots"] >= 0
        k = _exact_norm_rope(s["k"], s["kw"], *more)
        filled = [(s["key_cache"], k), (s["value_cache"], s["v"])] + ([(s["bias_cache"], s["k_bias"])] if case["R"] else [])
        caches = []
        for cache, rows in filled:
            flat = torch.zeros(cache.shape, dtype=torch.float64, device=cache.device)
            flat.flatten(0, 1)[s["slots"][live]] = rows.double()[live]
            caches.append(flat)
        return (_exact_norm_rope(s["q"], s["qw"], *more), *caches)
    Hq, Hk, D, page = (case[n] for n in ("Hq", "Hk", "D", "page"))
    G, out, n0 = Hq // Hk, [], 0
    for b, (ctx, new) in enumerate(zip(s["host_lens"], s["host_new"])):
        total = ctx + new
        pages = s["table"][b, : -(-total // page)].long()
        k, v = (s[c][pages].reshape(-1, Hk, D)[:total].double().movedim(1, 0) for c in ("key_cache", "value_cache"))
        q = s["q"][n0 : n0 + new].double().view(new, Hk, G, D).permute(1, 2, 0, 3)
        z = (q.reshape(Hk, G * new, D) @ k.mT).view(Hk, G, new, total) * s["scale"]
        if s["q_bias"] is not None:
            qb = s["q_bias"][n0 : n0 + new].double().view(new, Hk, G, -1).permute(1, 2, 0, 3)
            kb = s["bias_cache"][pages].reshape(pages.numel() * page, Hk, -1)[:total].double().movedim(1, 0)
            z = z + qb @ kb.mT[:, None]
        pos = s["positions"][n0 : n0 + new].double() if s["positions"] is not None else ctx + torch.arange(new, device=z.device).double()
        if s["slopes"] is not None:
            key_pos = torch.cat([torch.arange(ctx, device=z.device).double(), pos])
            z = z + s["slopes"].double().view(Hk, G, 1, 1) * (key_pos[None, :] - pos[:, None])
        if s["tree_mask"] is not None:
            word = s["tree_mask"][n0 : n0 + new]
            sees = torch.stack([(word[:, i // 64] >> (i % 64)) & 1 for i in range(new)], 1) == 1
        else:
            sees = torch.ones(new, new, dtype=torch.bool, device=z.device).tril()
        z[..., ctx:].masked_fill_(~sees, -math.inf)
        o = torch.softmax(z, -1) @ v[:, None]
        out.append(o.permute(2, 0, 1, 3).reshape(new, Hq, D))
        n0 += new
    return torch.cat(out)
