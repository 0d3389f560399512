"""Keys, values and factors on their way into pages: what is written, and what is left as it was."""
import pytest
import torch

from flashbias_b200 import check_device_status, norm_rope_func, paged_append

pytestmark = pytest.mark.gpu


def inputs(N, Hq, Hk, D, rot, R, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(N, (Hq + 2 * Hk) * D, generator=g).to(dtype).cuda()
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, Hk * D, Hk * D], 1))
    w = [(1.0 + 0.2 * torch.randn(D, generator=g)).cuda() for _ in range(2)]
    f = (10000.0 ** (-torch.arange(0, rot, 2).double() / max(rot, 1))).float().cuda()
    pos = torch.randint(0, 5000, (N,), generator=g).cuda()
    return q, k, v, w, f, pos, torch.randn(N, Hk, R, generator=g).to(dtype).cuda() if R else None


def check(q, k, v, w, f, pos, kb, page, pages, slots, order, il=False, axes=None):
    """Against norm_rope_func, which has its own tests: the same bits in the slots, everything else untouched."""
    N, Hk, D = k.shape
    R = 0 if kb is None else kb.shape[2]

    def cache(heads, cols):
        c = torch.randn(pages, page, heads, cols, device="cuda").to(k.dtype)
        return c.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) if order == "hpd" else c

    kc, vc, bc = cache(Hk, D), cache(Hk, D), cache(kb.shape[1], R) if R else None
    want = [c.clone() if c is not None else None for c in (kc, vc, bc)]
    got = paged_append(q, k, v, kc, vc, slots, pos, f, w[0], w[1], axes, il, k_bias=kb, bias_cache=bc)
    torch.cuda.synchronize()
    check_device_status()
    p4 = None if pos is None else pos[..., None, :]
    wk, wq = norm_rope_func(k[None], None if q is None else q[None], p4, f, w[1], w[0], axes, il)
    for n, s in enumerate(slots.tolist()):
        if s >= 0:
            want[0][s // page, s % page], want[1][s // page, s % page] = wk[0, n], v[n]
            if R:
                want[2][s // page, s % page] = kb[n]
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]) and (not R or torch.equal(bc, want[2]))
    assert (got is None) if q is None else torch.equal(got, wq[0])


@pytest.mark.parametrize("N,Hq,Hk,D,rot,page,R,dtype,order", [
    (1, 8, 2, 128, 128, 16, 0, torch.bfloat16, "phd"),
    (33, 4, 4, 64, 64, 16, 2, torch.float16, "phd"),
    (100, 6, 2, 80, 20, 7, 5, torch.bfloat16, "hpd"),
    (257, 3, 1, 96, 96, 64, 8, torch.bfloat16, "hpd"),
    (50, 2, 2, 20, 20, 1, 3, torch.float16, "phd"),
    (40, 2, 1, 7, 6, 5, 1, torch.float16, "phd"),
    (700, 16, 8, 128, 64, 32, 16, torch.float16, "phd"),
])
def test_rows_land_in_their_slots(N, Hq, Hk, D, rot, page, R, dtype, order):
    q, k, v, w, f, pos, kb = inputs(N, Hq, Hk, D, rot, R, dtype, N)
    pages = -(-N // page) + 3
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(N))[:N]
    slots[::5] = -1
    slots[N // 2:N // 2 + 1] = -12345
    check(q, k, v, w, f, pos, kb, page, pages, slots.cuda(), order)
    check(q, k, v, w, f, pos.int(), kb, page, pages, slots.int().cuda(), order, il=True)


def test_plain_write_and_shared_bias_head():
    q, k, v, _, _, _, kb = inputs(30, 4, 4, 64, 64, 4, torch.float16, 1)
    slots = torch.arange(30, device="cuda") + 5
    check(None, k, v, [None, None], None, None, kb[:, :1], 16, 4, slots, "phd")
    check(q, k, v, [None, None], None, None, kb[:, :1], 16, 4, slots, "hpd")


def test_several_axes_and_strided_slots():
    q, k, v, w, f, pos, _ = inputs(30, 4, 2, 64, 64, 0, torch.bfloat16, 2)
    axes = [0] * 10 + [1] * 11 + [2] * 11
    slots = torch.arange(60, device="cuda")[::2]
    check(q, k, v, w, f, torch.stack([pos, pos + 3, pos // 2]), None, 16, 5, slots, "phd", axes=axes)


def test_unaligned_inputs_and_caches():
    q, k, v, w, f, pos, _ = inputs(21, 4, 2, 64, 64, 0, torch.float16, 3)
    shift = lambda t: torch.cat([t, t[..., :1]], -1)[..., 1:]  # noqa: E731
    check(shift(q), shift(k), shift(v), w, f, pos, None, 16, 4, torch.arange(21, device="cuda"), "phd")
    big = torch.zeros(4, 16, 2, 65, device="cuda", dtype=torch.float16)
    kc, vc = big[..., 1:], torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.float16)
    paged_append(None, k, v, kc, vc, torch.arange(21, device="cuda"))
    assert torch.equal(kc.flatten(0, 1)[:21], k) and torch.equal(vc.flatten(0, 1)[:21], v) and (big[..., 0] == 0).all()


def test_values_that_are_copied_keep_their_bits():
    q, k, v, _, _, _, _ = inputs(8, 2, 2, 64, 64, 0, torch.bfloat16, 4)
    v = v.clone()
    v[0, 0, 0], v[0, 0, 1], v[0, 0, 2], v[0, 0, 3] = float("nan"), float("inf"), 1e-39, -0.0
    kc, vc = (torch.zeros(1, 8, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    paged_append(None, v, v, kc, vc, torch.arange(8, device="cuda"))
    assert torch.equal(vc[0].view(torch.int16), v.view(torch.int16)) and torch.equal(kc[0].view(torch.int16), v.view(torch.int16))


def test_a_slot_behind_the_cache_is_reported_and_not_written():
    q, k, v, w, f, pos, _ = inputs(4, 2, 2, 64, 64, 0, torch.float16, 5)
    pool = torch.zeros(6, 8, 2, 64, device="cuda", dtype=torch.float16)
    kc, vc = pool[:2], torch.zeros_like(pool[:2])
    out = paged_append(q, k, v, kc, vc, torch.tensor([16, 3, 2 ** 40, 17], device="cuda"), pos, f)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="out of range"):
        check_device_status()
    assert (pool[2:] == 0).all() and torch.equal(vc[0, 3], v[1]) and vc.count_nonzero() == v[1].count_nonzero()
    assert torch.equal(out, norm_rope_func(q[None], None, pos, f)[0][0])


def test_no_tokens_and_versions():
    q, k, v, _, _, _, _ = inputs(4, 2, 2, 64, 64, 0, torch.float16, 6)
    kc, vc = (torch.zeros(2, 8, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    slots = torch.arange(4, device="cuda")
    assert paged_append(q[:0], k[:0], v[:0], kc, vc, slots[:0]).shape == (0, 2, 64)
    before = kc._version
    paged_append(q, k, v, kc, vc, slots)
    assert kc._version > before  # autograd sees that a tensor it may have saved has changed


def test_captured_append():
    q, k, v, w, f, pos, _ = inputs(9, 4, 2, 64, 64, 0, torch.float16, 7)
    kc, vc = (torch.zeros(4, 8, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    slots = torch.arange(9, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_append(q, k, v, kc, vc, slots, pos, f, *w)
    slots += 20
    graph.replay()
    ref = [torch.zeros_like(kc) for _ in range(2)]
    want = paged_append(q, k, v, *ref, slots, pos, f, *w)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(kc, ref[0]) and torch.equal(vc, ref[1])


@pytest.mark.parametrize("bad", [dict(k=torch.zeros(4, 2, 64)), dict(v=torch.zeros(4, 1, 64).half()), dict(q=torch.zeros(3, 2, 64).half()),
                                 dict(key_cache=torch.zeros(2, 8, 2, 64)), dict(key_cache=torch.zeros(2, 8, 1, 64).half()),
                                 dict(value_cache=torch.zeros(3, 8, 2, 64).half()), dict(key_cache=torch.zeros(2, 8, 64, 2).half().transpose(2, 3)),
                                 dict(value_cache=torch.zeros(2, 8, 1, 64).half().expand(2, 8, 2, 64)), dict(slots=torch.arange(3)),
                                 dict(slots=torch.zeros(4)), dict(k_bias=torch.zeros(4, 2, 3).half()),
                                 dict(k_bias=torch.zeros(4, 2, 3).half(), bias_cache=torch.zeros(2, 8, 1, 3).half()),
                                 dict(k_bias=torch.zeros(4, 3, 3).half(), bias_cache=torch.zeros(2, 8, 3, 3).half()),
                                 dict(positions=torch.arange(4)), dict(positions=torch.arange(3), inv_freq=torch.ones(4))], ids=lambda b: "-".join(b))
def test_refusals(bad):
    args = dict(q=torch.zeros(4, 2, 64).half(), k=torch.zeros(4, 2, 64).half(), v=torch.zeros(4, 2, 64).half(),
                key_cache=torch.zeros(2, 8, 2, 64).half(), value_cache=torch.zeros(2, 8, 2, 64).half(), slots=torch.arange(4))
    dev = {n: v.cuda() for n, v in args.items()}
    paged_append(**dev)
    with pytest.raises(AssertionError):
        paged_append(**{**dev, **{n: v.cuda() if n != "value_cache" or v.stride(2) else v[:, :, :1].cuda().expand(v.shape) for n, v in bad.items()}})


def test_rows_that_lie_in_a_cache_are_refused():
    """Moving accepted tokens up: from a copy, because a slot may be another token's source; one arena for everything is fine."""
    arena = torch.randn(2 * 4 * 8 * 2 * 16 + 4 * 2 * 16, generator=torch.Generator().manual_seed(5)).half().cuda()
    kc, vc = arena[:1024].view(4, 8, 2, 16), arena[1024:2048].view(4, 8, 2, 16)
    fresh = arena[2048:].view(4, 2, 16)
    slots = torch.tensor([3, 4, 5, 6], device="cuda")
    k, v = kc.view(32, 2, 16)[4:8], vc.view(32, 2, 16)[4:8]
    for bad in ((k, fresh), (fresh, v), (fresh, k), (v, fresh)):
        with pytest.raises(AssertionError):
            paged_append(None, *bad, kc, vc, slots)
    paged_append(None, fresh, fresh, kc, vc, slots)
    assert torch.equal(kc.view(32, 2, 16)[3:7], fresh) and torch.equal(vc.view(32, 2, 16)[3:7], fresh)
    want = kc.view(32, 2, 16)[4:8].clone(), vc.view(32, 2, 16)[4:8].clone()
    paged_append(None, *want, kc, vc, slots)
    assert torch.equal(kc.view(32, 2, 16)[3:7], want[0]) and torch.equal(vc.view(32, 2, 16)[3:7], want[1])


def test_caches_that_share_elements_are_refused_and_interleaved_ones_are_not():
    _, k, v, _, _, _, kb = inputs(9, 2, 2, 16, 0, 16, torch.float16, 11)
    pool = torch.zeros(6, 2, 8, 2, 16, device="cuda", dtype=torch.float16)  # keys beside values, page by page
    slots = torch.arange(9, device="cuda") + 5
    for kc, vc in ((pool[:, 0], pool[:, 0]), (pool.flatten(0, 1)[:6], pool.flatten(0, 1)[2:8])):
        with pytest.raises(AssertionError, match="share"):
            paged_append(None, k, v, kc, vc, slots)
    other = torch.zeros(6, 8, 2, 16, device="cuda", dtype=torch.float16)
    for bc in (pool[:, 0], pool[:, 1]):
        with pytest.raises(AssertionError, match="share"):
            paged_append(None, k, v, pool[:, 0], pool[:, 1], slots, k_bias=kb, bias_cache=bc)
    assert pool.count_nonzero() == 0
    paged_append(None, k, v, pool[:, 0], pool[:, 1], slots, k_bias=kb, bias_cache=other)
    torch.cuda.synchronize()
    for c, rows in ((pool[:, 0], k), (pool[:, 1], v), (other, kb)):
        assert torch.equal(c.flatten(0, 1)[5:14], rows) and c.count_nonzero() == rows.count_nonzero()
    wide = torch.zeros(6, 8, 2, 32, device="cuda", dtype=torch.float16)  # ... column by column
    paged_append(None, k, v, wide[..., :16], wide[..., 16:], slots)
    assert torch.equal(wide.flatten(0, 1)[5:14], torch.cat([k, v], -1))
