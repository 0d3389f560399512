"""Attention over pages against 64 bits: single tokens, runs, trees, head groups, biases, page sizes, layouts; places that no
request owns hold NaN throughout."""
import math

import pytest
import torch

from flashbias_b200 import check_device_status, flash_bias_alibi_func, flash_bias_paged_func
from oracle import serving_oracle as orc
from tests.serving_helpers import FP32, assert_within, half_step, paged_inputs, tree

pytestmark = pytest.mark.gpu


def dev(kw):
    return {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in kw.items()}


def bounds(want, weight, size, D, dtype):
    """o: the result is rounded once, the probabilities too (the tensor path), the fp32 logits by D + 64 steps of the sum of
    magnitudes behind them, the exponentials by 2^-21; lse: the logits' error and a few steps of its own."""
    logit = (D + 64) * FP32 * (size + 1.0)
    u = half_step(dtype)
    tiny = torch.finfo(dtype).smallest_normal * u
    o = u * want.abs() + (1.01 * u + 2 * logit[..., None] + 2.0 ** -19) * weight + tiny
    return o, logit


def check(kw, **more):
    kw = {**kw, **more}
    want, lse, weight, size = orc.paged_attention(**{{"block_table": "table", "cu_tokens": "cu", "softmax_scale": "scale"}.get(n, n): v for n, v in kw.items()})
    o, got = flash_bias_paged_func(**dev(kw), return_lse=True)
    torch.cuda.synchronize()
    check_device_status()
    D = kw["q"].shape[2] + (kw["q_bias"].shape[2] if kw.get("q_bias") is not None else 0)
    bo, bl = bounds(want, weight, size, D, kw["q"].dtype)
    assert_within("o", o, want, bo)
    empty = lse == -math.inf
    assert (got.cpu()[empty] == -math.inf).all() and (o.cpu()[empty] == 0).all()
    # (lse is held in fp32, a few roundings of its own size)
    assert_within("lse", got.cpu()[~empty], lse[~empty], (bl + 8 * FP32 * lse.abs() + 1e-6)[~empty])
    return o


SHAPES = [
    # lens, new, Hq, Hk, D, page
    ([0], [1], 1, 1, 64, 16),                          # the first token of a request
    ([1], [1], 4, 2, 128, 16),
    ([700], [1], 32, 8, 128, 16),
    ([63, 64, 65, 127, 128, 129], [1] * 6, 4, 4, 64, 32),  # ends at the edges of tiles
    ([300, 5, 0, 77], [1, 1, 1, 1], 8, 1, 96, 7),      # page size that divides nothing
    ([200, 31], [2, 5], 4, 2, 32, 1),                  # pages of one place
    ([90, 0, 400], [17, 3, 1], 6, 3, 80, 64),
    ([500], [33], 8, 2, 128, 16),                      # 132 rows per key head
    ([129, 1000], [64, 40], 2, 2, 64, 128),
    ([0, 0], [100, 61], 2, 1, 72, 16),                 # nothing cached
    ([250], [7], 24, 2, 24, 16),
    ([60], [3], 5, 5, 8, 16),
    ([45, 46], [3, 2], 4, 2, 20, 16),                  # head_dim that is no whole number of vectors
    ([30], [4], 2, 1, 7, 4),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "L%sT%sH%d-%dD%dp%d" % ("_".join(map(str, s[0])), "_".join(map(str, s[1])), *s[2:]))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", ["none", "slopes", "factors"])
def test_runs(shape, dtype, bias):
    lens, new, Hq, Hk, D, page = shape
    R = {"none": 0, "slopes": 0, "factors": 3}[bias]
    kw = paged_inputs(lens, new, Hq, Hk, D, page, dtype, sum(lens) + D, R, order="hpd" if page == 16 else "phd")
    if bias == "slopes":
        kw["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)])
    check(kw)


@pytest.mark.parametrize("lens,new,Hq,Hk,D,page", [([100, 0, 33], [9, 5, 64], 4, 2, 64, 16), ([513], [60], 8, 2, 128, 32), ([20, 400], [1, 2], 4, 4, 128, 8),
                                                   ([70, 10], [64, 64], 16, 2, 96, 16), ([40], [5], 2, 1, 20, 16)])
@pytest.mark.parametrize("bias", ["none", "slopes", "factors"])
def test_trees(lens, new, Hq, Hk, D, page, bias):
    kw = paged_inputs(lens, new, Hq, Hk, D, page, torch.bfloat16, 3, 8 if bias == "factors" else 0, 1 if Hk > 1 else None)
    _, mask, depth = tree(new, 4)
    first = torch.repeat_interleave(kw["lens"], torch.tensor(new))
    if bias == "slopes":
        kw["slopes"] = torch.linspace(0.5, 0.01, Hq)
    check(kw, tree_mask=mask, positions=(first + depth).int())
    if bias == "slopes":  # positions without a tree, a tree without positions
        check(kw, positions=(first + depth).int())
        check(kw, tree_mask=mask)


@pytest.mark.parametrize("T,words", [(65, 2), (130, 3), (200, 2), (64, 4)])
def test_masks_of_several_words(T, words):
    kw = paged_inputs([50, 9], [T, 3], 2, 1, 64, 16, torch.float16, 5)
    _, mask, _ = tree([T, 3], 6, words)
    check(kw, tree_mask=mask)


def test_mask_rows_that_see_nothing_and_masks_without_the_token_itself():
    kw = paged_inputs([0, 40, 0], [4, 3, 70], 4, 2, 64, 16, torch.bfloat16, 7)
    mask = torch.randint(-2 ** 62, 2 ** 62, (77, 2), generator=torch.Generator().manual_seed(8))
    mask[0] = 0
    mask[2] = 2
    mask[5] = 0
    mask[30:50] = 0
    o = check(kw, tree_mask=mask)
    assert (o[0] == 0).all() and (o[5] != 0).any()
    check(kw, tree_mask=torch.full((77,), -1, dtype=torch.int64))  # one word as a vector: all of the first 64


def test_tokens_of_no_request_and_refused_requests():
    kw = paged_inputs([30, -1, 12], [2, 3, 1], 4, 2, 64, 16, torch.float16, 9)
    kw["q"] = torch.cat([kw["q"], torch.full((3, 4, 64), float("nan"), dtype=torch.float16)])
    o = check(kw)
    assert (o[2:5] == 0).all() and (o[6:] == 0).all()


def test_values_of_unseen_keys_do_not_count():
    """Drafted keys and values that are infinite or NaN touch only the rows that see them."""
    new = [6, 40]
    kw = paged_inputs([70, 3], new, 4, 2, 64, 16, torch.bfloat16, 10)
    _, mask, _ = tree(new, 11)
    clean = check(kw, tree_mask=mask)
    for b, t, what in ((0, 4, float("nan")), (1, 20, float("inf"))):
        place = int(kw["lens"][b]) + t
        at = int(kw["block_table"][b, place // 16]), place % 16
        kw["key_cache"][at] = what
        kw["value_cache"][at] = what
    o = flash_bias_paged_func(**dev(kw), tree_mask=mask.cuda())
    seen = torch.tensor([bool(mask[n, 0] >> (4 if n < 6 else 20) & 1) for n in range(46)])
    assert torch.equal(o.cpu()[~seen], clean.cpu()[~seen]) and not o.cpu()[seen].isfinite().any()


def test_large_logits_and_scales():
    kw = paged_inputs([200], [3], 2, 2, 64, 16, torch.bfloat16, 12)
    check(kw, softmax_scale=4.0)
    check(kw, softmax_scale=-0.3)
    kw["slopes"] = torch.tensor([50.0, -3.0])  # the newest key, and the oldest, take all
    check(kw)
    kw = paged_inputs([200], [3], 2, 2, 64, 16, torch.bfloat16, 12, R=2)
    kw["bias_cache"].nan_to_num_()[..., 0] = -3.0e38  # every logit is the type's lowest value or below
    kw["q_bias"][..., 0] = 1.0
    o, lse = flash_bias_paged_func(**dev(kw), return_lse=True)
    assert o.isfinite().all() and (lse < -1e38).all()


def test_one_run_equals_the_dense_operator():
    """The whole prompt in one step over an empty cache: causal attention with slopes."""
    T, H, D = 150, 4, 64
    kw = paged_inputs([0], [T], H, H, D, 16, torch.float16, 13)
    pages = kw["block_table"][0, :-(-T // 16)].long()
    k, v = (kw[c][pages].flatten(0, 1)[:T] for c in ("key_cache", "value_cache"))
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.01])
    want = flash_bias_alibi_func(kw["q"][None].cuda(), k[None].cuda(), v[None].cuda(), slopes.cuda(), True)[0]
    got = check(kw, slopes=slopes)
    assert (got.float() - want.float()).abs().max() < 4e-3  # two fp16 results of values up to about three


@pytest.mark.parametrize("T", [1, 40])
def test_bad_pages_are_left_out_and_reported(T):
    kw = paged_inputs([100], [T], 4, 2, 64, 16, torch.float16, 14)
    kw["tree_mask"] = torch.full((T, 1), -1, dtype=torch.int64)
    d = dev(kw)
    pool = kw["key_cache"].shape[0]
    for bad in (-1, pool, 2 ** 31 - 1):
        d["block_table"][0, 2] = bad
        o = flash_bias_paged_func(**d)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="out of range"):
            check_device_status()
        # the other keys' result: their pages moved together, sixteen places fewer
        k2 = dict(kw, block_table=torch.cat([kw["block_table"][:, :2], kw["block_table"][:, 3:]], 1), lens=kw["lens"] - 16)
        want, _, weight, size = orc.paged_attention(k2["q"], k2["key_cache"], k2["value_cache"], k2["block_table"], k2["lens"], k2["cu_tokens"], k2["tree_mask"])
        assert_within("o", o, want, bounds(want, weight, size, 64, torch.float16)[0])


def test_a_table_that_is_too_short_and_offsets_out_of_range():
    kw = paged_inputs([40], [1], 4, 2, 64, 16, torch.float16, 15)
    d = dev(kw)
    d["block_table"] = d["block_table"][:, :2].contiguous()
    o = flash_bias_paged_func(**d)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="out of range"):
        check_device_status()
    assert o.isfinite().all()
    d = dev(kw)
    for cu in ([0, 100], [-5, 1], [7, 3]):
        d["cu_tokens"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        flash_bias_paged_func(**d)  # offsets are held within the tokens
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="out of range"):
            check_device_status()


def test_strided_queries_tables_and_empty_steps():
    kw = paged_inputs([100, 20], [3, 2], 4, 2, 64, 16, torch.bfloat16, 16)
    want = check(kw)
    d = dev(kw)
    d["q"] = torch.cat([d["q"].flatten(1), d["q"].flatten(1)], 1)[:, :256].unflatten(1, (4, 64))
    wide = torch.full((2, 31), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + d["block_table"].shape[1]] = d["block_table"]
    d["block_table"] = wide[:, 2:]
    assert torch.equal(flash_bias_paged_func(**d), want)
    d["q"] = torch.cat([d["q"], d["q"][..., :1]], -1)[..., 1:].roll(1, -1)  # another order in memory, contiguous values
    d["q"] = torch.stack([kw["q"], kw["q"]], -1).cuda()[..., 0]
    assert torch.equal(flash_bias_paged_func(**d), want)
    d["q"], d["cu_tokens"] = d["q"][:0], torch.zeros(3, dtype=torch.int32, device="cuda")
    assert flash_bias_paged_func(**d).shape == (0, 4, 64)


def test_results_repeat_and_streams():
    kw = paged_inputs([3000, 100, 1500], [2, 9, 1], 8, 2, 128, 16, torch.bfloat16, 17)
    d = dev(kw)
    want = flash_bias_paged_func(**d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [flash_bias_paged_func(**d) for _ in range(4)]
    here = [flash_bias_paged_func(**d) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for o in others + here)


def test_a_graph_follows_the_lengths():
    """Captured once; lengths, offsets, table and values change between replays."""
    kw = paged_inputs([500, 40, 7], [1, 1, 1], 8, 2, 128, 16, torch.bfloat16, 18, extra_pages=40)
    d = dev(kw)
    d["block_table"] = torch.nn.functional.pad(d["block_table"], (0, 20), value=-1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = flash_bias_paged_func(**d)
    other = paged_inputs([3, 600, 300], [1, 2, 0], 8, 2, 128, 16, torch.bfloat16, 19)
    pages = other["key_cache"].shape[0]
    d["q"].copy_(other["q"])
    for c in ("key_cache", "value_cache"):
        d[c][:pages] = other[c].cuda()[:d[c].shape[0]]
    d["block_table"].fill_(-1)
    d["block_table"][:, :other["block_table"].shape[1]] = other["block_table"].cuda()
    d["lens"].copy_(other["lens"])
    d["cu_tokens"].copy_(other["cu_tokens"])
    graph.replay()
    torch.cuda.synchronize()
    check_device_status()
    want, _, weight, size = orc.paged_attention(other["q"], other["key_cache"], other["value_cache"], other["block_table"], other["lens"], other["cu_tokens"])
    assert_within("o", o, want, bounds(want, weight, size, 128, torch.bfloat16)[0])


def test_cache_offsets_beyond_32_bits():
    """A pool whose last pages lie more than 2^31 elements from its start."""
    pages, page, Hk, D = 2100, 256, 32, 128  # 2.2e9 elements each
    kc, vc = (torch.empty(pages, page, Hk, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kw = paged_inputs([300], [2], Hk, Hk, D, page, torch.bfloat16, 20, extra_pages=0)
    table = kw["block_table"].clone()
    used = (table >= 0).sum()
    for c, src in ((kc, kw["key_cache"]), (vc, kw["value_cache"])):
        for i in range(used):
            c[pages - 1 - i] = src[table[0, i]].cuda()
    far = torch.full_like(table, -1)
    far[0, :used] = torch.tensor([pages - 1 - i for i in range(used)], dtype=torch.int32)
    want = check(kw)
    got = flash_bias_paged_func(kw["q"].cuda(), kc, vc, far.cuda(), kw["lens"].cuda(), kw["cu_tokens"].cuda())
    assert torch.equal(got, want)


@pytest.mark.parametrize("bad", [dict(q=torch.zeros(2, 4, 64)), dict(q=torch.zeros(2, 3, 64).half()), dict(q=torch.zeros(2, 4, 32).half()),
                                 dict(key_cache=torch.zeros(3, 8, 2, 64)), dict(value_cache=torch.zeros(3, 8, 1, 64).half()),
                                 dict(block_table=torch.zeros(1, 3).long()), dict(block_table=torch.zeros(3).int()), dict(lens=torch.zeros(2).int()),
                                 dict(lens=torch.zeros(1).long()), dict(cu_tokens=torch.zeros(1).int()), dict(tree_mask=torch.zeros(2, 1).int()),
                                 dict(tree_mask=torch.zeros(3, 1).long()), dict(positions=torch.zeros(3).int()), dict(slopes=torch.zeros(3)),
                                 dict(q_bias=torch.zeros(2, 4, 2).half(), bias_cache=torch.zeros(3, 8, 3, 2).half()),
                                 dict(q_bias=torch.zeros(2, 4, 2).half(), bias_cache=torch.zeros(3, 8, 2, 3).half()),
                                 dict(q_bias=torch.zeros(2, 3, 2).half(), bias_cache=torch.zeros(3, 8, 2, 2).half()),
                                 dict(q_bias=torch.zeros(2, 4, 2).half(), bias_cache=torch.zeros(3, 8, 2, 2).half(), slopes=torch.zeros(4))],
                         ids=lambda b: "-".join(b))
def test_refusals(bad):
    args = dict(q=torch.zeros(2, 4, 64).half(), key_cache=torch.zeros(3, 8, 2, 64).half(), value_cache=torch.zeros(3, 8, 2, 64).half(),
                block_table=torch.zeros(1, 3).int(), lens=torch.zeros(1).int(), cu_tokens=torch.tensor([0, 2]).int())
    flash_bias_paged_func(**dev(args))
    with pytest.raises(AssertionError):
        flash_bias_paged_func(**dev({**args, **bad}))
    with pytest.raises(RuntimeError, match="together"):
        flash_bias_paged_func(**dev(args), q_bias=torch.zeros(2, 4, 2).half().cuda())


def kernel_of(kw, flags=0):
    """The kernel (flashbias_b200._lib.PAGED_KERNELS) of a call with contiguous tensors like these."""
    import ctypes as C

    from flashbias_b200 import _lib
    p = _lib.FbPagedParams()
    q, kc, bc = kw["q"], kw["key_cache"], kw.get("bias_cache")
    p.N, p.Hq, p.D, p.B, p.Hk, p.page_size, p.num_pages = *q.shape, kw["lens"].numel(), kc.shape[2], kc.shape[1], kc.shape[0]
    p.dtype, p.table_width, p.softmax_scale, p.flags = _lib.FB_DTYPE_BF16, kw["block_table"].shape[1], kw.get("softmax_scale", 1.0), flags
    for n in ("q", "key_cache", "value_cache", "block_table", "lens", "cu_tokens", "o"):
        setattr(p, n, 0x1000)
    p.q_stride = p.o_stride = _lib.I64x2(q.shape[1] * q.shape[2], q.shape[2])
    p.key_cache_stride = p.value_cache_stride = _lib.I64x3(kc.stride(0), kc.stride(1), kc.stride(2))
    if bc is not None:
        p.R, p.bias_heads, p.q_bias, p.bias_cache = bc.shape[3], bc.shape[2], 0x1000, 0x1000
    return _lib.PAGED_KERNELS[_lib.load().fb_paged_kernel(C.byref(p))]


@pytest.mark.parametrize("R,heads", [(1, 2), (2, 2), (4, 1), (5, 2), (6, 2), (7, 1), (10, 2), (12, 2), (16, 1), (17, 2), (20, 2), (40, 1)])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (32, 8), (96, 7)])
def test_ranks(R, heads, D, page):
    """Every way of reading factors: copied in pieces of 4, 8 or 16 bytes, odd ranks, and ranks beyond one product."""
    kw = paged_inputs([75, 0, 33], [1, 5, 3], 4, 2, D, page, torch.float16, R, R, heads)
    assert kernel_of(kw) == "split"
    check(kw)


def test_factors_at_an_odd_offset():
    kw = paged_inputs([75, 3], [1, 5], 4, 2, 64, 16, torch.float16, 1, 4)
    want = check(kw)
    d = dev(kw)
    d["bias_cache"] = torch.cat([d["bias_cache"][..., :1], d["bias_cache"]], -1)[..., 1:]
    assert torch.equal(flash_bias_paged_func(**d), want)


@pytest.mark.parametrize("Hq,D,page", [(4, 128, 32), (8, 64, 16), (3, 96, 128), (2, 40, 8), (6, 128, 256)])
@pytest.mark.parametrize("bias", ["none", "slopes"])
def test_tile_and_split_kernels_agree(Hq, D, page, bias):
    """The same call through both kernels: requests that end anywhere in a tile of 128 keys or rows, none cached, refused ones."""
    from flashbias_b200 import _lib
    from flashbias_b200.flash_bias import _op
    lens, new = [127, 128, 129, 0, -1, 513, 1000], [60, 1, 130, 97, 20, 33, 64]
    kw = paged_inputs(lens, new, Hq, 1 if Hq == 3 else 2, D, page, torch.bfloat16, D)
    _, mask, depth = tree(new, 23, 3)
    kw["tree_mask"] = mask
    if bias == "slopes":
        kw["slopes"] = torch.linspace(0.5, 0.02, Hq)
        kw["positions"] = (torch.repeat_interleave(kw["lens"], torch.tensor(new)) + depth).int()
    assert kernel_of(kw) == "tile" and kernel_of(kw, _lib.FB_FLAG_PAGED_SPLIT) == "split"
    check(kw)
    d = dev(kw)
    args = [d["q"], d["key_cache"], d["value_cache"], d["block_table"], d["lens"], d["cu_tokens"], d["tree_mask"], d.get("positions"), d.get("slopes")]
    got, lse = _op().paged_forward(*args, None, None, None, True, _lib.FB_FLAG_PAGED_SPLIT)
    gen, gl = _op().paged_forward(*args, None, None, None, True, _lib.FB_FLAG_FORCE_GENERAL)
    want, l64, weight, size = orc.paged_attention(kw["q"], kw["key_cache"], kw["value_cache"], kw["block_table"], kw["lens"], kw["cu_tokens"], mask,
                                                  kw.get("positions"), kw.get("slopes"))
    b = bounds(want, weight, size, D, torch.bfloat16)[0]
    assert_within("split", got, want, b)
    assert_within("general", gen, want, b)
    live = l64 > -math.inf
    assert (lse.cpu()[~live] == -math.inf).all() and (lse.cpu()[live] - l64[live]).abs().max() < 1e-3 and (gl.cpu()[live] - l64[live]).abs().max() < 1e-3


@pytest.mark.parametrize("T,Hq", [(1, 2), (40, 2), (20, 6)])
def test_many_requests(T, Hq):
    """More requests than a block of the schedule has threads, most of them short, some empty."""
    g = torch.Generator().manual_seed(T)
    B = 900 if T == 1 else 450
    lens, new = torch.randint(0, 40, (B,), generator=g).tolist(), torch.randint(0, T + 1, (B,), generator=g).tolist()
    new[0] = T
    kw = paged_inputs(lens, new, Hq, 2, 64, 16, torch.float16, 24)
    assert kernel_of(kw) == ("tile" if T * Hq / 4 > 32 else "split")
    check(kw)


def test_long_request_among_short_ones():
    """One request holds nearly all keys: its key tiles are spread over the GPU, and joined."""
    for T, Hq in ((1, 8), (2, 4), (24, 8)):
        kw = paged_inputs([20000, 1, 30, 0], [T, 1, T, T], Hq, 4, 64, 64, torch.bfloat16, 25)
        check(kw, slopes=torch.full((Hq,), 0.003))


def test_non_finite_values_in_a_tile_of_many_rows():
    """As test_values_of_unseen_keys_do_not_count, at every kernel, with values in the cached part as well."""
    from flashbias_b200 import _lib
    from flashbias_b200.flash_bias import _op
    new = [50, 40]
    kw = paged_inputs([200, 3], new, 4, 2, 128, 16, torch.bfloat16, 26)
    _, mask, _ = tree(new, 27)
    d = dev(kw)
    args = lambda d: [d["q"], d["key_cache"], d["value_cache"], d["block_table"], d["lens"], d["cu_tokens"], mask.cuda(), None, None, None, None, None, False]  # noqa: E731
    flags = (0, _lib.FB_FLAG_PAGED_SPLIT, _lib.FB_FLAG_FORCE_GENERAL)
    assert kernel_of(kw) == "tile"
    clean = [_op().paged_forward(*args(d), f)[0].cpu() for f in flags]
    for b, t, what in ((0, 4, float("nan")), (1, 20, -float("inf"))):
        place = int(kw["lens"][b]) + t
        kw["value_cache"][int(kw["block_table"][b, place // 16]), place % 16, :, 3:70] = what
    d = dev(kw)
    seen = torch.tensor([bool(mask[n, 0] >> (4 if n < 50 else 20) & 1) for n in range(90)])
    for f, c in zip(flags, clean):
        o = _op().paged_forward(*args(d), f)[0].cpu()
        assert torch.equal(o[~seen], c[~seen])
        assert not o[seen][:, :, 3:70].isfinite().any() and torch.equal(o[seen][:, :, :3], c[seen][:, :, :3])
    d["value_cache"][int(kw["block_table"][1, 0]), 1, 0, 5] = float("inf")  # a cached key that all of request 1 see
    for f in flags:
        o = _op().paged_forward(*args(d), f)[0].cpu()
        assert not o[50:, :2, 5].isfinite().any()


def test_two_graphs_and_an_eager_call_do_not_share_their_scratch():
    kw = [paged_inputs([3000, 70], [T, 1], 8, 2, 128, 16, torch.bfloat16, 28 + T) for T in (1, 30)]
    ds = [dev(k) for k in kw]
    want = [flash_bias_paged_func(**d) for d in ds]
    graphs, outs = [], []
    for d in ds:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(flash_bias_paged_func(**d))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in ds]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        eager = flash_bias_paged_func(**ds[0])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)) and torch.equal(eager, want[0])


@pytest.mark.parametrize("lens,new,Hq,Hk,D", [([1000], [1], 8, 4, 128), ([5], [1], 8, 4, 64), ([40, 700], [1, 1], 4, 1, 64), ([300, 0, -1, 90], [1, 2, 1, 0], 4, 2, 128),
                                              ([129], [1], 16, 2, 96), ([2100, 17], [2, 1], 16, 2, 32), ([33, 64, 0], [1, 5, 9], 4, 1, 128)])
@pytest.mark.parametrize("bias", ["none", "slopes", "factors", "tree"])
def test_few_requests_with_narrow_and_wide_tables(lens, new, Hq, Hk, D, bias):
    """Short tables: each item is a cluster's, and the parts meet in shared memory; long ones: the schedule over the whole GPU."""
    kw = paged_inputs(lens, new, Hq, Hk, D, 16, torch.bfloat16, 26, 4 if bias == "factors" else 0)
    if bias == "slopes":
        kw["slopes"] = torch.linspace(0.3, 0.01, Hq)
    if bias == "tree":
        kw["tree_mask"] = tree(new, 27, 1)[1]
    # two tokens behind the last request stay unowned
    kw["q"] = torch.cat([kw["q"], kw["q"][-1:].expand(2, -1, -1)])
    for n in ("q_bias", "tree_mask"):
        if kw.get(n) is not None:
            kw[n] = torch.cat([kw[n], kw[n][-1:].expand(2, *kw[n].shape[1:])])
    wide = torch.nn.functional.pad(kw["block_table"], (0, 600), value=-1)
    assert kernel_of(kw) == kernel_of({**kw, "block_table": wide}) == "split"
    a = check(kw)
    b = check(kw, block_table=wide)
    assert (a[-2:] == 0).all() and (b[-2:] == 0).all()
