"""The kernels of attention over pages at work that fills the GPU several times: segments of many key tiles, many segments per
CTA, parts joined from dozens of CTAs, four key heads per CTA, prompts behind a cached prefix."""
import math

import pytest
import torch

from flashbias_b200 import _lib, check_device_status
from flashbias_b200.flash_bias import _op
from oracle import serving_oracle as orc
from tests.serving_helpers import FP32, assert_within, paged_inputs, tree
from tests.test_paged_attention_gpu import bounds, kernel_of

pytestmark = pytest.mark.gpu


def on_device(kw):
    return {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in kw.items()}


def forward(d, flags=0):
    o, lse = _op().paged_forward(*[d.get(n) for n in ("q", "key_cache", "value_cache", "block_table", "lens", "cu_tokens", "tree_mask", "positions",
                                                      "slopes", "q_bias", "bias_cache", "softmax_scale")], True, flags)
    torch.cuda.synchronize()
    check_device_status()
    return o, lse


def in_64_bits(d):
    """serving_oracle.paged_attention in products over a request's keys, on the device: (o, lse, weight, size)."""
    q = d["q"].double()
    N, Hq, D = q.shape
    page, Hk = d["key_cache"].shape[1:3]
    scale = d.get("softmax_scale") or 1.0 / math.sqrt(D)
    o, lse = torch.zeros_like(q), torch.full((N, Hq), -math.inf, dtype=torch.float64, device="cuda")
    weight, size = torch.zeros_like(o), torch.zeros_like(lse)
    lens, cu = d["lens"].tolist(), d["cu_tokens"].tolist()
    for b, ctx in enumerate(lens):
        first, T = cu[b], cu[b + 1] - cu[b]
        if ctx < 0 or T == 0:
            continue
        keys, rows = ctx + T, slice(first, first + T)
        pages = d["block_table"][b, :-(-keys // page)].long()
        new = torch.arange(T, device="cuda")
        if d.get("tree_mask") is None:
            seen = new[:, None] >= new
        else:
            words = d["tree_mask"][rows]
            words = torch.nn.functional.pad(words, (0, max(0, -(-T // 64) - words.shape[1])))
            seen = (words[:, new // 64] >> (new % 64) & 1).bool()
        seen = torch.cat([torch.ones(T, ctx, dtype=torch.bool, device="cuda"), seen], 1)
        at = torch.arange(keys, device="cuda")
        if d.get("positions") is not None:
            at = torch.cat([at[:ctx], d["positions"][rows].long()])
        for h in range(Hq):
            hk = h // (Hq // Hk)
            k, v = (d[c][pages].flatten(0, 1)[:keys, hk].double() for c in ("key_cache", "value_cache"))
            z, mag = q[rows, h] @ k.T * scale, q[rows, h].abs() @ k.abs().T * abs(scale)
            if d.get("slopes") is not None:
                bias = d["slopes"][h].double() * (at - at[ctx:, None]).double()
                z, mag = z + bias, mag + bias.abs()
            if d.get("q_bias") is not None:
                qb = d["q_bias"][rows].double().expand(-1, Hq, -1)[:, h]
                kb = d["bias_cache"][pages].flatten(0, 1)[:keys].double()
                kb = kb[:, hk if kb.shape[1] > 1 else 0]
                z, mag = z + qb @ kb.T, mag + qb.abs() @ kb.abs().T
            z = z.masked_fill(~seen, -math.inf)
            lse[rows, h] = torch.logsumexp(z, 1)
            p = torch.softmax(z, 1).nan_to_num_()
            o[rows, h], weight[rows, h] = p @ v, p @ v.abs()
            size[rows, h] = mag.masked_fill(~seen, 0.0).amax(1)
    return [t.cpu() for t in (o, lse, weight, size)]


def check(kw, kernel, flags=(0,), want=None):
    assert kernel_of(kw) == kernel
    d = on_device(kw)
    want = want or in_64_bits(d)
    o64, lse64, weight, size = want
    D = kw["q"].shape[2] + (kw["q_bias"].shape[2] if kw.get("q_bias") is not None else 0)
    bo, bl = bounds(o64, weight, size, D, kw["q"].dtype)
    empty = lse64 == -math.inf
    for f in flags:
        o, lse = forward(d, f)
        assert_within(f"o {f}", o, o64, bo)
        assert (o.cpu()[empty] == 0).all() and (lse.cpu()[empty] == -math.inf).all()
        assert_within(f"lse {f}", lse.cpu()[~empty], lse64[~empty], (bl + 8 * FP32 * lse64.abs() + 1e-6)[~empty])
    return d


BOTH = (0, _lib.FB_FLAG_PAGED_SPLIT)


@pytest.mark.parametrize("bias", ["none", "slopes", "factors"])
@pytest.mark.parametrize("masked", [False, True])
def test_the_restatement_on_the_device_is_the_oracle(bias, masked):
    kw = paged_inputs([70, 0, -1, 9], [5, 66, 3, 1], 4, 2, 16, 8, torch.float16, 50, 3 if bias == "factors" else 0, 1)
    if bias == "slopes":
        kw["slopes"], kw["positions"] = torch.tensor([0.5, 0.2, 0.1, 0.05]), torch.randint(0, 90, (75,)).int()
    if masked:
        kw["tree_mask"] = tree([5, 66, 3, 1], 51, 1)[1]
    want = orc.paged_attention(**{{"block_table": "table", "cu_tokens": "cu"}.get(n, n): v for n, v in kw.items()})
    for a, b in zip(in_64_bits(on_device(kw)), want):
        finite = b.isfinite()
        assert (a[finite] - b[finite]).abs().max() < 1e-9 and torch.equal(a[~finite], b[~finite])


# key tiles of 128 on the tile kernel: 640, 408, 1680 (segments of 4 to 11 per CTA), then short requests alone (11 segments of one)
LONG = [([20000], [60], 8, 4, 64, 64), ([9000, 3000, 1, 700], [40, 33, 64, 50], 8, 4, 128, 32), ([6000, 5000, 2000], [30, 33, 31], 32, 16, 64, 16),
        ([6100, 4900, 2100], [30, 33, 31], 32, 16, 128, 128)]


@pytest.mark.parametrize("lens,new,Hq,Hk,D,page", LONG, ids=lambda v: "_".join(map(str, v)) if isinstance(v, list) else str(v))
@pytest.mark.parametrize("bias", ["none", "slopes", "tree"])
def test_segments_of_many_key_tiles(lens, new, Hq, Hk, D, page, bias):
    kw = paged_inputs(lens, new, Hq, Hk, D, page, torch.bfloat16 if D == 64 else torch.float16, 52)
    units = sum(-(-(a + t) // 128) * -(-t * (Hq // Hk) // 128) for a, t in zip(lens, new)) * Hk
    assert units > 2 * 148
    if bias != "none":
        kw["slopes"] = torch.logspace(-1, -4, Hq)
    if bias == "tree":
        _, kw["tree_mask"], depth = tree(new, 53)
        kw["positions"] = (torch.repeat_interleave(kw["lens"], torch.tensor(new)) + depth).int()
    check(kw, "tile", BOTH)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("order", ["rising", "falling", "zigzag"])
def test_a_maximum_that_moves_from_tile_to_tile(D, order):
    """Logits change by 8 (a factor of 2^11) from each tile of 128 keys to the next: the reference moves at every tile, at none, or at
    every other one."""
    lens, new = [3000, 2500, 2000], [30, 33, 31]
    kw = paged_inputs(lens, new, 32, 16, D, 16, torch.bfloat16, 54)
    kw["q"] = (1.0 + 0.03 * torch.randn(kw["q"].shape, generator=torch.Generator().manual_seed(55))).bfloat16()
    for b, (ctx, T) in enumerate(zip(lens, new)):
        for j in range(ctx + T):
            tile = j // 128
            level = {"rising": -8.0 * tile, "falling": 8.0 * tile, "zigzag": 8.0 * (tile // 2 - 3 * (tile % 2))}[order]
            kw["key_cache"][kw["block_table"][b, j // 16], j % 16] += level / math.sqrt(D)
    check(kw, "tile", BOTH)


@pytest.mark.parametrize("D,Hq", [(64, 32), (128, 16)])
def test_many_segments_per_cta(D, Hq):
    g = torch.Generator().manual_seed(56)
    lens, new = torch.randint(0, 300, (110,), generator=g).tolist(), torch.randint(25, 60, (110,), generator=g).tolist()
    lens[7], new[9] = -1, 0
    kw = paged_inputs(lens, new, Hq, 16, D, 32, torch.float16, 57)
    _, kw["tree_mask"], depth = tree(new, 58)
    kw["slopes"] = torch.linspace(0.4, 0.01, Hq)
    kw["positions"] = (torch.repeat_interleave(kw["lens"], torch.tensor(new)) + depth).int()
    d = check(kw, "tile")
    first = forward(d)
    for _ in range(5):  # the order of all sums is fixed
        assert all(torch.equal(a, b) for a, b in zip(first, forward(d)))


@pytest.mark.parametrize("D,Hq,Hk,T,kernel", [(64, 8, 2, 60, "tile"), (128, 4, 2, 60, "tile"), (64, 4, 2, 40, "split")])
def test_more_requests_than_the_schedule_has_threads(D, Hq, Hk, T, kernel):
    """A thread of the schedule adds up several requests' tiles."""
    g = torch.Generator().manual_seed(59)
    B = 850
    lens, new = torch.randint(0, 40, (B,), generator=g).tolist(), torch.randint(0, T + 1, (B,), generator=g).tolist()
    lens[400] = 2000
    kw = paged_inputs(lens, new, Hq, Hk, D, 16, torch.bfloat16, 60)
    check(kw, kernel)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,kernel", [(64, "tile"), (6, "split")])
def test_few_items_joined_from_dozens_of_parts(D, T, kernel):
    kw = paged_inputs([11772], [T], 4, 2, D, 32, torch.bfloat16, 61)
    check(kw, kernel, BOTH)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T,Hq,Hk,B,bias,R", [(1, 8, 4, 460, "none", 0), (1, 8, 4, 460, "slopes", 0), (1, 8, 4, 460, "factors", 8), (1, 8, 4, 460, "factors", 3),
                                              (1, 8, 4, 460, "factors", 20), (3, 16, 8, 300, "slopes", 0), (3, 16, 8, 300, "factors", 8),
                                              (14, 8, 4, 460, "none", 0), (14, 8, 4, 460, "factors", 3)])
def test_four_key_heads_per_cta(D, T, Hq, Hk, B, bias, R):
    """The split kernel's form for many requests (four key heads of a CTA, a warp each), with one long request whose parts are joined."""
    assert B * Hk >= 4 * 3 * torch.cuda.get_device_properties(0).multi_processor_count
    g = torch.Generator().manual_seed(62)
    lens, new = torch.randint(0, 150, (B,), generator=g).tolist(), torch.randint(T // 2 + 1, T + 1, (B,), generator=g).tolist()
    lens[B // 3], lens[5], lens[-1] = 9000, -1, 0
    kw = paged_inputs(lens, new, Hq, Hk, D, 16, torch.float16 if T == 1 else torch.bfloat16, 63, R)
    if bias == "slopes":
        kw["slopes"] = torch.logspace(-0.5, -4, Hq)
    check(kw, "split")


@pytest.mark.parametrize("ctx,T", [(0, 2500), (1700, 700), (129, 1024)])
@pytest.mark.parametrize("D,Hq,Hk", [(64, 8, 2), (128, 4, 4)])
@pytest.mark.parametrize("bias", ["none", "slopes", "factors"])
def test_prompts_and_chunks_of_them(ctx, T, D, Hq, Hk, bias):
    """Dozens of row tiles over dozens of key tiles, a second request of one token beside them."""
    kw = paged_inputs([ctx, 40], [T, 1], Hq, Hk, D, 64, torch.bfloat16, 64, 4 if bias == "factors" else 0)
    if bias == "slopes":
        kw["slopes"] = torch.logspace(-0.5, -3, Hq)
    check(kw, "split" if bias == "factors" else "tile")
