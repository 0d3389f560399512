"""Attention over pages at the ends of the number range, against 64 bits."""
import math

import pytest
import torch

from flashbias_b200 import _lib, check_device_status
from flashbias_b200.flash_bias import _op
from oracle import serving_oracle as orc
from tests.serving_helpers import FP32, assert_within, half_step, paged_inputs, tree
from tests.test_paged_attention_gpu import bounds, kernel_of

pytestmark = pytest.mark.gpu

FLAGS = {"own": 0, "split": _lib.FB_FLAG_PAGED_SPLIT, "general": _lib.FB_FLAG_FORCE_GENERAL}


def forward(kw, kernel):
    d = {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    o, lse = _op().paged_forward(*[d.get(n) for n in ("q", "key_cache", "value_cache", "block_table", "lens", "cu_tokens", "tree_mask", "positions",
                                                      "slopes", "q_bias", "bias_cache", "softmax_scale")], True, FLAGS[kernel])
    torch.cuda.synchronize()
    check_device_status()
    return o.cpu(), lse.cpu()


def oracle(kw):
    return orc.paged_attention(**{{"block_table": "table", "cu_tokens": "cu", "softmax_scale": "scale"}.get(n, n): v for n, v in kw.items()})


def weights_alone(want, weight, dtype):
    """bounds() of rows whose logits are equal or so far apart that the lower ones weigh nothing: no error of a logit counts."""
    u = half_step(dtype)
    return u * want.abs() + (1.01 * u + 2.0 ** -19) * weight + torch.finfo(dtype).smallest_normal * u


def used_places(kw, b=0):
    page = kw["key_cache"].shape[1]
    n = int(kw["lens"][b]) + int(kw["cu_tokens"][b + 1] - kw["cu_tokens"][b])
    return [(int(kw["block_table"][b, j // page]), j % page) for j in range(n)]


@pytest.mark.parametrize("kernel", ["own", "general"])
@pytest.mark.parametrize("lens,T,width", [(200, 3, 0), (900, 1, 0), (900, 2, 600), (4000, 12, 600)])
@pytest.mark.parametrize("value", [torch.finfo(torch.bfloat16).min, -3.0e38, -2.4e38, 3.0e38])
def test_a_bias_of_any_finite_size_in_all_keys(kernel, lens, T, width, value):
    """A padding mask of the type's lowest value as a factor: beside it the rest of a logit vanishes, so a row whose keys all carry
    it is the mean of its values (a step of 2.4e38 is 2e31 in 32 bits and 2.7e22 in 64; q.k is below 1e3)."""
    kw = paged_inputs([lens], [T], 2, 2, 64, 16, torch.bfloat16, 31, R=2)
    kw["block_table"] = torch.nn.functional.pad(kw["block_table"], (0, width), value=-1)
    kw["bias_cache"][..., 0] = value
    kw["q_bias"][..., 0] = 1.0
    want, lse, weight, _ = oracle(kw)
    assert lse.isfinite().all() and want.abs().max() > 0.01
    o, got = forward(kw, kernel)
    assert_within("o", o, want, weights_alone(want, weight, torch.bfloat16))
    assert_within("lse", got, lse, 8 * FP32 * lse.abs())


@pytest.mark.parametrize("kernel", ["own", "general"])
def test_huge_biases_keep_their_order(kernel):
    """Every third key carries -2.5e38, the others -3.3e38: the first kind alone counts."""
    kw = paged_inputs([400], [3], 4, 2, 64, 16, torch.bfloat16, 32, R=1)
    kw["bias_cache"][:] = -3.3e38
    for j, at in enumerate(used_places(kw)):
        if j % 3 == 0:
            kw["bias_cache"][at] = -2.5e38
    kw["q_bias"][:] = 1.0
    want, lse, weight, _ = oracle(kw)
    o, got = forward(kw, kernel)
    assert_within("o", o, want, weights_alone(want, weight, torch.bfloat16))
    assert_within("lse", got, lse, 8 * FP32 * lse.abs())


@pytest.mark.parametrize("kernel", ["own", "split", "general"])
@pytest.mark.parametrize("exponent,scale", [(40, None), (70, 0.3), (123, 24.0)])
@pytest.mark.parametrize("dtype,T,lens", [(torch.bfloat16, 40, 500), (torch.bfloat16, 1, 300), (torch.bfloat16, 64, 0)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_equal_logits_of_any_finite_size(kernel, exponent, scale, dtype, T, lens, sign):
    """All keys alike: however large q.k is, the values' mean.  (Logits up to 2.5e38: 24 * 2^123.)"""
    kw = paged_inputs([lens], [T], 4, 2, 128, 16, dtype, 33)
    for at in used_places(kw):
        kw["key_cache"][at] = 0.0
        kw["key_cache"][at][..., 5] = 2.0 ** (exponent // 2)
    kw["q"] = torch.randn(kw["q"].shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    kw["q"][..., 5] = sign * 2.0 ** (exponent - exponent // 2)
    kw["q"][1:, 1:, 5] *= 0.7109375  # (exact in bf16) and logits that are no powers of two
    if scale:
        kw["softmax_scale"] = scale
    if kernel == "own":
        assert kernel_of(kw) == ("tile" if T > 12 else "split")
    want, lse, weight, _ = oracle(kw)
    o, got = forward(kw, kernel)
    assert_within("o", o, want, weights_alone(want, weight, dtype))
    assert_within("lse", got, lse, 8 * FP32 * lse.abs())


@pytest.mark.parametrize("kernel", ["own", "split", "general"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_huge_logits_beside_tiles_of_which_a_row_sees_nothing(kernel, sign):
    """400 new tokens whose rows see the keys of one stretch of 64 alone, with logits of 2.5e38; 512 key tiles, several in a row per CTA."""
    kw = paged_inputs([0], [400], 32, 32, 128, 16, torch.bfloat16, 42)
    for at in used_places(kw):
        kw["key_cache"][at] = 0.0
        kw["key_cache"][at][..., 5] = 2.0 ** 61
    kw["q"][..., 5] = sign * 2.0 ** 62
    kw["softmax_scale"] = 24.0
    kw["tree_mask"] = torch.zeros(400, 7, dtype=torch.int64)
    for n in range(400):
        kw["tree_mask"][n, n // 32 % 6] = -1
    want, lse, weight, _ = oracle(kw)
    o, got = forward(kw, kernel)
    assert_within("o", o, want, weights_alone(want, weight, torch.bfloat16))
    assert_within("lse", got, lse, 8 * FP32 * lse.abs())


@pytest.mark.parametrize("kernel", ["own", "split"])
@pytest.mark.parametrize("T", [30, 64])
def test_large_logits_of_two_kinds(kernel, T):
    """Logits near 2^50 with steps of their own between the keys: the largest of a row takes all, the earlier tiles' are forgotten."""
    kw = paged_inputs([700], [T], 4, 2, 128, 16, torch.bfloat16, 34)
    best = {}
    for j, at in enumerate(used_places(kw)):
        kw["key_cache"][at] = 0.0
        size = (j * 37 % 101) + 128  # 8 bits: exact in bf16
        kw["key_cache"][at][..., 3] = size * 2.0 ** 17
        best.setdefault(size, []).append(j)
    kw["q"][..., 3] = 2.0 ** 26
    want, lse, weight, _ = oracle(kw)
    o, got = forward(kw, kernel)
    assert_within("o", o, want, weights_alone(want, weight, torch.bfloat16))
    assert_within("lse", got, lse, 8 * FP32 * lse.abs())


@pytest.mark.parametrize("kernel", ["own", "split", "general"])
@pytest.mark.parametrize("T,lens,slope", [(60, 0, 0.7), (130, 70, 0.7), (7, 0, 0.7), (60, 0, 20.0)])
def test_positions_of_one_request_that_are_far_from_one_another(kernel, T, lens, slope):
    """Two groups of new tokens, each near itself, that do not see one another."""
    kw = paged_inputs([lens], [T], 4, 2, 64, 16, torch.float16, 43)
    t = torch.arange(T)
    far = t % 3 != 0
    kw["positions"] = (t // 5 + torch.where(far, 1_234_567, lens)).int()
    kw["slopes"] = slope * torch.tensor([1.0, 0.4, 0.2, 0.1])
    seen = (far[:, None] == far) & (t[:, None] >= t)
    kw["tree_mask"] = torch.zeros(T, -(-T // 64), dtype=torch.int64)
    for i in range(T):
        word = kw["tree_mask"][:, i // 64]
        word |= torch.where(seen[:, i], -2 ** 63 if i % 64 == 63 else 2 ** (i % 64), 0)
    want, lse, weight, size = oracle(kw)
    if lens:  # the far tokens' cached keys weigh nothing: a request without them has the size of what counts
        kw0 = dict(kw, lens=kw["lens"] * 0, block_table=torch.arange(T, dtype=torch.int32)[None])
        for c in ("key_cache", "value_cache"):
            kw0[c] = torch.stack([kw[c][p] for p in used_places(kw)[lens:]]).unsqueeze(1)
        w0, _, weight0, size0 = oracle(kw0)
        assert (w0 - want)[far].abs().max() < 1e-12
        weight[far], size[far] = weight0[far], size0[far]
    o, got = forward(kw, kernel)
    bo, bl = bounds(want, weight, size, 64, torch.float16)
    assert_within("o", o, want, bo)
    assert_within("lse", got, lse, bl + 8 * FP32 * lse.abs() + 1e-6)


@pytest.mark.parametrize("kernel", ["own", "split", "general"])
@pytest.mark.parametrize("T,D", [(5, 64), (9, 128), (64, 128), (5, 32)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("depth", [19.0, 150.0])
def test_a_value_that_is_not_finite_counts_however_small_its_weight(kernel, T, D, dtype, depth):
    """A drafted key with a logit of `depth` below the others (a weight that fp16, or 32 bits, cannot hold) and a value that is not
    finite: the rows that see it are not finite, the others as if it were not there (but for the order of their fp32 sums: the kernel
    for few rows adds such a tile key by key.  Two orders of a sum of n terms p v differ by 2 n 2^-24 of the sum of |p v|, which is
    |v|'s largest at most, and each result is rounded once)."""
    kw = paged_inputs([70], [T], 4, 2, D, 16, dtype, 39)
    g = torch.Generator().manual_seed(40)
    kw["q"] = (1.0 + 0.05 * torch.randn(kw["q"].shape, generator=g)).to(dtype)
    _, mask, _ = tree([T], 41)
    kw["tree_mask"] = mask
    at = used_places(kw)[70 + 1]
    kw["key_cache"][at] = -depth / math.sqrt(D)
    clean, _ = forward(kw, kernel)
    largest = max(float(kw["value_cache"][p].abs().max()) for p in used_places(kw))
    allowed = 2 * half_step(dtype) * clean.double().abs() + 2 * (70 + T) * FP32 * largest
    for what in (float("inf"), float("nan"), -float("inf")):
        kw["value_cache"][at] = what
        o, _ = forward(kw, kernel)
        seen = (mask[:, 0] >> 1 & 1).bool()
        assert seen.any() and not seen.all()
        assert ((o.double() - clean.double()).abs() <= allowed)[~seen].all() and not o[seen].isfinite().any()


@pytest.mark.parametrize("kernel", ["own", "split", "general"])
@pytest.mark.parametrize("lens,T,width", [(9000, 1, 0), (6000, 1, 600), (7000, 30, 0), (3000, 2, 600)])
def test_many_small_weights_beside_a_large_one(kernel, lens, T, width):
    """fp16: the first key takes nearly all of the softmax and holds zeros; the rest weighs e^-19 = 2^-27.4 each, less than the
    smallest 16-bit number (2^-24), and is all of the result."""
    kw = paged_inputs([lens], [T], 4, 2, 128, 16, torch.float16, 35)
    kw["block_table"] = torch.nn.functional.pad(kw["block_table"], (0, width), value=-1)
    g = torch.Generator().manual_seed(36)
    kw["q"] = (1.0 + 0.02 * torch.randn(kw["q"].shape, generator=g)).half()
    for at in used_places(kw):
        kw["key_cache"][at] = 0.02 * torch.randn(2, 128, generator=g).half()
        kw["value_cache"][at] = (400.0 + 20.0 * torch.randn(2, 128, generator=g)).half()
    kw["key_cache"][used_places(kw)[0]] = 19.0 / math.sqrt(128)
    kw["value_cache"][used_places(kw)[0]] = 0.0
    want, lse, weight, size = oracle(kw)
    assert (want.abs() > 2.0 ** -14).all()
    o, got = forward(kw, kernel)
    bo, bl = bounds(want, weight, size, 128, torch.float16)
    assert_within("o", o, want, bo)
    assert_within("lse", got, lse, bl + 8 * FP32 * lse.abs() + 1e-6)


@pytest.mark.parametrize("kernel", ["own", "split", "general"])
@pytest.mark.parametrize("T,lens", [(7, 0), (60, 0), (12, 100), (130, 300)])
@pytest.mark.parametrize("offset", [1_000_000, 12_345_678, -700_001])
def test_positions_far_from_the_places(kernel, T, lens, offset):
    """Positions count by their differences: a request whose tokens stand far from their places (or whose cached keys, at theirs,
    weigh nothing) sees small biases between its new tokens."""
    kw = paged_inputs([lens], [T], 4, 2, 64, 16, torch.bfloat16, 37)
    _, mask, depth = tree([T], 38, 3)
    kw["tree_mask"] = mask
    kw["positions"] = (depth + offset).int()
    kw["slopes"] = torch.tensor([0.7, 0.31, 0.11, 0.05]) * (1 if offset > 0 else -1)
    want, lse, weight, size = oracle(kw)
    if lens:  # the cached keys' logits are below -20000 and weigh nothing: what counts is the size of the others
        kw0 = dict(kw, lens=kw["lens"] * 0)
        at = used_places(kw)
        for c in ("key_cache", "value_cache"):
            kw0[c] = torch.stack([kw[c][p] for p in at[lens:]]).unsqueeze(1)
        kw0["block_table"] = torch.arange(T, dtype=torch.int32)[None]
        w0, l0, weight, size = oracle(kw0)
        assert (w0 - want).abs().max() < 1e-12
    o, got = forward(kw, kernel)
    bo, bl = bounds(want, weight, size, 64, torch.bfloat16)
    assert_within("o", o, want, bo)
    assert_within("lse", got, lse, bl + 8 * FP32 * lse.abs() + 1e-6)
