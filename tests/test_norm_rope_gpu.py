"""Norm with rotation against the formulas in 64 bits: layouts, head sizes, kinds of pairs, axes, types, and gradients."""
import pytest
import torch

from flashbias_b200 import check_device_status, flash_bias_func, norm_rope_func
from oracle import serving_oracle as orc
from tests.serving_helpers import FP32, assert_within, half_step, rounded

pytestmark = pytest.mark.gpu


def inputs(B, S, Hq, Hk, D, rot, naxes, dtype, wtype, seed, far=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, S, (Hq + 2 * Hk) * D, generator=g).to(dtype)
    q, k = qkv[..., :Hq * D].unflatten(-1, (Hq, D)), qkv[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D))
    w = [1.0 + 0.2 * torch.randn(D, generator=g) for _ in range(2)]
    w = [x.to(wtype) for x in w] if wtype else [None, None]
    inv_freq = (10000.0 ** (-torch.arange(0, rot, 2).double() / max(rot, 1))).float() if rot else None
    pos = axes = None
    if rot:
        pos = torch.randint(-5, 200, (naxes, B, S), generator=g) + far
        if naxes == 1:
            pos = pos[0]
        else:
            axes = [i * naxes // (rot // 2) for i in range(rot // 2)]
    return q, k, w, pos, inv_freq, axes


CASES = [
    # B, S, Hq, Hk, D, rot, axes, interleaved, dtype, weights
    (2, 33, 4, 2, 128, 128, 1, False, torch.bfloat16, torch.bfloat16),
    (1, 1, 1, 1, 64, 64, 1, True, torch.float16, torch.float32),       # one token, one head
    (1, 70, 8, 1, 64, 32, 1, False, torch.bfloat16, torch.float32),    # half the head rotated
    (2, 19, 3, 3, 80, 20, 1, False, torch.float16, None),              # pairs that are no whole vectors apart, no norm
    (1, 41, 5, 5, 96, 96, 3, False, torch.bfloat16, torch.bfloat16),   # three axes, twelve lanes a row
    (2, 17, 2, 1, 32, 32, 2, True, torch.float16, torch.float16),
    (1, 9, 2, 2, 20, 20, 1, True, torch.bfloat16, torch.float32),      # rows that are no whole vectors
    (1, 9, 2, 2, 7, 6, 1, False, torch.float16, torch.float32),        # odd head
    (1, 12, 3, 2, 8, 8, 1, True, torch.bfloat16, torch.bfloat16),      # one vector a row
    (3, 50, 16, 4, 128, 0, 1, False, torch.float16, torch.float16),    # norm alone
    (1, 23, 2, 2, 72, 48, 4, False, torch.bfloat16, torch.float16),
    (1, 15, 2, 1, 128, 64, 1, True, torch.bfloat16, None),
    (1, 300, 40, 8, 128, 128, 1, False, torch.bfloat16, torch.float32),
    (1, 31, 7, 4, 40, 40, 1, False, torch.float16, torch.float32),     # 5, 6, 9, 10 lanes a row: lanes of the warp that have none
    (1, 31, 16, 5, 48, 24, 1, False, torch.bfloat16, torch.float32),
    (2, 11, 25, 8, 72, 36, 2, False, torch.float16, torch.float16),    # runs of two columns
    (1, 21, 10, 10, 80, 80, 1, True, torch.bfloat16, torch.float32),
    (1, 90, 13, 2, 80, 20, 1, False, torch.bfloat16, torch.bfloat16),
    (1, 13, 4, 3, 88, 22, 1, False, torch.float16, torch.float32),     # of one
    (1, 13, 9, 1, 40, 10, 1, False, torch.bfloat16, None),
    (1, 13, 5, 5, 24, 18, 1, True, torch.float16, torch.float16),      # the rotated columns end inside a lane's
    (1, 37, 7, 3, 36, 36, 1, False, torch.bfloat16, torch.float32),    # rows end inside a lane's columns
    (2, 9, 12, 4, 44, 20, 2, True, torch.float16, torch.float16),
    (1, 9, 5, 2, 100, 100, 1, False, torch.float16, torch.float32),
    (1, 9, 5, 2, 126, 126, 1, True, torch.bfloat16, torch.float32),
    (2, 33, 7, 3, 20, 10, 1, False, torch.bfloat16, torch.bfloat16),
    (1, 9, 33, 3, 6, 6, 1, False, torch.float16, torch.float16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "B%dS%dH%d-%dD%dr%da%d%s" % (*c[:7], "i" if c[7] else ""))
@pytest.mark.parametrize("layout", ["fused", "contiguous", "odd"])
def test_forward_and_gradients(case, layout):
    B, S, Hq, Hk, D, rot, naxes, il, dtype, wtype = case
    q, k, w, pos, f, axes = inputs(B, S, Hq, Hk, D, rot, naxes, dtype, wtype, S + D)
    to = (lambda t: None if t is None else t.cuda())
    if layout == "fused":  # slices of one projection
        qkv = torch.cat([q.flatten(2), k.flatten(2)], -1).cuda()
        qd, kd = qkv[..., :Hq * D].unflatten(-1, (Hq, D)), qkv[..., Hq * D:].unflatten(-1, (Hk, D))
    elif layout == "contiguous":  # heads outside the rows
        qd, kd = (t.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3) for t in (q, k))
    else:  # rows that start anywhere
        qd, kd = (torch.cat([t, t[..., :3]], -1).cuda()[..., 1:D + 1] for t in (q, k))
        q, k = qd.cpu(), kd.cpu()
    qd, kd = qd.detach().requires_grad_(True), kd.detach().requires_grad_(True)
    wd = [None if x is None else x.cuda().requires_grad_(True) for x in w]
    qo, ko = norm_rope_func(qd, kd, to(pos), to(f), wd[0], wd[1], axes, il)
    g = torch.Generator().manual_seed(1)
    gq, gk = torch.randn(q.shape, generator=g).to(dtype), torch.randn(k.shape, generator=g).to(dtype)
    leaves = [qd, kd] + [x for x in wd if x is not None]
    grads = torch.autograd.grad((qo, ko), leaves, (gq.cuda(), gk.cuda()))
    torch.cuda.synchronize()
    check_device_status()
    ang = None if f is None else orc.rope_angles(pos, f, axes)
    for name, x, wt, out, go, dx, dw in (("q", q, w[0], qo, gq, grads[0], grads[2] if wtype else None),
                                         ("k", k, w[1], ko, gk, grads[1], grads[3] if wtype else None)):
        want = orc.norm_rope(x, wt, ang, il)
        size = orc.norm_rope(x, wt).abs().amax(-1, keepdim=True)
        assert_within(name, out, want, rounded(want, dtype, size))
        wdx, wdw, size, total = orc.norm_rope_grads(x, go, wt, ang, il)
        assert_within("d" + name, dx, wdx, rounded(wdx, dtype, size.amax(-1, keepdim=True)))
        if wt is not None:
            # a sum of B S H terms in fp32 and one rounding
            assert_within("dw" + name, dw, wdw, half_step(wtype) * wdw.abs() * 1.001 + (B * S * x.shape[2] + 64) * FP32 * total)


def test_far_positions_keep_their_angle():
    """A 32-bit product position * frequency would be off by 2^-24 * 2e6 = 0.1 rad here."""
    q, k, w, pos, f, axes = inputs(1, 64, 2, 2, 64, 64, 1, torch.float16, None, 3, far=2_000_000)
    for p in (pos, -pos, pos.int()):
        qo, _ = norm_rope_func(q.cuda(), None, p.cuda(), f.double().cuda())
        want = orc.norm_rope(q, None, orc.rope_angles(p, f))
        assert_within("q", qo, want, rounded(want, torch.float16, q.double().abs().amax(-1, keepdim=True)))


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("axes", [None, [0, 2, 1, 1]])
def test_shapes_of_positions(axes, shared):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, 5, 2, 8, generator=g).half()
    f = torch.tensor([1.0, 0.5, 0.1, 0.01])
    pos = torch.randint(0, 50, (3, 1 if shared else 3, 5), generator=g)
    if axes is None:
        pos = pos[0]
    ang = orc.rope_angles(pos, f, axes)
    want = orc.norm_rope(x, None, ang)
    forms = [pos, pos.squeeze(-2)] if shared else [pos, pos.transpose(-1, -2).contiguous().transpose(-1, -2)]
    for p in forms:
        out, none = norm_rope_func(x.cuda(), None, p.cuda(), f.cuda(), axes=axes)
        assert none is None
        assert_within("x", out, want, rounded(want, torch.float16, x.double().abs().amax(-1, keepdim=True)))


def test_zero_rows_and_non_finite_values():
    x = torch.randn(1, 4, 1, 16).bfloat16()
    x[0, 0] = 0
    x[0, 1, 0, 3] = float("inf")
    x[0, 2, 0, 5] = float("nan")
    w = torch.ones(16)
    out, _ = norm_rope_func(x.cuda(), None, None, None, w.cuda())
    out = out.cpu()
    assert (out[0, 0] == 0).all()
    assert out[0, 1, 0, 3].isnan() and (out[0, 1, 0, :3] == 0).all()  # inf * (1 / inf), and finite values times 0
    assert out[0, 2].isnan().all()
    want = orc.norm_rope(x[:, 3:], w)
    assert_within("x", out[:, 3:], want, rounded(want, torch.bfloat16, want.abs().amax()))


@pytest.mark.parametrize("D", [40, 64, 72, 80, 128, 20, 44, 102, 27])
@pytest.mark.parametrize("rot", [2, 4, 10, 12, 16, 20])
@pytest.mark.parametrize("interleaved", [False, True])
def test_columns_behind_the_rotated_ones_keep_their_bits_and_touch_nothing(D, rot, interleaved):
    g = torch.Generator().manual_seed(D + rot)
    x = torch.randn(1, 6, 11, D, generator=g).half()
    x.view(torch.int16)[..., rot:] = torch.randint(-2 ** 15, 2 ** 15, x[..., rot:].shape, generator=g).short()  # any bits, NaN and inf too
    pos, f = torch.arange(6).cuda(), torch.rand(rot // 2, generator=g).cuda()
    xd = x.cuda().requires_grad_(True)
    out, _ = norm_rope_func(xd, None, pos, f, interleaved=interleaved)
    dx, = torch.autograd.grad(out, xd, x.cuda())
    for y in (out, dx):
        assert torch.equal(y.cpu()[..., rot:].view(torch.int16), x[..., rot:].view(torch.int16))
        assert y[..., :rot].isfinite().all()
    assert (out[..., :rot].float().norm(dim=-1).cpu() - x[..., :rot].float().norm(dim=-1)).abs().max() < 1e-2  # (20 roundings of 4 at most)


def test_partial_gradients_and_expanded_ones():
    q, k, w, pos, f, _ = inputs(2, 9, 2, 1, 64, 64, 1, torch.bfloat16, torch.float32, 4)
    qd, kd, pos, f = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True), pos.cuda(), f.cuda()
    wd = [x.cuda().requires_grad_(True) for x in w]
    qo, ko = norm_rope_func(qd, kd, pos, f, *wd)
    ang = orc.rope_angles(pos, f)
    dq, dqw = torch.autograd.grad(qo.sum(), [qd, wd[0]], retain_graph=True)  # the gradient is an expanded scalar; k_out unused
    wdx, wdw, size, total = orc.norm_rope_grads(q, torch.ones_like(q), w[0], ang)
    assert_within("dq", dq, wdx, rounded(wdx, torch.bfloat16, size.amax(-1, keepdim=True)))
    assert_within("dqw", dqw, wdw, half_step(torch.float32) * wdw.abs() + 100 * FP32 * total)
    assert torch.autograd.grad(qo.sum(), [kd, wd[1]], retain_graph=True, allow_unused=True) == (None, None)
    dk, = torch.autograd.grad(ko.sum(), [kd])
    wdx, _, size, _ = orc.norm_rope_grads(k, torch.ones_like(k), w[1], ang)
    assert_within("dk", dk, wdx, rounded(wdx, torch.bfloat16, size.amax(-1, keepdim=True)))
    # weights alone, and a tensor without a weight beside one that has it
    qo, ko = norm_rope_func(q.cuda(), k.cuda(), pos, f, wd[0], None)
    dqw2, = torch.autograd.grad(qo, [wd[0]], torch.ones_like(qo))
    assert torch.equal(dqw2, dqw)


@pytest.mark.parametrize("normed", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("heads_first", [False, True])
def test_tensors_without_a_weight_may_change_before_the_backward(normed, heads_first):
    """Their gradient needs the upstream one alone; that of a tensor with a weight reads it again, and autograd finds the change."""
    q, k, w, pos, f, _ = inputs(2, 300, 8, 4, 64, 48, 1, torch.bfloat16, torch.float32, 7)
    if heads_first:
        q, k = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k))
    gq, gk = (torch.randn(t.shape, generator=torch.Generator().manual_seed(1)).to(t.dtype) for t in (q, k))
    leaves = [t.cuda().requires_grad_(True) for t in (q, k)]
    rows = [t * 1 for t in leaves]
    w = [x.cuda() if n else None for x, n in zip(w, normed)]
    out = norm_rope_func(*rows, pos.cuda(), f.cuda(), *w)
    with torch.no_grad():
        for t, n in zip(rows, normed):
            if not n:
                t.zero_()
    grads = torch.autograd.grad(out, leaves, (gq.cuda(), gk.cuda()), retain_graph=True)
    ang = orc.rope_angles(pos, f)
    for name, got, leaf, t, go, wt in (("dq", grads[0], leaves[0], q, gq, w[0]), ("dk", grads[1], leaves[1], k, gk, w[1])):
        want, _, size, _ = orc.norm_rope_grads(t, go, wt, ang)
        assert_within(name, got, want, rounded(want, torch.bfloat16, size.amax(-1, keepdim=True)))
        assert got.stride() == leaf.stride()
    for t, n in zip(rows, normed):
        if n:
            with torch.no_grad():
                t.zero_()
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                torch.autograd.grad(out, leaves, (gq.cuda(), gk.cuda()))


def test_gradients_of_expanded_tensors_without_a_weight():
    q, k, _, pos, f, _ = inputs(1, 50, 4, 2, 64, 64, 1, torch.float16, None, 8)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k)]
    out = norm_rope_func(*[t.expand(3, -1, -1, -1) for t in leaves], pos.cuda(), f.cuda())
    go = [torch.randn(t.shape, generator=torch.Generator().manual_seed(2)).half() for t in out]
    for x, g, got in zip((q, k), go, torch.autograd.grad(out, leaves, [g.cuda() for g in go])):
        want = orc.norm_rope_grads(x, g, None, orc.rope_angles(pos, f))[0]
        # each of three gradients is rounded, and so are their two sums
        assert_within("dx", got, want.sum(0, keepdim=True), 5 * rounded(want, torch.float16, g.double().abs().amax(-1, keepdim=True)).sum(0, keepdim=True))


def test_a_fused_projection_is_freed_between_the_passes():
    pos, f = torch.arange(4096).cuda(), torch.rand(32).cuda()
    leaf = torch.randn(1, 4096, 24 * 64, device="cuda").half().requires_grad_(True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    qkv = leaf * 1
    out = norm_rope_func(qkv[..., :512].unflatten(-1, (8, 64)), qkv[..., 512:1024].unflatten(-1, (8, 64)), pos, f)
    del qkv
    held = torch.cuda.memory_allocated() - before - sum(t.numel() * 2 for t in out)
    assert held < 2 ** 20  # (the projection is 12 MB)
    torch.autograd.grad(out, leaf, [torch.ones_like(t) for t in out])


def test_a_second_derivative_is_refused():
    q, k, w, pos, f, _ = inputs(1, 9, 2, 1, 64, 64, 1, torch.bfloat16, torch.float32, 4)
    qd, wd = q.cuda().requires_grad_(True), w[0].cuda().requires_grad_(True)
    out, _ = norm_rope_func(qd, None, pos.cuda(), f.cuda(), wd)
    dq, dw = torch.autograd.grad(out, [qd, wd], torch.ones_like(out), create_graph=True)
    for g in (dq, dw):
        with pytest.raises(RuntimeError, match="twice"):
            torch.autograd.grad(g.sum(), qd, retain_graph=True)
    plain = torch.autograd.grad(norm_rope_func(qd, None, pos.cuda(), f.cuda(), wd)[0], [qd, wd], torch.ones_like(out))
    assert torch.equal(dq, plain[0]) and torch.equal(dw, plain[1])


def test_weight_gradients_repeat_bit_for_bit():
    q, k, w, pos, f, _ = inputs(1, 700, 8, 2, 128, 128, 1, torch.bfloat16, torch.float32, 6)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, *w)]
    def grads():
        out = norm_rope_func(leaves[0], leaves[1], pos.cuda(), f.cuda(), leaves[2], leaves[3])
        return torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])
    first = grads()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, grads()))


def test_empty_tensors():
    x = torch.randn(0, 7, 2, 16, device="cuda", dtype=torch.float16, requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    out, _ = norm_rope_func(x, None, None, None, w)
    dx, dw = torch.autograd.grad(out.sum(), [x, w])
    assert out.shape == x.shape == dx.shape and (dw == 0).all()


def test_captured_step_replays_on_new_values():
    """Forward and backward in one graph, replayed on other inputs; an eager pass over the same leaves runs before and after."""
    q, k, w, pos, f, _ = inputs(1, 65, 4, 2, 64, 64, 1, torch.float16, torch.float32, 8)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, *w)]
    pos, f = pos.cuda(), f.cuda()
    def step():
        out = norm_rope_func(leaves[0], leaves[1], pos, f, leaves[2], leaves[3])
        return out + torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        for t in leaves:
            t.copy_(torch.randn_like(t))
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_on_a_side_stream():
    q, k, w, pos, f, _ = inputs(2, 129, 4, 2, 64, 64, 1, torch.float16, torch.float32, 9)
    a = [t.cuda() for t in (q, k, pos, f, *w)]
    want = norm_rope_func(*a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm_rope_func(*a)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("bad", [dict(k=torch.zeros(1, 4, 2, 8)), dict(k=torch.zeros(1, 5, 2, 16)), dict(positions=torch.zeros(4)),
                                 dict(positions=torch.arange(5)), dict(positions=torch.zeros(2, 4, dtype=torch.int64)),
                                 dict(inv_freq=None), dict(inv_freq=torch.ones(9)), dict(inv_freq=torch.ones(8).half()),
                                 dict(q_weight=torch.ones(15)), dict(q_weight=torch.ones(16).half()), dict(q_weight=torch.ones(16).double()),
                                 dict(eps=-1.0), dict(eps=float("inf")), dict(axes=[0] * 8), dict(axes=[0] * 7, positions=torch.zeros(1, 4).long()),
                                 dict(axes=[1] * 8, positions=torch.zeros(1, 4).long()), dict(axes=[0] * 8, positions=torch.zeros(5, 4).long()),
                                 dict(axes=[-1] * 8, positions=torch.zeros(1, 4).long()), dict(q=torch.zeros(1, 4, 2, 16)),
                                 dict(q=torch.zeros(4, 2, 16).half()), dict(q=torch.zeros(1, 4, 2, 130).half(), k=None, q_weight=None)],
                         ids=lambda b: "-".join(b))
def test_refusals(bad):
    args = dict(q=torch.zeros(1, 4, 2, 16).half(), k=torch.zeros(1, 4, 2, 16).half(), positions=torch.arange(4), inv_freq=torch.ones(8),
                q_weight=torch.ones(16), k_weight=torch.ones(16))
    put = (lambda v: v.cuda() if isinstance(v, torch.Tensor) else v)
    norm_rope_func(**{n: put(v) for n, v in args.items()})
    bad = {n: v.half() if n == "k" and v is not None else v for n, v in bad.items()}
    with pytest.raises(AssertionError):
        norm_rope_func(**{n: put(v) for n, v in {**args, **bad}.items()})


def test_beside_the_attention_operator():
    """Projection, norm and rotation, attention with a low-rank bias: the gradient of the whole chain."""
    import math

    from oracle import flashbias_oracle
    B, S, H, D, R = 1, 70, 2, 32, 2
    q, k, w, pos, f, _ = inputs(B, S, H, H, D, D, 1, torch.float16, torch.float32, 11)
    g = torch.Generator().manual_seed(12)
    v, do = (torch.randn(B, S, H, D, generator=g).half() for _ in range(2))
    qb, kb = (torch.randn(1, S, H, R, generator=g).half() for _ in range(2))
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, *w)]
    qr, kr = norm_rope_func(leaves[0], leaves[1], pos.cuda(), f.cuda(), leaves[2], leaves[3])
    o = flash_bias_func(qr, kr, v.cuda(), qb.cuda(), kb.cuda(), None, True)
    grads = torch.autograd.grad(o, leaves, do.cuda())
    # the same chain in 64 bits, from the rotated values as the operator rounded them
    ang = orc.rope_angles(pos, f)
    ref = [t.detach().double().cpu() for t in (qr, kr, v, qb, kb)]
    scale = 1.0 / math.sqrt(D)
    o_ref, lse = flashbias_oracle.attention_forward(*[t.float() for t in ref], None, True, scale)
    dqr, dkr = flashbias_oracle.attention_backward(do.float(), *[t.float() for t in ref[:3]], o_ref, lse, *[t.float() for t in ref[3:]],
                                                   None, True, scale)[:2]
    for name, got, x, dr, wt in (("dq", grads[0], q, dqr, w[0]), ("dk", grads[1], k, dkr, w[1])):
        want, _, size, _ = orc.norm_rope_grads(x, dr, wt, ang)
        # the gradient that the attention hands over has been rounded twice (P, dS and the result): 2e-3 of its size in fp16
        assert_within(name, got, want, rounded(want, torch.float16, size) + 4e-3 * size.amax())
