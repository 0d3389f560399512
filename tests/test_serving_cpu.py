"""The operators around a paged cache, as far as no device is needed: what the C ABI refuses on the host, and the oracle's
gradients against differences."""
import ctypes as C

import pytest
import torch

from flashbias_b200 import _lib, flash_bias_paged_func, norm_rope_func, paged_append, paged_plan
from oracle import serving_oracle as orc

OK_STRIDE = _lib.I64x3(4096, 64, 256)


def rope_params():
    p = _lib.FbRopeParams()
    p.B, p.S, p.Hq, p.Hk, p.D, p.dtype, p.weight_dtype = 1, 16, 4, 2, 64, _lib.FB_DTYPE_BF16, _lib.FB_DTYPE_F32
    p.rot, p.naxes, p.position_bits, p.freq_dtype, p.eps = 64, 1, 64, _lib.FB_DTYPE_F32, 1e-6
    for n in ("q", "k", "q_weight", "k_weight", "positions", "inv_freq", "q_out", "k_out", "dq_out", "dk_out", "dq", "dk", "dq_weight",
              "dk_weight", "v", "key_cache", "value_cache", "slots"):
        setattr(p, n, 0x1000)  # never dereferenced on the host
    for n, t in p._fields_:
        if t is _lib.I64x3:
            setattr(p, n, OK_STRIDE)
    p.slot_stride, p.slot_bits, p.page_size, p.num_pages = 1, 64, 16, 8
    return p


def plan_params():
    p = _lib.FbPlanParams()
    p.B, p.num_tokens, p.page_size, p.table_width, p.stack_size, p.mask_words, p.table_stride = 2, 8, 16, 4, 10, 1, 4
    for n, t in p._fields_:
        if t is C.c_void_p and n != "status":
            setattr(p, n, 0x1000)
    return p


def paged_params():
    p = _lib.FbPagedParams()
    p.N, p.B, p.Hq, p.Hk, p.D, p.dtype, p.page_size, p.table_width, p.num_pages = 4, 2, 4, 2, 64, _lib.FB_DTYPE_F16, 16, 4096, 8
    p.softmax_scale, p.table_stride = 0.125, 4096
    for n in ("q", "key_cache", "value_cache", "block_table", "lens", "cu_tokens", "o"):
        setattr(p, n, 0x1000)
    for n in ("key_cache_stride", "value_cache_stride"):
        setattr(p, n, OK_STRIDE)
    p.q_stride = p.o_stride = _lib.I64x2(256, 64)
    return p


def refused(call, make, change):
    p = make()
    for n, v in change.items():
        setattr(p, n, v)
    code = getattr(_lib.load(), call)(C.byref(p), None)
    assert code < 0 and "unknown" not in _lib.strerror(code)
    return code


BAD_STRIDE = _lib.I64x3(1, -1, 1)
ROPE = [(dict(q=None), -1), (dict(B=0), -2), (dict(S=-1), -2), (dict(D=129), -2), (dict(Hq=0, Hk=0), -2), (dict(Hq=-1), -2), (dict(dtype=2), -3),
        (dict(weight_dtype=3), -3), (dict(eps=-1.0), -2), (dict(eps=float("nan")), -2), (dict(rot=66), -12), (dict(rot=3), -12),
        (dict(positions=None), -12), (dict(inv_freq=None), -12), (dict(naxes=5), -12), (dict(naxes=0), -12), (dict(position_bits=16), -3),
        (dict(freq_dtype=1), -3), (dict(q_stride=BAD_STRIDE), -4), (dict(pair_axis=(C.c_uint8 * 64)(0, 1)), -12)]


@pytest.mark.parametrize("change,code", ROPE + [(dict(q_out=None), -1), (dict(k_out_stride=BAD_STRIDE), -4)], ids=str)
def test_norm_rope_refuses(change, code):
    assert refused("fb_norm_rope", rope_params, change) == code


@pytest.mark.parametrize("change,code", ROPE + [(dict(dq_out=None), -1), (dict(dk=None), -1), (dict(dk_stride=BAD_STRIDE), -4),
                                                (dict(q_weight=None), -1), (dict(workspace=None), -6),
                                                (dict(workspace=0x1000, workspace_bytes=16), -6),
                                                (dict(workspace=0x1010, workspace_bytes=1 << 30), -6)], ids=str)
def test_norm_rope_backward_refuses(change, code):
    assert refused("fb_norm_rope_bwd", rope_params, change) == code


@pytest.mark.parametrize("change,code", ROPE + [(dict(B=2), -2), (dict(Hk=0), -2), (dict(v=None), -1), (dict(key_cache=None), -1), (dict(slots=None), -1),
                                                (dict(slot_bits=8), -3), (dict(slot_stride=-1), -4), (dict(page_size=0), -13), (dict(num_pages=0), -13),
                                                (dict(value_cache_stride=BAD_STRIDE), -4), (dict(R=4), -7), (dict(R=-1), -2), (dict(R=257), -2),
                                                (dict(bias_cache=0x1000), -7),
                                                (dict(R=4, k_bias=0x1000, bias_cache=0x1000, bias_heads=3), -7)], ids=str)
def test_paged_append_refuses(change, code):
    assert refused("fb_paged_append", rope_params, change) == code


@pytest.mark.parametrize("change,code", [(dict(B=0), -2), (dict(num_tokens=-1), -2), (dict(stack_size=-1), -2), (dict(page_size=0), -13),
                                         (dict(table_width=0), -13), (dict(page_size=1 << 30), -13), (dict(table_stride=3), -4),
                                         (dict(block_table=None), -1), (dict(free_count=None), -1), (dict(lens_out=None), -1),
                                         (dict(free_pages=None), -1), (dict(slots=None), -1), (dict(tree_mask=None), -5),
                                         (dict(mask_words=0), -5), (dict(mask_words=65), -5)], ids=str)
def test_paged_plan_refuses(change, code):
    assert refused("fb_paged_plan", plan_params, change) == code


@pytest.mark.parametrize("change,code", [(dict(N=0), -2), (dict(B=0), -2), (dict(Hq=3), -2), (dict(Hk=0), -2), (dict(D=0), -2), (dict(D=129), -2),
                                         (dict(R=257), -2), (dict(dtype=2), -3), (dict(page_size=0), -13), (dict(num_pages=0), -13),
                                         (dict(table_width=1 << 30), -13), (dict(q=None), -1), (dict(cu_tokens=None), -1), (dict(o=None), -1),
                                         (dict(R=4), -7), (dict(q_bias=0x1000), -7), (dict(R=4, q_bias=0x1000, bias_cache=0x1000, bias_heads=3), -7),
                                         (dict(R=4, q_bias=0x1000, bias_cache=0x1000, bias_heads=2, slopes=0x1000), -7),
                                         (dict(tree_mask=0x1000), -5), (dict(key_cache_stride=BAD_STRIDE), -4), (dict(q_stride=_lib.I64x2(-1, 1)), -4),
                                         (dict(workspace=None), -6), (dict(workspace=0x1000, workspace_bytes=64), -6)],
                         ids=str)
def test_paged_attention_refuses(change, code):
    assert refused("fb_paged_fwd", paged_params, change) == code


@pytest.mark.parametrize("change,code", [(dict(page_size=65537, table_width=32767), -13), (dict(page_size=1, table_width=2 ** 31 - 1), -13),
                                         (dict(page_size=65536, table_width=32768 - 1), -6), (dict(N=2147450000 // 4), -2),
                                         (dict(N=2147410000 // 4), -6)], ids=str)
def test_paged_attention_refuses_what_its_tiles_would_count_beyond_31_bits(change, code):
    """The last tile of the keys or rows, and copies that run ahead of it, are counted in 32 bits."""
    assert refused("fb_paged_fwd", paged_params, change) == code


@pytest.mark.parametrize("change", [dict(num_tokens=2 ** 31 - 2), dict(num_tokens=2 ** 31 - 2 ** 16 + 1), dict(B=2 ** 31 - 2)], ids=str)
def test_paged_plan_refuses_what_its_counters_would_pass(change):
    """A thread's next token is as far on as a cluster has threads, counted in 32 bits."""
    assert refused("fb_paged_plan", plan_params, change) == -2
    if "B" in change:
        assert refused("fb_paged_fwd", paged_params, change) == -2


def test_null_parameter_blocks_are_refused():
    lib = _lib.load()
    for call in ("fb_norm_rope", "fb_norm_rope_bwd", "fb_paged_append", "fb_paged_plan", "fb_paged_fwd"):
        assert getattr(lib, call)(None, None) == -1
    assert lib.fb_norm_rope_bwd_workspace_bytes(None) == 0 and lib.fb_paged_workspace_bytes(None) == 0


def test_operators_refuse_host_tensors_and_gradients():
    x = torch.randn(1, 4, 2, 8).half()
    with pytest.raises(AssertionError, match="device memory"):
        norm_rope_func(x, x)
    cache = torch.zeros(2, 4, 2, 8).half()
    ints = [torch.zeros(n, dtype=torch.int32) for n in (1, 2)]
    table = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="device memory"):
        paged_append(x[0], x[0], x[0], cache, cache, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(AssertionError, match="device memory"):
        paged_plan(table, ints[0], ints[1], ints[0], ints[0], ints[0], 4, 4)
    with pytest.raises(AssertionError, match="device memory"):
        flash_bias_paged_func(x[0], cache, cache, table, ints[0], ints[1])
    grad = x[0].clone().requires_grad_(True)
    with pytest.raises(AssertionError, match="inference"):
        paged_append(x[0], grad, x[0], cache, cache, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(AssertionError, match="inference"):
        flash_bias_paged_func(grad, cache, cache, table, ints[0], ints[1])
    with pytest.raises(AssertionError, match="constant"):
        norm_rope_func(x, x, torch.arange(4), torch.ones(4, requires_grad=True))


@pytest.mark.parametrize("which", range(4))
def test_tangents_are_refused(which):
    import torch.autograd.forward_ad as fwAD
    t = [torch.randn(1, 4, 2, 8).half(), torch.randn(1, 4, 2, 8).half(), torch.ones(8).half(), torch.ones(8).half()]
    with fwAD.dual_level():
        t[which] = fwAD.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            norm_rope_func(t[0], t[1], None, None, t[2], t[3])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_oracle_gradients_against_differences(norm, interleaved):
    g = torch.Generator().manual_seed(5)
    x, d = (torch.randn(1, 3, 2, 10, generator=g, dtype=torch.float64) for _ in range(2))
    w = torch.rand(10, generator=g, dtype=torch.float64) + 0.5 if norm else None
    ang = orc.rope_angles(torch.tensor([0, 5, -3]), torch.tensor([1.0, 0.3, 0.01]))
    dx, dw, _, _ = orc.norm_rope_grads(x, d, w, ang, interleaved)
    h = 1e-6
    for i in range(x.numel()):
        e = torch.zeros(x.numel(), dtype=torch.float64)
        e[i] = h
        e = e.view_as(x)
        num = ((orc.norm_rope(x + e, w, ang, interleaved) - orc.norm_rope(x - e, w, ang, interleaved)) * d).sum() / (2 * h)
        assert abs(float(num - dx.flatten()[i])) < 1e-7  # (differences of second order: h^2, and 1e-16 / h)
    for i in range(10 if norm else 0):
        e = torch.zeros(10, dtype=torch.float64)
        e[i] = h
        num = ((orc.norm_rope(x, w + e, ang, interleaved) - orc.norm_rope(x, w - e, ang, interleaved)) * d).sum() / (2 * h)
        assert abs(float(num - dw[i])) < 1e-7


@pytest.mark.parametrize("change,kernel", [
    (dict(), "split"), (dict(N=48), "split"), (dict(N=49), "tile"), (dict(N=96, Hq=2), "split"), (dict(N=97, Hq=2), "tile"), (dict(N=80, D=32), "split"),
    (dict(N=81, D=32), "tile"), (dict(N=24, D=128), "split"), (dict(N=25, D=128), "tile"),
    (dict(N=50, page_size=8), "tile"), (dict(N=50, page_size=24), "split"), (dict(N=50, page_size=4), "split"), (dict(N=50, page_size=256), "tile"),
    (dict(N=50, softmax_scale=-1.0), "split"), (dict(N=50, flags=_lib.FB_FLAG_PAGED_SPLIT), "split"), (dict(D=20), "general"),
    (dict(N=34, D=128, o_stride=_lib.I64x2(512, 128)), "tile"), (dict(key_cache=0x1008), "general"), (dict(key_cache_stride=_lib.I64x3(4096, 64, 257)), "general"),
    (dict(N=50, key_cache_stride=_lib.I64x3(4096, 0, 256)), "split"), (dict(flags=_lib.FB_FLAG_FORCE_GENERAL), "general"),
    (dict(N=50, R=4, q_bias=0x1000, bias_cache=0x1000, bias_heads=2), "split")], ids=str)
def test_the_query_names_the_kernel_of_paged_attention(change, kernel):
    p = paged_params()
    for n, v in change.items():
        setattr(p, n, v)
    assert _lib.PAGED_KERNELS[_lib.load().fb_paged_kernel(C.byref(p))] == kernel
    assert (_lib.load().fb_paged_workspace_bytes(C.byref(p)) > 0) == (kernel != "general")


@pytest.mark.parametrize("change,workspace", [(dict(), True), (dict(table_width=512), False), (dict(table_width=513), True),
                                              (dict(table_width=512, N=8, B=8), False), (dict(table_width=512, N=64, B=64), True)], ids=str)
def test_few_requests_over_short_tables_need_no_workspace(change, workspace):
    p = paged_params()
    for n, v in change.items():
        setattr(p, n, v)
    assert _lib.PAGED_KERNELS[_lib.load().fb_paged_kernel(C.byref(p))] == "split"
    assert (_lib.load().fb_paged_workspace_bytes(C.byref(p)) > 0) == workspace
