"""The operators of a serving step together: prompts, single tokens and trees of drafted tokens of several requests, step after
step through plan, append and attention, against dense attention over everything that each request has seen."""
import math

import pytest
import torch

from flashbias_b200 import check_device_status, flash_bias_paged_func, paged_append, paged_plan
from oracle import serving_oracle as orc
from tests.serving_helpers import assert_within, half_step, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bias", ["slopes", "factors"])
def test_prompts_tokens_and_trees(bias):
    g = torch.Generator().manual_seed(21)
    B, Hq, Hk, D, page, pool, dtype, R = 3, 4, 2, 64, 8, 40, torch.bfloat16, 4
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    state = [ints([[-1] * 20] * B), ints([0] * B), torch.randperm(pool, generator=g).int().cuda(), ints([pool])]
    kc, vc = (torch.full((pool, page, Hk, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    bc = torch.full((pool, page, 1, R), float("nan"), dtype=dtype, device="cuda") if bias == "factors" else None
    slopes = torch.tensor([0.5, 0.2, 0.1, 0.01]) if bias == "slopes" else None
    f = (10000.0 ** (-torch.arange(0, D, 2).double() / D)).float()
    w = [1.0 + 0.1 * torch.randn(D, generator=g) for _ in range(2)]
    past = [dict(k=torch.zeros(0, Hk, D), v=torch.zeros(0, Hk, D), b=torch.zeros(0, 1, R), pos=torch.zeros(0)) for _ in range(B)]
    lens = [0] * B
    # (new tokens, drafted as a tree, kept per request: a prefix of the step's tokens, None: the request ends)
    steps = [([30, 0, 11], False, [30, 0, 11]), ([1, 9, 1], False, [1, 9, 1]), ([12, 5, 1], True, [1, 1, 1]), ([1, 1, 0], False, [1, 1, None]),
             ([1, 20, 40], False, [1, 20, 40]), ([7, 7, 7], True, [1, 1, 1])]
    for new, drafted, kept in steps:
        N = sum(new) + 2  # two rows of padding
        parents, masks, depth = tree(new, N)
        pad = torch.full((2,), -1, dtype=torch.int32)
        plan = paged_plan(*state, ints(lens), ints(new), page, N, torch.cat([parents, pad]).cuda() if drafted else None)
        q, k, v = (torch.randn(N, h, D, generator=g).to(dtype) for h in (Hq, Hk, Hk))
        qb, kb = (torch.randn(N, h, R, generator=g).to(dtype) for h in (Hq, 1))
        more = dict(k_bias=kb.cuda(), bias_cache=bc) if bc is not None else {}
        qr = paged_append(q.cuda(), k.cuda(), v.cuda(), kc, vc, plan.slots, plan.positions, f.cuda(), w[0].cuda(), w[1].cuda(), **more)
        more = dict(q_bias=qb.cuda(), bias_cache=bc) if bc is not None else dict(slopes=slopes.cuda())
        o = flash_bias_paged_func(qr, kc, vc, state[0], plan.lens, plan.cu_tokens, plan.tree_mask, plan.positions, **more).double().cpu()
        check_device_status()
        assert plan.lens.tolist() == lens
        n = 0
        for b in range(B):
            for t in range(new[b]):
                pos = lens[b] + (int(depth[n]) if drafted else t)
                assert int(plan.positions[n]) == pos
                seen = [i for i in range(new[b]) if masks[n, 0] >> i & 1] if drafted else range(t + 1)
                rows = [n - t + i for i in seen]
                at = torch.tensor([[lens[b] + (int(depth[r]) if drafted else r - n + t)] for r in rows])
                # queries and keys as the operator before rounded them: within half a step of the formula
                mine = orc.norm_rope(q[n][None, None], w[0], orc.rope_angles(torch.tensor([pos]), f))[0, 0].to(dtype).double()
                keys = torch.stack([orc.norm_rope(k[r][None, None], w[1], orc.rope_angles(a, f))[0, 0] for r, a in zip(rows, at)]).to(dtype).double()
                K, V = torch.cat([past[b]["k"].double(), keys]), torch.cat([past[b]["v"].double(), v[rows].double()])
                z = torch.einsum("hd,khd->hk", mine, K.repeat_interleave(Hq // Hk, 1)) / math.sqrt(D)
                if bc is None:
                    z += slopes.double()[:, None] * (torch.cat([past[b]["pos"], at[:, 0]]).double() - pos)
                else:
                    z += torch.einsum("hr,kr->hk", qb[n].double(), torch.cat([past[b]["b"].double(), kb[rows].double()])[:, 0])
                p = torch.softmax(z, -1)
                V = V.repeat_interleave(Hq // Hk, 1)
                want, weight = torch.einsum("hk,khd->hd", p, V), torch.einsum("hk,khd->hd", p, V.abs())
                # a few of the keys round the other way than here (their fp32 values differ in the last bits): a step of one
                # value of D each, far below the half step of the probabilities that is counted
                u = half_step(dtype)
                assert_within("o", o[n], want, u * want.abs() + 2 * u * weight)
                n += 1
        assert (o[n:] == 0).all()
        # accepted tokens: a prefix (for a tree its root), moved to their final place by writing them again
        n = 0
        for b in range(B):
            if kept[b] is None:
                lens[b], past[b] = 0, {x: y[:0] for x, y in past[b].items()}
            else:
                for t in range(kept[b]):
                    kr = orc.norm_rope(k[n + t][None, None], w[1], orc.rope_angles(torch.tensor([lens[b] + t]), f))[0].to(dtype)
                    past[b]["k"], past[b]["v"] = torch.cat([past[b]["k"], kr]), torch.cat([past[b]["v"], v[n + t][None]])
                    past[b]["b"], past[b]["pos"] = torch.cat([past[b]["b"], kb[n + t][None]]), torch.cat([past[b]["pos"], torch.tensor([lens[b] + t])])
                lens[b] += kept[b]
            n += new[b]
    # all requests end: the pool is whole again
    paged_plan(*state, ints([0] * B), ints([0] * B), page, 0)
    assert state[3].tolist() == [pool] and sorted(state[2].tolist()) == list(range(pool)) and state[1].tolist() == [0] * B


def test_a_captured_step_runs_on():
    """Plan, append and attention of one decoding step in one graph, replayed: each replay appends a token to every request."""
    B, Hq, Hk, D, page, pool = 2, 4, 2, 64, 4, 30
    g = torch.Generator().manual_seed(22)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    make = lambda h: torch.randn(B, h, D, generator=g).half().cuda()  # noqa: E731
    state = [ints([[-1] * 12] * B), ints([0] * B), torch.arange(pool).int().cuda(), ints([pool])]
    kc, vc = (torch.full((pool, page, Hk, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    q, k, v, lens, one = make(Hq), make(Hk), make(Hk), ints([0] * B), ints([1] * B)

    def step():
        plan = paged_plan(*state, lens, one, page, B)
        qr = paged_append(q, k, v, kc, vc, plan.slots)
        return flash_bias_paged_func(qr, kc, vc, state[0], plan.lens, plan.cu_tokens)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    ks, vs = [], []
    for i in range(30):
        for t, h in ((q, Hq), (k, Hk), (v, Hk)):
            t.copy_(make(h))
        ks.append(k.double().cpu()), vs.append(v.double().cpu())
        graph.replay()
        K, V = (torch.stack(x, 1).repeat_interleave(2, 2) for x in (ks, vs))
        p = torch.softmax(torch.einsum("bhd,bkhd->bhk", q.double().cpu(), K) / 8.0, -1)
        want, weight = torch.einsum("bhk,bkhd->bhd", p, V), torch.einsum("bhk,bkhd->bhd", p, V.abs())
        u = half_step(torch.float16)
        assert_within("o", o, want, u * want.abs() + 1.1 * u * weight)
        lens += 1
    check_device_status()
