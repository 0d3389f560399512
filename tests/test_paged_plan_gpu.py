"""The plan of a serving step against sequential code: pages given back and taken, refusals, trees, many requests and tokens."""
import pytest
import torch

from flashbias_b200 import check_device_status, paged_plan
from oracle import serving_oracle as orc
from tests.serving_helpers import pool_of, tree

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def run(state, lens, new, page, N, parents=None, max_tree=64):
    table, held, stack, count = state
    dev = [ints(table), ints(held), ints(stack), ints([count])]
    step = paged_plan(*dev, ints(lens), ints(new), page, N, None if parents is None else parents.cuda(), max_tree)
    return dev, step


def check(state, lens, new, page, N, parents=None, max_tree=64):
    want = orc.plan(*state, lens, new, page, N, None if parents is None else parents.tolist(), max_tree)
    (table, held, stack, count), step = run(state, lens, new, page, N, parents, max_tree)
    torch.cuda.synchronize()
    check_device_status()
    assert table.tolist() == want["table"] and held.tolist() == want["held"]
    assert count.tolist() == [want["count"]] and stack.tolist()[:want["count"]] == want["stack"][:want["count"]]
    assert step.lens.tolist() == want["lens"] and step.cu_tokens.tolist() == want["cu"]
    assert step.slots.tolist() == want["slots"] and step.positions.tolist() == want["positions"]
    if parents is not None:
        assert step.tree_mask.tolist() == want["masks"]
    return want


@pytest.mark.parametrize("B,longest,T,page", [(1, 0, 1, 16), (1, 5, 1, 1), (3, 40, 1, 16), (17, 100, 9, 7), (64, 500, 3, 32), (1000, 60, 2, 8),
                                              (1024, 30, 1, 16), (1025, 30, 4, 16), (3000, 10, 5, 4), (2, 3000, 20000, 64), (5, 900, 4000, 16)])
def test_growth(B, longest, T, page):
    g = torch.Generator().manual_seed(B + T)
    lens, new = torch.randint(0, longest + 1, (B,), generator=g).tolist(), torch.randint(0, T + 1, (B,), generator=g).tolist()
    width = max(-(-(a + b) // page) for a, b in zip(lens, new)) + 1
    N = sum(new) + 3
    want = check(pool_of(lens, new, page, width, B), lens, new, page, N)
    assert -1 not in want["lens"] and want["slots"][-3:] == [-1] * 3


def test_requests_that_end_give_their_pages_to_those_that_grow():
    page, lens = 8, [40, 17, 64, 3]
    state = pool_of(lens, [0] * 4, page, 12, 1, spare=1)
    # requests 0 and 2 end (13 pages), 1 shrinks, 3 grows beyond what was free before
    want = check(state, [0, 5, 0, 3], [0, 0, 0, 80], page, 80)
    assert want["lens"] == [0, 5, 0, 3] and want["held"] == [0, 1, 0, 11]
    # everything back: the stack holds every page once
    want = check((want["table"], want["held"], want["stack"], want["count"]), [0] * 4, [0] * 4, page, 0)
    assert want["count"] == len(state[2]) and sorted(want["stack"]) == list(range(len(state[2])))


def test_growing_and_shrinking_back_restores_the_stack():
    page, lens, new = 16, [33, 0, 100, 15], [20, 64, 1, 2]
    state = pool_of(lens, new, page, 10, 2, spare=5)
    dev, _ = run(state, lens, new, page, sum(new))
    before = [ints(x) for x in (state[1], state[2], [state[3]])]
    paged_plan(*dev, ints(lens), ints([0] * 4), page, 0)
    assert all(torch.equal(a, b) for a, b in zip(dev[1:], before))


def test_refusals_of_requests():
    page, lens = 8, [8, 8, 8, -1, 8, 8, 8, 0]
    new = [8, 9, 8, 1, -3, 60, 8, 70]
    state = pool_of(lens, [0] * 8, page, 8, 3, spare=3)
    # 0 takes one page, 1 two, then none is left: 2 and 6 are refused, negative lengths (3, 4), a row too short (5, 7)
    want = check(state, lens, new, page, 300)
    assert want["lens"] == [8, 8, -1, -1, -1, -1, -1, -1] and want["count"] == 0
    # what needs no page is served all the same
    want = check(state, [8, 8, 8, 0, 8, 8, 8, 0], [16, 16, 0, 0, 8, 0, 0, 0], page, 100)
    assert want["lens"] == [8, -1, 8, 0, -1, 8, 8, 0] and want["count"] == 1


def test_tokens_beyond_the_step_are_refused():
    want = check(pool_of([5, 5, 5], [4, 4, 0], 4, 4, 4), [5, 5, 5], [4, 4, 0], 4, 6)
    assert want["lens"] == [5, -1, -1] and want["cu"] == [0, 4, 6, 6] and want["slots"][4:] == [-1, -1]


@pytest.mark.parametrize("new,max_tree", [([1], 64), ([64, 1, 0, 33], 64), ([65, 64], 64), ([65, 130, 200], 200), ([7] * 40, 64), ([256, 3], 256)])
def test_trees(new, max_tree):
    lens = [10 + 3 * b for b in range(len(new))]
    parents, masks, depth = tree(new, 5, -(-max_tree // 64))
    state = pool_of(lens, new, 16, 30, 5)
    want = check(state, lens, new, 16, sum(new), parents, max_tree)
    for b, T in enumerate(new):
        assert (want["lens"][b] == -1) == (T > -(-max_tree // 64) * 64)
    if -1 not in want["lens"]:
        assert want["masks"] == masks.tolist()


def test_deep_tree_and_padding():
    new = [300, 5]
    parents = torch.tensor([t - 1 for t in range(300)] + [-1, 0, 0, 2, -1] + [9, 9], dtype=torch.int32)
    want = check(pool_of([0, 7], new, 32, 12, 6), [0, 7], new, 32, 307, parents, 320)
    assert want["positions"][299] == 299 and want["positions"][300:] == [7, 8, 8, 9, 7, 0, 0]


def test_a_parent_that_is_not_before_its_token_ends_the_path():
    state = pool_of([0], [4], 8, 2, 7)
    _, step = run(state, [0], [4], 8, 4, torch.tensor([-1, 0, 2, 9], dtype=torch.int32))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="out of range"):
        check_device_status()
    assert step.tree_mask.flatten().tolist() == [1, 3, 4, 8] and step.positions.tolist() == [0, 1, 0, 0]


def test_a_page_count_beyond_the_row_is_refused_and_reported():
    table, held, stack, count = pool_of([8, 8], [1, 1], 8, 3, 8)
    (t, h, _, c), step = run((table, [9, 1], stack, count), [8, 8], [1, 1], 8, 2)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="out of range"):
        check_device_status()
    assert step.lens.tolist() == [-1, 8] and h.tolist() == [9, 2] and c.tolist() == [count - 1]


@pytest.mark.parametrize("B", [2, 1500])
@pytest.mark.parametrize("count,counted", [(-3, 0), (10 ** 9, None)])
def test_a_count_of_free_pages_beyond_the_stack_is_reported(B, count, counted):
    """Taken for the nearest one that the stack can have."""
    lens, new = [8] * B, [1] * B
    table, held, stack, _ = pool_of(lens, new, 8, 3, 10)
    stack = stack[:next(i for i, x in enumerate(stack + [-9]) if x < 0)]  # free pages alone
    want = orc.plan(table, held, stack, len(stack) if counted is None else counted, lens, new, 8, B)
    (t, h, _, c), step = run((table, held, stack, count), lens, new, 8, B)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="out of range"):
        check_device_status()
    assert t.tolist() == want["table"] and h.tolist() == want["held"] and c.tolist() == [want["count"]] and step.lens.tolist() == want["lens"]


def test_a_graph_of_the_plan_follows_the_lengths():
    page, lens, new = 16, [30, 50], [1, 1]
    state = pool_of(lens, [60, 60], page, 10, 9)
    dev = [ints(state[0]), ints(state[1]), ints(state[2]), ints([state[3]])]
    l, n = ints(lens), ints(new)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = paged_plan(*dev, l, n, page, 2)
    want = state
    for _ in range(40):
        graph.replay()
        w = orc.plan(*want, l.tolist(), new, page, 2)
        assert dev[0].tolist() == w["table"] and step.slots.tolist() == w["slots"]
        want = (w["table"], w["held"], w["stack"], w["count"])
        l += n
    check_device_status()


@pytest.mark.parametrize("bad", [dict(block_table=torch.zeros(2, 3)), dict(block_table=torch.zeros(0, 3).int()), dict(pages_held=torch.zeros(3).int()),
                                 dict(lens=torch.zeros(2).long()), dict(new_lens=torch.zeros(3).int()), dict(free_count=torch.zeros(2).int()),
                                 dict(page_size=0), dict(page_size=2 ** 30), dict(num_tokens=-1), dict(parents=torch.zeros(5).int()),
                                 dict(parents=torch.zeros(4).int(), max_tree=0), dict(parents=torch.zeros(4).int(), max_tree=4097)], ids=lambda b: "-".join(b))
def test_refusals(bad):
    args = dict(block_table=torch.zeros(2, 3).int(), pages_held=torch.zeros(2).int(), free_pages=torch.arange(9).int(), free_count=ints([9]),
                lens=torch.zeros(2).int(), new_lens=torch.ones(2).int(), page_size=4, num_tokens=4)
    put = (lambda v: v.cuda() if isinstance(v, torch.Tensor) else v)
    paged_plan(**{n: put(v).clone() if isinstance(v, torch.Tensor) else v for n, v in args.items()})
    with pytest.raises(AssertionError):
        paged_plan(**{n: put(v) for n, v in {**args, **bad}.items()})
