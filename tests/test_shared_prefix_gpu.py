"""Attention of single tokens whose requests share a prefix, against 64 bits."""
import math

import pytest
import torch

from cache8_cases import Step, check

pytestmark = pytest.mark.gpu
FORMS = [("bf16", "bf16"), ("f32", "f32"), ("int8", "bf16"), ("e4m3", "bf16"), ("int8", "f32"), ("e4m3", "f32")]


def shared(step, groups, lens, window=0, max_own=0):
    from swifttransformer_b200 import ops
    plan = ops.shared_prefix_plan(groups, lens, step.heads, step.kv, "cuda", max_own)
    return ops.attention_shared_prefix(step.q, step.pool, step.layer, step.out(), plan, step.positions, step.seq, step.slots, step.table,
                                       step.heads, step.scale, window, scales=step.scales, status=step.status)


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (8, 2, 64), (4, 4, 128), (6, 2, 80), (2, 1, 96), (3, 3, 48), (2, 1, 13), (1, 1, 256), (24, 1, 32),
                                          (100, 1, 16)])
def test_groups(form, act, heads, kv, dim):
    """A group of five behind 200 keys, one of two behind 33, one alone behind 40, two that share nothing."""
    requests = [(200, 1), (217, 1), (208, 1), (300, 1), (201, 1), (33, 1), (60, 1), (45, 1), (10, 1), (0, 1)]
    groups, lens = [[0, 1, 2, 3, 4], [6, 5], [7], [8, 9]], [200, 33, 40, 0]
    step = Step(requests, heads, kv, dim, form, act, 16, seed=dim, shared=[([0, 1, 2, 3, 4], 200), ([6, 5], 33)], pad=2)
    check(step, shared(step, groups, lens))
    assert int(step.status) == 0
    check(step, shared(step, groups, lens, max_own=101))
    # a window that begins behind the prefix for some and inside it for others; values that are hidden from some rows of a tile are finite
    check(step, shared(step, groups, lens, window=20), window=20)


@pytest.mark.parametrize("form,act", [f for f in FORMS if f[0] != "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (8, 2, 128), (24, 2, 64), (6, 2, 80)])
def test_own_keys_dealt_out_as_one_line(form, act, heads, kv, dim):
    """With room for so many keys in the block table that the tokens' own keys are dealt out run by run: tokens with many of them, with
    one, inside the prefix with none, and in a group that shares nothing."""
    requests = [(200, 1), (1500, 1), (208, 1), (300, 1), (201, 1), (33, 1), (60, 1), (45, 1), (10, 1), (0, 1)]
    groups, lens = [[0, 1, 2, 3, 4], [6, 5], [7], [8, 9]], [200, 33, 46, 0]
    step = Step(requests, heads, kv, dim, form, act, 16, seed=dim, shared=[([0, 1, 2, 3, 4], 200), ([6, 5], 33)], pad=2, table_wide=5000)
    check(step, shared(step, groups, lens))
    check(step, shared(step, groups, lens, window=20), window=20)
    assert int(step.status) == 0


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("page_size", [1, 7, 8, 64])
def test_pages(form, act, page_size):
    requests = [(150, 1), (140, 1), (151, 2)]
    step = Step(requests, 4, 2, 64, form, act, page_size, seed=page_size, shared=[([0, 1, 2], 139)])
    check(step, shared(step, [[0, 1, 2, 3]], [139]))


@pytest.mark.parametrize("form,act,dim", [("bf16", "bf16", 64), ("bf16", "bf16", 128), ("int8", "bf16", 64), ("e4m3", "bf16", 128), ("f32", "f32", 64),
                                          ("int8", "f32", 64)])
@pytest.mark.parametrize("members,prefix", [(150, 130), (40, 2500), (1, 1000)])
def test_many_members_and_long_prefixes(form, act, dim, members, prefix):
    step = Step([(prefix + 3 * i % 50, 1) for i in range(members)], 2, 2, dim, form, act, 16, seed=members, shared=[(list(range(members)), prefix)],
                layers=1, layer=0)
    check(step, shared(step, [list(range(members))], [prefix], max_own=50))


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 24])
def test_positions_inside_the_prefix(form, act, dim):
    """Tokens that stand inside the shared keys, some of one request, and padding: each sees what lies before it."""
    step = Step([(100, 1), (3, 1), (126, 4), (0, 1)], 4, 2, dim, form, act, 16, seed=dim, pad=1)
    for r in (0, 1, 3):                                                 # shorter requests: their first keys are those of request 2
        n = step.requests[r][0] + 1
        step.k[r], step.v[r] = step.k[2][:, :n], step.v[2][:, :n]
    check(step, shared(step, [[2, 0, 1, 3, 4, 5, 6, 7]], [128]))


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 40])
@pytest.mark.parametrize("gone", [[0], [0, 1, 3], [0, 1, 2, 3]])
def test_members_that_have_left(form, act, dim, gone):
    """Members that are padding now, the first of the group among them: their requests and slots may be anything."""
    step = Step([(70, 1), (75, 1), (64, 1), (90, 1), (20, 1)], 4, 2, dim, form, act, 16, seed=1, shared=[([0, 1, 2, 3], 64)])
    step.positions[gone] = -1
    step.seq[gone] = -1000000000
    got = shared(step, [[0, 1, 2, 3], [4]], [64, 0])
    left = [t for t in range(5) if t not in gone]
    check(step, got, rows=left)
    assert float(got[gone].min()) == 77.0 and float(got[gone].max()) == 77.0
    assert int(step.status) == 0


@pytest.mark.parametrize("form,act", [("bf16", "bf16"), ("f32", "f32"), ("e4m3", "bf16")])
def test_a_pool_of_more_than_four_gigabytes(form, act):
    step = Step([(500, 1), (530, 1), (690, 1)], 8, 8, 128, form, act, 64, seed=9, shared=[([0, 1, 2], 490)], spare=20000)
    assert step.pool.numel() > 2 ** 32
    check(step, shared(step, [[0, 1, 2]], [490]))


def test_tokens_without_a_group_stay():
    step = Step([(40, 1), (41, 1), (42, 1)], 2, 2, 64, "bf16", "bf16", 16, shared=[([0, 2], 32)])
    got = shared(step, [[0, 2]], [32])
    check(step, got, rows=[0, 2])
    assert float(got[1].min()) == 77.0 and float(got[1].max()) == 77.0


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_keys_without_a_page(form, act, dim):
    step = Step([(70, 1), (75, 1), (20, 1)], 2, 2, dim, form, act, 8, seed=1, shared=[([0, 1], 64)])
    s = step.slots.tolist()
    step.table[s[0], 2] = -1                               # inside the prefix, as the group's first request has it
    step.table[s[1], 8] = -1                               # behind it
    step.table[s[2], :] = 99999
    hidden = [(r, j) for r in (0, 1) for j in range(16, 24)] + [(1, j) for j in range(64, 72)] + [(2, j) for j in range(21)]
    check(step, shared(step, [[0, 1], [2]], [64, 8]), hidden=hidden)
    assert int(step.status) == 1


@pytest.mark.parametrize("form,act", [f for f in FORMS if f[0] != "bf16"])
def test_a_row_that_is_not_finite_stays_behind_the_window(form, act):
    step = Step([(100, 1), (140, 1)], 2, 2, 64, form, act, 16, seed=3, shared=[([0, 1], 96)])
    page, off = step.table[int(step.slots[0])].long()[5], 10       # key 90: token 0's window of 30 holds it, token 1's does not
    if step.scales is not None:
        step.scales[page, step.layer, 1, 0, off] = math.nan
    else:
        step.pool[page, step.layer, 1, 0, off] = math.inf
    got = shared(step, [[0, 1]], [96], window=30)
    check(step, got, window=30, rows=[1])
    assert not torch.isfinite(got[0, :64]).any() and torch.isfinite(got[0, 64:]).all()


@pytest.mark.parametrize("form,act", [("bf16", "bf16"), ("int8", "bf16"), ("f32", "f32")])
def test_steps_of_a_batch_captured(form, act):
    """A step captured once and replayed while its tokens move on, beside the same steps launched one by one; two captured graphs on
    two streams at the same time."""
    from swifttransformer_b200 import ops
    steps, plans = [], []
    for seed in (1, 2):
        steps.append(Step([(160 + 20 * i, 1) for i in range(6)], 4, 2, 64, form, act, 16, seed=seed, shared=[(list(range(6)), 160)]))
        plans.append(ops.shared_prefix_plan([list(range(6))], [160], 4, 2, "cuda", 120))

    def go(i, out):
        s = steps[i]
        ops.attention_shared_prefix(s.q, s.pool, s.layer, out, plans[i], s.positions, s.seq, s.slots, s.table, 4, s.scale, scales=s.scales,
                                    status=s.status)

    outs, graphs, streams = [s.out() for s in steps], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in (0, 1):
        go(i, outs[i])
    torch.cuda.synchronize()
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            go(i, outs[i])
        graphs.append(g)
    for back in (0, 1, 5):
        for s in steps:
            s.pos_list = [160 + 20 * i - min(back, 20 * i) for i in range(6)]
            s.positions.copy_(torch.tensor(s.pos_list, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for i in (0, 1):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            check(steps[i], outs[i])
            alone = steps[i].out()
            go(i, alone)
            assert torch.equal(alone, outs[i])


def test_agrees_with_the_single_token_attention():
    """Over a bfloat16 cache: the rows of attention_decode, to the sum of both operators' bounds."""
    from swifttransformer_b200 import ops
    step = Step([(320 + i, 1) for i in range(8)], 4, 4, 64, "bf16", "bf16", 16, seed=8, shared=[(list(range(8)), 320)])
    one = shared(step, [list(range(8))], [320]).double()
    two = ops.attention_decode(step.q, step.pool, step.layer, step.out(), None, step.n, step.positions, step.seq, step.slots, step.table, 4,
                               step.scale).double()
    _, tol = step.expected()
    assert bool(((one - two).abs() <= 2 * tol).all())
