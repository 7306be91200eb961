"""The 8-bit cache: rows as they are written and read back, and attention over it, against 64 bits."""
import math

import pytest
import torch

from cache8_cases import TINY, TOP, TYPES, Step, check, e4m3_grid, quantise

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ written and read back
def write(qkv, bias, nh, nkv, d, form, page_size, positions, seq, slots, table, n_pages, layers=2, layer=1, q_out=True, **more):
    from swifttransformer_b200 import ops
    pool, scales = ops.cache8_pool(n_pages, layers, nkv, page_size, d, TYPES[form], "cuda")
    q = torch.full((qkv.shape[0], nh * d), 77.0, dtype=qkv.dtype, device="cuda") if q_out else None
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.qkv_to_cache8(qkv, bias, q, pool, scales, layer, positions, seq, slots, table, nh, nkv, d, status, **more)
    return pool, scales, q, status


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("nh,nkv,d,page_size,n,bias", [(4, 4, 64, 16, 5, True), (8, 2, 128, 8, 3, False), (3, 3, 80, 7, 9, True), (2, 1, 256, 16, 2, True),
                                                       (5, 5, 13, 1, 4, True), (1, 1, 1, 3, 6, False), (32, 32, 64, 32, 40, True), (2, 2, 24, 4, 700, True)])
def test_rows_written_and_read_back(form, act, nh, nkv, d, page_size, n, bias):
    """Codes, scales and queries to the last bit."""
    from swifttransformer_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn((n, (nh + 2 * nkv) * d), generator=gen, device="cuda") * torch.exp(2 * torch.randn((n, 1), generator=gen, device="cuda"))
    x[0] = 0.0                                            # a row of zeros
    x[1, nh * d:] *= 1e-38                                # below the least scale
    x[-1, nh * d:] *= 1e30
    qkv = x.to(TYPES[act])
    b = torch.randn(x.shape[1], generator=gen, device="cuda") if bias else None
    if bias:
        b[nh * d:] *= 1e-39
    pages = -(-n // page_size)
    order = torch.randperm(pages + 1, generator=torch.Generator().manual_seed(n)).tolist()
    table = ints([[-1] * pages, order[:pages]])
    positions, seq, slots = ints(list(range(n))), ints([0] * n), ints([1])
    pool, scales, q, status = write(qkv, b, nh, nkv, d, form, page_size, positions, seq, slots, table, pages + 1)
    assert int(status) == 0
    f = qkv.float() + b if bias else qkv.float()
    assert torch.equal(q, f[:, :nh * d].to(qkv.dtype))
    code, scale = quantise(f[:, nh * d:].reshape(n, 2, nkv, d).contiguous(), form)
    page = table[1].long()[torch.arange(n, device="cuda") // page_size]
    off = torch.arange(n, device="cuda") % page_size
    got_scale = scales[page, 1][torch.arange(n), :, :, off]
    assert torch.equal(got_scale, scale)
    got = pool.view(torch.int8)[page, 1][torch.arange(n), :, :, off].view(TYPES[form]).double()
    assert torch.equal(got, code)
    assert float(scales[:, 0].abs().max()) == 0 and int(pool.view(torch.int8)[:, 0].abs().max()) == 0       # the other layer
    for out_type in (torch.float32, torch.bfloat16):
        back = ops.cache8_rows(pool, scales, 1, torch.full((n, 2 * nkv * d), 77.0, dtype=out_type, device="cuda"), positions, seq, slots,
                               table, status)
        want = (code.float() * scale.unsqueeze(-1)).reshape(n, -1).to(out_type)
        assert torch.equal(back, want)
    assert int(status) == 0


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 13])
def test_borders_between_codes(form, d):
    """Numbers on and next to the middle between two codes, behind a largest element that fixes the scale."""
    rows = []
    grid = [float(i) for i in range(127)] if form == "int8" else e4m3_grid()
    for s in (1.0, 0.37, 3.3e-5, 1.7e20):
        mids = [(a + b) / 2 for a, b in zip(grid, grid[1:])]
        top = torch.tensor(TOP[form] * s, dtype=torch.float32)
        scale = float((top.double() / TOP[form]).float())
        near = []
        for m in mids:
            x = torch.tensor(m * scale, dtype=torch.float32)
            near += [x, torch.nextafter(x, torch.tensor(math.inf)), torch.nextafter(x, torch.tensor(-math.inf)), -x]
        for i in range(0, len(near), d - 1):
            part = near[i:i + d - 1]
            rows.append(torch.stack([top] + part + [torch.tensor(0.0)] * (d - 1 - len(part))))
    x = torch.stack(rows).cuda()
    n = x.shape[0]
    qkv = torch.cat([torch.zeros_like(x), x, x.flip(0)], dim=1)
    pool, scales, _, _ = write(qkv, None, 1, 1, d, form, n, ints(list(range(n))), ints([0] * n), ints([0]), ints([[0]]), 1, 1, 0)
    code, scale = quantise(torch.stack([x, x.flip(0)], 0), form)
    assert torch.equal(scales[0, 0, :, 0], scale)
    assert torch.equal(pool[0, 0, :, 0].double(), code)


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 30])
@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_rows_that_are_not_finite(form, act, d):
    from swifttransformer_b200 import ops
    n, x = 6, torch.randn((6, 6 * d), device="cuda")
    x[1, 2 * d + 3], x[2, 3 * d], x[3, 5 * d + 1] = math.nan, math.inf, -math.inf
    pos, seq, slots, table = ints([0, 1, 2, 3, 4, 5]), ints([0] * n), ints([0]), ints([[1, 0]])
    pool, scales, _, _ = write(x.to(TYPES[act]), None, 2, 2, d, form, 4, pos, seq, slots, table, 2)
    back = ops.cache8_rows(pool, scales, 1, torch.empty((n, 4 * d), device="cuda"), pos, seq, slots, table).view(n, 4, d)
    odd = torch.zeros((n, 4), dtype=torch.bool, device="cuda")
    odd[1, 0] = odd[2, 1] = odd[3, 3] = True
    assert torch.equal(torch.isnan(back).all(-1), odd) and torch.equal(torch.isnan(back).any(-1), odd)
    assert int(pool.view(torch.int8)[1, 1, 0, 0, 1].abs().max()) == 0


def test_padding_holes_and_queries_in_place():
    from swifttransformer_b200 import ops
    qkv = torch.randn((5, 3 * 64), device="cuda").bfloat16()
    pos, seq, slots, table = ints([0, -1, 20, 1, 500]), ints([0, 0, 0, 0, 0]), ints([0]), ints([[2, -1]])
    pool, scales, q, status = write(qkv, None, 1, 1, 64, "int8", 16, pos, seq, slots, table, 3)
    assert int(status) == 1
    assert torch.equal(q, qkv[:, :64])
    live = scales[:, 1, 0, 0].nonzero().tolist()
    assert live == [[2, 0], [2, 1]] and float(scales[:2].abs().max()) == 0
    status.zero_()
    back = ops.cache8_rows(pool, scales, 1, torch.full((5, 128), 77.0, device="cuda"), pos, seq, slots, table, status)
    assert int(status) == 1
    assert float(back[1].min()) == 77.0 and float(back[2].abs().max()) == 0 and float(back[4].abs().max()) == 0
    assert float(back[0].abs().max()) > 0 and float(back[3].abs().max()) > 0
    bad = ints([[7, 0]])                                   # a page the pool does not have
    pool2, scales2, _, status = write(qkv, None, 1, 1, 64, "int8", 16, ints([0, 1, 2, 3, 4]), seq, slots, bad, 3)
    assert int(status) == 1 and float(scales2.abs().max()) == 0
    pool3, scales3, _, status = write(qkv, None, 1, 1, 64, "int8", 16, ints([0, 1, 2, 3, 4]), seq, slots, table, 3, q_out=False, write_kv=False)
    assert int(status) == 0 and float(scales3.abs().max()) == 0


# ------------------------------------------------------------------ single tokens
def single(step, window=0, items=None, n_items=None, max_kv=0):
    from swifttransformer_b200 import ops
    out = step.out()
    return ops.attention_cache8_single(step.q, step.pool, step.scales, step.layer, out, items, n_items if n_items is not None else step.n,
                                       step.positions, step.seq, step.slots, step.table, step.heads, step.scale, window, max_kv, step.status)


HEADS = [(4, 4, 64), (4, 4, 128), (8, 2, 64), (2, 2, 80), (6, 2, 96), (2, 1, 32), (24, 2, 128), (12, 1, 64), (16, 1, 80), (40, 2, 32), (10, 1, 96), (3, 3, 40),
         (2, 1, 13), (1, 1, 256), (4, 1, 1)]


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_single_tokens(form, act, heads, kv, dim):
    step = Step([(0, 1), (1, 1), (6, 1), (15, 1), (16, 1), (31, 1), (32, 1), (300, 1), (77, 1)], heads, kv, dim, form, act, 16, seed=dim, pad=2)
    check(step, single(step))
    assert int(step.status) == 0
    check(step, single(step, window=9), window=9)
    check(step, single(step, window=64, max_kv=301), window=64)


@pytest.mark.parametrize("page_size", [1, 4, 7, 8, 24, 64])
@pytest.mark.parametrize("form,act", [("int8", "bf16"), ("e4m3", "f32")])
def test_single_tokens_over_pages(page_size, form, act):
    step = Step([(200, 1), (63, 1), (64, 1), (7, 3)], 4, 2, 64, form, act, page_size, seed=page_size)
    check(step, single(step))
    check(step, single(step, window=50), window=50)


@pytest.mark.parametrize("form,act,dim", [("int8", "bf16", 64), ("e4m3", "bf16", 128), ("int8", "f32", 128), ("e4m3", "f32", 24)])
@pytest.mark.parametrize("context", [2000, 9000])
def test_single_token_over_a_long_cache(form, act, dim, context):
    """One request: its keys go to a cluster of blocks."""
    step = Step([(context, 1)], 2, 1, dim, form, act, 16, seed=context, layers=1, layer=0)
    check(step, single(step, max_kv=context))
    check(step, single(step, window=1500), window=1500)


@pytest.mark.parametrize("form,act", [("int8", "bf16"), ("e4m3", "f32")])
def test_many_single_tokens(form, act):
    step = Step([(5 * i % 97, 1) for i in range(300)], 8, 8, 64, form, act, 16, seed=3)
    check(step, single(step))


@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (8, 2, 128), (24, 2, 64), (12, 3, 80), (6, 2, 96), (2, 2, 32), (20, 2, 128)])
@pytest.mark.parametrize("form,act", [("int8", "bf16"), ("e4m3", "bf16"), ("int8", "f32"), ("e4m3", "f32")])
def test_tokens_dealt_out_as_one_line(form, act, heads, kv, dim):
    """A block table with room for so many keys that the calls are dealt out run by run: units in one warp, cut by one warp's end, by many."""
    step = Step([(0, 1), (2900, 1), (40, 2), (7, 1), (640, 1), (33, 1), (64, 1)], heads, kv, dim, form, act, 16, seed=dim + 1, pad=2, table_wide=4000)
    check(step, single(step))
    assert int(step.status) == 0
    check(step, single(step, window=70), window=70)
    got = single(step, items=ints([6, -1, 1, 9, 3]), n_items=5)
    check(step, got, rows=[1, 3, 6])
    others = [0, 2, 4, 5, 7, 8, 9]
    assert float(got[others].min()) == 77.0 and float(got[others].max()) == 77.0
    assert torch.equal(single(step), single(step))
    s = step.slots.tolist()
    step.table[s[1], 3] = -1
    step.table[s[4], :] = 99999
    hidden = [(1, j) for j in range(48, 64)] + [(4, j) for j in range(641)]
    check(step, single(step), hidden=hidden)
    assert int(step.status) == 1


@pytest.mark.parametrize("form,act,heads,dim", [("int8", "bf16", 8, 64), ("e4m3", "bf16", 16, 128), ("e4m3", "f32", 8, 64)])
def test_a_line_of_windows(form, act, heads, dim):
    """So many windows that the call is dealt out as one line: whole ones, ones that reach before the first key, empty lengths."""
    step = Step([(11 * i % 700, 1) for i in range(190)], heads, 8, dim, form, act, 16, seed=6)
    check(step, single(step, window=400), window=400)
    assert int(step.status) == 0


def test_more_tokens_than_a_line_takes():
    step = Step([(13 * i % 61, 1) for i in range(1100)], 4, 2, 64, "int8", "bf16", 16, seed=7, table_wide=40)
    check(step, single(step))


@pytest.mark.parametrize("form,act,dim", [("int8", "bf16", 64), ("e4m3", "f32", 128), ("int8", "f32", 24)])
@pytest.mark.parametrize("table_wide", [0, 5000])
@pytest.mark.parametrize("far", [3, 2 ** 31 - 1])
def test_positions_past_the_block_table(form, act, dim, table_wide, far):
    """A token that stands behind all keys the table has room for sees those that are there; one whose window lies behind them sees none."""
    step = Step([(31, 1), (47, 1), (20, 1)], 4, 2, dim, form, act, 16, seed=dim, table_wide=table_wide)
    reach = step.table.shape[1] * 16
    step.positions[1] = reach + far if far < 1000 else far
    check(step, single(step))
    assert int(step.status) == 1
    got = single(step, window=3)
    check(step, got, window=3, rows=[0, 2])
    assert float(got[1].abs().max()) == 0.0


@pytest.mark.parametrize("table_wide", [0, 5000])
def test_the_same_token_twice_and_padding_alone(table_wide):
    step = Step([(40, 1), (700, 1), (9, 1)], 4, 2, 64, "int8", "bf16", 16, seed=8, pad=2, table_wide=table_wide)
    check(step, single(step, items=ints([1, 0, 1, 1, 2, 0]), n_items=6), rows=[0, 1, 2])
    assert float(single(step, items=ints([3, 4, -1]), n_items=3).min()) == 77.0


@pytest.mark.parametrize("form,act", [("int8", "bf16"), ("e4m3", "f32")])
def test_a_pool_of_more_than_four_gigabytes(form, act):
    """Pages all over it, for single tokens, for portions, for the write and for rows read back."""
    step = Step([(500, 40), (100, 1), (290, 7)], 8, 8, 128, form, act, 64, seed=9, spare=20000)
    assert step.pool.numel() > 2 ** 32
    check(step, single(step))
    check(step, portion(step))
    from swifttransformer_b200 import ops
    rows = torch.empty((step.n, 2 * 8 * 128), dtype=TYPES[act], device="cuda")
    ops.cache8_rows(step.pool, step.scales, step.layer, rows, step.positions, step.seq, step.slots, step.table, step.status)
    qkv = torch.cat([step.q, rows], dim=1)
    before, scales = rows.clone(), step.scales.nan_to_num()
    ops.qkv_to_cache8(qkv, None, None, step.pool, step.scales, step.layer, step.positions, step.seq, step.slots, step.table, 8, 8, 128, step.status)
    ops.cache8_rows(step.pool, step.scales, step.layer, rows, step.positions, step.seq, step.slots, step.table, step.status)
    assert torch.allclose(rows.float(), before.float(), rtol=2.0 ** -3, atol=2.0 ** -6 * float(before.abs().max()))
    changed = (step.scales.nan_to_num() != scales).sum()
    assert int(changed) <= step.n * 2 * 8 and int(step.status) == 0


@pytest.mark.parametrize("form,act", [("int8", "bf16"), ("e4m3", "f32")])
def test_captured_steps_on_two_streams_at_once(form, act):
    """Single tokens as one line, and portions, recorded in two graphs that replay beside one another; a third graph on the first one's
    stream, and eager calls between: the bits of calls made one by one."""
    steps = [Step([(0, 30), (900 + 100 * i, 3), (250, 140)], 4, 2, 64, form, act, 16, seed=i, table_wide=4000) for i in range(3)]
    streams, graphs, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [], []

    def both(step):
        return torch.stack([single(step), portion(step)])

    for step in steps:
        both(step)
    from swifttransformer_b200 import ops
    plans = [ops.portion_plan([n for _, n in s.requests], [b for b, _ in s.requests], 4, 2, 0, "cuda") for s in steps]
    torch.cuda.synchronize()
    for i, s in enumerate(steps):
        out, g = [s.out(), s.out()], torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i % 2]):
            ops.attention_cache8_single(s.q, s.pool, s.scales, s.layer, out[0], None, s.n, s.positions, s.seq, s.slots, s.table, 4, s.scale,
                                        status=s.status)
            ops.attention_cache8_tiles(s.q, s.pool, s.scales, s.layer, out[1], plans[i], s.positions, s.slots, s.table, 4, s.scale,
                                       status=s.status)
        graphs.append(g)
        outs.append(out)
    for turn in range(4):
        for i, s in enumerate(steps):
            s.q.copy_(torch.randn(s.q.shape, generator=torch.Generator(device="cuda").manual_seed(10 * turn + i), device="cuda"))
            s.positions[-1] = 389 - 30 * turn
        torch.cuda.synchronize()
        for i in (0, 1, 2, 0, 1):
            with torch.cuda.stream(streams[i % 2]):
                graphs[i].replay()
        between = both(steps[1])
        torch.cuda.synchronize()
        for i, s in enumerate(steps):
            want = both(s)
            assert torch.equal(torch.stack(outs[i]), want), (turn, i)
        assert torch.equal(between, both(steps[1]))


def test_listed_tokens_only():
    step = Step([(40, 3), (0, 2), (9, 1)], 4, 4, 64, "int8", "bf16", 16, seed=5)
    got = single(step, items=ints([4, -1, 2, 0]), n_items=4)
    check(step, got, rows=[0, 2, 4])
    assert float(got[[1, 3, 5]].min()) == 77.0 and float(got[[1, 3, 5]].max()) == 77.0
    assert float(single(step, n_items=0).min()) == 77.0


@pytest.mark.parametrize("dim", [64, 40])
def test_keys_without_a_page(dim):
    step = Step([(70, 1), (20, 1), (40, 1)], 2, 2, dim, "e4m3", "bf16", 8, seed=1)
    s = step.slots.tolist()
    step.table[s[0], 2] = -1
    step.table[s[1], :] = -1
    step.table[s[2], 1] = 12345
    hidden = [(0, j) for j in range(16, 24)] + [(1, j) for j in range(21)] + [(2, j) for j in range(8, 16)]
    check(step, single(step), hidden=hidden)
    assert int(step.status) == 1


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 40])
def test_sizes_of_rows(act, dim):
    """Values whose scales differ by 2^60, zero rows, queries far from one: powers of two leave the sums as exact as they were."""
    step = Step([(130, 1), (64, 1)], 4, 2, dim, "int8", act, 16, seed=2, q_std=1e-9, k_std=1e9)
    for r in range(2):
        at = step.table[int(step.slots[r])].long()
        step.scales[at[0], step.layer, 1, :, :4] *= 2.0 ** -60
        step.v[r][:, :4] *= 2.0 ** -60
        step.pool.view(torch.int8)[at[1], step.layer, 1, :, 3] = 0
        step.scales[at[1], step.layer, 1, :, 3] = TINY
        step.v[r][:, 19] = 0.0
        step.scales[at[2], step.layer, 1, :, 5] *= 2.0 ** 40
        step.v[r][:, 37] *= 2.0 ** 40
    check(step, single(step))


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 40])
def test_rows_that_are_not_finite_reach_who_sees_them(act, dim):
    step = Step([(60, 1), (30, 1)], 2, 2, dim, "int8", act, 16, seed=2)
    step.scales[step.table[int(step.slots[0])].long()[1], step.layer, 1, 0, 4] = math.nan       # key 20 of request 0, head 0: its values
    got = single(step)
    assert torch.isnan(got[0, :dim]).all() and not torch.isnan(got[0, dim:]).any() and not torch.isnan(got[1]).any()
    check(step, single(step, window=40), window=40)          # keys 21 .. 60
    step.q[1, 0] = math.nan
    got = single(step)
    assert torch.isnan(got[1, :dim]).all() and not torch.isnan(got[1, dim:]).any()


# ------------------------------------------------------------------ portions
def portion(step, window=0, q=None):
    from swifttransformer_b200 import ops
    plan = ops.portion_plan([n for _, n in step.requests], [b for b, _ in step.requests], step.heads, step.kv, window, "cuda")
    return ops.attention_cache8_tiles(step.q if q is None else q, step.pool, step.scales, step.layer, step.out(), plan, step.positions,
                                      step.slots, step.table, step.heads, step.scale, window, step.status)


@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (4, 1, 64), (2, 2, 128), (6, 2, 80), (1, 1, 16), (3, 1, 48), (2, 1, 13), (1, 1, 256), (40, 1, 32), (100, 1, 16)])
@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_portions(form, act, heads, kv, dim):
    step = Step([(0, 1), (0, 150), (200, 20), (127, 2), (63, 65)], heads, kv, dim, form, act, 16, seed=dim, pad=3)
    check(step, portion(step))
    check(step, portion(step, window=40), window=40)
    assert int(step.status) == 0


@pytest.mark.parametrize("page_size", [1, 4, 7, 8, 24, 64])
@pytest.mark.parametrize("form,act", [("int8", "bf16"), ("e4m3", "f32")])
def test_portions_over_pages(page_size, form, act):
    step = Step([(30, 100), (0, 9)], 4, 2, 64, form, act, page_size, seed=page_size)
    check(step, portion(step))


@pytest.mark.parametrize("form,act,dim", [("int8", "bf16", 64), ("e4m3", "bf16", 128), ("int8", "f32", 64)])
def test_a_long_prompt_and_a_portion_behind_a_long_cache(form, act, dim):
    step = Step([(0, 700), (3000, 130)], 2, 2, dim, form, act, 16, seed=4, layers=1, layer=0)
    check(step, portion(step))
    check(step, portion(step, window=500), window=500)


def test_queries_inside_the_projection():
    step = Step([(0, 70), (5, 3)], 2, 2, 64, "int8", "bf16", 16, seed=4)
    wide = torch.randn((step.n, 6 * 64), device="cuda").bfloat16()
    wide[:, :128] = step.q
    check(step, portion(step, q=wide[:, :128]))


@pytest.mark.parametrize("act,dim", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_portions_with_keys_without_a_page(act, dim):
    step = Step([(70, 20), (0, 30), (40, 2)], 2, 2, dim, "e4m3", act, 8, seed=1)
    s = step.slots.tolist()
    step.table[s[0], 2] = -1
    step.table[s[1], :] = -1
    step.table[s[2], 1] = 12345
    hidden = [(0, j) for j in range(16, 24)] + [(1, j) for j in range(30)] + [(2, j) for j in range(8, 16)]
    check(step, portion(step), hidden=hidden)
    assert int(step.status) == 1


@pytest.mark.parametrize("act,dim", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_sizes_of_rows_in_portions(act, dim):
    step = Step([(30, 100), (0, 40)], 2, 1, dim, "int8", act, 16, seed=2, q_std=1e-9, k_std=1e9)
    for r in range(2):
        at = step.table[int(step.slots[r])].long()
        step.scales[at[0], step.layer, 1, :, :4] *= 2.0 ** -60
        step.v[r][:, :4] *= 2.0 ** -60
        step.pool.view(torch.int8)[at[1], step.layer, 1, :, 3] = 0
        step.scales[at[1], step.layer, 1, :, 3] = TINY
        step.v[r][:, 19] = 0.0
        step.scales[at[2], step.layer, 1, :, 5] *= 2.0 ** 40
        step.v[r][:, 37] *= 2.0 ** 40
    check(step, portion(step))


@pytest.mark.parametrize("act,dim", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_a_row_that_is_not_finite_in_a_portion(act, dim):
    """Key 20's values are NaN: the rows before it are as if it were not there."""
    step = Step([(0, 60)], 2, 2, dim, "int8", act, 16, seed=2)
    step.scales[step.table[int(step.slots[0])].long()[1], step.layer, 1, 0, 4] = math.nan
    got = portion(step)
    check(step, got, rows=list(range(20)))
    assert torch.isnan(got[20:, :dim]).all() and not torch.isnan(got[:, dim:]).any()


def test_the_same_bits_again():
    step = Step([(0, 400), (900, 60)], 4, 4, 64, "int8", "bf16", 16, seed=4)
    first = portion(step)
    for _ in range(3):
        assert torch.equal(portion(step), first)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_a_request_from_its_prompt_on(form, act):
    """A prompt in two portions, then single tokens, each step's rows written before they are read: every row as in 64 bits over
    the rows the cache holds, and the whole run again as captured graphs on another stream."""
    from swifttransformer_b200 import ops
    nh, nkv, d, page, total = 4, 2, 64, 16, 90
    gen = torch.Generator(device="cuda").manual_seed(9)
    qkv = torch.randn((total, (nh + 2 * nkv) * d), generator=gen, device="cuda").to(TYPES[act])
    bias = 0.1 * torch.randn(qkv.shape[1], generator=gen, device="cuda")
    table, slots = ints([[3, 0, 5, 1, 2, 4]]), ints([0])
    steps = [(0, 50), (50, 35)] + [(p, 1) for p in range(85, total)]

    def run(pool, scales, outs, data):
        for (start, n), out, (pos, seq, plan, x) in zip(steps, outs, data):
            q = torch.empty((n, nh * d), dtype=x.dtype, device="cuda")
            ops.qkv_to_cache8(x, bias, q, pool, scales, 0, pos, seq, slots, table, nh, nkv, d)
            if n > 1:
                ops.attention_cache8_tiles(q, pool, scales, 0, out, plan, pos, slots, table, nh, d ** -0.5)
            else:
                ops.attention_cache8_single(q, pool, scales, 0, out, None, 1, pos, seq, slots, table, nh, d ** -0.5, max_kv=start + 1)

    data = [(ints(list(range(s, s + n))), ints([0] * n), ops.portion_plan([n], [s], nh, nkv, device="cuda"), qkv[s:s + n].contiguous())
            for s, n in steps]
    outs = [torch.empty((n, nh * d), dtype=qkv.dtype, device="cuda") for _, n in steps]
    pool, scales = ops.cache8_pool(6, 1, nkv, page, d, TYPES[form], "cuda")
    run(pool, scales, outs, data)
    whole = torch.cat(outs)
    f = qkv.float() + bias
    step = Step([(0, total)], nh, nkv, d, form, act, page)
    code, s = quantise(f[:, nh * d:].reshape(total, 2, nkv, d).contiguous(), form)
    rows = (code * s.double().unsqueeze(-1)).permute(1, 2, 0, 3)
    step.q, step.k, step.v = f[:, :nh * d].to(qkv.dtype), [rows[0]], [rows[1]]
    check(step, whole)
    assert ops.kernel_status("cuda") == 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pool2, scales2 = ops.cache8_pool(6, 1, nkv, page, d, TYPES[form], "cuda")
    outs2 = [torch.empty_like(o) for o in outs]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run(pool2, scales2, outs2, data)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(torch.cat(outs2), whole)
        assert torch.equal(pool2.view(torch.int8), pool.view(torch.int8)) and torch.equal(scales2, scales)
