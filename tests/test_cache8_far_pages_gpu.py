"""Writes to and reads from pages beyond 4 GB of a pool, against what was meant."""
import pytest
import torch

from cache8_cases import TYPES, Step, quantise

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form,act,dim", [("int8", "bf16", 128), ("e4m3", "f32", 128), ("int8", "f32", 130)])
def test_rows_lie_where_they_belong(form, act, dim):
    """The rows of a step's tokens as they were laid out, then other rows written over them: those places have the new codes and scales, every
    other byte of the pool and every other scale is what it was."""
    from swifttransformer_b200 import ops
    heads, page = 8, 64
    step = Step([(500, 40), (100, 1), (290, 7)], heads, heads, dim, form, act, page, seed=9, spare=20000)
    pool, scales, n = step.pool.view(torch.int8), step.scales, step.n
    assert pool.numel() > 2 ** 32
    at = torch.tensor([int(step.table[int(step.slots[r]), p // page]) for p, r in zip(step.pos_list, step.seq_list)], device="cuda")
    assert int(at.max()) * pool[0].numel() > 2 ** 32 and int(at.min()) * pool[0].numel() < 2 ** 32
    off = step.positions.long() % page
    rows = torch.full((n, 2 * heads * dim), 77.0, dtype=TYPES[act], device="cuda")
    ops.cache8_rows(step.pool, scales, step.layer, rows, step.positions, step.seq, step.slots, step.table, step.status)
    want = torch.stack([torch.stack([x[r][:, p] for x in (step.k, step.v)]) for p, r in zip(step.pos_list, step.seq_list)])
    assert torch.equal(rows, want.float().to(TYPES[act]).view(n, -1))
    gen = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn((n, 3 * heads * dim), generator=gen, device="cuda").to(TYPES[act])
    meant, meant_scales = pool.clone(), scales.clone()
    code, s = quantise(qkv[:, heads * dim:].float().view(n, 2, heads, dim), form)
    meant[at, step.layer, :, :, off] = code.float().to(TYPES[form]).view(torch.int8)
    meant_scales[at, step.layer, :, :, off] = s
    ops.qkv_to_cache8(qkv, None, None, step.pool, scales, step.layer, step.positions, step.seq, step.slots, step.table, heads, heads, dim, step.status)
    assert torch.equal(pool, meant) and torch.equal(scales.view(torch.int32), meant_scales.view(torch.int32))
    assert int(step.status) == 0
