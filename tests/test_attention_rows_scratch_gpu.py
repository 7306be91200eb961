"""What a call of portions takes beside its inputs and results."""
import pytest
import torch

from cache8_cases import Step, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,dim", [("bf16", 128), ("f32", 64)])
def test_workspace_of_a_long_prompt(act, dim):
    """It follows the device, not the prompt: two parts of 128 rows, (dim + 2) floats each, for two or three walkers on every SM (large
    blocks come in segments of whole 2 MB)."""
    from swifttransformer_b200 import ops
    n, heads = 30000 if act == "bf16" else 6000, 16
    pages = -(-n // 16)
    pool, scales = ops.cache8_pool(pages, 1, heads, 16, dim, torch.int8, "cuda")
    q = torch.zeros((n, heads * dim), dtype={"bf16": torch.bfloat16, "f32": torch.float32}[act], device="cuda")
    out = torch.empty_like(q)
    positions, slots = torch.arange(n, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(1, -1)
    plan = ops.portion_plan([n], [0], heads, heads)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.attention_cache8_tiles(q, pool, scales, 0, out, plan, positions, slots, table, heads, 0.1)
    torch.cuda.synchronize()
    most = torch.cuda.max_memory_allocated() - before
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert most <= 2 * (2 if dim == 128 else 3) * sms * 128 * (dim + 2) * 4 + (2 << 20), most
    assert float(out.abs().max()) == 0.0


@pytest.mark.parametrize("form,act,dim", [("int8", "bf16", 64), ("e4m3", "bf16", 128), ("int8", "f32", 64), ("e4m3", "f32", 130)])
def test_cuts_anywhere(form, act, dim):
    """Units of one chunk to many, so that walkers begin and end in the middle of units, at their ends, and several to a unit."""
    from swifttransformer_b200 import ops
    step = Step([(0, 5), (2500, 130), (64, 64), (0, 300), (900, 1), (63, 2)], 6, 3, dim, form, act, 16, seed=dim)
    for window in (0, 200):
        plan = ops.portion_plan([n for _, n in step.requests], [b for b, _ in step.requests], 6, 3, window, "cuda")
        got = ops.attention_cache8_tiles(step.q, step.pool, step.scales, step.layer, step.out(), plan, step.positions, step.slots, step.table, 6,
                                         step.scale, window, step.status)
        check(step, got, window=window)
    assert int(step.status) == 0
