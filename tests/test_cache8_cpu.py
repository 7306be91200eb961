"""Plans of the row attention, and what its operations refuse (no GPU)."""
import random

import pytest
import torch

from swifttransformer_b200 import ops
from swifttransformer_b200.ops import KernelError
from swifttransformer_b200.ops.cache8 import ROWS_CHUNK as CHUNK
from swifttransformer_b200.ops.cache8 import ROWS_PER_TILE
from swifttransformer_b200.ops.cache8 import ROWS_UNIT as UNIT


def walk(plan, ctas):
    """The pieces every block gets, as the kernels cut the line of chunks."""
    tiles = plan.tiles.view(-1, 6).tolist()
    run = -(-plan.total // ctas)
    bounds = [min(run * c, plan.total) for c in range(ctas + 1)]
    pieces = []
    for c in range(ctas):
        for x in range(bounds[c], bounds[c + 1]):
            t = max(i for i, r in enumerate(tiles) if r[5] <= x and chunks(r) > 0)
            head, place = divmod(x - tiles[t][5], chunks(tiles[t]) + UNIT)
            if place >= UNIT:                           # the first places stand for what a unit costs beside its chunks
                pieces.append((c, t, head, place - UNIT))
    return pieces


def chunks(tile):
    lo, hi = tile[3], tile[4]
    return -(-(hi - lo // CHUNK * CHUNK) // CHUNK) if hi > lo else 0


@pytest.mark.parametrize("seed", range(6))
def test_every_key_of_every_row_is_in_one_chunk(seed):
    rng = random.Random(seed)
    nkv = rng.choice([1, 2, 5])
    nh = nkv * rng.choice([1, 3, 4, 100])
    window = rng.choice([0, 0, 50, 300])
    lens = [rng.choice([0, 1, 2, 127, 128, 129, rng.randint(1, 600)]) for _ in range(rng.randint(1, 5))]
    starts = [rng.choice([0, 1, 128, rng.randint(0, 900)]) for _ in lens]
    plan = ops.portion_plan(lens, starts, nh, nkv, window, "cpu")
    tiles = plan.tiles.view(-1, 6).tolist() if plan.n_tiles else []
    assert plan.n_tokens == sum(lens) and plan.total == sum(chunks(t) + UNIT for t in tiles if chunks(t)) * nkv
    rows = []
    first = 0
    for seq, (n, s) in enumerate(zip(lens, starts)):
        for j in range(n):
            pos = s + j
            rows.append((first + j, seq, max(0, pos - window + 1) if window else 0, pos + 1))
        first += n
    seen = {r[0]: 0 for r in rows}
    for token, n, seq, lo, hi, _ in tiles:
        assert n * (nh // nkv) <= 128
        for t in range(token, token + n):
            row = rows[t]
            assert row[1] == seq and lo <= row[2] and row[3] <= hi
            seen[t] += 1
    assert all(v == 1 for v in seen.values())
    if plan.total:
        for ctas in (1, 2, 7, 148):
            got = walk(plan, min(ctas, plan.total))
            assert len(got) == len(set(p[1:] for p in got)) == sum(chunks(t) for t in tiles) * nkv


def test_the_plans_sizes_are_the_librarys():
    lib = ops.lib()
    assert (ROWS_PER_TILE, CHUNK, UNIT) == (lib.st_attention_rows_per_tile(), lib.st_attention_rows_chunk(), lib.st_attention_rows_unit())


def test_shared_plan():
    plan = ops.shared_prefix_plan([[5, 2, 9], [], [0], [7, 8]], [300, 10, 0, 128], 64, 1, "cpu", 17)
    assert plan.tokens_per_tile == 2 and plan.items.tolist() == [5, 2, 9, 0, 7, 8]
    assert plan.tiles.view(-1, 6).tolist() == [[0, 2, -1, 0, 300, 0], [2, 1, -1, 0, 300, 8], [3, 1, -1, 0, 0, 16], [4, 2, -1, 0, 128, 16]]
    assert plan.info.view(-1, 3).tolist() == [[300, 0, 0], [300, 0, 1], [300, 1, 0], [0, 2, 0], [128, 3, 0], [128, 3, 1]]
    assert plan.total == 21 and plan.n_items == 6 and plan.max_rows == 128 and plan.n_tokens == 10 and plan.max_own == 17


@pytest.mark.parametrize("make", [
    lambda: ops.portion_plan([1, 2], [0], 4, 4, device="cpu"),
    lambda: ops.portion_plan([-1], [0], 4, 4, device="cpu"),
    lambda: ops.portion_plan([1], [-1], 4, 4, device="cpu"),
    lambda: ops.portion_plan([1], [0], 4, 3, device="cpu"),
    lambda: ops.portion_plan([1], [0], 129, 1, device="cpu"),
    lambda: ops.portion_plan([1], [0], 4, 4, window=-1, device="cpu"),
    lambda: ops.portion_plan([1 << 24], [1 << 30], 64, 64, device="cpu"),
    lambda: ops.shared_prefix_plan([[1, 1]], [4], 4, 4, device="cpu"),
    lambda: ops.shared_prefix_plan([[1], [1]], [4, 5], 4, 4, device="cpu"),
    lambda: ops.shared_prefix_plan([[-1]], [4], 4, 4, device="cpu"),
    lambda: ops.shared_prefix_plan([[1]], [-4], 4, 4, device="cpu"),
    lambda: ops.shared_prefix_plan([[1]], [4, 4], 4, 4, device="cpu"),
    lambda: ops.cache8_pool(1, 1, 1, 16, 64, torch.bfloat16, "cpu"),
])
def test_plans_refuse(make):
    with pytest.raises(KernelError):
        make()


def test_an_empty_cache_reads_as_zeros():
    pool, scales = ops.cache8_pool(3, 2, 1, 16, 64, torch.float8_e4m3fn, "cpu")
    assert pool.shape == (3, 2, 2, 1, 16, 64) and scales.shape == (3, 2, 2, 1, 16)
    assert float(pool.float().abs().max()) == 0 and float(scales.max()) == 0


def test_cpu_tensors_are_refused():
    pool, scales = ops.cache8_pool(3, 2, 1, 16, 64, torch.int8, "cpu")
    i = torch.zeros(4, dtype=torch.int32)
    q = torch.zeros((4, 64))
    with pytest.raises(KernelError, match="CUDA"):
        ops.qkv_to_cache8(torch.zeros((4, 192)), None, q, pool, scales, 0, i, i, i, i.view(2, 2), 1, 1, 64)
    with pytest.raises(KernelError, match="CUDA"):
        ops.cache8_rows(pool, scales, 0, torch.zeros((4, 128)), i, i, i, i.view(2, 2))
    with pytest.raises(KernelError, match="CUDA"):
        ops.attention_cache8_single(q, pool, scales, 0, q, None, 4, i, i, i, i.view(2, 2), 1, 0.1)
    with pytest.raises(KernelError, match="CUDA"):
        ops.attention_cache8_tiles(q, pool, scales, 0, q, ops.portion_plan([4], [0], 1, 1, device="cpu"), i, i, i.view(2, 2), 1, 0.1)
    with pytest.raises(KernelError, match="CUDA"):
        ops.attention_shared_prefix(q, q, 0, q, ops.shared_prefix_plan([[0]], [1], 1, 1, device="cpu"), i, i, i, i.view(2, 2), 1, 0.1)


class Fake:
    """Stands for a CUDA tensor where only shapes and types are looked at."""

    def __init__(self, t, device=0):
        self.t, self.index = t, device

    is_cuda = True
    dtype = property(lambda self: self.t.dtype)
    shape = property(lambda self: self.t.shape)
    device = property(lambda self: torch.device("cuda", self.index))
    get_device = lambda self: self.index  # noqa: E731
    dim = lambda self: self.t.dim()  # noqa: E731
    is_contiguous = lambda self: self.t.is_contiguous()  # noqa: E731
    numel = lambda self: self.t.numel()  # noqa: E731
    stride = lambda self, i: self.t.stride(i)  # noqa: E731
    data_ptr = lambda self: self.t.data_ptr()  # noqa: E731


@pytest.fixture()
def fake(monkeypatch):
    from swifttransformer_b200.ops import cache8
    monkeypatch.setattr(cache8, "_current_device", lambda: 0)

    def reached(*a, **k):
        raise AssertionError("the call reached the library")

    class Lib:
        def __getattr__(self, name):
            return reached

    monkeypatch.setattr(cache8, "lib", Lib)
    return Fake


def base(fake, **over):
    pool, scales = ops.cache8_pool(3, 2, 2, 16, 64, torch.int8, "cpu")
    i = lambda *s: fake(torch.zeros(s, dtype=torch.int32))  # noqa: E731
    a = dict(q=fake(torch.zeros((4, 256))), pool=fake(pool), scales=fake(scales), layer=0, out=fake(torch.zeros((4, 256))), items=None, n_items=4,
             positions=i(4), seq_of_token=i(4), slots=i(2), block_table=i(2, 3), nh=4, scale=0.125, window=0, status=i(1))
    a.update(over)
    return a


@pytest.mark.parametrize("what,change", [
    ("type", lambda f: dict(q=f(torch.zeros((4, 256), dtype=torch.float16)))),
    ("types differ", lambda f: dict(out=f(torch.zeros((4, 256), dtype=torch.bfloat16)))),
    ("shape", lambda f: dict(q=f(torch.zeros((4, 128))))),
    ("rows", lambda f: dict(out=f(torch.zeros((3, 256))))),
    ("strided", lambda f: dict(q=f(torch.zeros((4, 512))[:, :256]))),
    ("columns apart", lambda f: dict(q=f(torch.zeros((4, 512))[:, ::2]))),
    ("scales missing", lambda f: dict(scales=None)),
    ("scales' shape", lambda f: dict(scales=f(torch.zeros((3, 2, 2, 2, 8))))),
    ("scales' type", lambda f: dict(scales=f(torch.zeros((3, 2, 2, 2, 16), dtype=torch.float64)))),
    ("pool's type", lambda f: dict(pool=f(torch.zeros((3, 2, 2, 2, 16, 64), dtype=torch.uint8)))),
    ("pool without scales", lambda f: dict(pool=f(torch.zeros((3, 2, 2, 2, 16, 64))))),
    ("pool strided", lambda f: dict(pool=f(torch.zeros((3, 2, 2, 2, 16, 128), dtype=torch.int8)[..., :64]))),
    ("layer", lambda f: dict(layer=2)),
    ("layer", lambda f: dict(layer=-1)),
    ("heads", lambda f: dict(nh=3)),
    ("positions' type", lambda f: dict(positions=f(torch.zeros(4, dtype=torch.int64)))),
    ("few positions", lambda f: dict(positions=f(torch.zeros(3, dtype=torch.int32)))),
    ("few requests", lambda f: dict(seq_of_token=f(torch.zeros(3, dtype=torch.int32)))),
    ("table", lambda f: dict(block_table=f(torch.zeros(6, dtype=torch.int32)))),
    ("slots", lambda f: dict(slots=f(torch.zeros((2, 2), dtype=torch.int32)[:, 0]))),
    ("items", lambda f: dict(n_items=5)),
    ("items", lambda f: dict(items=f(torch.zeros(3, dtype=torch.int32)))),
    ("items", lambda f: dict(items=f(torch.zeros(4, dtype=torch.int64)))),
    ("scale", lambda f: dict(scale=0.0)),
    ("scale", lambda f: dict(scale=float("nan"))),
    ("window", lambda f: dict(window=-1)),
    ("device", lambda f: dict(pool=f(ops.cache8_pool(3, 2, 2, 16, 64, torch.int8, "cpu")[0], 1))),
])
def test_single_tokens_refuse(fake, what, change):
    with pytest.raises(KernelError):
        ops.attention_cache8_single(**base(fake, **change(fake)))


def test_another_device_than_the_current_one(fake, monkeypatch):
    from swifttransformer_b200.ops import cache8
    monkeypatch.setattr(cache8, "_current_device", lambda: 1)
    with pytest.raises(KernelError, match="current device"):
        ops.attention_cache8_single(**base(fake))


@pytest.mark.parametrize("kind", ["heads", "tokens", "requests", "window", "kind", "strided"])
def test_portions_refuse(fake, kind):
    a = base(fake)
    for name in ("items", "n_items", "seq_of_token"):
        a.pop(name)
    plan = ops.portion_plan([2, 2], [0, 0], 4, 2, device="cpu")
    if kind == "heads":
        plan = ops.portion_plan([2, 2], [0, 0], 4, 4, device="cpu")
    if kind == "tokens":
        plan = ops.portion_plan([2, 3], [0, 0], 4, 2, device="cpu")
    if kind == "requests":
        plan = ops.portion_plan([2, 1, 1], [0, 0, 0], 4, 2, device="cpu")
    if kind == "window":
        a["window"] = 7
    if kind == "kind":
        plan = ops.shared_prefix_plan([[0]], [4], 4, 2, device="cpu")
    if kind == "strided":
        a["q"] = fake(torch.zeros(1024).as_strided((4, 256), (200, 1)))
    plan.tiles = fake(plan.tiles)
    with pytest.raises(KernelError):
        ops.attention_cache8_tiles(**a, plan=plan)


@pytest.mark.parametrize("kind", ["heads", "tokens", "kind", "type", "scales", "strided"])
def test_shared_prefixes_refuse(fake, kind):
    a = base(fake)
    a.pop("items"), a.pop("n_items")
    plan = ops.shared_prefix_plan([[0, 1, 2, 3]], [4], 4, 2, device="cpu")
    if kind == "heads":
        plan = ops.shared_prefix_plan([[0, 1, 2, 3]], [4], 2, 2, device="cpu")
    if kind == "tokens":
        plan = ops.shared_prefix_plan([[0, 4]], [4], 4, 2, device="cpu")
    if kind == "kind":
        plan = ops.portion_plan([2, 2], [0, 0], 4, 2, device="cpu")
    if kind == "type":
        a.update(pool=fake(torch.zeros((3, 2, 2, 2, 16, 64), dtype=torch.bfloat16)), scales=None)
    if kind == "scales":
        a.update(pool=fake(torch.zeros((3, 2, 2, 2, 16, 64))))
    if kind == "strided":
        a["q"] = fake(torch.zeros((4, 512))[:, :256])
    plan.tiles = fake(plan.tiles)
    with pytest.raises(KernelError):
        ops.attention_shared_prefix(**a, plan=plan)


@pytest.mark.parametrize("change", [
    lambda f: dict(qkv=f(torch.zeros((4, 511)))), lambda f: dict(qkv=f(torch.zeros((4, 512), dtype=torch.float16))),
    lambda f: dict(qkv=f(torch.zeros((4, 1024))[:, :512])), lambda f: dict(bias=f(torch.zeros(512, dtype=torch.bfloat16))),
    lambda f: dict(bias=f(torch.zeros(511))), lambda f: dict(q_out=f(torch.zeros((4, 255)))),
    lambda f: dict(q_out=f(torch.zeros((4, 256), dtype=torch.bfloat16))), lambda f: dict(d=32), lambda f: dict(nkv=1),
    lambda f: dict(positions=f(torch.zeros(3, dtype=torch.int32))), lambda f: dict(scales=None), lambda f: dict(layer=7),
    lambda f: dict(pool=f(torch.zeros((3, 2, 2, 2, 16, 64))), scales=None),
])
def test_the_write_refuses(fake, change):
    a = base(fake)
    w = dict(qkv=fake(torch.zeros((4, 512))), bias=None, q_out=fake(torch.zeros((4, 256))), nkv=2, d=64,
             **{k: a[k] for k in ("pool", "scales", "layer", "positions", "seq_of_token", "slots", "block_table", "nh", "status")})
    w.update(change(fake))
    with pytest.raises(KernelError):
        ops.qkv_to_cache8(**w)
