"""The 4-bit K/V cache and rotated appends on the GPU: codes, scales and rows
against plain restatements, bit for bit; the attention over it against the
formula in 64 bits."""
import math

import numpy as np
import pytest
import torch

from oracle import kv_reference as ref
from test_gpu_paged_attention import Served

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def make_rows(rng, n, heads, dim, dtype):
    """Rows whose groups of 32 differ by 2^12, some of them on the borders between codes."""
    x = rng.standard_normal((n, heads, dim // 32, 32)) * np.exp2(rng.uniform(-6, 6, (n, heads, dim // 32, 1)))
    x[::3, :, 0] = rng.choice([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, -0.25, -2.5, -5], (len(x[::3]), heads, 32))
    return torch.from_numpy(x.reshape(n, heads, dim)).to(dtype)


def same(got, want):
    return torch.equal(torch.nan_to_num(got.double(), nan=1e30), torch.nan_to_num(want.double(), nan=1e30))


def table_of(rotary, positions):
    rows = rotary.table.cpu()[torch.as_tensor(positions)]
    return rows[..., 0], rows[..., 1]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,dim,block", [(1, 64, 16), (3, 128, 16), (2, 128, 32), (2, 64, 64), (5, 64, 32), (1, 128, 64)])
def test_append_and_read_exact(gpu, dtype, heads, dim, block):
    """Prompts, single tokens, idle slots, in any order: values bit for bit, what stands next to them as it was."""
    from next_step_ai_amd.kv_cache import KvCache

    rng = np.random.RandomState(heads * 100 + dim + block)
    blocks = 7
    cache, plain = KvCache(blocks, heads, dim, block_tokens=block, fmt="e2m1"), ref.PlainCache(blocks, heads, dim, block, "e2m1")
    every = list(range(blocks * block))
    free = list(rng.permutation(every))
    for n in (1, 2, 37, 3, 64, 5):
        slots = [int(free.pop()) for _ in range(min(n, len(free)))]
        slots[n // 2: n // 2] = [-1, blocks * block]
        k, v = (make_rows(rng, len(slots), heads, dim, dtype) for _ in range(2))
        cache.append(k.to(gpu), v.to(gpu), torch.tensor(slots, device=gpu))
        stored = [s if s < blocks * block else -1 for s in slots]
        plain.append(k.float().numpy(), v.float().numpy(), stored)
        for out in DTYPES:
            got = cache.read(torch.tensor(every + [-1, blocks * block], device=gpu), out)
            for which, name in ((0, "k"), (1, "v")):
                want = torch.from_numpy(plain.values(every + [-1, -1], which))
                assert torch.equal(got[name].cpu().float(), want) and got[name].dtype == out


def test_every_value(gpu):
    """All finite fp16 and bf16 values as a group's largest, next to halves of the least step."""
    from next_step_ai_amd.kv_cache import KvCache

    for dtype in DTYPES:
        bits = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16)
        top = bits.view(dtype)
        top = top[top.isfinite()]
        n = top.numel() // 64 * 64
        x = torch.zeros(n // 64, 1, 64, 32, dtype=torch.float64)
        x[:, 0] = top[:n].double().view(-1, 64, 1) * torch.linspace(-1, 1, 32, dtype=torch.float64)
        x[:, 0, :, 0] = top[:n].double().view(-1, 64)
        rows = x.to(dtype).view(n // 2, 1, 64)
        cache = KvCache(n // 2 // 64 + 1, 1, 64, block_tokens=64, fmt="e2m1")
        slots = torch.arange(n // 2, device=gpu)
        cache.append(rows.to(gpu), rows.to(gpu), slots)
        codes, scale = ref.encode4(rows.float().numpy())
        want = torch.from_numpy(codes * np.repeat(scale, 32, -1))
        got = cache.read(slots, dtype)
        assert torch.equal(got["k"].cpu().float(), want) and torch.equal(got["v"].cpu().float(), want)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(gpu, dim, value):
    """A token's head whose K or V holds one reads as NaN, K and V, until it is written again; nothing else does."""
    from next_step_ai_amd.kv_cache import KvCache

    cache = KvCache(2, 2, dim, fmt="e2m1")
    x = torch.randn(20, 2, dim, device=gpu).half()
    slots = torch.arange(20, device=gpu)
    k, v = x.clone(), x.clone()
    k[3, 1, dim - 1], v[4, 0, 5] = value, value
    cache.append(k, v, slots)
    got = cache.read(slots)
    bad = torch.zeros(20, 2, dtype=torch.bool, device=gpu)
    bad[3, 1] = bad[4, 0] = True
    for name in ("k", "v"):
        assert torch.equal(got[name].isnan().all(-1), bad) and torch.equal(got[name].isnan().any(-1), bad)
        assert cache.read(slots, torch.bfloat16)[name].isnan().any(-1).equal(bad)
    cache.append(x[3:5], x[3:5], slots[3:5])
    again = cache.read(slots)
    cache.append(x, x, slots)
    clean = cache.read(slots)
    assert all(torch.equal(again[name], clean[name]) for name in ("k", "v"))


@pytest.mark.parametrize("fmt", ["e2m1", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Hq,H,dim,block", [(1, 1, 64, 16), (6, 2, 128, 16), (12, 3, 128, 32), (9, 3, 64, 64), (5, 5, 64, 32),
                                            (7, 1, 128, 64)])
def test_rotated_append_exact(gpu, fmt, dtype, interleaved, Hq, H, dim, block):
    """Stored values and query rows are those of rows rotated beforehand, bit for bit, over several steps and idle slots."""
    from next_step_ai_amd.kv_cache import KvCache
    from next_step_ai_amd.rotary import Rotary

    rng = np.random.RandomState(Hq + dim + block)
    rotary = Rotary(dim, 5000, base=500000.0, interleaved=interleaved)
    blocks = 9
    cache, plain = (make(blocks, H, dim, **kw) for make, kw in ((KvCache, dict(block_tokens=block, fmt=fmt)),
                                                                (ref.PlainCache, dict(block=block, fmt=fmt))))
    at, start = [0, 0, 0], [0, 4000, 37]
    for new in ([block + 3, 1, 0], [1, 1, 2 * block], [2, block - 3, 1], [1, 1, 1], [1, 0, 0]):
        slots, pos = [], []
        for r, n in enumerate(new):
            slots += [(3 * r + p // block) * block + p % block for p in range(at[r], at[r] + n)] + [-1]
            pos += [start[r] + p for p in range(at[r], at[r] + n)] + [-1]
            at[r] += n
        n = len(slots)
        k, v, q = (make_rows(rng, n, heads, dim, dtype) for heads in (H, H, Hq))
        k_dev = k.to(gpu)
        out = torch.full((n, Hq, dim), 7.0, dtype=dtype, device=gpu)
        got = cache.append_rotated(k_dev, v.to(gpu), torch.tensor(slots, device=gpu),
                                   torch.tensor(pos, dtype=torch.int32, device=gpu), rotary, q=q.to(gpu), q_out=out)
        assert got is out and torch.equal(k_dev.cpu(), k)
        cos, sin = table_of(rotary, [max(p, 0) for p in pos])
        want_q = ref.rotate(q, cos, sin, interleaved)
        want_q[torch.tensor(pos) < 0] = 7.0
        assert torch.equal(got.cpu(), want_q)
        plain.append(ref.rotate(k, cos, sin, interleaved).float().numpy(), v.float().numpy(), slots)
        every = [s for r in range(3) for s in range(3 * r * block, 3 * r * block + at[r])]
        data = cache.read(torch.tensor(every, device=gpu), dtype)
        for which, name in ((0, "k"), (1, "v")):
            assert torch.equal(data[name].cpu(), torch.from_numpy(plain.values(every, which)).to(dtype))


@pytest.mark.parametrize("fmt", ["e2m1", "int8", "e4m3"])
def test_rotated_append_in_place_and_strides(gpu, fmt):
    """Slices of one projection, the queries turned where they lie; a table that ends before a position."""
    from next_step_ai_amd.kv_cache import KvCache
    from next_step_ai_amd.rotary import Rotary

    n, Hq, H, dim = 21, 6, 2, 128
    rotary = Rotary(dim, 30)
    both = torch.randn(n, (Hq + 2 * H) * dim, device=gpu).bfloat16()
    q, k, v = (t.view(n, -1, dim) for t in both.split([Hq * dim, H * dim, H * dim], 1))
    before = both.clone()
    slots, pos = torch.arange(n, device=gpu), torch.arange(10, 10 + n, dtype=torch.int32, device=gpu)
    cache, other = KvCache(2, H, dim, fmt=fmt), KvCache(2, H, dim, fmt=fmt)
    pos[-1], pos[4] = 30, -1  # past the table; of no request, but with a slot
    got = cache.append_rotated(k, v, slots, pos, rotary, q=q, q_out=q)
    assert got is q
    cos, sin = table_of(rotary, pos.cpu().clamp(0, 29).long())
    want = ref.rotate(before[:, : Hq * dim].view(n, Hq, dim).cpu(), cos, sin, False)
    want[-1] = math.nan
    want[4] = before[4, : Hq * dim].view(Hq, dim).cpu()
    assert same(q.cpu(), want) and torch.equal(both[:, Hq * dim:], before[:, Hq * dim:])
    k2 = ref.rotate(before[:, Hq * dim: (Hq + H) * dim].view(n, H, dim).cpu(), cos, sin, False)
    k2[-1] = k2[4] = math.nan
    other.append(k2.to(gpu), v, slots)
    assert torch.equal(cache.data, other.data)
    if fmt != "e2m1":
        assert same(cache.scale, other.scale)
    # no queries; queries whose memory the kernels cannot read in pieces of 16 bytes
    again = KvCache(2, H, dim, fmt=fmt)
    assert again.append_rotated(k, v, slots, pos, rotary) is None
    assert torch.equal(again.data, cache.data)
    odd = torch.zeros(n, Hq, dim + 1, dtype=torch.bfloat16, device=gpu)[:, :, 1:]
    odd.copy_(before[:, : Hq * dim].view(n, Hq, dim))
    new = again.append_rotated(k, v, slots, pos, rotary, q=odd)
    keep = torch.arange(n) != 4  # (a new tensor holds anything there)
    assert same(new.cpu()[keep], want[keep])
    # pieces of a wider buffer: nothing around them is written
    wide = torch.full((n, Hq + 2, dim + 8), 3.0, dtype=torch.bfloat16, device=gpu)
    again.append_rotated(k, v, slots, pos, rotary, q=odd, q_out=wide[:, 1:-1, 8:])
    assert same(wide[:, 1:-1, 8:].cpu()[keep], want[keep]) and (wide[4] == 3).all()
    assert (wide[:, [0, -1]] == 3).all() and (wide[:, :, :8] == 3).all()


def test_rotation_error_in_64_bits(gpu):
    """Far positions: an angle is off by no more than its cos and sin's rounding to fp32."""
    from next_step_ai_amd.kv_cache import KvCache
    from next_step_ai_amd.rotary import Rotary, rotary_frequencies

    dim, reach = 128, 300000
    rotary = Rotary(dim, reach, base=500000.0)
    f = rotary_frequencies(dim, 500000.0)
    pos = torch.tensor([0, 1, 2, 8191, 131071, 262143, 262144, reach - 1], dtype=torch.int32, device=gpu)
    n = pos.numel()
    q = torch.randn(n, 3, dim, device=gpu).half()
    k = torch.zeros(n, 1, dim, dtype=torch.float16, device=gpu)
    got = KvCache(1, 1, dim, fmt="e2m1").append_rotated(k, k, torch.full((n,), -1, device=gpu), pos, rotary, q=q).cpu().double()
    turn = torch.polar(torch.ones(n, dim // 2, dtype=torch.float64), pos.cpu().double()[:, None] * f)
    z = torch.complex(*q.cpu().double().split(dim // 2, -1)) * turn[:, None]
    want = torch.cat([z.real, z.imag], -1)
    size = q.cpu().double().abs()
    both = size + size.roll(dim // 2, -1)
    # rounding to fp32 and fp16, cos and sin's (2^-25 each where they are near 1), an angle's in 64 bits (2^18 times 2^-53, twice)
    assert ((got - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -24) + both * (2.0 ** -24 + 2.0 ** -33) + 2.0 ** -25).all()


def test_positions_of_a_plan(gpu):
    """Positions count a request's stored tokens; -1 where a token has no slot."""
    from next_step_ai_amd.kv_cache import KvBatch

    batch = KvBatch(100, 16, max_requests=4, max_blocks=3, q_heads=4, kv_heads=4)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    step = batch.plan(ints([5, 0, 17, 49]), 75)
    assert step.positions.tolist() == [*range(5), *range(17), *[-1] * 49, *[-1] * 4] and step.positions.dtype == torch.int32
    batch.commit()
    again = batch.plan(ints([1, 2, 16, 0]), 19)
    assert again.positions.tolist() == [5, 0, 1, *range(17, 33)]
    assert batch.plan(ints([3, 0, 1, 2]), 6, step=None).positions.tolist() == [5, 6, 7, 17, 0, 1]
    assert batch.plan(ints([0] * 4), 0).positions.numel() == 0


def test_positions_are_a_view_of_their_own(gpu):
    """Looking at a step's other outputs makes no view for them, as steps without a rotation have no use for one."""
    from next_step_ai_amd.kv_cache import KvBatch

    batch = KvBatch(10, 16, max_requests=2, max_blocks=3, q_heads=4, kv_heads=4)
    step = batch.plan(torch.tensor([3, 4], dtype=torch.int32, device=gpu), 7)
    assert step.q_start.tolist() == [0, 3, 7] and step.kv_len.tolist() == [3, 4] and step.info.tolist()[2:] == [0, 7]
    assert len(step._split) == 5 and step._positions is None
    assert step.positions is step.positions and step.positions.tolist() == [0, 1, 2, 0, 1, 2, 3]
    assert step.positions.data_ptr() == step._view.positions


def test_refusals(gpu):
    from next_step_ai_amd.kv_cache import KvCache
    from next_step_ai_amd.rotary import Rotary

    c, rotary = KvCache(4, 2, 64, fmt="e2m1"), Rotary(64, 10)
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device=gpu)
    s, p = torch.arange(3, device=gpu), torch.arange(3, dtype=torch.int32, device=gpu)
    for args, kw in (((x, x, s, p.long(), rotary), {}), ((x, x, s, p[:2], rotary), {}), ((x, x, s, p.cpu(), rotary), {}),
                     ((x, x, s, p, Rotary(128, 10)), {}), ((x, x.bfloat16(), s, p, rotary), {}), ((x, x, s.int(), p, rotary), {}),
                     ((x, x, s, p, rotary), dict(q=x.float())), ((x, x, s, p, rotary), dict(q=x.bfloat16())),
                     ((x, x, s, p, rotary), dict(q=x[:2])), ((x, x, s, p, rotary), dict(q=x[:, :, :32])),
                     ((x, x, s, p, rotary), dict(q=x[:, 0])), ((x, x, s, p, rotary), dict(q=x[:, :0])),
                     ((x, x, s, p, rotary), dict(q_out=x)),
                     ((x, x, s, p, rotary), dict(q=x, q_out=x[:, :1])), ((x, x, s, p, rotary), dict(q=x, q_out=x.bfloat16())),
                     ((x, x, s, p, rotary), dict(q=x, q_out=x.transpose(0, 2).contiguous().transpose(0, 2))),
                     ((x, x, s, p, rotary), dict(q=x, q_out=x[:1].expand(3, 2, 64)))):
        with pytest.raises(RuntimeError):
            c.append_rotated(*args, **kw)
    long = torch.zeros(5, 2, 64, dtype=torch.float16, device=gpu)
    with pytest.raises(RuntimeError, match="overlaps"):
        c.append_rotated(x, x, s, p, rotary, q=long[:3], q_out=long[1:4])
    assert c.append_rotated(x[:0], x[:0], s[:0], p[:0], rotary, q=x[:0]).shape == (0, 2, 64)


# ------------------------------------------------------------- attention --
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,H,D,block", [(4, 4, 64, 16), (16, 1, 128, 16), (14, 2, 128, 32), (6, 2, 64, 64), (40, 2, 128, 16)])
def test_decode(gpu, dtype, Hq, H, D, block):
    """One token each at lengths around a tile, a block and a workgroup's share, the first token of a request among them."""
    lengths = [(0, 1), (1, 1), (14, 1), (15, 1), (16, 1), (0, 0), (31, 1), (32, 1), (63, 1), (64, 1), (127, 1), (130, 1), (400, 1),
               (1000, 1)]
    s = Served(gpu, lengths, Hq, H, D, block, "e2m1", dtype, seed=Hq + D)
    s.check(*s.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,H,D,block,lengths", [
    (4, 1, 128, 16, [(0, 5), (7, 4), (100, 2), (33, 1)]),
    (6, 2, 64, 32, [(50, 7), (0, 1), (0, 40), (129, 3), (1, 0)]),
    (16, 1, 128, 16, [(20, 37), (300, 1), (0, 65)]),
    (2, 2, 128, 64, [(0, 130), (257, 65)]),
    (3, 1, 64, 16, [(5, 200)]),
])
def test_several_tokens(gpu, dtype, Hq, H, D, block, lengths):
    """Drafts, prompts and chunks next to single tokens: every row's own end."""
    s = Served(gpu, lengths, Hq, H, D, block, "e2m1", dtype, seed=len(lengths))
    s.check(*s.run())


@pytest.mark.parametrize("D,block", [(128, 16), (64, 32)])
def test_keys_shared_out(gpu, D, block):
    """Few rows and many keys: partial results joined, more than 64 blocks per wave, in both lists."""
    s = Served(gpu, [(9001, 1)], 4, 1, D, block, "e2m1", torch.float16, seed=9)
    s.check(*s.run())
    s = Served(gpu, [(9001, 7), (300, 40)], 4, 1, D, block, "e2m1", torch.bfloat16, seed=10)
    s.check(*s.run())
