"""The paged 8-bit K/V cache on the GPU: plan, commit, append and read against
plain restatements, exactly."""
import numpy as np
import pytest
import torch

from oracle import kv_reference as ref

pytestmark = pytest.mark.gpu


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def check_plan(batch, plain, step, want, new, total):
    assert step.slots.tolist() == want["slots"]
    assert step.kv_len.tolist() == want["kv_len"]
    assert step.q_start.tolist() == want["q_start"]
    head, free, refused, tokens = step.info.tolist()
    assert (free, refused, tokens) == (want["free"], want["refused"], sum(new))
    table = step.table.cpu()
    for r, blocks in enumerate(want["blocks"]):
        assert table[r, : len(blocks)].tolist() == blocks


@pytest.mark.parametrize("requests,block,steps,seed", [(1, 16, 6, 1), (5, 32, 8, 2), (70, 16, 5, 3), (1100, 64, 3, 4)])
def test_plan_and_commit_over_steps(gpu, requests, block, steps, seed):
    """Random steps with waiting requests, prompts, ends of requests; the ring
    runs dry now and then, so that some requests are refused."""
    from next_step_ai_amd.kv_cache import KvBatch

    rng = np.random.RandomState(seed)
    pool, width = 3 * requests + 4, 9
    order = rng.permutation(pool)
    batch = KvBatch(pool, block, max_requests=requests, max_blocks=width, q_heads=8, kv_heads=2,
                    free_blocks=torch.from_numpy(order))
    plain = ref.PlainBatch(pool, block, requests, width, order)
    refusals = 0
    for _ in range(steps):
        new = [int(rng.choice([0, 1, 1, 1, block - 1, block, 2 * block + 3, 5 * block])) for _ in range(requests)]
        if sum(new) == 0:
            new[0] = 1
        total = sum(new)
        want = plain.plan(new, total)
        for _ in range(2):  # a plan that is not committed can be made again
            step = batch.plan(ints(new, gpu), total, max_new=max(new))
        check_plan(batch, plain, step, want, new, total)
        refusals += want["refused"]
        ended = [r for r in range(requests) if rng.rand() < 0.3]
        flags = [0] * requests
        for r in ended:
            flags[r] = 1
        plain.commit(ended)
        batch.commit(ints(flags, gpu))
        assert batch.cached.tolist() == plain.cached
        head, free = batch.state.tolist()
        ring = batch.ring.tolist()
        assert [ring[(head + i) % pool] for i in range(free)] == plain.free
    assert requests < 5 or refusals > 0


def test_plan_limits(gpu):
    """Requests longer than the table or than max_new are refused, others are
    not touched by it; tokens past the sum have no slot; zero-length steps."""
    from next_step_ai_amd.kv_cache import KvBatch

    batch = KvBatch(100, 16, max_requests=4, max_blocks=3, q_heads=4, kv_heads=4)
    plain = ref.PlainBatch(100, 16, 4, 3)
    for new, total, most in (([48, 49, 0, 1], 98, 0), ([1, 5, 40, 2], 48, 39), ([0, 0, 0, 0], 5, 0), ([0, 3, 0, 0], 9, 0)):
        want = plain.plan(new, total, most)
        check_plan(batch, plain, batch.plan(ints(new, gpu), total, max_new=most), want, new, total)
        plain.commit()
        batch.commit()
        assert batch.cached.tolist() == plain.cached
    step = batch.plan(ints([0, 3, 0, 0], gpu), 9)
    with pytest.raises(RuntimeError, match="planned for 9 tokens"):
        step.check()
    step = batch.plan(ints([0, 100, 0, 0], gpu), 100)
    with pytest.raises(RuntimeError, match="1 requests were refused"):
        step.check()
    assert batch.plan(ints([0] * 4, gpu), 0).slots.numel() == 0


def make_rows(rng, n, heads, dim, dtype, grow):
    x = rng.standard_normal((n, heads, dim)) * np.exp2(rng.uniform(-3, 3, (n if grow else 1, heads, 1)))
    return torch.from_numpy(x).to(dtype)


def stored(cache, slots, dtype=torch.bfloat16):
    got = cache.read(torch.tensor(slots, dtype=torch.int64, device=cache.device), dtype)
    return got["k"].cpu(), got["v"].cpu()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,dim,block", [(1, 64, 16), (3, 128, 16), (2, 128, 32), (2, 64, 64)])
def test_append_and_read_exact(gpu, fmt, dtype, heads, dim, block):
    """Prompts, single tokens that raise the scale, idle slots: scales and
    values bit for bit, recoded tokens among them."""
    from next_step_ai_amd.kv_cache import KvCache

    rng = np.random.RandomState(heads * 100 + dim + block)
    blocks = 12
    cache = KvCache(blocks, heads, dim, block_tokens=block, fmt=fmt)
    plain = ref.PlainCache(blocks, heads, dim, block, fmt)
    place = rng.permutation(blocks)
    lengths = [0, 0, 0]
    own = [place[0:4], place[4:8], place[8:12]]
    seen = []
    for new in ([block + 3, 1, 0], [1, 1, 2 * block], [2, block - 3, 1], [5, 1, 1], [1, 1, 1]):
        slots = []
        for r, n in enumerate(new):
            slots += [int(own[r][p // block]) * block + p % block for p in range(lengths[r], lengths[r] + n)] + [-1]
            lengths[r] += n
        seen += [s for s in slots if s >= 0]
        k, v = (make_rows(rng, len(slots), heads, dim, dtype, True) for _ in range(2))
        cache.append(k.to(gpu), v.to(gpu), torch.tensor(slots, dtype=torch.int64, device=gpu))
        plain.append(k.float().numpy(), v.float().numpy(), slots)
        assert np.array_equal(cache.scale.cpu().numpy(), plain.scale)
        for out in (torch.float16, torch.bfloat16):
            got = stored(cache, seen, out)
            for which in (0, 1):
                want = torch.from_numpy(plain.values(seen, which)).to(out)
                assert torch.equal(got[which], want)
    assert (stored(cache, [-1, seen[0], blocks * block])[0][[0, 2]] == 0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_error_in_64_bits(gpu, fmt):
    """A block written in one call: every value within half a step of its own
    (int8: scale / 2; e4m3: 2^-4 of the value, 2^-10 scale below the normals)."""
    from next_step_ai_amd.kv_cache import KvCache

    rng = np.random.RandomState(5)
    cache = KvCache(4, 2, 128, fmt=fmt)
    x = make_rows(rng, 64, 2, 128, torch.float16, True)
    slots = torch.arange(64, device=gpu)
    cache.append(x.to(gpu), (x * 2).to(gpu), slots)
    data = cache.read(slots, torch.float16)
    for which, (name, src) in enumerate((("k", x), ("v", x * 2))):
        s = cache.scale.cpu().double()[:, :, which].repeat_interleave(16, 0)[:, :, None]
        y, z = src.double(), data[name].cpu().double()
        step = s / 2 if fmt == "int8" else torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10)
        # read's own rounding to fp16 (2^-11) and the division's in fp32 (2^-23 of a step's position) come on top
        assert ((y - z).abs() <= step * (1 + 2.0 ** -15) + z.abs() * 2.0 ** -11 + 2.0 ** -25).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_strides_zeros_and_values_that_are_not_finite(gpu, fmt):
    from next_step_ai_amd.kv_cache import KvCache

    rng = np.random.RandomState(6)
    cache, same = KvCache(4, 2, 64, fmt=fmt), KvCache(4, 2, 64, fmt=fmt)
    slots = torch.arange(20, device=gpu)
    both = make_rows(rng, 20, 6, 64, torch.bfloat16, False).to(gpu)
    k, v = both[:, 1:3], both[:, 3:5]  # a fused projection's slices
    cache.append(k, v, slots)
    same.append(k.contiguous(), v.contiguous(), slots)
    assert torch.equal(cache.data, same.data) and torch.equal(cache.scale, same.scale)
    odd = torch.zeros(20, 2, 65, dtype=torch.bfloat16, device=gpu)[:, :, 1:]
    odd.copy_(k)
    same.append(odd, v, slots)
    assert torch.equal(cache.data, same.data)
    # zeros: the smallest scale; a block started anew forgets its old one
    zero = torch.zeros(16, 2, 64, dtype=torch.bfloat16, device=gpu)
    cache.append(zero, zero, slots[:16])
    assert (cache.scale[0] == 2.0 ** -100).all() and (cache.read(slots[:16])["k"] == 0).all()
    # one infinite and one NaN value: their (block, head) alone, until it is started anew
    bad = k[:2].clone()
    bad[0, 0, 5], bad[1, 1, 7] = float("inf"), float("nan")
    cache.append(bad, v[:2], torch.tensor([32, 48], device=gpu))
    assert cache.scale[2, 0, 0].isnan() and cache.scale[3, 1, 0].isnan()
    assert not cache.scale[2, 1].isnan().any() and not cache.scale[2, 0, 1].isnan()
    cache.append(k[:1], v[:1], torch.tensor([33], device=gpu))
    assert cache.scale[2, 0, 0].isnan()
    cache.append(k[:1], v[:1], torch.tensor([32], device=gpu))
    assert not cache.scale.isnan()[2].any()


def test_refusals(gpu):
    from next_step_ai_amd.kv_cache import KvBatch, KvCache

    for bad in (dict(fmt="int4"), dict(block_tokens=24), dict(block_tokens=128)):
        with pytest.raises(RuntimeError):
            KvCache(4, 2, 128, **bad)
    for shape in ((0, 2, 128), (4, 0, 128), (4, 2, 96)):
        with pytest.raises(RuntimeError):
            KvCache(*shape)
    c = KvCache(4, 2, 64)
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device=gpu)
    s = torch.arange(3, device=gpu)
    for args in ((x.float(), x, s), (x, x.bfloat16(), s), (x[:2], x, s), (x, x, s.int()), (x, x, s[:2]), (x[:, :1], x, s),
                 (x.cpu(), x, s), (x, x, s.cpu())):
        with pytest.raises(RuntimeError):
            c.append(*args)
    with pytest.raises(RuntimeError, match="dtype"):
        c.read(s, torch.float32)
    c.append(x[:0], x[:0], s[:0])
    assert c.read(s[:0])["k"].shape == (0, 2, 64)
    kw = dict(max_requests=2, max_blocks=4, q_heads=4, kv_heads=2)
    for bad in (dict(q_heads=0), dict(max_requests=4097), dict(max_requests=0), dict(max_blocks=0)):
        with pytest.raises(RuntimeError):
            KvBatch(8, 16, **{**kw, **bad})
    with pytest.raises(RuntimeError):
        KvBatch(8, 24, **kw)
    b = KvBatch(8, 16, **kw)
    for new in (torch.zeros(3, dtype=torch.int32, device=gpu), torch.zeros(2, device=gpu, dtype=torch.int64),
                torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="new_tokens"):
            b.plan(new, 1)
    with pytest.raises(RuntimeError, match="total"):
        b.plan(torch.zeros(2, dtype=torch.int32, device=gpu), -1)
    with pytest.raises(RuntimeError, match="finished"):
        b.commit(torch.zeros(2, device=gpu))
