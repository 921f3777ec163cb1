"""The 4-bit cache's attention, rotated appends and log probabilities where they can go wrong: rows that see nothing,
tokens that are not finite, bad tables, far offsets, many short requests, other streams, captured steps, a run of them
together."""
import math

import numpy as np
import pytest
import torch

from oracle import kv_reference as ref
from test_gpu_kv_edges import rows_against_formula
from test_gpu_paged_attention import Served

pytestmark = pytest.mark.gpu


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def formula(q, k, v, cached):
    """One request's rows in 64 bits: q [n, Hq, D], k and v [cached + n, H, D] -> out, and sum_j p_j |v_j|."""
    n, G = q.shape[0], q.shape[1] // k.shape[1]
    k, v = (t.double().repeat_interleave(G, 1).transpose(0, 1).contiguous() for t in (k, v))  # [Hq, keys, D]
    s = torch.matmul(q.double().transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) * q.shape[-1] ** -0.5
    hidden = torch.arange(k.shape[1], device=q.device)[None] > cached + torch.arange(n, device=q.device)[:, None]
    p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
    return torch.matmul(p, v).transpose(0, 1), torch.matmul(p, v.abs()).transpose(0, 1)


def within(out, want, spread, keys):
    """The output's rounding, the weights' to fp16 (2^-11 each at most, and 2^-25 of the largest where one is subnormal),
    fp32 scores (2^-15)."""
    u = 2.0 ** -11 if out.dtype == torch.float16 else 2.0 ** -8
    bound = u * want.abs() + (2.0 ** -11 + 2.0 ** -15) * spread + keys * 2.0 ** -25 * 64 + 2.0 ** -24
    return ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("D,new,most", [(128, 1, 1), (64, 3, 3), (128, 20, 20), (64, 40, 0)])
def test_rows_that_see_nothing(gpu, D, new, most):
    """A refused request's tokens get zeros and -inf; rows past the step's tokens are left alone."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    b = KvBatch(8, 16, max_requests=3, max_blocks=4, q_heads=4, kv_heads=2, head_dim=D)
    c = KvCache(8, 2, D, fmt="e2m1")
    total = 2 * new + 70 + 5
    st = b.plan(ints([new, 70, new], gpu), total, max_new=0 if most == 0 else max(most, 70))
    k = torch.randn(total, 2, D, device=gpu).half()
    c.append(k, k, st.slots)
    q = torch.randn(total, 4, D, device=gpu).half()
    out, lse = torch.full_like(q, 7.0), torch.full((total, 4), 7.0, device=gpu)
    paged_attention(q, c, st, out=out, lse=lse)
    assert (out[new: new + 70] == 0).all() and (lse[new: new + 70] == -math.inf).all()
    assert (out[-5:] == 7).all() and (lse[-5:] == 7).all()
    got = c.read(st.slots)
    for t0 in (0, new + 70):
        rows = slice(t0, t0 + new)
        assert within(out[rows], *formula(q[rows], got["k"][rows], got["v"][rows], 0), new)
        assert lse[rows].isfinite().all()


@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("Hq,H,D,block,cached,new,bad", [
    (4, 2, 128, 16, 70, 1, 33), (4, 2, 64, 32, 0, 9, 4), (8, 1, 128, 16, 100, 50, 120), (256, 128, 64, 16, 40, 520, 300),
    (2, 2, 128, 64, 2000, 1, 1999)])
def test_a_token_that_is_not_finite(gpu, value, which, Hq, H, D, block, cached, new, bad):
    """Only rows that see the token, of its K/V head, are NaN; the others are as if it were any other."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    n, pool = cached + new, (cached + new) // block + 2
    g = torch.Generator(device=gpu).manual_seed(7)
    k, v = (torch.randn(n, H, D, device=gpu, generator=g).half() for _ in range(2))
    q = torch.randn(new, Hq, D, device=gpu, generator=g).half()
    outs = []
    for spoil in (False, True):
        b = KvBatch(pool, block, max_requests=1, max_blocks=pool, q_heads=Hq, kv_heads=H, head_dim=D)
        c = KvCache(pool, H, D, block_tokens=block, fmt="e2m1")
        # what the cache's blocks held before: a token that is not finite in every place
        junk = torch.full((pool * block, H, D), math.nan, dtype=torch.float16, device=gpu)
        c.append(junk, junk, torch.arange(pool * block, device=gpu))
        if spoil:
            (k if which == "k" else v)[bad, H - 1, D // 2] = value
        for lo, hi in ((0, cached), (cached, n)):
            if hi > lo:
                st = b.plan(ints([hi - lo], gpu), hi - lo, max_new=hi - lo)
                c.append(k[lo:hi], v[lo:hi], st.slots)
                if lo == 0 and cached:
                    b.commit()
        outs.append(paged_attention(q, c, st))
    clean, spoilt = (o.view(new, H, Hq // H, D) for o in outs)
    assert clean.isfinite().all()
    sees = cached + torch.arange(new, device=gpu) >= bad
    assert spoilt[sees, H - 1].isnan().all()
    assert torch.equal(spoilt[:, : H - 1], clean[:, : H - 1]) and torch.equal(spoilt[~sees], clean[~sees])


def test_table_entry_that_is_no_block(gpu):
    """Its keys are hidden, in the first window of pages and in a later one, for single tokens and for tiles."""
    for lengths, Hq, hide in (([(3000, 1)], 4, {(0, 2), (0, 187)}), ([(100, 1), (1500, 30)], 8, {(1, 3), (1, 70)}),
                              ([(40, 1), (2100, 1), (33, 1)], 2, {(1, 100)})):
        s = Served(gpu, lengths, Hq, 2, 64, 16, "e2m1", torch.float16, seed=11)
        for r, j in hide:
            s.batch.table[r, j] = -1 if j % 2 else 10 ** 6
        from next_step_ai_amd import _runtime

        ws = _runtime.workspace(s.step.workspace_bytes(64), gpu)
        ws[:4] = 0
        out, lse = s.run()
        assert ws[:4].view(torch.int32).item() == 1
        ws[:4] = 0
        t0 = 0
        for r, (c, n) in enumerate(s.lengths):
            keep = [p for p in range(c + n) if (r, p // 16) not in hide]
            slots = [s.slots_of(r, c + n)[p] for p in keep]
            k, v = (torch.from_numpy(s.plain.values(slots, w)).to(gpu) for w in (0, 1))
            want, spread = formula(s.q[t0: t0 + n], k, v, len(keep) - n)
            assert within(out[t0: t0 + n], want, spread, c + n), r
            t0 += n


def test_offsets_past_32_bits(gpu):
    """Blocks whose bytes lie past 2^32: the same bits as in a small cache."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    blocks = (1 << 32) // (8 * 64 * 128 * 17 // 16) + 40
    small = None
    for first in (blocks - 5, 0):
        c = KvCache(blocks if small is None else 5, 8, 128, block_tokens=64, fmt="e2m1")
        order = torch.arange(first, first + 5)
        b = KvBatch(c.num_blocks, 64, max_requests=1, max_blocks=8, q_heads=16, kv_heads=8, free_blocks=order)
        g = torch.Generator(device=gpu).manual_seed(3)
        x, y, q = (torch.randn(300, h, 128, device=gpu, generator=g).half() for h in (8, 8, 16))
        st = b.plan(ints([299], gpu), 299)
        c.append(x[:299], y[:299], st.slots)
        chunk = paged_attention(q[:299], c, st)
        b.commit()
        st1 = b.plan(ints([1], gpu), 1, max_new=1)
        c.append(x[299:], y[299:], st1.slots)
        got = chunk, paged_attention(q[299:], c, st1), c.read(torch.cat([st.slots, st1.slots]))["v"]
        assert small is not None or int(st.slots.max()) // 64 * 8 * 64 * 128 * 17 // 16 > 1 << 32
        if small is None:
            small = got
        else:
            assert all(torch.equal(a, b) for a, b in zip(got, small))


@pytest.mark.parametrize("requests,H,D", [(2500, 8, 64), (700, 2, 128), (300, 16, 128)])
def test_many_short_requests(gpu, requests, H, D):
    """More units in a workgroup's share than it lists at a time; requests without a token, refused ones, a single key."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    rng = np.random.RandomState(requests)
    cached = rng.randint(0, 70, requests)
    cached[::50] = rng.randint(300, 900, len(cached[::50]))
    new = (rng.rand(requests) < 0.9).astype(int)
    Hq, width = 2 * H, 60
    need = int(sum(-(-(c + n) // 16) for c, n in zip(cached, new)))
    b = KvBatch(need, 16, max_requests=requests, max_blocks=width, q_heads=Hq, kv_heads=H, head_dim=D,
                free_blocks=torch.from_numpy(rng.permutation(need)))
    c = KvCache(need, H, D, fmt="e2m1")
    g = torch.Generator(device=gpu).manual_seed(1)
    st = b.plan(ints(cached.tolist(), gpu), int(cached.sum()))
    x, y = (torch.randn(int(cached.sum()), H, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    c.append(x, y, st.slots)
    b.commit()
    total = int(new.sum())
    asked = new.copy()
    refused = [r for r in range(7, requests, 97) if new[r]]
    asked[refused] = 1000  # more blocks than the table's width: refused
    T = int(asked.sum())
    st = b.plan(ints(asked.tolist(), gpu), T, max_new=1)
    x, y = (torch.randn(T, H, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    c.append(x, y, st.slots)
    q = torch.randn(T, Hq, D, device=gpu, generator=g).bfloat16()
    lse = torch.empty(T, Hq, device=gpu)
    out = paged_attention(q, c, st, lse=lse)
    assert total > 0 and st.info.tolist()[2] == len(refused)
    starts, table = st.q_start.tolist(), st.table.cpu()
    for r in {*range(0, requests, max(1, requests // 60)), *range(0, requests, 50), *refused[:5], requests - 1}:
        rows = slice(starts[r], starts[r + 1])
        if r in refused:
            assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()
        elif new[r]:
            n = int(cached[r]) + 1
            p = torch.arange(n)
            got = c.read((table[r][p // 16].long() * 16 + p % 16).to(gpu))
            assert within(out[rows], *formula(q[rows], got["k"], got["v"], n - 1), n), r


@pytest.mark.parametrize("size", [1.0, 40.0, 3000.0, 40000.0])
@pytest.mark.parametrize("Hq,H,D,block,cached,new", [(4, 2, 128, 16, 300, 1), (4, 2, 128, 32, 200, 60), (256, 128, 64, 16, 100, 520)])
def test_scores_of_any_size(gpu, size, Hq, H, D, block, cached, new):
    """Queries that are keys of the cache, scores to 1e10: a row is its key's value where that stands alone, and the mean
    of its values where all keys are the same."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    n, G, pool = cached + new, Hq // H, (cached + new) // block + 1
    g = torch.Generator(device=gpu).manual_seed(3)
    signs = torch.randint(0, 2, (n, H, D), device=gpu, generator=g) * 2 - 1
    for same in (False, True):
        b = KvBatch(pool, block, max_requests=1, max_blocks=pool, q_heads=Hq, kv_heads=H, head_dim=D)
        c = KvCache(pool, H, D, block_tokens=block, fmt="e2m1")
        k = torch.full((n, H, D), size, device=gpu).half() if same else (signs * size).half()
        v = torch.randn(n, H, D, device=gpu, generator=g).half()
        st = b.plan(ints([cached], gpu), cached)
        c.append(k[:cached], v[:cached], st.slots)
        b.commit()
        st = b.plan(ints([new], gpu), new, max_new=new)
        c.append(k[cached:], v[cached:], st.slots)
        ask = (7 * torch.arange(new, device=gpu)) % (cached + 1 + torch.arange(new, device=gpu))
        q = k[ask].repeat_interleave(G, 1)
        out = paged_attention(q, c, st)
        at = torch.arange(n, device=gpu)
        got = c.read(st.table[0][at // block].long() * block + at % block)
        want, spread = formula(q, got["k"], got["v"], cached)
        assert within(out, want, spread, n)


def test_bf16_of_far_exponents(gpu):
    """Queries of 2^60 and 2^-60, keys at both ends of what 4 bits hold."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    for q_size, k_size, new in ((2.0 ** 60, 2.0 ** -22, 1), (2.0 ** -60, 40000.0, 30), (2.0 ** -126, 1.0, 30), (1.0, 1e30, 1), (1.0, 1e-30, 30)):
        b = KvBatch(20, 16, max_requests=1, max_blocks=20, q_heads=4, kv_heads=2, head_dim=64)
        c = KvCache(20, 2, 64, fmt="e2m1")
        g = torch.Generator(device=gpu).manual_seed(2)
        k, v = (torch.randn(200 + new, 2, 64, device=gpu, generator=g) for _ in range(2))
        k, v = (k * k_size).bfloat16(), v.bfloat16()
        q = (torch.randn(new, 4, 64, device=gpu, generator=g) * q_size).bfloat16()
        st = b.plan(ints([200], gpu), 200)
        c.append(k[:200], v[:200], st.slots)
        b.commit()
        st = b.plan(ints([new], gpu), new, max_new=new)
        c.append(k[200:], v[200:], st.slots)
        out = paged_attention(q, c, st)
        p = torch.arange(200 + new, device=gpu)
        got = c.read(st.table[0][p // 16].long() * 16 + p % 16, torch.bfloat16)
        want, spread = formula(q, got["k"], got["v"], 200)
        assert out.isfinite().all()
        # (scores of 2^40: which of two close ones is larger is fp32's to say; there the row is a mix of values all the same)
        assert q_size > 1 or within(out, want, spread, 200 + new)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,block", [(128, 16), (128, 64), (64, 32)])
def test_tiles_of_256_rows(gpu, dtype, D, block):
    """What long prompts run (128 K/V heads: from 1024 rows a head on, 8 waves a workgroup): a chunk with more than 64 blocks
    of 16 tokens behind it, next to a draft, single tokens and a request that waits; with and without log sums, the same
    bits. The bound is the output's rounding, the weights' to fp16 (2^-11 each, 2^-25 of the largest value where one is
    subnormal) and fp32 scores."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    Hq, H, cached, new = 256, 128, [1500, 700, 0, 40, 0], [520, 1, 0, 6, 1]
    pool = sum(-(-(c + n) // block) for c, n in zip(cached, new)) + 2
    b = KvBatch(pool, block, max_requests=5, max_blocks=pool, q_heads=Hq, kv_heads=H, head_dim=D,
                free_blocks=torch.randperm(pool, generator=torch.Generator().manual_seed(1)))
    c = KvCache(pool, H, D, block_tokens=block, fmt="e2m1")
    g = torch.Generator(device=gpu).manual_seed(D + block)
    for lengths in (cached, new):
        T = sum(lengths)
        st = b.plan(ints(lengths, gpu), T, max_new=max(lengths))
        k, v = ((torch.randn(T, H, D, device=gpu, generator=g) * torch.randn(T, H, 1, device=gpu, generator=g).exp2()).to(dtype)
                for _ in range(2))
        c.append(k, v, st.slots)
        if lengths is cached:
            b.commit()
    assert T * 2 // 256 * H >= 512
    q = (torch.randn(T, Hq, D, device=gpu, generator=g) * 1.5).to(dtype)
    lse = torch.full((T, Hq), 7.0, device=gpu)
    out = paged_attention(q, c, st, lse=lse)
    assert torch.equal(paged_attention(q, c, st), out)
    starts, u = st.q_start.tolist(), 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    for r, (have, n) in enumerate(zip(cached, new)):
        if n == 0:
            continue
        at, rows = torch.arange(have + n, device=gpu), slice(starts[r], starts[r + 1])
        got = c.read(st.table[r][at // block].long() * block + at % block)  # (every value is an fp16 number)
        rows_against_formula(q[rows], got["k"], got["v"], out[rows], have, u, 2)
        hidden = at[None] > have + torch.arange(n, device=gpu)[:, None]
        for h in range(0, Hq, 15):
            e = (q[rows, h].double() @ got["k"][:, h // 2].double().t().contiguous() * D ** -0.5).masked_fill(hidden, -math.inf)
            want = torch.logsumexp(e, 1)
            assert ((lse[rows, h].double() - want).abs() <= 2.0 ** -14 + 2.0 ** -20 * want.abs()).all(), (r, h)


@pytest.mark.parametrize("size", [2.0 ** 60, 2.0 ** 100])
@pytest.mark.parametrize("Hq,H,D,block,cached,new", [(4, 2, 128, 16, 300, 1), (4, 2, 64, 16, 200, 6), (4, 2, 128, 32, 200, 60),
                                                     (256, 128, 64, 16, 100, 520), (256, 128, 128, 16, 100, 520)])
def test_bf16_queries_far_above_their_keys(gpu, size, Hq, H, D, block, cached, new):
    """Queries of 2^60 and 2^100 along a key each: that key's value, which 4 bits and a power of two make exact."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    n = cached + new
    pool = n // block + 1
    b = KvBatch(pool, block, max_requests=1, max_blocks=pool, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(pool, H, D, block_tokens=block, fmt="e2m1")
    g = torch.Generator(device=gpu).manual_seed(6)
    k = (torch.randint(0, 2, (n, H, D), device=gpu, generator=g) * 2 - 1).bfloat16()
    v = torch.randn(n, H, D, device=gpu, generator=g).bfloat16()
    st = b.plan(ints([cached], gpu), cached)
    c.append(k[:cached], v[:cached], st.slots)
    b.commit()
    st = b.plan(ints([new], gpu), new, max_new=new)
    c.append(k[cached:], v[cached:], st.slots)
    ask = (7 * torch.arange(new, device=gpu)) % (cached + 1 + torch.arange(new, device=gpu))
    out = paged_attention((k[ask].float() * size).bfloat16().repeat_interleave(Hq // H, 1), c, st)
    slots = st.table[0][ask // block].long() * block + ask % block
    assert torch.equal(out, c.read(slots, torch.bfloat16)["v"].repeat_interleave(Hq // H, 1))


def test_streams(gpu):
    """Two streams at once, each with its own cache and workspace; the same bits as one after the other."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention
    from next_step_ai_amd.lm_head import token_logprobs
    from next_step_ai_amd.rotary import Rotary

    rotary = Rotary(128, 5000)

    def work(seed):
        g = torch.Generator(device=gpu).manual_seed(seed)
        b = KvBatch(400, 16, max_requests=3, max_blocks=300, q_heads=8, kv_heads=2)
        c = KvCache(400, 2, 128, fmt="e2m1")
        outs = []
        for new in ([4000, 30, 0], [1, 1, 1], [1, 20, 1]):
            T = sum(new)
            st = b.plan(ints(new, gpu), T, max_new=max(new))
            k, v = (torch.randn(T, 2, 128, device=gpu, generator=g).half() for _ in range(2))
            q = torch.randn(T, 8, 128, device=gpu, generator=g).half()
            q = c.append_rotated(k, v, st.slots, st.positions, rotary, q=q)
            outs.append(paged_attention(q, c, st))
            b.commit()
        z = torch.randn(2, 128256, device=gpu, generator=g)
        outs += token_logprobs(z, torch.tensor([5, 9], device=gpu), top=3).values()
        return outs

    want = [work(1), work(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(i + 1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


@pytest.mark.parametrize("fmt", ["e2m1", "int8"])
def test_step_in_a_graph(gpu, fmt):
    """Plan, rotated append, attention, log probabilities and commit captured once, replayed with other lengths next to an
    eager batch that does the same, eager work and synchronisation between the replays."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention
    from next_step_ai_amd.lm_head import token_logprobs
    from next_step_ai_amd.rotary import Rotary

    R, Hq, H, D, T = 4, 8, 2, 128, 9
    rotary = Rotary(D, 3000)
    order = torch.randperm(200, generator=torch.Generator().manual_seed(1))

    def fresh():
        return (KvBatch(200, 16, max_requests=R, max_blocks=50, q_heads=Hq, kv_heads=H, head_dim=D, free_blocks=order),
                KvCache(200, H, D, fmt=fmt))

    g = torch.Generator(device=gpu).manual_seed(4)
    steps = [[3, 4, 1, 1], [0, 7, 1, 1], [1, 1, 6, 1], [2, 2, 2, 3], [9, 0, 0, 0], [1, 1, 1, 6]]
    k, v = (torch.empty(T, H, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    q, w = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=gpu), torch.randn(Hq * D, 40000, device=gpu, generator=g).bfloat16()
    new = torch.zeros(R, dtype=torch.int32, device=gpu)
    tokens = torch.arange(T, device=gpu)

    def fill(i):
        gi = torch.Generator(device=gpu).manual_seed(100 + i)
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, device=gpu, generator=gi))
        new.copy_(ints(steps[i], gpu))

    def one(b, c, step=None):
        st = b.plan(new, T, max_new=9, step=step)
        turned = c.append_rotated(k, v, st.slots, st.positions, rotary, q=q)
        out = paged_attention(turned, c, st)
        lp = token_logprobs(out.view(T, -1) @ w, tokens, top=4)
        b.commit()
        return st, (out, st.positions, *lp.values())

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        eager, plain = fresh(), fresh()
        fill(0)
        one(*eager)  # kernels loaded, workspaces allocated
        b, c = fresh()
        step, _ = one(b, c)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            _, captured = one(b, c, step)
        one(*plain)
        for i in range(1, len(steps)):
            fill(i)
            graph.replay()
            _, want = one(*plain)
            stream.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(captured, want)), i
            assert torch.equal(b.cached, plain[0].cached)


@pytest.mark.parametrize("fmt", ["e2m1", "int8"])
@pytest.mark.parametrize("n,H,D,layout", [(1, 3, 64, "rows"), (37, 1, 128, "rows"), (37, 4, 64, "rows"), (70, 4, 128, "heads"),
                                          (21, 3, 64, "stacked"), (21, 3, 64, "turned")])
def test_queries_turned_next_to_keys_and_values(gpu, fmt, n, H, D, layout):
    """In place in a buffer that holds K and V too, whatever the order of its dimensions; over K or V it is refused."""
    from next_step_ai_amd.kv_cache import KvCache
    from next_step_ai_amd.rotary import Rotary

    g = torch.Generator(device=gpu).manual_seed(n)
    if layout == "rows":  # [n, 3 H, D]
        both = torch.randn(n, 3 * H, D, device=gpu, generator=g).half()
        q, k, v = both.split(H, 1)
    elif layout == "heads":  # [n, H, 3, D]
        both = torch.randn(n, H, 3, D, device=gpu, generator=g).half()
        q, k, v = both.unbind(2)
    elif layout == "stacked":  # [3, n, H, D]
        both = torch.randn(3, n, H, D, device=gpu, generator=g).half()
        q, k, v = both.unbind(0)
    else:  # [3 H, n, D]
        both = torch.randn(3 * H, n, D, device=gpu, generator=g).half()
        q, k, v = (t.transpose(0, 1) for t in both.split(H, 0))
    rotary = Rotary(D, 100, interleaved=layout == "heads")
    slots, pos = torch.arange(n, device=gpu), torch.arange(5, 5 + n, dtype=torch.int32, device=gpu)
    apart, cache = (KvCache(5, H, D, fmt=fmt) for _ in range(2))
    q0, k0, v0 = (t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
    want = apart.append_rotated(k0, v0, slots, pos, rotary, q=q0)
    for over in (k, v):
        with pytest.raises(RuntimeError, match="overlaps k or v"):
            cache.append_rotated(k, v, slots, pos, rotary, q=q0, q_out=over)
    assert torch.equal(q, q0) and torch.equal(k, k0) and not cache.data.any()
    assert cache.append_rotated(k, v, slots, pos, rotary, q=q, q_out=q) is q
    assert torch.equal(q, want) and torch.equal(k, k0) and torch.equal(v, v0)
    assert torch.equal(cache.data, apart.data)


@pytest.mark.parametrize("fmt", ["e2m1", "int8"])
def test_queries_turned_into_the_other_half_of_their_buffer(gpu, fmt):
    """Slices of one buffer that have no element in common, in rows, in heads and in dims."""
    from next_step_ai_amd.kv_cache import KvCache
    from next_step_ai_amd.rotary import Rotary

    n, Hq, H, D = 19, 4, 2, 64
    g = torch.Generator(device=gpu).manual_seed(2)
    rotary = Rotary(D, 100)
    slots, pos = torch.arange(n, device=gpu), torch.arange(n, dtype=torch.int32, device=gpu)
    k, v = (torch.randn(n, H, D, device=gpu, generator=g).half() for _ in range(2))
    q = torch.randn(n, Hq, D, device=gpu, generator=g).half()
    cache = KvCache(2, H, D, fmt=fmt)
    want = cache.append_rotated(k, v, slots, pos, rotary, q=q)
    for shape, parts in (((n, 2 * Hq, D), lambda t: (t[:, :Hq], t[:, Hq:])), ((n, 2 * Hq, D), lambda t: (t[:, ::2], t[:, 1::2])),
                         ((n, Hq, 2 * D), lambda t: (t[:, :, D:], t[:, :, :D])), ((2 * n, Hq, D), lambda t: (t[::2], t[1::2]))):
        both = torch.full(shape, 7.0, dtype=torch.float16, device=gpu)
        mine, out = parts(both)
        mine.copy_(q)
        assert cache.append_rotated(k, v, slots, pos, rotary, q=mine, q_out=out) is out
        assert torch.equal(out, want) and torch.equal(mine, q)


def test_a_run_of_them(gpu):
    """Steps of a small model's layer as a server makes them: fused projection, rotated append in place, attention, a head,
    log probabilities; against the same in 64 bits from what the cache gives back, and against the 8-bit cache's."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention
    from next_step_ai_amd.lm_head import dense_linear_nf4, lm_head_forward, lm_head_nf4_meta, token_logprobs
    from next_step_ai_amd.rotary import Rotary
    from next_step_ai_amd._runtime import nf4_code
    from next_step_ai_amd.synth import synth_nf4

    hidden, Hq, H, D, vocab = 1024, 8, 2, 128, 5000
    widths = [Hq * D, H * D, H * D]
    qkv = synth_nf4(3, sum(widths) * hidden, 64, hidden ** -0.5, gpu)
    head = synth_nf4(4, vocab * Hq * D, 64, (Hq * D) ** -0.5, gpu)
    meta = lm_head_nf4_meta(*head, nf4_code(gpu), vocab, Hq * D, 64)
    rotary = Rotary(D, 400, base=500000.0)
    results = {}
    for fmt in ("e2m1", "int8"):
        g = torch.Generator(device=gpu).manual_seed(9)
        b = KvBatch(60, 16, max_requests=3, max_blocks=20, q_heads=Hq, kv_heads=H, head_dim=D)
        c = KvCache(60, H, D, fmt=fmt)
        done, all_lp = [0, 0, 0], []
        for new in ([200, 33, 1], [1, 1, 1], [5, 1, 60], [1, 1, 1]):
            T = sum(new)
            st = b.plan(ints(new, gpu), T, max_new=max(new))
            x = torch.randn(T, hidden, device=gpu, generator=g).half()
            both = dense_linear_nf4(x, *qkv, nf4_code(gpu), sum(widths), hidden, 64)
            q, k, v = (t.view(T, -1, D) for t in both.split(widths, 1))
            plain_q = q.clone()
            turned = c.append_rotated(k, v, st.slots, st.positions, rotary, q=q, q_out=q)
            assert turned is q
            cos, sin = (rotary.table.cpu()[st.positions.cpu().long()][..., i] for i in (0, 1))
            assert torch.equal(q.cpu(), ref.rotate(plain_q.cpu(), cos, sin, False))
            out = paged_attention(q, c, st)
            starts, table = st.q_start.tolist(), st.table.cpu()
            for r, n in enumerate(new):
                rows, keys = slice(starts[r], starts[r] + n), done[r] + n
                p = torch.arange(keys)
                got = c.read((table[r][p // 16].long() * 16 + p % 16).to(gpu), torch.float16)
                if fmt == "e2m1":  # (every value is an fp16 number)
                    assert within(out[rows], *formula(q[rows], got["k"], got["v"], done[r]), keys)
                done[r] = keys
            b.commit()
            ends = torch.tensor(starts[1:], device=gpu) - 1
            logits = lm_head_forward(out.view(T, -1)[ends][None], meta)[0]
            lp = token_logprobs(logits, logits.argmax(-1), top=3)
            z = torch.log_softmax(logits.double(), -1)
            assert torch.equal(lp["top_ids"][:, 0], (logits == logits.amax(-1, keepdim=True)).int().argmax(-1))
            assert ((lp["logprob"].double() - z.amax(-1)).abs() <= 2.0 ** -16).all()
            assert ((lp["entropy"].double() + (z.exp() * z).sum(-1)).abs() <= 2.0 ** -14).all()
            all_lp.append(z)
        results[fmt] = torch.cat(all_lp)
    # the two caches' distributions are close: a code of 4 bits is off by a sixth of its group's largest at most
    kl = (results["int8"].exp() * (results["int8"] - results["e2m1"])).sum(-1)
    assert (kl >= -1e-6).all() and (kl < 0.5).all()


def test_tensors_of_a_device_that_is_not_the_current_one(gpu, monkeypatch):
    """Every call makes its tensors' device current and gives the same (here there is one: the current one is said to be another)."""
    from next_step_ai_amd import kv_cache, lm_head
    from next_step_ai_amd.rotary import Rotary

    g = torch.Generator(device=gpu).manual_seed(1)
    k, v, q = (torch.randn(5, h, 64, device=gpu, generator=g).half() for h in (2, 2, 4))
    z = torch.randn(3, 500, device=gpu, generator=g)
    entered = []
    real = torch.cuda.device

    class Noted(real):
        def __enter__(self):
            super().__enter__()
            entered.append(self.idx)
            monkeypatch.setattr(kv_cache, "current_device", lambda: 0)
            monkeypatch.setattr(lm_head, "current_device", lambda: 0)

    def elsewhere():
        monkeypatch.setattr(kv_cache, "current_device", lambda: 1)
        monkeypatch.setattr(lm_head, "current_device", lambda: 1)

    results = []
    for other in (False, True):
        if other:
            monkeypatch.setattr(torch.cuda, "device", Noted)
        away = elsewhere if other else lambda: None
        b = kv_cache.KvBatch(4, 16, max_requests=1, max_blocks=4, q_heads=4, kv_heads=2, head_dim=64)
        c = kv_cache.KvCache(4, 2, 64, fmt="e2m1")
        rotary = Rotary(64, 10)
        away()
        st = b.plan(ints([5], gpu), 5)
        away()
        c.append(k, v, st.slots)
        away()
        turned = c.append_rotated(k, v, st.slots, st.positions, rotary, q=q)
        away()
        got = c.read(st.slots)
        away()
        out = kv_cache.paged_attention(turned, c, st)
        away()
        b.commit()
        away()
        lp = lm_head.token_logprobs(z, top=3)
        results.append([turned, got["k"], out, b.cached.clone(), *lp.values()])
    assert all(torch.equal(x, y) for x, y in zip(*results)) and entered == [0] * 7
