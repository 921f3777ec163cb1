"""The paged 8-bit cache and its attention where a step refuses requests, holds
values that are not finite, or reaches an end of a type's range."""
import numpy as np
import pytest
import torch

from oracle import kv_reference as ref

pytestmark = pytest.mark.gpu


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ------------------------------------------------------------- refusals --
def owned(batch, pool):
    """Asserts that the requests' blocks and the free ones are the pool, each once; returns the requests'."""
    table, (head, free), ring = batch.table.tolist(), batch.state.tolist(), batch.ring.tolist()
    blocks = [table[r][: -(-n // batch.block_tokens)] for r, n in enumerate(batch.cached.tolist())]
    ids = [b for own in blocks for b in own] + [ring[(head + i) % pool] for i in range(free)]
    assert sorted(ids) == list(range(pool))
    return blocks


def test_blocks_after_a_request_longer_than_max_new(gpu):
    """A request refused for its length takes nothing: those after it get the ring's next entries, and no block has two owners."""
    from next_step_ai_amd.kv_cache import KvBatch

    batch = KvBatch(20, 16, max_requests=3, max_blocks=8, q_heads=8, kv_heads=2)
    step = batch.plan(ints([40, 5, 5], gpu), 50, max_new=16)
    assert step.kv_len.tolist() == [0, 5, 5] and step.info.tolist() == [2, 18, 1, 50]
    assert step.slots.tolist() == [-1] * 40 + list(range(0, 5)) + list(range(16, 21))
    batch.commit()
    assert owned(batch, 20) == [[], [0], [1]]
    batch.plan(ints([1, 12, 16], gpu), 29, max_new=16).check()
    batch.commit()
    assert owned(batch, 20) == [[2], [0, 3], [1, 4]]


@pytest.mark.parametrize("requests,block,seed", [(3, 16, 1), (70, 32, 2), (300, 16, 3), (1100, 64, 4)])
def test_blocks_over_steps_with_every_refusal(gpu, requests, block, seed):
    """Random steps in which requests are refused for max_new, for the table's width and for want of blocks, against the
    plain batch; after each, every block has one owner."""
    from next_step_ai_amd.kv_cache import KvBatch

    rng = np.random.RandomState(seed)
    pool, width = 3 * requests, 5
    order = rng.permutation(pool)
    batch = KvBatch(pool, block, max_requests=requests, max_blocks=width, q_heads=8, kv_heads=2,
                    free_blocks=torch.from_numpy(order))
    plain = ref.PlainBatch(pool, block, requests, width, order)
    for _ in range(8):
        new = [int(rng.choice([0, 1, 1, block // 2, block, 2 * block + 1, 6 * block])) for _ in range(requests)]
        total, most = max(1, sum(new)), int(rng.choice([0, block, 3 * block]))
        want = plain.plan(new, total, most)
        step = batch.plan(ints(new, gpu), total, max_new=most)
        assert step.slots.tolist() == want["slots"] and step.kv_len.tolist() == want["kv_len"]
        assert step.info.tolist()[1:] == [want["free"], want["refused"], sum(new)]
        ended = [r for r in range(requests) if rng.rand() < 0.2]
        plain.commit(ended)
        batch.commit(ints([int(r in ended) for r in range(requests)], gpu))
        assert batch.cached.tolist() == plain.cached and owned(batch, pool) == plain.blocks


@pytest.mark.parametrize("dtype,D", [(torch.float16, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("group,most", [(8, 1), (2, 6), (16, 1), (1, 16), (40, 1)])
def test_rows_of_a_request_longer_than_max_new(gpu, dtype, D, group, most):
    """Zeros and -inf in all of them, next to requests that are served, also where no request of max_new tokens fills
    more than one tile of 16 rows."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    H, new = 2, [1, 40, 0, most, most + 1, 1]
    total = sum(new)
    b = KvBatch(20, 16, max_requests=len(new), max_blocks=4, q_heads=H * group, kv_heads=H)
    c = KvCache(20, H, D)
    g = torch.Generator(device=gpu).manual_seed(group)
    st = b.plan(ints(new, gpu), total + 1, max_new=most)
    assert st.kv_len.tolist() == [1, 0, 0, most, 0, 1]
    k, v, q = (torch.randn(total + 1, h, D, device=gpu, generator=g).to(dtype) for h in (H, H, H * group))
    c.append(k, v, st.slots)
    for with_lse in (True, False):
        out = torch.full_like(q, 3.0)
        lse = torch.full(q.shape[:2], 3.0, device=gpu) if with_lse else None
        paged_attention(q, c, st, out=out, lse=lse)
        t0 = 0
        for n in new:
            refused = n > most
            rows = out[t0: t0 + n]
            assert bool((rows == 0).all()) if refused else bool((rows.abs().amax(-1) > 0).all())
            if with_lse:
                assert ((lse[t0: t0 + n] == -np.inf) == refused).all()
            t0 += n
        assert (out[total:] == 3).all() and (lse is None or (lse[total:] == 3).all())
        # one key: the row is its value, read back
        assert torch.equal(out[0].view(H, group, D), c.read(st.slots[:1], dtype)["v"][0][:, None].expand(H, group, D))


# --------------------------------------------- values that are not finite --
def rows_against_formula(q, keys, values, out, first, u, group):
    """Rows i < len(q), which see keys 0 .. first + i, against the formula in 64 bits; the tolerance of an output's
    rounding u, the weights' to fp16 (2^-11 each, 2^-25 of the largest value where one is subnormal) and fp32 scores."""
    D = q.shape[-1]
    k, v = keys.double(), values.double()
    n = k.shape[0]
    hidden = torch.arange(n, device=q.device)[None] > first + torch.arange(q.shape[0], device=q.device)[:, None]
    for h in range(q.shape[1]):
        kh, vh = k[:, h // group].contiguous(), v[:, h // group].contiguous()
        e = (q[:, h].double() @ kh.t().contiguous() * D ** -0.5).masked_fill(hidden, -np.inf)
        p = torch.softmax(e, 1)
        want, spread = p @ vh, p @ vh.abs()
        bound = u * want.abs() + (2.0 ** -11 + 2.0 ** -15) * spread + n * 2.0 ** -25 * float(vh.abs().max()) + 2.0 ** -24
        assert ((out[:, h].double() - want).abs() <= bound).all(), h


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("Hq,H,D,block,cached,new,bad", [
    (4, 2, 64, 16, 13, 6, 5),         # a draft: 16 rows streamed, the block begins inside it
    (8, 8, 128, 16, 30, 9, 4),
    (4, 2, 64, 16, 20, 40, 30),       # a chunk: a tile of 128 rows
    (6, 1, 128, 32, 0, 100, 70),
    (256, 128, 64, 16, 100, 520, 333),  # tiles of 256 rows
])
def test_a_value_that_is_not_finite_reaches_only_rows_that_see_its_block(gpu, which, value, fmt, Hq, H, D, block, cached, new, bad):
    """Appended in a step's later token: rows that end before its block are as the formula says, rows that see the
    block are NaN, and so is what is read back, in its head alone."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    dtype = torch.bfloat16
    pool = (cached + new) // block + 2
    b = KvBatch(pool, block, max_requests=1, max_blocks=pool, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(pool, H, D, block_tokens=block, fmt=fmt)
    g = torch.Generator(device=gpu).manual_seed(new)

    def rows(n, h):
        return torch.randn(n, h, D, device=gpu, generator=g).to(dtype)

    if cached:
        st = b.plan(ints([cached], gpu), cached)
        c.append(rows(cached, H), rows(cached, H), st.slots)
        b.commit()
    st = b.plan(ints([new], gpu), new, max_new=new)
    kv, head, G = {"k": rows(new, H), "v": rows(new, H)}, H - 1, Hq // H
    kv[which][bad, head, 3] = value
    q = rows(new, Hq)
    c.append(kv["k"], kv["v"], st.slots)
    lse = torch.empty(new, Hq, device=gpu)
    out = paged_attention(q, c, st, lse=lse)
    start = (cached + bad) // block * block  # the block's first token
    clean = start - cached                   # rows that end before it
    assert 0 < clean < new
    at = torch.arange(cached + new, device=gpu)
    stored = c.read(st.table[0][at // block].long() * block + at % block, dtype)
    poisoned = torch.zeros(cached + new, H, dtype=torch.bool, device=gpu)
    poisoned[start: start + block, head] = True
    assert torch.equal(stored[which].isnan().all(-1), poisoned) and torch.equal(stored[which].isnan().any(-1), poisoned)
    assert not stored["v" if which == "k" else "k"].isnan().any()
    mine = slice(head * G, (head + 1) * G)
    assert out[clean:, mine].isnan().all() and lse[clean:, mine].isnan().all()
    assert not out[:clean].isnan().any() and not out[:, : head * G].isnan().any()
    assert lse[:clean].isfinite().all() and lse[:, : head * G].isfinite().all()
    if fmt == "e4m3":  # rounded to bf16 without loss: 4 bits and a power of two
        rows_against_formula(q[:clean], stored["k"][:start], stored["v"][:start], out[:clean], cached, 2.0 ** -8, G)


# ------------------------------------------------------- far into a request --
def test_a_table_entry_that_is_no_block_in_a_later_window_of_pages(gpu):
    """A wave that starts 32 tokens into a block of 64 takes its second window of 64 pages between the two tiles of a
    pair: a bad entry there hides its keys as one in the first window does, whatever block 0 holds."""
    from next_step_ai_amd._runtime import StatusWord, workspace
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    H, D, B, n = 256, 64, 64, 16500  # one share for all keys, a quarter (4128, rounded up to 32) for each wave
    blocks = -(-n // B)
    b = KvBatch(blocks + 1, B, max_requests=1, max_blocks=blocks, q_heads=H, kv_heads=H, head_dim=D,
                free_blocks=torch.arange(1, blocks + 1))
    c = KvCache(blocks + 1, H, D, block_tokens=B)
    g = torch.Generator(device=gpu).manual_seed(1)
    q = torch.randn(1, H, D, device=gpu, generator=g).half()
    big = (4 * q).expand(B, H, D)  # block 0: keys that a softmax would not overlook, with large values
    c.append(big, torch.full_like(big, 100.0), torch.arange(B, device=gpu))
    st = b.plan(ints([n - 1], gpu), n - 1)
    for at in range(0, n - 1, 4 * 1024):  # (blocks whole in every call)
        to = min(at + 4 * 1024, n - 1)
        k, v = (torch.randn(to - at, H, D, device=gpu, generator=g).half() for _ in range(2))
        c.append(k, v, st.slots[at:to])
    b.commit()
    st = b.plan(ints([1], gpu), 1, max_new=1)
    c.append(q, q, st.slots)
    slots = (st.table[0][torch.arange(n, device=gpu) // B].long() * B + torch.arange(n, device=gpu) % B)
    heads = (0, 1, 100, 255)
    stored = c.read(slots)
    scale = c.scale[slots // B]  # (tokens, heads, 2)
    for page in (64, 127, 128, 129, blocks - 1):
        was = b.table[0, page].clone()
        b.table[0, page] = -1
        out = paged_attention(q, c, st)
        b.table[0, page] = was
        keep = torch.arange(n, device=gpu) // B != page
        for h in heads:
            # the codes' values exactly: what is read back, rounded to fp16, over the scale is a whole number
            k, v = (torch.round(stored[x][:, h].double() / scale[:, h, i, None].double()) * scale[:, h, i, None].double()
                    for i, x in ((0, "k"), (1, "v")))
            e = (k[keep] @ q[0, h].double()) * D ** -0.5
            p = torch.softmax(e, 0)
            want, spread = p @ v[keep], p @ v[keep].abs()
            bound = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -15) * spread + n * 2.0 ** -25 * float(v.abs().max()) + 2.0 ** -24
            assert ((out[0, h].double() - want).abs() <= bound).all(), (page, h)
    StatusWord(gpu, "paged attention").clear(workspace(1 << 20, gpu))


def test_a_captured_step_after_a_larger_call_on_its_stream(gpu, monkeypatch):
    """The graph's workspace is its own still when a later call has made the stream's larger: partial results and
    arrival counters of every replay, next to memory that others have filled since."""
    from next_step_ai_amd import _runtime
    from next_step_ai_amd._runtime import workspace
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    monkeypatch.setattr(_runtime, "_workspaces", {})  # streams that no test has used
    lengths, Hq, H, D = [5000, 700, 3100], 8, 2, 128
    g = torch.Generator(device=gpu).manual_seed(6)
    b = KvBatch(600, 16, max_requests=3, max_blocks=400, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(600, H, D)
    st = b.plan(ints(lengths, gpu), sum(lengths))
    k, v = (torch.randn(sum(lengths), H, D, device=gpu, generator=g).half() for _ in range(2))
    c.append(k, v, st.slots)
    b.commit()
    st = b.plan(ints([1, 1, 1], gpu), 3, max_new=1)
    c.append(k[:3], v[:3], st.slots)
    q, out = (torch.randn(3, Hq, D, device=gpu, generator=g).half() for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_attention(q, c, st, out=out)
        small = workspace(1, gpu).numel()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        paged_attention(q, c, st, out=out)
    big = KvBatch(600, 16, max_requests=1, max_blocks=400, q_heads=4 * Hq, kv_heads=4 * H, head_dim=D)
    wide = KvCache(600, 4 * H, D)
    with torch.cuda.stream(side):
        long = big.plan(ints([300], gpu), 300)
        x = torch.randn(300, 4 * H, D, device=gpu, generator=g).half()
        wide.append(x, x, long.slots)
        paged_attention(x.repeat(1, 4, 1), wide, long)
        assert workspace(1, gpu).numel() > small
        fill = [torch.full((small + 256,), 0x7F, dtype=torch.uint8, device=gpu) for _ in range(8)]
    torch.cuda.synchronize()
    for _ in range(4):
        q.normal_(generator=g)
        out.fill_(3.0)
        want = paged_attention(q, c, st)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all((f == 0x7F).all() for f in fill)


def test_a_step_captured_without_a_call_before_it(gpu, monkeypatch):
    """Its workspace is made inside the capture: eager calls on that stream before the first replay have one of their
    own, and replays give what eager calls give."""
    from next_step_ai_amd import _runtime
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    monkeypatch.setattr(_runtime, "_workspaces", {})
    n, Hq, H, D = 4000, 8, 2, 128
    g = torch.Generator(device=gpu).manual_seed(7)
    b = KvBatch(300, 16, max_requests=1, max_blocks=300, q_heads=Hq, kv_heads=H, head_dim=D)
    caches = [KvCache(300, H, D) for _ in range(2)]
    st = b.plan(ints([n], gpu), n)
    for c in caches:
        c.append(*(torch.randn(n, H, D, device=gpu, generator=g).half() for _ in range(2)), st.slots)
    b.commit()
    st = b.plan(ints([1], gpu), 1, max_new=1)
    q, *outs = (torch.randn(1, Hq, D, device=gpu, generator=g).half() for _ in range(3))
    for c in caches:
        c.append(q[:, :H], q[:, :H], st.slots)
    want = [paged_attention(q, c, st) for c in caches]  # (and the kernels are loaded)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for c, out in zip(caches, outs):
            paged_attention(q, c, st, out=out)
    with torch.cuda.stream(side):
        eager = [paged_attention(q, c, st) for c in caches]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(eager, want))
    for _ in range(4):
        for out in outs:
            out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
        with torch.cuda.stream(side):
            assert torch.equal(paged_attention(q, caches[0], st), want[0])
        torch.cuda.synchronize()


# ------------------------------------------------------------- arguments --
def test_workspaces_that_the_kernels_cannot_use(gpu):
    """One in host memory, and one that is larger than its memory."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    b, c = KvBatch(8, 16, max_requests=2, max_blocks=4, q_heads=4, kv_heads=2, head_dim=64), KvCache(8, 2, 64)
    st = b.plan(ints([20, 3], gpu), 23)
    x = torch.ones(23, 4, 64, dtype=torch.float16, device=gpu)
    c.append(x[:, :2], x[:, :2], st.slots)
    for ws in (torch.zeros(1 << 25, dtype=torch.uint8), torch.zeros(256, dtype=torch.uint8, device=gpu).expand(1 << 17, 256)):
        with pytest.raises(RuntimeError, match="ws must be"):
            paged_attention(x, c, st, ws=ws)
    assert torch.equal(paged_attention(x, c, st), x)


def test_a_step_that_no_plan_has_written(gpu):
    """Its work lists hold anything: the attention refuses it until a plan has been made into it."""
    from next_step_ai_amd import _lib
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, KvStep, paged_attention

    b, c = KvBatch(8, 16, max_requests=2, max_blocks=4, q_heads=4, kv_heads=2, head_dim=64), KvCache(8, 2, 64)
    x = torch.ones(23, 4, 64, dtype=torch.float16, device=gpu)
    st = KvStep(b, 23, 0)
    with pytest.raises(RuntimeError, match="not been planned"):
        paged_attention(x, c, st)
    with _lib.injected_faults("kv_plan=hip:1"):
        with pytest.raises(RuntimeError, match="injected fault"):
            b.plan(ints([20, 3], gpu), 23, step=st)
    with pytest.raises(RuntimeError, match="not been planned"):
        paged_attention(x, c, st)
    assert b.plan(ints([20, 3], gpu), 23, step=st) is st
    c.append(x[:, :2], x[:, :2], st.slots)
    assert torch.equal(paged_attention(x, c, st), x)


def test_commit_that_fails_can_be_made_again(gpu):
    """A commit that raises has done nothing: the plan is still the one to commit."""
    from next_step_ai_amd import _lib
    from next_step_ai_amd.kv_cache import KvBatch

    b = KvBatch(8, 16, max_requests=2, max_blocks=4, q_heads=4, kv_heads=2)
    b.plan(ints([20, 3], gpu), 23)
    with _lib.injected_faults("kv_commit=hip:1"):
        with pytest.raises(RuntimeError, match="injected fault"):
            b.commit()
    assert b.cached.tolist() == [0, 0]
    b.commit()
    assert b.cached.tolist() == [20, 3]
    b.commit()
    assert b.cached.tolist() == [20, 3]


def test_one_token_or_one_head_of_any_stride(gpu):
    """A decode step's rows where they lie in a fused projection of odd width, and one K/V head of any stride."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    g = torch.Generator(device=gpu).manual_seed(8)
    for H in (1, 2):
        b, c, same = (KvBatch(8, 16, max_requests=1, max_blocks=4, q_heads=2 * H, kv_heads=H, head_dim=64),
                      KvCache(8, H, 64), KvCache(8, H, 64))
        st = b.plan(ints([1], gpu), 1, max_new=1)
        wide = torch.randn(4 * H * 64 + 3, device=gpu, generator=g).half()
        q = wide.as_strided((1, 2 * H, 64), (4 * H * 64 + 3, 64, 1))
        k = wide.as_strided((1, H, 64), (4 * H * 64 + 3, 64 if H > 1 else 77, 1), 2 * H * 64)
        v = wide.as_strided((1, H, 64), (4 * H * 64 + 3, 64 if H > 1 else 77, 1), 3 * H * 64)
        c.append(k, v, st.slots)
        same.append(k.reshape(-1).view(1, H, 64), v.reshape(-1).view(1, H, 64), st.slots)
        assert torch.equal(c.data, same.data) and torch.equal(c.scale, same.scale)
        assert torch.equal(paged_attention(q, c, st), paged_attention(q.reshape(-1).view(1, 2 * H, 64), c, st))


@pytest.mark.parametrize("value", [0.0, 2.0 ** -95])
@pytest.mark.parametrize("Hq,H,D,block,n,new", [
    (4, 1, 64, 64, 1200000, 1),      # streamed
    (4, 1, 64, 64, 1200000, 33),     # a tile of 128 rows, its keys in parts
    (128, 128, 64, 64, 1200000, 1100),  # tiles of 256 rows, whole requests
])
def test_many_keys_at_the_least_scale(gpu, value, Hq, H, D, block, n, new):
    """V scales of 2^-100 (values of zero among them) for all of a long request: the sums of the weights over the scales
    stay within fp32, so lse is finite and outputs keep their share."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    blocks = -(-n // block)
    b = KvBatch(blocks, block, max_requests=1, max_blocks=blocks, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(blocks, H, D, block_tokens=block, fmt="e4m3")
    g = torch.Generator(device=gpu).manual_seed(2)
    k = torch.randn(block, H, D, device=gpu, generator=g).bfloat16()  # every block holds the same keys
    v = torch.full((block, H, D), value, dtype=torch.bfloat16, device=gpu)
    st = b.plan(ints([n - new], gpu), n - new)
    b.commit()
    st = b.plan(ints([new], gpu), new, max_new=new)
    c.append(k, v, torch.arange(block, device=gpu))
    c.data[1:], c.scale[1:] = c.data[0], c.scale[0]
    assert (c.scale[:, :, 1] == 2.0 ** -100).all()
    q = (torch.randn(new, Hq, D, device=gpu, generator=g) * 0.25).bfloat16()
    lse = torch.empty(new, Hq, device=gpu)
    out = paged_attention(q, c, st, lse=lse)
    kept = c.read(torch.arange(block, device=gpu), torch.bfloat16)["k"].double()  # (exact: 4 bits and a power of two)
    seen = n - new + 1 + torch.arange(new, device=gpu)
    times = (seen[:, None] - torch.arange(block, device=gpu) + block - 1) // block  # how often a row sees each of the keys
    for h in range(0, Hq, max(1, Hq // 4)):
        e = q[:, h].double() @ kept[:, h * H // Hq].t().contiguous() * D ** -0.5
        want = torch.logsumexp(e + times.double().log(), 1)
        # fp32 sums of n / 64 tiles one after the other, each rounded (the same way, as the keys repeat): 2^-24 per tile
        sums = n / 64 * 2.0 ** -24
        assert ((lse[:, h].double() - want).abs() <= 2.0 ** -14 + sums + 2.0 ** -20 * want.abs()).all()
        # all values are the same: a row is that value, but for its own rounding (2^-9), the weights' (2^-11) and two sums
        assert ((out[:, h].double() - value).abs() <= (2.0 ** -9 + 2.0 ** -11 + 2.0 ** -15 + 2 * sums) * value).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("size", [1000.0, 3000.0, 60000.0])
@pytest.mark.parametrize("Hq,H,D,block,cached,new", [
    (4, 2, 128, 16, 300, 1),
    (4, 2, 128, 32, 200, 60),
    (256, 128, 64, 16, 100, 520),
])
def test_scores_of_any_size(gpu, fmt, size, Hq, H, D, block, cached, new):
    """Queries that are keys of the cache, with magnitudes up to fp16's largest: scores to 4e10, each row's own key far
    above the others, so that the row is that key's value."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    n, G = cached + new, Hq // H
    pool = n // block + 1
    b = KvBatch(pool, block, max_requests=1, max_blocks=pool, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(pool, H, D, block_tokens=block, fmt=fmt)
    g = torch.Generator(device=gpu).manual_seed(3)
    signs = torch.randint(0, 2, (n, H, D), device=gpu, generator=g) * 2 - 1
    k, v = (signs * size).half(), torch.randn(n, H, D, device=gpu, generator=g).half()
    if cached:
        st = b.plan(ints([cached], gpu), cached)
        c.append(k[:cached], v[:cached], st.slots)
        b.commit()
    st = b.plan(ints([new], gpu), new, max_new=new)
    c.append(k[cached:], v[cached:], st.slots)
    # row i asks for key (7 i) mod its last + 1: signs that agree in all dims, against about half of them
    ask = (7 * torch.arange(new, device=gpu)) % (cached + 1 + torch.arange(new, device=gpu))
    lse = torch.empty(new, Hq, device=gpu)
    q = k[ask].repeat_interleave(G, 1)
    out = paged_attention(q, c, st, lse=lse)
    at = torch.arange(n, device=gpu)
    slots = st.table[0][at // block].long() * block + at % block
    got = c.read(slots[ask])
    want = got["v"].repeat_interleave(G, 1)
    # the key's weight is 1 to 64 bits; the value was rounded to fp16 when read, and the row again
    assert ((out.double() - want.double()).abs() <= 2.0 ** -10 * want.double().abs() + 2.0 ** -24).all()
    top = (q.double() * got["k"].repeat_interleave(G, 1).double()).sum(-1) * D ** -0.5
    # 2^-11 of the keys read back (size 60000 passes fp16 by its code's rounding nowhere), fp32 sums of 128 products
    assert ((lse.double() - top).abs() <= (2.0 ** -11 + 2.0 ** -16) * top).all()


@pytest.mark.parametrize("fmt", ["e2m1", "int8", "e4m3"])
@pytest.mark.parametrize("which,value", [("k", float("nan")), ("k", float("inf")), ("v", -float("inf"))])
@pytest.mark.parametrize("Hq,H,D,block,cached,new,bad", [
    (4, 2, 128, 16, 600, 1, 0),       # single tokens: in a wave's first tile, in a later one, in the last
    (4, 2, 128, 16, 600, 1, 333),
    (4, 2, 64, 32, 600, 1, 600),
    (4, 2, 64, 16, 200, 6, 70),       # drafts
    (4, 2, 64, 16, 200, 6, 203),
    (4, 2, 128, 32, 200, 60, 5),      # tiles of 128 rows
    (4, 2, 128, 32, 200, 60, 236),
    (8, 8, 64, 16, 0, 40, 17),
    (256, 128, 64, 16, 100, 520, 40),  # of 256
    (256, 128, 64, 16, 100, 520, 433),
])
def test_a_value_that_is_not_finite_among_far_scores(gpu, fmt, which, value, Hq, H, D, block, cached, new, bad):
    """Queries that are keys of the cache, of size 3000, so that scores pass 2^20: rows that see the token (in 8 bits its
    block, whose scale is NaN) are NaN, the others their key's value."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    n, G, head = cached + new, Hq // H, H - 1
    pool = n // block + 1
    b = KvBatch(pool, block, max_requests=1, max_blocks=pool, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(pool, H, D, block_tokens=block, fmt=fmt)
    g = torch.Generator(device=gpu).manual_seed(3)
    k = ((torch.randint(0, 2, (n, H, D), device=gpu, generator=g) * 2 - 1) * 3000.0).half()
    v = torch.randn(n, H, D, device=gpu, generator=g).half()
    ask = (7 * torch.arange(new, device=gpu)) % (cached + 1 + torch.arange(new, device=gpu))
    q = k[ask].repeat_interleave(G, 1)
    kv = {"k": k, "v": v}
    kv[which][bad, head, 3] = value
    if cached:
        st = b.plan(ints([cached], gpu), cached)
        c.append(k[:cached], v[:cached], st.slots)
        b.commit()
    st = b.plan(ints([new], gpu), new, max_new=new)
    c.append(k[cached:], v[cached:], st.slots)
    lse = torch.empty(new, Hq, device=gpu)
    out = paged_attention(q, c, st, lse=lse)
    first = bad if fmt == "e2m1" else bad // block * block  # the first key that is not a number
    sees = (cached + torch.arange(new, device=gpu) >= first)[:, None] & (torch.arange(Hq, device=gpu) >= head * G)[None]
    assert sees.any() and not sees.all()
    assert torch.equal(out.isnan().all(-1), sees) and torch.equal(out.isnan().any(-1), sees)
    assert torch.equal(lse.isnan(), sees)
    at = torch.arange(n, device=gpu)
    slots = st.table[0][at // block].long() * block + at % block
    want = c.read(slots[ask])["v"].repeat_interleave(G, 1).double()
    off = (out.double() - want).abs() <= 2.0 ** -10 * want.abs() + 2.0 ** -24  # read and row rounded once each
    assert off.all(-1)[~sees].all()


@pytest.mark.parametrize("fmt", ["e2m1", "int8"])
@pytest.mark.parametrize("Hq,H,D,cached,new", [(16, 2, 128, [9000, 40, 3], [1, 1, 1]), (8, 2, 64, [5000, 0, 17], [3, 1, 40]),
                                               (256, 128, 64, [100], [520])])
def test_outputs_over_queries(gpu, fmt, Hq, H, D, cached, new):
    """In the queries' own memory: the same bits.  Anywhere else over them: refused, as other rows' queries would be lost."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    pool = sum(-(-(c + n) // 16) for c, n in zip(cached, new))
    b = KvBatch(pool, 16, max_requests=len(new), max_blocks=pool, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(pool, H, D, fmt=fmt)
    g = torch.Generator(device=gpu).manual_seed(5)
    for lengths in (cached, new):
        T = sum(lengths)
        st = b.plan(ints(lengths, gpu), T, max_new=max(lengths))
        k, v = (torch.randn(T, H, D, device=gpu, generator=g).half() for _ in range(2))
        c.append(k, v, st.slots)
        if lengths is cached:
            b.commit()
    wide = torch.randn(T + 1, Hq, D, device=gpu, generator=g).half()
    q = wide[:T]
    want = paged_attention(q, c, st)
    for over in (wide[1:], wide.view(-1)[8: 8 + q.numel()].view_as(q)):
        before = wide.clone()
        with pytest.raises(RuntimeError, match="overlaps q"):
            paged_attention(q, c, st, out=over)
        assert torch.equal(wide, before)
    fused = torch.randn(T, Hq + 2, D, device=gpu, generator=g).half()
    if T > 1:
        with pytest.raises(RuntimeError, match="overlaps q"):
            paged_attention(fused[:, :Hq], c, st, out=fused.view(-1)[: q.numel()].view_as(q))
    for _ in range(3):
        mine = q.clone()
        assert paged_attention(mine, c, st, out=mine) is mine and torch.equal(mine, want)


@pytest.mark.parametrize("new", [1, 60])
def test_scores_of_any_size_in_bf16(gpu, new):
    """The same with bf16 magnitudes of 2^40, whose scores pass 2^80."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    n, D, H = 200 + new, 128, 2
    b = KvBatch(20, 16, max_requests=1, max_blocks=20, q_heads=H, kv_heads=H, head_dim=D)
    c = KvCache(20, H, D, fmt="e4m3")
    g = torch.Generator(device=gpu).manual_seed(4)
    k = ((torch.randint(0, 2, (n, H, D), device=gpu, generator=g) * 2 - 1) * 2.0 ** 40).bfloat16()
    v = torch.randn(n, H, D, device=gpu, generator=g).bfloat16()
    st = b.plan(ints([200], gpu), 200)
    c.append(k[:200], v[:200], st.slots)
    b.commit()
    st = b.plan(ints([new], gpu), new, max_new=new)
    c.append(k[200:], v[200:], st.slots)
    ask = (7 * torch.arange(new, device=gpu)) % (200 + torch.arange(new, device=gpu))
    out = paged_attention(k[ask], c, st)
    slots = st.table[0][ask // 16].long() * 16 + ask % 16
    assert torch.equal(out, c.read(slots, torch.bfloat16)["v"])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("size", [30.0, 100.0, 3000.0, 60000.0])
@pytest.mark.parametrize("Hq,H,D,block,cached,new", [
    (4, 2, 128, 16, 300, 1),
    (4, 2, 128, 32, 200, 60),
    (256, 128, 64, 16, 100, 520),
])
def test_equal_scores_of_any_size(gpu, fmt, size, Hq, H, D, block, cached, new):
    """Keys and queries that are all the same: a row is the mean of its values, whose blocks have scales of their own."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    n, G = cached + new, Hq // H
    pool = n // block + 1
    b = KvBatch(pool, block, max_requests=1, max_blocks=pool, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(pool, H, D, block_tokens=block, fmt=fmt)
    g = torch.Generator(device=gpu).manual_seed(5)
    k = torch.full((n, H, D), size, dtype=torch.float16, device=gpu)
    v = torch.randn(n, H, D, device=gpu, generator=g) * torch.exp2(torch.arange(n, device=gpu) // block % 7 - 3.0)[:, None, None]
    v = v.half()
    st = b.plan(ints([cached], gpu), cached)
    c.append(k[:cached], v[:cached], st.slots)
    b.commit()
    st = b.plan(ints([new], gpu), new, max_new=new)
    c.append(k[cached:], v[cached:], st.slots)
    out = paged_attention(torch.full((new, Hq, D), size, dtype=torch.float16, device=gpu), c, st)
    at = torch.arange(n, device=gpu)
    stored = c.read(st.table[0][at // block].long() * block + at % block)["v"].double()
    seen = torch.arange(cached + 1, n + 1, device=gpu)[:, None, None].double()
    want, spread = ((x.cumsum(0)[cached:] / seen).repeat_interleave(G, 1) for x in (stored, stored.abs()))
    # roundings of the row, the weights and the values read back, 2^-11 each; the log of a scale next to a score below
    # 2^12 in powers of two, 2^-12
    assert ((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + (2.0 ** -10 + 2.0 ** -12 + 2.0 ** -15) * spread + 2.0 ** -24).all()


# ------------------------------------------------ variants, by their sizes --
@pytest.mark.parametrize("Hq,H,D,new", [
    (64, 8, 128, 32),  # 2048 rows to join: a wave for each
    (32, 4, 64, 8),    # 256: a workgroup for each
])
def test_rows_joined_from_many_parts(gpu, Hq, H, D, new):
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    n, dtype = 9000 + new, torch.bfloat16
    b = KvBatch(600, 16, max_requests=1, max_blocks=600, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(600, H, D, fmt="e4m3")
    g = torch.Generator(device=gpu).manual_seed(9)
    st = b.plan(ints([9000], gpu), 9000)
    c.append(*(torch.randn(9000, H, D, device=gpu, generator=g).to(dtype) for _ in range(2)), st.slots)
    b.commit()
    st = b.plan(ints([new], gpu), new, max_new=new)
    c.append(*(torch.randn(new, H, D, device=gpu, generator=g).to(dtype) for _ in range(2)), st.slots)
    q = torch.randn(new, Hq, D, device=gpu, generator=g).to(dtype)
    at = torch.arange(n, device=gpu)
    stored = c.read(st.table[0][at // 16].long() * 16 + at % 16, dtype)
    rows_against_formula(q, stored["k"], stored["v"], paged_attention(q, c, st), 9000, 2.0 ** -8, Hq // H)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block,D,lengths", [
    (16, 64, [1] * 300),                                  # 38400 runs' heads: a wave looks at 8 tokens
    (16, 128, [1] * 700 + [0, 333, 1, 2, 17] + [1] * 90),  # 146304: at 16
    (64, 64, [500, 1, 1, 63, 65, 1, 900]),
    (32, 64, [31, 33, 1] * 7),
])
def test_append_of_many_tokens(gpu, fmt, block, D, lengths):
    """A long call, whose waves look at several tokens each, stores what the same rows store request by request."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache

    R, H, n = len(lengths), 64, sum(lengths)
    cached = [(7 * r) % 40 for r in range(R)]
    need = [-(-(a + b) // block) for a, b in zip(cached, lengths)]
    pool = sum(need)
    g = torch.Generator(device=gpu).manual_seed(10)
    b = KvBatch(pool, block, max_requests=R, max_blocks=max(need), q_heads=H, kv_heads=H,
                free_blocks=torch.randperm(pool, generator=torch.Generator().manual_seed(1)))
    whole, single = KvCache(pool, H, D, block_tokens=block, fmt=fmt), KvCache(pool, H, D, block_tokens=block, fmt=fmt)
    for new in (cached, lengths):
        st = b.plan(ints(new, gpu), sum(new))
        st.check()
        k, v = (torch.randn(sum(new), H, D, device=gpu, generator=g) * torch.randn(sum(new), 1, 1, device=gpu, generator=g).exp2()
                for _ in range(2))
        k, v = k.half(), v.half()
        whole.append(k, v, st.slots)
        at = 0
        for m in new:
            to = at + m
            first = at  # whole blocks at a time, at most 255 tokens in a call
            while first < to:
                room = 192 - int(st.slots[first]) % block
                last = min(to, first + room)
                single.append(k[first:last], v[first:last], st.slots[first:last])
                first = last
            at = to
        b.commit()
        assert torch.equal(whole.data, single.data) and torch.equal(whole.scale, single.scale)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("H,block,D,lengths", [
    (32, 64, 64, [128]), (64, 16, 128, [1] * 100),                         # 1 token a wave, as tokens are few
    (16, 64, 64, [1] * 20 + [130, 107]), (32, 16, 128, [1] * 30 + [240]),  # 2
    (8, 32, 64, [1] * 70 + [300, 300, 355]), (4, 64, 128, [1] * 2049), (8, 16, 128, [1100]),  # 4
])
def test_append_of_some_tokens(gpu, fmt, H, block, D, lengths):
    """Calls between a few tokens and many, whose waves look at one to four: what the same rows store request by request,
    with a rotation too."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache
    from next_step_ai_amd.rotary import Rotary

    R = len(lengths)
    cached = [(7 * r) % 40 for r in range(R)]
    need = [-(-(a + b) // block) for a, b in zip(cached, lengths)]
    pool = sum(need)
    rotary = Rotary(D, 1200)
    g = torch.Generator(device=gpu).manual_seed(11)
    b = KvBatch(pool, block, max_requests=R, max_blocks=max(need), q_heads=H, kv_heads=H, head_dim=D,
                free_blocks=torch.randperm(pool, generator=torch.Generator().manual_seed(1)))
    whole, single, turned, turned1 = (KvCache(pool, H, D, block_tokens=block, fmt=fmt) for _ in range(4))
    for new in (cached, lengths):
        if sum(new) == 0:
            continue
        st = b.plan(ints(new, gpu), sum(new))
        st.check()
        k, v = ((torch.randn(sum(new), H, D, device=gpu, generator=g) * torch.randn(sum(new), 1, 1, device=gpu, generator=g).exp2())
                .bfloat16() for _ in range(2))
        whole.append(k, v, st.slots)
        turned.append_rotated(k, v, st.slots, st.positions, rotary)
        at = 0
        for m in new:
            first = at
            while first < at + m:  # whole blocks at a time, few tokens in a call
                last = min(at + m, first + 64 - int(st.slots[first]) % block)
                part = slice(first, last)
                single.append(k[part], v[part], st.slots[part])
                turned1.append_rotated(k[part], v[part], st.slots[part], st.positions[part], rotary)
                first = last
            at += m
        b.commit()
        for x, y in ((whole, single), (turned, turned1)):
            assert torch.equal(x.data, y.data) and torch.equal(x.scale, y.scale)


@pytest.mark.parametrize("fmt,Hq,H,D", [("e4m3", 32, 8, 128), ("int8", 16, 1, 64)])
def test_weights_of_single_tokens_are_not_rounded_in_bf16(gpu, fmt, Hq, H, D):
    """Streamed rows are the bf16 roundings of numbers within 2^-14 of the weights (fp32 scores up to 64 and sums) of the
    formula: one rounding, and where a weight's to fp16 would add 2^-11 none."""
    from next_step_ai_amd.kv_cache import KvBatch, KvCache, paged_attention

    lengths, dtype = [700, 61, 1, 2500], torch.bfloat16
    b = KvBatch(300, 16, max_requests=4, max_blocks=200, q_heads=Hq, kv_heads=H, head_dim=D)
    c = KvCache(300, H, D, fmt=fmt)
    g = torch.Generator(device=gpu).manual_seed(11)
    st = b.plan(ints(lengths, gpu), sum(lengths))
    c.append(*(torch.randn(sum(lengths), H, D, device=gpu, generator=g).to(dtype) for _ in range(2)), st.slots)
    b.commit()
    st = b.plan(ints([1] * 4, gpu), 4, max_new=1)
    c.append(*(torch.randn(4, H, D, device=gpu, generator=g).to(dtype) for _ in range(2)), st.slots)
    q = torch.randn(4, Hq, D, device=gpu, generator=g).to(dtype)
    out = paged_attention(q, c, st)
    for r, n in enumerate(lengths):
        at = torch.arange(n + 1, device=gpu)
        slots = st.table[r][at // 16].long() * 16 + at % 16
        scale = c.scale[slots // 16].double()
        # values as the codes say: what is read back, rounded to fp16, over the scale is near a code of 4 bits or a whole number
        back = c.read(slots)
        exact = []
        for i, x in ((0, "k"), (1, "v")):
            y = back[x].double() / scale[:, :, i, None]
            exact.append((torch.round(y) if fmt == "int8" else y.float().to(torch.float8_e4m3fn).double()) * scale[:, :, i, None])
        for h in range(Hq):
            k, v = (x[:, h * H // Hq].contiguous() for x in exact)
            p = torch.softmax(k @ q[r, h].double() * D ** -0.5, 0)
            want, near = p @ v, 2.0 ** -14 * (p @ v.abs()) + 2.0 ** -24
            assert ((want - near).to(dtype) <= out[r, h]).all() and (out[r, h] <= (want + near).to(dtype)).all()
