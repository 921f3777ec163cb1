"""Log probabilities of given tokens, entropies and alternatives against the formulas in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def reference(z, tokens, top):
    """Rows one by one in 64 bits; alternatives by a stable sort."""
    out = {"logprob": [], "entropy": [], "top_ids": [], "top_logprobs": []}
    for row, t in zip(z.double().cpu(), tokens.tolist()):
        m = row.max()
        e = torch.where(row == -math.inf, 0.0, (row - m).exp())
        log_l = e.sum().log()
        lp = row - m - log_l if m > -math.inf else torch.full_like(row, -math.inf)
        out["logprob"].append(lp[t] if 0 <= t < len(row) else torch.tensor(math.nan, dtype=torch.float64))
        out["entropy"].append(-(torch.where(e > 0, e / e.sum() * lp, 0.0)).sum() if m > -math.inf else torch.zeros((), dtype=torch.float64))
        ids = torch.sort(row, descending=True, stable=True).indices[:top]
        out["top_ids"].append(ids)
        out["top_logprobs"].append(lp[ids])
    return {k: torch.stack(v) for k, v in out.items()}


def check(got, want, spread):
    """An exponent d is rounded twice (2^-24 |d| each, log2 e 2^-25 |d| on top, exp2 2^-23): a weight is off by less than
    2^-22 (1 + spread) of itself, spread the largest |d| whose weight counts; sums over 2^17 logits by less than 2^-24 per
    addition of a lane (2^11 at most, in any direction: 2^-18) of themselves; log l and x / l and their difference by 2^-23
    of what they are."""
    assert torch.equal(got["top_ids"].cpu(), want["top_ids"]) and got["top_ids"].dtype == torch.int64
    slack = 2.0 ** -22 * (1 + spread) + 2.0 ** -18
    for name in ("logprob", "top_logprobs"):
        assert got[name].dtype == torch.float32
        g, w = got[name].cpu().double(), want[name]
        assert torch.equal(g.isnan(), w.isnan()) and torch.equal(g == -math.inf, w == -math.inf)
        fine = w.isfinite()
        assert ((g - w).abs()[fine] <= slack + 2.0 ** -22 * w.abs()[fine]).all(), (name, (g - w).abs()[fine].max())
    g, w = got["entropy"].cpu().double(), want["entropy"]
    assert ((g - w).abs() <= slack * (2 + w.abs()) * 2).all(), (g - w).abs().max()


def rows_of(rng, rows, vocab, dtype):
    z = rng.standard_normal((rows, vocab)) * 2
    for r in range(rows):
        z[r, rng.randint(vocab, size=min(vocab, 20))] += rng.uniform(0, 15, min(vocab, 20))
    return torch.from_numpy(z).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 7, 0), (1, 8, 8), (5, 63, 63), (4, 64, 64), (2, 511, 5),
                                            (3, 513, 64), (1, 2049, 20), (7, 5000, 20), (1, 8192, 33), (2, 8193, 1), (1, 50257, 64),
                                            (33, 4097, 40), (1, 128256, 20), (1100, 1000, 7), (1024, 777, 3)])
def test_rows(gpu, dtype, rows, vocab, top):
    """Rows that start at any address, alone and many, shorter and longer than a batch of vectors."""
    from next_step_ai_amd.lm_head import token_logprobs

    rng = np.random.RandomState(rows + vocab)
    z = rows_of(rng, rows, vocab, dtype)
    tokens = torch.from_numpy(rng.randint(-1, vocab + 1, rows))
    for offset in (0, 1, 3):
        flat = torch.full((rows * vocab + 16,), 60000.0, dtype=dtype, device=gpu)  # what is not the rows' would be seen
        mine = flat[offset: offset + rows * vocab].view(rows, vocab)
        mine.copy_(z)
        check(token_logprobs(mine, tokens.to(gpu), top=top), reference(z, tokens, top), 30)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes_and_strides(gpu, dtype):
    from next_step_ai_amd.lm_head import token_logprobs

    rng = np.random.RandomState(1)
    z = rows_of(rng, 6, 3001, dtype)
    tokens = torch.from_numpy(rng.randint(3001, size=6))
    want = reference(z, tokens, 4)
    dev = z.to(gpu)
    got = token_logprobs(dev.view(2, 3, 3001), tokens.view(2, 3).to(gpu), top=4)
    assert got["logprob"].shape == got["entropy"].shape == (2, 3) and got["top_ids"].shape == got["top_logprobs"].shape == (2, 3, 4)
    check({k: v.flatten(0, 1) for k, v in got.items()}, want, 30)
    wide = torch.full((6, 3100), 1e4, dtype=dtype, device=gpu)
    wide[:, 50:3051] = dev
    check(token_logprobs(wide[:, 50:3051], tokens.to(gpu), top=4), want, 30)
    check(token_logprobs(dev.t().contiguous().t(), tokens.to(gpu), top=4), want, 30)
    same = token_logprobs(dev[:1].expand(6, -1), tokens.to(gpu), top=4)
    assert (same["top_ids"] == same["top_ids"][0]).all()
    one = token_logprobs(dev[2], tokens[2].to(gpu), top=4)
    assert one["logprob"].shape == () and torch.equal(one["top_ids"].cpu(), want["top_ids"][2])
    none = token_logprobs(dev)
    assert set(none) == {"entropy", "top_ids", "top_logprobs"} and none["top_ids"].shape == (6, 0)
    assert token_logprobs(dev[:0], tokens[:0].to(gpu), top=2)["top_ids"].shape == (0, 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [100, 5000, 40000])
def test_order_of_equal_logits(gpu, dtype, vocab):
    """All equal, rising, falling, few values, zeros of either sign: the lower index first."""
    from next_step_ai_amd.lm_head import token_logprobs

    rng = np.random.RandomState(vocab)
    i = torch.arange(vocab, dtype=torch.float64)
    z = torch.stack([torch.zeros(vocab, dtype=torch.float64), i / vocab, -i / vocab, torch.from_numpy(rng.randint(4, size=vocab)) * 1.0,
                     torch.where(torch.from_numpy(rng.rand(vocab)) < 0.5, 0.0, -0.0), (i % 97) / 16, (i * 7919 % 1009) / 64]).to(dtype)
    tokens = torch.from_numpy(rng.randint(vocab, size=len(z)))
    for top in (1, 20, 64):
        check(token_logprobs(z.to(gpu), tokens.to(gpu), top=top), reference(z, tokens, top), 30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [300, 70000])
def test_masked_rows(gpu, dtype, vocab):
    """Logits of -inf and of the type's lowest value: most of a row, but one, and all of it."""
    from next_step_ai_amd.lm_head import token_logprobs

    rng = np.random.RandomState(3)
    low, inf = torch.finfo(dtype).min, -math.inf
    z = rows_of(rng, 8, vocab, dtype)
    hide = torch.from_numpy(rng.rand(vocab)) < 0.99
    z[0][hide], z[1][hide] = inf, low
    z[2], z[3], z[4], z[5] = inf, low, inf, low
    z[4][vocab - 1] = z[5][vocab - 1] = -3.0
    z[6][: vocab // 2], z[7][vocab // 2:] = inf, low
    tokens = torch.tensor([int((~hide).nonzero()[0]), int(hide.nonzero()[0]), 5, 5, vocab - 1, 7, 3, vocab - 2])
    got, want = token_logprobs(z.to(gpu), tokens.to(gpu), top=20), reference(z, tokens, 20)
    # far logits: their own size counts (fp32 differences)
    for name in ("logprob", "top_logprobs"):
        far = want[name] < -1000
        assert torch.allclose(got[name].cpu().double()[far], want[name][far].clamp(min=-math.inf), rtol=2.0 ** -22)
        got[name] = torch.where(far.to(gpu), 0.0, got[name])
        want[name] = torch.where(far, 0.0, want[name])
    check(got, want, 30)
    assert (got["entropy"][2] == 0) and (got["logprob"].cpu()[2] == 0 if want["logprob"][2] == 0 else True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [64, 300, 70000])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_values_that_are_not_numbers(gpu, dtype, vocab, value):
    """Such a row's numbers are NaN, its neighbours' are not; a NaN comes last in the order."""
    from next_step_ai_amd.lm_head import token_logprobs

    rng = np.random.RandomState(4)
    z = rows_of(rng, 3, vocab, dtype)
    z[1, vocab // 3] = value
    tokens = torch.tensor([1, 2, 3])
    got = {k: v.cpu() for k, v in token_logprobs(z.to(gpu), tokens.to(gpu), top=64).items()}
    for name in ("logprob", "entropy", "top_logprobs"):
        assert got[name][1].isnan().all() and not got[name][0].isnan().any() and not got[name][2].isnan().any()
    order = torch.sort(torch.nan_to_num(z[1].double(), nan=-1e300), descending=True, stable=True).indices[:64]
    assert torch.equal(got["top_ids"][1], order)
    z[1] = math.nan
    got = token_logprobs(z.to(gpu), tokens.to(gpu), top=64)
    assert got["top_ids"][1].tolist() == list(range(64)) and got["top_logprobs"][1].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits(gpu, dtype):
    """Logits of thousands: differences, not sizes, count."""
    from next_step_ai_amd.lm_head import token_logprobs

    rng = np.random.RandomState(5)
    z = torch.from_numpy(rng.randint(-60, 60, (4, 9000)) * 32.0 + np.array([[0], [30000], [-30000], [0]])).to(dtype)
    z[3] = z[3] * 30
    tokens = torch.from_numpy(rng.randint(9000, size=4))
    got, want = token_logprobs(z.to(gpu), tokens.to(gpu), top=10), reference(z, tokens, 10)
    check(got, want, 30)


def test_same_bits_every_time(gpu):
    """Whoever ends last: the same bits, with a workspace of the caller's and with the stream's; counters left at zero."""
    from next_step_ai_amd import _lib
    from next_step_ai_amd.lm_head import token_logprobs

    z = torch.randn(3, 128256, device=gpu).bfloat16()
    tokens = torch.tensor([5, 77, 128255], device=gpu)
    want = token_logprobs(z, tokens, top=20)
    n = _lib.lib().nsmlp_token_logprobs_workspace_bytes(3, 128256, 1, 20)
    ws = torch.full((n + 256,), 255, dtype=torch.uint8, device=gpu)
    ws = ws[(-ws.data_ptr()) % 256:][:n]
    _lib.call("nsmlp_workspace_init", ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    for i in range(30):
        got = token_logprobs(z, tokens, top=20, ws=ws if i % 2 else None)
        assert all(torch.equal(got[k], want[k]) for k in want)
    alone = token_logprobs(z[1:2], tokens[1:2], top=20)
    assert torch.equal(alone["top_ids"], want["top_ids"][1:2])
    assert torch.allclose(alone["logprob"], want["logprob"][1:2], rtol=1e-6, atol=1e-5)


def test_refusals(gpu):
    from next_step_ai_amd.lm_head import token_logprobs

    z = torch.zeros(2, 100, device=gpu)
    t = torch.zeros(2, dtype=torch.int64, device=gpu)
    for args, kw in (((z.double(),), {}), ((z.int(),), {}), ((z, t.int()), {}), ((z, t[:1]), {}), ((z, t.cpu()), {}), ((z, t), dict(top=65)),
                     ((z[:, :5], t), dict(top=6)), ((z, t), dict(top=-1)), ((z[:, :0], t), {}), ((z[0, 0],), {}),
                     ((torch.zeros(1, 100000, device=gpu),), dict(ws=t.view(torch.uint8))),
                     ((z, t), dict(ws=torch.zeros(8, dtype=torch.uint8)))):
        with pytest.raises(RuntimeError):
            token_logprobs(*args, **kw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 3), (3, 40), (2, 1000), (1, 70001), (300, 2000)])
def test_rows_of_one_token(gpu, dtype, rows, vocab):
    """One token has nearly all of a row: log p and the entropy to their own size, not to that of 1.

    With the others d = -12 to -20 below it (exact in fp32) and log p = -log(1 + r), r = sum e^d: a weight's
    exponent d log2 e is rounded once and its exp2 to an ulp, (20 * 1.45 + 2) 2^-24; the sums take at most 8 terms of a
    vector, 35 batches of 4 vectors, 6 joins of lanes, 3 of waves, 6 of workgroups: 60 roundings, r as it grows;
    log1p two ulps.  The entropy has x = sum e^d d next to it, with one rounding more each."""
    from next_step_ai_amd.lm_head import token_logprobs

    g = torch.Generator().manual_seed(vocab)
    z = (torch.randint(0, 33, (rows, vocab), generator=g) * 0.25 - 20.0).to(dtype)  # exact in all three
    at = torch.randint(vocab, (rows,), generator=g)
    z[torch.arange(rows), at] = 0.0
    got = token_logprobs(z.to(gpu), at.to(gpu), top=1)
    lp = z.double().log_softmax(-1)
    d = z.double()
    r = (d.exp() * (d < 0)).sum(-1)
    want = -torch.log1p(r)
    entropy = -(lp.exp() * lp).sum(-1)
    tol = (20 * 1.45 + 2 + 60 + 4) * 2.0 ** -24
    for name, w in (("logprob", want), ("entropy", torch.log1p(r) - (d.exp() * d).sum(-1) / (1 + r))):
        e = (got[name].double().cpu() - w).abs() / w.abs()
        assert float(e.max()) <= tol * (1 if name == "logprob" else 1.5), (name, float(e.max()), tol)
    assert torch.allclose(entropy, torch.log1p(r) - (d.exp() * d).sum(-1) / (1 + r), rtol=1e-9, atol=1e-13)
    assert torch.equal(got["top_ids"][:, 0].cpu(), at) and torch.equal(got["top_logprobs"][:, 0], got["logprob"])
    # several of the same: their logits are 1 each
    tied = token_logprobs(torch.zeros(2, vocab, dtype=dtype, device=gpu), torch.zeros(2, dtype=torch.int64, device=gpu))
    for name, sign in (("logprob", -1), ("entropy", 1)):
        assert torch.allclose(tied[name].double().cpu(), torch.full((2,), sign * math.log(vocab), dtype=torch.float64), rtol=2.0 ** -22, atol=0)


@pytest.mark.parametrize("rows,vocab,top", [(1, (1 << 32) + 5, 0), (1, 100, 1 << 32), (1, 100, -(1 << 32)), ((1 << 32) + 1, 1, 0)])
def test_sizes_past_32_bits(gpu, rows, vocab, top):
    """Numbers that would be small ones in 32 bits (broadcast logits: nothing is stored)."""
    from next_step_ai_amd.lm_head import token_logprobs

    z = torch.zeros(1, 1, dtype=torch.float16, device=gpu).expand(rows, vocab)
    with pytest.raises(RuntimeError, match="top"):
        token_logprobs(z, top=top)


def test_in_a_graph(gpu):
    """Captured and replayed with other logits, eager calls on the same stream between the replays."""
    from next_step_ai_amd.lm_head import token_logprobs

    z = torch.randn(2, 50257, device=gpu).half()
    tokens = torch.tensor([3, 50256], device=gpu)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        token_logprobs(z, tokens, top=5)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = token_logprobs(z, tokens, top=5)
        for seed in range(4):
            torch.manual_seed(seed)
            z.copy_(torch.randn(2, 50257, device=gpu))
            graph.replay()
            want = token_logprobs(z, tokens, top=5)
            stream.synchronize()
            assert all(torch.equal(out[k], want[k]) for k in want)


def test_alternatives_refused_before_memory_is_taken(gpu):
    """More of them than there may be: no outputs are made for them."""
    from next_step_ai_amd.lm_head import token_logprobs

    z = torch.zeros(200, 100000, dtype=torch.float16, device=gpu)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    for top in (65, 100000):
        with pytest.raises(RuntimeError, match=f"top {top}"):
            token_logprobs(z, top=top)
    # nor is a row of one broadcast logit written out
    with pytest.raises(RuntimeError, match="logits"):
        token_logprobs(z[:1, :1].expand(1, (1 << 30) + 1))
    assert torch.cuda.max_memory_allocated() == before


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [3, 300, 70000])
@pytest.mark.parametrize("top", [0, 3, 64])
def test_rows_of_nothing_but_minus_infinity(gpu, dtype, vocab, top):
    """Log probabilities of -inf, an entropy of 0, alternatives by index; and one logit among them has all of the row."""
    from next_step_ai_amd.lm_head import token_logprobs

    top = min(top, vocab)
    z = torch.full((4, vocab), -math.inf, dtype=dtype, device=gpu)
    z[1, vocab - 1] = z[3, 0] = -3.0
    tokens = torch.tensor([vocab - 1, vocab - 1, 0, vocab - 1], device=gpu)
    got = {k: v.cpu() for k, v in token_logprobs(z, tokens, top=top).items()}
    assert got["logprob"].tolist() == [-math.inf, 0.0, -math.inf, -math.inf] and got["entropy"].tolist() == [0.0] * 4
    for r, order in enumerate(([*range(vocab)], [vocab - 1, *range(vocab - 1)], [*range(vocab)], [*range(vocab)])):
        assert got["top_ids"][r].tolist() == order[:top]
        assert got["top_logprobs"][r].tolist() == ([0.0 if r % 2 else -math.inf] + [-math.inf] * (top - 1))[:top]
