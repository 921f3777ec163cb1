"""The paged K/V cache's C entry points on the host: what they refuse before
any device work, their sizes, and injected faults."""
import ctypes
import os

import pytest

EINVAL, ENOSPC, ENODEV, EIO = -22, -28, -19, -5


@pytest.fixture(scope="module")
def L():
    from next_step_ai_amd import _lib

    if not os.path.exists(_lib.LIB_PATH):
        from next_step_ai_amd import build_lib

        build_lib.build()
    yield _lib.lib()
    _lib.fault_inject(None)


@pytest.fixture()
def args():
    """Valid arguments of every call; the memory is the host's, as no call gets as far as a launch."""
    from next_step_ai_amd import _lib

    class Args:
        pass

    a = Args()
    a.keep = ctypes.create_string_buffer(1 << 16)
    a.p = (ctypes.addressof(a.keep) + 255) // 256 * 256
    a.cache = dict(num_blocks=8, kv_heads=2, head_dim=64, block_tokens=16, format=_lib.NSMLP_KV_INT8, data=a.p, scale=a.p)
    a.batch = dict(requests=3, max_blocks=4, num_blocks=8, block_tokens=16, q_heads=4, kv_heads=2, cached=a.p, table=a.p,
                   ring=a.p, state=a.p)
    a.step = dict(total=5, max_new=0, slots=a.p, q_start=a.p, kv_len=a.p, next=a.p, info=a.p, schedule=a.p,
                  schedule_bytes=1 << 20)
    a.views = lambda: (ctypes.byref(_lib.KvCacheView(**a.cache)), ctypes.byref(_lib.KvBatchView(**a.batch)),
                       ctypes.byref(_lib.KvStepView(**a.step)))
    return a


def append(L, a, **kw):
    x = dict(k=a.p, k_row=128, k_head=64, v=a.p, v_row=128, v_head=64, dtype=0, slots=a.p, n=3)
    x.update(kw)
    return L.nsmlp_kv_append(a.views()[0], x["k"], x["k_row"], x["k_head"], x["v"], x["v_row"], x["v_head"], x["dtype"],
                             x["slots"], x["n"], None)


def read(L, a, **kw):
    x = dict(slots=a.p, n=3, k=a.p, v=a.p, dtype=0)
    x.update(kw)
    return L.nsmlp_kv_read(a.views()[0], x["slots"], x["n"], x["k"], x["v"], x["dtype"], None)


def attend(L, a, **kw):
    x = dict(q=a.p, row=256, head=64, dtype=0, scale=0.125, out=a.p, lse=None, ws=a.p, ws_bytes=1 << 40)
    x.update(kw)
    c, b, s = a.views()
    return L.nsmlp_paged_attention(c, b, s, x["q"], x["row"], x["head"], x["dtype"], x["scale"], x["out"], x["lse"], x["ws"],
                                   x["ws_bytes"], None)


@pytest.mark.parametrize("field,value,text", [
    ("head_dim", 96, b"head_dim"), ("head_dim", 0, b"head_dim"), ("block_tokens", 24, b"block_tokens"), ("format", 2, b"format"),
    ("kv_heads", 0, b"kv_heads"), ("kv_heads", 1025, b"kv_heads"), ("num_blocks", 0, b"num_blocks"),
    ("num_blocks", (1 << 26) + 1, b"num_blocks"), ("data", None, b"non-NULL"), ("scale", None, b"non-NULL")])
def test_cache_refusals(L, args, field, value, text):
    args.cache[field] = value
    for call in (append, read, attend):
        assert call(L, args) == EINVAL and text in L.nsmlp_last_error()


def test_cache_alignment_and_null(L, args):
    args.cache["data"] += 8
    assert append(L, args) == EINVAL and b"aligned" in L.nsmlp_last_error()
    assert L.nsmlp_kv_read(None, args.p, 1, args.p, args.p, 0, None) == EINVAL and b"cache" in L.nsmlp_last_error()


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(dtype=-1), dict(n=-1), dict(n=(1 << 24) + 1), dict(slots=None),
                                dict(k=None), dict(v=None)])
def test_append_and_read_refusals(L, args, kw):
    assert append(L, args, **kw) == EINVAL
    assert read(L, args, **kw) == EINVAL


@pytest.mark.parametrize("kw", [dict(k_row=129), dict(k_head=63), dict(v_row=4), dict(v_head=-4)])
def test_append_strides(L, args, kw):
    assert append(L, args, **kw) == EINVAL and b"strides" in L.nsmlp_last_error()
    assert append(L, args, n=0, **kw) == 0  # nothing to store: nothing is looked at
    assert append(L, args, k=args.p + 8) == EINVAL


@pytest.mark.parametrize("field,value", [
    ("requests", 0), ("requests", 4097), ("max_blocks", 0), ("max_blocks", (1 << 24) + 1), ("num_blocks", 0),
    ("block_tokens", 8), ("q_heads", 0), ("kv_heads", 0), ("q_heads", 2049), ("cached", None), ("table", None),
    ("ring", None), ("state", None)])
def test_batch_refusals(L, args, field, value):
    args.batch[field] = value
    _, b, s = args.views()
    assert L.nsmlp_kv_schedule_bytes(b, 5, 0) == 0
    assert L.nsmlp_kv_plan(b, args.p, s, None) == EINVAL
    assert L.nsmlp_kv_commit(b, s, None, None) == EINVAL
    assert L.nsmlp_paged_attention_workspace_bytes(b, 5, 0, 64) == 0


@pytest.mark.parametrize("field,value,code", [
    ("total", -1, EINVAL), ("total", (1 << 24) + 1, EINVAL), ("max_new", -1, EINVAL), ("slots", None, EINVAL),
    ("q_start", None, EINVAL), ("kv_len", None, EINVAL), ("next", None, EINVAL), ("info", None, EINVAL),
    ("schedule", None, EINVAL), ("schedule_bytes", 64, ENOSPC)])
def test_step_refusals(L, args, field, value, code):
    args.step[field] = value
    _, b, s = args.views()
    assert L.nsmlp_kv_plan(b, args.p, s, None) == code
    assert attend(L, args) == code
    args.step["schedule"] = args.p + 8
    assert L.nsmlp_kv_plan(b, args.p, None, None) == EINVAL
    assert L.nsmlp_kv_plan(b, None, s, None) in (EINVAL, code)


def test_table_entries_and_rows_have_limits(L, args):
    args.batch.update(requests=4096, max_blocks=1 << 24)
    assert L.nsmlp_kv_schedule_bytes(args.views()[1], 1, 0) == 0 and b"2^30" in L.nsmlp_last_error()
    args.batch.update(requests=1, max_blocks=4, q_heads=1024, kv_heads=1)
    assert L.nsmlp_kv_schedule_bytes(args.views()[1], 1 << 19, 0) == 0 and b"too many rows" in L.nsmlp_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), EINVAL), (dict(out=None), EINVAL), (dict(row=100), EINVAL), (dict(head=60), EINVAL), (dict(dtype=3), EINVAL),
    (dict(scale=0.0), EINVAL), (dict(scale=-1.0), EINVAL), (dict(scale=float("inf")), EINVAL), (dict(scale=float("nan")), EINVAL),
    (dict(ws=None), ENOSPC), (dict(ws_bytes=1000), ENOSPC)])
def test_attention_refusals(L, args, kw, code):
    assert attend(L, args, **kw) == code
    assert attend(L, args, ws=args.p + 16) == EINVAL
    args.step["total"] = 0
    if "dtype" not in kw and "scale" not in kw:
        assert attend(L, args, **kw) == 0


@pytest.mark.parametrize("change", [dict(kv_heads=1), dict(num_blocks=9), dict(block_tokens=32), dict(q_heads=5)])
def test_cache_and_batch_that_do_not_fit(L, args, change):
    args.batch.update(change)
    assert attend(L, args) == EINVAL


def test_sizes(L, args):
    """A schedule holds a unit for every request and every tile of rows; the workspace grows only with the parts."""
    for total, most in ((1, 1), (64, 1), (4096, 0), (4096, 4096), (1 << 20, 0)):
        _, b, _ = args.views()
        n = L.nsmlp_kv_schedule_bytes(b, total, most)
        assert n % 4 == 0 and n >= 32 * (args.batch["requests"] + (total * 2 // 256 if most != 1 else 0))
        ws = L.nsmlp_paged_attention_workspace_bytes(b, total, most, 128)
        assert 0 < ws < 1 << 28
        assert L.nsmlp_paged_attention_workspace_bytes(b, total, most, 96) == 0
    assert L.nsmlp_kv_schedule_bytes(args.views()[1], 0, 0) > 0


@pytest.mark.parametrize("kind,code", [("hip", EIO), ("nospc", ENOSPC), ("nodev", ENODEV)])
def test_fault_points(L, args, kind, code):
    from next_step_ai_amd import _lib

    c, b, s = args.views()
    calls = {"kv_append": lambda: append(L, args), "kv_read": lambda: read(L, args), "paged_attention": lambda: attend(L, args),
             "kv_plan": lambda: L.nsmlp_kv_plan(b, args.p, s, None), "kv_commit": lambda: L.nsmlp_kv_commit(b, s, None, None)}
    for name, call in calls.items():
        with _lib.injected_faults(f"{name}={kind}:1"):
            assert call() == code
            assert b"injected fault" in L.nsmlp_last_error() and b"nsmlp_" + name.encode() in L.nsmlp_last_error()
        with _lib.injected_faults(f"{name}x={kind}"):
            args.cache["head_dim"] = 96
            args.batch["requests"] = 0
            c2, b2, _ = args.views()
            assert {"kv_append": lambda: append(L, args), "kv_read": lambda: read(L, args),
                    "paged_attention": lambda: attend(L, args), "kv_plan": lambda: L.nsmlp_kv_plan(b2, args.p, s, None),
                    "kv_commit": lambda: L.nsmlp_kv_commit(b2, s, None, None)}[name]() == EINVAL
            args.cache["head_dim"], args.batch["requests"] = 64, 3


def test_python_wants_a_gpu():
    import torch
    from next_step_ai_amd.kv_cache import KvBatch, KvCache

    for bad in (dict(fmt="fp8"), dict(block_tokens=8)):
        with pytest.raises(RuntimeError):
            KvCache(4, 2, 64, **bad)
    for shape in ((4, 2, 80), (0, 2, 64), (4, 0, 64)):
        with pytest.raises(RuntimeError):
            KvCache(*shape)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            KvCache(4, 2, 64)
        with pytest.raises(RuntimeError):
            KvBatch(4, 16, max_requests=1, max_blocks=2, q_heads=2, kv_heads=2)
