"""Rotated appends and the 4-bit cache on the host: what the calls refuse
before any device work, the angles' frequencies, the oracle's own codes."""
import ctypes
import math
import os

import numpy as np
import pytest
import torch

from oracle import kv_reference as ref

EINVAL, ENOSPC, ENODEV, EIO = -22, -28, -19, -5


@pytest.fixture(scope="module")
def L():
    from next_step_ai_amd import _lib

    if not os.path.exists(_lib.LIB_PATH):
        from next_step_ai_amd import build_lib

        build_lib.build()
    yield _lib.lib()
    _lib.fault_inject(None)


KEEP = ctypes.create_string_buffer(1 << 16)
MEM = (ctypes.addressof(KEEP) + 255) // 256 * 256


def call(L, **kw):
    """nsmlp_kv_append_rotated with valid arguments but for ``kw``; no call gets as far as a launch."""
    from next_step_ai_amd import _lib

    x = dict(num_blocks=8, kv_heads=2, head_dim=64, block_tokens=16, format=_lib.NSMLP_KV_E2M1, data=MEM, scale=None,
             reach=100, rot_dim=64, interleaved=0, table=MEM, k=MEM, k_row=128, k_head=64, v=MEM, v_row=128, v_head=64, dtype=0,
             slots=MEM, positions=MEM, n=3, q=MEM, q_row=256, q_head=64, q_heads=4, q_out=MEM, o_row=256, o_head=64,
             cache=True, rotary=True)
    x.update(kw)
    c = _lib.KvCacheView(num_blocks=x["num_blocks"], kv_heads=x["kv_heads"], head_dim=x["head_dim"], block_tokens=x["block_tokens"],
                         format=x["format"], data=x["data"], scale=x["scale"])
    r = _lib.RotaryView(positions=x["reach"], head_dim=x["rot_dim"], interleaved=x["interleaved"], table=x["table"])
    return L.nsmlp_kv_append_rotated(ctypes.byref(c) if x["cache"] else None, ctypes.byref(r) if x["rotary"] else None, x["k"],
                                     x["k_row"], x["k_head"], x["v"], x["v_row"], x["v_head"], x["dtype"], x["slots"],
                                     x["positions"], x["n"], x["q"], x["q_row"], x["q_head"], x["q_heads"], x["q_out"], x["o_row"],
                                     x["o_head"], None)


@pytest.mark.parametrize("kw,text", [
    (dict(cache=False), b"cache"), (dict(rotary=False), b"rotary"), (dict(table=None), b"rotary"), (dict(table=MEM + 8), b"aligned"),
    (dict(rot_dim=128), b"head_dim"), (dict(reach=0), b"positions"), (dict(interleaved=2), b"interleaved"),
    (dict(positions=None), b"positions"), (dict(slots=None), b"slots"), (dict(k=None), b"k must"), (dict(v=None), b"v must"),
    (dict(k_row=100), b"strides"), (dict(v_head=4), b"strides"), (dict(q_row=100), b"strides"), (dict(q_head=4), b"strides"),
    (dict(q=MEM + 8), b"aligned"), (dict(q_out=None), b"q_out"), (dict(q_out=MEM + 2), b"q_out"), (dict(o_row=12), b"q_out"),
    (dict(q_heads=0), b"q_heads"), (dict(q_heads=1 << 28), b"q_heads"), (dict(o_row=512), b"in place"), (dict(dtype=2), b"dtype"),
    (dict(n=-1), b"rows"), (dict(n=(1 << 24) + 1), b"rows"), (dict(format=3), b"format"), (dict(head_dim=96), b"head_dim"),
    (dict(data=None), b"non-NULL"), (dict(data=MEM + 8), b"aligned"), (dict(format=0), b"non-NULL")])
def test_refusals(L, kw, text):
    assert call(L, **kw) == EINVAL and text in L.nsmlp_last_error(), L.nsmlp_last_error()


def test_more_rows_than_a_launch_has_threads(L):
    """In 4 bits 16 threads have a row: 2^28 rows, which the 8-bit formats take, would be 2^32 threads."""
    from next_step_ai_amd import _lib

    assert call(L, n=1 << 24, kv_heads=16, q=None) == EINVAL and b"2^27" in L.nsmlp_last_error()
    c = _lib.KvCacheView(num_blocks=8, kv_heads=16, head_dim=64, block_tokens=16, format=_lib.NSMLP_KV_E2M1, data=MEM, scale=None)
    assert L.nsmlp_kv_append(ctypes.byref(c), MEM, 1024, 64, MEM, 1024, 64, 0, MEM, 1 << 24, None) == EINVAL
    assert L.nsmlp_kv_read(ctypes.byref(c), MEM, 1 << 24, MEM, MEM, 0, None) == EINVAL and b"2^27" in L.nsmlp_last_error()


@pytest.mark.parametrize("kw", [
    dict(q_out=MEM + 4096, k=MEM + 4096), dict(q_out=MEM + 4096, v=MEM + 4096),            # the same rows
    dict(q_out=MEM + 4096, k=MEM + 4096 + 2 * (2 * 256 + 3 * 64)),                          # the last query row, the first of K
    dict(q_out=MEM + 4096, v=MEM + 4096 - 2 * (2 * 128 + 64)),                              # the last row of V, the first query row
    dict(q_out=MEM + 4096, o_row=512, k=MEM + 4096 + 2 * 192, k_row=512),                   # in every row of one projection
    dict(q_out=MEM + 4096, o_row=512, k=MEM + 4096 + 2 * 512 * 2 - 2 * 64, k_row=512),      # K's rows begin before the queries'
    dict(q_out=MEM + 4096, o_head=192, o_row=768, v=MEM + 4096 + 2 * 56, v_head=192, v_row=768),  # in every head's
    dict(q_out=MEM + 4096, o_row=0, q_heads=1, k=MEM + 4096, k_row=0, n=1)])
def test_queries_over_keys_or_values(L, kw):
    """Other workgroups read K and V while rows of q_out are written."""
    x = dict(q=MEM + 32768, k=MEM + 16384, v=MEM + 16384)
    x.update(kw)
    assert call(L, **x) == EINVAL and b"q_out overlaps k or v" in L.nsmlp_last_error(), L.nsmlp_last_error()


@pytest.mark.parametrize("kw", [
    dict(q_out=MEM + 4096 + 16), dict(q_out=MEM + 4096 + 2 * 64), dict(q_out=MEM + 4096 - 2 * (2 * 256 + 3 * 64)),
    dict(q_out=MEM + 4096 + 2 * 192, q_row=512, o_row=512), dict(q_out=MEM + 4096 + 2 * 56, q_head=128, o_head=128, q_row=512, o_row=512),
    dict(q_out=MEM + 4096 + 2 * 56, q_row=0, q_head=0), dict(q_out=MEM + 4096 + 2 * 64, q_head=-64, o_row=256),
    dict(q_out=MEM + 4096 + 2 * 320, q_row=512, o_row=520)])  # (strides without a period: as if they met)
def test_queries_over_queries(L, kw):
    x = dict(q=MEM + 4096, k=MEM + 16384, v=MEM + 16384)
    x.update(kw)
    assert call(L, **x) == EINVAL and b"q_out overlaps q:" in L.nsmlp_last_error(), L.nsmlp_last_error()


def test_nothing_to_store(L):
    assert call(L, n=0, q=None) == 0 and call(L, n=0, positions=None, slots=None, k=None, v=None, q_out=None) == 0
    assert call(L, n=0, interleaved=5) == EINVAL


@pytest.mark.parametrize("kind,code", [("hip", EIO), ("nospc", ENOSPC), ("nodev", ENODEV)])
def test_fault_point(L, kind, code):
    from next_step_ai_amd import _lib

    with _lib.injected_faults(f"kv_append_rotated={kind}:1"):
        assert call(L, n=0) == code and b"nsmlp_kv_append_rotated" in L.nsmlp_last_error()
    with _lib.injected_faults(f"kv_append={kind}"):
        assert call(L, n=0) == 0


def test_frequencies():
    from next_step_ai_amd.rotary import rotary_frequencies

    f = rotary_frequencies(128, 500000.0)
    assert f.dtype == torch.float64 and f.shape == (64,) and f[0] == 1
    assert torch.allclose(f.log(), -math.log(500000.0) * torch.arange(64, dtype=torch.float64) / 64, rtol=0, atol=1e-13)
    assert torch.equal(rotary_frequencies(128, 500000.0, {"rope_type": "default"}), f)
    assert torch.equal(rotary_frequencies(128, 500000.0, {"type": "linear", "factor": 4}), f / 4)
    s = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
         "original_max_position_embeddings": 8192}
    g = rotary_frequencies(128, 500000.0, s)
    for a, b in zip(f.tolist(), g.tolist()):
        wave = 2 * math.pi / a
        if wave < 8192 / 4:
            want = a
        elif wave > 8192:
            want = a / 8
        else:
            x = (8192 / wave - 1) / 3
            want = (1 - x) * a / 8 + x * a
        assert b == pytest.approx(want, rel=1e-14)
    assert (g == f).any() and (g == f / 8).any() and ((g < f) & (g > f / 8)).any()


@pytest.mark.parametrize("kw", [dict(base=0.0), dict(base=float("inf")), dict(scaling={"rope_type": "other", "factor": 2}),
                                dict(scaling={"rope_type": "linear", "factor": 0.5}), dict(scaling={"rope_type": "linear"}),
                                dict(scaling={"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0}),
                                dict(scaling={"rope_type": "llama3", "factor": 8, "low_freq_factor": 4, "high_freq_factor": 4,
                                              "original_max_position_embeddings": 8192})])
def test_frequencies_refused(kw):
    from next_step_ai_amd.rotary import rotary_frequencies

    with pytest.raises(RuntimeError):
        rotary_frequencies(128, **kw)


def test_configurations_with_more_than_a_scaling():
    """What stands next to it in a model's configuration is checked: other angles than asked for come out of neither."""
    from next_step_ai_amd.rotary import rotary_frequencies

    plain = rotary_frequencies(64, 500000.0)
    for kind in ("default", None):
        same = {"rope_type": kind, "rope_theta": 500000, "partial_rotary_factor": 1.0}
        assert torch.equal(rotary_frequencies(64, 500000.0, same), plain)
    for other, text in (({"rope_theta": 10000.0}, "rope_theta"), ({"partial_rotary_factor": 0.5}, "part of a head")):
        for kind in ({"rope_type": "default"}, {"rope_type": "linear", "factor": 2.0}):
            with pytest.raises(RuntimeError, match=text):
                rotary_frequencies(64, 500000.0, {**kind, **other})
    # a factor on cos and sin, which frequencies do not hold, is named
    with pytest.raises(RuntimeError, match="square"):
        rotary_frequencies(64, 500000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096})


def test_rotary_refusals():
    from next_step_ai_amd.rotary import Rotary

    for args, kw in (((96, 10), {}), ((64, 0), {}), ((64, (1 << 29) + 1), {}), ((64, 10), dict(frequencies=torch.ones(64)))):
        with pytest.raises(RuntimeError):
            Rotary(*args, **kw)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            Rotary(64, 10)


def test_overlap_of_rows():
    from next_step_ai_amd.kv_cache import _overlap

    t = torch.zeros(4096, dtype=torch.float16)
    a, b = t[:1024].view(8, 2, 64), t[1024:2048].view(8, 2, 64)
    assert not _overlap(a, b) and not _overlap(b, a) and _overlap(a, a) and _overlap(a, t[1023:2047].view(8, 2, 64))
    assert _overlap(t.as_strided((4, 2, 64), (256, 64, 1)), t.as_strided((4, 2, 64), (256, 64, 1), 128))  # (between each other's rows)


@pytest.mark.parametrize("n,row,heads,head,meets", [
    (3, 128, 2, 64, False), (3, 127, 2, 64, True), (3, 64, 2, 64, True), (3, 64, 2, 192, False), (3, 64, 2, 128, True), (1, 0, 2, 64, False),
    (3, 0, 1, 64, True), (3, 64, 1, 64, False), (1, 8, 1, 8, False), (3, 1000, 2, 500, False), (3, 1000, 2, 32, True), (0, 0, 2, 64, False)])
def test_rows_that_meet_themselves(n, row, heads, head, meets):
    from next_step_ai_amd.kv_cache import _meets_itself

    assert _meets_itself(n, row, heads, head, 64) == meets
    places = [r * row + h * head + d for r in range(n) for h in range(heads) for d in range(64)]
    assert (len(set(places)) < len(places)) <= meets


def test_codes_of_the_oracle():
    """Ties to the even code, both ends of the exponents, signs: by hand."""
    x = np.zeros((1, 64))
    x[0, :16] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.26, -0.74, 1.3, 1.7, -2.6, 3.4, -5.1, 0.24]
    x[0, 32:36] = [7, 2.0 ** -30, -1, 0.5]
    codes, scale = ref.encode4(x)
    assert scale.tolist() == [[1.0, 2.0]]
    assert codes[0, :16].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -0.5, -0.5, 1.5, 1.5, -3, 3, -6, 0]
    assert codes[0, 32:36].tolist() == [4, 0, -0.5, 0]
    for most, want in ((0.0, 2.0 ** -23), (2.0 ** -26, 2.0 ** -23), (6 * 2.0 ** -23, 2.0 ** -23), (6.01 * 2.0 ** -23, 2.0 ** -22),
                       (49152.0, 2.0 ** 13), (65504.0, 2.0 ** 13), (1e30, 2.0 ** 13)):
        codes, scale = ref.encode4(np.full((1, 32), most))
        assert scale[0, 0] == want and codes.max() * want <= 49152
