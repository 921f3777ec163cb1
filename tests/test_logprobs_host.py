"""Token log probabilities on the host: what the call refuses before any device work, its sizes, injected faults."""
import ctypes
import os

import pytest
import torch

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
    x = dict(logits=MEM, stride=1000, dtype=0, rows=2, vocab=1000, tokens=MEM, top=3, logprob=MEM, entropy=MEM, top_ids=MEM,
             top_logprobs=MEM, ws=MEM, ws_bytes=1 << 40)
    x.update(kw)
    return L.nsmlp_token_logprobs(x["logits"], x["stride"], x["dtype"], x["rows"], x["vocab"], x["tokens"], x["top"], x["logprob"],
                                  x["entropy"], x["top_ids"], x["top_logprobs"], x["ws"], x["ws_bytes"], None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(rows=-1), EINVAL, b"rows"), (dict(rows=(1 << 24) + 1), EINVAL, b"rows"), (dict(vocab=0), EINVAL, b"vocabulary"),
    (dict(vocab=(1 << 30) + 1), EINVAL, b"vocabulary"), (dict(dtype=3), EINVAL, b"dtype"), (dict(top=-1), EINVAL, b"top"),
    (dict(top=65), EINVAL, b"top"), (dict(vocab=2), EINVAL, b"top"), (dict(tokens=None), EINVAL, b"go together"),
    (dict(logprob=None), EINVAL, b"go together"), (dict(top_ids=None), EINVAL, b"top_ids"),
    (dict(top_logprobs=None), EINVAL, b"top_ids"), (dict(logits=None), EINVAL, b"logits"), (dict(logits=MEM + 1), EINVAL, b"aligned"),
    (dict(dtype=2, logits=MEM + 2), EINVAL, b"aligned"), (dict(vocab=100000, ws=None), ENOSPC, b"workspace"),
    (dict(vocab=100000, ws_bytes=1000), ENOSPC, b"workspace"), (dict(vocab=100000, ws=MEM + 16), EINVAL, b"256-byte")])
def test_refusals(L, kw, code, text):
    assert call(L, **kw) == code and text in L.nsmlp_last_error(), L.nsmlp_last_error()


def test_more_rows_than_a_launch_has_threads(L):
    """256 threads have a row: 2^24 rows would be 2^32 threads."""
    assert call(L, rows=1 << 24) == EINVAL and b"rows" in L.nsmlp_last_error()
    with_ws = L.nsmlp_token_logprobs_workspace_bytes
    assert with_ws(1 << 24, 1000, 0, 3) == 0 and b"rows" in L.nsmlp_last_error()
    # one fewer is taken as far as its other arguments go
    assert call(L, rows=(1 << 24) - 1, logits=None) == EINVAL and b"logits" in L.nsmlp_last_error()


def test_no_rows(L):
    assert call(L, rows=0) == 0 and call(L, rows=0, logits=None, ws=None, ws_bytes=0) == 0


def test_sizes(L):
    """A workspace only where a row is shared out: few rows and many logits."""
    size = L.nsmlp_token_logprobs_workspace_bytes
    assert size(1, 1000, 0, 5) == 0 and size(4096, 128256, 1, 20) == 0 and size(0, 128256, 1, 20) == 0
    assert 0 < size(1, 128256, 0, 20) < 1 << 20 and size(1, 128256, 2, 20) >= size(1, 128256, 2, 0) > 0
    assert size(1, 128256, 0, 65) == 0 and size(1, 10, 0, 11) == 0 and size(1, 128256, 7, 1) == 0


@pytest.mark.parametrize("vocab", [5000, 10000, 16000, 20001, 32000, 50257, 100003, 128256, 262144])
@pytest.mark.parametrize("dtype,size", [(0, 2), (1, 2), (2, 4)])
def test_shares_of_whole_batches(L, vocab, dtype, size):
    """The workgroups of a row (16 + 8 top bytes of workspace for each) have 16 steps of 64 vectors, or a multiple."""
    bytes_of = L.nsmlp_token_logprobs_workspace_bytes
    steps = -(-vocab * size // 1024)
    for rows in (1, 2, 7, 61, 100, 205, 230, 256, 300, 511, 700, 1023, 1024, 5000):
        more = bytes_of(rows, vocab, dtype, 1) - bytes_of(rows, vocab, dtype, 0)
        shares = max(1, more // (8 * rows))
        assert shares == 1 or rows * shares < 1024 + rows
        assert shares <= 32 and any(-(-steps // each) == shares for each in range(16, steps + 17, 16)), (rows, shares)


@pytest.mark.parametrize("kind,code", [("hip", EIO), ("nospc", ENOSPC), ("nodev", ENODEV)])
def test_fault_point(L, kind, code):
    from next_step_ai_amd import _lib

    with _lib.injected_faults(f"token_logprobs={kind}:1"):
        assert call(L, rows=0) == code and b"nsmlp_token_logprobs" in L.nsmlp_last_error()
        assert call(L, rows=0) == 0


def test_python_wants_a_gpu():
    from next_step_ai_amd.lm_head import token_logprobs

    with pytest.raises(RuntimeError, match="GPU"):
        token_logprobs(torch.zeros(2, 5))


@pytest.mark.parametrize("rows,vocab,top,text", [
    (1 << 24, 10, 1, "16777216 rows"), (1 << 31, 1, 0, "2147483648 rows"), ((1 << 32) + 1, 1, 0, "4294967297 rows"),
    (1, (1 << 30) + 1, 0, "of 1073741825 logits"), (1, (1 << 32) + 5, 0, "of 4294967301 logits"), (2, 0, 0, "of 0 logits"),
    (1, 1000, 65, "top 65"), (1, 10, 11, "top 11"), (1, 100, -1, "top -1"), (1, 100, 1 << 32, "top 4294967296")])
def test_sizes_refused_before_anything_is_made(rows, vocab, top, text):
    """Each by what is wrong with it."""
    from next_step_ai_amd.lm_head import _check_sizes

    with pytest.raises(RuntimeError, match=text):
        _check_sizes(rows, vocab, top)


def test_sizes_taken():
    from next_step_ai_amd.lm_head import _check_sizes

    for sizes in ((0, 5, 5), ((1 << 24) - 1, 1 << 30, 64), (1, 1, 1), (3, 64, 64), (3, 1000, 0)):
        _check_sizes(*sizes)
