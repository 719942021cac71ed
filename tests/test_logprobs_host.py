"""What token log probabilities refuse, without a GPU (addresses are never dereferenced)."""
import pytest

from llm_infer_rust_amd import _native

A = 0x10000


def call(rows=4, vocab=100, stride=None, dtype=0, top=2, cus=256, logits=A, ids=A, workspace=None,
         room=0):
    return _native.lib().mi355x_token_logprobs(
        logits, rows, vocab, vocab if stride is None else stride, dtype, A, top, A, A, ids, A,
        workspace, room, cus, None)


@pytest.mark.parametrize("kwargs,what", [
    (dict(rows=-1), b"shape"),
    (dict(vocab=0, top=0), b"shape"),
    (dict(vocab=(1 << 24) + 1), b"shape"),
    (dict(top=65), b"shape"),
    (dict(vocab=3, top=4), b"shape"),
    (dict(top=-1), b"shape"),
    (dict(dtype=3), b"shape"),
    (dict(cus=0), b"shape"),
    (dict(rows=1 << 31), b"shape"),
    (dict(logits=None), b"null"),
    (dict(ids=None), b"null"),
    (dict(stride=99), b"overlap"),
    (dict(logits=A + 1), b"overlap"),
    (dict(vocab=151936), b"workspace"),
    (dict(vocab=151936, workspace=A, room=64), b"workspace"),
    (dict(rows=1 << 24, vocab=8193), b"too many rows"),
    (dict(rows=1 << 26, vocab=50), b"too many rows"),
])
def test_refused(kwargs, what):
    err = call(**kwargs)
    assert err is not None and what in err


def test_no_rows():
    assert call(rows=0, logits=None) is None


def test_workspace_bytes():
    need = _native.lib().mi355x_token_logprobs_workspace_bytes
    assert need(0, 151936, 5, 256) == 0
    assert need(256, 151936, 20, 256) == 0  # a workgroup a row
    assert need(1, 100, 5, 256) == 0
    assert need(1, 151936, 5, 256) == 64 * (16 + 8 * 5)
    assert need(1, 1 << 24, 64, 256) == 64 * (16 + 8 * 64)
    assert need(1, (1 << 24) + 1, 5, 256) == -1
    assert need(1, 4, 5, 256) == -1
