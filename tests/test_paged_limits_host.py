"""The sizes up to which the paged cache's calls and the verification of drafts go, as the
header states them, without a GPU: the first size beyond is refused, the last one within
is not (it goes on to ask for the device)."""
import re

import pytest

import forge_hip as fh

A = 1 << 20  # an aligned address that is never read


def cache(nSeq, nKV=1):
    return fh.ref(fh.PagedCache(1, nSeq, nKV, 32, 16, 9, 3, 1, A, A, A, A))


def calls(name, nSeq, T, nH=1):
    c = cache(nSeq)
    return {"paged_append": lambda: fh.lib.fg_paged_append(c, 0, None, None, A, A, 32, 0, T, None, None, None, 0, 0, 0),
            "paged_read": lambda: fh.lib.fg_paged_read(c, 0, A, A, 32, 0, T),
            "paged_attn": lambda: fh.lib.fg_paged_attn(c, 0, A, 2 * A, nH, 1.0, T, None, 0, 0)}[name]()


def check(over, within):
    # (1024 sequences of 1023 drafts pass the limit on drafts at the same number)
    assert over() == -1 and re.search("too many|bad dimensions", fh.last_error()), fh.last_error()
    if fh.device_count() == 0:  # (with one the call would run)
        assert within() == -4, fh.last_error()


@pytest.mark.parametrize("name", ["paged_append", "paged_read"])
@pytest.mark.parametrize("T", [1, 4])
def test_rows(name, T):
    check(lambda: calls(name, (1 << 23) // T, T), lambda: calls(name, ((1 << 23) - 1) // T, T))


@pytest.mark.parametrize("T,nH", [(1, 1), (1, 32), (7, 1), (64, 8), (8192, 32)])
def test_attention(T, nH):
    n = ((1 << 23) - 9) // (T * nH)
    check(lambda: calls("paged_attn", (1 << 23) // (T * nH) + 1, T, nH), lambda: calls("paged_attn", max(n, 1), T, nH))


def test_one_sequence_beyond():
    """32 sequences of 8192 tokens with 32 heads are one row above."""
    check(lambda: calls("paged_attn", 32, 8192, 32), lambda: calls("paged_attn", 31, 8192, 32))


@pytest.mark.parametrize("D,V", [(0, 1 << 20), (3, 128256), (1023, 32000)])
@pytest.mark.parametrize("two", [False, True])
def test_verification(D, V, two):
    chunks, rows = -(-V // 4096), D + 1 + (D if two else 0)
    n = ((1 << 23) - 1) // (chunks * rows)
    y = A if two else None
    go = lambda s: fh.lib.fg_draft_verify(A, A, A, V, y, V, A, None, A, 1.0, s, D, V)  # noqa: E731
    check(lambda: go(n + 1), lambda: go(n))
