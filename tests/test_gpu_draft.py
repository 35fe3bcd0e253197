"""Verification of drafted tokens on the device (fg_draft_verify) against the plain
64-bit form of oracle/paged_ref.py, token by token."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def run(fh, logits, draft_logits, draft, u, temperature, drafted=None, pad=0, pad_draft=0):
    nSeq, D1, V = logits.shape
    D = D1 - 1
    up = fh.DeviceArray.from_numpy

    def rows(x, extra):
        wide = np.full((x.shape[0] * x.shape[1], V + extra), np.nan, np.float32)
        wide[:, :V] = x.reshape(-1, V)
        return up(wide)
    x, y = rows(logits, pad), rows(draft_logits, pad_draft) if draft_logits is not None else None
    d, du = up(np.ascontiguousarray(draft, np.int32)) if D else None, up(u) if u is not None else None
    n = up(np.array(drafted, np.int32)) if drafted is not None else None
    token, count = up(np.full((nSeq, D1), -9, np.int32)), up(np.full(nSeq, -9, np.int32))
    fh.call("draft_verify", token, count, x, V + pad, y, V + pad_draft, d, n, du, temperature, nSeq, D, V)
    return token.numpy(), count.numpy()


def compare(got, logits, draft_logits, draft, u, temperature, drafted=None):
    token, count = got
    for s in range(len(logits)):
        want = ref.verify(logits[s], None if draft_logits is None else draft_logits[s], draft[s], u[s] if u is not None else None,
                          temperature, len(draft[s]) if drafted is None else drafted[s])
        assert count[s] == want[1] and (token[s] == want[0]).all(), (s, token[s], want)


def case(rng, nSeq, D, V, noise=0.5):
    logits = (rng.standard_normal((nSeq, D + 1, V)) * 2).astype(np.float32)
    draft_logits = (logits[:, :D] + rng.standard_normal((nSeq, D, V)) * noise).astype(np.float32)
    draft = np.zeros((nSeq, D), np.int32)
    for s in range(nSeq):
        for t in range(D):
            draft[s, t] = ref.draw(ref.softmax(draft_logits[s, t], 1.0), rng.random())
    return logits, draft_logits, draft, rng.random((nSeq, D + 1)).astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 31, 64, 257, 1000, 4096, 4099, 32000])
@pytest.mark.parametrize("nSeq,D,pad", [(1, 0, 0), (3, 1, 1), (2, 4, 0), (9, 7, 2)])
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_verify(fh, V, nSeq, D, pad, temperature):
    rng = np.random.default_rng(V + D)
    logits, draft_logits, draft, u = case(rng, nSeq, D, V)
    compare(run(fh, logits, draft_logits, draft, u, temperature, pad=pad, pad_draft=2 * pad), logits, draft_logits, draft, u, temperature)
    compare(run(fh, logits, None, draft, u, temperature, pad=pad), logits, None, draft, u, temperature)


@pytest.mark.parametrize("V", [1, 33, 1000, 32000, 50001])
@pytest.mark.parametrize("nSeq,D", [(1, 0), (4, 3), (2, 12)])
def test_greedy(fh, V, nSeq, D):
    """Temperature 0: ties go to the lowest token, and neither draft_logits nor u is read."""
    rng = np.random.default_rng(V + D)
    logits = np.round(rng.standard_normal((nSeq, D + 1, V)) * 2).astype(np.float32)
    draft = np.array([[ref.best(logits[s, t]) if rng.random() < 0.8 else rng.integers(0, V) for t in range(D)] for s in range(nSeq)], np.int32)
    draft = draft.reshape(nSeq, D)
    compare(run(fh, logits, None, draft, None, 0.0), logits, None, draft, None, 0.0)


def test_long_vocabulary(fh):
    rng = np.random.default_rng(8)
    logits, draft_logits, draft, u = case(rng, 3, 3, 128256)
    for y in (draft_logits, None):
        compare(run(fh, logits, y, draft, u, 1.0), logits, y, draft, u, 1.0)


@pytest.mark.parametrize("V", [262145, 700001])
def test_more_chunks_than_lanes(fh, V):
    """A lane adds up more than one of a row's chunks, whose greatest logits differ; a masked one, and one that is no number."""
    rng = np.random.default_rng(V)
    logits, draft_logits, draft, u = case(rng, 3, 2, V)
    logits[:, :, 262144:] += 8
    logits[1, :, 4096:8192] = -np.inf
    for y in (draft_logits, None):
        compare(run(fh, logits, y, draft, u, 1.0), logits, y, draft, u, 1.0)
    logits[2, 0, V - 1] = np.nan
    got = run(fh, logits, draft_logits, draft, u, 1.0)
    compare(got, logits, draft_logits, draft, u, 1.0)
    assert got[1][2] == 1 and got[0][2, 0] == -1
    compare(run(fh, logits, None, draft, None, 0.0), logits, None, draft, None, 0.0)


@pytest.mark.parametrize("nSeq,D,V", [(2, 40, 64), (1, 1023, 8), (300, 2, 4500), (20, 1, 9000), (70, 1, 20000)])
def test_many_rows(fh, nSeq, D, V):
    """Long drafts, most of which stand, and more sequences than there are units: every share of a row that a thread may have."""
    rng = np.random.default_rng(nSeq + D)
    logits, draft_logits, _, u = case(rng, nSeq, D, V, noise=0.05)
    draft = np.array([[ref.draw(ref.softmax(draft_logits[s, t], 1.0), rng.random()) for t in range(D)] for s in range(nSeq)], np.int32)
    u[:, :D] *= 0.9
    got = run(fh, logits, draft_logits, draft, u, 1.0)
    compare(got, logits, draft_logits, draft, u, 1.0)
    compare(run(fh, logits, None, draft, u, 1.0), logits, None, draft, u, 1.0)
    assert D < 40 or got[1].max() > 20


def test_own_numbers_of_drafts(fh):
    rng = np.random.default_rng(4)
    logits, draft_logits, draft, u = case(rng, 8, 5, 500, noise=0.05)
    drafted = [5, 0, -1, 3, 9, 1, -2147483648, 2]
    got = run(fh, logits, draft_logits, draft, u, 1.0, drafted)
    compare(got, logits, draft_logits, draft, u, 1.0, drafted)
    assert got[1][2] == 0 and (got[0][2] == -1).all() and got[1][1] == 1
    draft = np.array([[ref.best(logits[s, t]) for t in range(5)] for s in range(8)], np.int32)
    got = run(fh, logits, None, draft, None, 0.0, drafted)
    compare(got, logits, None, draft, None, 0.0, drafted)
    assert got[1].tolist() == [6, 1, 0, 4, 6, 2, 0, 3]


@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_masked_tokens_and_no_numbers(fh, temperature):
    """Logits of -inf have no probability; a row with NaN, an infinite logit or nothing left ends the sequence with -1."""
    rng = np.random.default_rng(6)
    V, D = 300, 3
    logits, draft_logits, draft, u = case(rng, 9, D, V, noise=0.01)
    draft = np.array([[ref.best(logits[s, t]) for t in range(D)] for s in range(9)], np.int32)
    u[:, :D] *= 0.01
    mask = rng.random(logits.shape) < 0.5
    logits = np.where(mask & (np.arange(V) != np.pad(draft, ((0, 0), (0, 1)))[..., None]), -np.inf, logits).astype(np.float32)
    logits[1, 1, 7] = np.nan
    logits[2, 0] = -np.inf
    logits[3, 2, 9] = np.inf
    logits[4, 3] = np.nan
    draft_logits[5, 1, 3] = np.nan     # a draft that nothing is known of does not stand, the target's own token does
    draft_logits[6, 0] = -np.inf
    draft_logits[7] = -np.inf          # what the draft model gave all its weight
    draft_logits[7, np.arange(D), draft[7]] = 3.0
    logits[8, 1, draft[8, 1]] = -np.inf
    got = run(fh, logits, draft_logits, draft, u, temperature)
    compare(got, logits, draft_logits, draft, u, temperature)
    if temperature:
        assert [int(got[0][s, got[1][s] - 1]) for s in (1, 2, 3, 4)] == [-1, -1, -1, -1]
        assert (got[0][[5, 6], got[1][[5, 6]] - 1] >= 0).all()


def test_drafts_outside_the_vocabulary(fh):
    rng = np.random.default_rng(12)
    logits, draft_logits, draft, u = case(rng, 4, 2, 64, noise=0.01)
    draft[0, 0], draft[1, 0], draft[2, 1], draft[3, 0] = -1, 64, 2 ** 31 - 1, -2147483648
    u[:, 0] = 0.0
    for y in (draft_logits, None):
        compare(run(fh, logits, y, draft, u, 1.0), logits, y, draft, u, 1.0)
    compare(run(fh, logits, None, draft, None, 0.0), logits, None, draft, None, 0.0)


@pytest.mark.parametrize("V,pad,pad_draft", [(1000, 0, 1), (1000, 3, 2), (4099, 1, 0), (40000, 0, 3)])
def test_equal_rows(fh, V, pad, pad_draft):
    """Rows of one distribution that lie apart and are shifted, so that they are summed in other orders: a draft outside the
    vocabulary leaves no weight, and the next token is drawn from the target's own row."""
    rng = np.random.default_rng(V + pad)
    logits = (np.round(rng.standard_normal((6, 3, V)) * 16) / 8).astype(np.float32)
    draft_logits = logits[:, :2] + np.float32(4)  # exact: no bit is lost
    draft = np.array([[V, 0], [-1, 0], [V + 5, V]] * 2, np.int32)
    u = rng.random((6, 3)).astype(np.float32)
    u[0, 2], u[1, 2] = 0, np.float32(1 - 2.0 ** -24)
    got = run(fh, logits, draft_logits, draft, u, 1.0, pad=pad, pad_draft=pad_draft)
    assert (got[1] == 1).all()
    compare(got, logits, draft_logits, draft, u, 1.0)


def test_numbers_at_the_ends(fh):
    """u of 0 takes the first token of any weight, one of nearly 1 the last that it reaches; equal rows leave no rest and every draft stands."""
    rng = np.random.default_rng(14)
    V = 700
    logits, _, _, u = case(rng, 4, 1, V)
    logits[:, :, :5] = -np.inf
    u[0], u[1], u[2], u[3] = 0.0, 1 - 2.0 ** -24, [0.999, 0.0], [1 - 2.0 ** -24, 0.5]
    draft = np.array([[0], [0], [ref.best(logits[2, 0])], [ref.best(logits[3, 0])]], np.int32)
    compare(run(fh, logits, None, draft, u, 1.0), logits, None, draft, u, 1.0)
    same = logits[:, :1].copy()
    got = run(fh, logits, same, draft, u, 1.0)
    compare(got, logits, same, draft, u, 1.0)
    assert got[1][2] == 2 and got[1][3] == 2


def test_frequencies(fh):
    """Whatever the drafts are drawn from, the first token comes out as the target model has it: of 65536 sequences each
    token's share is within 6 standard deviations of its probability."""
    rng = np.random.default_rng(20)
    n, V = 65536, 8
    p_logits, q_logits = rng.standard_normal(V).astype(np.float32), (rng.standard_normal(V) * 1.5).astype(np.float32)
    p, q = ref.softmax(p_logits, 1.0), ref.softmax(q_logits, 1.0)
    logits, draft_logits = np.broadcast_to(p_logits, (n, 2, V)), np.broadcast_to(q_logits, (n, 1, V))
    draft = np.searchsorted(np.cumsum(q), rng.random(n)).clip(0, V - 1).astype(np.int32)[:, None]
    token, count = run(fh, logits, draft_logits, draft, rng.random((n, 2)).astype(np.float32), 1.0)
    share = np.bincount(token[:, 0], minlength=V) / n
    assert (np.abs(share - p) <= 6 * np.sqrt(p * (1 - p) / n)).all()
    accept = np.minimum(p, q).sum()
    assert abs((count == 2).mean() - accept) <= 6 * np.sqrt(accept * (1 - accept) / n)
