"""How long sums are dealt out to shares, on CPU: a share without a term would never be finished."""
import ctypes
import random

import pytest

from hp_rms_norm_b200 import capi


def piece(rows, hidden, vocab, k):
    out = (ctypes.c_int64 * 4)()
    status = capi.load().hprn_test_loss_backward_piece(rows, hidden, vocab, k, out)
    assert status == capi.OK, capi.load().hprn_last_error()
    return tuple(out)


def check(rows, hidden, vocab):
    count, cols, _, _ = piece(rows, hidden, vocab, 0)
    total = 0
    for k in {0, count - 1}:
        _, cols_k, stages, shares = piece(rows, hidden, vocab, k)
        assert 1 <= cols_k <= cols and stages == -(-cols_k // 64)
        assert 1 <= shares <= stages, (rows, hidden, vocab, k, stages, shares)
        total = k * cols + cols_k
    assert total == vocab
    return count


# Vocabularies of many pieces whose last one is a few columns long.
@pytest.mark.parametrize("case", [(62100, 8, 69642), (63130, 10, 61441), (39915, 16, 452707),
                                  (27990, 224, 738832), (12134, 1070, 3786829), (24576, 256, 462464),
                                  (44032, 64, 159000)], ids=str)
def test_short_last_piece(case):
    count = check(*case)
    assert piece(*case, count - 1)[1] <= 128  # what makes the case one


def test_every_share_has_a_term():
    rng = random.Random(5)
    spread = lambda hi: int(round(hi ** rng.random()))
    many = sum(check(spread(1 << 17), spread(8192), spread(1 << 22)) > 1 for _ in range(20000))
    assert many > 1000


def test_refusals():
    out = (ctypes.c_int64 * 4)()
    for bad in ((8, 8, 8, 1), (8, 8, 8, -1), (-1, 8, 8, 0), (8, 8, 0, 0)):
        assert capi.load().hprn_test_loss_backward_piece(*bad, out) == capi.ERR_INVALID_ARGUMENT
