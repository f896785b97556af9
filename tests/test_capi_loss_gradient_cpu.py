"""What the C entries of the losses' deferred gradient refuse, before anything is launched."""

import pytest

from rbf_attention_b200 import _lib

P = 1 << 20                        # never followed
BAD_ARGUMENT, BAD_LAYOUT, OK = 1, 2, 0


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _refused(lib, rc, code, word):
    assert rc == code and word.encode() in lib.rbf_b200_last_error(), (rc, lib.rbf_b200_last_error())


def test_loss_gradient(lib):
    good = dict(logits=P, tokens=P, stats=P, factor=P, grad=P, rows=1, cols=10, ld=10, ld_out=10, ignore=-100, stream=None)
    for change, code, word in ((dict(rows=-1), BAD_ARGUMENT, "rows"), (dict(cols=0), BAD_ARGUMENT, "cols"), (dict(ld=9), BAD_ARGUMENT, "pitch"),
                               (dict(ld_out=9), BAD_ARGUMENT, "pitch"), (dict(logits=None), BAD_ARGUMENT, "NULL"),
                               (dict(tokens=None), BAD_ARGUMENT, "NULL"), (dict(stats=None), BAD_ARGUMENT, "NULL"),
                               (dict(factor=None), BAD_ARGUMENT, "NULL"), (dict(grad=None), BAD_ARGUMENT, "NULL"),
                               (dict(logits=P + 1), BAD_LAYOUT, "aligned"), (dict(stats=P + 4), BAD_LAYOUT, "aligned"),
                               (dict(grad=P + 2), BAD_LAYOUT, "alignment"), (dict(rows=2, ld_out=11), BAD_LAYOUT, "alignment")):
        _refused(lib, lib.rbf_b200_loss_gradient(*{**good, **change}.values()), code, word)
    assert lib.rbf_b200_loss_gradient(*{**good, "rows": 0}.values()) == OK


def test_policy_loss_rows(lib):
    good = dict(logits=P, tokens=P, old=P, adv=P, ref=None, weights=None, loss=P, lp=P, stats=P, ws=P, bytes=1 << 20, rows=1, cols=10,
                ld=10, ignore=-100, low=0.2, high=0.2, kl=0.0, dtype=1, stream=None)
    for change, code, word in ((dict(rows=-1), BAD_ARGUMENT, "rows"), (dict(ld=9), BAD_ARGUMENT, "pitch"), (dict(stats=None), BAD_ARGUMENT, "NULL"),
                               (dict(old=None), BAD_ARGUMENT, "NULL"), (dict(low=-1.0), BAD_ARGUMENT, "clip"),
                               (dict(stats=P + 4), BAD_LAYOUT, "row_stats")):
        _refused(lib, lib.rbf_b200_policy_loss_rows(*{**good, **change}.values()), code, word)
