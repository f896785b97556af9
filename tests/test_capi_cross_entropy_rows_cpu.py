"""What the C entry for the losses of float16 logits refuses, before anything is launched."""

from rbf_attention_b200 import _lib

P = 1 << 20                        # never followed


def test_cross_entropy_rows(built_library):
    lib = _lib.load()
    good = dict(logits=P, targets=P, scale=P, loss=P, stats=P, rows=4, cols=64, ld=64, ignore=-100, stream=None)
    for change, code, word in ((dict(rows=-1), 1, "rows"), (dict(cols=0), 1, "cols"), (dict(ld=32), 1, "pitch"), (dict(logits=None), 1, "NULL"),
                               (dict(scale=None), 1, "NULL"), (dict(stats=None), 1, "NULL"), (dict(stats=P + 4), 2, "row_stats")):
        rc = lib.rbf_b200_cross_entropy_rows(*{**good, **change}.values())
        assert rc == code and word.encode() in lib.rbf_b200_last_error(), (change, rc)
    assert lib.rbf_b200_cross_entropy_rows(*{**good, "rows": 0}.values()) == 0
