"""The C entries of the cache and the policy loss without a GPU: bad arguments are refused before any CUDA work."""

import ctypes

import pytest

from rbf_attention_b200 import _lib

OK, BAD_ARGUMENT, BAD_LAYOUT, WORKSPACE, LAUNCH = 0, 1, 2, 3, 5
S = _lib.I64x3(64, 64, 64)
P = 4096                        # an address that is never followed


def _refused(lib, rc, code, word):
    assert rc == code, lib.rbf_b200_last_error()
    assert word in lib.rbf_b200_last_error().decode()


def test_page_bytes(built_library):
    lib = _lib.load()
    assert [lib.rbf_b200_cache_page_bytes(d) for d in (8, 64, 72, 128)] == [36992, 36992, 73856, 73856]
    assert lib.rbf_b200_cache_page_bytes(0) == lib.rbf_b200_cache_page_bytes(129) == 0


def _append(lib, **change):
    a = dict(pages=P, table=P, lengths=P, new=None, k=P, v=P, ks=S, vs=S, B=1, H=1, T=1, D=64, max_pages=1, num_pages=1, dtype=0,
             stream=None)
    return lib.rbf_b200_cache_append(*{**a, **change}.values())


def _read(lib, **change):
    a = dict(pages=P, table=P, lengths=P, first=None, k=P, v=P, B=1, H=1, D=64, count=4, max_pages=1, num_pages=1, dtype=0, stream=None)
    return lib.rbf_b200_cache_read(*{**a, **change}.values())


def _attend(lib, **change):
    a = dict(q=P, qs=S, pages=P, table=P, lengths=P, new=None, out=P, ws=P, bytes=0, B=1, H=1, G=1, T=1, D=64, max_pages=1,
             num_pages=1, dtype=0, softmax=1, gamma=0.1, stream=None)
    return lib.rbf_b200_cache_attention(*{**a, **change}.values())


SHARED = [(dict(D=0), BAD_ARGUMENT, "head dim"), (dict(D=136), BAD_ARGUMENT, "head dim"), (dict(D=60), BAD_ARGUMENT, "head dim"),
          (dict(H=0), BAD_ARGUMENT, "H must"), (dict(B=-1), BAD_ARGUMENT, "B,"), (dict(max_pages=-1), BAD_ARGUMENT, "max_pages"),
          (dict(dtype=2), BAD_ARGUMENT, "dtype"), (dict(pages=None), BAD_ARGUMENT, "NULL"), (dict(table=None), BAD_ARGUMENT, "NULL"),
          (dict(lengths=None), BAD_ARGUMENT, "NULL"), (dict(pages=P + 8), BAD_LAYOUT, "aligned")]


@pytest.mark.parametrize("call", [_append, _read, _attend])
@pytest.mark.parametrize("change,code,word", SHARED)
def test_a_cache_that_is_none(built_library, call, change, code, word):
    lib = _lib.load()
    _refused(lib, call(lib, **change), code, word)


@pytest.mark.parametrize("call,change,code,word", [
    (_append, dict(T=-1), BAD_ARGUMENT, "T must"), (_append, dict(k=None), BAD_ARGUMENT, "k is NULL"),
    (_append, dict(v=P + 2), BAD_LAYOUT, "v must"), (_append, dict(T=2, ks=_lib.I64x3(64, 64, 60)), BAD_LAYOUT, "stride[2]"),
    (_append, dict(B=60000, H=60000), BAD_ARGUMENT, "too large"), (_read, dict(count=-1), BAD_ARGUMENT, "count"),
    (_read, dict(k=None), BAD_ARGUMENT, "NULL"), (_read, dict(v=P + 8), BAD_LAYOUT, "aligned"),
    (_read, dict(B=60000, H=60000), BAD_ARGUMENT, "too large"), (_attend, dict(G=0), BAD_ARGUMENT, "G must"),
    (_attend, dict(T=-1), BAD_ARGUMENT, "T at least"), (_attend, dict(gamma=0.0), BAD_ARGUMENT, "gamma"),
    (_attend, dict(gamma=float("nan")), BAD_ARGUMENT, "gamma"), (_attend, dict(q=P + 4), BAD_LAYOUT, "q must"),
    (_attend, dict(out=None), BAD_LAYOUT, "out"), (_attend, dict(H=2**20, G=2**12), BAD_ARGUMENT, "too many"),
    (_attend, dict(T=2**20, H=64, max_pages=4096, num_pages=4096), BAD_ARGUMENT, "too many"),
])
def test_bad_rows_and_sizes(built_library, call, change, code, word):
    lib = _lib.load()
    _refused(lib, call(lib, **change), code, word)


def test_nothing_to_do_is_done(built_library):
    lib = _lib.load()
    for call, change in ((_append, dict(B=0)), (_append, dict(T=0)), (_append, dict(num_pages=0)), (_read, dict(B=0)), (_read, dict(count=0)),
                         (_attend, dict(B=0)), (_attend, dict(T=0))):
        assert call(lib, **change) == OK


def test_lists_of_pages(built_library):
    lib = _lib.load()

    def copy(src, dst, pages=P, layers=1, num=8, size=32):
        a = (ctypes.c_int * max(len(src), 1))(*src)
        b = (ctypes.c_int * max(len(dst), 1))(*dst)
        return lib.rbf_b200_cache_copy_pages(pages, layers, num, size, a, b, len(src), None)

    assert copy([], []) == OK and copy([1], [2], layers=0) == OK and copy([1], [2], size=0) == OK
    for src, dst, word in (([0], [8], "[0, 8)"), ([8], [0], "[0, 8)"), ([-1], [0], "[0, 8)"), ([0, 1], [2, 2], "twice"),
                           ([0, 1], [1, 2], "a source and"), ([3], [3], "a source and")):
        _refused(lib, copy(src, dst), BAD_ARGUMENT, word)
    _refused(lib, copy([0], [1], size=24), BAD_ARGUMENT, "multiple of 16")
    _refused(lib, copy([0], [1], pages=None), BAD_ARGUMENT, "NULL")
    _refused(lib, copy([0], [1], pages=P + 8), BAD_LAYOUT, "aligned")
    assert lib.rbf_b200_cache_copy_pages(P, 1, 8, 32, None, None, 1, None) == BAD_ARGUMENT


def test_logits(built_library):
    lib = _lib.load()
    probs = dict(logits=P, tokens=P, lp=P, rows=1, cols=10, ld=10, ignore=-100, dtype=0, stream=None)
    loss = dict(logits=P, tokens=P, old=P, adv=P, ref=None, weights=None, loss=P, lp=P, grad=P, ws=P, bytes=1 << 20, rows=1, cols=10,
                ld=10, ld_out=10, ignore=-100, low=0.2, high=0.2, kl=0.0, dtype=0, stream=None)
    for change, code, word in ((dict(rows=-1), BAD_ARGUMENT, "rows"), (dict(cols=0), BAD_ARGUMENT, "cols"), (dict(ld=9), BAD_ARGUMENT, "pitch"),
                               (dict(dtype=3), BAD_ARGUMENT, "dtype"), (dict(tokens=None), BAD_ARGUMENT, "NULL"),
                               (dict(logits=P + 1), BAD_LAYOUT, "aligned")):
        _refused(lib, lib.rbf_b200_token_log_probs(*{**probs, **change}.values()), code, word)
        _refused(lib, lib.rbf_b200_policy_loss(*{**loss, **change}.values()), code, word)
    for change, code, word in ((dict(old=None), BAD_ARGUMENT, "NULL"), (dict(loss=None), BAD_ARGUMENT, "NULL"), (dict(low=-1.0), BAD_ARGUMENT, "clip"),
                               (dict(high=float("nan")), BAD_ARGUMENT, "clip"), (dict(ld_out=9), BAD_ARGUMENT, "pitch"),
                               (dict(grad=P + 2), BAD_LAYOUT, "alignment"), (dict(rows=2, ld_out=11), BAD_LAYOUT, "alignment")):
        _refused(lib, lib.rbf_b200_policy_loss(*{**loss, **change}.values()), code, word)
    assert lib.rbf_b200_token_log_probs(*{**probs, "rows": 0}.values()) == OK
