"""The paged 8-bit cache and RBF attention over it, against the definitions in 64 bits."""

import math

import pytest
import torch

from rbf_attention_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE, BLOCK = 256, 16
BF16, FP16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


class Pool:
    """A pool with scattered pages, its table and lengths, and the tokens that were appended."""

    def __init__(self, B, H, D, tokens, dtype, seed=0, extra=3, long=False):
        self.B, self.H, self.D, self.dtype = B, H, D, dtype
        self.max_pages = -(-tokens // PAGE)
        n = B * self.max_pages + extra
        self.pages = torch.randint(0, 256, (n, H, ops.cache_page_bytes(D)), dtype=torch.uint8, device=DEV, generator=_gen(seed))
        self.table = torch.randperm(n, device=DEV, generator=_gen(seed + 1))[:B * self.max_pages].to(torch.int32)
        self.table = self.table.view(B, self.max_pages)
        if long:            # room for 8192 tokens: another kernel than for short sequences, whatever their lengths
            self.table = torch.cat([self.table, self.table.new_full((B, 32 - self.max_pages), -1)], 1)
        self.lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
        self.k = [torch.zeros(H, 0, D, dtype=dtype, device=DEV) for _ in range(B)]
        self.v = [torch.zeros(H, 0, D, dtype=dtype, device=DEV) for _ in range(B)]

    def append(self, k, v, new=None):
        ops.cache_append(self.pages, self.table, self.lengths, k, v, None if new is None else _ints(new))
        for b in range(self.B):
            n = k.shape[2] if new is None else new[b]
            self.k[b] = torch.cat([self.k[b], k[b, :, :n]], 1)
            self.v[b] = torch.cat([self.v[b], v[b, :, :n]], 1)
        if new is None:
            self.lengths += k.shape[2]
        else:
            self.lengths += _ints(new)

    def held(self, which, b):
        """The sequence's tokens as the cache holds them, fp64: whole blocks as code * scale, the rest as they came."""
        x = (self.k if which == "k" else self.v)[b].double()
        whole = x.shape[1] // BLOCK * BLOCK
        blocks = x[:, :whole].float().view(self.H, whole // BLOCK, BLOCK, self.D)
        amax = blocks.abs().amax((2, 3), keepdim=True)
        ok = amax >= 1e-30
        top = torch.full_like(amax, 127.0)
        code = torch.where(ok, torch.round(blocks * torch.where(ok, top / amax, 0 * amax)), 0 * blocks)
        scale = torch.where(ok, amax / top, 0 * amax)
        return torch.cat([(code.double() * scale.double()).reshape(self.H, whole, self.D), x[:, whole:]], 1)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _randn(*shape, dtype=BF16, std=1.0, seed=0):
    return (torch.randn(shape, device=DEV, generator=_gen(seed)) * std).to(dtype)


def _reference(pool, q, before, new, softmax):
    """Attention in 64 bits over what the cache holds."""
    B, Hq, T, D = q.shape
    G, gamma = Hq // pool.H, 1 / math.sqrt(D)
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        k, v = (pool.held(x, b).repeat_interleave(G, 0) for x in "kv")
        for i in range(new[b]):
            n = before[b] + i + 1
            x = q[b, :, i].double()
            logits = -gamma * (x[:, None] - k[:, :n]).square().sum(-1)
            w = torch.softmax(logits, -1) if softmax else logits.exp()
            out[b, :, i] = (w[:, None] @ v[:, :n])[:, 0]
    return out


def _check(got, want, dtype):
    """The output's rounding is half a step of its value. P is rounded once to fp16 (codes; relative 2^-11) or to the cache's type
    (the incomplete block), q once more to fp16 relative to its largest element: each moves a weighted mean by at most its half
    step of the values' mean magnitude. Whole-tensor norms: three half steps of the type bound all of it."""
    half = torch.finfo(dtype).eps / 2
    rel = ((got.double() - want).norm() / want.norm().clamp(min=1e-30)).item()
    assert rel <= 3 * half + 2 * 2.0**-11, rel


LENGTHS = [[1], [15, 16, 17], [255, 256, 257, 300], [1, 700, 64, 0, 513]]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128, 80, 8])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_what_was_appended_is_held(D, lengths, dtype):
    """Bit by bit: codes and scales are IEEE operations, the value is rounded once to the type."""
    pool = Pool(len(lengths), 3, D, 1024, dtype, seed=D)
    T = max(lengths)
    pool.append(_randn(pool.B, 3, T, D, dtype=dtype, seed=1), _randn(pool.B, 3, T, D, dtype=dtype, seed=2), lengths)
    k, v = ops.cache_read(pool.pages, pool.table, pool.lengths, D, dtype, T + 5)
    for b, n in enumerate(lengths):
        for got, which in ((k, "k"), (v, "v")):
            want = pool.held(which, b)
            assert torch.equal(got[b, :, :n], want.float().to(dtype)), (b, which)
            assert not got[b, :, n:].any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_portions_do_not_matter(D, dtype):
    """One call or many portions of any size: the same bytes in codes, scales and incomplete blocks."""
    B, H, N = 3, 2, 611
    k, v = _randn(B, H, N, D, dtype=dtype, seed=3), _randn(B, H, N, D, dtype=dtype, seed=4)
    whole, parts = Pool(B, H, D, 768, dtype), Pool(B, H, D, 768, dtype)
    whole.append(k, v)
    at = 0
    for T in [1, 1, 14, 1, 16, 3, 30, 200, 5, 256, 1, 40, 15, 1, 27]:
        parts.append(k[:, :, at:at + T], v[:, :, at:at + T])
        at += T
    assert at == N
    for a, b in zip(*(ops.cache_read(p.pages, p.table, p.lengths, D, dtype, N) for p in (whole, parts))):
        assert torch.equal(a, b)


def test_reading_a_range():
    pool = Pool(4, 2, 64, 1024, BF16)
    pool.append(_randn(4, 2, 900, 64, seed=5), _randn(4, 2, 900, 64, seed=6), [900, 37, 0, 256])
    k, v = ops.cache_read(pool.pages, pool.table, pool.lengths, 64, BF16, 900)
    for first in ([0, 5, 0, 250], [899, 36, 3, 255], [-4, 16, 100, 256], [433, 1000, 2**31 - 1, 2]):
        for count in (1, 7, 64):
            kk, vv = ops.cache_read(pool.pages, pool.table, pool.lengths, 64, BF16, count, first=_ints(first))
            for b, f in enumerate(first):
                f = max(f, 0)
                for got, full in ((kk, k), (vv, v)):
                    want = torch.zeros_like(got[b])
                    have = full[b, :, f:f + count]
                    want[:, :have.shape[1]] = have
                    assert torch.equal(got[b], want), (first, count, b)


@pytest.mark.parametrize("softmax", [True, False])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128, 80, 8])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("long", [False, True])
def test_single_tokens(long, D, lengths, dtype, softmax):
    std = 1.0 if softmax else 0.5
    pool = Pool(len(lengths), 2, D, 1024, dtype, seed=D, long=long)
    T = max(lengths)
    k, v = _randn(pool.B, 2, T, D, dtype=dtype, seed=7, std=std), _randn(pool.B, 2, T, D, dtype=dtype, seed=8)
    new = [min(n, 1) for n in lengths]
    before = [n - x for n, x in zip(lengths, new)]
    pool.append(k, v, before)
    last = [torch.stack([x[b, :, max(n - 1, 0)] for b, n in enumerate(lengths)])[:, :, None] for x in (k, v)]
    start = pool.lengths.clone()
    pool.append(*last, new)
    q = _randn(pool.B, 2, 1, D, dtype=dtype, seed=9, std=std)
    got = ops.cache_attention(q, pool.pages, pool.table, start, _ints(new), softmax=softmax)
    _check(got, _reference(pool, q, before, new, softmax), dtype)


@pytest.mark.parametrize("softmax", [True, False])
@pytest.mark.parametrize("G,T", [(2, 1), (4, 3), (1, 9), (8, 1), (16, 2), (3, 37), (1, 100)])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, FP16), (80, BF16)])
@pytest.mark.parametrize("long", [False, True])
def test_several_columns(long, D, dtype, G, T, softmax):
    """Heads that share keys and chunks of tokens, padded to one length, histories that end anywhere."""
    std = 1.0 if softmax else 0.5
    before, new = [0, 3, 250, 600], [T, max(T - 1, 1), T, T // 2]
    pool = Pool(4, 2, D, 768, dtype, seed=T, long=long)
    pool.append(_randn(4, 2, 600, D, dtype=dtype, seed=10, std=std), _randn(4, 2, 600, D, dtype=dtype, seed=11), before)
    start = pool.lengths.clone()
    pool.append(_randn(4, 2, T, D, dtype=dtype, seed=12, std=std), _randn(4, 2, T, D, dtype=dtype, seed=13), new)
    q = _randn(4, 2 * G, T, D, dtype=dtype, seed=14, std=std)
    got = ops.cache_attention(q, pool.pages, pool.table, start, _ints(new), softmax=softmax)
    _check(got, _reference(pool, q, before, new, softmax), dtype)
    for b in range(4):
        assert not got[b, :, new[b]:].any()


@pytest.mark.parametrize("B,H,N", [(1, 1, 20000), (1, 1, 4096), (3, 5, 2500), (1, 8, 5000), (40, 3, 330), (300, 1, 40)])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_shares_of_the_work(D, long, B, H, N):
    """Few long sequences that many warps share, many short ones of which a warp has several, all at once."""
    g = torch.Generator().manual_seed(N)
    new = [N] + [int(torch.randint(0, N + 1, (1,), generator=g)) for _ in range(B - 1)]
    pool = Pool(B, H, D, N, BF16, long=long and N <= 4096)
    pool.append(_randn(B, H, N, D, seed=15), _randn(B, H, N, D, seed=16), new)
    one = [min(n, 1) for n in new]
    before = [n - x for n, x in zip(new, one)]
    q = _randn(B, H, 1, D, seed=17)
    got = ops.cache_attention(q, pool.pages, pool.table, _ints(before), _ints(one))
    _check(got, _reference(pool, q, before, one, True), BF16)


def test_layouts_of_the_tensors():
    """The projection's layout, slices and unaligned rows; tables and lengths that are views."""
    pool = Pool(3, 4, 64, 512, BF16)
    B, H, T, D = 3, 4, 21, 64
    qkv = _randn(B, T, 3, H, D, seed=18)
    q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)
    odd = _randn(B, H, T, D + 3, seed=19)[..., 1:D + 1]
    start = pool.lengths.clone()
    pool.append(k, odd)
    want = _reference(pool, q, [0] * 3, [T] * 3, True)
    _check(ops.cache_attention(q, pool.pages, pool.table, start), want, BF16)
    wide = torch.stack([pool.table, pool.table + 1], 2)[..., 0]
    lengths = torch.stack([start, start + 9], 1)[:, 0]
    odd_q = torch.cat([q, q[..., :1]], -1)[..., :D]
    assert not wide.is_contiguous() and not lengths.is_contiguous()
    _check(ops.cache_attention(odd_q, pool.pages, wide, lengths), want, BF16)
    first = ops.cache_attention(q[:1].expand(3, H, T, D), pool.pages, pool.table[:1].expand(3, -1), start)
    assert torch.equal(first[0], first[1]) and torch.equal(first[0], first[2])


@pytest.mark.parametrize("T", [1, 12])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("long", [False, True])
def test_pages_outside_the_pool_and_lengths_beyond_the_table(long, D, T):
    """They count as absent tokens; what is in the pool behind other pages stays as it was."""
    pool = Pool(3, 2, D, 512, BF16, extra=2, long=long)
    k, v = _randn(3, 2, 300, D, seed=20), _randn(3, 2, 300, D, seed=21)
    pool.append(k, v)
    start = pool.lengths - T
    q = _randn(3, 2, T, D, seed=22)
    good = ops.cache_attention(q, pool.pages, pool.table, start)
    table = pool.table.clone()
    table[0, 0], table[1, 1] = -1, pool.pages.shape[0]
    got = ops.cache_attention(q, pool.pages, table, start)
    assert torch.equal(got[2], good[2]) and got.isfinite().all()
    for b, (lo, hi) in ((0, (256, 300)), (1, (0, 256))):
        kk, vv = (pool.held(x, b)[:, lo:hi] for x in "kv")
        for i in range(T):
            n = max(0, min(300 - T + i + 1, hi) - lo)
            w = torch.softmax(-(q[b, :, i, None].double() - kk[:, :n]).square().sum(-1) / math.sqrt(D), -1)
            _check(got[b, :, i], (w[:, None] @ vv[:, :n])[:, 0], BF16)
    table[:] = -5
    assert not ops.cache_attention(q, pool.pages, table, start).any()
    before = pool.pages.clone()
    ops.cache_append(pool.pages, table, pool.lengths, k, v)
    ops.cache_append(pool.pages, pool.table, _ints([8192, 2**31 - 1, 9000] if long else [512, 2**31 - 1, 600]), k, v)
    assert torch.equal(before, pool.pages)
    kk, vv = ops.cache_read(pool.pages, table, pool.lengths, D, BF16, 300)
    assert not kk.any() and not vv.any()
    assert ops.cache_attention(q, pool.pages, pool.table, _ints([-7, 2**31 - 1, 512])).shape == q.shape


@pytest.mark.parametrize("D", [64, 128])
def test_blocks_that_are_not_finite(D):
    """NaN and infinities stay in their block, their head, and in the rows that see them."""
    pool = Pool(2, 2, D, 256, FP16)
    k, v = _randn(2, 2, 60, D, dtype=FP16, seed=23), _randn(2, 2, 60, D, dtype=FP16, seed=24)
    v[0, 0, 55, 3] = math.inf              # incomplete block
    v[1, 1, 37, 5] = math.nan              # a whole one
    pool.append(k, v)
    q = _randn(2, 2, 30, D, dtype=FP16, seed=25)
    got = ops.cache_attention(q, pool.pages, pool.table, _ints([30, 30]))
    # token i sees 30 + i: the block of token 37 is 32 to 47, seen from row 2 on, token 55 from row 25 on
    assert got[0, 1].isfinite().all() and got[1, 0].isfinite().all()
    assert got[0, 0, :25].isfinite().all() and not got[0, 0, 25:, 3].isfinite().any()
    assert got[0, 0, 25:, 4:].isfinite().all() and got[0, 0, 25:, :3].isfinite().all()
    assert got[1, 1, :2].isfinite().all() and got[1, 1, 2:].isnan().all()
    kk, vv = ops.cache_read(pool.pages, pool.table, pool.lengths, D, FP16, 60)
    assert kk.isfinite().all() and vv[1, 1, 32:48].isnan().all() and vv[1, 1, :32].isfinite().all()
    clean = pool.v[1].clone()
    clean[1, 37, 5] = 0
    pool.v[1] = clean
    want = _reference(pool, q, [30, 30], [30, 30], True)
    _check(got[1, 1, :2], want[1, 1, :2], FP16)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 6])
def test_blocks_that_are_not_finite_and_few_rows(T, D, long):
    pool = Pool(2, 2, D, 256, FP16, long=long)
    k, v = _randn(2, 2, 60, D, dtype=FP16, seed=23), _randn(2, 2, 60, D, dtype=FP16, seed=24)
    v[0, 0, 59 - T // 2, 3] = math.inf     # incomplete block, seen by the last rows only
    v[1, 1, 37, 5] = math.nan              # a whole one, seen by all
    pool.append(k, v)
    q = _randn(2, 2, T, D, dtype=FP16, seed=25)
    got = ops.cache_attention(q, pool.pages, pool.table, _ints([60 - T, 60 - T]))
    first = T - 1 - T // 2
    assert got[0, 1].isfinite().all() and got[1, 0].isfinite().all() and got[1, 1].isnan().all()
    assert got[0, 0, :first].isfinite().all() and not got[0, 0, first:, 3].isfinite().any()
    assert got[0, 0, first:, 4:].isfinite().all() and got[0, 0, first:, :3].isfinite().all()


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [6, 12, 30, 50])
def test_a_key_that_is_not_finite_in_the_incomplete_block(T, D, dtype, bad):
    """Rows that do not see it have what they had without it."""
    pool = Pool(1, 2, D, 256, dtype)
    k, v = _randn(1, 2, 60, D, dtype=dtype, seed=27), _randn(1, 2, 60, D, dtype=dtype, seed=28)
    k[0, 1, 57, 5] = bad
    pool.append(k, v)
    q = _randn(1, 2, T, D, dtype=dtype, seed=29)
    got = ops.cache_attention(q, pool.pages, pool.table, _ints([60 - T]))
    clean = Pool(1, 2, D, 256, dtype)
    k[0, 1, 57, 5] = 0
    clean.append(k, v)
    want = _reference(clean, q, [60 - T], [T], True)
    _check(got[0, 0], want[0, 0], dtype)
    _check(got[0, 1, :-3], want[0, 1, :-3], dtype)
    if math.isnan(bad):
        assert got[0, 1, -3:].isnan().all()


def test_extreme_queries_and_keys():
    """Large and tiny queries, keys far from every query, blocks of zeros."""
    pool = Pool(4, 1, 64, 512, BF16)
    k, v = _randn(4, 1, 300, 64, seed=26), _randn(4, 1, 300, 64, seed=27)
    k[0] *= 20
    k[1, :, :200] = 0
    v[1, :, :100] = 0
    k[2] *= 2.0**-20
    v[2] *= 2.0**100
    k[3], v[3] = k[3] * 1e-33, v[3] * 1e-35
    pool.append(k, v)
    q = _randn(4, 1, 1, 64, seed=28)
    q[0] *= 30
    q[2] *= 2.0**-30
    got = ops.cache_attention(q, pool.pages, pool.table, _ints([299] * 4))
    want = _reference(pool, q, [299] * 4, [1] * 4, True)
    for b in range(3):
        _check(got[b], want[b], BF16)
    _check(ops.cache_attention(q, pool.pages, pool.table, _ints([299] * 4), softmax=False)[1:3],
           _reference(pool, q, [299] * 4, [1] * 4, False)[1:3], BF16)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_values_of_very_different_sizes(D, long):
    """Blocks whose scales jump by large powers of two either way, seen by queries that attend to the large or the small ones."""
    pool = Pool(3, 2, D, 512, BF16, long=long)
    N = 300
    k, v = _randn(3, 2, N, D, seed=60), _randn(3, 2, N, D, seed=61)
    size = torch.ones(3, 1, N, 1, device=DEV)
    size[0, 0, 32:64], size[0, 0, 64:80], size[0, 0, 200:] = 2.0**40, 2.0**-60, 2.0**90
    size[1, 0, :100], size[1, 0, 100:250], size[1, 0, 250:] = 2.0**100, 2.0**-90, 2.0**-20
    size[2, 0, ::7] = 2.0**30
    v = (v.float() * size).to(BF16)
    k[1, :, :100] *= 40                     # far from every query: weight zero
    pool.append(k, v)
    q = _randn(3, 2, 4, D, seed=62)
    got = ops.cache_attention(q, pool.pages, pool.table, _ints([N - 4] * 3))
    want = _reference(pool, q, [N - 4] * 3, [4] * 3, True)
    for b in range(3):
        scale = want[b].abs().max()
        _check(got[b].double() / scale, want[b] / scale, BF16)


def test_copied_pages():
    for layers in (None, 1, 3):
        for copies in (1, 7, 600):
            n = 3 * copies + 2
            shape = (n, 2, 2048) if layers is None else (layers, n, 2, 2048)
            pages = torch.randint(0, 256, shape, dtype=torch.uint8, device=DEV)
            order = torch.randperm(n).tolist()
            dst = order[:copies]
            src = [order[copies + i % (copies + 1)] for i in range(copies)]
            want = pages.clone()
            want.index_copy_(-3, torch.tensor(dst, device=DEV), pages.index_select(-3, torch.tensor(src, device=DEV)))
            ops.cache_copy_pages(pages, src, dst)
            assert torch.equal(pages, want)
    before = pages.clone()
    ops.cache_copy_pages(pages, [], [])
    assert torch.equal(before, pages)


def test_empty_calls():
    pool = Pool(2, 2, 64, 256, BF16)
    none = torch.empty(2, 2, 0, 64, dtype=BF16, device=DEV)
    ops.cache_append(pool.pages, pool.table, pool.lengths, none, none)
    assert ops.cache_attention(none, pool.pages, pool.table, pool.lengths).shape == none.shape
    k, v = ops.cache_read(pool.pages, pool.table, pool.lengths, 64, BF16, 0)
    assert k.shape == none.shape
    nobody = torch.empty(0, 2, 3, 64, dtype=BF16, device=DEV)
    table, lengths = pool.table[:0], pool.lengths[:0]
    ops.cache_append(pool.pages, table, lengths, nobody, nobody)
    assert ops.cache_attention(nobody, pool.pages, table, lengths).shape == nobody.shape
    no_pages = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    x = _randn(2, 2, 3, 64)
    ops.cache_append(pool.pages, no_pages, pool.lengths, x, x)
    assert not ops.cache_attention(x, pool.pages, no_pages, pool.lengths).any()
    assert not ops.cache_attention(x, pool.pages[:0], pool.table, pool.lengths).any()
    assert not ops.cache_attention(x, pool.pages, pool.table, pool.lengths, _ints([0, 0])).any()


@pytest.mark.parametrize("D,T,G", [(64, 1, 1), (128, 5, 4)])
def test_captured_and_replayed_while_the_sequences_grow(D, T, G):
    """Lengths, tables and tokens are read by the kernels: one graph serves every step."""
    steps, B, H = 40 // T, 3, 2
    pools = [Pool(B, H, D, 768, BF16, seed=1) for _ in range(2)]
    for p in pools:
        p.append(_randn(B, H, 250, D, seed=29), _randn(B, H, 250, D, seed=30), [250, 100, 7])
    q, k, v = (torch.empty(B, H * g, T, D, dtype=BF16, device=DEV) for g in (G, 1, 1))
    a, b = pools

    def step(p):
        ops.cache_append(p.pages, p.table, p.lengths, k, v)
        out = ops.cache_attention(q, p.pages, p.table, p.lengths)
        p.lengths += T
        return out

    keep = a.pages.clone(), a.lengths.clone()
    for x in (q, k, v):
        x.zero_()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(a)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(a)
    torch.cuda.synchronize()
    a.pages.copy_(keep[0])
    a.lengths.copy_(keep[1])
    for i in range(steps):
        for j, x in enumerate((q, k, v)):
            x.copy_(_randn(*x.shape, seed=100 * i + j))
        graph.replay()
        want = step(b)
        assert torch.equal(out, want), i
    assert torch.equal(a.lengths, b.lengths)


def test_two_streams_at_once():
    pools = [Pool(4, 4, 64, 2048, BF16, seed=s) for s in (1, 2)]
    qs = [_randn(4, 4, 1, 64, seed=31 + s) for s in (0, 1)]
    for s, p in enumerate(pools):
        p.append(_randn(4, 4, 2000, 64, seed=40 + s), _randn(4, 4, 2000, 64, seed=50 + s))
    alone = [ops.cache_attention(q, p.pages, p.table, p.lengths - 1) for q, p in zip(qs, pools)]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (s, q, p) in enumerate(zip(streams, qs, pools)):
            with torch.cuda.stream(s):
                outs[i].append(ops.cache_attention(q, p.pages, p.table, p.lengths - 1))
    torch.cuda.synchronize()
    for i, many in enumerate(outs):
        assert all(torch.equal(x, alone[i]) for x in many)


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GB whose last pages are used."""
    n = 2**32 // ops.cache_page_bytes(64) + 4
    pages = torch.empty(n, 1, ops.cache_page_bytes(64), dtype=torch.uint8, device=DEV)
    small = Pool(1, 1, 64, 512, BF16)
    k, v, q = _randn(1, 1, 400, 64, seed=33), _randn(1, 1, 400, 64, seed=34), _randn(1, 1, 1, 64, seed=35)
    small.append(k, v)
    table, zero = _ints([[n - 1, n - 2]]), _ints([0])
    ops.cache_append(pages, table, zero, k, v)
    assert torch.equal(ops.cache_attention(q, pages, table, _ints([399])),
                       ops.cache_attention(q, small.pages, small.table, _ints([399])))
    ops.cache_copy_pages(pages, [n - 1, n - 2], [n - 3, 0])
    assert torch.equal(ops.cache_attention(q, pages, _ints([[n - 3, 0]]), _ints([399])),
                       ops.cache_attention(q, small.pages, small.table, _ints([399])))


def test_refusals():
    pool = Pool(2, 4, 64, 256, BF16)
    x = _randn(2, 4, 3, 64)
    P, t, n = pool.pages, pool.table, pool.lengths
    append = dict(pages=P, page_table=t, lengths=n, k=x, v=x, new_lengths=_ints([1, 2]))
    attend = dict(q=x, pages=P, page_table=t, lengths=n, new_lengths=_ints([1, 2]), softmax=True)
    read = dict(pages=P, page_table=t, lengths=n, head_dim=64, dtype=BF16, count=4, first=_ints([0, 0]))
    shared = [{"pages": P[0]}, {"pages": P.float()}, {"pages": P[..., :-16]}, {"pages": P[:, :, ::2]}, {"pages": P.cpu()},
              {"page_table": t.long()}, {"page_table": t[0]}, {"page_table": t.cpu()}, {"page_table": t[:1]}, {"lengths": n.long()},
              {"lengths": n[:1]}, {"lengths": n.cpu()}, {"lengths": n[:, None]}]
    bad = {ops.cache_append: (append, [{"k": x[:, :2]}, {"v": x[:, :, :2]}, {"k": x.half()}, {"k": x.float(), "v": x.float()}, {"k": x[0]},
                                       {"k": x[..., :60], "v": x[..., :60]}, {"k": x.cpu()}, {"v": x.cpu()}, {"k": x[:1], "v": x[:1]},
                                       {"new_lengths": _ints([1])}, {"new_lengths": torch.ones(2, device=DEV)},
                                       {"new_lengths": _ints([1, 2]).cpu()}, {"k": _randn(2, 4, 3, 128), "v": _randn(2, 4, 3, 128)}]),
           ops.cache_attention: (attend, [{"q": x[:, :3]}, {"q": x.float()}, {"q": x[0]}, {"q": x[..., :60]}, {"q": x.cpu()}, {"q": x[:1]},
                                          {"new_lengths": _ints([1])}, {"q": _randn(2, 4, 3, 128)}]),
           ops.cache_read: (read, [{"head_dim": 128}, {"head_dim": 0}, {"dtype": torch.float32}, {"count": -1}, {"first": _ints([0])},
                                   {"first": torch.zeros(2, device=DEV)}])}
    for call, (good, changes) in bad.items():
        call(**good)
        for change in changes + shared:
            with pytest.raises((ValueError, RuntimeError)):
                call(**{**good, **change})
    grown = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.cache_attention(**{**attend, "q": grown})
    with torch.no_grad():
        ops.cache_attention(**{**attend, "q": grown})
    number = P.shape[0]
    for src, dst in (([0], [number]), ([number], [0]), ([-1], [0]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [0]),
                     ([2**40], [0]), ([0.5], [1])):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            ops.cache_copy_pages(P, src, dst)
    for pages in (P[0, 0], P.float(), P[:, :, ::2], P.cpu()):
        with pytest.raises((ValueError, RuntimeError)):
            ops.cache_copy_pages(pages, [0], [1])


def test_through_the_registered_operators():
    """Under a dispatch mode the operators run as registered: the same bytes and numbers."""
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    pools = [Pool(2, 2, 64, 256, FP16) for _ in range(2)]
    k, v, q = (_randn(2, 2, 21, 64, dtype=FP16, seed=s) for s in (70, 71, 72))
    outs = []
    for i, p in enumerate(pools):
        start = p.lengths.clone()

        def run():
            ops.cache_append(p.pages, p.table, start, k, v)
            ops.cache_copy_pages(p.pages, [int(p.table[0, 0])], [max(set(range(5)) - set(p.table.flatten().tolist()))])
            return ops.cache_attention(q, p.pages, p.table, start), *ops.cache_read(p.pages, p.table, start + 21, 64, FP16, 21)

        if i:
            with Mode():
                outs.append(run())
        else:
            outs.append(run())
    assert torch.equal(pools[0].pages, pools[1].pages) and all(torch.equal(a, b) for a, b in zip(*outs))
    for name in ("cache_append", "cache_copy_pages", "cache_attention", "cache_read"):
        assert any(name in s for s in seen)


def test_inference_mode_and_versions():
    p = Pool(1, 1, 64, 256, BF16)
    x = _randn(1, 1, 4, 64)
    version = p.pages._version
    ops.cache_append(p.pages, p.table, p.lengths, x, x)
    ops.cache_copy_pages(p.pages, [0], [1])
    assert p.pages._version > version
    with torch.inference_mode():
        pages = torch.zeros_like(p.pages)
        ops.cache_append(pages, p.table, p.lengths, x, x)
        ops.cache_copy_pages(pages, [0], [1])
        assert ops.cache_attention(x, pages, p.table, p.lengths).isfinite().all()


def test_another_stream_than_the_default_and_reused_memory():
    """Results of a side stream whose workspaces the allocator hands on at once."""
    p = Pool(3, 4, 64, 8192, BF16)
    k, v = _randn(3, 4, 5000, 64, seed=73), _randn(3, 4, 5000, 64, seed=74)
    p.append(k, v)
    q = _randn(3, 8, 2, 64, seed=75)
    want = ops.cache_attention(q, p.pages, p.table, p.lengths - 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        outs = []
        for _ in range(30):
            outs.append(ops.cache_attention(q, p.pages, p.table, p.lengths - 2))
            torch.full((1 << 20,), float("nan"), device=DEV)
    stream.synchronize()
    assert all(torch.equal(x, want) for x in outs)
