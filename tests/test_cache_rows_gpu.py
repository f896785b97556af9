"""Attention over the 8-bit cache row by row: every row of every head and sequence within the bound that its own weights and values
give, so that one wrong row, or a token that one of them misses, is seen."""

import math

import pytest
import torch

from rbf_attention_b200 import ops
from test_cache_gpu import BF16, BLOCK, DEV, FP16, Pool, _ints, _randn

pytestmark = pytest.mark.gpu


def _rows(pool, q, before, new, softmax):
    """In 64 bits: the rows, and how far each (in its norm) may be off but for the output's own rounding. Weights are rounded once,
    to fp16 - 2^-11 of each - or in the block that is not complete to the cache's type where there are up to 8 query rows, so a row
    is off by at most the sum of that half step of every weight times its value's norm. Scores are sums of D products in fp32,
    off by D half steps of the sum of their magnitudes at most, and a weight by as much of it; twice that covers the rest."""
    B, Hq, T, D = q.shape
    G, gamma, half = Hq // pool.H, 1 / math.sqrt(D), torch.finfo(q.dtype).eps / 2
    out, off = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV), torch.zeros(B, Hq, T, dtype=torch.float64, device=DEV)
    for b in range(B):
        k, v = (pool.held(x, b).repeat_interleave(G, 0) for x in "kv")
        n, total = new[b], before[b] + new[b]
        if n == 0:
            continue
        x = q[b, :, :n].double()
        k_sq, x_sq = k.square().sum(-1), x.square().sum(-1)
        score = gamma * (2 * (x @ k.mT) - k_sq[:, None] - x_sq[..., None])
        size = gamma * (2 * (x.norm(dim=-1)[..., None] * k.norm(dim=-1)[:, None]) + k_sq[:, None] + x_sq[..., None])
        hidden = torch.arange(total, device=DEV) > before[b] + torch.arange(n, device=DEV)[:, None]
        w = score.masked_fill(hidden, -math.inf)
        w = torch.softmax(w, -1) if softmax else w.exp()
        unit = torch.full((total,), 2.0**-11, dtype=torch.float64, device=DEV)
        unit[total // BLOCK * BLOCK:] = max(half, 2.0**-11)
        out[b, :, :n] = w @ v
        off[b, :, :n] = (w * (unit + 2 * D * 2.0**-24 * (size + 1)) * v.norm(dim=-1)[:, None]).sum(-1)
    return out, off


def _check_rows(got, want, off, tiny=0.0):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).norm(dim=-1)
    bound = half * want.norm(dim=-1) + (1 + half) * off + tiny * math.sqrt(got.shape[-1])
    assert (err <= bound).all(), ((err / bound).max().item(), (err > bound).nonzero()[:5].tolist())


@pytest.mark.parametrize("softmax", [True, False])
@pytest.mark.parametrize("G,T", [(1, 1), (8, 1), (3, 2), (4, 4), (1, 30), (2, 33)])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (64, FP16), (128, BF16), (80, FP16), (24, BF16)])
@pytest.mark.parametrize("long", [False, True])
def test_every_row(long, D, dtype, G, T, softmax):
    std = 1.0 if softmax else 0.5
    before, new = [0, 15, 16, 255, 256, 700, 989], [T, T, max(T - 1, 0), T, T, T // 2, T]
    pool = Pool(7, 2, D, 1280, dtype, seed=T, long=long)
    most = max(before)
    pool.append(_randn(7, 2, most, D, dtype=dtype, seed=1, std=std), _randn(7, 2, most, D, dtype=dtype, seed=2), before)
    start = pool.lengths.clone()
    pool.append(_randn(7, 2, T, D, dtype=dtype, seed=3, std=std), _randn(7, 2, T, D, dtype=dtype, seed=4), new)
    q = _randn(7, 2 * G, T, D, dtype=dtype, seed=5, std=std)
    got = ops.cache_attention(q, pool.pages, pool.table, start, _ints(new), softmax=softmax)
    _check_rows(got, *_rows(pool, q, before, new, softmax))
    for b in range(7):
        assert not got[b, :, new[b]:].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,N,T", [(1, 1, 20000, 1), (1, 2, 9000, 12), (24, 3, 700, 1), (200, 2, 90, 2), (3, 4, 2100, 70)])
def test_every_row_of_shared_work(B, H, N, T, D):
    """Sequences of any length whose blocks several warps share."""
    g = torch.Generator().manual_seed(N)
    total = [N] + [int(torch.randint(T, N + 1, (1,), generator=g)) for _ in range(B - 1)]
    pool = Pool(B, H, D, N, FP16, seed=B)
    pool.append(_randn(B, H, N, D, dtype=FP16, seed=6), _randn(B, H, N, D, dtype=FP16, seed=7), total)
    before = [n - T for n in total]
    # the last T tokens' rows are what the cache holds when they are the newest, also of the incomplete block
    q = _randn(B, H, T, D, dtype=FP16, seed=8)
    _check_rows(ops.cache_attention(q, pool.pages, pool.table, _ints(before)), *_rows(pool, q, before, [T] * B, True))


@pytest.mark.parametrize("size,tiny", [(1e-31, 0.0), (1e-35, 2.0**-126)])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 1), (64, 10)])
@pytest.mark.parametrize("long", [False, True])
def test_blocks_held_as_zeros(long, D, T, size, tiny):
    """Keys and values whose complete blocks are below what is held, with an incomplete block of theirs behind them: value scales
    of zero, then tiny values. (Below 2^-126 fp32 numbers may be zeros.)"""
    pool = Pool(2, 1, D, 512, BF16, long=long)
    k, v = _randn(2, 1, 300, D, seed=9), _randn(2, 1, 300, D, seed=10)
    pool.append(k * (size * 1e-2), v * size)
    kk, vv = ops.cache_read(pool.pages, pool.table, pool.lengths, D, BF16, 300)
    assert not kk[:, :, :288].any() and not vv[:, :, :288].any()
    for b in range(2):
        assert torch.equal(kk[b, :, 288:], pool.k[b][:, 288:]) and torch.equal(vv[b, :, 288:], pool.v[b][:, 288:])
    q = _randn(2, 1, T, D, seed=11)
    got = ops.cache_attention(q, pool.pages, pool.table, _ints([300 - T] * 2))
    want, off = _rows(pool, q, [300 - T] * 2, [T] * 2, True)
    assert (want.abs().amax((1, 2, 3)) > 0).all()
    _check_rows(got, want, off, tiny)


@pytest.mark.parametrize("D,T", [(64, 1), (128, 6), (64, 30)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_an_infinite_key_in_the_incomplete_block(dtype, D, T):
    """Rows that see it are NaN, or have what they had without it where its product with the query makes it infinitely far."""
    pools = [Pool(1, 2, D, 256, dtype) for _ in range(2)]
    k, v = _randn(1, 2, 60, D, dtype=dtype, seed=12), _randn(1, 2, 60, D, dtype=dtype, seed=13)
    q = _randn(1, 2, T, D, dtype=dtype, seed=14)
    outs = []
    for pool, at in zip(pools, (math.inf, None)):
        k[0, :, 57, 5] = at if at is not None else 0.0
        if at is None:
            k[0, :, 57] = 200.0             # so far that its weight is zero
        pool.append(k, v)
        outs.append(ops.cache_attention(q, pool.pages, pool.table, _ints([60 - T])))
    got, without = outs
    nan = got.isnan().all(-1)
    assert (nan | got.isfinite().all(-1)).all()
    seen = torch.arange(60 - T, 60, device=DEV) >= 57
    assert not nan[:, :, ~seen].any()
    toward = (q[..., 5] >= 0) & seen
    assert torch.equal(nan, toward)
    want, off = _rows(pools[1], q, [60 - T], [T], True)
    _check_rows(torch.where(nan[..., None], without, got), want, off)
