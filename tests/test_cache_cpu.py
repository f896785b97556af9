"""The cache's bookkeeping of pages, without a GPU: the operators that move bytes are played by indexing."""

import random

import pytest
import torch

from rbf_attention_b200 import cache as cache_module
from rbf_attention_b200 import ops
from rbf_attention_b200.cache import PAGE_TOKENS, PagedCache


@pytest.fixture
def copies(monkeypatch):
    """Copies as they were asked for; the pages really move."""
    seen = []

    def copy(pages, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        seen.append(list(zip(src, dst)))
        pages[:, dst] = pages[:, src].clone()

    monkeypatch.setattr(cache_module.ops, "cache_copy_pages", copy)
    return seen


def _cache(sequences=4, length=1000, pages=None, layers=2):
    return PagedCache(layers, 2, 64, sequences, length, pages, device="cpu")


def _step(c, new, sequences=None):
    c.begin(new, sequences)
    c.end()


def _check(c):
    """Host lists, reference counts, free pages and the device's tensors agree."""
    users = [0] * c.num_pages
    for s in range(c.max_sequences):
        pages = c._held[s]
        assert len(pages) >= -(-c.length(s) // PAGE_TOKENS)
        assert c.page_table[s].tolist() == pages + [-1] * (c.page_table.shape[1] - len(pages))
        assert c.lengths[s] == c.length(s)
        for p in pages:
            users[p] += 1
    assert users == c._users
    assert sorted(c._free) == [p for p, n in enumerate(users) if n == 0]


def test_pages_come_with_the_tokens(copies):
    c = _cache()
    assert c.num_pages == 16 and c.free_pages == 16 and c.pages.shape == (2, 16, 2, ops.cache_page_bytes(64))
    _step(c, [1, 256, 257, 0])
    assert [len(h) for h in c._held] == [1, 1, 2, 0] and c.free_pages == 12
    _check(c)
    _step(c, 255)
    assert [len(h) for h in c._held] == [1, 2, 2, 1]
    _step(c, 1)
    assert [len(h) for h in c._held] == [2, 2, 3, 1]
    _step(c, [3], [2])
    assert [c.length(s) for s in range(4)] == [257, 512, 516, 256]
    _check(c)
    c.free([1, 2])
    assert c.free_pages == 16 - 3 and c.length(2) == 0
    _check(c)
    assert not copies


def test_a_batch_of_some_sequences(copies):
    c = _cache()
    _step(c, [5, 9], [3, 1])
    c.begin(2, [1, 3])
    assert c.positions.tolist() == [9, 5] and c.counts == [2, 2]
    c.end()
    assert c.lengths.tolist() == [0, 11, 0, 7]
    _check(c)


def test_forks_share_full_pages_and_copy_the_last(copies):
    c = _cache(5)
    _step(c, [600], [0])
    c.pages[:, c._held[0]] = torch.arange(3, dtype=torch.uint8)[:, None, None]
    c.fork(0, [1, 2, 4])
    _check(c)
    assert c.free_pages == 20 - 3 and c._held[4] == c._held[0] and c.length(4) == 600
    _step(c, 1, [1, 2])                                     # two of the four write: both get copies
    assert len(copies) == 1 and len(copies[0]) == 2
    assert c._held[1][:2] == c._held[0][:2] and len({h[2] for h in (c._held[0], c._held[1], c._held[2])}) == 3
    assert (c.pages[:, c._held[1][2]] == 2).all()
    _check(c)
    _step(c, 1, [0, 4])                                     # the last two: one copy, the other keeps the page
    assert len(copies[1]) == 1
    _check(c)
    c.free([0])
    assert c._held[1][:2] == c._held[2][:2]
    _check(c)
    full = _cache(2)
    _step(full, [512], [0])
    full.fork(0, [1])
    _step(full, 1)
    assert len(copies) == 2 and full._held[0][:2] == full._held[1][:2] and full._held[0][2] != full._held[1][2]


def test_compaction_keeps_the_contents(copies):
    random.seed(0)
    c = _cache(6, 2000)
    for _ in range(60):
        s = random.randrange(6)
        if random.random() < 0.3 and c.length(s):
            c.free([s])
        elif c.length(s) == 0 and random.random() < 0.5:
            source = random.choice([x for x in range(6) if x != s])
            if c.length(source):
                c.fork(source, [s])
        elif c.length(s) < 1500:
            _step(c, [random.randrange(1, 400)], [s])
        for s in range(6):
            for p in c._held[s]:
                if c._users[p] == 1:
                    c.pages[:, p] = (17 * s + p) % 251
        _check(c)
        before = [c.pages[:, h].clone() for h in c._held]
        if random.random() < 0.3:
            used = sum(1 for n in c._users if n)
            moved = c.compact()
            assert all(p < used for h in c._held for p in h) and moved <= used
            assert c.compact() == 0
            _check(c)
            for h, b in zip(c._held, before):
                assert torch.equal(c.pages[:, h], b)
    used = sum(1 for n in c._users if n)
    before = [c.pages[:, h].clone() for h in c._held]
    c.resize(used + 1)
    assert c.num_pages == used + 1 and c.free_pages == 1
    for h, b in zip(c._held, before):
        assert torch.equal(c.pages[:, h], b)
    _check(c)


def test_what_does_not_fit_changes_nothing(copies):
    c = _cache(3, 700, pages=4)
    _step(c, [300, 10, 0])
    state = ([list(h) for h in c._held], list(c._tokens), list(c._users), sorted(c._free), c.page_table.clone())

    def same():
        assert state[:4] == ([list(h) for h in c._held], c._tokens, c._users, sorted(c._free))
        assert torch.equal(state[4], c.page_table) and c._step is None
        _check(c)

    for new, sequences, error in (([0, 300, 300], None, RuntimeError), ([401, 0, 0], None, ValueError), ([1, 1], None, ValueError),
                                  ([-1, 0, 0], None, ValueError), ([1, 1], [0, 0], ValueError), ([1], [3], ValueError),
                                  ([1], [-1], ValueError)):
        with pytest.raises(error):
            c.begin(new, sequences)
        same()
    c.fork(0, [2])
    with pytest.raises(RuntimeError, match="full"):
        c.begin([214, 0, 1])                                # a copy and a new page, one is free
    c.free([2])
    same()
    for call in (lambda: c.fork(0, [1]), lambda: c.fork(0, [0]), lambda: c.fork(0, [2, 2]), lambda: c.fork(5, [2]),
                 lambda: c.free([3]), lambda: c.resize(2), lambda: c.length(3)):
        with pytest.raises(ValueError):
            call()
        same()


def test_calls_have_their_place(copies):
    c = _cache()
    for call in (lambda: c.append(0, None, None), lambda: c.attend(0, None), c.end, c.abort, lambda: c.positions, lambda: c.counts):
        with pytest.raises(RuntimeError, match="begin"):
            call()
    c.begin(3)
    for call in (lambda: c.begin(1), lambda: c.fork(0, [1]), lambda: c.free([0]), c.compact, lambda: c.resize(20)):
        with pytest.raises(RuntimeError, match="between begin"):
            call()
    bad = torch.zeros(4, 2, 3, 64)
    for q in (bad, bad.bfloat16()[..., :32], bad.bfloat16()[:, :, :2]):
        with pytest.raises(ValueError):
            c.attend(0, q)
    with pytest.raises(ValueError, match="layer"):
        c.attend(2, bad.bfloat16())
    c.abort()
    assert c.lengths.tolist() == [0] * 4 and c.length(0) == 0
    for args in ((0, 2, 64, 1, 1), (1, 2, 64, 0, 1), (1, 2, 64, 1, 0), (1, 2, 65, 1, 1), (1, 2, 136, 1, 1)):
        with pytest.raises(ValueError):
            PagedCache(*args, device="cpu")
    with pytest.raises(ValueError):
        PagedCache(1, 2, 64, 1, 1, dtype=torch.float32, device="cpu")


def test_a_step_that_has_written_is_freed_when_it_is_left(copies, monkeypatch):
    c = _cache()
    _step(c, [20, 30, 0, 0])
    monkeypatch.setattr(cache_module.ops, "cache_append", lambda *a: None)
    c.begin([1, 0, 1, 0])
    c.append(0, *[torch.zeros(4, 2, 1, 64, dtype=torch.bfloat16)] * 2)
    c.abort()
    assert [c.length(s) for s in range(4)] == [0, 30, 0, 0]
    _check(c)


def test_cpu_tensors_and_gradients_are_refused():
    pages = torch.zeros(3, 2, ops.cache_page_bytes(64), dtype=torch.uint8)
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.cache_append(pages, table, lengths, x, x), lambda: ops.cache_attention(x, pages, table, lengths),
                 lambda: ops.cache_read(pages, table, lengths, 64, torch.bfloat16, 4), lambda: ops.cache_copy_pages(pages, [0], [1]),
                 lambda: ops.token_log_probs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    leaf = x.clone().requires_grad_(True)
    for call in (lambda: ops.cache_append(pages, table, lengths, leaf, x), lambda: ops.cache_attention(leaf, pages, table, lengths),
                 lambda: ops.token_log_probs(torch.zeros(2, 3, requires_grad=True), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    row = torch.zeros(2)
    with pytest.raises(RuntimeError, match="detach"):
        ops.policy_loss(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64), row, row.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="ref_log_probs"):
        ops.policy_loss(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64), row, row, kl_weight=0.1)
    for D in (0, 4, 65, 136):
        with pytest.raises(ValueError):
            ops.cache_page_bytes(D)


def test_fake_kernels():
    pages = torch.empty(3, 2, ops.cache_page_bytes(64), dtype=torch.uint8, device="meta")
    table = torch.empty(5, 2, dtype=torch.int32, device="meta")
    lengths = torch.empty(5, dtype=torch.int32, device="meta")
    q = torch.empty(5, 6, 1, 64, dtype=torch.float16, device="meta").transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.ops.rbf_attn_b200.cache_attention(q, pages, table, lengths, None, True).shape == q.shape
    k, v = torch.ops.rbf_attn_b200.cache_read(pages, table, lengths, 64, torch.float16, 7, None)
    assert k.shape == v.shape == (5, 2, 7, 64) and k.dtype == torch.float16
    logits = torch.empty(4, 50257, dtype=torch.bfloat16, device="meta")
    t, row = torch.empty(4, dtype=torch.int64, device="meta"), torch.empty(4, device="meta")
    loss, lp, grad = torch.ops.rbf_attn_b200.policy_loss_fwd(logits, t, row, row, None, None, 0.2, 0.2, 0.0, -100, True)
    assert loss.shape == () and lp.shape == (4,) and grad.shape == logits.shape and grad.dtype == logits.dtype
    assert torch.ops.rbf_attn_b200.token_log_probs(logits, t, -100).dtype == torch.float32


def test_pages_of_a_step_that_was_left_are_not_shared(copies):
    """A step that was begun and left before anything was written has its pages back: a fork afterwards shares only held tokens,
    and the page that the sequence writes into next is its own."""
    c = _cache(3)
    _step(c, [100, 0, 0])
    c.begin([300, 0, 0])
    c.abort()
    assert len(c._held[0]) == 1 and c.free_pages == c.num_pages - 1
    _check(c)
    c.fork(0, [1])
    _step(c, [200, 200, 0])
    assert not set(c._held[0]) & set(c._held[1])
    _check(c)
