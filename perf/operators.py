"""Answering from a cache and fine-tuning from rewards, as measurable cases: RBF attention over a paged 8-bit cache, writing
tokens into it, copying its pages, log-probabilities of given tokens and the clipped policy loss with its gradient.

``listed()`` are fixed cases, ``draw(rng)`` gives another one of the same ranges. ``prepare(case, seed)`` builds what a program
holds before the call, ``run(state)`` is one pass (plain torch, or the package's operators where ``own`` is set),
``work(case)`` its unavoidable bytes and operations, ``exact(case, seed)`` the outputs in 64 bits.

A page holds 256 tokens of every head: 16 blocks of 16 tokens. Per head its bytes are a header of 16 fp32 pairs (key scale, value
scale), then 18 slots of 32 * P bytes (P: the head dim rounded up to 64 or 128). Slots 0 to 15 hold the codes of complete blocks
(code + 128 as uint8, value = code * scale, scale = largest magnitude / 127): 16 * P bytes of keys ordered
[P / 64][half][8 rows][64 dims], row g of a half being token 4 * (g // 2) + 2 * half + g % 2, and 16 * P bytes of values ordered
[P / 32][8][4 token quads][4 dims][4 tokens]. Slots 16 and 17 hold the keys and values of the block that is not complete yet,
16 rows of P 16-bit numbers each."""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
PAGE, BLOCK, HEADER = 256, 16, 128
PER_PAGE = PAGE // BLOCK
TINY = 1e-30                       # blocks whose largest magnitude is below this are held as zeros
IGNORE = -100
CLIP_LOW, CLIP_HIGH, KL_WEIGHT = 0.2, 0.28, 0.04


def _attend(name, B, H, G, D, T, L, dtype, softmax=True):
    """B sequences of up to L tokens in the cache, the last T of them new; H key/value heads shared by G query heads each."""
    return {"name": name, "kind": "attend", "B": B, "H": H, "G": G, "D": D, "T": T, "L": L, "dtype": dtype, "softmax": softmax}


def listed():
    return [
        # one user, the language model of the training benchmark (8 heads of 64): the smallest step, latency counts
        _attend("decode_1x1000", 1, 8, 1, 64, 1, 1000, "bf16"),
        # a batch of users of that model, every sequence another length up to its 1024 tokens and 4 registers
        _attend("decode_64_ragged", 64, 8, 1, 64, 1, 1028, "bf16"),
        # long contexts with wide heads and keys shared by four query heads: the largest read
        _attend("decode_16x32k_shared", 16, 8, 4, 128, 1, 32768, "fp16"),
        # a chunk of a prompt on top of a cached history, the variant without a softmax denominator, an odd length
        _attend("chunk_37_no_softmax", 6, 16, 1, 64, 37, 5003, "bf16", softmax=False),
        # one new token for each of 64 sequences: a sixteenth of them complete a block
        {"name": "append_64_tokens", "kind": "append", "B": 64, "H": 8, "D": 64, "T": 1, "L": 1028, "dtype": "bf16"},
        # prompts written into the cache as a whole, their last block incomplete
        {"name": "append_8_prompts", "kind": "append", "B": 8, "H": 16, "D": 128, "T": 8190, "L": 0, "dtype": "fp16"},
        # one sequence gets its own copy of a shared page of one layer
        {"name": "copy_1_page", "kind": "pages", "layers": 1, "H": 8, "D": 64, "pages": 40, "copies": 1},
        # compaction of an 8-layer cache: a third of its pages move
        {"name": "compact_8_layers", "kind": "pages", "layers": 8, "H": 8, "D": 64, "pages": 400, "copies": 131},
        # the answers of a few samples scored under the model, logits as the projection pads them
        {"name": "log_probs_500", "kind": "log_probs", "rows": 500, "cols": 50304, "dtype": "bf16"},
        # the unpadded vocabulary in float32: rows without any alignment
        {"name": "log_probs_4111_fp32", "kind": "log_probs", "rows": 4111, "cols": 50257, "dtype": "fp32"},
        # the update on a handful of short answers, rows of an odd length
        {"name": "policy_333", "kind": "policy", "rows": 333, "cols": 50257, "dtype": "fp16"},
        # the update on 16 answers of the model's full length
        {"name": "policy_16k", "kind": "policy", "rows": 16384, "cols": 50304, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["attend"] * 6 + ["append"] * 2 + ["pages"] + ["log_probs"] + ["policy"] * 2)
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "attend":
        B, H, G = _log_int(rng, 1, 64), rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 1, 2, 3, 4, 8])
        D = rng.choice([64, 64, 64, 128, 128, 80])
        T = 1 if rng.random() < 0.6 else _log_int(rng, 2, 200)
        most = min(65536, 2**28 // (B * H * (128 if D > 64 else 64)), 2**25 // (B * H * G * T))
        case = _attend("", B, H, G, D, T, _log_int(rng, min(8, most), most), dtype, rng.random() < 0.75)
        del case["name"]
        return case
    if kind == "append":
        H, D = rng.choice([1, 4, 8, 16]), rng.choice([64, 128, 80])
        if rng.random() < 0.5:
            return {"kind": kind, "B": _log_int(rng, 1, 128), "H": H, "D": D, "T": 1, "L": _log_int(rng, 1, 2000), "dtype": dtype}
        B = _log_int(rng, 1, 16)
        return {"kind": kind, "B": B, "H": H, "D": D, "T": _log_int(rng, 2, 65536 // B), "L": 0, "dtype": dtype}
    if kind == "pages":
        layers, H, D = rng.choice([1, 4, 8]), rng.choice([2, 8, 16]), rng.choice([64, 128])
        most = max(2, 2**29 // (layers * H * _page_bytes(D)))
        pages = _log_int(rng, 2, min(400, most))
        return {"kind": kind, "layers": layers, "H": H, "D": D, "pages": pages, "copies": rng.randint(1, pages // 2)}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    cols = rng.choice([50304, 50257, 50304, _log_int(rng, 100, 130000)])
    return {"kind": kind, "rows": _log_int(rng, 16, min(8192, 2**31 // (cols * 4))), "cols": cols, "dtype": dtype}


# ------------------------------------------------------------------ the cache's geometry
def _columns(D):
    return 64 if D <= 64 else 128


def _page_bytes(D):
    return HEADER + (PER_PAGE + 2) * 32 * _columns(D)


def _lengths(case):
    """Tokens in the cache before the call, sequence by sequence: the first has the full length, the others spread below it."""
    L, T = case["L"], case["T"]
    most = max(0, L - T) if case["kind"] == "attend" else L
    return [most if b == 0 else (b * 2654435761 % 4294967296) * (most + 1) // 4294967296 for b in range(case["B"])]


def _quantise(x):
    """(..., 16, P) fp32 -> int codes as floats and the block's scale (...)."""
    amax = x.abs().amax((-2, -1))
    held = amax >= TINY
    top = torch.full_like(amax, 127.0)
    scale = torch.where(held, amax / top, torch.zeros_like(amax))
    inverse = torch.where(held, top / amax, torch.zeros_like(amax))
    return torch.round(x * inverse[..., None, None]), scale


def _pack_keys(code):
    """(..., 16, P) codes -> (..., 16 * P) bytes."""
    lead, P = code.shape[:-2], code.shape[-1]
    n = len(lead)
    x = (code + 128).to(torch.uint8).reshape(*lead, 4, 2, 2, P // 64, 64)          # quad, half, low bit, dims
    return x.permute(*range(n), n + 3, n + 1, n, n + 2, n + 4).reshape(*lead, 16 * P)


def _pack_values(code):
    lead, P = code.shape[:-2], code.shape[-1]
    n = len(lead)
    x = (code + 128).to(torch.uint8).reshape(*lead, 4, 4, P // 32, 8, 4)           # quad, token, chunk, row, dim
    return x.permute(*range(n), n + 2, n + 3, n, n + 4, n + 1).reshape(*lead, 16 * P)


def _unpack(pages, ids, D, dtype):
    """The pages ``ids`` (B, M) as (keys, values) in fp32, (B, H, M * 256, P), and their incomplete blocks (B, M, H, 16, P)."""
    P, (B, M), H = _columns(D), ids.shape, pages.shape[1]
    raw = pages[ids]                                                               # (B, M, H, bytes)
    scale = raw[..., :HEADER].contiguous().view(torch.float32).view(B, M, H, PER_PAGE, 2)
    slots = raw[..., HEADER:].reshape(B, M, H, PER_PAGE + 2, 32 * P)
    k = slots[..., :PER_PAGE, :16 * P].reshape(B, M, H, PER_PAGE, P // 64, 2, 4, 2, 64).permute(0, 2, 1, 3, 6, 5, 7, 4, 8)
    v = slots[..., :PER_PAGE, 16 * P:].reshape(B, M, H, PER_PAGE, P // 32, 8, 4, 4, 4).permute(0, 2, 1, 3, 6, 8, 4, 5, 7)
    both = []
    for codes, s in ((k, scale[..., 0]), (v, scale[..., 1])):
        codes = codes.reshape(B, H, M, PER_PAGE, BLOCK, P).float() - 128.0
        both.append((codes * s.permute(0, 2, 1, 3)[..., None, None]).reshape(B, H, M * PAGE, P))
    tails = [slots[..., PER_PAGE + i, :].contiguous().view(dtype).view(B, M, H, BLOCK, P).float() for i in (0, 1)]
    return *both, *tails


def _held(pages, table, total, first_page, M, D, dtype):
    """Keys and values of the M pages from page ``first_page`` (B,) on, fp32 (B, H, M * 256, D), zeros from token ``total`` (B,)
    on, and the tokens' positions (B, M * 256)."""
    B = table.shape[0]
    column = first_page[:, None] + torch.arange(M, device=table.device)
    ids = table.long().gather(1, column.clamp(max=table.shape[1] - 1))
    k, v, tk, tv = _unpack(pages, ids, D, dtype)
    pos = first_page[:, None] * PAGE + torch.arange(M * PAGE, device=table.device)
    last = total // BLOCK                                                          # the incomplete block
    at = (last // PER_PAGE - first_page).clamp(0, M - 1)
    row = torch.arange(B, device=table.device)
    inside = (pos < total[:, None])[:, None, :, None]
    in_tail = (pos >= (last * BLOCK)[:, None])[:, None, :, None]
    out = []
    for x, tail in ((k, tk), (v, tv)):
        t = tail[row, at].repeat(1, 1, M * PER_PAGE, 1)
        out.append(torch.where(inside, torch.where(in_tail, t, x), torch.zeros_like(x))[..., :D])
    return *out, pos


# ------------------------------------------------------------------ states
def _cache(case, g, before, total, values_std):
    """Pages that hold the first ``before`` tokens of each sequence, in pages scattered over the pool."""
    B, H, D, P = case["B"], case["H"], case["D"], _columns(case["D"])
    dtype = DTYPES[case["dtype"]]
    M = max(1, -(-max(total) // PAGE)) + 1
    pages = torch.zeros(B * M + 3, H, _page_bytes(D), dtype=torch.uint8, device=DEVICE)
    table = torch.randperm(B * M + 3, generator=g, device=DEVICE)[:B * M].view(B, M).to(torch.int32)
    for b, n in enumerate(before):
        if n == 0:
            continue
        m = -(-n // PAGE)
        spread = torch.exp(0.3 * torch.randn(H, m * PAGE, 1, generator=g, device=DEVICE))
        page = torch.zeros(H, m, _page_bytes(D), dtype=torch.uint8, device=DEVICE)
        slots = page[..., HEADER:].view(H, m, PER_PAGE + 2, 32 * P)
        scales = page[..., :HEADER].view(torch.float32).view(H, m, PER_PAGE, 2)
        for i, pack in ((0, _pack_keys), (1, _pack_values)):
            x = torch.randn(H, m * PAGE, D, generator=g, device=DEVICE) * values_std
            x = torch.nn.functional.pad((x * spread if i == 0 else x).to(dtype), (0, P - D)).view(H, m, PER_PAGE, BLOCK, P)
            code, scale = _quantise(x.float())
            slots[:, :, :PER_PAGE, i * 16 * P:(i + 1) * 16 * P] = pack(code)
            scales[..., i] = scale
            if n % BLOCK:
                last = n // BLOCK
                slots[:, last // PER_PAGE, PER_PAGE + i] = x[:, last // PER_PAGE, last % PER_PAGE].reshape(H, -1).view(torch.uint8)
        pages[table[b, :m].long()] = page.transpose(0, 1)
    return pages, table


def _logits(case, g):
    rows, cols = case["rows"], case["cols"]
    x = torch.empty(rows, cols, dtype=DTYPES[case["dtype"]], device=DEVICE)
    for r in range(0, rows, 1024):
        part = torch.randn(min(1024, rows - r), cols, generator=g, device=DEVICE) * 2.5
        if cols == 50304:
            part[:, 50257:] = -math.inf                                            # the padding of the vocabulary projection
        x[r:r + 1024] = part.to(x.dtype)
    tokens = torch.randint(0, min(cols, 50257), (rows,), generator=g, device=DEVICE)
    # half of the tokens are what the model finds likely, as sampled answers are; a tenth of the rows are prompt or padding
    likely = torch.rand(rows, generator=g, device=DEVICE) < 0.5
    tokens = torch.where(likely, x.argmax(-1), tokens)
    tokens[torch.rand(rows, generator=g, device=DEVICE) < 0.1] = IGNORE
    tokens[0] = 1
    return x, tokens


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = case["kind"]
    if kind in ("attend", "append"):
        before = _lengths(case)
        std = 1.0 if case.get("softmax", True) else 0.5
        T, D, dtype = case["T"], case["D"], DTYPES[case["dtype"]]
        total = [n + T for n in before]
        pages, table = _cache(case, g, total if kind == "attend" else before, total, std)
        state = {"kind": kind, "pages": pages, "table": table, "D": D, "dtype": dtype,
                 "lengths": torch.tensor(before, dtype=torch.int32, device=DEVICE)}
        if kind == "attend":
            q = torch.randn(case["B"], case["H"] * case["G"], T, D, generator=g, device=DEVICE) * std
            return state | {"q": q.to(dtype), "softmax": case["softmax"]}
        k, v = (torch.randn(case["B"], T, case["H"], D, generator=g, device=DEVICE).to(dtype).transpose(1, 2) for _ in range(2))
        first = [n // BLOCK * BLOCK for n in before]
        return state | {"k": k, "v": v, "first": torch.tensor(first, dtype=torch.int32, device=DEVICE),
                        "count": BLOCK if T == 1 else T,
                        "total": torch.tensor(total, dtype=torch.int32, device=DEVICE)}
    if kind == "pages":
        size = (case["layers"], case["pages"], case["H"], _page_bytes(case["D"]))
        pages = torch.randint(0, 256, size, generator=g, device=DEVICE, dtype=torch.uint8)
        order = torch.randperm(case["pages"], generator=g, device=DEVICE).tolist()
        return {"kind": kind, "pages": pages, "src": order[:case["copies"]], "dst": order[case["copies"]:2 * case["copies"]]}
    logits, tokens = _logits(case, g)
    state = {"kind": kind, "logits": logits, "tokens": tokens}
    if kind == "policy":
        rows = case["rows"]
        logp = _plain_log_probs(state)
        old = logp + 0.2 * torch.randn(rows, generator=g, device=DEVICE)
        ref = logp + 0.3 * torch.randn(rows, generator=g, device=DEVICE)
        adv = torch.randn(rows, generator=g, device=DEVICE)
        state |= {"old": old, "ref": ref, "adv": adv, "logits": logits.requires_grad_(True)}
    return state


# ------------------------------------------------------------------ plain forms
def _plain_attend(s):
    q, D = s["q"].float(), s["D"]
    B, Hq, T, _ = q.shape
    lengths = s["lengths"].long()
    M = s["table"].shape[1]
    k, v, pos = _held(s["pages"], s["table"], lengths + T, torch.zeros_like(lengths), M, D, s["dtype"])
    H = k.shape[1]
    q = q.reshape(B, H, Hq // H * T, D)
    gamma = 1.0 / math.sqrt(D)
    hidden = pos[:, None, :] > (lengths[:, None] + torch.arange(T, device=q.device))[:, :, None]        # (B, T, tokens)
    hidden = hidden.repeat(1, Hq // H, 1)[:, None]
    logits = 2.0 * gamma * (q @ k.mT) - gamma * k.square().sum(-1)[:, :, None]
    if s["softmax"]:
        logits = torch.where(hidden, -math.inf, logits)
        p = torch.exp(logits - logits.amax(-1, keepdim=True))
        out = (p @ v) / p.sum(-1, keepdim=True)
    else:
        logits = logits - gamma * q.square().sum(-1, keepdim=True)
        out = torch.where(hidden, 0.0, torch.exp(logits)) @ v
    return out.reshape(B, Hq, T, D).to(s["q"].dtype)


def _plain_append(s):
    pages, table, lengths, D, dtype = s["pages"], s["table"].long(), s["lengths"].long(), s["D"], s["dtype"]
    B, H, T, _ = s["k"].shape
    P = _columns(D)
    blocks = (T + BLOCK - 2) // BLOCK + 1                  # blocks that the new tokens can touch
    base = lengths // BLOCK
    pos = base[:, None] * BLOCK + torch.arange(blocks * BLOCK, device=table.device)
    at = pos - lengths[:, None]                            # index of the new token, negative for the incomplete block's
    block = base[:, None] + torch.arange(blocks, device=table.device)
    page = table.gather(1, block // PER_PAGE)              # (B, blocks)
    slot = block % PER_PAGE
    complete = ((block + 1) * BLOCK <= lengths[:, None] + T)[..., None, None]
    page_now = table.gather(1, (base // PER_PAGE)[:, None])[:, 0]
    end = lengths + T
    last = (end // BLOCK - base).clamp(max=blocks - 1)     # the incomplete block afterwards, if there is one
    page_then = table.gather(1, (end // BLOCK // PER_PAGE)[:, None])[:, 0]
    row = torch.arange(B, device=table.device)
    new_tail = ((at >= 0) & (at < T)).view(B, blocks, BLOCK)[row, last] & (end // BLOCK - base < blocks)[:, None]
    slots = pages[..., HEADER:].view(pages.shape[0], H, PER_PAGE + 2, 32 * P)
    scales = pages[..., :HEADER].view(torch.float32).view(pages.shape[0], H, PER_PAGE, 2)
    for i, (x, pack) in enumerate(((s["k"], _pack_keys), (s["v"], _pack_values))):
        x = torch.nn.functional.pad(x, (0, P - D))
        tail = slots[page_now, :, PER_PAGE + i].view(dtype).view(B, H, BLOCK, P).repeat(1, 1, blocks, 1)
        fresh = x.gather(2, at.clamp(0, T - 1)[:, None, :, None].expand(B, H, blocks * BLOCK, P))
        x = torch.where((at < 0)[:, None, :, None], tail, fresh).view(B, H, blocks, BLOCK, P)
        code, scale = _quantise(x.float())
        code, scale = pack(code).transpose(1, 2), scale.transpose(1, 2)            # (B, blocks, H, bytes), (B, blocks, H)
        old = slots[page, :, slot, i * 16 * P:(i + 1) * 16 * P]
        slots[page, :, slot, i * 16 * P:(i + 1) * 16 * P] = torch.where(complete, code, old)
        scales[page, :, slot, i] = torch.where(complete[..., 0], scale, scales[page, :, slot, i])
        old = slots[page_then, :, PER_PAGE + i].view(dtype).view(B, H, BLOCK, P)
        kept = torch.where(new_tail[:, None, :, None], x[row, :, last], old)
        slots[page_then, :, PER_PAGE + i] = kept.reshape(B, H, BLOCK * P).view(torch.uint8)
    # read back
    first = s["first"].long()
    M = 1 if s["count"] <= BLOCK else -(-s["count"] // PAGE)
    k, v, pos = _held(pages, s["table"], end, first // PAGE, M, D, dtype)
    want = (first - first // PAGE * PAGE)[:, None] + torch.arange(s["count"], device=table.device)
    want = want[:, None, :, None].expand(B, H, s["count"], D)
    return k.gather(2, want).to(dtype), v.gather(2, want).to(dtype)


def _plain_pages(s):
    index = torch.tensor([s["src"], s["dst"]], device=s["pages"].device)
    s["pages"][:, index[1]] = s["pages"][:, index[0]]
    return s["pages"]


def _plain_log_probs(s):
    x, t = s["logits"].detach().float(), s["tokens"]
    counted = t != IGNORE
    top = x.amax(-1, keepdim=True)
    lse = torch.log(torch.exp(x - top).sum(-1)) + top[:, 0]
    return torch.where(counted, x.gather(1, t.clamp(min=0)[:, None])[:, 0] - lse, 0.0)


def _plain_policy(s):
    x, t = s["logits"].detach().float(), s["tokens"]
    counted = t != IGNORE
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    target = t.clamp(min=0)[:, None]
    logp = torch.where(counted, (x.gather(1, target) - top - torch.log(total))[:, 0], 0.0)
    ratio = torch.exp(logp - s["old"])
    plain, clipped = ratio * s["adv"], ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * s["adv"]
    gap = s["ref"] - logp
    away = torch.exp(gap)
    weight = counted.float() / counted.sum()
    loss = (weight * (KL_WEIGHT * (away - gap - 1.0) - torch.minimum(plain, clipped))).sum()
    slope = weight * (KL_WEIGHT * (1.0 - away) - torch.where(plain <= clipped, plain, 0.0))
    grad = p * (-slope[:, None] / total)
    grad.scatter_add_(1, target, slope[:, None])
    return loss, logp, grad.to(s["logits"].dtype)


# ------------------------------------------------------------------ the package's operators
def _own(s):
    from rbf_attention_b200 import ops

    kind = s["kind"]
    if kind == "attend":
        return ops.cache_attention(s["q"], s["pages"], s["table"], s["lengths"], softmax=s["softmax"])
    if kind == "append":
        ops.cache_append(s["pages"], s["table"], s["lengths"], s["k"], s["v"])
        return ops.cache_read(s["pages"], s["table"], s["total"], s["D"], s["dtype"], s["count"], first=s["first"])
    if kind == "pages":
        ops.cache_copy_pages(s["pages"], s["src"], s["dst"])
        return s["pages"]
    if kind == "log_probs":
        return ops.token_log_probs(s["logits"], s["tokens"])
    s["logits"].grad = None
    loss, logp = ops.policy_loss(s["logits"], s["tokens"], s["old"], s["adv"], ref_log_probs=s["ref"], clip_low=CLIP_LOW,
                                 clip_high=CLIP_HIGH, kl_weight=KL_WEIGHT)
    loss.backward()
    return loss.detach(), logp, s["logits"].grad


def run(state):
    if own:
        return _own(state)
    plain = {"attend": _plain_attend, "append": _plain_append, "pages": _plain_pages, "log_probs": _plain_log_probs,
             "policy": _plain_policy}
    return plain[state["kind"]](state)


# ------------------------------------------------------------------ unavoidable work
def work(case):
    kind = case["kind"]
    if kind == "attend":
        B, H, G, D, T = (case[n] for n in ("B", "H", "G", "D", "T"))
        total = [n + T for n in _lengths(case)]
        held = sum(H * 2 * (n // BLOCK * (BLOCK * D + 4) + n % BLOCK * 2 * D) for n in total)
        seen = sum(T * (n - T) + T * (T + 1) // 2 for n in total)
        return {"bytes": float(held + 2 * B * H * G * T * D * 2), "flops": 4.0 * H * G * D * seen}
    if kind == "append":
        B, H, D, T = (case[n] for n in ("B", "H", "D", "T"))
        moved = written = 0
        for n in _lengths(case):
            done, rest = (n + T) // BLOCK - n // BLOCK, (n + T) % BLOCK
            moved += T * 2 * D + (n % BLOCK * 2 * D if done else 0)
            written += done * (BLOCK * D + 4) + min(rest, T) * 2 * D
        count = BLOCK if T == 1 else T
        return {"bytes": 2.0 * H * (moved + 2 * written + B * count * 2 * D), "flops": 0.0}
    if kind == "pages":
        return {"bytes": 2.0 * case["copies"] * case["layers"] * case["H"] * _page_bytes(case["D"]), "flops": 0.0}
    size = case["rows"] * case["cols"]
    if kind == "log_probs":
        return {"bytes": float(size * BYTES[case["dtype"]] + case["rows"] * 12), "flops": 4.0 * size}
    return {"bytes": float(2 * size * BYTES[case["dtype"]] + case["rows"] * 24), "flops": 8.0 * size}


# ------------------------------------------------------------------ 64 bits
def _bytes_at(page, P, token, is_value):
    """The codes (tokens, P) of the tokens ``token`` of one head's pages (M, bytes), by address."""
    block, r = token % PAGE // BLOCK, token % BLOCK
    d = torch.arange(P, device=page.device)[None]
    r = r[:, None]
    if is_value:
        inner = 16 * P + d // 32 * 512 + (d % 32 // 4 * 4 + r // 4) * 16 + d % 4 * 4 + r % 4
    else:
        inner = (d // 64 * 2 + r // 2 % 2) * 512 + (r // 4 * 2 + r % 2) * 64 + d % 64
    return page[(token // PAGE)[:, None], HEADER + block[:, None] * 32 * P + inner].double() - 128.0


def _exact_attend(case, s):
    B, H, G, D, T = (case[n] for n in ("B", "H", "G", "D", "T"))
    P, gamma = _columns(D), D ** -0.5
    out = torch.zeros(B, H * G, T, D, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(_lengths(case)):
        total = n + T
        token = torch.arange(total, device=DEVICE)
        whole = total // BLOCK * BLOCK
        for h in range(H):
            page = s["pages"][s["table"][b].long(), h]
            held = []
            for i in (0, 1):
                x = _bytes_at(page, P, token, i == 1)
                scale = page[:, :HEADER].contiguous().view(torch.float32).double()
                x = x * scale[token // PAGE, token % PAGE // BLOCK * 2 + i][:, None]
                if whole < total:
                    at = HEADER + (PER_PAGE + i) * 32 * P
                    x[whole:] = page[whole // PAGE, at:at + 32 * P].view(s["dtype"]).view(BLOCK, P)[:total - whole].double()
                held.append(x[:, :D])
            k, v = held
            q = s["q"][b, h * G:(h + 1) * G].double()
            distance = (q.square().sum(-1)[..., None] if not case["softmax"] else 0.0) + k.square().sum(-1) - 2.0 * (q @ k.T)
            weight = -gamma * distance
            seen = token[None] <= n + torch.arange(T, device=DEVICE)[:, None]
            weight = weight.masked_fill(~seen[None], -math.inf)
            weight = torch.softmax(weight, -1) if case["softmax"] else weight.exp()
            out[b, h * G:(h + 1) * G] = weight @ v
    return out


def _exact_append(case, s):
    T, D, P = case["T"], case["D"], _columns(case["D"])
    outs = []
    for i, x in enumerate((s["k"], s["v"])):
        out = torch.zeros(case["B"], case["H"], s["count"], D, dtype=torch.float64, device=DEVICE)
        for b, n in enumerate(_lengths(case)):
            start = n // BLOCK * BLOCK
            page = s["pages"][s["table"][b, n // PAGE].long()]
            at = HEADER + (PER_PAGE + i) * 32 * P
            tail = page[:, at:at + 32 * P].contiguous().view(s["dtype"]).view(-1, BLOCK, P)[:, :n - start, :D]
            have = torch.cat([tail.double(), x[b].double()], 1)
            whole = have.shape[1] // BLOCK * BLOCK
            block = have[:, :whole].reshape(case["H"], whole // BLOCK, BLOCK, D)
            step = block.abs().amax((2, 3), keepdim=True) / 127
            have[:, :whole] = (torch.round(block / step) * step).reshape(case["H"], whole, D)
            out[b, :, :have.shape[1]] = have
        outs.append(out)
    return tuple(outs)


def exact(case, seed):
    kind = case["kind"]
    if kind == "pages":
        return None
    if kind == "attend" and case["B"] * case["H"] > 2048:
        return None
    s = prepare(case, seed)
    if kind == "attend":
        return _exact_attend(case, s)
    if kind == "append":
        return _exact_append(case, s)
    t, rows = s["tokens"], case["rows"]
    keep = t != IGNORE
    logp = torch.zeros(rows, dtype=torch.float64, device=DEVICE)
    logits = s["logits"].detach()
    for r in range(0, rows, 512):
        logp[r:r + 512] = torch.log_softmax(logits[r:r + 512].double(), -1).gather(1, t[r:r + 512].clamp(min=0)[:, None])[:, 0]
    logp = logp * keep
    if kind == "log_probs":
        return logp
    lp = logp.clone().requires_grad_(True)
    ratio = (lp - s["old"].double()).exp()
    adv, gap = s["adv"].double(), s["ref"].double() - lp
    gain = torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
    loss = (KL_WEIGHT * (gap.exp() - gap - 1) - gain)[keep].mean()
    (slope,) = torch.autograd.grad(loss, lp)
    if rows * case["cols"] > 2**29:
        return loss.detach(), logp, None
    grad = torch.zeros(rows, case["cols"], dtype=torch.float64, device=DEVICE)
    for r in range(0, rows, 512):
        part = -torch.softmax(logits[r:r + 512].double(), -1)
        part.scatter_add_(1, t[r:r + 512].clamp(min=0)[:, None], torch.ones(part.shape[0], 1, dtype=torch.float64, device=DEVICE))
        grad[r:r + 512] = part * slope[r:r + 512, None]
    return loss.detach(), logp, grad
