"""The language model with a cache: answers to prompts, samples that share a prompt's pages, and a policy-gradient step on them,
against the model's definition in 64 bits over what the cache holds."""

import copy
import math

import pytest
import torch
import torch.nn.functional as F

from rbf_attention_b200 import lm, ops
from rbf_attention_b200.cache import PagedCache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
VOCAB = 517


def _model(kind="rbf_triton", pos="rope", registers=3, heads=2, width=128, layers=2, dtype=torch.bfloat16, seed=0, xsa=False):
    torch.manual_seed(seed)
    model = lm.CausalLM(VOCAB, d_model=width, num_layers=layers, num_heads=heads, max_seq_len=700, pos_emb_type=pos,
                        num_registers=registers, attention_type=kind)
    with torch.no_grad():
        for p in model.parameters():
            p.mul_(1.5)
        if registers:
            model.register_tokens.normal_()
    for block in model.blocks:
        block.attn.apply_xsa = xsa
    return model.to(DEV, dtype).requires_grad_(False)


def _ids(B, T, seed=1):
    return torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _snapshot(cache):
    """What the cache holds of every sequence now: per layer, keys and values."""
    return [cache.read(layer) for layer in range(cache.pages.shape[0])]


def _reference(model, ids, steps, held, b):
    """Logits (T, vocab) in 64 bits of sequence b whose tokens came in portions of ``steps``: the first portion attends to itself,
    later ones to what the cache holds when theirs has been added (``held``: after every portion, as _snapshot has it). What it
    holds is looked at too: every key and value within half a step of its block's scale of the reference's."""
    m = copy.deepcopy(model).double().to(DEV)
    R = m.num_registers
    outs, kept, done = [], [], 0
    for i, n in enumerate(steps):
        x = m.token_emb(ids[done:done + n])
        at = torch.arange(done, done + n, device=DEV)
        if m.pos_emb_type == "learned":
            x = x + m.pos_emb(at)
        skip = R if i == 0 else 0
        if skip:
            x = torch.cat([m.register_tokens, x])
        before = 0 if i == 0 else done + R
        place = torch.arange(before, before + x.shape[0], device=DEV)
        for li, block in enumerate(m.blocks):
            a = block.attn
            H, D = a.num_heads, a.head_dim
            q, k, v = a.qkv_proj(block.ln1(x)).view(-1, 3, H, D).permute(1, 2, 0, 3)
            if a.positional_encoding_type == "susie":
                emb = a.susie_cache.double()[(place - R).clamp(min=0)] * a.pos_weight[0].repeat(1, 1, 2)
                if R:
                    emb = torch.where((place < R)[:, None], a.reg_pos_emb[0][:, place.clamp(max=R - 1)], emb)
                q, k = q + emb, k + emb
            if li == len(kept):
                kept.append([k[:, :0], v[:, :0]])
            kept[li] = [torch.cat([kept[li][0], k], 1), torch.cat([kept[li][1], v], 1)]
            kk, vv = kept[li]
            total = kk.shape[1]
            for mine, there in zip(kept[li], held[i][li]):
                there = there[b, :, :total].double()
                whole = total // 16 * 16
                step = torch.zeros(H, total, 1, dtype=torch.float64, device=DEV)
                step[:, :whole] = (mine[:, :whole].reshape(H, whole // 16, 16 * D).abs().amax(-1) / 127).repeat_interleave(16, 1)[..., None]
                off = (there - mine).abs() - 0.51 * step
                assert off.max() <= _bound(model) * mine.abs().max(), (i, li)
            if i > 0:
                kk, vv = (x2[b, :, :total].double() for x2 in held[i][li])
            logits = -(q[:, :, None] - kk[:, None]).square().sum(-1) / math.sqrt(D)
            hidden = torch.arange(total, device=DEV)[None] > place[:, None]
            logits = logits.masked_fill(hidden, -math.inf)
            w = logits.exp() if a.attention_type == "rbf_non_softmax" else logits.softmax(-1)
            o = w @ vv
            if a.apply_xsa:
                vh = F.normalize(v, dim=-1)
                o = o - (o * vh).sum(-1, keepdim=True) * vh
            x = x + a.proj(o.transpose(0, 1).reshape(-1, H * D))
            x = x + block.ff(block.ln2(x))
        outs.append(m.to_logits(m.ln_f(x))[skip:])
        done += n
    return torch.cat(outs)


# Roundings between an id and its logit: about twelve per layer (projections, the position, q, k, v, P, the output, two residual
# sums, two norms, three of the MLP) and three around them, each half a step of the type, independent: their squares add up, and
# the residual stream carries them on at its own scale. Twice that root covers how the layers weigh them.
def _bound(model):
    n = 12 * len(model.blocks) + 3
    return 2 * math.sqrt(n) * torch.finfo(next(model.parameters()).dtype).eps / 2


@pytest.mark.parametrize("kind,pos,registers,heads,width,dtype,xsa", [
    ("rbf_triton", "rope", 3, 2, 128, torch.bfloat16, False),
    ("rbf_triton", "rope", 0, 1, 128, torch.float16, False),
    ("rbf_non_softmax", "rope", 4, 2, 128, torch.float16, False),
    ("rbf_triton", "learned", 2, 2, 256, torch.bfloat16, True),
    ("rbf_flex", "none", 0, 4, 192, torch.float16, True),
])
def test_portions_of_a_sequence(kind, pos, registers, heads, width, dtype, xsa):
    model = _model(kind, pos, registers, heads, width, dtype=dtype, xsa=xsa)
    steps = [[40, 1, 1, 13, 1, 200, 1], [7, 20, 1, 1, 1, 1, 1], [250, 1, 1, 5, 1, 60, 2]]
    T = [sum(s) for s in steps]
    ids = _ids(3, max(T))
    cache = model.new_cache(3, 400)
    got, held = [[] for _ in range(3)], []
    done = [0, 0, 0]
    for i in range(len(steps[0])):
        new = [s[i] for s in steps]
        part = torch.stack([F.pad(ids[b, done[b]:done[b] + new[b]], (0, max(new) - new[b]), value=VOCAB - 1) for b in range(3)])
        full = i % 2 == 0
        logits = model.forward_cached(part, cache, new, all_logits=full)
        for b, n in enumerate(new):
            got[b].append(logits[b, :n] if full else logits[b:b + 1])
        done = [d + n for d, n in zip(done, new)]
        held.append(_snapshot(cache))
    for b in range(3):
        want = _reference(model, ids[b], steps[b], held, b)
        at = 0
        for i, (n, part) in enumerate(zip(steps[b], got[b])):
            ref = want[at:at + n][-part.shape[0]:]
            rel = ((part.double() - ref).norm() / ref.norm()).item()
            assert rel <= _bound(model), (b, i, rel)
            at += n
        assert cache.length(b) == T[b] + registers


def test_the_first_portion_is_the_models_forward():
    model = _model()
    ids = _ids(2, 90)
    cache = model.new_cache(2, 100)
    got = model.forward_cached(ids, cache, all_logits=True)
    want = model(ids)[0]
    assert torch.equal(got, want)
    k, v = cache.read(0)
    assert k.shape == (2, 2, 93, 64) and k.isfinite().all() and v.isfinite().all()


def test_greedy_answers_are_the_most_likely_ones():
    """Every chosen id is the argmax of the 64-bit logits, or as good as it: within twice what the logits may be off."""
    model = _model(dtype=torch.float16)
    ids = _ids(3, 30)
    lengths = [30, 4, 17]
    out = model.generate(ids, 25, lengths)
    assert out.shape == (3, 25)
    cache, held = model.new_cache(3, 60), []
    model.forward_cached(ids, cache, lengths)               # the same steps again, for what the cache held after each
    held.append(_snapshot(cache))
    for t in range(24):
        assert torch.equal(model.forward_cached(out[:, t:t + 1], cache).argmax(-1), out[:, t + 1])
        held.append(_snapshot(cache))
    for b, n in enumerate(lengths):
        whole = torch.cat([ids[b, :n], out[b]])
        want = _reference(model, whole[:-1], [n] + [1] * 24, held, b)[n - 1:]
        off = 2 * _bound(model) * want.norm(dim=-1) / math.sqrt(VOCAB) * 5       # five times the root mean square: a maximum
        assert (want.gather(1, out[b][:, None])[:, 0] >= want.amax(-1) - off).all()


def test_samples_share_their_prompts_pages():
    """Several samples of a prompt are what the same calls give one by one."""
    model = _model()
    ids = _ids(2, 290)
    cache = model.new_cache(6, 330)
    before = cache.free_pages
    out = model.generate(ids, 20, [290, 250], samples=3, cache=cache)
    assert out.shape == (6, 20) and (out[0] == out[1]).all() and (out[3] == out[5]).all()
    # the first prompt's full page once, its last page three times; the second's page three times, as many go over its end
    assert before - cache.free_pages == (1 + 3) + (3 + 3)
    alone = model.generate(ids, 20, [290, 250])
    assert torch.equal(alone, out[::3])
    g = torch.Generator(device=DEV).manual_seed(5)
    drawn = model.generate(ids, 12, samples=4, temperature=1.0, generator=g)
    assert drawn.shape == (8, 12) and len({tuple(r.tolist()) for r in drawn}) > 4
    again = model.generate(ids, 12, samples=4, temperature=1.0, generator=torch.Generator(device=DEV).manual_seed(5))
    assert torch.equal(drawn, again)


def test_compaction_in_the_middle_of_an_answer():
    model = _model(dtype=torch.float16)
    ids = _ids(4, 300)
    caches = [model.new_cache(4, 400, num_pages=12) for _ in range(2)]
    outs = []
    for i, c in enumerate(caches):
        logits = [model.forward_cached(ids, c)]
        c.free([0, 2])
        if i:
            assert c.compact() > 0
            c.resize(5)
        for t in range(10):
            logits.append(model.forward_cached(ids[1::2, t:t + 1], c, sequences=[1, 3]))
        outs.append(torch.cat(logits))
    assert torch.equal(*outs)


def test_one_graph_for_all_steps_of_an_answer():
    model = _model()
    ids = _ids(2, 100)
    caches = [model.new_cache(2, 400) for _ in range(2)]
    first = [model.forward_cached(ids, c).argmax(-1) for c in caches]
    token = first[0][:, None].clone()

    def step(cache):                        # between begin() and end()
        x, pending = model.token_emb(token), None
        for i, block in enumerate(model.blocks):
            x, pending = block.forward_cached(x, cache, i, False, pending)
        return model.to_logits(lm.apply_add_layer_norm(model.ln_f, x, pending)[1])[:, -1]

    a, b = caches
    with torch.no_grad():
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            a.begin(1)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = step(a)
        torch.cuda.current_stream().wait_stream(stream)
        other = first[1][:, None]
        for i in range(200):                # over the end of a page
            if i > 0:
                a.begin(1)
            graph.replay()
            a.end()
            want = model.forward_cached(other, b)
            assert torch.equal(out.argmax(-1), want.argmax(-1)) and (out - want).abs().max() <= 0.1 * want.abs().max(), i
            other = want.argmax(-1)[:, None]
            token.copy_(out.argmax(-1)[:, None])


def _policy_reference(logits, tokens, old, adv, ref):
    lp = torch.log_softmax(logits.float(), -1).gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    keep = tokens != -100
    r = (lp - old).exp()
    gap = ref - lp
    value = 0.1 * (gap.exp() - gap - 1) - torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv)
    return (value * keep).sum() / keep.sum()


def test_a_step_of_fine_tuning_on_sampled_answers():
    """Prompts, several answers to each, their log-probabilities, the loss, and gradients of every parameter."""
    model = _model()
    prompts, samples, T = _ids(2, 20), 4, 30
    answers = model.generate(prompts, T, samples=samples, temperature=1.0, generator=torch.Generator(device=DEV).manual_seed(0))
    ids = torch.cat([prompts.repeat_interleave(samples, 0), answers], 1)
    tokens = ids[:, 1:].clone()
    tokens[:, :19] = -100                   # the prompt is not the model's to learn
    with torch.no_grad():
        logits = model(ids[:, :-1], padded_logits=True)[0]
    old = lm.token_log_probs(logits, tokens)
    assert old.shape == tokens.shape and not old[:, :19].any() and (old[:, 19:] < 0).all()
    ref = old + 0.1 * torch.randn_like(old)
    adv = torch.randn(2 * samples, 1, device=DEV).expand_as(old)
    old = old + 0.15 * torch.randn_like(old)
    grads = []
    for own in (True, False):
        m = copy.deepcopy(model).requires_grad_(True)
        logits = m(ids[:, :-1], padded_logits=own)[0]
        if own:
            loss, lp = lm.policy_loss(logits, tokens, old, adv, ref_log_probs=ref, kl_weight=0.1)
            assert lp.shape == tokens.shape and not lp.requires_grad
        else:
            loss = _policy_reference(logits, tokens, old, adv, ref)
        loss.backward()
        grads.append([p.grad.double() for p in m.parameters()] + [loss.detach().double()])
    # both sides round the same gradient of the logits to bfloat16, one from fp32 in one step: it and all that follows from it
    # differ by roundings, as the logits of two paths through the model do
    for i, (a, b) in enumerate(zip(*grads)):
        assert (a - b).norm() <= 2 * _bound(model) * b.norm() + 1e-6, i


def test_refusals():
    model = _model()
    ids = _ids(2, 10)
    cache = model.new_cache(2, 20)
    with pytest.raises(ValueError, match="positions end"):
        model.new_cache(1, 701)
    for call in (lambda: model.forward_cached(ids, cache, [11, 1]), lambda: model.forward_cached(ids[:1], cache),
                 lambda: model.forward_cached(ids, cache, [1]), lambda: model.generate(ids, 0), lambda: model.generate(ids, 3, [0, 4]),
                 lambda: model.generate(ids, 3, cache=model.new_cache(3, 20)), lambda: model.forward_cached(_ids(2, 30), cache)):
        with pytest.raises(ValueError):
            call()
    model.forward_cached(ids, cache, [10, 0])
    with pytest.raises(ValueError, match="two calls"):
        model.forward_cached(ids, cache, [1, 1])
    model.forward_cached(ids, cache, [0, 10])
    assert [cache.length(s) for s in (0, 1)] == [13, 13]
    with pytest.raises(ValueError, match="no cached form"):
        other = lm.CausalLM(VOCAB, 128, 1, 2, 64, attention_type="standard").to(DEV, torch.bfloat16)
        other.forward_cached(ids, PagedCache(1, 2, 64, 2, 64))
    with pytest.raises(ValueError, match="float32"):
        lm.CausalLM(VOCAB, 128, 1, 2, 64, attention_type="rbf_triton").to(DEV).new_cache(1, 10)
    ops.check_device_status()


@pytest.mark.parametrize("pos", ["rope", "learned"])
def test_positions_end_with_the_model(pos):
    """A cache of the caller's own may be longer than the model's positions: the token behind the last one is refused, before
    anything is written."""
    model = _model(pos=pos)
    limit = 700
    cache = PagedCache(len(model.blocks), 2, 64, 1, 2000, device=DEV)
    with pytest.raises(ValueError, match="positions end"):
        model.forward_cached(_ids(1, limit + 1), cache)
    model.forward_cached(_ids(1, limit - 1), cache)
    assert model.forward_cached(_ids(1, 1), cache).isfinite().all()
    held = cache.length(0)
    assert held == limit + model.num_registers
    with pytest.raises(ValueError, match="positions end"):
        model.forward_cached(_ids(1, 1), cache)
    assert cache.length(0) == held
