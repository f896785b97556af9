"""Causal language model around the RBF attention block, with the reference's module and parameter names
(``train_rbf_transformer.py:113-244``: ``token_emb``, ``register_tokens``, ``blocks.<i>.{attn, ln1, ff, ln2}``,
``ln_f``, ``to_logits``), so that reference checkpoints load and the data-parallel training step of the benchmark
runs the same architecture: pre-LayerNorm blocks, 4x GELU MLP, zero-initialised register tokens prepended to the
sequence and sliced off before the final norm, untied output projection."""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops
from .attention import CustomCausalAttention
from .cache import PagedCache


def vocab_projection(linear: nn.Linear, x: torch.Tensor, keep_padding: bool = False) -> torch.Tensor:
    """``linear(x)`` for an output width (the vocabulary) whose rows are not 16-byte aligned in 16-bit types. With the
    reference's vocabulary of 50257 the logits' row pitch is odd, and the GEMM library falls back to kernels of an old
    architecture for all three products of this layer (measured on B200: 77 of the 116 ms of a training step). The
    product is evaluated at the width rounded up to a multiple of 64 - the weight is zero-padded on the fly, 51 MB -
    and the caller gets the first ``out_features`` columns as a view; parameters and state dict are unchanged.
    With ``keep_padding`` the padded width is returned as it is, the extra columns holding -inf (probability zero,
    gradient zero): a loss evaluated on it equals the loss on the sliced logits and saves the copies a strided view of
    6.6 GB of logits costs on its way through log-softmax and back."""
    V = linear.out_features
    pad = (-V) % 64
    if pad == 0 or not x.is_cuda or x.dtype == torch.float32:
        return linear(x)
    weight = F.pad(linear.weight, (0, 0, 0, pad))
    if keep_padding:
        bias = torch.zeros(V, dtype=x.dtype, device=x.device) if linear.bias is None else linear.bias
        return F.linear(x, weight, F.pad(bias, (0, pad), value=float("-inf")))
    bias = None if linear.bias is None else F.pad(linear.bias, (0, pad))
    return F.linear(x, weight, bias)[..., :V]


def apply_layer_norm(ln: nn.LayerNorm, x: torch.Tensor) -> torch.Tensor:
    """``ln(x)``: 16-bit CUDA activations of a supported width go through the library's one-pass kernels
    (``ops.layer_norm``, a warp per row; PyTorch's kernels reach a sixth of the memory bandwidth at 512 columns),
    anything else through PyTorch."""
    if x.is_cuda and len(ln.normalized_shape) == 1 and ln.elementwise_affine:
        weight, bias = ln.weight, ln.bias           # once: a module's parameters are found through __getattr__
        if ops.layer_norm_supported(x, weight, bias):
            return ops.layer_norm(x, weight, bias, ln.eps)
    return ln(x)


def apply_add_layer_norm(ln: nn.LayerNorm, x: torch.Tensor, delta):
    """``x = x + delta; return x, ln(x)`` (``delta`` None: ``x, ln(x)``): the residual addition rides on the
    LayerNorm that follows it, forward and backward, where the library's kernels apply."""
    if delta is None:
        return x, apply_layer_norm(ln, x)
    if x.is_cuda and len(ln.normalized_shape) == 1 and ln.elementwise_affine and delta.shape == x.shape \
            and delta.dtype == x.dtype:
        weight, bias = ln.weight, ln.bias
        if ops.layer_norm_supported(x, weight, bias):
            return ops.add_layer_norm(x, delta, weight, bias, ln.eps)
    x = x + delta
    return x, ln(x)


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """The training loss of the reference (``torch.nn.CrossEntropyLoss(ignore_index=-100)`` on flattened logits,
    train_rbf_transformer.py:282, 340-345). CUDA logits go through the library's single-kernel loss + gradient
    (``ops.cross_entropy``: one read and one write of the logits instead of four passes and an fp32 copy); anything
    else (the CPU oracle runs of the tests) is PyTorch's."""
    logits = logits.reshape(-1, logits.shape[-1])
    targets = targets.reshape(-1)
    if logits.is_cuda:
        return ops.cross_entropy(logits, targets, ignore_index)
    return F.cross_entropy(logits, targets, ignore_index=ignore_index)


class TransformerBlock(nn.Module):
    def __init__(self, emb_dim, num_heads, max_seq_len, use_rope, attention_type, use_qk_norm=False, use_xsa=False,
                 num_registers=0):
        super().__init__()
        self.attention_type = attention_type
        self.use_qk_norm = use_qk_norm
        self.use_xsa = use_xsa
        self.attn = CustomCausalAttention(num_heads, emb_dim, max_seq_len, use_rope, attention_type, use_qk_norm,
                                          use_xsa, num_registers)
        self.ln1 = nn.LayerNorm(emb_dim)
        self.ff = nn.Sequential(nn.Linear(emb_dim, 4 * emb_dim), nn.GELU(), nn.Linear(4 * emb_dim, emb_dim))
        self.ln2 = nn.LayerNorm(emb_dim)

    def forward(self, x):
        x, mlp_out, attn_weights = self.forward_deferred(x)
        return x + mlp_out, attn_weights

    def forward_deferred(self, x, pending=None):
        """The block on ``x + pending`` with its own last residual addition left to the caller: returns
        (x, mlp_out, attention weights) with the block's output being ``x + mlp_out``. A stack of blocks hands
        ``mlp_out`` to the next block as ``pending``, so that every residual addition is made by the LayerNorm pass
        that follows it."""
        x, normed = apply_add_layer_norm(self.ln1, x, pending)
        attn_out, attn_weights = self.attn(normed)
        x, normed = apply_add_layer_norm(self.ln2, x, attn_out)
        return x, self._mlp(normed), attn_weights

    def forward_cached(self, x, cache, layer, from_empty=False, pending=None):
        """``forward_deferred`` for the new tokens of a step of ``cache``, see CustomCausalAttention.forward_cached."""
        x, normed = apply_add_layer_norm(self.ln1, x, pending)
        x, normed = apply_add_layer_norm(self.ln2, x, self.attn.forward_cached(normed, cache, layer, from_empty))
        return x, self._mlp(normed)

    def _mlp(self, x):
        """``self.ff(x)`` (Linear, GELU, Linear) with the activation, its backward and the bias gradients of both
        projections from the library."""
        if x.is_cuda:
            up, act, down = self.ff[0], self.ff[1], self.ff[2]
            exact_gelu = isinstance(act, nn.GELU) and act.approximate == "none"
            hidden = ops.linear_gelu(up, x) if exact_gelu else act(ops.linear(up, x))
            return ops.linear(down, hidden)
        return self.ff(x)


class CausalLM(nn.Module):
    def __init__(self, vocab_size, d_model=256, num_layers=4, num_heads=4, max_seq_len=1024, pos_emb_type="none",
                 use_qk_norm=False, num_registers=0, attention_type="standard"):
        super().__init__()
        if use_qk_norm and attention_type.startswith("rbf"):
            raise AssertionError("QK-Norm requires standard attention")
        if pos_emb_type not in ("none", "rope", "learned"):
            raise ValueError(f"Unsupported pos_emb_type: {pos_emb_type}")
        self.num_registers = num_registers
        self.use_qk_norm = use_qk_norm
        self.pos_emb_type = pos_emb_type
        if num_registers > 0:
            if attention_type.startswith("rbf"):
                # zero registers start at distance |q|^2 from every query (the reference's choice for RBF)
                init = torch.zeros(num_registers, d_model)
            elif attention_type.startswith("standard"):
                init = torch.randn(num_registers, d_model) * d_model**-0.5
            else:
                raise ValueError(f"Unsupported attention type: {attention_type}")
            self.register_tokens = nn.Parameter(init)
        self.token_emb = nn.Embedding(vocab_size, d_model)
        if pos_emb_type == "learned":
            self.pos_emb = nn.Embedding(max_seq_len, d_model)
        self.use_rope = pos_emb_type == "rope"
        self.blocks = nn.ModuleList(
            TransformerBlock(d_model, num_heads, max_seq_len, self.use_rope, attention_type, use_qk_norm=use_qk_norm,
                             use_xsa=False, num_registers=num_registers)
            for _ in range(num_layers)
        )
        self.ln_f = nn.LayerNorm(d_model)
        self.to_logits = nn.Linear(d_model, vocab_size)

    def forward(self, idx, padded_logits: bool = False):
        """Returns (logits, attention weights per block). ``padded_logits`` (not in the reference): the logits keep the
        vocabulary rounded up to a multiple of 64 with -inf in the extra columns, see ``vocab_projection``."""
        bsz, seq = idx.shape
        x = self.token_emb(idx)
        if self.pos_emb_type == "learned":
            x = x + self.pos_emb(torch.arange(seq, device=idx.device))
        if self.num_registers > 0:
            x = torch.cat([self.register_tokens.unsqueeze(0).expand(bsz, -1, -1).to(x.dtype), x], dim=1)
        weights = []
        pending = None                      # the last block's MLP output, added by the next LayerNorm pass
        for block in self.blocks:
            x, pending, w = block.forward_deferred(x, pending)
            weights.append(w)
        _, normed = apply_add_layer_norm(self.ln_f, x, pending)     # row-wise: the register rows are dropped after it
        if self.num_registers > 0:
            # contiguous: F.linear takes a strided 3-D input through matmul + a separate bias pass over the logits
            normed = normed[:, self.num_registers:, :].contiguous()
        return vocab_projection(self.to_logits, normed, keep_padding=padded_logits), weights

    # -- answers ---------------------------------------------------------------------------------
    def new_cache(self, max_sequences: int, max_length: int, num_pages: int | None = None) -> PagedCache:
        """A cache for ``max_sequences`` sequences of up to ``max_length`` tokens (the register tokens come on top)."""
        attn = self.blocks[0].attn
        self._check_positions(max_length)
        weight = self.to_logits.weight
        return PagedCache(len(self.blocks), attn.num_heads, attn.head_dim, max_sequences, max_length + self.num_registers,
                          num_pages, weight.dtype, weight.device)

    def _check_positions(self, length: int) -> None:
        """Refuses sequences that the model has no positions for."""
        table = getattr(self.blocks[0].attn, "susie_cache", None)
        for limit in (None if table is None else table.shape[0],
                      self.pos_emb.num_embeddings if self.pos_emb_type == "learned" else None):
            if limit is not None and length > limit:
                raise ValueError(f"the model's positions end at {limit} tokens, {length} are asked for")

    @torch.no_grad()
    def forward_cached(self, idx, cache: PagedCache, new=None, sequences=None, all_logits: bool = False):
        """Logits (batch, vocab) behind each sequence's last new token - with ``all_logits`` (batch, T, vocab) behind every one -
        of the ``idx`` (batch, T) that follow what ``cache`` holds; ``new``: how many of the T are real, per sequence (default:
        all; what is behind them is padding, which may be longer than the model's positions and has logits of zero or no meaning),
        ``sequences``: which of the cache's these are (default: all). Either all or none of those that get tokens are
        empty. A sequence without new tokens has logits of no meaning. If it raises, no sequence has got tokens; where a layer had
        been written, those that would have got some are empty (``PagedCache.abort``)."""
        bsz, seq = idx.shape
        batch = range(cache.max_sequences) if sequences is None else sequences
        new = [seq] * bsz if new is None else [int(n) for n in new]
        if len(batch) != bsz or len(new) != bsz or any(not 0 <= n <= seq for n in new):
            raise ValueError(f"{len(batch)} sequences, new tokens {new} and ids {tuple(idx.shape)} do not go together")
        empty = {cache.length(s) == 0 for s, n in zip(batch, new) if n}
        if len(empty) > 1:
            raise ValueError("some of the sequences are empty, others are not: give them their tokens in two calls")
        from_empty = empty == {True}
        self._check_positions(max((cache.length(s) + n - (0 if from_empty else self.num_registers) for s, n in zip(batch, new) if n),
                                  default=0))
        idx = idx[:, :max([1, *new])]          # no sequence has a place for what is behind
        cut, seq = seq - idx.shape[1], idx.shape[1]
        skip = self.num_registers if from_empty else 0
        cache.begin([n + skip if n else 0 for n in new], sequences)
        try:
            x = self.token_emb(idx)
            if self.pos_emb_type == "learned":
                at = cache.positions[:, None] + torch.arange(seq, device=idx.device) - (0 if from_empty else self.num_registers)
                x = x + self.pos_emb(at.clamp(0, self.pos_emb.num_embeddings - 1))
            if skip:
                x = torch.cat([self.register_tokens.unsqueeze(0).expand(bsz, -1, -1).to(x.dtype), x], dim=1)
            pending = None
            for i, block in enumerate(self.blocks):
                x, pending = block.forward_cached(x, cache, i, from_empty, pending)
            _, normed = apply_add_layer_norm(self.ln_f, x, pending)
            if all_logits:
                normed = normed[:, skip:].contiguous()
            else:
                last = torch.tensor([skip + max(n - 1, 0) for n in new]).to(idx.device)
                normed = normed[torch.arange(bsz, device=idx.device), last]
            logits = vocab_projection(self.to_logits, normed)
            if all_logits and cut:
                logits = F.pad(logits, (0, 0, 0, cut))
        except BaseException:
            cache.abort()
            raise
        cache.end()
        return logits

    @torch.no_grad()
    def generate(self, idx, max_new_tokens: int, lengths=None, samples: int = 1, temperature: float = 0.0, generator=None,
                 cache: PagedCache | None = None):
        """(batch * samples, max_new_tokens) ids that follow the prompts ``idx`` (batch, T), of ``lengths`` tokens each where
        they are padded: the most likely ones (the reference's generation, train_rbf_transformer.py:446-530), or drawn at
        ``temperature``. A prompt's ``samples`` answers are rows beside one another and share its pages. ``cache``: an empty one
        of batch * samples sequences, left with what the model has read."""
        bsz, seq = idx.shape
        lengths = [seq] * bsz if lengths is None else [int(n) for n in lengths]
        if max_new_tokens < 1 or samples < 1 or len(lengths) != bsz or any(not 0 < n <= seq for n in lengths):
            raise ValueError(f"prompts {tuple(idx.shape)} of {lengths} tokens, {max_new_tokens} new ones, {samples} samples")
        rows = bsz * samples
        if cache is None:
            cache = self.new_cache(rows, max(lengths) + max_new_tokens - 1)        # the last ids are not read again
        if cache.max_sequences != rows or any(cache.length(s) for s in range(rows)):
            raise ValueError(f"the cache must be an empty one of {rows} sequences")

        def choose(logits):
            if temperature == 0.0:
                return logits.argmax(-1)
            return torch.multinomial(torch.softmax(logits.float() / temperature, -1), 1, generator=generator)[:, 0]

        first = [b * samples for b in range(bsz)]
        logits = self.forward_cached(idx, cache, lengths, first).repeat_interleave(samples, 0)
        for s in first:
            cache.fork(s, range(s + 1, s + samples))
        out = [choose(logits)]
        while len(out) < max_new_tokens:
            out.append(choose(self.forward_cached(out[-1][:, None], cache)))
        return torch.stack(out, 1)


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """Log-probabilities (the shape of ``tokens``, fp32, no gradient) of given tokens under logits (..., vocab); 0 where the token
    is ``ignore_index``. CUDA logits go through the library's single read (``ops.token_log_probs``)."""
    logits = logits.detach()
    flat, t = logits.reshape(-1, logits.shape[-1]), tokens.reshape(-1)
    if logits.is_cuda:
        return ops.token_log_probs(flat, t, ignore_index).view(tokens.shape)
    counted = (t != ignore_index) & (t >= 0) & (t < flat.shape[-1])
    lp = torch.log_softmax(flat.float(), -1).gather(1, torch.where(counted, t, 0)[:, None])[:, 0]
    return torch.where(counted, lp, 0.0).view(tokens.shape)


def policy_loss(logits, tokens, old_log_probs, advantages, ref_log_probs=None, weights=None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_weight: float = 0.0, ignore_index: int = -100):
    """Clipped policy loss with a KL term (``ops.policy_loss``) of logits (..., vocab) and tokens, old_log_probs, advantages,
    ref_log_probs and weights of the leading shape: (loss, log_probs). CUDA logits only."""
    shape = tokens.shape
    rows = [None if t is None else t.reshape(-1) for t in (tokens, old_log_probs, advantages, ref_log_probs, weights)]
    loss, lp = ops.policy_loss(logits.reshape(-1, logits.shape[-1]), *rows, clip_low=clip_low, clip_high=clip_high,
                               kl_weight=kl_weight, ignore_index=ignore_index)
    return loss, lp.view(shape)


def zipf_token_ids(batch, seq_len, vocab_size, exponent=1.1, seed=0):
    """(batch, seq_len) int64 token ids with P(id = k) proportional to (k + 1)^-exponent, seeded, on the CPU."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    probs = torch.arange(1, vocab_size + 1, dtype=torch.float64).pow(-exponent)
    return torch.multinomial(probs / probs.sum(), batch * seq_len, replacement=True, generator=g).view(batch, seq_len)
