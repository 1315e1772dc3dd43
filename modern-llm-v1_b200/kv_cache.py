"""Per-layer KV cache for token-by-token sampling (csrc/kv_cache.cuh, csrc/attn_decode.cuh).

The reference's sampler keeps no cache: every generated token re-runs the model over the whole
T-token window (llm/apps/infer_modern_gpt.cu:13,253-255), and the cache is listed as future work
(TODO.md, "KV cache for inference").  This class is the attention side of that cache for a
ModernGPT block (llm/src/model/modern_gpt.cu:351-378): per layer a BF16 K and V buffer
[B, Hkv, L_cap, D]; `append` does split_heads + RoPE at the true positions + QK-Norm for the newest
tokens and stores their k and v, `attend` runs attention for them (causal forward over the prompt,
or the split-KV decode kernel for one token), `advance` moves the length once every layer is done.
The B sequences advance in lock step until `set_lengths` gives each its own length (a batch of
prompts of different lengths); from then on `append` and `attend` take one token per sequence at the
sequence's own position.

For long contexts a cache can also
  - rotate in other layouts (`pairs`, `rotary_dim`), with scaled frequencies (`scaling`, `factor`, `trained`, `turns_fast`,
    `turns_slow`) and without the QK-norm (gammas None), see rotary.py;
  - continue prompts that several of its sequences share (`prefix`: a KVCache that holds them; sequence b continues prompt
    b // (B // prefix.B)): the prompts' keys and values are kept and read once, not once per sequence;
  - keep the attention weight that each cached key has received and its position (`track_weights`), and cut itself down by it
    (`evict`): rows and positions then part ways, `next_position` is what counts on.
Like the reference's operators, the caller allocates every
input and output; bad arguments raise ValueError, CUDA failures RuntimeError; there is no CPU or
PyTorch fallback.
"""
from __future__ import annotations

import torch

from . import _lib
from .rope_norm import make_rope_cache
from .rotary import make_rotary_cache


def kv_evict(kcache, vcache, weights, positions, weights_out, positions_out, B, L, Hkv, D, keep, recent, lens=None, L_cap=None):
    """Cuts the first lens[b] rows (int32 [B] on the device; None: L) of every (batch, KV head) down to at most `keep`: the rows whose
    position is above newest - recent stay, then those of the largest weight, of equal ones the lower row (csrc/kv_evict.cuh).  kcache,
    vcache [B, Hkv, L_cap, D] BF16 change in place: rows below `keep` that stay are not moved, the j-th row that stays behind them goes
    to the j-th free place.  weights (FP32) and positions (int32, distinct within a head) [B, Hkv, L_cap] are read, weights_out and
    positions_out written whole, with 0 and -1 behind the rows that stayed."""
    _lib.host().kv_evict(kcache, vcache, weights, positions, weights_out, positions_out, B, L, Hkv, D, keep, recent, lens, L_cap)


class KVCache:
    def __new__(cls, *args, **kwargs):
        """The reference's rotation, a cache of its own, no weights.  (What every append, attend and advance asks are attributes of the
        instance alone: one that the class has as well costs a lookup of some 20 ns.)"""
        self = super().__new__(cls)
        self._plain = self._alone = True
        self.prefix, self.track_weights = None, False
        self._shift = 0  # a token's position minus its row, where all sequences agree
        self._pos = None  # else: the next token's position per sequence [B] int32 on the device
        self._evicted, self._prompts = False, None
        self._changes = 0  # times that the tokens which count have changed
        return self

    def __init__(self, n_layers: int, B: int, Hq: int, Hkv: int, D: int, L_cap: int, device="cuda",
                 rope_base=None, eps=None, *, rotary_dim=None, pairs="interleaved", scaling="none",
                 factor: float = 1.0, trained=None, T_max=None, prefix=None, track_weights: bool = False, turns_fast=None,
                 turns_slow=None):
        """rope_base is 10000 and eps 1e-5 where they are left out, or what the prompts' cache has (`prefix`); turns_fast and
        turns_slow are make_rotary_cache's, for "parts"."""
        if min(n_layers, B, Hq, Hkv, D, L_cap) <= 0 or Hq % Hkv != 0:
            raise ValueError("KVCache: sizes must be positive and Hq a multiple of Hkv")
        if D not in (64, 128):
            raise ValueError("KVCache: d_h must be 64 or 128")
        _lib.load()  # fail now, not at the first token, when the CUDA library is missing
        self.n_layers, self.B, self.Hq, self.Hkv, self.D, self.L_cap = n_layers, B, Hq, Hkv, D, L_cap
        self.eps = 1e-5 if eps is None else float(eps)
        self.device = torch.device(device)
        self.k = torch.zeros((n_layers, B, Hkv, L_cap, D), dtype=torch.bfloat16, device=self.device)
        self.v = torch.zeros_like(self.k)
        self.prefix, self.track_weights = prefix, bool(track_weights)
        self._alone = prefix is None and not self.track_weights
        turns = (turns_fast, turns_slow)
        own = (rotary_dim, pairs, scaling) != (None, "interleaved", "none")
        if prefix is None:
            self._rotary_setup(10000.0 if rope_base is None else rope_base, rotary_dim, pairs, scaling, factor, trained, turns, T_max, own)
        else:
            self._prefix_setup(prefix, own, T_max, rope_base, eps, factor, trained, turns)
        if self.track_weights:
            if prefix is not None:
                raise ValueError("KVCache: a cache that continues shared prompts keeps no weights")
            shape = (B, Hkv, L_cap)
            new = lambda: (torch.zeros(shape, device=self.device), torch.full(shape, -1, dtype=torch.int32, device=self.device))  # noqa: E731
            pairs_ = [new() for _ in range(n_layers + 1)]  # one more than layers: what an eviction writes to
            self.weights, self.positions = [w for w, _ in pairs_[:-1]], [p for _, p in pairs_[:-1]]
            self._spare = pairs_[-1]
        # the layers' own tensors, for the calls that take them
        self._kl, self._vl = list(self.k.unbind(0)), list(self.v.unbind(0))
        self.length = 0  # tokens held by every layer (the longest sequence's, once lengths differ)
        self.lengths = None  # per-sequence lengths [B] int32 on the device, once set_lengths was called
        self._lens_next = None  # lengths + 1: what the decode kernel reads while the newest token is being attended
        self._lengths_host = None

    def _rotary_setup(self, base, rotary_dim, pairs, scaling, factor, trained, turns, T_max, own):
        R = self.D if rotary_dim is None else int(rotary_dim)
        if pairs not in ("interleaved", "half"):
            raise ValueError("KVCache: pairs must be interleaved or half")
        if R <= 0 or R > self.D or R % 16 != 0:
            raise ValueError("KVCache: rotary_dim must be a multiple of 16, at most d_h")
        T = self.L_cap if T_max is None else int(T_max)
        if T < self.L_cap:
            raise ValueError("KVCache: T_max is less than the capacity")
        self._R, self._pairs, self._base = R, _lib.PAIRS_HALF if pairs == "half" else _lib.PAIRS_INTERLEAVED, base
        fast, slow = (default if x is None else float(x) for x, default in zip(turns, (32.0, 1.0)))
        self._scaled = (scaling, factor, trained, fast, slow)
        self._reference = not own
        self._plain = not own and not self.track_weights and T_max is None  # the reference's rotation, rows are positions
        self.cos, self.sin = self._tables(T)

    def _tables(self, T):
        if self._reference:  # the reference's rotation has its values, of angles in 32 bits
            return make_rope_cache(T, self.D, self._base, device=self.device)
        return make_rotary_cache(T, self._R, self._base, *self._scaled, device=self.device)

    def _prefix_setup(self, prefix, own, T_max, base, eps, factor, trained, turns):
        given = [(base, prefix._base), (eps, prefix.eps), *zip((None if factor == 1.0 else factor, trained, *turns), prefix._scaled[1:])]
        if own or T_max is not None or any(x is not None and x != theirs for x, theirs in given):
            raise ValueError("KVCache: a cache that continues prompts rotates and normalises as theirs does")
        if (prefix.n_layers, prefix.Hq, prefix.Hkv, prefix.D) != (self.n_layers, self.Hq, self.Hkv, self.D) or prefix.prefix is not None:
            raise ValueError("KVCache: prefix must be a cache of prompts with the same layers and heads")
        if prefix.track_weights:
            raise ValueError("KVCache: prefix must not keep weights")
        if self.B % prefix.B != 0:
            raise ValueError("KVCache: B must be a multiple of the number of prompts")
        self._R, self._pairs, self._scaled, self._base, self._reference = prefix._R, prefix._pairs, prefix._scaled, prefix._base, prefix._reference
        self._plain, self.eps = False, prefix.eps
        self.cos, self.sin = self._tables(prefix.L_cap + self.L_cap)

    def reset(self) -> None:
        """Forgets every token (the buffers keep their bytes; rows >= length are never read)."""
        self._changes += 1
        self.length = 0
        self.lengths = self._lens_next = self._lengths_host = None
        self._shift, self._pos, self._evicted, self._prompts = 0, None, False, None
        if self.track_weights:
            for w, p in zip(self.weights, self.positions):
                w.zero_()
                p.fill_(-1)

    def _place(self):
        """(first position, positions or None, rows or None) of the next tokens; behind prompts of different lengths they are made when
        the first token comes"""
        if self.prefix is not None and self._prompts is None:
            if self.prefix.length == 0:
                raise ValueError("KVCache: the prompts are empty")
            self._shift, self._prompts = self.prefix.length, self.prefix._changes
            if self.prefix.lengths is not None:
                self._pos = self.prefix.lengths.repeat_interleave(self.B // self.prefix.B)
        elif self.prefix is not None and self.prefix._changes != self._prompts:
            raise ValueError("KVCache: the prompts have changed since their first continuation (reset this cache)")
        return self.length + self._shift, self._pos, self.lengths

    @property
    def next_position(self):
        """The position of the next token: an int, or int32 [B] on the device where the sequences differ."""
        pos0, pos, rows = self._place()
        return pos.clone() if pos is not None else pos0 if rows is None else rows + self._shift

    def set_lengths(self, lengths) -> None:
        """Gives every sequence its own length (e.g. after a padded prompt batch went through `append` /
        `attend` / `advance` with the longest prompt's length): rows at and beyond a sequence's length are
        treated as not yet written.  With track_weights those rows' weights become 0 and their positions -1; what their tokens gave to the
        rows that stay remains."""
        host = [int(x) for x in lengths]
        if len(host) != self.B or min(host) < 0 or max(host) > self.L_cap:
            raise ValueError("KVCache.set_lengths: need B lengths in [0, L_cap]")
        if self._evicted or self.prefix is not None:
            raise ValueError("KVCache.set_lengths: not after an eviction, nor behind shared prompts")
        self._changes += 1
        self._lengths_host = host
        self.length = max(host)
        self.lengths = torch.tensor(host, dtype=torch.int32, device=self.device)
        self._lens_next = self.lengths + 1
        if self.track_weights:
            gone = torch.arange(self.L_cap, device=self.device) >= self.lengths[:, None, None]
            for w, p in zip(self.weights, self.positions):
                w.masked_fill_(gone, 0.0)
                p.masked_fill_(gone, -1)

    def append(self, layer: int, xq, xk, xv, gamma_q, gamma_k, q_out) -> None:
        """xq [B, n_new, Hq, D], xk / xv [B, n_new, Hkv, D] (the projection outputs, FP32 or BF16, all the
        same type) are the n_new tokens after the `length` cached ones.  Writes q_out [B, Hq, n_new, D] BF16
        (rotated, normalised, times gamma_q) and the tokens' rows of this layer's K (same chain with gamma_k)
        and V (converted to BF16); with track_weights these rows begin without weight.  Except in a cache with the reference's
        rotation and nothing else, gamma_q and gamma_k may both be None: no norm."""
        if self._plain:
            return (_lib._host or _lib.host()).kv_append(self, layer, xq, xk, xv, gamma_q, gamma_k, q_out)
        self._layer_ok("append", layer)
        pos0, pos, rows = self._place()
        if rows is not None and pos is None:
            pos = rows if self._shift == 0 else rows + self._shift
        if rows is not None and isinstance(xq, torch.Tensor) and xq.dim() == 4 and xq.shape[1] != 1:
            raise ValueError("KVCache.append: one token per sequence once the lengths differ")
        _lib.host().append_rotary(xq, xk, xv, gamma_q, gamma_k, q_out, self._kl[layer], self._vl[layer],
                                  self.positions[layer] if self.track_weights else None, self.cos, self.sin, self._R, self._pairs, pos, pos0,
                                  rows, self.length, self.B, self.L_cap, self.Hq, self.Hkv, self.D, self.eps,
                                  self.weights[layer] if self.track_weights else None)

    def _layer_ok(self, what, layer):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"KVCache.{what}: layer {layer} out of range")

    def attend(self, layer: int, q, ctx, lse, n_new: int = 1, softmax_scale=None, new_lens=None) -> None:
        """Attention of the n_new appended tokens over the length + n_new cached ones.  q, ctx: [B, Hq, n_new, D]
        BF16; lse: [B, Hq, n_new] FP32 (may be None for n_new == 1).  n_new == 1 is the split-KV decode kernel;
        n_new > 1 is the causal forward of the new tokens over the cache: a whole prompt into an empty cache, or a
        further chunk of it behind the tokens already cached (chunked prefill; lock-step sequences only).
        Behind shared prompts: one token, over the prompt and the sequence's own tokens.  With track_weights the keys' weights grow by
        what these tokens give them; new_lens (int32 [B] on the device) says how many of the n_new tokens of each sequence are
        tokens and not padding, where the prompts of a batch differ in length (`set_lengths` follows)."""
        if self._alone and new_lens is None:
            return (_lib._host or _lib.host()).kv_attend(self, layer, q, ctx, lse, n_new, softmax_scale)
        if new_lens is not None and (not self.track_weights or n_new == 1):
            raise ValueError("KVCache.attend: new_lens is for several tokens at once, with track_weights")
        self._layer_ok("attend", layer)
        if n_new <= 0 or self.length + n_new > self.L_cap:
            raise ValueError("KVCache.attend: n_new out of range")
        h, k, v, L = _lib.host(), self._kl[layer], self._vl[layer], self.length + n_new
        if self.prefix is not None:
            if n_new != 1:
                raise ValueError("KVCache.attend: one token per sequence behind shared prompts")
            self._place()
            p = self.prefix
            h.decode_shared(q, p._kl[layer], p._vl[layer], k, v, ctx, lse, self.B, p.B, p.length, L, self.Hq, self.Hkv, self.D, p.lengths,
                            self._lens_next, softmax_scale, p.L_cap, self.L_cap)
        elif n_new == 1:
            h.decode_weights(q, k, v, ctx, lse, self.weights[layer], self.B, L, self.Hq, self.Hkv, self.D, self._lens_next, softmax_scale,
                             self.L_cap)
        else:
            h.kv_attend(self, layer, q, ctx, lse, n_new, softmax_scale)
            h.key_weights(q, k, lse, self.weights[layer], self.B, n_new, self.length, self.Hq, self.Hkv, self.D, softmax_scale, self.L_cap, "BHTD",
                          new_lens)

    def evict(self, keep: int, recent: int) -> None:
        """Cuts every layer down to at most `keep` rows per (sequence, KV head): the newest `recent` tokens and those of the largest
        weight (csrc/kv_evict.cuh).  Between steps, after `advance`.  Later tokens go on at their positions."""
        if not self.track_weights:
            raise ValueError("KVCache.evict: the cache keeps no weights (track_weights)")
        if keep <= 0 or not 0 <= recent <= keep:
            raise ValueError("KVCache.evict: need 0 <= recent <= keep and keep > 0")
        if self.length <= keep:
            return
        for i in range(self.n_layers):
            w2, p2 = self._spare
            _lib.host().kv_evict(self._kl[i], self._vl[i], self.weights[i], self.positions[i], w2, p2, self.B, self.length, self.Hkv, self.D, keep,
                                 recent, self.lengths, self.L_cap)
            self._spare = (self.weights[i], self.positions[i])
            self.weights[i], self.positions[i] = w2, p2
        self._changes += 1
        self._evicted = True
        if self.lengths is None:
            self._shift += self.length - keep
        else:
            if self._pos is None:
                self._pos = self.lengths + self._shift
            self._lengths_host = [min(x, keep) for x in self._lengths_host]
            self.lengths = self.lengths.clamp(max=keep)
            self._lens_next = self.lengths + 1
        self.length = keep

    def advance(self, n_new: int = 1) -> None:
        """Call once per step, after every layer has appended and attended."""
        if n_new <= 0 or self.length + n_new > self.L_cap:
            raise ValueError("KVCache.advance: n_new out of range")
        self._changes += 1
        self.length += n_new
        if self.lengths is not None:
            self._lengths_host = [x + n_new for x in self._lengths_host]
            self.lengths += n_new
            self._lens_next += n_new
        if self._pos is not None:
            self._pos += n_new
