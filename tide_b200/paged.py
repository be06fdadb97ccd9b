"""A paged KV cache and live decoding over it: requests of different lengths,
which come, grow and end on their own.

The cache keeps every request's keys and values in pages of one pool; which
pages those are, the free ones, and where the new tokens of a step go is worked
out on the GPU from the requests' lengths (tide_page_tables), so that a decode
step reads nothing back and can be captured as a CUDA graph.  The reference has
no counterpart: its decode loop keeps the model's own cache and one length for
the whole batch (python/TIDE/runtime.py:223-313).
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from tide_b200.live import LiveDecoder, _StepBuffers


class PagedKVCache:
    """Keys and values [n_pages, kv_heads, page_size, head_dim] per layer, and
    the requests' block tables and lengths, on the device."""

    def __init__(self, n_layers: int, n_requests: int, n_pages: int, page_size: int, kv_heads: int,
                 head_dim: int, max_len: int, dtype: torch.dtype, device: torch.device,
                 error_word: Optional[torch.Tensor] = None):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two of at least 16")
        if not 1 <= n_requests <= 8192:
            raise ValueError("1 to 8192 requests")
        shape = (n_pages, kv_heads, page_size, head_dim)
        self.k = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.page_size, self.max_len, self.n_requests = page_size, max_len, n_requests

        def i32(*size, value=0):
            return torch.full(size, value, dtype=torch.int32, device=device)

        self.block_tables = i32(n_requests, -(-max_len // page_size), value=-1)
        self.kv_lens = i32(n_requests)
        self.free_pages = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.n_free = i32(1, value=n_pages)
        self.cu_seqlens = i32(n_requests + 1)
        self.error_word = i32(1) if error_word is None else error_word

    def advance(self, new_lens: torch.Tensor, slot_map: torch.Tensor, positions: torch.Tensor,
                done: Optional[torch.Tensor] = None) -> None:
        """Room for new_lens[r] (int32) more tokens of request r, whose slots
        and positions go to slot_map and positions (int64, as many entries as
        there are new tokens or more) and whose packed offsets to cu_seqlens;
        the requests with done[r] != 0 (int32) start over first."""
        from tide_b200 import _native

        _native.ops().page_tables(self.kv_lens, new_lens, done, self.free_pages, self.n_free,
                                  self.block_tables, self.page_size, self.n_free, self.kv_lens,
                                  self.cu_seqlens, slot_map, positions, self.error_word)

    def append(self, layer: int, k: Optional[torch.Tensor], v: Optional[torch.Tensor],
               slot_map: torch.Tensor, row_ids: Optional[torch.Tensor] = None,
               n_rows: Optional[torch.Tensor] = None) -> None:
        """Row i of k and v [n, kv_heads, head_dim] to slot_map[row_ids[i]]
        (None: zeros to every slot)."""
        from tide_b200 import _native

        _native.ops().paged_append(k, v, slot_map, row_ids, n_rows, self.k[layer], self.v[layer],
                                   self.error_word)

    def attend(self, layer: int, q: torch.Tensor, scale: float, *, chunk: bool,
               seq_ids: Optional[torch.Tensor] = None,
               n_seqs: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of q [n, heads, head_dim]: the packed new tokens of all
        requests (chunk), or one row per request, of request seq_ids[i]."""
        from tide_b200 import _native

        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _native.ops().paged_attention(q, self.k[layer], self.v[layer], self.block_tables,
                                      self.kv_lens, self.cu_seqlens if chunk else None, seq_ids, out,
                                      self.max_len, scale, self.error_word, n_seqs)
        return out


class PagedLiveDecoder(LiveDecoder):
    """LiveDecoder (per-row early exit that skips layers, each step one CUDA
    graph replay with graph=True) over a PagedKVCache: `extend` appends any
    number of prompt tokens to any of the requests, in one or several chunks,
    and starts requests over; `step` decodes one token of some or all of the
    requests, whatever their lengths.  A row that exits leaves zeros at its
    position in the later layers (the reference's "zero_pad",
    python/TIDE/runtime.py:194-221).  The host keeps the lengths too and
    refuses a step that the pool has no pages for."""

    def __init__(self, runtime, n_requests: int, max_len: int, n_pages: Optional[int] = None,
                 page_size: int = 64, graph: bool = False, fused_layers: bool = True):
        super().__init__(runtime, 1, 1, graph=graph, fused_layers=fused_layers)
        fam = self.fam
        if n_pages is None:
            n_pages = n_requests * -(-max_len // page_size)
        self.cache = PagedKVCache(len(fam.layers), n_requests, n_pages, page_size, fam.kv_heads(),
                                  fam.head_dim(), max_len, self.dtype, self.dev, self.err)
        self.k, self.v = self.cache.k, self.cache.v
        self.n_slots, self.max_len, self.n_pages = n_requests, max_len, n_pages
        self.lengths: List[int] = [0] * n_requests  # the device's kv_lens, as the host knows them
        self._requests: List[int] = []

    @property
    def length(self) -> int:
        """Positions held by the longest request."""
        return max(self.lengths)

    def fill_random(self, length: int, generator: torch.Generator) -> None:
        """Every request starts over with N(0,1) keys and values at positions
        0..length-1."""
        lens = self._take([0] * self.n_slots, [length] * self.n_slots)
        n = length * self.n_slots
        slot_map = torch.empty(max(n, 1), dtype=torch.int64, device=self.dev)
        self.cache.advance(self._i32([length] * self.n_slots), slot_map, torch.empty_like(slot_map),
                           self._i32([1] * self.n_slots))
        self.lengths = lens
        for c in self.k + self.v:
            c.copy_(torch.randn(c.shape, generator=generator, device=c.device))

    def _i32(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32, device=self.dev)

    def _take(self, lengths: Sequence[int], new: Sequence[int]) -> List[int]:
        """The lengths with `new` more positions each, or an error."""
        lens = [a + n for a, n in zip(lengths, new)]
        if max(lens) > self.max_len:
            raise RuntimeError("the live decoder's cache is full")
        if sum(-(-n // self.cache.page_size) for n in lens) > self.n_pages:
            raise RuntimeError("the live decoder's cache has no pages left")
        return lens

    # ---- one layer on rows whose slots and positions are known
    def _qkv(self, i: int, h: torch.Tensor, positions: torch.Tensor, places: torch.Tensor,
             n_live: Optional[torch.Tensor]):
        """Rotated q, rotated k, and v of rows h at the given positions
        (places: 0, 1, 2, ... in int32)."""
        from tide_b200 import _native

        fam, layer = self.fam, self.fam.layers[i]
        attn = layer.self_attn
        n = h.shape[0]
        if not self.fused:
            q, k, v = fam._qkv(layer, h, positions)
            return (q.to(self.dtype).contiguous(), k.to(self.dtype).contiguous(),
                    v.to(self.dtype).contiguous())
        x, _ = fam.rms_norm(layer.input_layernorm, h, n_live)
        w, b = fam._qkv_weight(i, attn)
        qkv = torch.nn.functional.linear(x, w, b)
        dq, dk = attn.q_proj.out_features, attn.k_proj.out_features
        q = qkv[:, :dq].view(n, -1, 128)
        k = qkv[:, dq:dq + dk].view(n, -1, 128)
        v = qkv[:, dq + dk:].view(n, -1, 128)
        qn, kn = getattr(attn, "q_norm", None), getattr(attn, "k_norm", None)
        q_rot = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        # (each row its own place in a cache of one position a row)
        k_new = torch.empty(n, k.shape[1], 1, 128, dtype=k.dtype, device=k.device)
        v_new = torch.empty_like(k_new)
        _native.ops().qk_norm_rope(
            q, k, v, qn.weight if qn is not None else None, kn.weight if kn is not None else None,
            float(qn.variance_epsilon) if qn is not None else 0.0, fam._inv_freq(),
            float(getattr(fam.rotary, "attention_scaling", 1.0)), 0, None, positions, places, n_live,
            q_rot, k_new, v_new, None)
        return q_rot, k_new.view(n, -1, 128), v_new.view(n, -1, 128)

    def _rest(self, i: int, h: torch.Tensor, o: torch.Tensor,
              n_live: Optional[torch.Tensor]) -> torch.Tensor:
        """The layer after its attention."""
        from tide_b200 import _native

        fam, layer = self.fam, self.fam.layers[i]
        o = layer.self_attn.o_proj(o.view(h.shape[0], -1))
        mlp = layer.mlp
        if not self.fused:
            h = h + o
            return h + mlp(layer.post_attention_layernorm(h))
        x, h = fam.rms_norm(layer.post_attention_layernorm, h, n_live, delta=o)
        g = mlp.gate_proj(x)
        act = torch.empty_like(g)
        _native.ops().silu_mul(g, mlp.up_proj(x), act, n_live)
        return h + mlp.down_proj(act)

    # ---- prompts
    @torch.no_grad()
    def extend(self, tokens: torch.Tensor, new_lens: Sequence[int],
               done: Optional[Sequence[bool]] = None) -> Optional[torch.Tensor]:
        """Append new_lens[r] of the packed tokens (in order of requests) to
        every request r, after the requests with done[r] have given their
        pages back and started over; every layer, no exits.  Returns the
        logits of each request's last new token [n_requests, V] (zeros for one
        without any), or None when there are no tokens at all.  Raises if a
        kernel has flagged a device error (what the call has added to the
        requests is then not to be used: they start over with done)."""
        new = [int(n) for n in new_lens]
        over = [False] * self.n_slots if done is None else [bool(d) for d in done]
        if len(new) != self.n_slots or len(over) != self.n_slots or min(new) < 0 \
                or sum(new) != tokens.numel():
            raise ValueError("new_lens and done: an entry for every request, and as many tokens as "
                             "new_lens adds up to")
        lens = self._take([0 if o else n for o, n in zip(over, self.lengths)], new)
        n = sum(new)
        tokens = tokens.reshape(1, -1).to(self.dev)
        slot_map = torch.empty(max(n, 1), dtype=torch.int64, device=self.dev)
        positions = torch.empty_like(slot_map)
        self.cache.advance(self._i32(new), slot_map, positions, self._i32([int(o) for o in over]))
        self.lengths = lens
        if n == 0:
            return None
        places = torch.arange(n, dtype=torch.int32, device=self.dev)
        h = self.fam.embed_tokens(tokens)
        for i in range(len(self.fam.layers)):
            q, k, v = self._qkv(i, h, positions, places, None)
            self.cache.append(i, k, v, slot_map)
            o = self.cache.attend(i, q, float(self.fam.layers[i].self_attn.scaling), chunk=True)
            h = self._rest(i, h, o, None)
        got = [r for r in range(self.n_slots) if new[r]]
        ends = torch.cumsum(torch.tensor(new), 0)[got] - 1
        ends = ends.to(self.dev)  # (waits for the layers)
        self.runner.check_errors()
        logits = self.rt._lm_head(self.fam.norm(h.index_select(0, ends)))
        if len(got) == self.n_slots:
            return logits
        full = logits.new_zeros(self.n_slots, logits.shape[1])
        return full.index_copy_(0, torch.tensor(got, device=self.dev), logits)

    def prefill(self, input_ids: torch.Tensor,
                attention_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The prompts of requests 0..B-1 without their padding, every request
        starting over; returns the last tokens' logits [B, V]."""
        B = input_ids.shape[0]
        if attention_mask is None:
            tokens, lens = input_ids.reshape(-1), [input_ids.shape[1]] * B
        else:
            if attention_mask.shape != input_ids.shape:
                raise ValueError("attention_mask must be [batch, seq]")
            keep = attention_mask.bool()
            tokens, lens = input_ids[keep], keep.sum(1).tolist()
        if B > self.n_slots or min(lens) < 1:
            raise ValueError("a prompt without tokens, or more prompts than requests")
        return self.extend(tokens, lens + [0] * (self.n_slots - B), [True] * self.n_slots)[:B]

    # ---- decode steps
    @torch.no_grad()
    def step(self, tokens: torch.Tensor, stats=None,
             requests: Optional[Sequence[int]] = None) -> torch.Tensor:
        """One decode step: tokens[i] is the next token of request requests[i]
        (ascending; None: of request i); the others stay as they are.  Returns
        the next logits [B, V] in the tokens' order, as LiveDecoder.step."""
        B = tokens.shape[0]
        req = list(range(B)) if requests is None else [int(r) for r in requests]
        if len(req) != B or B < 1 or req[0] < 0 or req[-1] >= self.n_slots \
                or any(a >= b for a, b in zip(req, req[1:])):
            raise ValueError("requests: ascending, one per token, below the number of requests")
        self._requests = req
        return super().step(tokens, stats)

    def _prepare(self, b: _StepBuffers) -> None:
        new = [0] * self.n_slots
        for r in self._requests:
            new[r] = 1
        self._next = self._take(self.lengths, new)
        if getattr(b, "requests", None) != self._requests:
            b.requests = list(self._requests)
            b.slots0.copy_(torch.tensor(self._requests, dtype=torch.int32))
            if not hasattr(b, "new_lens"):
                b.new_lens = self._i32(new)
            else:
                b.new_lens.copy_(torch.tensor(new, dtype=torch.int32))

    def _advanced(self, b: _StepBuffers) -> None:
        self.lengths = self._next

    def _begin(self, b: _StepBuffers) -> None:
        b.slot_map = torch.empty(b.B, dtype=torch.int64, device=self.dev)
        b.positions = torch.empty_like(b.slot_map)
        self.cache.advance(b.new_lens, b.slot_map, b.positions)
        b.places = torch.arange(b.B, dtype=torch.int32, device=self.dev)
        b.live_rows, b.row_ids, b.live_positions = b.rows0, b.places, b.positions

    def _layer(self, b: _StepBuffers, i: int, h: torch.Tensor, rows: torch.Tensor,
               slots: torch.Tensor, n_live: torch.Tensor) -> torch.Tensor:
        if rows is not b.live_rows:  # compacted since the last layer; past the live ones: anything
            b.live_rows, b.row_ids = rows, rows.to(torch.int32)
            b.live_positions = b.positions.index_select(0, rows.clamp(0, b.B - 1))
        q, k, v = self._qkv(i, h, b.live_positions, b.places, n_live)
        if rows is not b.rows0:  # some may have exited: zeros in their place
            self.cache.append(i, None, None, b.slot_map)
        self.cache.append(i, k, v, b.slot_map, b.row_ids, n_live)
        o = self.cache.attend(i, q, float(self.fam.layers[i].self_attn.scaling), chunk=False,
                              seq_ids=slots, n_seqs=n_live)
        return self._rest(i, h, o, n_live)

    def _end(self, b: _StepBuffers) -> None:
        pass

    def _state(self):
        return self.cache.kv_lens.clone(), self.cache.n_free.clone()

    def _undo(self, saved) -> None:
        # (what was written past the lengths is not read)
        self.cache.kv_lens.copy_(saved[0])
        self.cache.n_free.copy_(saved[1])
