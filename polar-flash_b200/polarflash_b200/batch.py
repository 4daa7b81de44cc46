"""Several conversations at once over packed layers: a paged KV cache, packed
prompts, batched decode steps and sampling.

``PFlashDecoder`` mirrors the reference's single-sequence forward
(polarflash_core/model_integration.py:203-254); ``BatchDecoder`` runs the same
blocks (RMSNorm :27-37, half-split RoPE :40-60, GQA attention :63-147, SwiGLU
:150-163) for up to ``max_seqs`` sequences of different lengths, with the
serving operators in place of the single-sequence kernels: ``paged_rope_kv``
writes rotated keys and values into pages, ``prompt_attention`` runs the
prompts packed into one batch, ``paged_attention`` the new tokens over the
pages, ``sample_logits`` draws the next ones.  There is no CPU path.
"""
import ctypes
from typing import Dict, List, Optional, Sequence

import torch

from . import _lib
from .decode import DecoderLayer
from .qweight import group_workspace_bytes, qlinear_multi
from .serving import (KVPages, PAGE_MODES, PAGE_SIZES, check_serving_status, paged_attention,
                      paged_attention_workspace_bytes, paged_rope_kv, prompt_attention, sample_logits)


def _p(t: Optional[torch.Tensor]):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


class PageAllocator:
    """Which pages are free (host side): the last ones given back go out first."""

    def __init__(self, num_pages: int):
        self._free = list(range(num_pages - 1, -1, -1))

    def __len__(self) -> int:
        return len(self._free)

    def take(self, n: int) -> List[int]:
        if n > len(self._free):
            raise RuntimeError(f"{n} cache pages needed, {len(self._free)} free")
        return [self._free.pop() for _ in range(n)]

    def give(self, pages: Sequence[int]) -> None:
        self._free.extend(reversed(pages))


class BatchDecoder:
    """Causal LM over packed layers for up to `max_seqs` sequences.

    config, layers, embed, final_norm and lm_head as PFlashDecoder's.  The cache
    is `num_pages` pages of `page_size` positions, shared by the sequences, each
    of at most `max_seq` tokens, in `kv_mode` ("fp16", "bf16", "int8", "2bit",
    "2bit_asym").  A prompt's own attention runs in `prompt_dtype` (fp16 or bf16)
    on its keys and values as they are; later tokens read them from the cache, as
    it holds them.  head_dim is 64 or 128.  Calls on one decoder stay on one
    stream of its device, which is the current one."""

    def __init__(self, config: Dict, layers: List[DecoderLayer], embed: torch.Tensor, final_norm: torch.Tensor,
                 lm_head: torch.Tensor, max_seqs: int, max_seq: int, num_pages: int, page_size: int = 64,
                 kv_mode: str = "int8", prompt_dtype: torch.dtype = torch.bfloat16):
        if kv_mode not in PAGE_MODES:
            raise ValueError(f"kv_mode {kv_mode!r}: one of {', '.join(PAGE_MODES)}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size {page_size}: one of {PAGE_SIZES}")
        if prompt_dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"prompt_dtype {prompt_dtype}: torch.float16 or torch.bfloat16")
        if max_seqs < 1 or max_seq < 1:
            raise ValueError("max_seqs and max_seq: at least one")
        self.hidden = int(config["hidden_size"])
        self.nh = int(config["num_attention_heads"])
        self.nkv = int(config["num_key_value_heads"])
        self.hd = self.hidden // self.nh
        if self.hd not in (64, 128):
            raise ValueError(f"head_dim {self.hd}: a paged cache holds heads of 64 or 128")
        self.eps = float(config.get("rms_norm_eps", 1e-6))
        self.layers, self.embed, self.final_norm, self.lm_head = layers, embed, final_norm, lm_head
        self.device = embed.device
        self.max_seqs, self.max_seq, self.page_size, self.prompt_dtype = max_seqs, max_seq, page_size, prompt_dtype
        self.width = -(-max_seq // page_size)
        dev = self.device
        half = self.hd // 2
        theta = float(config.get("rope_theta", 1000000.0))
        self.inv_freq = 1.0 / (theta ** (torch.arange(0, half, dtype=torch.float32, device=dev) / half))
        self.pages = [KVPages.empty(kv_mode, num_pages, page_size, self.nkv, self.hd, dev) for _ in layers]
        self.allocator = PageAllocator(num_pages)
        self.lengths = [0] * max_seqs                       # tokens of each slot; 0: free
        self.seq_pages: List[List[int]] = [[] for _ in range(max_seqs)]
        # what the step reads: a free slot has length 0 (its row is computed and means nothing)
        self._table = torch.full((max_seqs, self.width), -1, dtype=torch.int32, device=dev)
        self._lens = torch.zeros(max_seqs, dtype=torch.int32, device=dev)
        self._tok = torch.zeros(max_seqs, dtype=torch.long, device=dev)
        self._logits = torch.zeros(max_seqs, lm_head.shape[0], dtype=torch.float32, device=dev)
        need = 0
        for ly in layers:
            for group in ([ly.q, ly.k, ly.v], [ly.gate, ly.up], [ly.o], [ly.down]):
                need = max(need, group_workspace_bytes(group, max_seqs))
        self._ws = torch.zeros(need, dtype=torch.uint8, device=dev)
        self._attn_ws = torch.empty(paged_attention_workspace_bytes(self.nh, self.nkv, self.hd, max_seqs, dev),
                                    dtype=torch.uint8, device=dev)
        self._graph = None

    # ---- sequences ------------------------------------------------------------
    def active(self) -> List[int]:
        """The slots that hold a sequence."""
        return [i for i, n in enumerate(self.lengths) if n > 0]

    def _grow(self, slot: int, length: int) -> None:
        """Pages for `length` tokens of a slot, entered in its table row."""
        have = self.seq_pages[slot]
        more = -(-length // self.page_size) - len(have)
        if more > 0:
            new = self.allocator.take(more)
            self._table[slot, len(have):len(have) + more] = torch.tensor(new, dtype=torch.int32, device=self.device)
            have.extend(new)

    def release(self, slot: int) -> None:
        """Ends a slot's sequence; its pages are free."""
        self.allocator.give(self.seq_pages[slot])
        self.seq_pages[slot] = []
        self.lengths[slot] = 0
        self._lens[slot] = 0
        self._table[slot] = -1

    # ---- blocks -----------------------------------------------------------------
    def _norm(self, h: torch.Tensor, delta: Optional[torch.Tensor], w: torch.Tensor) -> torch.Tensor:
        """h += delta, and its RMSNorm (rows of fp32)."""
        out = torch.empty_like(h)
        st = ctypes.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)
        _lib.check(_lib.load().pf_add_rmsnorm(_p(h), _p(delta), _p(w), _p(out), h.shape[0], h.shape[1], self.eps, st),
                   "pf_add_rmsnorm")
        return out

    def _forward(self, ids: torch.Tensor, pos: torch.Tensor, attend, ws: Optional[torch.Tensor]) -> torch.Tensor:
        """The final norm's output of the tokens ids [T] at fp32 positions pos [T]."""
        L = _lib.load()
        f = pos[:, None] * self.inv_freq[None, :]
        cos, sin = torch.cos(f), torch.sin(f)
        h = self.embed.index_select(0, ids).float()
        T, delta = h.shape[0], None
        for li, ly in enumerate(self.layers):
            n = self._norm(h, delta, ly.input_norm)
            q, k, v = qlinear_multi([ly.q, ly.k, ly.v], n, ly.qkv_bias, workspace=ws)
            a = attend(li, q.view(T, self.nh, self.hd), k.view(T, self.nkv, self.hd), v.view(T, self.nkv, self.hd),
                       cos, sin)
            o = qlinear_multi([ly.o], a.view(T, self.hidden), workspace=ws)[0]
            g, u = qlinear_multi([ly.gate, ly.up], self._norm(h, o, ly.post_norm), workspace=ws)
            act = torch.empty_like(g)
            st = ctypes.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)
            _lib.check(L.pf_silu_mul(_p(g), _p(u), _p(act), g.numel(), st), "pf_silu_mul")
            delta = qlinear_multi([ly.down], act, workspace=ws)[0]
        return self._norm(h, delta, self.final_norm)

    def _head(self, hn: torch.Tensor) -> torch.Tensor:
        if self.lm_head.dtype == torch.float32:
            return hn @ self.lm_head.t()
        return (hn.to(self.lm_head.dtype) @ self.lm_head.t()).float()

    # ---- prompts ------------------------------------------------------------------
    def add(self, prompts: Sequence[torch.Tensor]):
        """Starts a sequence for each prompt (1-D token ids of the vocabulary, not
        empty) in a free slot: (slots, logits [len(prompts), vocab] of the
        prompts' last tokens).  Refused as a whole where slots or pages lack; taken
        back, with RuntimeError, where a wait of the prompts' attention gave up."""
        ids = [p.reshape(-1).to(self.device, torch.long) for p in prompts]
        lens = [len(i) for i in ids]
        free = [i for i, n in enumerate(self.lengths) if n == 0]
        if not ids:
            raise ValueError("no prompts")
        if min(lens) < 1 or max(lens) > self.max_seq:
            raise ValueError(f"prompts of {lens} tokens: 1 to {self.max_seq} each")
        if len(ids) > len(free):
            raise RuntimeError(f"{len(ids)} prompts, {len(free)} free slots")
        need = sum(-(-n // self.page_size) for n in lens)
        if need > len(self.allocator):
            raise RuntimeError(f"{need} cache pages needed, {len(self.allocator)} free")
        packed = torch.cat(ids)
        lo, hi = (int(x) for x in packed.aminmax())
        if lo < 0 or hi >= self.embed.shape[0]:
            raise ValueError(f"token ids {lo}..{hi}: 0 to {self.embed.shape[0] - 1}")
        slots = free[:len(ids)]
        try:
            out = self._add(slots, packed, lens)
            check_serving_status(self.device)
            return out
        except BaseException:
            for s in slots:
                self.release(s)
            raise

    def _add(self, slots: List[int], packed: torch.Tensor, lens: List[int]):
        for s, n in zip(slots, lens):
            self._grow(s, n)
        dev = self.device
        at = torch.tensor(slots, device=dev)
        lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
        cu = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
        table = self._table[at]
        pos = torch.cat([torch.arange(n, dtype=torch.float32, device=dev) for n in lens])

        def attend(li, q, k, v, cos, sin):
            q16, k16, v16 = paged_rope_kv(q, k, v, cos, sin, self.pages[li], table, lens_t, cu,
                                          out_dtype=self.prompt_dtype, return_kv=True)
            return prompt_attention(q16, k16, v16, cu)

        hn = self._forward(packed, pos, attend, None)
        self._lens[at] = lens_t
        for s, n in zip(slots, lens):
            self.lengths[s] = n
        return slots, self._head(hn[cu[1:].long() - 1])

    # ---- decode steps -----------------------------------------------------------------
    def _step_body(self):
        def attend(li, q, k, v, cos, sin):
            q, _, _ = paged_rope_kv(q, k, v, cos, sin, self.pages[li], self._table, self._lens, q_out=q)
            return paged_attention(q, self.pages[li], self._table, self._lens, workspace=self._attn_ws)

        hn = self._forward(self._tok, (self._lens - 1).clamp_min(0).float(), attend, self._ws)
        self._logits.copy_(self._head(hn))

    def capture(self):
        """Captures the step as a CUDA graph, replayed by every later step().
        No sequence may be active (the captured step runs once for real)."""
        if self.active():
            raise RuntimeError("BatchDecoder.capture: before the first prompt, or after the last release")
        dev = self.device
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            self._step_body()  # no slot has a token: nothing is cached
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                self._step_body()
        torch.cuda.current_stream(dev).wait_stream(s)
        self._graph = g
        return g

    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """Appends one token to every active sequence: tokens [max_seqs] (int64,
        on the device; free slots' entries are not looked at, an id outside the
        vocabulary counts as the nearest one in it) -> logits [max_seqs, vocab],
        in a buffer that the next step overwrites (free slots' rows mean
        nothing)."""
        act = self.active()
        if tokens.shape != (self.max_seqs,):
            raise ValueError(f"tokens {tuple(tokens.shape)}: [{self.max_seqs}] is needed")
        if tokens.device != self.device or tokens.is_floating_point() or tokens.is_complex():
            raise ValueError(f"tokens: token ids on {self.device} are needed, not {tokens.dtype} on {tokens.device}")
        if any(self.lengths[s] >= self.max_seq for s in act):
            raise ValueError(f"a sequence holds {self.max_seq} tokens")
        need = sum(self.lengths[s] % self.page_size == 0 for s in act)
        if need > len(self.allocator):
            raise RuntimeError(f"{need} cache pages needed, {len(self.allocator)} free")
        for s in act:
            self.lengths[s] += 1
            self._grow(s, self.lengths[s])
        on = self._lens > 0
        # -1 is drawn where no logit is above -inf: every id that is looked up is one of the embedding's
        self._tok.copy_(torch.where(on, tokens, 0).clamp(0, self.embed.shape[0] - 1))
        self._lens += on
        if self._graph is not None:
            self._graph.replay()
        else:
            self._step_body()
        return self._logits

    # ---- sampling ------------------------------------------------------------------
    def generate(self, prompts: Sequence[torch.Tensor], max_new_tokens: int, temperature=1.0, top_k=0, top_p=1.0,
                 min_p=0.0, eos: Optional[int] = None, generator: Optional[torch.Generator] = None) -> List[List[int]]:
        """The tokens drawn after each prompt (sample_logits' parameters, numbers
        for all sequences): max_new_tokens each, or up to and with `eos`.  The
        uniform numbers come from `generator` (on the device).  No other sequence
        may be active; these are released at the end.  Without `eos` a call that
        max_seq or the pages cannot hold is refused before it starts; with it a
        sequence that finds no room for its next token ends there, shorter."""
        if self.active():
            raise RuntimeError("BatchDecoder.generate: other sequences are active")
        if max_new_tokens < 1:
            return [[] for _ in prompts]
        if eos is None:
            held = [p.numel() + max_new_tokens - 1 for p in prompts]  # the last token drawn is not cached
            if held and max(held) > self.max_seq:
                raise ValueError(f"a sequence of {max(held)} tokens: at most {self.max_seq}")
            need = sum(-(-n // self.page_size) for n in held)
            if need > len(self.allocator):
                raise RuntimeError(f"{need} cache pages needed, {len(self.allocator)} free")
        slots, logits = self.add(prompts)
        kw = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        rand = lambda n: torch.rand(n, generator=generator, device=self.device)  # noqa: E731
        at = torch.tensor(slots, device=self.device)
        tokens = torch.zeros(self.max_seqs, dtype=torch.long, device=self.device)
        drawn = []
        live = set(slots)
        ends = {}  # tokens of the sequences that found no room

        def full(s):
            ends[s] = len(drawn)
            live.discard(s)
            self.release(s)

        try:
            tokens[at] = sample_logits(logits, rand(len(slots)), **kw)
            drawn.append(tokens[at].clone())
            for _ in range(max_new_tokens - 1):
                if eos is not None:  # the only reason to look at the tokens on the way
                    for s, t in zip(slots, drawn[-1].tolist()):
                        if t == eos and s in live:
                            live.discard(s)
                            self.release(s)
                    for s in [s for s in slots if s in live and self.lengths[s] >= self.max_seq]:
                        full(s)
                    turn = [s for s in slots if s in live and self.lengths[s] % self.page_size == 0]
                    while len(turn) > len(self.allocator):  # the last one's pages go to the others
                        full(turn.pop())
                    if not live:
                        break
                tokens.copy_(sample_logits(self.step(tokens), rand(self.max_seqs), **kw))
                drawn.append(tokens[at].clone())
            rows = torch.stack(drawn, 1).tolist()
            check_serving_status(self.device)
        finally:
            for s in live:
                self.release(s)
        if eos is None:
            return rows
        rows = [r[:ends.get(s)] for s, r in zip(slots, rows)]
        return [r[:r.index(eos) + 1] if eos in r else r for r in rows]
