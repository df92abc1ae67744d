"""Text from a trained GPT-mode model: ``python -m cme213_final_project_b200.generate --checkpoint model.ck --data inp.txt``.

The parts, each usable alone:

* :class:`PagedCache` -- keys and values of all layers in pages that sequences take and give back, so that sequences of different and
  growing lengths share one piece of memory.  One table serves all layers.  It holds the model's type, or 8-bit integers with a scale
  for each block of tokens and head (half the bytes of bf16, a quarter of fp32's).
* :class:`Generator` -- the model over such a cache: prompts in chunks, then one token per sequence and step.  Attention reads the cache
  (``ops.paged_attention``) after the new tokens' keys and values have joined it (``ops.cache_append``); ``ops.next_token`` makes the next
  tokens of the logits.  A decoding step stays on the device from its tokens to the next ones and replays as one CUDA graph.
  :meth:`Generator.beam_search` keeps several continuations of each prompt: ``ops.beam_step`` picks them and ``ops.cache_reorder`` lets them
  go on from one another's past.

The reference has no counterpart: it trains and reports its loss (``FINAL_CLEAN_CODE_/src/main.cu:134-495``).
"""
from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import torch

from .arena import ArenaLayout
from .config import ModelConfig


class CacheFull(RuntimeError):
    """No page is left for the tokens asked for."""


class PagedCache:
    """Keys and values of ``seqs`` sequences in ``pages`` pages of ``page`` slots, ``[layers, pages, heads, page, head_dim]`` each.

    The host keeps the books (which page belongs to whom, how long a sequence is); ``table`` is their copy on the device, where an
    entry of -1 means that a sequence has no page there.

    ``dtype`` int8: ``k_scales``, ``v_scales`` are ``[layers, pages, heads, page // block]``, a scale for each ``block`` slots (a multiple of 8
    that divides a page; 16 where that does, else 8).  For other types ``scales(layer)`` is empty."""

    def __init__(self, layers: int, heads: int, head_dim: int, seqs: int, max_len: int, pages: int, page: int = 16,
                 dtype=torch.bfloat16, device="cuda", block: Optional[int] = None) -> None:
        if page < 8 or page % 8:
            raise ValueError(f"pages of {page} slots: a multiple of 8 is needed")
        block = (8 if page % 16 else 16) if block is None else block
        if block < 8 or block % 8 or page % block:
            raise ValueError(f"scales of {block} slots: a multiple of 8 that divides a page of {page} is needed")
        self.page, self.max_len = page, max_len
        self.k = torch.empty(layers, pages, heads, page, head_dim, dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.k_scales = self.v_scales = None
        if dtype == torch.int8:
            self.k_scales = torch.empty(layers, pages, heads, page // block, dtype=torch.float32, device=device)
            self.v_scales = torch.empty_like(self.k_scales)
        self.table = torch.full((seqs, -(-max_len // page)), -1, dtype=torch.int32, device=device)
        self.lengths = [0] * seqs
        self.owned: List[List[int]] = [[] for _ in range(seqs)]
        self.free = list(range(pages - 1, -1, -1))
        self.shared = False                                # after fork(): pages of one sequence are in others' tables

    def scales(self, layer: Optional[int] = None) -> dict:
        """What ``ops.cache_append`` and ``ops.paged_attention`` are told of an int8 cache's layer, ``ops.cache_reorder`` of all."""
        if self.k_scales is None:
            return {}
        return {"k_scales": self.k_scales, "v_scales": self.v_scales} if layer is None else {"k_scales": self.k_scales[layer],
                                                                                             "v_scales": self.v_scales[layer]}

    def grow(self, new: Sequence[int]) -> None:
        """Give sequence ``b`` room for ``new[b]`` more tokens and count them as its own.  All sequences or none: raises
        :class:`CacheFull` or ``ValueError`` (beyond ``max_len``, or after :meth:`fork`) before anything has changed."""
        if self.shared:
            raise ValueError("the sequences of a search with beams have all the pages that they get")
        need = []
        for b, n in enumerate(new):
            length = self.lengths[b] + n
            if n < 0 or length > self.max_len:
                raise ValueError(f"sequence {b}: {length} tokens, {self.max_len} at the most")
            need.append(max(0, -(-length // self.page) - len(self.owned[b])))
        if sum(need) > len(self.free):
            raise CacheFull(f"{sum(need)} pages are needed, {len(self.free)} are free")
        rows, cols, ids = [], [], []
        for b, n in enumerate(need):
            for _ in range(n):
                rows.append(b)
                cols.append(len(self.owned[b]))
                ids.append(self.free.pop())
                self.owned[b].append(ids[-1])
            self.lengths[b] += new[b]
        if ids:
            at = torch.tensor([rows, cols, ids], dtype=torch.int64).to(self.table.device)
            self.table[at[0], at[1]] = at[2].to(torch.int32)

    def release(self, b: int) -> None:
        """Sequence ``b`` is over: its pages are free again."""
        if self.shared:
            raise ValueError("the sequences of a search with beams end together: clear()")
        self.free += reversed(self.owned[b])
        self.owned[b] = []
        self.lengths[b] = 0
        self.table[b] = -1

    def fits(self, lengths: Sequence[int]) -> None:
        """Raises what :meth:`grow` would if sequences of these lengths were all that is there."""
        for b, n in enumerate(lengths):
            if n > self.max_len:
                raise ValueError(f"sequence {b}: {n} tokens, {self.max_len} at the most")
        need, pages = sum(-(-n // self.page) for n in lengths), self.k.shape[1]
        if need > pages:
            raise CacheFull(f"{need} pages are needed, the cache has {pages}")

    def forked(self, lengths: Sequence[int], beams: int, new: int) -> int:
        """Pages of groups of ``beams`` sequences that share a prompt of ``lengths[group]`` tokens and get ``new`` more each.  Raises
        what :meth:`fits` raises."""
        need, pages = 0, self.k.shape[1]
        for g, n in enumerate(lengths):
            if n + new > self.max_len:
                raise ValueError(f"sequence {g}: {n + new} tokens, {self.max_len} at the most")
            full = n // self.page
            need += full + beams * (-(-(n + new) // self.page) - full + (beams > 1))
        if need > pages:
            raise CacheFull(f"{need} pages are needed, the cache has {pages}")
        return need

    def fork(self, beams: int, new: int) -> torch.Tensor:
        """The first sequence of each group of ``beams`` holds a prompt, the others nothing: give all of them room for ``new`` more
        tokens, and a spare page each (-1: a beam alone, which goes on from none but itself, needs none).  Returns these (int32 ``[seqs]``), as
        ``ops.cache_reorder`` takes them; that call with all parents 0 then lets the others go on from the prompt.  Until :meth:`clear` no
        sequence grows or is released.  Raises :class:`CacheFull` or ``ValueError`` before anything has changed."""
        if self.shared:
            raise ValueError("the sequences are beams already: clear()")
        if beams < 1 or len(self.owned) % beams or new < 0:
            raise ValueError(f"{len(self.owned)} sequences in groups of {beams}, room for {new} more tokens")
        if any(o for b, o in enumerate(self.owned) if b % beams):
            raise ValueError("the first sequence of each group has to be the only one that holds something")
        self.forked([self.lengths[b] for b in range(0, len(self.owned), beams)], beams, new)
        rows, cols, ids, spare = [], [], [], []
        for b in range(len(self.owned)):
            n = self.lengths[b - b % beams]
            for col in range(len(self.owned[b]) if b % beams == 0 else n // self.page, -(-(n + new) // self.page)):
                rows.append(b)
                cols.append(col)
                ids.append(self.free.pop())
                self.owned[b].append(ids[-1])
            spare.append(self.free.pop() if beams > 1 else -1)
            if beams > 1:
                self.owned[b].append(spare[-1])
        self.shared = True
        device = self.table.device
        if ids:
            at = torch.tensor([rows, cols, ids], dtype=torch.int64).to(device)
            self.table[at[0], at[1]] = at[2].to(torch.int32)
        return torch.tensor(spare, dtype=torch.int32).to(device)

    def clear(self) -> None:
        """All sequences are over."""
        self.shared = False
        for b in reversed(range(len(self.owned))):
            self.free += reversed(self.owned[b])
            self.owned[b] = []
            self.lengths[b] = 0
        self.table.fill_(-1)


@dataclass
class Sampling:
    """How a row's next token is picked (see ``ops.next_token``)."""
    temperature: float = 0.0            # 0: the most likely token
    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: Optional[dict] = None         # token -> what is added to its logit
    allowed: Optional[Sequence[int]] = None      # tokens that may follow; None: all

    def tensors(self, rows: int, vocab: int, device) -> dict:
        full = lambda v: torch.full((rows,), float(v), device=device)
        kw = dict(temperature=full(self.temperature), repetition=full(self.repetition), presence=full(self.presence),
                  frequency=full(self.frequency))
        if self.bias:
            kw["bias_ids"] = torch.tensor([list(self.bias)] * rows, dtype=torch.int32, device=device)
            kw["bias_values"] = torch.tensor([list(self.bias.values())] * rows, dtype=torch.float32, device=device)
        if self.allowed is not None:
            if any(not 0 <= t < vocab for t in self.allowed):
                raise ValueError(f"allowed tokens have to be of the vocabulary, 0 to {vocab - 1}")
            bits = torch.zeros(-(-vocab // 32) * 32, dtype=torch.int64)
            bits[torch.as_tensor(list(self.allowed), dtype=torch.int64)] = 1
            words = (bits.view(-1, 32) << torch.arange(32)).sum(1)
            kw["allowed"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).view(1, -1).to(device)
        return kw


class Generator:
    """The model with weights ``params`` (the flat arena of ``layout``, bf16 or fp32 on a GPU) and a cache for ``seqs`` sequences.
    fp32 weights are multiplied exactly, or with ``tf32`` on the tensor cores, as by the trainer's ``--compute-dtype fp32`` and ``tf32``.
    ``cache8``: the cache holds 8-bit integers.  ``beams``: for :meth:`beam_search`, so many of the sequences belong to one prompt."""

    def __init__(self, cfg: ModelConfig, layout: ArenaLayout, params: torch.Tensor, seqs: int, pages: Optional[int] = None,
                 page: int = 16, tf32: bool = False, cache8: bool = False, beams: int = 1) -> None:
        if cfg.mode != "gpt" or not cfg.causal or cfg.head_layout != "split":
            raise ValueError("generation needs a causal model (mode gpt): the parity model's attention looks ahead")
        if cfg.head_dim not in (32, 64, 128):
            raise ValueError(f"head size {cfg.head_dim}: the cache's kernels take 32, 64 and 128")
        if not 1 <= beams <= 32 or seqs % beams:
            raise ValueError(f"{beams} beams for {seqs} sequences: 1 to 32 that divide them are needed")
        self.cfg, self.seqs, self.beams = cfg, seqs, beams
        self.products = {"allow_tf32": 2 if tf32 else False} if params.dtype == torch.float32 else {}
        self.P = layout.views(params)
        columns = -(-cfg.seq_len // page)
        pages = pages or seqs * (columns + (beams > 1))   # (a spare page for each beam)
        self.cache = PagedCache(cfg.layers, cfg.heads, cfg.head_dim, seqs, cfg.seq_len, pages, page, torch.int8 if cache8 else params.dtype,
                                params.device)

    # -- the model over the cache -----------------------------------------------------------------
    def forward(self, tokens: torch.Tensor, positions: torch.Tensor, offsets: torch.Tensor, lengths: torch.Tensor,
                last: torch.Tensor) -> torch.Tensor:
        """Logits ``[seqs, vocab]`` after row ``last[b]`` of each sequence.  ``tokens``, ``positions``: of all new rows;
        ``offsets``, ``lengths``: as ``ops.paged_attention`` takes them."""
        from . import ops
        cfg, P, c = self.cfg, self.P, self.cache
        gemm = lambda *args, **kw: ops.gemm(*args, **kw, **self.products)
        N, D, H, HD = tokens.shape[0], cfg.hidden, cfg.heads, cfg.head_dim
        x = ops.add(P["tok_embed"].index_select(0, tokens), P["pos_embed"].index_select(0, positions))
        for l in range(cfg.layers):
            w = lambda name: P[f"h{l}.{name}"]
            h = ops.layernorm_fwd(x, w("ln1_gamma"), w("ln1_beta"), cfg.ln_eps)[0]
            qkv = gemm(h, w("Wqkv")).view(N, 3, H, HD)
            ops.cache_append(qkv[:, 1], qkv[:, 2], c.k[l], c.v[l], c.table, offsets, lengths, **c.scales(l))
            a, _ = ops.paged_attention(qkv[:, 0], c.k[l], c.v[l], c.table, offsets, lengths, **c.scales(l))
            x = gemm(a.view(N, D), w("Wo"), residual=x)
            h = ops.layernorm_fwd(x, w("ln2_gamma"), w("ln2_beta"), cfg.ln_eps)[0]
            f = gemm(h, w("W1"), bias=w("b1"), act=cfg.activation)
            x = gemm(f, w("W2"), bias=w("b2"), residual=x)
        x = x.index_select(0, last)
        if cfg.final_layernorm:
            x = ops.layernorm_fwd(x, P["lnf_gamma"], P["lnf_beta"], cfg.ln_eps)[0]
        return gemm(x, P["tok_embed"], b_trans=True) if cfg.tied_embeddings else gemm(x, P["Wout"])

    def prefill(self, prompts: Sequence[Sequence[int]], chunk: int = 512) -> torch.Tensor:
        """Start new sequences: take the prompts into the cache, up to ``chunk`` tokens of each at a time; logits after each prompt's last
        token.  What the cache held, of an earlier call or of one that failed, is given back first."""
        if len(prompts) != self.seqs or any(len(p) == 0 for p in prompts):
            raise ValueError(f"{self.seqs} prompts with a token at least are needed")
        if any(not 0 <= t < self.cfg.vocab_size for p in prompts for t in p):
            raise ValueError(f"prompts have to have tokens of the vocabulary, 0 to {self.cfg.vocab_size - 1}")
        if chunk < 1:
            raise ValueError(f"a chunk of {chunk} tokens: one at least is needed")
        self.cache.fits([len(p) for p in prompts])
        self.cache.clear()
        return self._take(prompts, chunk)

    def _take(self, prompts, chunk):
        """Prompts (some may be empty) into sequences that hold nothing."""
        device = self.cache.table.device
        out = None
        done = [0] * self.seqs
        while any(d < len(p) for d, p in zip(done, prompts)):
            part = [list(p[d:d + chunk]) for d, p in zip(done, prompts)]
            n = [len(t) for t in part]
            self.cache.grow(n)
            offsets = [0]
            for k in n:
                offsets.append(offsets[-1] + k)
            i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(device)
            tokens = i32([t for row in part for t in row])
            positions = i32([d + i for d, k in zip(done, n) for i in range(k)])
            logits = self.forward(tokens, positions, i32(offsets), i32(self.cache.lengths), i32([max(0, o - 1) for o in offsets[1:]]))
            done = [d + k for d, k in zip(done, n)]
            # rows whose prompt ended in this chunk
            ended = i32([k > 0 and d == len(p) for d, k, p in zip(done, n, prompts)]).bool()
            out = logits if out is None else torch.where(ended[:, None], logits, out)
        return out

    # -- a run ------------------------------------------------------------------------------------
    def generate(self, prompts: Sequence[Sequence[int]], max_new: int, sampling: Optional[Sampling] = None, seed: int = 0,
                 chunk: int = 512, cuda_graph: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
        """``max_new`` tokens after each prompt, as new sequences: ``(tokens [seqs, max_new], log-probabilities)`` on the device.  -1
        where the sampling's mask left no token (and from there on)."""
        from . import ops
        s, cfg, device = sampling or Sampling(), self.cfg, self.cache.table.device
        if max_new < 1:
            raise ValueError(f"max_new of {max_new}: one token at least is needed")
        if max(len(p) for p in prompts) + max_new > cfg.seq_len + 1:
            raise ValueError(f"prompts of up to {max(map(len, prompts))} tokens and {max_new} more: the model's positions end at {cfg.seq_len}")
        kw = s.tensors(self.seqs, cfg.vocab_size, device)
        self.cache.fits([len(p) + max_new - 1 for p in prompts])          # (the last token's key is not needed)
        logits = self.prefill(prompts, chunk)
        start = list(self.cache.lengths)
        self.cache.grow([max_new - 1] * self.seqs)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(device)
        given = i32(start)
        history = torch.zeros(self.seqs, cfg.seq_len + 1, dtype=torch.int32, device=device)
        for b, p in enumerate(prompts):
            history[b, :len(p)] = i32(list(p))
        told = given.clone()                                              # tokens of a sequence so far, on the device
        rows, noise = torch.arange(self.seqs, device=device), None
        offsets = i32(list(range(self.seqs + 1)))
        uniform = torch.Generator(device=device).manual_seed(seed)
        if s.temperature > 0:
            noise = torch.empty(self.seqs, cfg.vocab_size, device=device)

        def pick(logits):
            if noise is not None:
                kw["noise"] = -torch.log(-torch.log(noise))
            token, logprob, _ = ops.next_token(logits, history=history, lengths=told, prompts=given, **kw)
            history[rows, told.long()] = token
            told.add_(1)
            return token, logprob

        def step():
            told_now = told - 1                                           # the position of the newest token
            token = history[rows, told_now.long()].clamp_min(0)
            return pick(self.forward(token, told_now, offsets, told, rows))

        def draw():
            if noise is not None:
                noise.uniform_(1e-9, 1 - 1e-7, generator=uniform)

        draw()
        token, logprob = pick(logits)
        tokens, logprobs = [token], [logprob]
        graph = None
        for i in range(1, max_new):
            draw()
            if not cuda_graph or i < 3:                                   # two steps warm everything up
                token, logprob = step()
            else:
                if graph is None:
                    torch.cuda.synchronize(device)
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        token, logprob = step()
                graph.replay()
            tokens.append(token.clone())
            logprobs.append(logprob.clone())
        return self._ended(torch.stack(tokens, 1), torch.stack(logprobs, 1))

    # -- several continuations of a prompt -----------------------------------------------------------
    def beam_search(self, prompts: Sequence[Sequence[int]], max_new: int, end: Optional[int] = None, allowed: Optional[Sequence[int]] = None,
                    length_power: float = 0.0, chunk: int = 512, cuda_graph: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
        """The ``beams`` best continuations of each prompt that a search with so many beams finds, as new sequences: ``(tokens
        [prompts, beams, max_new], scores [prompts, beams])`` on the device, best first.  A score is the sum of the tokens'
        log-probabilities.  A continuation ends with token ``end`` (-1 behind it) and then stays as it is among the others, as long as its score is one
        of the best.  ``length_power``: the order of the results is that of score / (number of tokens) ** power.  ``allowed``: tokens that may
        follow.  A place for which no continuation was found has -1 and ``-inf``."""
        from . import ops
        cfg, n, device = self.cfg, self.beams, self.cache.table.device
        groups = self.seqs // n
        if len(prompts) != groups or any(len(p) == 0 for p in prompts):
            raise ValueError(f"{groups} prompts with a token at least are needed")
        if any(not 0 <= t < cfg.vocab_size for p in prompts for t in p):
            raise ValueError(f"prompts have to have tokens of the vocabulary, 0 to {cfg.vocab_size - 1}")
        if end is not None and not 0 <= end < cfg.vocab_size:
            raise ValueError(f"the end has to be a token of the vocabulary, 0 to {cfg.vocab_size - 1}")
        if chunk < 1:
            raise ValueError(f"a chunk of {chunk} tokens: one at least is needed")
        if max_new < 1:
            raise ValueError(f"max_new of {max_new}: one token at least is needed")
        if max(len(p) for p in prompts) + max_new > cfg.seq_len + 1:
            raise ValueError(f"prompts of up to {max(map(len, prompts))} tokens and {max_new} more: the model's positions end at {cfg.seq_len}")
        allowed = Sampling(allowed=allowed).tensors(1, cfg.vocab_size, device).get("allowed")
        c = self.cache
        c.forked([len(p) for p in prompts], n, max_new - 1)               # (the last token's key is not needed)
        c.clear()
        logits = self._take([list(prompts[b // n]) if b % n == 0 else [] for b in range(self.seqs)], chunk)[::n]
        start = [c.lengths[b] for b in range(0, self.seqs, n)]
        spare = c.fork(n, max_new - 1)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(device)
        held = i32(start)                                                 # tokens of a group's beams in the cache
        rows, offsets = torch.arange(self.seqs, device=device), i32(list(range(self.seqs + 1)))
        first_row = (rows // n * n).view(groups, n)
        history = torch.full((self.seqs, max_new), -1, dtype=torch.int32, device=device)
        finished = torch.zeros(groups, n, dtype=torch.bool, device=device)
        scores = torch.zeros(groups, 1, device=device)
        newest = torch.zeros((), dtype=torch.int64, device=device)        # column of the newest tokens

        def keep(parents, token):
            """The beams that were picked take the places of their parents."""
            pages, new_spare = ops.cache_reorder(c.k, c.v, c.table, spare, parents, held, **c.scales())
            c.table.copy_(pages)
            spare.copy_(new_spare)
            of = parents.long()
            history.copy_(history[(first_row + of).view(-1)])
            history.index_copy_(1, newest.view(1), token.view(-1, 1))
            history.masked_fill_((scores == -torch.inf).view(-1, 1), -1)      # (no continuation: none of a past one either)
            over = finished.gather(1, of)
            finished.copy_(over if end is None else over | (token == end))

        def step():
            token = history.index_select(1, newest.view(1)).view(-1).clamp_min(0)
            positions = held.repeat_interleave(n)
            held.add_(1)
            newest.add_(1)
            logits = self.forward(token, positions, offsets, positions + 1, rows)
            parents, token, best = ops.beam_step(logits, scores, finished=finished, allowed=allowed)
            scores.copy_(best)
            keep(parents, token)

        parents, token, scores = ops.beam_step(logits, scores, n, allowed=allowed)      # (the parents are all the first one)
        keep(torch.zeros_like(parents), token)
        graph = None
        for i in range(1, max_new):
            if end is not None and i % 16 == 0 and bool((finished | (scores == -torch.inf)).all()):
                break
            if not cuda_graph or i < 3:                                   # two steps warm everything up
                step()
            else:
                if graph is None:
                    torch.cuda.synchronize(device)
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        step()
                graph.replay()
        tokens = history.view(groups, n, max_new)
        if length_power:
            count = (tokens >= 0).sum(2).clamp_min(1)
            order = (scores / count ** length_power).sort(dim=1, descending=True, stable=True).indices
            tokens, scores = tokens.gather(1, order[:, :, None].expand_as(tokens)), scores.gather(1, order)
        return tokens, scores

    @staticmethod
    def _ended(tokens, logprobs):
        over = (tokens < 0).cumsum(1) > 0
        return torch.where(over, -1, tokens), torch.where(over, float("-inf"), logprobs)


# --------------------------------------------------------------------------------------------------
# Command line
# --------------------------------------------------------------------------------------------------
def build_parser() -> argparse.ArgumentParser:
    p = argparse.ArgumentParser(prog="generate", description="text from a trained GPT-mode model")
    p.add_argument("--checkpoint", required=True, help="written by train --save-checkpoint")
    p.add_argument("--data", help="the corpus that the model was trained on: its characters are the vocabulary (else token numbers are printed)")
    p.add_argument("--prompt", action="append", help="text, or token numbers with commas without --data; may come several times")
    p.add_argument("--max-new", type=int, default=128)
    p.add_argument("--temperature", type=float, help="0: the most likely token every time (default: 0.8)")
    p.add_argument("--repetition", type=float, default=1.0)
    p.add_argument("--presence", type=float, default=0.0)
    p.add_argument("--frequency", type=float, default=0.0)
    p.add_argument("--beams", type=int, default=0, help="search for the most likely texts with so many beams (up to 32), and print them all")
    p.add_argument("--end", help="with --beams: the character of the corpus (without --data: the token number) that ends a text")
    p.add_argument("--length-power", type=float, default=0.0, help="with --beams: order by log-probability / tokens ** power")
    p.add_argument("--allow", help="only these characters of the corpus may come (with --data)")
    p.add_argument("--seed", type=int, default=0)
    p.add_argument("--chunk", type=int, default=512, help="tokens of a prompt that are taken in at a time")
    p.add_argument("--page", type=int, default=16, help="slots of a cache page")
    p.add_argument("--compute-dtype", default="bf16", choices=("bf16", "tf32", "fp32"))
    p.add_argument("--cache-dtype", default="model", choices=("model", "int8"),
                   help="int8: keys and values as 8-bit integers with a scale for each block of tokens and head")
    p.add_argument("--no-cuda-graph", action="store_true")
    return p


def main(argv: Optional[Sequence[str]] = None) -> int:
    a = build_parser().parse_args(argv)
    from .checkpoint import load_checkpoint
    from .data import CharTokenizer, read_file
    try:
        layout, flat, _, _, _, header = load_checkpoint(a.checkpoint, None)
        tok = CharTokenizer().build(read_file(a.data)) if a.data else None
    except (OSError, ValueError) as e:
        print(f"Error: {e}", file=sys.stderr)
        return 1
    cfg = layout.cfg
    if tok is not None and tok.vocab_size != cfg.vocab_size:
        print(f"Error: {a.data} has {tok.vocab_size} characters, the model {cfg.vocab_size}", file=sys.stderr)
        return 1
    texts = a.prompt or (["\n"] if tok else ["0"])
    try:
        prompts = [tok.encode(t).tolist() if tok else [int(i) for i in t.split(",")] for t in texts]
        if any(not 0 <= t < cfg.vocab_size for p in prompts for t in p) or not all(prompts):
            raise ValueError("prompts have to have tokens of the model's vocabulary")
        allowed = None
        if a.allow is not None:
            if tok is None:
                raise ValueError("--allow names characters: it needs --data")
            allowed = tok.encode(a.allow).tolist()
            if not allowed or len(allowed) < len(a.allow.encode("utf-8")):
                raise ValueError(f"--allow has to name characters of {a.data}")
        if not 0 <= a.beams <= 32:
            raise ValueError(f"--beams of {a.beams}: up to 32")
        if a.beams and (a.temperature is not None or a.repetition != 1.0 or a.presence or a.frequency):
            raise ValueError("--beams finds the most likely texts: --temperature and penalties are not for it")
        if not a.beams and (a.end is not None or a.length_power):
            raise ValueError("--end and --length-power go with --beams")
        end = None
        if a.end is not None:
            ends = tok.encode(a.end).tolist() if tok else [int(a.end)]
            if len(ends) != 1 or not 0 <= ends[0] < cfg.vocab_size or (tok and len(a.end.encode("utf-8")) != 1):
                raise ValueError("--end has to name one token of the model's vocabulary")
            end = ends[0]
        if not torch.cuda.is_available():
            raise ValueError("generation needs a GPU")
        dtype = torch.bfloat16 if a.compute_dtype == "bf16" else torch.float32
        # (on the device tensors start at multiples of 64 elements, as the engine lays them)
        aligned = ArenaLayout(cfg, align=64)
        params = torch.zeros(aligned.total, dtype=dtype, device="cuda")
        for name, view in layout.views(flat).items():
            aligned.views(params)[name].copy_(view)
        beams = max(1, a.beams)
        gen = Generator(cfg, aligned, params, len(prompts) * beams, page=a.page, tf32=a.compute_dtype == "tf32", cache8=a.cache_dtype == "int8",
                        beams=beams)
        if a.beams:
            tokens, scores = gen.beam_search(prompts, a.max_new, end, allowed, a.length_power, a.chunk, not a.no_cuda_graph)
        else:
            sampling = Sampling(0.8 if a.temperature is None else a.temperature, a.repetition, a.presence, a.frequency, None, allowed)
            tokens, logprobs = gen.generate(prompts, a.max_new, sampling, a.seed, a.chunk, not a.no_cuda_graph)
    except (ValueError, CacheFull) as e:
        print(f"Error: {e}", file=sys.stderr)
        return 1
    from . import ops
    rows = tokens.tolist()
    if ops.attention_check_status() or ops.gemm_check_status():
        print("Error: a bounded device wait ran out", file=sys.stderr)
        return 1
    if a.beams:
        for p, found, best in zip(prompts, rows, scores.tolist()):
            for row, score in zip(found, best):
                row = [i for i in row if i >= 0]
                print((tok.decode(p + row).decode("utf-8", "replace")) if tok else ",".join(map(str, p + row)))
                print(f"-- {len(row)} tokens, log-probability {score:.3f}")
        return 0
    for t, p, row, lp in zip(texts, prompts, rows, logprobs.tolist()):
        row = [i for i in row if i >= 0]
        print((tok.decode(p + row).decode("utf-8", "replace")) if tok else ",".join(map(str, p + row)))
        print(f"-- {len(row)} tokens, mean log-probability {sum(lp[:len(row)]) / max(1, len(row)):.3f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
