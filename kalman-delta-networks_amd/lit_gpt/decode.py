"""Token-by-token decoding of a KDN ``GPT`` with the layers' recurrent state kept on the GPU.

The reference has no decoding path for KDN models (``model.py:104,184`` refuse caching).  Every
KDN layer's history is a fixed-size state (``KDNLayerState``), so a decode step costs the same at
any context length: the chunked scan consumes the prompt (``prefill``), then each ``step`` runs
one token through every block, the mixers through ``kdn_kalman_step``.

One decode step is a chain of small dependent kernels (5 to 9 per block for a bf16 model, ``decode_block``;
about 20 otherwise), so at small batch the step is bound by launch overhead as much as by the GPU.  With
``use_graph=True`` the step is captured once as a HIP graph (``torch.cuda.CUDAGraph``) over fixed buffers -- the token ids, the
logits and every layer's state -- and each later step is one graph replay.  The decoder's layer
states are in-place states (``KDNLayerState.inplace``): each layer advances its own buffers, the
mixers through ``kdn_kalman_step`` (the single-token gain and memory update in one launch).

A captured step reads the weights where they lay when it was captured.  The decoder keeps them, and the packed copies
beside them, from being released; it captures again at the first step after ``quantize_mx4``, and after a ``prefill``
that finds a parameter, buffer or part of the model exchanged or written since.
"""
from __future__ import annotations

import torch

from ._inference import StepSources
from .kdn_ops.sampling import sample_tokens
from .kdn_state import KDNLayerState


class KDNDecoder:
    def __init__(self, model, batch_size: int, *, use_graph: bool = True):
        self.model = model
        self.B = int(batch_size)
        self.use_graph = bool(use_graph)
        self.state = None
        self.graph = None
        self._sources = None
        dev = next(model.parameters()).device
        self.tokens = torch.zeros(self.B, 1, dtype=torch.long, device=dev)
        self.logits = None

    @torch.no_grad()
    def prefill(self, idx: torch.Tensor) -> torch.Tensor:
        """Run the prompt ``idx`` [B,T] (T >= 1) through the chunked scan; returns its logits [B,T,V]
        and keeps the state after it (copied into this decoder's fixed buffers)."""
        if idx.ndim != 2 or idx.shape[0] != self.B:
            raise ValueError(f"idx must have shape [{self.B}, T], got {tuple(idx.shape)}")
        if self.graph is not None and not self._sources.current():
            self._release()
        logits, state = self.model(idx, return_state=True)
        if self.state is None:
            self.state = [KDNLayerState(tuple(c.clone() for c in s.conv), s.memory.clone(), s.precision.clone(),
                                        s.seen_tokens, inplace=True) for s in state]
        else:
            self._assign(state)
            for s, n in zip(self.state, state):
                s.seen_tokens = n.seen_tokens
        return logits

    def _assign(self, new):
        for s, n in zip(self.state, new):
            s.memory.copy_(n.memory)
            s.precision.copy_(n.precision)
            for c, nc in zip(s.conv, n.conv):
                c.copy_(nc)

    def _release(self):
        """Drop the captured step, and what was kept for it: replays may still be running on any stream."""
        torch.cuda.synchronize(self.tokens.device)
        self.graph = self._sources = None

    def _eager_step(self):
        # the states are in-place states: the layers advance their buffers themselves
        logits, _ = self.model(self.tokens, state=self.state, return_state=True)
        # (captured, this tensor is the graph's own output buffer, rewritten by every replay)
        self.logits = logits[:, -1]

    def _capture(self):
        # warm up (library handles, allocator) on a side stream without advancing the state
        saved = [(s.memory.clone(), s.precision.clone(), tuple(c.clone() for c in s.conv), s.seen_tokens)
                 for s in self.state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                self._eager_step()
        torch.cuda.current_stream().wait_stream(side)
        for s, (m, p, cs, n) in zip(self.state, saved):
            s.memory.copy_(m)
            s.precision.copy_(p)
            for c, sc in zip(s.conv, cs):
                c.copy_(sc)
            s.seen_tokens = n
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._eager_step()
        self.graph, self._sources = graph, StepSources(self.model)
        for s, (_, _, _, n) in zip(self.state, saved):
            s.seen_tokens = n  # capture records the step without running it

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """Feed one token per sequence (``tokens`` [B] or [B,1]); returns the next-token logits [B,V]
        (with the graph a view of its output buffer, overwritten by the next step)."""
        if self.state is None:
            raise RuntimeError("call prefill() before step()")
        self.tokens.copy_(tokens.view(self.B, 1))
        if not self.use_graph:
            self._eager_step()  # advances seen_tokens itself
        else:
            if self.graph is not None and not self._sources.same_parts(self.model):
                self._release()
            if self.graph is None:
                self._capture()
            self.graph.replay()
            for s in self.state:
                s.seen_tokens += 1
        return self.logits

    @torch.no_grad()
    def generate(self, idx: torch.Tensor, max_new_tokens: int, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                 generator=None, vocab_size=None):
        """Runs the prompt ``idx`` [B,T] and draws ``max_new_tokens`` tokens after it, one per sequence and step, with
        ``sample_tokens`` (its settings: a number, or one per sequence); the random numbers come from ``generator``.
        ``vocab_size``: only the first so many tokens can be drawn (the model's logits are as many as its
        ``padded_vocab_size``, and no tokenizer has the padding's; the probabilities are those of the rest).
        Returns ``(tokens [B, max_new_tokens] int64, logprobs fp32)``.  A sequence without a token that can be drawn (its
        logits are all -inf or NaN) gets token -1, and goes on as if it were 0."""
        if max_new_tokens < 0:
            raise ValueError(f"max_new_tokens must be >= 0, got {max_new_tokens}")
        logits = self.prefill(idx)[:, -1]
        V = logits.shape[1] if vocab_size is None else vocab_size
        if not 1 <= V <= logits.shape[1]:
            raise ValueError(f"vocab_size must be 1 to {logits.shape[1]}, got {vocab_size}")
        dev = logits.device
        tokens = torch.empty((self.B, max_new_tokens), device=dev, dtype=torch.int64)
        logprobs = torch.empty((self.B, max_new_tokens), device=dev, dtype=torch.float32)
        greedy = not isinstance(temperature, torch.Tensor) and temperature == 0
        noise = None if greedy else torch.empty((self.B, V), device=dev, dtype=torch.float32)
        for i in range(max_new_tokens):
            if i:
                logits = self.step(tokens[:, i - 1].clamp_min(0))  # (-1 is no row of the embedding)
            if noise is not None:
                noise.exponential_(generator=generator)
            tokens[:, i], logprobs[:, i] = sample_tokens(logits if vocab_size is None else logits[:, :V], noise,
                                                         temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        return tokens, logprobs


__all__ = ("KDNDecoder",)
