"""What the requests of one batch share, and what sets them apart.

A :class:`~leanstack_b200.engine.DecodeEngine` runs a batch of sequences through
one set of weights.  Three resident objects let them be different requests of
one deployment (no counterpart in the reference, which runs one request):

* :class:`SharedPrefix`: the keys and values of a prompt prefix that all of them
  share (a system prompt, a document), held once per layer;
* :class:`AdapterBank`: low-rank adapters of the decoder linears, one per
  request or none;
* :class:`TokenRules`: each request's penalties, biases and grammar mask for the
  greedy pick, and the token counts that the penalties read.

All of their state lives in device tensors of fixed address, so a captured step
follows whatever is written into them between replays.
"""

from __future__ import annotations

import torch

from . import kernels as K
from .config import QwenGeometry


class SharedPrefix:
    """Key / value arenas ``[L, Hkv, capacity, D]``, the first ``length`` positions in use."""

    def __init__(self, geometry: QwenGeometry, capacity: int, device, dtype=torch.bfloat16):
        if capacity < 1:
            raise ValueError("prefix capacity must be positive")
        g = geometry
        shape = (g.num_hidden_layers, g.num_key_value_heads, capacity, g.head_dim)
        self.key = torch.zeros(shape, device=device, dtype=dtype)
        self.value = torch.zeros(shape, device=device, dtype=dtype)
        self.capacity = capacity
        self.length = 0


class AdapterBank:
    """Low-rank adapters of the decoder linears, stacked so that one launch serves every request of a batch.

    Per layer and target, ``a [adapters, rank, in]`` and ``b [adapters, out,
    rank]`` (bf16) beside the fused projections: ``qkv`` (q, k and v rows),
    ``o``, ``gate_up`` (gate rows, then up rows) and ``down``.  ``scaling`` is
    fp32 per adapter.  An adapter of a lower rank leaves the rest zero.
    """

    TARGETS = ("qkv", "o", "gate_up", "down")

    def __init__(self, geometry: QwenGeometry, adapters: int, rank: int, device, targets=TARGETS):
        if adapters < 1:
            raise ValueError("the bank needs room for an adapter")
        if rank < 8 or rank > 128 or rank % 8:
            raise ValueError(f"adapter rank {rank}: a multiple of 8 up to 128")
        unknown = [t for t in targets if t not in self.TARGETS]
        if unknown:
            raise ValueError(f"unknown adapter targets {unknown}; choose from {self.TARGETS}")
        self.shapes = self.linear_shapes(geometry)
        self.adapters, self.rank = adapters, rank
        self.targets = tuple(t for t in self.TARGETS if t in targets)
        self.scaling = torch.zeros(adapters, device=device, dtype=torch.float32)

        def z(*shape):
            return torch.zeros(shape, device=device, dtype=torch.bfloat16)

        self.layers = [{t: (z(adapters, rank, self.shapes[t][0]), z(adapters, self.shapes[t][1], rank))
                        for t in self.targets} for _ in range(geometry.num_hidden_layers)]

    @staticmethod
    def linear_shapes(g: QwenGeometry) -> dict[str, tuple[int, int]]:
        """(inputs, outputs) of each target's linear."""
        return {"qkv": (g.hidden_size, g.qkv_dim), "o": (g.q_dim, g.hidden_size),
                "gate_up": (g.hidden_size, 2 * g.intermediate_size), "down": (g.intermediate_size, g.hidden_size)}

    def load(self, index: int, weights: dict, scaling: float) -> None:
        """Put an adapter at ``index``: ``weights[(layer, target)] = (a [r, in], b [out, r])`` with r up to
        the bank's rank; linears that it does not name are left as they are by it."""
        if not 0 <= index < self.adapters:
            raise ValueError(f"adapter {index} outside the bank of {self.adapters}")
        for (layer, target), (a, b) in weights.items():
            if not 0 <= layer < len(self.layers) or target not in self.targets:
                raise ValueError(f"no {target!r} adapter in layer {layer} of this bank")
            k, n = self.shapes[target]
            r = a.shape[0]
            if a.shape != (r, k) or b.shape != (n, r) or r > self.rank:
                raise ValueError(f"{target}: a {tuple(a.shape)} and b {tuple(b.shape)} do not fit "
                                 f"[r <= {self.rank}, {k}] and [{n}, r]")
        for pair in (p for layer in self.layers for p in layer.values()):
            for t in pair:
                t[index].zero_()
        for (layer, target), (a, b) in weights.items():
            sa, sb = self.layers[layer][target]
            sa[index, :a.shape[0]].copy_(a)
            sb[index, :, :a.shape[0]].copy_(b)
        self.scaling[index] = float(scaling)


class TokenRules:
    """Penalties, biases and grammar masks of each sequence for the greedy pick (:func:`kernels.constrained_argmax`).

    ``seen`` marks the tokens of prompt and answer, ``counts`` counts the
    answer's; the engine keeps both.  The tokens of a shared prefix belong to
    every prompt: ``prefix_seen`` holds them, and whatever empties a row leaves
    them in it.  ``allowed`` (with ``grammar=True``) holds one bit per token, all
    set until a request's grammar writes its words.
    """

    def __init__(self, batch: int, vocab: int, device, max_biases: int = 0, grammar: bool = False):
        self.batch, self.vocab, self.words = batch, vocab, (vocab + 31) // 32

        def full(shape, value, dtype):
            return torch.full(shape, value, device=device, dtype=dtype)

        self.counts = full((batch, vocab), 0, torch.int32)
        self.seen = full((batch, self.words), 0, torch.int32)
        self.prefix_seen = full((1, self.words), 0, torch.int32)
        self.repetition = full((batch,), 1.0, torch.float32)
        self.frequency = full((batch,), 0.0, torch.float32)
        self.presence = full((batch,), 0.0, torch.float32)
        self.bias_ids = full((batch, max_biases), -1, torch.int32) if max_biases else None
        self.bias_values = full((batch, max_biases), 0.0, torch.float32) if max_biases else None
        self.allowed = full((batch, self.words), -1, torch.int32) if grammar else None
        self.workspace = torch.empty(K.constrained_argmax_workspace_bytes(batch, vocab), device=device,
                                     dtype=torch.uint8)

    def set_request(self, row: int, repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0,
                    biases: dict[int, float] | None = None) -> None:
        """The rules of the request in ``row``; its token counts start anew, behind the present prefix."""
        if not 0 <= row < self.batch:
            raise ValueError(f"row {row} outside the batch of {self.batch}")
        if not repetition > 0:
            raise ValueError("repetition must be positive")
        biases = biases or {}
        room = 0 if self.bias_ids is None else self.bias_ids.shape[1]
        if len(biases) > room:
            raise ValueError(f"{len(biases)} biases, room for {room}")
        if any(not 0 <= t < self.vocab for t in biases):
            raise ValueError("biased token outside the vocabulary")
        self.repetition[row], self.frequency[row], self.presence[row] = repetition, frequency, presence
        if room:
            ids = list(biases) + [-1] * (room - len(biases))
            values = list(biases.values()) + [0.0] * (room - len(biases))
            self.bias_ids[row].copy_(torch.tensor(ids, dtype=torch.int32))
            self.bias_values[row].copy_(torch.tensor(values, dtype=torch.float32))
        if self.allowed is not None:
            self.allowed[row].fill_(-1)
        self.counts[row].zero_()
        self.seen[row].copy_(self.prefix_seen[0])

    def restart(self) -> None:
        """Empty sequences in every row: no answer, and of the prompt only the shared prefix.  The rules stay."""
        self.counts.zero_()
        self.seen.copy_(self.prefix_seen.expand_as(self.seen))

    def set_prefix(self, ids: torch.Tensor) -> None:
        """The tokens ``ids [P]`` as every prompt's shared prefix, in place of the one before; the sequences are empty."""
        self.counts.zero_()
        self.seen.bitwise_and_(~self.prefix_seen)
        self.prefix_seen.zero_()
        K.token_stats_add(ids.view(1, -1), self.prefix_seen, self.vocab)
        self.seen.bitwise_or_(self.prefix_seen)

    def note_prompt(self, ids: torch.Tensor) -> None:
        """Mark the prompt tokens ``ids [batch, n]`` (negative: padding) as seen."""
        K.token_stats_add(ids, self.seen, self.vocab)

    def pick(self, logits: torch.Tensor, out_ids: torch.Tensor) -> None:
        """The next token of every sequence under its rules into ``out_ids``, entered into the counts."""
        K.constrained_argmax(logits, counts=self.counts, seen=self.seen, repetition=self.repetition,
                             frequency=self.frequency, presence=self.presence, bias_ids=self.bias_ids,
                             bias_values=self.bias_values, allowed=self.allowed, record=True, out_ids=out_ids,
                             workspace=self.workspace)
