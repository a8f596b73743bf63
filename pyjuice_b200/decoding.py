"""Answers of a language-model circuit: next-token distributions and beam search of a homogeneous hidden Markov model.

The circuit of an HMM (``structures.HMM``) evaluates a sentence from its end to its beginning; what decoding needs is the
other direction, the distribution of the next hidden state given the tokens so far.  :class:`HMMDecoder` carries that
distribution for every beam, one column each, and advances it with the sum and leaf kernels of two small circuits that hold
the model's parameters: one of the transitions, one of the emissions.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib, lm
from .model import TensorCircuit, compile
from .nodes import Categorical, inputs, multiply, summate


def _power_of_two(n: int, most: int) -> int:
    return min(n & -n, most)


def _padded(n: int) -> int:
    """States as the decoder holds them: in blocks of 64 nodes at least, so that the tiles of parameters are few and large (1000 states
    and 8000 tokens in blocks of 8: more than a second of host time for every layout)."""
    return -(-n // 64) * 64


def _dense(pc: TensorCircuit, ns) -> torch.Tensor:
    """Parameters of a fully connected sum vector, ``[nodes, children]``."""
    p = pc.get_node_params(ns)
    out = torch.zeros(ns.num_node_blocks, ns.num_ch_node_blocks, ns.block_size, ns.ch_block_size, device=p.device)
    out[ns.edge_ids[0].to(p.device), ns.edge_ids[1].to(p.device)] = p
    return out.permute(0, 2, 1, 3).reshape(ns.num_nodes, -1)


def _set_dense(pc: TensorCircuit, ns, weights: torch.Tensor):
    """Writes ``weights`` ``[nodes, children]`` into the parameters of a fully connected sum vector, as they are; the nodes and
    children that it lacks get zeros."""
    s, e = ns._param_range
    order = ((ns._param_ids - s) // (ns.block_size * ns.ch_block_size)).to(pc.device)
    rows, cols = ns.edge_ids[0].to(pc.device), ns.edge_ids[1].to(pc.device)
    full = torch.zeros(ns.num_node_blocks * ns.block_size, ns.num_ch_node_blocks * ns.ch_block_size, device=pc.device)
    full[:weights.size(0), :weights.size(1)] = weights
    full = full.view(ns.num_node_blocks, ns.block_size, ns.num_ch_node_blocks, ns.ch_block_size)
    tiles = pc.params[s:e].view(order.numel(), ns.ch_block_size, ns.block_size)      # (tables derived from them follow)
    some = max(1, (1 << 24) // (ns.block_size * ns.ch_block_size))                   # 64 MB of tiles at a time
    for at in range(0, order.numel(), some):
        i, j, k = rows[at:at + some], cols[at:at + some], order[at:at + some]
        tiles[k] = full[i, :, j].transpose(1, 2)


class HMMDecoder:
    """Next-token distributions of a compiled homogeneous HMM, for any number of beams.

    The parameters are taken over when the decoder is made and on ``reload()``; training the circuit later does not change
    it.  The arithmetic is the circuit's present ``sum_mode``.  A decoder serves one call at a time: all of them use its circuits'
    buffers.

    A state is a ``[num_latents, N]`` tensor: column n holds the logarithm of the distribution of beam n's next hidden state
    given its tokens, up to a constant, which ``log_probs`` takes out.  As in every circuit, a sum is at least 1e-24 of its
    largest term: what has a probability of zero beside others that have not has that one."""

    def __init__(self, pc: TensorCircuit):
        pc._require_cuda()
        self.pc, self.device = pc, pc.device
        root = pc.root_ns
        chain = self._chain(root)
        self._root, self._transition, self._emission = root, chain[0], chain[1]
        self.num_latents = self._emission.num_nodes
        self.vocab = self._emission.dist.num_cats
        V, L = self.vocab, _padded(self.num_latents)
        bs = _power_of_two(L, 1024)
        # emissions: sum nodes are tokens, padded to whole blocks with nodes of probability zero
        vbs = 1
        while vbs < min(V, bs, 128):                 # (no block larger than the states': leaves come before all other rows)
            vbs *= 2
        self._v_pad = -(-V // vbs) * vbs
        state = inputs(0, num_node_blocks=L // bs, block_size=bs, dist=Categorical(1))
        self._heard_ns = state
        self._speak_ns = summate(state, num_node_blocks=self._v_pad // vbs, block_size=vbs)
        # transitions: the state of the previous position times the emission of its token
        state = inputs(0, num_node_blocks=L // bs, block_size=bs, dist=Categorical(1))
        # (two categories more: a token that the vocabulary does not have, one that is not known)
        self._said_ns = inputs(1, num_node_blocks=L // bs, block_size=bs, dist=Categorical(V + 2))
        self._said_ns.set_params(torch.full((L, V + 2), 1.0 / (V + 2)), normalize=False)
        self._step_ns = summate(multiply(state, self._said_ns), num_node_blocks=L // bs, block_size=bs)
        self._state_ns = state
        self._speak = compile(self._speak_ns, verbose=False).to(self.device)
        self._step = compile(self._step_ns, verbose=False).to(self.device)
        for small in (self._speak, self._step):
            small.use_cuda_graphs = False            # a decoding loop may be captured as a whole
        self.reload()

    @staticmethod
    def _chain(root):
        """(transition vector, emission vector) that all positions share."""
        def refuse():
            raise ValueError("decoding needs the circuit of a homogeneous HMM (structures.HMM(..., homogeneous=True)) of at least "
                             "two positions")
        source = lambda ns: ns.get_source_ns() if ns.is_tied() else ns
        transitions, emissions, ns, variable = set(), [], root, 0
        if not root.is_sum() or root.num_nodes != 1:
            refuse()
        transition = None
        while True:
            if len(ns.chs) != 1:
                refuse()
            below = ns.chs[0]
            if below.is_prod() and len(below.chs) == 1:          # (compilation puts one between a sum and its leaves)
                below = below.chs[0]
            if below.is_input():
                leaf, ns = below, None
            elif below.is_prod() and len(below.chs) == 2 and below.chs[0].is_input() and below.chs[1].is_sum():
                leaf, ns = below.chs
            else:
                refuse()
            if leaf.scope.to_list() != [variable] or leaf.dist.get_signature() != "Categorical":
                refuse()
            variable += 1
            emissions.append(source(leaf))
            if ns is None:
                break
            transition = source(ns)
            transitions.add(id(transition))
        if len(transitions) != 1 or len({id(e) for e in emissions}) != 1:
            refuse()
        L = emissions[0].num_nodes
        if transition.num_nodes != L or any(v.edge_ids.size(1) != v.num_node_blocks * v.num_ch_node_blocks for v in (root, transition)):
            refuse()
        return transition, emissions[0]

    @torch.no_grad()
    def reload(self):
        """Takes over the circuit's present parameters."""
        L, V = self.num_latents, self.vocab
        layer = next(l for l in self.pc.input_layer_group if any(n is self._emission for n in l.nodes))
        s, e = self._emission._param_range
        emission = layer.params.data[s:e].view(L, V)
        self._initial = _dense(self.pc, self._root).view(L).log()
        _set_dense(self._step, self._step_ns, _dense(self.pc, self._transition).t())
        _set_dense(self._speak, self._speak_ns, emission.t())
        leaf = self._step.input_layer_group[0]
        s, e = self._said_ns._param_range
        said = leaf.params[s:e].view(-1, V + 2)
        said[:L, :V], said[:L, V], said[:L, V + 1], said[L:] = emission, 0.0, 1.0, 0.0

    def start(self, n: int) -> torch.Tensor:
        """States of ``n`` beams without tokens."""
        return self._initial.unsqueeze(1).expand(-1, n).contiguous()

    def _check(self, state):
        if state.dim() != 2 or state.size(0) != self.num_latents or state.dtype != torch.float32 or state.device != self.device:
            raise ValueError(f"a state is a float32 [{self.num_latents}, N] tensor on {self.device}")

    @torch.no_grad()
    def log_probs(self, state: torch.Tensor) -> torch.Tensor:
        """Log-probabilities of every beam's next token, ``[N, vocab]``, whatever the columns' sums; -inf for a column of -inf."""
        self._check(state)
        mass = state.logsumexp(0)
        return self._next(state - mass.masked_fill_(mass == float("-inf"), 0.0))

    def _next(self, state: torch.Tensor) -> torch.Tensor:
        """As `log_probs`, joint with what a column's sum holds."""
        N = state.size(1)
        if N == 0:
            return torch.empty(0, self.vocab, device=self.device)
        self._speak.sum_mode = self.pc.sum_mode
        rows = self._speak._values_of_inner([(self._heard_ns, state)], N)
        W = rows.size(1)
        out = torch.empty(W, self._v_pad, device=self.device)
        _lib.call("pcx_teacher_turn", out, rows, self._v_pad, W, self._v_pad, 0)
        return out[:N, :self.vocab]

    @torch.no_grad()
    def advance(self, state: torch.Tensor, tokens: torch.Tensor, log_probs: Optional[torch.Tensor] = None) -> torch.Tensor:
        """States after one more token each: ``tokens`` ``[N]``; ``log_probs`` ``[N]``: what the tokens had, which keeps the
        probabilities of a column at a sum of one (without it they go on as joint probabilities with the tokens).  A negative
        token is one that is not known: the state goes on by the transition alone.  A token that is impossible, or that the
        vocabulary does not have, leaves a column of -inf."""
        self._check(state)
        N = state.size(1)
        if tokens.shape != (N,) or tokens.is_floating_point():
            raise ValueError("one token per beam is needed")
        if N == 0:
            return state.clone()
        if log_probs is not None:
            state = state - log_probs.nan_to_num(0.0, neginf=0.0)
        return self._advance(state, self._categories(tokens.long()))

    def _categories(self, tokens: torch.Tensor) -> torch.Tensor:
        """What `_advance` takes: the vocabulary's tokens as they are, then one that it does not have, one that is not known."""
        return tokens.clamp(-1, self.vocab).remainder_(self.vocab + 2)

    def _advance(self, state: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
        N = state.size(1)
        x = torch.stack([torch.zeros_like(tokens), tokens], 1)
        self._step.sum_mode = self.pc.sum_mode
        return self._step._values_of_inner([(self._state_ns, state)], N, x)[:self.num_latents, :N].clone()


@torch.no_grad()
def beam_search(pc, prompts: Optional[torch.Tensor] = None, num_tokens: int = 1, num_beams: int = 4, batch: int = 1,
                eos_id: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The likeliest continuations of ``prompts`` ``[B, P]`` (integer; None: ``batch`` empty ones) under an HMM circuit or an
    :class:`HMMDecoder` (a circuit is laid out for decoding in every call: keep a decoder to ask more than once): tokens ``[B,
    num_beams, num_tokens]`` (int64) and their log-probabilities ``[B, num_beams]``, best first.  A beam that says ``eos_id`` is
    finished and goes on with ``eos_id`` at no cost.  Where there are fewer continuations than beams the rest has the score -inf and
    tokens -1.

    A negative token of a prompt is one that is not known (its position is marginalised, as a circuit's variable without slots);
    after one that is impossible, or that the vocabulary does not have, there are no continuations."""
    decoder = pc if isinstance(pc, HMMDecoder) else HMMDecoder(pc)
    V, device = decoder.vocab, decoder.device
    if num_tokens < 1 or not 1 <= num_beams <= lm.MAX_TOP:
        raise ValueError(f"at least one token, and 1 to {lm.MAX_TOP} beams")
    if eos_id is not None and not 0 <= eos_id < V:
        raise ValueError("`eos_id` is not in the vocabulary")
    if prompts is None:
        prompts = torch.empty(batch, 0, dtype=torch.int64, device=device)
    if prompts.dim() != 2 or prompts.is_floating_point():
        raise ValueError("prompts must be integer [B, P]")
    prompts = prompts.to(device)
    B, K = prompts.size(0), num_beams
    state = decoder.start(B)
    prompts = prompts.long()
    said, at, unknown = decoder._categories(prompts), prompts.clamp(0, V - 1), prompts < 0
    for t in range(prompts.size(1) if B > 0 else 0):
        heard = decoder._next(state).gather(1, at[:, t:t + 1])[:, 0]
        state = decoder._advance(state - heard.masked_fill_(unknown[:, t], 0.0).nan_to_num_(0.0, neginf=0.0), said[:, t])
    scores = torch.zeros(B, 1, device=device)
    finished = torch.zeros(B, 1, dtype=torch.bool, device=device)
    tokens = torch.empty(B, 0, dtype=torch.int64, device=device)
    pad = 0 if eos_id is None else eos_id
    for t in range(num_tokens):
        k = scores.size(1)
        n = min(K, k * V)
        logits = decoder._next(state).unflatten(0, (B, k))         # (the selection normalises)
        scores, parents, said = lm.beam_select(logits, scores, n, finished if eos_id is not None else None, pad)
        finished, tokens = lm.reorder(parents, finished.reshape(B * k), tokens.reshape(B * k, t))
        state, = lm.reorder(parents, state, dim=1)
        picked = logits[torch.arange(B, device=device)[:, None], parents, said.clamp_min(0)]
        tokens = torch.cat([tokens.view(B, n, t), said[..., None]], 2)
        if eos_id is not None:
            finished = finished.view(B, n) | (said == eos_id)
        else:
            finished = finished.view(B, n)
        if t + 1 < num_tokens and B > 0:
            state = decoder._advance(state - picked.reshape(-1), said.reshape(-1).clamp_min(0))        # (of dead beams: anything)
    if scores.size(1) < K:
        scores = torch.nn.functional.pad(scores, (0, K - scores.size(1)), value=float("-inf"))
        tokens = torch.nn.functional.pad(tokens, (0, 0, 0, K - tokens.size(1)), value=-1)
    return tokens.masked_fill((scores == float("-inf"))[..., None], -1), scores
