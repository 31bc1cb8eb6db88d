"""The sampling part of ContinuousBatchingEngine::step (src/inference.rs:
103-141), one device call per step for the whole batch.

The reference loops over the running sequences, and for each one runs the
model, calls Model::sample_with_params(logits, state.temperature,
state.top_p) (src/model.rs:484-486 -> src/decoder.rs:35-100), pushes the
token and updates the sequence's counters. BatchStep does the same updates
for every live sequence at once, given the step's logits already on the
device (one row per live sequence, in the order `live()` returns):

  semantics "ref_exact" (default): rl_decoder_sample, the reference's own
      sample_with_params per row -- the same tokens as the reference's loop
      for the same uniforms;
  semantics "spec": rl_sample_batch with each sequence's optional top_k and
      penalties over its last HISTORY tokens (the batched pipeline).

SpeculativeStep is the sampling part of SpeculativeDecoder::generate
(src/inference.rs:260-333) for a batch of sequences, with the drafts verified
against both models' distributions (rl_specdec_verify_draft) in place of the
reference's comparison of the target's probability with itself.

SequenceState mirrors src/inference.rs:31-40 and carries the optional
sampler fields the batched path adds (all off by default).
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np

import rlsampler

HISTORY = 64  # tokens of a sequence's history the penalties see (Sampler::prev_tokens)


@dataclass
class SequenceState:
    """src/inference.rs:31-40, plus the batched path's optional fields."""

    seq_id: int
    tokens: list = field(default_factory=list)
    position: int = 0
    finished: bool = False
    generated_tokens: int = 0
    max_tokens: int = 0
    temperature: float = 1.0
    top_p: float = 0.9
    # batched path only (0 / 1.0 = off)
    top_k: int = 0
    repeat_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0

    def live(self) -> bool:
        """The reference's skip test (src/inference.rs:117-119), negated."""
        return not self.finished and self.generated_tokens < self.max_tokens


def live(states):
    """The sequences a step samples, in order."""
    return [s for s in states if s.live()]


def params_of(states) -> np.ndarray:
    p = np.zeros(len(states), rlsampler.ROW_PARAMS_DTYPE)
    for i, s in enumerate(states):
        p[i] = (s.temperature, s.top_p, s.top_k, s.repeat_penalty, s.presence_penalty, s.frequency_penalty)
    return p


def history_of(states, width=HISTORY):
    """[B, width] int32 ids (each sequence's last `width` tokens) and [B] lengths."""
    h = np.zeros((len(states), width), np.int32)
    n = np.zeros(len(states), np.int32)
    for i, s in enumerate(states):
        t = s.tokens[-width:]
        h[i, : len(t)] = t
        n[i] = len(t)
    return h, n


def apply(states, tokens) -> dict:
    """The reference's per-sequence updates (src/inference.rs:128-138) for the
    sampled tokens; returns {seq_id: token}."""
    out = {}
    for s, t in zip(states, tokens):
        t = int(t)
        s.tokens.append(t)
        s.generated_tokens += 1
        s.position += 1
        out[s.seq_id] = t
        if t == 0 or s.generated_tokens >= s.max_tokens:
            s.finished = True
    return out


class BatchStep:
    """One device sampling call per engine step (see the module docstring)."""

    def __init__(self, vocab: int, max_batch: int, device: int = 0, semantics: str = "ref_exact", uniform=None):
        if semantics not in ("ref_exact", "spec"):
            raise ValueError(f"semantics {semantics!r}")
        self.V = vocab
        self.semantics = semantics
        self.device = device
        self.sampler = rlsampler.Sampler(device, max_batch=max_batch, max_vocab=vocab, max_history=HISTORY)
        rng = np.random.Generator(np.random.PCG64())
        self.uniform = uniform or (lambda n: (rng.random(n) * (1.0 - 2.0 ** -24)).astype(np.float32))

    def sample(self, states, logits, uniforms=None):
        """Tokens for `states` (the live sequences, in order) from device logits
        [len(states), V] f32; the states are not changed."""
        import torch

        B = len(states)
        if logits.shape[0] != B or logits.shape[1] != self.V:
            raise ValueError(f"logits {tuple(logits.shape)} for {B} sequences of vocabulary {self.V}")
        dev = logits.device
        u = np.ascontiguousarray(self.uniform(B) if uniforms is None else uniforms, np.float32)
        du = torch.from_numpy(u).to(dev)
        if self.semantics == "ref_exact":
            T = torch.tensor([s.temperature for s in states], dtype=torch.float32, device=dev)
            P = torch.tensor([s.top_p for s in states], dtype=torch.float32, device=dev)
            tok, _ = self.sampler.decoder_sample(logits, T, P, du)
            return tok.cpu().numpy()
        h, n = history_of(states)
        tok, _, st = self.sampler.sample(logits, rlsampler.params_tensor(params_of(states), dev), du,
                                         torch.from_numpy(h).to(dev), torch.from_numpy(n).to(dev))
        st = st.cpu().numpy()
        if (st != 0).any():
            bad = int(np.flatnonzero(st)[0])
            raise rlsampler.RLError(int(st[bad]), f"sequence {states[bad].seq_id}: row status {int(st[bad])}")
        return tok.cpu().numpy()

    def step(self, states, logits, uniforms=None) -> dict:
        """Samples the live sequences (logits: one row per live sequence, in
        order) and applies the reference's updates; returns {seq_id: token}."""
        act = live(states)
        if not act:
            return {}
        return apply(act, self.sample(act, logits, uniforms))

    def close(self):
        self.sampler.close()


def apply_tokens(states, tokens) -> dict:
    """apply() for several tokens a sequence (rows of a [B, n] array, -1 behind a
    row's last): a sequence takes its tokens until it is finished. Returns
    {seq_id: [tokens taken]}."""
    out = {}
    for s, row in zip(states, tokens):
        taken = out.setdefault(s.seq_id, [])
        for t in row:
            if t < 0 or not s.live():
                break
            apply([s], [t])
            taken.append(int(t))
    return out


def speculative_params(states, cutoffs: bool) -> np.ndarray:
    """The sampling parameters of a speculative step's sequences: their
    temperatures, with `cutoffs` their top_p and top_k too. What the step would
    drop is refused: penalties, which change a row's logits with every accepted
    token, and a top_k without `cutoffs`."""
    p = params_of(states)
    for s in states:
        if (s.repeat_penalty, s.presence_penalty, s.frequency_penalty) != (1.0, 0.0, 0.0):
            raise ValueError(f"sequence {s.seq_id}: a speculative step applies no penalties")
        if s.top_k > 0 and not cutoffs:
            raise ValueError(f"sequence {s.seq_id}: top_k {s.top_k} needs SpeculativeStep(cutoffs=True)")
    if not cutoffs:
        p["top_p"], p["top_k"] = 1.0, 0
    return p


class SpeculativeStep:
    """Draft and verify for the live sequences of a batch: `draft` draws one
    token a sequence from the draft model's logits (called once for each
    position of the drafts), `verify` checks the drafts against the target's
    logits and gives each sequence its accepted drafts and one more token,
    distributed as the target's own samples are. Both models sample at the
    sequences' temperatures, over whole distributions (a sequence's top_p is not
    applied), or with `cutoffs` over what its top_k and top_p keep of each row.
    Sequences with penalties are refused."""

    def __init__(self, vocab: int, max_batch: int, max_draft: int, device: int = 0, uniform=None, cutoffs: bool = False):
        if max_draft < 1 or max_draft + 1 > rlsampler.VERIFY_MAX_NODES:
            raise ValueError(f"max_draft {max_draft}")
        self.V, self.K, self.device, self.max_batch, self.cutoffs = vocab, max_draft, device, max_batch, cutoffs
        self.sampler = rlsampler.Sampler(device, max_batch=max_batch, max_vocab=vocab, max_history=1)
        rng = np.random.Generator(np.random.PCG64())
        self.uniform = uniform or (lambda n: (rng.random(n) * (1.0 - 2.0 ** -24)).astype(np.float32))

    def _uniforms(self, shape, dev):
        import torch

        return torch.from_numpy(np.ascontiguousarray(self.uniform(int(np.prod(shape))), np.float32).reshape(shape)).to(dev)

    def _rows(self, states, params, logits, each):
        """The distributions of `each` rows a sequence."""
        import torch

        dev = logits.device
        T = torch.tensor([s.temperature for s in states], dtype=torch.float32, device=dev)
        if not self.cutoffs:
            return rlsampler.DistRows(logits, T)
        p = rlsampler.params_tensor(np.repeat(params, each), dev)
        size, u = params.dtype.itemsize, torch.zeros(self.max_batch, device=dev)
        cut = torch.empty(len(logits), dtype=torch.int32, device=dev)
        for r in range(0, len(logits), self.max_batch):
            n = min(self.max_batch, len(logits) - r)
            # rows that are not finite have no cutoff; verify reports those it looks at
            cut[r : r + n] = self.sampler.sample_debug(logits[r : r + n], p[r * size : (r + n) * size], u[:n], list_cap=1)[6][:, 2]
        return rlsampler.DistRows(logits, T, cut=cut)

    def draft(self, states, logits):
        """One drafted token [B] (device) a sequence from draft logits [B, V]."""
        if tuple(logits.shape) != (len(states), self.V):
            raise ValueError(f"draft logits {tuple(logits.shape)} for {len(states)} sequences of vocabulary {self.V}")
        p = rlsampler.params_tensor(speculative_params(states, self.cutoffs), logits.device)
        tok, _, _ = self.sampler.sample(logits, p, self._uniforms((len(states),), logits.device))
        return tok

    def verify(self, states, target_logits, drafts, draft_logits=None, n_draft=None):
        """target_logits [B * (K + 1), V] (a sequence's rows after 0 .. K drafts),
        drafts [B, K] int32 and the logits [B * K, V] they were drawn from
        (None: given drafts), n_draft [B] of them (None: K). Returns the
        device tensors (accepted [B], tokens [B, K + 1]); the states are not
        changed."""
        import torch

        B, dev = len(states), target_logits.device
        if tuple(drafts.shape) != (B, self.K) or tuple(target_logits.shape) != (B * (self.K + 1), self.V):
            raise ValueError(f"drafts {tuple(drafts.shape)} and target logits {tuple(target_logits.shape)} for {B} sequences")
        if draft_logits is not None:
            if len(draft_logits) < B * self.K or draft_logits.shape[-1] != self.V:
                raise ValueError(f"draft logits {tuple(draft_logits.shape)} for {B} sequences of {self.K} drafts")
            draft_logits = draft_logits[: B * self.K]
        params = speculative_params(states, self.cutoffs)
        n = torch.full((B,), self.K, dtype=torch.int32, device=dev) if n_draft is None else n_draft
        acc, tok, _, st = self.sampler.specdec_verify_draft(
            self._rows(states, params, target_logits, self.K + 1), drafts, n, self._uniforms((B, self.K), dev),
            self._uniforms((B,), dev), draft=None if draft_logits is None else self._rows(states, params, draft_logits, self.K))
        bad = st.cpu().numpy()
        if (bad != 0).any():
            i = int(np.flatnonzero(bad)[0])
            raise rlsampler.RLError(int(bad[i]), f"sequence {states[i].seq_id}: row status {int(bad[i])}")
        return acc, tok

    def step(self, states, target_logits, drafts, draft_logits=None, n_draft=None) -> dict:
        """verify() and the per-sequence updates; returns {seq_id: [tokens]}."""
        return apply_tokens(states, self.verify(states, target_logits, drafts, draft_logits, n_draft)[1].cpu().numpy())

    def close(self):
        self.sampler.close()
