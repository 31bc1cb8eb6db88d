"""engine.SpeculativeStep over what top_k and top_p keep, and what it refuses."""
import numpy as np
import pytest

import engine
import rlsampler
import verify as ref

torch = pytest.importorskip("torch")


def seq(**kw):
    return engine.SequenceState(seq_id=3, max_tokens=5, **kw)


@pytest.mark.parametrize("cutoffs", [False, True])
@pytest.mark.parametrize("kw", [dict(repeat_penalty=1.1), dict(presence_penalty=0.2), dict(frequency_penalty=-0.1)])
def test_penalties_are_refused(cutoffs, kw):
    with pytest.raises(ValueError, match="sequence 3: .*penalties"):
        engine.speculative_params([seq(), seq(**kw)], cutoffs)


def test_parameters():
    states = [seq(top_p=0.8, temperature=0.5), seq(top_p=1.0, top_k=7)]
    with pytest.raises(ValueError, match="top_k 7"):
        engine.speculative_params(states, False)
    p = engine.speculative_params(states, True)
    assert p["top_k"].tolist() == [0, 7] and p["top_p"].tolist() == [np.float32(0.8), 1.0]
    p = engine.speculative_params(states[:1], False)
    assert p["top_k"].tolist() == [0] and p["top_p"].tolist() == [1.0] and p["temperature"].tolist() == [0.5]


@pytest.mark.gpu
@pytest.mark.parametrize("given", [False, True])
def test_cutoffs(given):
    """Drafts and tokens lie in what the sequence's top_k and top_p keep, and the
    tokens are those of the 64-bit walk over the kept ids, away from borders. More
    rows than the handle takes at once."""
    dev, B, K, V = "cuda:0", 9, 3, 4000
    rng = np.random.default_rng(9)
    kept = []

    def uniform(n):
        kept.append((rng.random(n) * (1 - 2.0 ** -24)).astype(np.float32))
        return kept[-1]

    step = engine.SpeculativeStep(V, 10, K, uniform=uniform, cutoffs=True)
    states = [engine.SequenceState(seq_id=b, tokens=[1], max_tokens=50, temperature=0.6 + 0.1 * b, top_k=[0, 5, 40][b % 3],
                                   top_p=[0.7, 1.0, 0.9][b // 3]) for b in range(B)]
    states[4].temperature = 0.0
    x = rng.normal(0, 3, (B, K + 1, V)).astype(np.float32)
    y = (0.95 * x[:, :K] + rng.normal(0, 0.4, (B, K, V))).astype(np.float32)
    rows = [torch.from_numpy(np.ascontiguousarray(a.reshape(-1, V))).to(dev) for a in (x, y)]
    drafts = torch.stack([step.draft(states, rows[1].view(B, K, V)[:, i].contiguous()) for i in range(K)], 1).contiguous()
    d = drafts.cpu().numpy()
    del kept[:]
    out = step.step(states, rows[0], drafts, None if given else rows[1])
    u, du = kept[0].reshape(B, K), kept[1]

    def cut(row, s):
        """The last id kept, from 64 bits: the sampler keeps the shortest head with top_p of the whole row's mass, top_k at most."""
        order = np.argsort(-row.astype(np.float64), kind="stable")
        e = np.exp((row[order].astype(np.float64) - row.max()) / np.float32(s.temperature))
        run = np.cumsum(e) / e.sum()
        n = V if s.top_p >= 1 else int(np.flatnonzero(run >= np.float32(s.top_p))[0]) + 1
        return int(order[min(n, s.top_k or V) - 1])

    same = 0
    for b, s in enumerate(states):
        T = float(np.float32(s.temperature))
        pc = [cut(x[b, i], s) if T > 0 else None for i in range(K + 1)]
        qc = [cut(y[b, i], s) if T > 0 else None for i in range(K)]
        for i in range(K):
            assert ref.dist(y[b, i], T, cut=qc[i])[d[b, i]] > 0, (b, i)
        r = ref.walk(lambda i: ref.dist(x[b, i], T, cut=pc[i]), lambda i: None if given or T <= 0 else ref.dist(y[b, i], T, cut=qc[i]),
                     lambda i: [i + 1] if i < K else [], lambda c: int(d[b, c - 1]), lambda c: u[b, c - 1], du[b], greedy=T <= 0)
        for i, t in enumerate(out[s.seq_id]):
            assert ref.dist(x[b, i], T, cut=pc[i])[t] > 0, (b, i)
        want = r.tokens[: r.tokens.index(0) + 1] if 0 in r.tokens else r.tokens
        same += out[s.seq_id] == want
    assert same >= B - 1, (same, B)
    with pytest.raises(ValueError, match="penalties"):
        step.draft([engine.SequenceState(seq_id=1, max_tokens=2, repeat_penalty=1.2)], rows[1][:1])
    with pytest.raises(ValueError, match="draft logits"):
        step.verify(states, rows[0], drafts, rows[1][:-1])
    if not given:  # rows behind the last sequence's are not looked at
        acc, tok = step.verify(states, rows[0], drafts, torch.cat([rows[1], torch.full((2, V), float("nan"), device=dev)]))
        assert tuple(tok.shape) == (B, K + 1) and (acc >= 0).all()
    step.close()
