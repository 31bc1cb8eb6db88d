"""The speculative step over a batch (engine.SpeculativeStep): its host logic on
the CPU, and on the GPU the operators in a row as a serving step has them: a
4-bit draft head proposes, the bf16 target head scores the drafts, both models'
rows are verified, and the sequences take what came out."""
import numpy as np
import pytest

import engine
import rlsampler
import verify as ref

torch = pytest.importorskip("torch")


def test_apply_tokens_stops_where_a_sequence_ends():
    a = engine.SequenceState(seq_id=1, tokens=[5], max_tokens=2)
    b = engine.SequenceState(seq_id=2, tokens=[6], max_tokens=9)
    c = engine.SequenceState(seq_id=3, tokens=[7], max_tokens=9, finished=True)
    out = engine.apply_tokens([a, b, c], np.array([[3, 4, 8], [9, 0, 5], [1, 2, -1]]))
    assert out == {1: [3, 4], 2: [9, 0], 3: []}
    assert a.finished and a.tokens == [5, 3, 4]  # max_tokens
    assert b.finished and b.tokens == [6, 9, 0]  # token 0 ends a sequence
    assert c.tokens == [7]
    d = engine.SequenceState(seq_id=4, tokens=[], max_tokens=9)
    assert engine.apply_tokens([d], np.array([[2, -1, -1]])) == {4: [2]} and d.live()


def test_refusals_before_any_device_work():
    with pytest.raises(ValueError):
        engine.SpeculativeStep(100, 4, 0)
    with pytest.raises(ValueError):
        engine.SpeculativeStep(100, 4, rlsampler.VERIFY_MAX_NODES)


def test_tensors_on_another_device_are_refused():
    s = rlsampler.Sampler.__new__(rlsampler.Sampler)
    s.h, s.device = None, 0
    i32, f32, bf16 = torch.int32, torch.float32, torch.bfloat16
    n, du = torch.zeros(2, dtype=i32), torch.zeros(2)
    with pytest.raises(ValueError, match="on cpu"):
        s.specdec_verify_draft(rlsampler.DistRows(torch.zeros(8, 40)), torch.zeros(2, 3, dtype=i32), n, torch.zeros(2, 3), du)
    with pytest.raises(ValueError, match="on cpu"):
        s.specdec_verify_tree(rlsampler.DistRows(torch.zeros(6, 40)), torch.zeros(2, 3, dtype=i32), torch.zeros(2, 3, dtype=i32), n,
                              torch.zeros(2, 3, dtype=f32), du)
    w = rlsampler.Q4Weight(torch.zeros(6, 64, dtype=torch.uint8), torch.zeros(6, 2, dtype=bf16), 64)
    x = torch.zeros(2, 128, dtype=bf16)
    for call in (lambda: s.lmhead_q4_logits(x, w), lambda: s.lmhead_q4_greedy(x, w), lambda: s.lmhead_q4_sample(x, w, n, du),
                 lambda: s.lmhead_q4_quantize(torch.zeros(6, 128, dtype=bf16), 64)):
        with pytest.raises(ValueError, match="on cpu"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("given", [False, True])
def test_draft_head_target_head_verify(given):
    """The tokens are those the 64-bit walk over the same logits gives (away from
    borders), and every sequence gets at least one."""
    dev, B, K, V, H = "cuda:0", 6, 3, 5000, 512
    g = torch.Generator(device=dev).manual_seed(7)
    rng = np.random.default_rng(7)
    kept = []

    def uniform(n):
        kept.append((rng.random(n) * (1 - 2.0 ** -24)).astype(np.float32))
        return kept[-1]

    step = engine.SpeculativeStep(V, B * (K + 1), K, uniform=uniform)
    weight = (torch.randn(V, H, generator=g, device=dev) * (3.0 / H ** 0.5)).to(torch.bfloat16)
    small = step.sampler.lmhead_q4_quantize(weight, 64)
    states = [engine.SequenceState(seq_id=10 + b, tokens=[1], max_tokens=50, temperature=0.7 + 0.1 * b) for b in range(B)]
    states[0].temperature = 0.0
    hidden = torch.randn(B, K + 1, H, generator=g, device=dev).to(torch.bfloat16)
    logits, drafts = [], []
    for i in range(K):  # the draft model's steps
        x = step.sampler.lmhead_q4_logits(hidden[:, i].contiguous(), small)
        drafts.append(step.draft(states, x))
        logits.append(x)
    drafts = torch.stack(drafts, 1).contiguous()
    draft_rows = torch.stack(logits, 1).reshape(B * K, V)
    target_rows = step.sampler.lmhead_logits(hidden.reshape(B * (K + 1), H), weight)
    del kept[:]
    out = step.step(states, target_rows, drafts, None if given else draft_rows)
    u, du = kept[0].reshape(B, K), kept[1]
    x, y, d = target_rows.cpu().numpy(), draft_rows.cpu().numpy(), drafts.cpu().numpy()
    same = 0
    for b, s in enumerate(states):
        T = float(np.float32(s.temperature))
        r = ref.walk(lambda i: ref.dist(x[b * (K + 1) + i], T),
                     lambda i: None if given or T <= 0 else ref.dist(y[b * K + i], T),
                     lambda i: [i + 1] if i < K else [], lambda c: int(d[b, c - 1]), lambda c: u[b, c - 1], du[b], greedy=T <= 0)
        assert len(out[s.seq_id]) >= 1 and s.tokens[1:] == out[s.seq_id]
        want = r.tokens
        if 0 in want:
            want = want[: want.index(0) + 1]  # token 0 ends a sequence
        same += out[s.seq_id] == want
    # a test or a draw within the rounding of f32 weights may fall otherwise
    assert same >= B - 1, (same, B)
    assert sum(len(t) for t in out.values()) > B  # drafts are accepted
    step.close()


@pytest.mark.gpu
def test_verify_reports_a_bad_sequence():
    step = engine.SpeculativeStep(64, 8, 1)
    states = [engine.SequenceState(seq_id=b, max_tokens=5) for b in range(2)]
    x = torch.zeros(4, 64, device="cuda:0")
    x[2, 3] = float("nan")
    with pytest.raises(rlsampler.RLError) as e:
        step.step(states, x, torch.ones(2, 1, dtype=torch.int32, device="cuda:0"))
    assert e.value.status == rlsampler.RL_ERR_NONFINITE and "sequence 1" in str(e.value)
    with pytest.raises(ValueError):
        step.draft(states, x)
    step.close()
