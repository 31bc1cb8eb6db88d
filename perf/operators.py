"""The operators of speculative decoding and of the 4-bit LM head: cases, plain forms, work.

  verify   a chain of drafted tokens checked against the target's distributions (rl_specdec_verify_draft)
  tree     a tree of drafted tokens checked against the target's distributions (rl_specdec_verify_tree)
  head     an LM head with 4-bit weights and group scales: logits, or greedy tokens (rl_lmhead_q4_*)
"""
import os
import sys

import torch

own = False

DEV = "cuda"
#: nibble e of a packed 32-bit word (element 8 i + e) starts at this bit
SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)


def _package():
    """The framework's Python front end."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust-llm_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import rlsampler

    return rlsampler


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one conversation, the command line's vocabulary, three drafts: latency is all
        dict(name="verify b1 k3 v32000", op="verify", B=1, K=3, V=32000, dtype="f32", draft="rows", ragged=False, mask=False, cut=False, greedy=False, pad=0),
        # a serving step: 64 sequences, four drafts each, f32 logits
        dict(name="verify b64 k4 v128256", op="verify", B=64, K=4, V=128256, dtype="f32", draft="rows", ragged=False, mask=False, cut=False, greedy=False, pad=0),
        # a large step: drafts of unequal length, bf16 logits, greedy requests among the sampled, rows with padding behind them
        dict(name="verify b128 k7 v151936 bf16", op="verify", B=128, K=7, V=151936, dtype="bf16", draft="rows", ragged=True, mask=False, cut=False, greedy=True, pad=64),
        # grammar-constrained requests with top-k: allowed sets and cutoffs for both models
        dict(name="verify b24 k5 v32000 mask cut", op="verify", B=24, K=5, V=32000, dtype="f32", draft="rows", ragged=True, mask=True, cut=True, greedy=False, pad=0),
        # one conversation with a small tree
        dict(name="tree b1 3.2 v32000", op="tree", B=1, branch="3.2", V=32000, dtype="f32", draft="rows", ragged=False, greedy=False, pad=0),
        # a serving step with sampled trees
        dict(name="tree b16 4.2.1.1 v128256", op="tree", B=16, branch="4.2.1.1", V=128256, dtype="f32", draft="rows", ragged=True, greedy=True, pad=0),
        # many requests whose trees hold the draft's best tokens (no draft distribution)
        dict(name="tree b64 3.2.1 v151936 given", op="tree", B=64, branch="3.2.1", V=151936, dtype="bf16", draft="given", ragged=False, greedy=False, pad=0),
        # one token of one conversation through a small head
        dict(name="head b1 h2048 v32000 g32", op="head", B=1, H=2048, V=32000, group=32, out="f32"),
        # one token, a large head
        dict(name="head b1 h4096 v128256 g128", op="head", B=1, H=4096, V=128256, group=128, out="f32"),
        # the drafted positions of three sequences, greedy: the logits stay in the kernel
        dict(name="head b12 h4096 v128256 greedy", op="head", B=12, H=4096, V=128256, group=64, out="greedy"),
        # a serving batch, bf16 logits, a vocabulary that no tile divides
        dict(name="head b37 h2560 v50257 bf16", op="head", B=37, H=2560, V=50257, group=32, out="bf16"),
        # a step of 64 sequences with verification rows
        dict(name="head b128 h4096 v128256 g128", op="head", B=128, H=4096, V=128256, group=128, out="f32"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of its range."""
    import math

    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["verify", "tree", "head"])
    V = _log(rng, 600, 151936)
    if rng.random() < 0.5:
        V |= 1
    if op == "head":
        group = rng.choice([32, 64, 128])
        H = 128 * _log(rng, 2, 48)
        V = max(257, min(V, 128256 * 4096 // H))
        return dict(op="head", B=_log(rng, 1, 128), H=H, V=V, group=group, out=rng.choice(["f32", "bf16", "greedy"]))
    dtype = rng.choice(["f32", "bf16"])
    pad = rng.choice([0, 0, 3, 8, 64])
    greedy = rng.random() < 0.3
    if op == "verify":
        K = rng.randint(1, 8)
        B = _log(rng, 1, 128)
        while B * (2 * K + 1) * V > 64 * 9 * 128256:
            B = max(1, B // 2)
        mask = rng.random() < 0.3
        return dict(op="verify", B=B, K=K, V=V, dtype=dtype, draft=rng.choice(["rows", "rows", "given"]), ragged=rng.random() < 0.5, mask=mask,
                    cut=rng.random() < 0.3, greedy=greedy, pad=pad)
    branch = rng.choice(["2", "4", "2.2", "3.1.1", "4.2", "2.2.2", "5.3", "1.2.3", "8", "3.2.1.1"])
    B = _log(rng, 1, 64)
    while B * _nodes(branch) * V > 16 * 29 * 128256:
        B = max(1, B // 2)
    return dict(op="tree", B=B, branch=branch, V=V, dtype=dtype, draft=rng.choice(["rows", "rows", "given"]), ragged=rng.random() < 0.5, greedy=greedy, pad=pad)


def _parents(branch):
    """Parents of a tree in level order (the root is node 0, parent -1): every node of level l has branch[l] children."""
    parent, level = [-1], [0]
    for m in (int(x) for x in branch.split(".")):
        nxt = []
        for node in level:
            for _ in range(m):
                nxt.append(len(parent))
                parent.append(node)
        level = nxt
    return parent


def _nodes(branch):
    return len(_parents(branch))


def _lengths(case, most):
    """Drafts (or tree nodes behind the root) of each sequence: all alike, or unequal."""
    return [((5 * b + 3) % (most + 1)) if case["ragged"] else most for b in range(case["B"])]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * seed + 17)
    return g


def _rows(x, dtype, pad):
    """The rows [R, V] as a program holds them: the type of the model's output, rows `pad` elements apart."""
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    buf = torch.zeros(x.shape[0], x.shape[1] + pad, dtype=t, device=DEV)
    buf[:, : x.shape[1]] = x
    return buf[:, : x.shape[1]]


def _gumbel(shape, g):
    return -torch.log(-torch.log(torch.rand(shape, generator=g, device=DEV).clamp_(1e-7, 1 - 1e-7)))


def _speculative(case, N, seed):
    """Logits of both models over N positions a sequence, temperatures, and the generator."""
    g = _gen(seed)
    B, V = case["B"], case["V"]
    # a language model's logits: a few likely tokens, a long tail; the draft model agrees with most of it
    target = torch.randn(B * N, V, generator=g, device=DEV).mul_(3.0)
    draft = torch.randn(B * N, V, generator=g, device=DEV).mul_(0.6).add_(target, alpha=0.95)
    T = torch.rand(B, generator=g, device=DEV) * 0.6 + 0.6
    if case["greedy"]:
        T[::3] = 0.0
    return g, _rows(target, case["dtype"], case["pad"]), _rows(draft, case["dtype"], case["pad"]), T


def _prepare_verify(case, seed):
    B, K, V = case["B"], case["K"], case["V"]
    g, target, draft, T = _speculative(case, K + 1, seed)
    draft = _rows(draft.unflatten(0, (B, K + 1))[:, :K].flatten(0, 1), case["dtype"], case["pad"])
    s = dict(target=target, draft=draft, T=T, mask=None, draft_mask=None, cut=None, draft_cut=None)
    seen = draft.float()
    if case["mask"]:
        W = (V + 31) // 32
        words = torch.randint(-(1 << 31), 1 << 31, (B, K + 1, W), generator=g, device=DEV, dtype=torch.int64)
        words &= torch.randint(-(1 << 31), 1 << 31, (B, K + 1, W), generator=g, device=DEV, dtype=torch.int64)
        words[:, ::4] = torch.where((torch.arange(B, device=DEV) % 8 == 5)[:, None, None], 0, words[:, ::4])  # a state that constrains nothing
        s["mask"] = words.to(torch.int32).reshape(B * (K + 1), W)
        s["draft_mask"] = words[:, :K].to(torch.int32).reshape(B * K, W)
        seen = seen.masked_fill(~_allowed(s["draft_mask"], V), float("-inf"))
    if case["cut"]:
        def last_kept(x, rows):
            k = torch.randint(8, 50, (rows, 1), generator=g, device=DEV)
            return torch.topk(x, 50, dim=1).indices.gather(1, k).to(torch.int32).reshape(rows)

        full = target.float()
        if case["mask"]:
            full = full.masked_fill(~_allowed(s["mask"], V), float("-inf"))
        s["cut"], s["draft_cut"] = last_kept(full, B * (K + 1)), last_kept(seen, B * K)
        floor = seen.gather(1, s["draft_cut"].long()[:, None])
        seen = seen.masked_fill(seen < floor, float("-inf"))
    hot = torch.where(T > 0, T, torch.ones_like(T)).repeat_interleave(K)[:, None]
    drafts = (seen / hot + _gumbel(seen.shape, g) * (T > 0).repeat_interleave(K)[:, None]).argmax(1)
    s["drafts"] = drafts.to(torch.int32).view(B, K)
    s["n"] = torch.tensor(_lengths(case, K), dtype=torch.int32, device=DEV)
    s["accept_u"] = torch.rand(B, K, generator=g, device=DEV)
    s["draw_u"] = torch.rand(B, generator=g, device=DEV)
    if case["draft"] == "given":
        s["draft"] = s["draft_mask"] = s["draft_cut"] = None
    return s


def _prepare_tree(case, seed):
    parents = _parents(case["branch"])
    B, N, V = case["B"], len(parents), case["V"]
    g, target, draft, T = _speculative(case, N, seed)
    parent = torch.tensor(parents, device=DEV)
    x = draft.float()
    hot = torch.where(T > 0, T, torch.ones_like(T)).repeat_interleave(N)[:, None]
    tokens = torch.full((B, N), -1, dtype=torch.int64, device=DEV)
    rank = torch.zeros(N, dtype=torch.int64, device=DEV)
    for i in range(1, N):
        rank[i] = sum(p == parents[i] for p in parents[:i])
    if case["draft"] == "given":  # a node's children are its draft row's best tokens
        best = torch.topk(x, 8, dim=1).indices.view(B, N, 8)
        tokens[:, 1:] = best[:, parent[1:], rank[1:]]
    else:  # drawn from the node's draft row
        for j in range(int(rank.max()) + 1):
            pick = (x / hot + _gumbel(x.shape, g)).argmax(1).view(B, N)
            which = torch.nonzero((rank == j) & (parent >= 0)).flatten()
            tokens[:, which] = pick[:, parent[which]]
    s = dict(target=target, draft=None if case["draft"] == "given" else draft, T=T, tokens=tokens.to(torch.int32))
    s["parent"] = parent.to(torch.int32).repeat(B, 1)
    s["n"] = torch.tensor([1 + k for k in _lengths(case, N - 1)], dtype=torch.int32, device=DEV)
    s["accept_u"] = torch.rand(B, N, generator=g, device=DEV)
    s["draw_u"] = torch.rand(B, generator=g, device=DEV)
    s["most"] = max(sum(p == i for p in parents) for i in range(N))
    s["depth"] = len(case["branch"].split("."))
    return s


def _prepare_head(case, seed):
    g = _gen(seed)
    B, H, V, G = case["B"], case["H"], case["V"], case["group"]
    hidden = torch.randn(B, H, generator=g, device=DEV)
    hidden[:, ::97] *= 12.0  # a final norm's output has a few large channels
    q = torch.empty(V, H // 2, dtype=torch.uint8, device=DEV)
    scale = torch.empty(V, H // G, dtype=torch.bfloat16, device=DEV)
    for v0 in range(0, V, 16384):  # rows as round-to-nearest quantisation leaves them
        n = min(16384, V - v0)
        w = torch.randn(n, H // G, G, generator=g, device=DEV).mul_(0.02)
        top = w.abs().amax(2, keepdim=True)
        s = (top / 8).to(torch.bfloat16)
        code = torch.clamp(torch.round(w / s.float()) + 8, 0, 15).to(torch.int64).view(n, H // 8, 8)
        word = (code << torch.tensor(SHIFTS, device=DEV)).sum(2)
        q[v0 : v0 + n] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32).view(torch.uint8)
        scale[v0 : v0 + n] = s[:, :, 0]
    return dict(hidden=hidden.to(torch.bfloat16), q=q, scale=scale)


def prepare(case, seed):
    s = {"verify": _prepare_verify, "tree": _prepare_tree, "head": _prepare_head}[case["op"]](case, seed)
    s["case"] = case
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _allowed(mask, V):
    """Bit-packed rows as truth values [R, V]; a row without a bit allows every id."""
    ids = torch.arange(V, device=DEV)
    bits = ((mask[:, ids >> 5] >> (ids & 31).to(torch.int32)) & 1) != 0
    return bits | ~bits.any(1, keepdim=True)


def _dist(x, T, mask=None, cut=None):
    """Rows of probabilities [R, V] in 64 bits (draws lie next to borders): softmax(x / T) over the kept ids; T <= 0: one at the maximum."""
    x = x.double()
    ids = torch.arange(x.shape[1], device=DEV)
    if mask is not None:
        x = x.masked_fill(~_allowed(mask, x.shape[1]), float("-inf"))
    if cut is not None:
        at = cut.long()[:, None]
        xc = x.gather(1, at)
        x = x.masked_fill((x < xc) | ((x == xc) & (ids > at)), float("-inf"))
    top = x.amax(1, keepdim=True)
    first = torch.where(x == top, ids, x.shape[1]).amin(1, keepdim=True)
    hot = torch.where(T > 0, T, torch.ones_like(T)).double()[:, None]
    e = torch.exp((x - top) / hot)
    e /= e.sum(1, keepdim=True)
    return torch.where((T > 0)[:, None], e, (ids == first).double())


def _pick(w, u):
    """The first id whose running sum of w is over u times the whole."""
    run = w.cumsum(1)
    at = (run <= (u.double() * run[:, -1])[:, None]).sum(1)
    last = torch.where(w > 0, torch.arange(w.shape[1], device=DEV), -1).amax(1)
    return torch.minimum(at, last)


def _plain_verify(s):
    B, K = s["drafts"].shape
    V = s["target"].shape[1]
    at = torch.arange(B, device=DEV)
    p = _dist(s["target"], s["T"].repeat_interleave(K + 1), s["mask"], s["cut"]).view(B, K + 1, V)
    drafts = s["drafts"].long()
    given = torch.nn.functional.one_hot(drafts, V).double() if s["draft"] is None or bool(s["case"]["greedy"]) else None
    if s["draft"] is None:
        q = given
    else:
        q = _dist(s["draft"], s["T"].repeat_interleave(K), s["draft_mask"], s["draft_cut"]).view(B, K, V)
        if given is not None:
            q = torch.where((s["T"] > 0)[:, None, None], q, given)
    px, qx = (d.gather(2, drafts[:, :, None])[:, :, 0] for d in (p[:, :K], q))
    inside = torch.arange(K, device=DEV) < s["n"][:, None]
    ok = (s["accept_u"].double() * qx < px) & inside
    acc = ok.long().cumprod(1).sum(1)
    refused = acc < s["n"]
    w = p[at, acc]
    w = torch.where(refused[:, None], (w - q[at, acc.clamp(max=K - 1)]).clamp(min=0), w)
    last = _pick(w, s["draw_u"])
    place = torch.arange(K + 1, device=DEV)
    tok = torch.nn.functional.pad(drafts, (0, 1), value=-1)
    tok = torch.where(place < acc[:, None], tok, torch.where(place == acc[:, None], last[:, None], -1))
    prob = torch.where(tok >= 0, p.gather(2, tok.clamp(min=0)[:, :, None])[:, :, 0], 0.0)
    return acc.to(torch.int32), tok.to(torch.int32), prob.float()


def _plain_tree(s):
    B, N = s["tokens"].shape
    V = s["target"].shape[1]
    at, ids = torch.arange(B, device=DEV), torch.arange(V, device=DEV)
    tokens, parent, hot = s["tokens"].long(), s["parent"].long(), s["T"] > 0
    p = _dist(s["target"], s["T"].repeat_interleave(N)).view(B, N, V)
    q = None if s["draft"] is None else _dist(s["draft"], s["T"].repeat_interleave(N)).view(B, N, V)
    inside = torch.arange(N, device=DEV) < s["n"][:, None]
    cur = torch.zeros(B, dtype=torch.long, device=DEV)
    walking = torch.ones(B, dtype=torch.bool, device=DEV)
    path, tok = torch.full((B, N), -1, device=DEV), torch.full((B, N), -1, device=DEV)
    prob = torch.zeros(B, N, dtype=torch.float64, device=DEV)
    acc = torch.zeros(B, dtype=torch.long, device=DEV)
    w = p[:, 0].clone()
    for _ in range(s["depth"] + 1):
        here = cur.clone()
        w = torch.where(walking[:, None], p[at, here], w)
        went = torch.zeros(B, dtype=torch.bool, device=DEV)
        kids = (parent == here[:, None]) & inside
        order = torch.where(kids, torch.arange(N, device=DEV), N).sort(1).values
        for j in range(s["most"]):
            c = order[:, j].clamp(max=N - 1)
            there = walking & ~went & (order[:, j] < N)
            x = tokens[at, c]
            sharp = (ids == x[:, None]).double()
            d = sharp if q is None else torch.where(hot[:, None], q[at, here], sharp)
            whole = w.sum(1)
            yes = there & (s["accept_u"][at, c].double() * d[at, x] * whole < w[at, x])
            less = (w - whole[:, None] * d).clamp(min=0) if q is not None else w * (1 - d)
            less = torch.where(hot[:, None], less, w * (1 - d))
            w = torch.where((there & ~yes)[:, None], less, w)
            path[at, acc] = torch.where(yes, c, path[at, acc])
            tok[at, acc] = torch.where(yes, x, tok[at, acc])
            prob[at, acc] = torch.where(yes, p[at, here, x], prob[at, acc])
            acc = acc + yes
            cur = torch.where(yes, c, cur)
            went = went | yes
        walking = went
    last = _pick(w, s["draw_u"])
    tok[at, acc] = last
    prob[at, acc] = p[at, cur, last]
    return acc.to(torch.int32), path.to(torch.int32), tok.to(torch.int32), prob.float()


def _codes(q):
    """[V, H / 2] packed bytes as codes 0..15 [V, H]."""
    word = q.view(torch.int32)
    return ((word[:, :, None] >> torch.tensor(SHIFTS, dtype=torch.int32, device=DEV)) & 15).flatten(1)


def _plain_head(s):
    G = s["case"]["group"]
    w = (_codes(s["q"]).float() - 8).unflatten(1, (-1, G)).mul_(s["scale"].float()[:, :, None]).flatten(1)
    y = s["hidden"].float() @ w.T
    if s["case"]["out"] == "bf16":
        return y.to(torch.bfloat16)
    if s["case"]["out"] == "greedy":  # the last of equal maxima, as the framework's greedy sampling
        top = y.amax(1, keepdim=True)
        return torch.where(y == top, torch.arange(y.shape[1], device=DEV), -1).amax(1).to(torch.int32)
    return y


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
#: The handles that a program keeps for all of its calls, one a device: made at a device's first call, whatever its inputs.
_handles = {}


def _handle(rl):
    device = torch.cuda.current_device()
    if device not in _handles:
        _handles[device] = rl.Sampler(device, max_batch=256, max_vocab=64, max_history=1)
    return _handles[device]


def _own(s):
    rl, op = _package(), s["case"]["op"]
    h = _handle(rl)
    if op == "head":
        w = rl.Q4Weight(s["q"], s["scale"], s["case"]["group"])
        if s["case"]["out"] == "greedy":
            return h.lmhead_q4_greedy(s["hidden"], w)[0]
        return h.lmhead_q4_logits(s["hidden"], w, out_dtype=torch.bfloat16 if s["case"]["out"] == "bf16" else torch.float32)
    if op == "verify":
        target = rl.DistRows(s["target"], s["T"], mask=s["mask"], cut=s["cut"])
        draft = None if s["draft"] is None else rl.DistRows(s["draft"], s["T"], mask=s["draft_mask"], cut=s["draft_cut"])
        acc, tok, prob, _ = h.specdec_verify_draft(target, s["drafts"], s["n"], s["accept_u"], s["draw_u"], draft=draft)
        return acc, tok, prob
    target = rl.DistRows(s["target"], s["T"])
    draft = None if s["draft"] is None else rl.DistRows(s["draft"], s["T"])
    acc, path, tok, prob, _ = h.specdec_verify_tree(target, s["tokens"], s["parent"], s["n"], s["accept_u"], s["draw_u"], draft=draft)
    return acc, path, tok, prob


def run(state):
    if own:
        return _own(state)
    return {"verify": _plain_verify, "tree": _plain_tree, "head": _plain_head}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------------------------------------------------
#: Share of drafted tokens that the target accepts on these inputs (drawn from the draft's rows, or given). A walk stops
#: at its first refusal and the rows behind it need not be read, so what a pass has to read follows from it.
AGREE = {"rows": 0.70, "given": 0.10}


def work(case):
    if case["op"] == "head":
        B, H, V = case["B"], case["H"], case["V"]
        out = {"f32": 4 * B * V, "bf16": 2 * B * V, "greedy": 4 * B}[case["out"]]
        return {"bytes": V * H // 2 + 2 * V * (H // case["group"]) + 2 * B * H + out, "flops": 2.0 * B * V * H}
    V, size = case["V"], 2 if case["dtype"] == "bf16" else 4
    rows = 0.0
    both = 2 if case["draft"] == "rows" else 1
    agree = AGREE[case["draft"]]
    if case["op"] == "verify":
        for n in _lengths(case, case["K"]):
            rows += sum(agree**i * (both if i < n else 1) for i in range(n + 1))
        rows_bytes = V * size + (((V + 31) // 32) * 4 if case["mask"] else 0)
        small = case["B"] * (12 * case["K"] + 20)
    else:
        parents = _parents(case["branch"])
        for n in _lengths(case, len(parents) - 1):
            level, reach = 0, 1.0
            while reach > 0 and level <= n:
                kids = sum(p == level for p in parents[: n + 1])
                rows += reach * (both if kids else 1)
                reach *= 1 - (1 - agree) ** kids if kids else 0.0
                level = parents.index(level) if level in parents else n + 1
        rows_bytes = V * size
        small = case["B"] * (20 * len(parents) + 20)
    return {"bytes": int(rows * rows_bytes + small), "flops": 4.0 * rows * V}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, written apart from the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _row64(row, T, mask, cut):
    """log p of one row; None for one-hot rows, and the id that holds all."""
    x = row.double().clone()
    if mask is not None:
        word = mask.long() & 0xFFFFFFFF
        allow = (word[:, None] >> torch.arange(32, device=DEV)).bitwise_and(1).flatten()[: len(x)].bool()
        if bool(allow.any()):
            x[~allow] = float("-inf")
    if cut is not None:
        c = int(cut)
        order = torch.argsort(x, descending=True, stable=True)
        place = int((order == c).nonzero())
        x[order[place + 1 :]] = float("-inf")
    if T <= 0:
        one = torch.full_like(x, float("-inf"))
        one[int((x == x.max()).nonzero()[0])] = 0.0
        return one
    return torch.log_softmax(x / T, 0)


def _walk64(s, b, children, token, prow, qrow, u_of):
    """One sequence: [(node, token, probability)], the last one drawn."""
    node, out = 0, []
    while True:
        logp = prow(b, node)
        p = logp.exp()
        w, went = p.clone(), False
        for c in children(b, node):
            x, q = token(b, c), qrow(b, node)
            if q is None:
                if u_of(b, c) * float(w.sum()) < float(w[x]):
                    went = True
                else:
                    w[x] = 0.0
            else:
                if u_of(b, c) * float(q[x]) * float(w.sum()) < float(w[x]):
                    went = True
                else:
                    w = torch.relu(w - w.sum() * q)
            if went:
                out.append((c, x, float(p[x])))
                node = c
                break
        if not went:
            t = float(s["draw_u"][b]) * float(w.sum())
            x = int((torch.cumsum(w, 0) > t).nonzero()[0])
            return out + [(-1, x, float(p[x]))]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "head":
        if case["out"] == "greedy":
            return None
        B, H, V, G = case["B"], case["H"], case["V"], case["group"]
        y = torch.empty(B, V, dtype=torch.float64, device=DEV)
        h = s["hidden"].double().view(B, H // G, G)
        bytes_ = s["q"].view(V, H // 8, 4)
        for v0 in range(0, V, 8192):
            c = bytes_[v0 : v0 + 8192].to(torch.int32)
            # byte 0: elements 0, 2; byte 1: 4, 6; byte 2: 1, 3; byte 3: 5, 7 (low, high)
            e = torch.stack([c[..., 0] % 16, c[..., 2] % 16, c[..., 0] // 16, c[..., 2] // 16, c[..., 1] % 16, c[..., 3] % 16, c[..., 1] // 16, c[..., 3] // 16], 2)
            d = torch.einsum("vgk,bgk->bvg", e.reshape(-1, H // G, G).double() - 8.0, h)
            y[:, v0 : v0 + 8192] = (d * s["scale"][v0 : v0 + 8192].double()).sum(2)
        return y
    B = case["B"]
    T = [float(t) for t in s["T"]]
    u = s["accept_u"].double().cpu()
    n = [int(k) for k in s["n"]]
    if case["op"] == "verify":
        N = case["K"] + 1
        prow = lambda b, i: _row64(s["target"][b * N + i], T[b], None if s["mask"] is None else s["mask"][b * N + i], None if s["cut"] is None else s["cut"][b * N + i])  # noqa: E731
        at = lambda b, i: b * (N - 1) + i  # noqa: E731
        qrow = lambda b, i: None if s["draft"] is None or T[b] <= 0 else _row64(  # noqa: E731
            s["draft"][at(b, i)], T[b], None if s["draft_mask"] is None else s["draft_mask"][at(b, i)], None if s["draft_cut"] is None else s["draft_cut"][at(b, i)]).exp()
        children = lambda b, i: [i + 1] if i < n[b] else []  # noqa: E731
        token = lambda b, c: int(s["drafts"][b, c - 1])  # noqa: E731
        u_of = lambda b, c: float(u[b, c - 1])  # noqa: E731
    else:
        N = s["tokens"].shape[1]
        prow = lambda b, i: _row64(s["target"][b * N + i], T[b], None, None)  # noqa: E731
        qrow = lambda b, i: None if s["draft"] is None or T[b] <= 0 else _row64(s["draft"][b * N + i], T[b], None, None).exp()  # noqa: E731
        parents = s["parent"].cpu().tolist()
        children = lambda b, i: [c for c in range(n[b]) if parents[b][c] == i]  # noqa: E731
        token = lambda b, c: int(s["tokens"][b, c])  # noqa: E731
        u_of = lambda b, c: float(u[b, c])  # noqa: E731
    prob = torch.zeros(B, N, dtype=torch.float64)
    for b in range(B):
        for i, (_, _, p) in enumerate(_walk64(s, b, children, token, prow, qrow, u_of)):
            prob[b, i] = p
    return (None, None, prob) if case["op"] == "verify" else (None, None, None, prob)
