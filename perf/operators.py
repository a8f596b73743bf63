"""Workloads by which the speed of the language-model operators is judged (``pyjuice_b200.lm``).

A case is one call of one operator:

    top      ``lm.top_logits``: the largest logits of a teacher's rows, with the rows' log-normalisers
    teach    ``lm.expected_log_probs``: log-probabilities of leaf tables expected under a teacher's top logits, forward
             and (``grad``) backward; ``tied``: one table for all positions, as the emissions of a homogeneous HMM
    beam     ``lm.beam_select``: the best continuations over beams and vocabulary
    reorder  ``lm.reorder``: states of the beams that were continued

With ``own`` false every operator is computed in its plain form from elementary torch operations.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "int64": torch.int64}
NEG_INF = float("-inf")


def _top(rows, vocab, k, dtype, temperature=1.0, **more):
    return dict(op="top", rows=rows, vocab=vocab, k=k, dtype=dtype, temperature=temperature, **more)


def _teach(length, latents, cats, batch, k, dtype, tied, grad, temperature=1.0, **more):
    return dict(op="teach", length=length, latents=latents, cats=cats, batch=batch, k=k, dtype=dtype, tied=tied,
                grad=grad, temperature=temperature, **more)


def _beam(batch, beams, vocab, n, dtype, normalize=True, **more):
    return dict(op="beam", batch=batch, beams=beams, vocab=vocab, n=n, dtype=dtype, normalize=normalize, **more)


def _reorder(batch, beams, n, latents, dtype, dim, tokens=0, **more):
    return dict(op="reorder", batch=batch, beams=beams, n=n, latents=latents, dtype=dtype, dim=dim, tokens=tokens, **more)


def listed():
    return [
        # the next token of one sequence: latency
        _top(1, 50257, 8, "bfloat16", name="top-1x50257-k8-bf16"),
        # a teacher's logits over a training batch of 64 sequences of 128 tokens
        _top(8192, 32768, 32, "bfloat16", 2.0, name="top-8192x32768-k32-bf16"),
        # odd sizes, many slots, 32-bit logits of a scored test set
        _top(1001, 50257, 100, "float32", name="top-1001x50257-k100-fp32"),
        # a hidden tree over 14 x 14 pixels learns from a teacher's pixel distributions: a table for each variable
        _teach(196, 256, 256, 100, 16, "float32", False, True, name="teach-hclt-196v-k256-b100"),
        # language-model HMM with tied emissions, distilled from a teacher's top 32 of 32768 logits: the largest work
        _teach(128, 4096, 32768, 64, 32, "bfloat16", True, True, 2.0, name="teach-hmm-128t-k4096-b64"),
        # a mid-size HMM with an odd batch and a small vocabulary
        _teach(64, 512, 1000, 77, 10, "float32", True, True, name="teach-hmm-64t-k512-b77"),
        # one sequence scored against a teacher, forward only
        _teach(128, 1024, 50257, 1, 50, "float16", True, False, name="score-hmm-128t-k1024-b1"),
        # a student that is itself a language model: every position has a row of its own
        _teach(2048, 1, 32768, 1, 64, "bfloat16", False, True, name="teach-rows-2048x32768"),
        # one prompt, four beams: latency of a decoding step
        _beam(1, 4, 50257, 8, "float32", name="beam-b1-k4-v50257"),
        # a serving batch of wide beams, some of them finished
        _beam(64, 16, 32768, 32, "bfloat16", name="beam-b64-k16-v32768"),
        # HMM states, one column a beam
        _reorder(64, 16, 16, 4096, "float32", 1, name="reorder-hmm-k4096-64x16"),
        # a small batch of beams with their states and the tokens so far, one row a beam
        _reorder(4, 4, 4, 1024, "bfloat16", 0, 128, name="reorder-rows-k1024-4x4"),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(["top", "teach", "teach", "beam", "reorder"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "top":
        vocab = _spread(rng, 16, 131072)
        return _top(_spread(rng, 1, min(8192, (1 << 27) // vocab)), vocab, _spread(rng, 1, min(128, vocab)), dtype,
                    rng.choice([0.5, 1.0, 2.0]))
    if op == "beam":
        vocab, beams = _spread(rng, 64, 131072), _spread(rng, 1, 32)
        return _beam(_spread(rng, 1, max(1, min(64, (1 << 25) // (vocab * beams)))), beams, vocab, rng.choice([beams, 2 * beams]),
                     dtype, rng.choice([True, True, False]))
    if op == "reorder":
        beams = _spread(rng, 1, 32)
        return _reorder(_spread(rng, 1, 64), beams, rng.choice([beams, 2 * beams]), _spread(rng, 16, 8192), dtype,
                        rng.randint(0, 1), rng.choice([0, 0, _spread(rng, 1, 512)]))
    k, grad = _spread(rng, 1, 64), rng.choice([True, True, False])
    if rng.random() < 0.6:
        cats, latents = _spread(rng, 64, 50257), _spread(rng, 16, 2048)
        length = _spread(rng, 1, 128)
        batch = _spread(rng, 1, max(1, min(128, (1 << 28) // (length * latents * k))))
        return _teach(length, latents, cats, batch, min(k, cats), dtype, True, grad, rng.choice([1.0, 2.0]))
    cats, latents, length = _spread(rng, 2, 256), _spread(rng, 1, 256), _spread(rng, 16, 400)
    k = min(k, cats)
    batch = _spread(rng, 8, max(8, min(512, (1 << 28) // (length * latents * k))))
    return _teach(length, latents, cats, batch, k, dtype, False, grad, rng.choice([1.0, 2.0]))


# ---- inputs --------------------------------------------------------------------------------------------------------

def _vocabulary_logits(g, rows, vocab):
    """Logits of a language model: word frequencies follow Zipf's law, each row has its own preferences."""
    rank = torch.randperm(vocab, device=DEVICE, generator=g).float() + 1.0
    x = torch.randn(rows, vocab, device=DEVICE, generator=g)
    return x.mul_(2.0).sub_(rank.log())


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case)
    if case["op"] == "top":
        s["logits"] = _vocabulary_logits(g, case["rows"], case["vocab"]).to(TYPES[case["dtype"]])
    elif case["op"] == "beam":
        B, K, V = case["batch"], case["beams"], case["vocab"]
        x = _vocabulary_logits(g, B * K, V).view(B, K, V)
        if not case["normalize"]:
            x = x.log_softmax(-1)
        if V > 8:
            x[..., 5:7] = NEG_INF                       # tokens that may not be said
        s["logits"] = x.to(TYPES[case["dtype"]])
        s["scores"] = torch.rand(B, K, device=DEVICE, generator=g).mul_(-6.0).sub_(12.0)
        s["finished"] = torch.rand(B, K, device=DEVICE, generator=g) < 0.1
        if B > 2:
            s["scores"][1, 1:] = NEG_INF                # a sequence at its first step: one live beam
    elif case["op"] == "reorder":
        B, K, n, L, d = case["batch"], case["beams"], case["n"], case["latents"], TYPES[case["dtype"]]
        s["parents"] = torch.randint(K, (B, n), device=DEVICE, generator=g)
        s["states"] = [torch.randn((B * K, L) if case["dim"] == 0 else (L, B * K), device=DEVICE, generator=g).to(d)]
        if case["tokens"]:
            shape = (B * K, case["tokens"]) if case["dim"] == 0 else (case["tokens"], B * K)
            s["states"].append(torch.randint(50257, shape, device=DEVICE, generator=g))
    else:
        T, M, C, B, K = (case[name] for name in ("length", "latents", "cats", "batch", "k"))
        table = torch.randn((1 if case["tied"] else T) * M, C, device=DEVICE, generator=g).mul_(1.5).log_softmax(-1)
        s["log_probs"] = (table if case["tied"] else table.view(T, M, C)).requires_grad_(case["grad"])
        x = _vocabulary_logits(g, T * B, C)
        values, ids = x.topk(K, dim=-1)
        values, ids = values.view(B, T, K), ids.view(B, T, K)
        if K > 2:                                       # some positions have fewer slots, the ends of some sequences none
            ids[torch.rand(B, T, device=DEVICE, generator=g) < 0.1, -1] = -1
        if T > 4:
            ids[torch.rand(B, device=DEVICE, generator=g) < 0.25, -(T // 4):] = -1
        s["ids"], s["logits"] = ids, values.to(TYPES[case["dtype"]])
        if case["grad"]:
            s["flow"] = torch.rand(T, M, B, device=DEVICE, generator=g)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _keys(x):
    """Whole numbers in the order of the 32-bit values `x` (a last dimension of places), a lower place first among equals."""
    x = torch.where(x == 0, torch.zeros_like(x), x)     # (one zero)
    bits = x.view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    return (bits << 31) - torch.arange(x.size(-1), device=x.device)


def _largest(x, k):
    """The places of the k largest values of each row, a lower place first among equals."""
    return _keys(x).topk(k, dim=-1).indices


def _plain_top(s):
    x = s["logits"].float()
    x = torch.where(x.isnan(), NEG_INF, x)
    ids = _largest(x, s["k"])
    values = x.gather(-1, ids)
    z = x.double() / s["temperature"]
    m = z.amax(-1, keepdim=True)
    norm = ((z - m).exp().sum(-1).log() + m[:, 0]).float()
    return dict(ids=torch.where(values == NEG_INF, -1, ids), logits=values.to(s["logits"].dtype), log_norm=norm)


def _plain_beam(s):
    B, K, V = s["logits"].shape
    x, score = s["logits"].float(), s["scores"].double().unsqueeze(-1)
    x = torch.where(x.isnan(), NEG_INF, x)
    only = torch.where(torch.arange(V, device=x.device) == 0, 0.0, NEG_INF)
    x = torch.where(s["finished"].unsqueeze(-1), only, x)
    own_best = _largest(x, min(s["n"], V)).sort(-1).values           # places ascending, so that a stable sort settles ties
    best = x.gather(-1, own_best).double()
    if s["normalize"]:
        z = x.double()
        m = z.amax(-1, keepdim=True)
        norm = (z - m).exp().sum(-1, keepdim=True).log() + m
        best = best - torch.where(s["finished"].unsqueeze(-1), 0.0, norm)
    flat = torch.where(best == NEG_INF, NEG_INF, best + score).reshape(B, -1)
    got, at = flat.sort(dim=-1, descending=True, stable=True)
    got, at = got[:, :s["n"]], at[:, :s["n"]]
    none = got == NEG_INF
    tokens = own_best.reshape(B, -1).gather(1, at)
    parents = at // own_best.size(-1)
    return dict(scores=got.float(), parents=torch.where(none, 0, parents), tokens=torch.where(none, -1, tokens))


def _plain_reorder(s):
    B, K = s["batch"], s["beams"]
    at = (s["parents"] + K * torch.arange(B, device=s["parents"].device).unsqueeze(1)).reshape(-1)
    return [x.index_select(s["dim"], at) for x in s["states"]]


def _plain_teach(s):
    table = s["log_probs"].detach().view(-1, s["latents"], s["cats"])
    ids, x = s["ids"].transpose(0, 1), s["logits"].float().transpose(0, 1) / s["temperature"]       # [T, B, K]
    x = torch.where(ids >= 0, x, NEG_INF)
    m = x.amax(-1, keepdim=True)
    e = torch.where(ids >= 0, (x - torch.where(m == NEG_INF, 0.0, m)).exp(), 0.0)
    q = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    T, B, K = ids.shape
    at = ids.clamp_min(0) + (0 if s["tied"] else s["cats"] * torch.arange(T, device=ids.device).view(T, 1, 1))
    rows = table.transpose(1, 2).reshape(-1, s["latents"])           # [categories of all tables, nodes]
    picked = rows[at.reshape(-1)].view(T, B, K, -1)
    values = (picked * q.unsqueeze(-1)).sum(2).transpose(1, 2).contiguous()
    if not s["grad"]:
        return dict(values=values)
    spread = s["flow"].transpose(1, 2).unsqueeze(2) * q.unsqueeze(-1)                               # [T, B, K, M]
    grad = torch.zeros_like(rows).index_add_(0, at.reshape(-1), spread.reshape(-1, s["latents"]))
    grad = grad.view(table.size(0), s["cats"], s["latents"]).transpose(1, 2).reshape(s["log_probs"].shape)
    return dict(values=values, grad=grad)


def run(state):
    s = state
    if not own:
        return {"top": _plain_top, "beam": _plain_beam, "reorder": _plain_reorder, "teach": _plain_teach}[s["op"]](s)
    from pyjuice_b200 import lm
    if s["op"] == "top":
        top = lm.top_logits(s["logits"], s["k"], temperature=s["temperature"])
        return dict(ids=top.ids, logits=top.logits, log_norm=top.log_norm)
    if s["op"] == "beam":
        scores, parents, tokens = lm.beam_select(s["logits"], s["scores"], s["n"], finished=s["finished"], pad_id=0,
                                                 normalize=s["normalize"])
        return dict(scores=scores, parents=parents, tokens=tokens)
    if s["op"] == "reorder":
        return lm.reorder(s["parents"], *s["states"], dim=s["dim"])
    values = lm.expected_log_probs(s["log_probs"], lm.TopLogits(s["ids"], s["logits"], temperature=s["temperature"]))
    if not s["grad"]:
        return dict(values=values)
    grad, = torch.autograd.grad(values, s["log_probs"], s["flow"])
    return dict(values=values.detach(), grad=grad)


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "reorder":
        beam = torch.arange(case["batch"] * case["n"], device=DEVICE) // case["n"] * case["beams"] + s["parents"].flatten()
        first = s["states"][0].double()
        return [first[beam] if case["dim"] == 0 else first[:, beam]] + [None] * (len(s["states"]) - 1)
    if case["op"] == "top":
        parts = []
        for x in s["logits"].split(1024):
            parts.append(torch.logsumexp(x.double() / case["temperature"], -1))
        return dict(ids=None, logits=None, log_norm=torch.cat(parts))
    if case["op"] == "beam":
        B, K, V = s["logits"].shape
        found = []
        for x, score, done in zip(s["logits"], s["scores"].double(), s["finished"]):
            total = x.double() - (torch.logsumexp(x.double(), -1, keepdim=True) if case["normalize"] else 0.0) + score[:, None]
            total[done] = NEG_INF
            total[done, 0] = score[done]
            best = total.reshape(-1).topk(min(case["n"], K * V)).values
            found.append(best)
        return dict(scores=torch.stack(found), parents=None, tokens=None)
    T, M, C, B, K = (case[name] for name in ("length", "latents", "cats", "batch", "k"))
    tables = s["log_probs"].detach().view(-1, M, C)
    values = torch.zeros(T, M, B, dtype=torch.float64, device=DEVICE)
    grad = torch.zeros(tables.size(0), C, M, dtype=torch.float64, device=DEVICE) if case["grad"] else None
    turned = tables[0].t().contiguous() if case["tied"] else None
    for t in range(T):
        ids, z = s["ids"][:, t], s["logits"][:, t].double() / case["temperature"]
        z = z.masked_fill(ids < 0, NEG_INF)
        q = torch.softmax(z, -1).nan_to_num(0.0)
        table = turned if case["tied"] else tables[t].t()
        for k in range(K):
            row = ids[:, k].clamp_min(0)
            values[t] += (table[row].double() * q[:, k, None]).t()
            if grad is not None:
                grad[0 if case["tied"] else t].index_add_(0, row, s["flow"][t].t().double() * q[:, k, None])
    if grad is None:
        return dict(values=values)
    return dict(values=values, grad=grad.transpose(1, 2).reshape(s["log_probs"].shape))


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    """Inputs read once, outputs written once.  The operations: one exponential and one sum per logit of a vocabulary
    row; one product and one sum per slot of the teacher, node and sample, once for each direction."""
    size = {"float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
    if case["op"] == "top":
        read, written = case["rows"] * case["vocab"] * size, case["rows"] * (case["k"] * (size + 8) + 4)
        return {"bytes": float(read + written), "flops": 2.0 * case["rows"] * case["vocab"]}
    if case["op"] == "beam":
        rows = case["batch"] * case["beams"]
        return {"bytes": float(rows * (case["vocab"] * size + 5) + case["batch"] * case["n"] * 20),
                "flops": 2.0 * rows * case["vocab"]}
    if case["op"] == "reorder":
        row = case["latents"] * size + case["tokens"] * 8
        rows = case["batch"] * min(case["beams"], case["n"])
        return {"bytes": float(rows * row + case["batch"] * case["n"] * (row + 8)), "flops": 0.0}
    table = 4.0 * case["latents"] * case["cats"] * (1 if case["tied"] else case["length"])
    slots = 1.0 * case["length"] * case["batch"] * case["k"]
    out = 4.0 * case["length"] * case["batch"] * case["latents"]
    # no more of the tables is needed than the slots name
    read = min(table, 4.0 * slots * case["latents"])
    once = slots * (size + 8) + read + out
    return {"bytes": once + (out + table if case["grad"] else 0.0),
            "flops": 2.0 * slots * case["latents"] * (2 if case["grad"] else 1)}
