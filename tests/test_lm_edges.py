"""Operators of language-model circuits at the edges: rows of large logits, continuations whose scores are equal or nearly so, tokens
and slots that say something unusual, every form of the selection at every cut of a row."""
import math

import pytest
import torch

from pyjuice_b200 import lm

NEG_INF, NAN, INF = float("-inf"), float("nan"), float("inf")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
STEP = 2.0 ** -24                    # half a step of fp32, relative


def norm_tol(vocab):
    """How far a log-normaliser may be off before it is rounded to fp32, in steps of 2^-24 of the sum: an exponential of 2^-22 (4); its
    argument, rounded twice, whose distance from the maximum is at most log2(vocab) + 2 bits on average under the weights (2 ln 2
    each); up to 34 sums in a tile; per tile of a lane (128 logits of a part or more) a sum, and a product with an
    exponential where the maximum rises (6); and as many joins of lanes (5 + 5, arguments of 2 log2(vocab) bits)."""
    bits = math.log2(vocab) + 2
    return (4 + 2 * 0.7 * bits + 34 + 6 * (vocab // 1024 + 1) + 10 + 2 * 0.7 * bits) * STEP


def exact_norm(row):
    """log sum exp of a list, the sum rounded once (NaN counts nothing)."""
    row = [v for v in row if v > NEG_INF]
    if not row:
        return NEG_INF
    m = max(row)
    return INF if m == INF else m + math.log(math.fsum(math.exp(v - m) for v in row))


def best(x, scores, n, finished=None, pad=0):
    """The n best continuations of one sequence, ``x`` [K, V], by the definition in 64 bits: [(score, parent, token)]."""
    found = []
    for k, (row, s) in enumerate(zip(x.double().tolist(), scores.double().tolist())):
        if not s > NEG_INF:
            continue
        if finished is not None and bool(finished[k]):
            found.append((-s, k, pad))
            continue
        norm = exact_norm(row)
        found += sorted((-((s + v) - norm), k, t) for t, v in enumerate(row) if v > NEG_INF and norm < INF)[:n]
    found = sorted(found)[:n]
    return [(-s, k, t) for s, k, t in found] + [(NEG_INF, 0, -1)] * (n - len(found))


def check_best(x, scores, n, finished=None, pad=0):
    got = [t.cpu() for t in lm.beam_select(x, scores, n, finished, pad)]
    for b in range(x.size(0)):
        want = best(x[b], scores[b], n, None if finished is None else finished[b], pad)
        assert got[1][b].tolist() == [w[1] for w in want] and got[2][b].tolist() == [w[2] for w in want]
        for s, w in zip(got[0][b].tolist(), want):
            assert s == w[0] or abs(s - w[0]) <= norm_tol(x.size(2)) + abs(w[0]) * STEP


LARGE = [-1e9, 1e9, 1e5, -1e6, 3e7, -1e12, -1e30, 2e38, torch.finfo(torch.float32).min]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", LARGE)
def test_rows_of_large_logits_have_their_normaliser(value, dtype):
    """A row that a mask's number fills altogether, or in part, scores as any other row: what counts is how far logits are apart."""
    value = max(min(value, torch.finfo(dtype).max), torch.finfo(dtype).min)
    for B, K, V in ((1, 4, 5003), (700, 4, 257), (2, 4, 60)):
        x = torch.randn(1, K, V, generator=torch.Generator().manual_seed(V))
        x[:, 0] = value
        x[:, 1] += value
        x[:, 2, ::7] = value
        x = x.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)
        scores = torch.tensor([[-3.0, -5.0, -4.0, -6.0]])
        got = [t.cpu() for t in lm.beam_select(x.expand(B, K, V).contiguous().cuda(), scores.expand(B, K).cuda(), 9)]
        want = best(x[0], scores[0], 9)
        for b in (0, B - 1):
            assert got[1][b].tolist() == [w[1] for w in want] and got[2][b].tolist() == [w[2] for w in want]
            for s, w in zip(got[0][b].tolist(), want):
                assert abs(s - w[0]) <= norm_tol(V) + abs(w[0]) * STEP
        for temperature in (0.5, 1.0, 2.0, 30.0):
            norm = lm.top_logits(x[0].cuda(), 1, temperature).log_norm.double().cpu().tolist()
            for row, n in zip(x[0].double().tolist(), norm):
                want = exact_norm([v / temperature for v in row])
                # (a normaliser beyond the range of fp32 is infinite)
                if abs(want) < torch.finfo(torch.float32).max:
                    assert abs(n - want) <= norm_tol(V) + abs(want) * STEP, (temperature, n, want)


def check_all_alike(x, scores, n, B, finished=None):
    """One sequence, B times."""
    rows = lambda t: t.expand(B, *t.shape[1:]).contiguous().cuda()
    got = [t.cpu() for t in lm.beam_select(rows(x), rows(scores), n, None if finished is None else rows(finished), 3)]
    want = best(x[0], scores[0], n, None if finished is None else finished[0], 3)
    assert bool((got[1] == torch.tensor([w[1] for w in want])).all()) and bool((got[2] == torch.tensor([w[2] for w in want])).all())
    for s, w in zip(got[0][0].tolist(), want):
        assert s == w[0] or abs(s - w[0]) <= norm_tol(x.size(2)) + abs(w[0]) * STEP


# (a warp a row, a CTA a row, parts of a row; a beam's rows begin at other places of 16 bytes than its neighbours')
CUTS = [(2, 6, 257), (1, 6, 4501), (3, 5, 50257), (320, 6, 5001), (1, 128, 41)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V", CUTS)
def test_equal_beams_go_by_their_place(B, K, V, dtype):
    x = (torch.randn(1, 1, V, generator=torch.Generator().manual_seed(V)) * 3).to(dtype).expand(1, K, V)
    scores = torch.full((1, K), -3.0)
    for n in (1, K - 1, K, min(2 * K + 1, 128)):
        check_all_alike(x, scores, n, B)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V", CUTS)
def test_beams_whose_normalisers_differ_by_little(B, K, V, dtype):
    """Rows that differ in a logit of next to no weight: the order of their continuations is that of their normalisers in 64 bits,
    which are 1e-10 to 1e-6 apart."""
    g = torch.Generator().manual_seed(K + V)
    x = (torch.randn(1, 1, V, generator=g) * 3).to(dtype).expand(1, K, V).clone()
    low = x[0, 0].float().argmin()
    x[0, :, low] += (torch.randperm(K, generator=g).float() * (8.0 / K)).to(dtype)
    scores = torch.full((1, K), -3.0)
    norms = [exact_norm(row) for row in x[0].double().tolist()]
    assert K < 10 and 1e-11 < max(norms) - min(norms) < 1e-4 or K == 128
    for n in (2, K - 1, min(3 * K, 128)):
        check_all_alike(x, scores, n, B)
    # finished beams in between, at scores within a rounding of a continuation's
    finished = torch.zeros(1, K, dtype=torch.bool)
    finished[0, 1::3] = True
    top = x[0, 0].double().max() - 3.0
    for k in range(1, K, 3):
        scores[0, k] = float(top) - norms[0]
    check_all_alike(x, scores, K, B, finished)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [3, 40, 300])
def test_logits_of_plus_infinity_share_the_weight_under_a_given_normaliser(K):
    ids = torch.arange(K).expand(1, 3, K)
    x = torch.randn(1, 3, K, generator=torch.Generator().manual_seed(1))
    x[0, 0, 1], x[0, 0, K - 1], x[0, 1, 0] = INF, INF, INF
    log_probs = -torch.arange(1.0, K + 1).expand(2, K).contiguous()
    log_probs[0, 0] = 0.0                              # (nothing of an infinite weight times zero)
    norm = torch.tensor([[2.0, 0.0, 7.0]])
    lp = log_probs.cuda().requires_grad_()
    got = lm.expected_log_probs(lp, lm.TopLogits(ids.cuda(), x.cuda(), 1.0, norm.cuda()))
    assert got[0, :, 0].tolist() == [-(2.0 + K) / 2] * 2                     # two of them, a half each
    assert got[1, :, 0].tolist() == [0.0, -1.0]
    q = (x[0, 2].double() - 7.0).exp()                 # the position without any keeps its normaliser
    want = (q * log_probs.double()).sum(-1)
    assert float((got[2, :, 0].detach().double().cpu() - want).abs().max()) <= (K + 12) * 2 * STEP * float(want.abs().max())
    grad, = torch.autograd.grad(got[:2].sum(), lp)
    want = torch.zeros(K)
    want[1], want[K - 1], want[0] = 0.5, 0.5, 1.0
    assert torch.equal(grad.cpu(), want.expand(2, K))


# ---- decoding: three products of 8-bit-mantissa halves per factor (2^-16 each way) and fp32 sums over the states, per token
DECODE_TOL = 2.0 ** -13


def hmm(latents, vocab, length=4, seed=0):
    """A circuit and its (alpha, beta, gamma) in 64 bits."""
    import pyjuice_b200 as pj
    g = torch.Generator().manual_seed(seed)
    p = lambda *s: torch.rand(*s, generator=g).pow(3).add_(1e-4)
    alpha, beta, gamma = p(latents, latents), p(latents, vocab), p(latents)
    alpha, beta, gamma = alpha / alpha.sum(1, keepdim=True), beta / beta.sum(1, keepdim=True), gamma / gamma.sum()
    torch.manual_seed(seed)
    ns = pj.structures.HMM(seq_length=length, num_latents=latents, num_emits=vocab, alpha=alpha, beta=beta, gamma=gamma)
    return pj.compile(ns, verbose=False).to("cuda:0"), (alpha.double(), beta.double(), gamma.double())


@pytest.mark.gpu
def test_next_tokens_of_a_joint_state():
    """Without the tokens' log-probabilities a state goes on as a joint distribution; the next token's probabilities are the same."""
    from pyjuice_b200.decoding import HMMDecoder
    pc, (alpha, beta, z) = hmm(20, 33)
    decoder = HMMDecoder(pc)
    state = decoder.start(2)
    said = torch.tensor([[3, 7, 0, 32], [1, 1, 1, 1]])
    rows = [z, z]
    for t in range(4):
        state = decoder.advance(state, said[:, t].cuda())
        rows = [(r * beta[:, v]) @ alpha for r, v in zip(rows, said[:, t].tolist())]
        got = decoder.log_probs(state)
        want = torch.stack([((r / r.sum()) @ beta).log() for r in rows])
        assert float((got.double().cpu() - want).abs().max()) < (t + 2) * DECODE_TOL
        mass = torch.stack([r.sum().log() for r in rows])
        assert float((state.logsumexp(0).double().cpu() - mass).abs().max()) < (t + 2) * DECODE_TOL
    assert float((decoder.log_probs(state + 40) - got).abs().max()) < 40 * 8 * STEP + DECODE_TOL
    state[:, 1] = NEG_INF                              # nothing is possible
    got = decoder.log_probs(state)
    assert bool((got[1] == NEG_INF).all()) and bool(got[0].isfinite().all())


def after(model, tokens):
    """(log p(tokens), next-token log-probabilities) in 64 bits; None: a token that is not known."""
    alpha, beta, z = model
    total = 0.0
    for t in tokens:
        z = z if t is None else z * beta[:, t]
        total += math.log(float(z.sum())) if t is not None else 0.0
        z = (z / z.sum()) @ alpha
    return total, (z @ beta).log()


@pytest.mark.gpu
@pytest.mark.parametrize("latents,vocab", [(20, 33), (16, 9), (64, 700)])
def test_tokens_that_are_unknown_or_not_in_the_vocabulary(latents, vocab):
    from pyjuice_b200.decoding import HMMDecoder, beam_search
    pc, model = hmm(latents, vocab)
    decoder = HMMDecoder(pc)
    prompts = torch.tensor([[3, -1, 2], [-1, -7, -2 ** 40], [5, 1, -1], [5, vocab, 1], [2 ** 40, 1, 1], [4, 3, 2]])
    names = lambda row: [None if t < 0 else t for t in row]
    for ids in (torch.int64, torch.int32):
        rows = prompts.clamp(-2 ** 31, 2 ** 31 - 1).to(ids)
        tokens, scores = beam_search(decoder, rows, 1, 4)
        for b, row in enumerate(prompts.tolist()):
            if max(row) >= vocab:
                assert bool((scores[b] == NEG_INF).all()) and bool((tokens[b] == -1).all())
                continue
            want, at = after(model, names(row))[1].sort(descending=True)
            assert float((scores[b].double().cpu() - want[:4]).abs().max()) < 5 * DECODE_TOL
            if float((want[:4] - want[1:5]).min()) > 10 * DECODE_TOL:
                assert tokens[b, :, 0].tolist() == at[:4].tolist()
    # the same through `advance`, with and without the tokens' log-probabilities; unsigned tokens
    joint = own = decoder.start(6)
    for t in range(3):
        said = prompts[:, t].cuda()
        heard = decoder.log_probs(own).gather(1, said.clamp(0, vocab - 1)[:, None])[:, 0]
        own = decoder.advance(own, said, torch.where(said < 0, 0.0, heard))
        joint = decoder.advance(joint, said)
    a, b = decoder.log_probs(own).double().cpu(), decoder.log_probs(joint).double().cpu()
    for n, row in enumerate(prompts.tolist()):
        if max(row) >= vocab:
            assert bool((own[:, n] == NEG_INF).all()) and bool((joint[:, n] == NEG_INF).all()) and bool((a[n] == NEG_INF).all())
        else:
            total, want = after(model, names(row))
            assert float((a[n] - want).abs().max()) < 5 * DECODE_TOL and float((b[n] - want).abs().max()) < 5 * DECODE_TOL
            assert abs(float(joint[:, n].logsumexp(0)) - total) < 5 * DECODE_TOL
    assert torch.equal(decoder.advance(decoder.start(1), torch.tensor([7], dtype=torch.uint8).cuda()), decoder.advance(decoder.start(1), torch.tensor([7]).cuda()))


@pytest.mark.gpu
def test_an_impossible_token_ends_its_own_beam_alone():
    import pyjuice_b200 as pj
    from pyjuice_b200.decoding import HMMDecoder, beam_search
    eye = torch.eye(4)
    beta = torch.cat([eye, torch.zeros(4, 2)], 1)              # state z says token z; tokens 4 and 5 are never said
    alpha = torch.roll(eye, 1, 1)                              # and is followed by the next state
    ns = pj.structures.HMM(seq_length=3, num_latents=4, num_emits=6, alpha=alpha, beta=beta, gamma=torch.full((4,), 0.25))
    decoder = HMMDecoder(pj.compile(ns, verbose=False).to("cuda:0"))
    tokens, scores = beam_search(decoder, torch.tensor([[4], [1], [5], [-1]]), 3, 2)
    assert bool((scores[[0, 2]] == NEG_INF).all()) and bool((tokens[[0, 2]] == -1).all())
    assert tokens[1, 0].tolist() == [2, 3, 0] and abs(float(scores[1, 0])) < 3 * DECODE_TOL
    # a sum of the circuit's kernels is 1e-24 of its largest term at least, so that a sentence of probability zero has log(1e-24) (and
    # the selection's normaliser is off by 5 tokens of it: nothing)
    assert abs(float(scores[1, 1]) - math.log(1e-24)) < 3 * DECODE_TOL + 55.3 * STEP
    assert bool((scores[3] + math.log(4)).abs().max() < 3 * DECODE_TOL)


def test_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad
    lp, parents = torch.zeros(4, 9), torch.zeros(2, 3, dtype=torch.int64)
    teacher = lm.TopLogits(torch.zeros(2, 3, 5, dtype=torch.int64), torch.zeros(2, 3, 5))
    calls = (lambda x: lm.expected_log_probs(x, teacher), lambda x: lm.reorder(parents, x)[0])
    for f in calls:
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(forward_ad.make_dual(lp, torch.ones_like(lp)))
            with pytest.raises(NotImplementedError):               # (a tensor without a tangent: no CPU path, as ever)
                f(lp)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(f, (lp,), (torch.ones_like(lp),))
        with pytest.raises(NotImplementedError):
            f(lp)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        calls[0](forward_ad.make_dual(lp.clone().requires_grad_(), torch.ones_like(lp)))


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [True, False])
def test_more_samples_than_a_grid_has_rows(tied):
    """4.2 million samples, both directions: 65536 tiles of 64 samples and a few."""
    B, M, C = 65536 * 64 + 37, 2, 3
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(-1, C, (B, 1, 1), generator=g).cuda()
    lp = torch.randn(M, C, generator=g).cuda() if tied else torch.randn(1, M, C, generator=g).cuda()
    lp.requires_grad_()
    out = lm.expected_log_probs(lp, lm.TopLogits(ids, torch.zeros(B, 1, 1, device="cuda")))
    table, at = lp.detach().view(M, C), ids.flatten()
    assert torch.equal(out.detach()[0], torch.where(at >= 0, table[:, at.clamp_min(0)], 0.0))
    flow = torch.randint(0, 3, (1, M, B), generator=g).float().cuda()            # (sums of whole numbers below 2^24 are exact)
    grad, = torch.autograd.grad(out, lp, flow)
    want = torch.stack([flow[0][:, at == c].double().sum(1) for c in range(C)], 1)
    assert float(want.max()) < 2 ** 24 and torch.equal(grad.view(M, C).double(), want)


@pytest.mark.gpu
def test_batches_of_many_slot_counts_leave_no_passes_behind():
    """Captured passes of two slot counts at most, whatever comes; each replays on the buffer it was captured with."""
    pc, _ = hmm(128, 700, length=16)
    g = torch.Generator().manual_seed(0)
    top = lambda K: lm.TopLogits(torch.randint(700, (32, 16, K), generator=g).cuda(), torch.randn(32, 16, K, generator=g).cuda())

    def step(teacher):
        pc.init_param_flows(flows_memory=0.0)
        lls = pc(teacher).detach().clone()
        pc.backward(teacher)
        return lls, pc.input_layer_group[0].param_flows.clone()

    held, counts = [], []
    for K in (3, 3, 3, 8, 8, 3, 8, 3, 5, 5, 5, 3, 3, 3, 1, 1, 1, 9, 9, 9, 12, 12, 12, 20, 20, 20, 3, 3, 3):
        teacher = top(K)
        held.append((teacher, step(teacher)))
        counts.append((len(pc._graphs), len(pc._bk_par_pending)))
    # a first pass and those after it (with and without new tables), twice, forward and backward
    assert max(c for c, _ in counts[8:]) <= max(c for c, _ in counts[:8]) and max(c for _, c in counts) <= 4
    assert len(pc._teacher_bufs) == 2
    pc.use_cuda_graphs = False
    for teacher, (lls, flows) in held:
        eager = step(teacher)
        assert torch.equal(eager[0], lls) and torch.equal(eager[1], flows)


@pytest.mark.gpu
@pytest.mark.parametrize("latents,vocab", [(1, 5), (2, 1), (3, 70), (20, 33), (64, 65), (65, 300), (96, 1000), (130, 9), (201, 500), (1000, 2001)])
def test_decoders_of_any_number_of_states(latents, vocab):
    """Blocks of 64 states at least, few tiles of parameters, and the distributions of the definition."""
    from pyjuice_b200.decoding import HMMDecoder, beam_search
    pc, model = hmm(latents, vocab)
    decoder = HMMDecoder(pc)
    for ns in (decoder._speak_ns, decoder._step_ns):
        assert ns.edge_ids.size(1) <= (latents / 64 + 1) * (max(latents, vocab) / 64 + 2)
    said = torch.randint(vocab, (3, 3), generator=torch.Generator().manual_seed(1))
    state, joint = decoder.start(3), decoder.start(3)
    for t in range(3):
        got, again = decoder.log_probs(state), decoder.log_probs(joint)
        assert state.shape == (latents, 3) and got.shape == (3, vocab)
        want = torch.stack([after(model, row[:t].tolist())[1] for row in said])
        assert float((got.double().cpu() - want).abs().max()) < (t + 1) * DECODE_TOL
        assert float((again.double().cpu() - want).abs().max()) < (t + 1) * DECODE_TOL
        tokens = said[:, t].cuda()
        state = decoder.advance(state, tokens, got.gather(1, tokens[:, None])[:, 0])
        joint = decoder.advance(joint - 400.0, tokens)             # (a state of any size: what it lacks does not show)
    before = decoder.log_probs(state)
    decoder.reload()
    assert torch.equal(decoder.log_probs(state), before)
    tokens, scores = beam_search(decoder, said, 2, 3)
    assert tokens.shape == (3, 3, 2) and bool(scores[:, :min(3, vocab)].isfinite().all())


@pytest.mark.gpu
def test_no_sequences_and_no_prompts():
    from pyjuice_b200.decoding import HMMDecoder, beam_search
    decoder = HMMDecoder(hmm(20, 33)[0])
    for prompts in (torch.empty(0, 4, dtype=torch.int64), None):
        tokens, scores = beam_search(decoder, prompts, 3, 5, batch=0)
        assert tokens.shape == (0, 5, 3) and scores.shape == (0, 5)
    a, b = beam_search(decoder, torch.empty(2, 0, dtype=torch.int32), 3, 5), beam_search(decoder, None, 3, 5, batch=2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert decoder.advance(decoder.start(0), torch.empty(0, dtype=torch.int64, device="cuda")).shape == (20, 0)
    assert decoder.log_probs(decoder.start(0)).shape == (0, 33)


@pytest.mark.gpu
def test_a_decoder_follows_its_circuits_arithmetic():
    from pyjuice_b200.decoding import HMMDecoder
    pc, _ = hmm(256, 1024)
    x = torch.randint(1024, (32, 2), generator=torch.Generator().manual_seed(0)).cuda()

    def answers(decoder):
        state = decoder.start(32)
        for t in range(2):
            state = decoder.advance(state, x[:, t])
        return decoder.log_probs(state)

    decoder = HMMDecoder(pc)
    seen = {}
    for mode in (None, 0, 2, 1, 0, None):
        pc.sum_mode = mode
        got = answers(decoder)
        assert torch.equal(got, answers(HMMDecoder(pc)))
        assert mode not in seen or torch.equal(got, seen[mode])
        seen[mode] = got
    assert not torch.equal(seen[0], seen[2]) and torch.equal(seen[1], seen[None])


def rows_of_all_kinds(vocab, dtype, seed=0):
    """[9, vocab] at an odd place of a wider tensor."""
    g = torch.Generator().manual_seed(seed)
    at = torch.arange(vocab, dtype=torch.float32)
    noise = torch.randn(vocab, generator=g)
    rows = [noise * 3, torch.full((vocab,), -3.5), at / 512, -at / 512, torch.where(at % 977 == 5, noise, NEG_INF), at % 2,
            torch.where(at % 3 == 0, NAN, noise), torch.where(at % 4001 == 7, noise, -1e9 if dtype != torch.float16 else -6e4),
            torch.full((vocab,), torch.finfo(dtype).min)]
    wide = torch.zeros(len(rows), vocab + 5)
    wide[:, 3:3 + vocab] = torch.stack(rows)
    return wide.to(dtype).cuda()[:, 3:3 + vocab]


@pytest.fixture(params=[0, 1, 2, 7, 32], ids=lambda s: "a warp a row" if s == 0 else f"{s} parts")
def cut(request, monkeypatch):
    """Every row is walked in this form, whatever the rule for its size."""
    splits = request.param
    monkeypatch.setattr(lm, "_scratch", lambda rows, row_bytes, n, device:
                        (torch.empty(rows * (max(splits, 1) + 1) * (8 * n + 16), dtype=torch.uint8, device=device), splits))
    return splits


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,dtype", [(32769, torch.bfloat16), (100003, torch.bfloat16), (40001, torch.float16), (16385, torch.float32),
                                         (50257, torch.float32), (16384, torch.float32), (77, torch.float32)])
def test_every_form_at_every_cut(vocab, dtype, cut):
    """A warp a row over one, two and four chunks of its tiles, CTAs a row with and without parts (more of them than the row has groups
    too): the same entries."""
    x = rows_of_all_kinds(vocab, dtype)
    values = x.double().cpu()
    values = torch.where(values.isnan(), NEG_INF, values)
    want, ids = values.sort(dim=1, descending=True, stable=True)
    norms = [exact_norm(row) for row in values.tolist()]
    for k in (1, 40, min(128, vocab)):
        got = lm.top_logits(x, k)
        assert torch.equal(got.logits.double().cpu(), want[:, :k])
        assert torch.equal(got.ids.cpu(), torch.where(want[:, :k] == NEG_INF, -1, ids[:, :k]))
        for a, b in zip(got.log_norm.double().cpu().tolist(), norms):
            assert a == b or abs(a - b) <= norm_tol(vocab) + abs(b) * STEP


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,dtype", [(33001, torch.bfloat16), (40001, torch.float32)])
def test_beams_in_every_form(vocab, dtype, cut):
    x = rows_of_all_kinds(vocab, dtype)
    beams = torch.stack([x[[0, 2, 6]], x[[4, 7, 4]], x[[8, 1, 5]]])
    scores = torch.tensor([[-1.0, -3.0, -1.5], [-2.0, -2.0, -2.0], [-1.0, -1.0, -1.0]]).cuda()
    for n in (1, 9, 128):
        check_best(beams, scores, n)


@pytest.mark.gpu
@pytest.mark.parametrize("eos", [None, 3])
def test_a_captured_search_replays_on_other_prompts(eos):
    from pyjuice_b200.decoding import HMMDecoder, beam_search
    decoder = HMMDecoder(hmm(64, 700)[0])
    g = torch.Generator().manual_seed(0)
    prompts = torch.randint(700, (5, 3), generator=g).cuda()
    for _ in range(2):
        beam_search(decoder, prompts, 4, 6, eos_id=eos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = beam_search(decoder, prompts, 4, 6, eos_id=eos)
    for _ in range(3):
        prompts.copy_(torch.randint(-1, 700, (5, 3), generator=g))
        graph.replay()
        got = [t.clone() for t in held]
        for a, b in zip(got, beam_search(decoder, prompts, 4, 6, eos_id=eos)):
            assert torch.equal(a, b)


def test_tables_of_more_nodes_than_are_addressed_are_refused():
    teacher = lambda T: lm.TopLogits(torch.zeros(2, T, 1, dtype=torch.int64), torch.zeros(2, T, 1))
    for shape, T in (((2 ** 30 - 3, 1), 1), ((1, 2 ** 30, 1), 1), ((2 ** 30 - 4, 1), 3), ((2, 2 ** 30 - 4, 1), 2)):
        fits = T * shape[-2] < 2 ** 31 and shape[-2] <= 2 ** 30 - 4
        with pytest.raises(NotImplementedError if fits else ValueError):
            lm.expected_log_probs(torch.zeros(1, 1).expand(shape), teacher(T))


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("T,M,C,B,K", [(2, 6, 200000, 2600, 2), (2, 40, 200000, 3000, 2), (3, 70, 900, 500, 4), (2, 300, 64, 700, 3), (1, 3, 5, 50, 2)])
def test_a_category_that_has_half_of_all_slots(T, M, C, B, K, tied):
    """Both forms of the backward pass: only categories that occur (few slots in large tables), tiles of categories."""
    g = torch.Generator().manual_seed(T + C)
    ids = torch.randint(C, (B, T, K), generator=g)
    ids[torch.rand(B, T, K, generator=g) < 0.5] = C // 3
    lp = torch.randn(*((M, C) if tied else (T, M, C)), generator=g).cuda().requires_grad_()
    out = lm.expected_log_probs(lp, lm.TopLogits(ids.cuda(), torch.zeros(B, T, K, device="cuda")))
    # (weights 1 / K; sums of small whole numbers over it: K a power of two or not, every sum is off by its terms' roundings at most)
    flow = torch.randint(0, 3, out.shape, generator=g).float().cuda()
    grad, = torch.autograd.grad(out, lp, flow)
    want = torch.zeros(T, C, M, dtype=torch.float64)
    q = float(torch.tensor(1.0) / K)
    for t in range(T):
        for k in range(K):
            want[t].index_add_(0, ids[:, t, k], flow[t].t().double().cpu() * q)
    want = want.sum(0).t() if tied else want.transpose(1, 2)
    terms = B * K * (T if tied else 1)
    assert bool(((grad.double().cpu() - want).abs() <= (terms * STEP) * want).all())
