"""Decoding of HMM circuits: next-token distributions and beam search against the same in 64 bits on the host."""
import math

import pytest
import torch

import pyjuice_b200 as pj
from pyjuice_b200.decoding import HMMDecoder, beam_search

NEG_INF = float("-inf")
# Three products of 8-bit-mantissa halves per factor (2^-16 each way) and fp32 sums over the states, per token
TOL = 2.0 ** -13


def hmm(latents, vocab, length, seed=0, **kwargs):
    g = torch.Generator().manual_seed(seed)
    p = lambda *s: torch.rand(*s, generator=g).pow(3).add_(1e-4)
    alpha, beta, gamma = p(latents, latents), p(latents, vocab), p(latents)
    alpha, beta, gamma = alpha / alpha.sum(1, keepdim=True), beta / beta.sum(1, keepdim=True), gamma / gamma.sum()
    torch.manual_seed(seed)
    ns = pj.structures.HMM(seq_length=length, num_latents=latents, num_emits=vocab, alpha=alpha, beta=beta, gamma=gamma, **kwargs)
    pc = pj.compile(ns, verbose=False).to("cuda:0")
    return pc, (alpha.double(), beta.double(), gamma.double())


def next_log_probs(model, tokens):
    """[vocab] after a list of tokens, in 64 bits."""
    alpha, beta, z = model
    for t in tokens:
        z = z * beta[:, t]
        z = (z / z.sum()) @ alpha
    return (z @ beta).log()


def search(model, prompt, steps, K, eos=None):
    """Beam search on the host: [(score, tokens)], best first, a lower (beam, token) first among equals."""
    beams = [(0.0, [], False)]
    for _ in range(steps):
        found = []
        for k, (score, said, done) in enumerate(beams):
            if done:
                found.append((-score, k, eos))
                continue
            lp = next_log_probs(model, prompt + said)
            lp = lp - lp.logsumexp(0)
            found += [(-(score + float(v)), k, t) for t, v in enumerate(lp.tolist())]
        found = sorted(found)[:K]
        beams = [(-s, beams[k][1] + [t], t == eos if eos is not None else False) for s, k, t in found]
    return beams


@pytest.mark.gpu
@pytest.mark.parametrize("latents,vocab,length", [(16, 9, 6), (20, 33, 2), (128, 1000, 4), (256, 130, 5), (3, 5, 3)])
def test_next_token_distributions(latents, vocab, length):
    pc, model = hmm(latents, vocab, length)
    decoder = HMMDecoder(pc)
    x = torch.randint(vocab, (5, 7), generator=torch.Generator().manual_seed(1))
    state = decoder.start(5)
    for t in range(7):
        got = decoder.log_probs(state)
        assert got.shape == (5, vocab)
        want = torch.stack([next_log_probs(model, row[:t].tolist()) for row in x])
        assert float((got.double().cpu() - want).abs().max()) < (t + 1) * TOL
        said = x[:, t].cuda()
        state = decoder.advance(state, said, got.gather(1, said[:, None])[:, 0])
        assert float(state.exp().sum(0).sub(1).abs().max()) < (t + 2) * TOL


@pytest.mark.gpu
def test_sentences_score_as_in_the_circuit():
    """The tokens' log-probabilities add up to the circuit's log-likelihood of the sentence; beams are such sentences."""
    pc, _ = hmm(64, 50, 8)
    tokens, scores = beam_search(pc, None, num_tokens=8, num_beams=6, batch=2)
    assert tokens.shape == (2, 6, 8) and torch.equal(tokens[0], tokens[1]) and bool((scores[:, :-1] >= scores[:, 1:]).all())
    lls = pc(tokens[0]).detach()[:, 0]
    assert float((lls - scores[0]).abs().max()) < 8 * TOL + 1e-3
    prompts = torch.randint(50, (3, 5), generator=torch.Generator().manual_seed(2)).cuda()
    tokens, scores = beam_search(pc, prompts, num_tokens=3, num_beams=4)
    decoder = HMMDecoder(pc)
    state, before = decoder.start(3), torch.zeros(3, device="cuda")
    for t in range(5):
        lp = decoder.log_probs(state).gather(1, prompts[:, t:t + 1])[:, 0]
        before, state = before + lp, decoder.advance(state, prompts[:, t], lp)
    whole = torch.cat([prompts[:, None].expand(-1, 4, -1), tokens], 2).reshape(12, 8)
    assert float((pc(whole).detach()[:, 0].view(3, 4) - before[:, None] - scores).abs().max()) < 8 * TOL + 1e-3


@pytest.mark.gpu
@pytest.mark.parametrize("eos", [None, 3])
@pytest.mark.parametrize("latents,vocab,K,steps", [(16, 9, 4, 5), (16, 9, 1, 6), (20, 33, 40, 3), (128, 300, 8, 4), (4, 2, 8, 5)])
def test_beam_search(latents, vocab, K, steps, eos):
    eos = None if eos is None else min(eos, vocab - 1)
    pc, model = hmm(latents, vocab, 4, seed=3)
    prompts = torch.randint(vocab, (3, 2), generator=torch.Generator().manual_seed(2))
    tokens, scores = beam_search(pc, prompts, steps, K, eos_id=eos)
    for b in range(3):
        want = search(model, prompts[b].tolist(), steps, K, eos)
        n = len(want)
        assert bool((scores[b, n:] == NEG_INF).all()) and bool((tokens[b, n:] == -1).all())
        for k in range(n):
            assert abs(float(scores[b, k]) - want[k][0]) < (steps + 2) * TOL
        # beams whose scores are apart are the same beams
        for k in range(n):
            apart = all(abs(want[k][0] - want[j][0]) > 4 * (steps + 2) * TOL for j in range(n) if j != k)
            if apart and k < n - 1:
                assert tokens[b, k].tolist() == want[k][1]


@pytest.mark.gpu
def test_a_decoder_keeps_its_parameters_until_it_reloads():
    pc, _ = hmm(16, 20, 5)
    decoder = HMMDecoder(pc)
    before = decoder.log_probs(decoder.start(2))
    opt = pj.optim.MiniBatchEM(pc, step_size=0.5, pseudocount=0.1)
    pc(torch.randint(20, (30, 5), device="cuda")).mean().backward()
    opt.step()
    assert torch.equal(decoder.log_probs(decoder.start(2)), before)
    decoder.reload()
    after = decoder.log_probs(decoder.start(2))
    assert float((after - before).abs().max()) > 1e-3
    assert torch.equal(after, HMMDecoder(pc).log_probs(decoder.start(2)))


@pytest.mark.gpu
def test_a_teacher_learned_and_answered():
    """The operators as they are used: a teacher's top logits train a circuit, which then continues a prompt."""
    pc, _ = hmm(32, 60, 6)
    g = torch.Generator().manual_seed(0)
    teacher = pj.lm.top_logits((torch.randn(40, 6, 60, generator=g) * 2).cuda(), 8, temperature=1.5)
    opt = pj.optim.MiniBatchEM(pc, step_size=0.3, pseudocount=0.1)
    first = None
    for _ in range(5):
        lls = pc(teacher)
        lls.mean().backward()
        opt.step()
    tokens, scores = beam_search(pc, torch.randint(60, (2, 3), generator=g), 4, 5, eos_id=0)
    assert tokens.shape == (2, 5, 4) and bool(scores.isfinite().all()) and bool(((tokens >= 0) & (tokens < 60)).all())


@pytest.mark.gpu
def test_other_circuits_and_arguments_are_refused():
    torch.manual_seed(0)
    for ns in (pj.structures.HMM(seq_length=4, num_latents=8, num_emits=5, homogeneous=False), pj.structures.HMM(seq_length=1, num_latents=8, num_emits=5),
               pj.structures.RAT_SPN(num_vars=8, num_latents=4, depth=2, num_repetitions=2, num_cats=3)):
        ns.init_parameters()
        with pytest.raises(ValueError):
            HMMDecoder(pj.compile(ns, verbose=False).to("cuda:0"))
    pc, _ = hmm(8, 6, 3)
    decoder = HMMDecoder(pc)
    for kwargs in (dict(num_tokens=0), dict(num_beams=0), dict(num_beams=129), dict(eos_id=6), dict(eos_id=-1),
                   dict(prompts=torch.zeros(3)), dict(prompts=torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(ValueError):
            beam_search(decoder, **kwargs)
    for state in (torch.zeros(8, 2), torch.zeros(7, 2, device="cuda"), torch.zeros(8, 2, device="cuda").double(), torch.zeros(8, device="cuda")):
        with pytest.raises(ValueError):
            decoder.log_probs(state)
    with pytest.raises(ValueError):
        decoder.advance(decoder.start(2), torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert decoder.log_probs(decoder.start(0)).shape == (0, 6)


def test_a_circuit_on_the_host_is_refused():
    torch.manual_seed(0)
    pc = pj.compile(pj.structures.HMM(seq_length=3, num_latents=4, num_emits=5), verbose=False)
    with pytest.raises(NotImplementedError):
        HMMDecoder(pc)
