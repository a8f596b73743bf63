"""Selection over a vocabulary (`lm.top_logits`, `lm.beam_select`) and `lm.reorder` against their definitions in 64 bits, at the
sizes, strides and masks where they can go wrong."""
import math

import pytest
import torch

from pyjuice_b200 import lm

NEG_INF, NAN, INF = float("-inf"), float("nan"), float("inf")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# A log-normaliser: sums of up to 2^17 rounded exponentials of 2 units in the last place, in fp32 partial sums of 16 * 32 terms
# a thread (each off by half a step of the partial sum), a final rounding to fp32 of a value of magnitude up to 64
NORM_TOL = (2 + 512 / 2) * 2.0 ** -23 + 64 * 2.0 ** -24


def _norm(x64):
    """log sum exp over the last dimension; NaN counts nothing."""
    return torch.logsumexp(torch.where(x64.isnan(), torch.full_like(x64, NEG_INF), x64), -1)


def _top(x, k):
    """(ids, values) of the definition, row by row."""
    x = x.double().cpu()
    ids, values = [], []
    for row in x.reshape(-1, x.size(-1)).tolist():
        order = sorted((v for v in range(len(row)) if row[v] > NEG_INF), key=lambda v: (-row[v], v))[:k]
        ids.append(order + [-1] * (k - len(order)))
        values.append([row[v] for v in order] + [NEG_INF] * (k - len(order)))
    lead = x.shape[:-1]
    return torch.tensor(ids).view(*lead, k), torch.tensor(values, dtype=torch.float64).view(*lead, k)


def _check_top(x, k, temperature=1.0):
    got = lm.top_logits(x, k, temperature)
    ids, values = _top(x, k)
    assert got.ids.dtype == torch.int64 and got.logits.dtype == x.dtype and got.log_norm.dtype == torch.float32
    assert got.ids.shape == got.logits.shape == ids.shape and got.log_norm.shape == x.shape[:-1]
    assert torch.equal(got.ids.cpu(), ids)
    assert torch.equal(got.logits.double().cpu(), values)
    norm = _norm(x.double().cpu() / temperature)
    torch.testing.assert_close(got.log_norm.double().cpu(), norm, rtol=0, atol=NORM_TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (1, 31, 8), (5, 128, 128), (2, 4096, 1), (7, 4097, 33),
                                          (1, 50257, 100), (700, 1000, 17), (1300, 513, 128), (3, 131071, 128)])
def test_top_logits(rows, vocab, k, dtype):
    g = torch.Generator().manual_seed(rows * vocab + k)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).cuda()
    _check_top(x, k, 0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["constant", "rising", "falling", "steps", "two", "zeros", "lowest"])
@pytest.mark.parametrize("vocab", [300, 9000, 20011])
def test_top_logits_of_ordered_and_equal_values(kind, vocab):
    at = torch.arange(vocab, dtype=torch.float32)
    x = {"constant": torch.full((vocab,), -3.5), "rising": at / 64, "falling": -at / 64, "steps": (at % 7) // 1,
         "two": (at % 2), "zeros": torch.where(at % 2 == 0, -0.0, 0.0),
         "lowest": torch.full((vocab,), torch.finfo(torch.float32).min)}[kind]
    got = lm.top_logits(x.cuda(), 40)
    ids, values = _top(x.unsqueeze(0), 40)
    assert torch.equal(got.ids.cpu(), ids[0]) and torch.equal(got.logits.double().cpu(), values[0])
    if kind == "lowest":
        assert abs(float(got.log_norm) / torch.finfo(torch.float32).min - 1) < 2 ** -23
    else:
        torch.testing.assert_close(float(got.log_norm), float(_norm(x.double())), rtol=2 ** -22, atol=NORM_TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_places_nan_and_infinities(dtype):
    x = torch.randn(8, 6000, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[0] = NEG_INF
    x[1] = NAN
    x[2, 5:] = NEG_INF
    x[3, ::2] = NAN
    x[4, 17], x[4, 4500] = INF, INF
    x[5, 3:] = NAN
    x[5, 0] = NEG_INF
    x[6] = torch.finfo(dtype).min
    x = x.cuda()
    got = lm.top_logits(x, 9)
    ids, values = _top(x, 9)
    assert torch.equal(got.ids.cpu(), ids) and torch.equal(got.logits.double().cpu(), values)
    norm = _norm(x.double().cpu())
    assert float(got.log_norm[0]) == NEG_INF == float(got.log_norm[1]) and float(got.log_norm[4]) == INF
    torch.testing.assert_close(got.log_norm.double().cpu(), norm, rtol=2 ** -22, atol=NORM_TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    base = torch.randn(9, 5003, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    for start in range(1, 8):
        _check_top(base[:, start:start + 4990], 20)
    _check_top(base.t()[:5000].t(), 5)                          # rows with a stride
    _check_top(base[:, ::3], 7)                                 # elements apart
    _check_top(base.t().contiguous().t(), 7)                    # columns first
    _check_top(base[:8].view(2, 4, 5003)[:, 1:3], 6)            # leading dimensions that are no one dimension
    _check_top(base[:1].expand(4, 5003), 3)
    _check_top(base[0], 3)


@pytest.mark.gpu
def test_no_rows():
    got = lm.top_logits(torch.empty(0, 7, 30, device="cuda"), 4)
    assert got.ids.shape == (0, 7, 4) and got.log_norm.shape == (0, 7)
    out = lm.beam_select(torch.empty(0, 2, 30, device="cuda"), torch.empty(0, 2, device="cuda"), 4)
    assert [t.shape for t in out] == [(0, 4)] * 3
    assert lm.reorder(torch.empty(0, 3, dtype=torch.int64, device="cuda"), torch.empty(0, 5, device="cuda"))[0].shape == (0, 5)


def _beam(x, scores, n, finished, pad, normalize):
    """The definition: all continuations of a sequence in 64 bits, sorted by (-score, place)."""
    x, scores = x.double().cpu(), scores.double().cpu()
    B, K, V = x.shape
    out = []
    for b in range(B):
        found = []
        for k in range(K):
            s = float(scores[b, k])
            if not s > NEG_INF:
                continue
            if finished is not None and bool(finished[b, k]):
                found.append((-s, k * V + pad))
                continue
            norm = float(_norm(x[b, k])) if normalize else 0.0
            total = s + x[b, k] - norm
            for v in torch.nonzero((total > NEG_INF) & (x[b, k] > NEG_INF)).flatten().tolist():
                found.append((-float(total[v]), k * V + v))
        found = sorted(found)[:n]
        out.append([(-s, p // V, p % V) for s, p in found] + [(NEG_INF, 0, -1)] * (n - len(found)))
    return torch.tensor(out, dtype=torch.float64)


def _check_beam(x, scores, n, finished=None, pad=0, normalize=True):
    got = lm.beam_select(x, scores, n, finished, pad, normalize)
    want = _beam(x, scores, n, finished, pad, normalize)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int64
    assert torch.equal(got[1].cpu(), want[..., 1].long()) and torch.equal(got[2].cpu(), want[..., 2].long())
    # the normaliser's error, and the rounding of the score
    torch.testing.assert_close(got[0].double().cpu(), want[..., 0], rtol=2.0 ** -24, atol=NORM_TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 4, 50257, 8), (3, 5, 33, 128), (2, 128, 40, 128), (200, 3, 257, 6),
                                     (4, 16, 5000, 32), (2, 32, 9001, 64)])
def test_beam_select(B, K, V, n, normalize, dtype):
    g = torch.Generator().manual_seed(B + 10 * K + V)
    x = (torch.randn(B, K, V, generator=g) * 3).to(dtype).cuda()
    scores = (torch.rand(B, K, generator=g) * -4 - 20).cuda()
    finished = (torch.rand(B, K, generator=g) < 0.2).cuda()
    _check_beam(x, scores, n, None, 0, normalize)
    _check_beam(x, scores, n, finished, V - 1, normalize)


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [True, False])
def test_beams_that_are_dead_finished_masked_or_equal(normalize):
    x = torch.randn(9, 4, 4500, generator=torch.Generator().manual_seed(5))
    scores = torch.full((9, 4), -3.0)
    finished = torch.zeros(9, 4, dtype=torch.bool)
    scores[0, 1:] = NEG_INF                       # the first step: one live beam
    scores[1] = NEG_INF                           # nothing lives
    scores[2, 0], scores[2, 3] = NAN, NEG_INF
    x[3] = NEG_INF                                # nothing may be said
    finished[4] = True                            # all finished
    x[4] = NAN
    finished[5, 2], scores[5, 2] = True, NEG_INF
    x[6] = x[6, :1]                               # equal rows at equal scores: a lower beam first
    x[7] = 0.0                                    # everything equal
    x[8, 1] = NAN
    x[8, 2, 7:] = NEG_INF
    x[8, 3, ::3] = NAN
    _check_beam(x.cuda(), scores.cuda(), 16, finished.cuda(), 11, normalize)


@pytest.mark.gpu
def test_a_row_of_plus_infinity_has_no_normaliser():
    x = torch.zeros(1, 2, 10)
    x[0, 0, 4] = INF
    s, p, t = lm.beam_select(x.cuda(), torch.zeros(1, 2).cuda(), 3)
    assert p.tolist() == [[1, 1, 1]] and t.tolist() == [[0, 1, 2]]
    s, p, t = lm.beam_select(x.cuda(), torch.zeros(1, 2).cuda(), 3, normalize=False)
    assert p.tolist() == [[0, 0, 0]] and t.tolist() == [[4, 0, 1]] and float(s[0, 0]) == INF


@pytest.mark.gpu
def test_beam_strides():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 4, 3001, generator=g).cuda()
    scores = torch.randn(4, 6, generator=g).cuda().t()
    _check_beam(x, scores, 9)
    _check_beam(x[::2, 1:], scores[::2, 1:], 9)
    _check_beam(x.permute(2, 0, 1).contiguous().permute(1, 2, 0), scores, 9)
    _check_beam(x[..., 1:3000].to(torch.bfloat16)[..., 3:], scores, 9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int64, torch.bool, torch.uint8, torch.float64])
@pytest.mark.parametrize("shape,dim", [((12, 5), 0), ((12,), 0), ((7, 12), 1), ((3, 12, 8), 1), ((12, 2, 33), -3), ((5, 2, 12, 1), 2),
                                       ((12, 0), 0), ((1, 12, 4096), 1)])
def test_reorder(shape, dim, dtype):
    g = torch.Generator().manual_seed(4)
    x = torch.randint(0, 2 if dtype == torch.bool else 100, shape, generator=g).to(dtype).cuda()
    for n, ids in ((1, torch.int32), (4, torch.int64), (9, torch.int64)):
        parents = torch.randint(0, 4, (3, n), generator=g).to(ids).cuda()
        at = (parents.long() + 4 * torch.arange(3, device="cuda")[:, None]).flatten()
        got, = lm.reorder(parents, x, dim=dim)
        assert got.is_contiguous() and torch.equal(got, x.index_select(dim, at))


@pytest.mark.gpu
def test_reorder_of_many_states_with_strides_and_bad_parents():
    g = torch.Generator().manual_seed(6)
    base = torch.randn(8, 6, 30, generator=g).cuda()
    states = [base, base[..., 1:], base[:, ::2], base.transpose(1, 2), base[:, :, 3], base[:, 0, :], base.half(), base[1:7].double()[[0, 1, 2, 3, 4, 5, 0, 1]],
              base.transpose(0, 1).contiguous().transpose(0, 1), (base > 0), base[:, :1].expand(8, 9, 30)]
    parents = torch.tensor([[3, 1, -1, 4], [0, 0, 2 ** 40, 3]]).cuda()
    ok = ((parents >= 0) & (parents < 4)).flatten()
    at = (parents.clamp(0, 3) + 4 * torch.arange(2, device="cuda")[:, None]).flatten()
    for x, got in zip(states, lm.reorder(parents, *states)):
        want = x.index_select(0, at)
        want[~ok] = 0
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_a_captured_step_replays_on_new_values():
    """Selection and reordering captured into a graph, replayed on other inputs, beside a second graph of other sizes."""
    def step(x, s, state):
        sc, p, t = lm.beam_select(x, s, 4)
        return (sc, p, t, *lm.reorder(p, state))

    def inputs(seed, V):
        g = torch.Generator().manual_seed(seed)
        return [torch.randn(*shape, generator=g).cuda() for shape in ((3, 4, V), (3, 4), (12, 50))]

    graphs = []
    for V in (9000, 700):
        held = inputs(0, V)
        step(*held)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*held)
        graphs.append((V, held, graph, out))
    for seed in (1, 2):
        for V, held, graph, out in graphs:
            for a, b in zip(held, inputs(seed, V)):
                a.copy_(b)
        for _, _, graph, _ in graphs:
            graph.replay()
        for _, held, _, out in graphs:
            for a, b in zip(out, step(*held)):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    x = torch.randn(2, 64, 30000, generator=torch.Generator().manual_seed(8)).cuda()
    want = [lm.top_logits(v, 50) for v in x]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(lm.top_logits(x[i], 50))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert torch.equal(r.ids, want[i].ids) and torch.equal(r.log_norm, want[i].log_norm)


def test_refusals():
    x = torch.randn(2, 3, 10)
    for bad in (0, 11, 129):
        with pytest.raises(ValueError):
            lm.top_logits(x, bad)
    with pytest.raises(ValueError):
        lm.top_logits(torch.empty(3, 0), 1)
    with pytest.raises(TypeError):
        lm.top_logits(x.double(), 2)
    for t in (0.0, -1.0, NAN, INF):
        with pytest.raises(ValueError):
            lm.top_logits(x, 2, temperature=t)
    with pytest.raises(NotImplementedError):
        lm.top_logits(x, 2)
    s = torch.zeros(2, 3)
    for args in ((x[0], s), (x, s[:1]), (x, s.double()), (x, s, 0), (x, s, 31), (x, s, 4, s > 0, 10), (x, s, 4, s > 0, -1), (x, s, 4, s),
                 (x, s, 4, (s > 0)[:1]), (torch.empty(1, 129, 2), torch.empty(1, 129))):
        with pytest.raises(ValueError):
            lm.beam_select(*args)
    with pytest.raises(TypeError):
        lm.beam_select(x.long(), s)
    with pytest.raises(NotImplementedError):
        lm.beam_select(x, s)
    parents = torch.zeros(2, 3, dtype=torch.int64)
    for args, dim in (((parents[0], s), 0), ((parents.float(), s), 0), ((parents, torch.zeros(5, 2)), 0), ((parents, s, torch.zeros(4, 2)), 0),
                      ((parents, s), 2), ((parents, torch.zeros(())), 0), ((parents, torch.zeros(2, 3, requires_grad=True)), 0),
                      ((parents, torch.zeros(0, 3)), 0)):
        with pytest.raises(ValueError):
            lm.reorder(*args, dim=dim)
    with pytest.raises(TypeError):
        lm.reorder(parents, s.to(torch.complex64))
    with pytest.raises(NotImplementedError):
        lm.reorder(parents, s)
