"""Leaf tables under a teacher's top logits (`lm.expected_log_probs`): values and gradients against the definition in 64 bits."""
import ctypes

import pytest
import torch

from pyjuice_b200 import _lib, lm

NEG_INF, NAN, INF = float("-inf"), float("nan"), float("inf")
STEP = 2.0 ** -24                    # half a step of fp32, relative


def weights(teacher):
    """The definition of the slots' weights, in 64 bits: [B, T, K]; empty slots 0."""
    ids, x = teacher.ids.cpu().long(), teacher.logits.detach().double().cpu()
    empty = (ids < 0) | ~(x > NEG_INF)
    z = torch.where(empty, torch.full_like(x, NEG_INF), x)
    top = z.amax(-1, keepdim=True) if z.size(-1) else z.new_zeros(*z.shape[:-1], 1)
    d = torch.where(z == top, torch.zeros_like(z), (z - torch.where(top == NEG_INF, torch.zeros_like(top), top)) / teacher.temperature)
    e = torch.where(empty, torch.zeros_like(z), d.exp())
    q = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    if teacher.log_norm is not None:
        norm = teacher.log_norm.double().cpu().unsqueeze(-1)
        q = torch.where(norm.isfinite(), torch.where(empty, torch.zeros_like(z), (z / teacher.temperature - norm).exp()), q)
    return q


# How far the exponents of the weights reach below 0 where the weights matter to fp32 (each exponent is rounded twice)
SPREAD = 110


def expected(log_probs, teacher):
    """Values [T, M, B] in 64 bits and the sum of the magnitudes that make them."""
    q, ids = weights(teacher), teacher.ids.cpu().long()
    lp = log_probs.detach().double().cpu()
    B, T, K = ids.shape
    M, C = lp.shape[-2:]
    values, size = torch.zeros(T, M, B, dtype=torch.float64), torch.zeros(T, M, B, dtype=torch.float64)
    for t in range(T):
        table = lp if lp.dim() == 2 else lp[t]
        table = torch.cat([table, torch.full((M, 1), NEG_INF, dtype=torch.float64)], 1)
        picked = table[:, ids[:, t].clamp(0, C)]                                            # [M, B, K]
        part = torch.where(q[:, t] > 2.0 ** -150, q[:, t] * picked, torch.zeros_like(picked))
        values[t], size[t] = part.sum(-1), part.abs().sum(-1)
    return values, size


def gradient(shape, teacher, g):
    """The gradient in 64 bits, the sum of the magnitudes that make it, and the number of its terms."""
    q, ids = weights(teacher), teacher.ids.cpu().long()
    B, T, K = ids.shape
    M, C = shape[-2:]
    out = [torch.zeros(T, C, M, dtype=torch.float64) for _ in range(3)]
    ok = (ids >= 0) & (ids < C) & (q > 0)
    for t in range(T):
        b, k = ok[:, t].nonzero(as_tuple=True)
        c = ids[b, t, k]
        part = q[b, t, k, None] * g[t].double().cpu().t()[b]
        for o, v in zip(out, (part, part.abs(), torch.ones_like(part))):
            o[t].index_add_(0, c, v)
    out = [o.transpose(1, 2) for o in out]
    return [o.sum(0) for o in out] if len(shape) == 2 else out


def check(log_probs, teacher, seed=0):
    B, T, K = teacher.ids.shape
    lp = log_probs.detach().clone().requires_grad_()
    got = lm.expected_log_probs(lp, teacher)
    want, size = expected(lp, teacher)
    assert got.shape == want.shape and got.dtype == torch.float32
    # K products and sums; of a weight: an exponential (two steps, and its argument rounded twice), a sum over the slots, a quotient
    terms = K + 12 + 2 * SPREAD
    ours = got.detach().double().cpu()
    finite = want.isfinite()
    assert torch.equal(finite, ours.isfinite()) and torch.equal(want[~finite], ours[~finite])
    # 2^-149: weights below the smallest fp32 number are 0
    assert bool(((ours - want).abs()[finite] <= (terms * 2 * STEP * size + 1e-40)[finite]).all())
    g = torch.randn(got.shape, generator=torch.Generator().manual_seed(seed)).cuda()
    grad, = torch.autograd.grad(got, lp, g)
    want, size, n = gradient(lp.shape, teacher, g)
    assert grad.shape == lp.shape and grad.dtype == torch.float32
    assert bool(((grad.double().cpu() - want).abs() <= (n + terms) * 2 * STEP * size + 1e-38).all())
    assert bool((grad.cpu()[n == 0] == 0).all())
    again = lm.expected_log_probs(lp, teacher)
    assert torch.equal(torch.autograd.grad(again, lp, g)[0], grad)                          # the same bits on every call
    return got


def make(T, M, C, B, K, tied, seed=0, ids=torch.int64, dtype=torch.float32, temperature=1.0, zipf=False):
    g = torch.Generator().manual_seed(seed + T * M + C)
    lp = (torch.randn(*((M, C) if tied else (T, M, C)), generator=g) * 2).log_softmax(-1)
    u = torch.rand(B, T, K, generator=g)
    x = ((C + 1.0) ** u - 1).long().clamp(0, C - 1) if zipf else (u * C).long().clamp(0, C - 1)
    x[torch.rand(B, T, K, generator=g) < 0.1] = -1
    x[torch.rand(B, T, generator=g) < 0.2] = -1
    logits = (torch.randn(B, T, K, generator=g) * 3).to(dtype)
    return lp.cuda(), lm.TopLogits(x.to(ids).cuda(), logits.cuda(), temperature)


# (forms of the forward pass: tables in place, in shared memory, turned; of the sort: one CTA a set, radix of 1 to 3 passes; of
# the backward pass: by categories that occur, by tiles of categories)
SIZES = [(1, 1, 1, 1, 1), (1, 1, 2, 1, 3), (3, 5, 7, 2, 4), (2, 128, 256, 33, 16), (5, 33, 100, 31, 9), (4, 130, 64, 40, 8), (7, 64, 31, 1, 1),
         (2, 16, 1600, 70, 12), (3, 9, 20000, 5, 10), (40, 1, 500, 3, 12), (2, 257, 1000, 65, 40), (1, 3, 200000, 2, 7), (2, 6, 70001, 90, 33),
         (2, 3, 400, 3, 300), (3, 2, 50, 2, 60), (8, 40, 600, 200, 4), (9, 300, 601, 200, 4), (8, 5, 70, 300, 3), (3, 70, 40, 500, 5),
         (3, 8, 1023, 160, 10), (3, 8, 1024, 160, 10)]      # the most categories of a sort in one pass, the fewest in two


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("size", SIZES)
def test_values_and_gradients(size, tied):
    check(*make(*size, tied, zipf=size[2] > 500))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_types_and_temperatures(ids, dtype):
    for temperature in (0.5, 2.0):
        check(*make(3, 20, 50, 9, 6, True, ids=ids, dtype=dtype, temperature=temperature))


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [True, False])
def test_masked_slots_infinities_and_repeated_ids(tied):
    T, M, C, B, K = 3, 37, 45, 8, 5
    lp, teacher = make(T, M, C, B, K, tied, seed=3)
    ids, x = teacher.ids.clamp_min(0), teacher.logits.clone()
    x[0, 0] = NEG_INF                                    # nothing left
    x[1, 0, 1:] = NAN
    ids[2, 0] = -7
    x[2, 0] = INF
    x[3, 0, 2], x[3, 0, 4] = INF, INF                    # share the weight
    x[4, 0] = torch.finfo(torch.float32).min             # the lowest value is a value
    ids[5, 0] = 4                                        # one category in every slot
    x[6, 0], x[6, 0, 0] = -1e30, 1e30                    # weights of zero ...
    ids[6, 0] = torch.arange(5) + 10
    with torch.no_grad():
        lp[..., 11], lp[..., 12] = NEG_INF, NEG_INF      # ... take nothing of -inf
        lp[..., 5, 4] = NEG_INF
    ids[7, 0, 1] = C                                     # no such category: -inf, and no gradient
    ids[7, 1, 0] = 2 ** 40
    x[7, 1, 0] = NEG_INF
    ids[7, 2, 0] = 2 ** 40
    got = check(lp, lm.TopLogits(ids, x))
    assert bool((got[0, :, 0] == 0).all()) and bool((got[0, :, 2] == 0).all())
    assert bool(got[0, :, 6].isfinite().all()) and bool((got[0, :, 7] == NEG_INF).all()) and bool((got[2, :, 7] == NEG_INF).all())


@pytest.mark.gpu
def test_given_normalisers():
    x = torch.randn(6, 4, 300, generator=torch.Generator().manual_seed(5)).cuda() * 2
    for temperature in (1.0, 3.0):
        top = lm.top_logits(x, 20, temperature)
        lp = (torch.randn(11, 300, generator=torch.Generator().manual_seed(6)) * 2).log_softmax(-1).cuda()
        check(lp, top)
        mass = weights(top).sum(-1)
        assert bool((mass < 1).all()) and bool((mass > 0.05).all())
        check(lp, top._replace(log_norm=torch.full_like(top.log_norm, INF)))        # not finite: the slots sum to one
        # all of the vocabulary kept: the teacher's whole distribution
        whole = lm.top_logits(x[..., :100], 100, temperature)
        a = lm.expected_log_probs(lp, whole)
        b = torch.einsum("btv,mv->tmb", (x[..., :100].double() / temperature).softmax(-1), lp[:, :100].double())
        assert float((a - b).abs().max()) < 300 * 20 * STEP


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [True, False])
def test_strides_and_slices(tied):
    T, M, C, B, K = 5, 21, 90, 7, 6
    lp, teacher = make(T, M, 2 * C + 1, B, K, tied)
    turned = lm.TopLogits((teacher.ids % C).permute(2, 0, 1).contiguous().permute(1, 2, 0), teacher.logits.transpose(0, 1).contiguous().transpose(0, 1))
    for table in (lp[..., 1:C + 1], lp[..., ::2][..., :C], lp.transpose(-1, -2).contiguous().transpose(-1, -2)[..., :C]):
        check(table, turned)
    one = lm.TopLogits(turned.ids[:1].expand(B, T, K), turned.logits[:, :1].expand(B, T, K))
    check(lp[..., :C], one)
    out = lm.expected_log_probs(lp.requires_grad_(), turned)                 # a gradient with strides
    g = torch.randn(B, M, T, device="cuda")
    a, = torch.autograd.grad(out, lp, g.permute(2, 1, 0), retain_graph=True)
    b, = torch.autograd.grad(out, lp, g.permute(2, 1, 0).contiguous())
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_empty_sizes():
    for shape, tied in (((0, 4, 5), True), ((2, 0, 5), True), ((2, 3, 0), True), ((2, 3, 0), False), ((2, 0, 5), False)):
        B, T, K = shape
        lp = torch.randn(*((6, 9) if tied else (T, 6, 9)), device="cuda", requires_grad=True)
        out = lm.expected_log_probs(lp, lm.TopLogits(torch.zeros(shape, dtype=torch.int64, device="cuda"), torch.zeros(shape, device="cuda")))
        assert out.shape == (T, 6, B) and bool((out == 0).all())
        out.sum().backward()
        assert bool((lp.grad == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [True, False])
def test_gradient_against_differences(tied):
    """The function is linear: a difference over any step is the gradient, but for the rounding of the values."""
    lp, teacher = make(4, 17, 40, 6, 7, tied, seed=8)
    lp = lp.requires_grad_()
    g = torch.rand(4, 17, 6, generator=torch.Generator().manual_seed(1)).cuda()
    grad, = torch.autograd.grad(lm.expected_log_probs(lp, teacher), lp, g)
    d = torch.randn(lp.shape, generator=torch.Generator().manual_seed(2)).cuda()
    up, down = (lm.expected_log_probs((lp + s * d).detach(), teacher) for s in (0.5, -0.5))
    difference = float(((up - down).double() * g.double()).sum())
    # values of up to |lp| + |d| / 2, each with K + 12 + 2 * SPREAD roundings, summed over 4 * 17 * 6 outputs with weights below 1
    tol = 408 * 2 * (19 + 220) * 2 * STEP * float(lp.detach().abs().max() + d.abs().max())
    assert abs(difference - float((grad.double() * d.double()).sum())) < tol


@pytest.mark.gpu
def test_a_second_derivative_is_refused():
    lp, teacher = make(2, 5, 9, 3, 4, True)
    lp.requires_grad_()
    g = torch.ones(2, 5, 3, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(lm.expected_log_probs(lp, teacher), lp, g, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("tied,C,B", [(True, 40, 6), (True, 2999, 20), (False, 60, 30)])
def test_captured_forward_and_backward(tied, C, B):
    """Captured after eager passes over the same leaf, replayed on other values beside more of them."""
    lp, teacher = make(5, 30, C, B, 12, tied)
    lp.requires_grad_()
    g = torch.randn(5, 30, B, device="cuda")

    def step():
        out = lm.expected_log_probs(lp, teacher)
        return out.detach(), torch.autograd.grad(out, lp, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    _, other = make(5, 30, C, B, 12, tied, seed=9)
    teacher.ids.copy_(other.ids)
    teacher.logits.copy_(other.logits)
    eager = lm.expected_log_probs(lp, teacher)
    graph.replay()
    for a, b in zip(held, step()):
        assert torch.equal(a, b)
    eager.sum().backward()
    graph.replay()
    for a, b in zip(held, step()):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("form", [0, 1, 2, 3])
@pytest.mark.parametrize("tied", [True, False])
def test_forms_of_the_forward_pass_agree(form, tied):
    """Every form through the library, at one size that all of them take."""
    T, M, C, B, K = 3, 36, 50, 37, 9
    lp, teacher = make(T, M, C, B, K, tied)
    entries = lm._prepare(teacher, B)
    geo = lm._Geo(flow_cols=T * M, positions=T, nodes=M, cats=C, tied=int(tied), n_segs=T, n_groups=1 if tied else T,
                  n_sets=1 if tied else T, max_vars=T if tied else 1, total_vars=T, width=B, slots=K)
    table, stride = lp, 0
    if form in (1, 3):
        rows, stride = lp.numel() // C, lp.numel() // C
        for take_log, source in ((0, lp), (1, lp.exp())):
            table = torch.full((C, stride), NAN, device="cuda")
            _lib.call("pcx_teacher_turn", table, source, rows, C, stride, take_log)
            assert float((table - lp.reshape(-1, C).t()).abs().max()) <= take_log * 4 * STEP * float(lp.abs().max()) * 8
    out = torch.full((T, M, B), NAN, device="cuda")
    _lib.call("pcx_teacher_fwd", out, table, entries, ctypes.addressof(geo), form, stride, 0)
    want, size = expected(lp, teacher)
    assert bool(((out.double().cpu() - want).abs() <= (K + 232) * 2 * STEP * size + 1e-40).all())


def test_refusals():
    lp = torch.zeros(4, 9)
    ids, x = torch.zeros(2, 3, 5, dtype=torch.int64), torch.zeros(2, 3, 5)
    T = lm.TopLogits
    for teacher in (T(ids.float(), x), T(ids.short(), x), T(ids, x.double()), T(ids, ids)):
        with pytest.raises(TypeError):
            lm.expected_log_probs(lp, teacher)
    for teacher in (T(ids[:1], x), T(ids[0], x[0]), T(ids, x, 0.0), T(ids, x, -2.0), T(ids, x, INF), T(ids, x, NAN),
                    T(ids, x, 1.0, x), T(ids, x, 1.0, x[..., 0].double())):
        with pytest.raises(ValueError):
            lm.expected_log_probs(lp, teacher)
    for table in (lp.double(), lp[0], lp[None, None], lp.half()):
        with pytest.raises(TypeError):
            lm.expected_log_probs(table, T(ids, x))
    for table in (lp.expand(4, 4, 9), torch.zeros(3, 4, 0), torch.empty(1, 1000001)):
        with pytest.raises(ValueError):
            lm.expected_log_probs(table, T(ids, x))
    with pytest.raises(ValueError):
        lm.expected_log_probs(lp, T(ids[:1, :1, :1].expand(2 ** 15, 2 ** 5, 2 ** 10), x[:1, :1, :1].expand(2 ** 15, 2 ** 5, 2 ** 10)))
    with pytest.raises(NotImplementedError):
        lm.expected_log_probs(lp, T(ids, x))
