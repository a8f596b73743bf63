"""Compiled circuits whose leaves see a teacher's top logits: likelihoods, flows and EM steps against an autograd evaluation of
the node DAG in 64 bits."""
import random

import numpy as np
import pytest
import torch

import pyjuice_b200 as pj
from dag_autograd import collect, evaluate
from helpers import LL_ATOL, folded_input_flows, rel_close
from pyjuice_b200 import lm
from test_lm_teacher import weights

NEG_INF = float("-inf")


def hclt(latents, cats, num_vars=12):
    tree = pj.structures.random_spanning_tree(num_vars, np.random.default_rng(0))
    return pj.structures.tree_to_hidden_circuit(tree, tree.center(), num_latents=latents, num_cats=cats)


STRUCTURES = {
    "hclt": lambda: hclt(8, 5),
    "hclt-wide": lambda: hclt(128, 300, 6),
    "hmm": lambda: pj.structures.HMM(seq_length=6, num_latents=16, num_emits=9),
    "hmm-shadow": lambda: pj.structures.HMM(seq_length=7, num_latents=32, num_emits=600),
    "hmm-vocabulary": lambda: pj.structures.HMM(seq_length=5, num_latents=32, num_emits=9001),
    "hmm-untied": lambda: pj.structures.HMM(seq_length=5, num_latents=20, num_emits=33, homogeneous=False),
    "hclt-many-cats": lambda: hclt(16, 700, 5),
    "pd": lambda: pj.structures.PD((4, 4), num_latents=8, split_points=[[2], [2]], num_cats=7),
    "rat": lambda: pj.structures.RAT_SPN(num_vars=16, num_latents=8, depth=2, num_repetitions=3, num_cats=6),
}


def circuit(name):
    torch.manual_seed(4)
    random.seed(4)
    np.random.seed(4)
    ns = STRUCTURES[name]()
    ns.init_parameters()
    return ns, pj.compile(ns, verbose=False).to("cuda:0")


def cats_of(pc):
    return min(int(layer.node_cats.min()) for layer in pc.input_layer_group)


def teacher_for(pc, B, K, seed=0, temperature=1.0):
    g = torch.Generator().manual_seed(seed)
    C, V = cats_of(pc), pc.num_vars
    ids = torch.rand(B, V, C, generator=g).topk(min(K, C), dim=-1).indices
    ids[torch.rand(B, V, ids.size(-1), generator=g) < 0.1] = -1
    ids[torch.rand(B, V, generator=g) < 0.2] = -1
    return lm.TopLogits(ids.cuda(), (torch.randn(ids.shape, generator=g) * 2).cuda(), temperature)


def reference(ns, pc, teacher):
    """Log-likelihoods and the gradients of the logarithms of every leaf table, by (layer, first parameter)."""
    q, ids = weights(teacher).to(pc.device), teacher.ids.to(pc.device).long()
    tables, leaves = {}, {}
    params = [layer.params.data.double() for layer in pc.input_layer_group]
    for n in collect(ns):
        if not n.is_input():
            continue
        layer = next(i for i, l in enumerate(pc.input_layer_group) if any(m is n for m in l.nodes))
        key, C, v = (layer, n._param_range[0]), n.dist.num_cats, n.scope.to_list()[0]
        if key not in tables:
            tables[key] = params[layer][n._param_range[0]:n._param_range[1]].view(-1, C).log().requires_grad_()
        at = ids[:, v]
        picked = tables[key][:, at.clamp(0, C - 1)]
        leaves[id(n)] = torch.where(q[:, v] > 0, q[:, v] * picked, 0.0).sum(-1)
    out, _ = evaluate(pc, ns, leaves)
    out.sum().backward()
    return out.detach().cpu(), {k: t.grad.cpu() for k, t in tables.items()}


def check(ns, pc, teacher, logspace=True, flows=True):
    want, grads = reference(ns, pc, teacher)
    pc.init_param_flows(flows_memory=0.0)
    lls = pc(teacher)
    assert lls.shape == want.t().shape
    assert float((lls.detach().double().cpu() - want.t()).abs().max()) < LL_ATOL
    if not flows:
        return
    pc.backward(teacher, logspace_flows=logspace)
    for i, layer in enumerate(pc.input_layer_group):
        got = folded_input_flows(layer, layer.param_flows)
        for (at, start), grad in grads.items():
            if at == i:
                source = next(n for n in layer.nodes if n._param_range[0] == start and not n.is_tied())
                f0, f1 = source._param_flow_range
                ok, err = rel_close(got[f0:f1], grad.reshape(-1))
                assert ok, f"flows of layer {i} rel err {err}"


@pytest.mark.gpu
@pytest.mark.parametrize("logspace", [True, False])
@pytest.mark.parametrize("name", list(STRUCTURES))
def test_likelihoods_and_flows(name, logspace):
    ns, pc = circuit(name)
    for B, K, temperature in ((5, 4, 1.0), (32, 3, 2.0), (5, 1, 1.0), (64, 40, 1.0)):
        check(ns, pc, teacher_for(pc, B, K, B + K, temperature), logspace)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(STRUCTURES))
def test_a_single_slot_is_an_observed_category(name):
    _, pc = circuit(name)
    x = torch.randint(cats_of(pc), (9, pc.num_vars), generator=torch.Generator().manual_seed(1)).cuda()
    flows = []
    for inputs in (x, lm.TopLogits(x.unsqueeze(-1), torch.randn(9, pc.num_vars, 1, device="cuda"))):
        pc.init_param_flows(flows_memory=0.0)
        lls = pc(inputs)
        pc.backward(inputs)
        flows.append([lls.detach()] + [folded_input_flows(layer, layer.param_flows) for layer in pc.input_layer_group])
    assert float((flows[0][0] - flows[1][0]).abs().max()) < LL_ATOL
    for a, b in zip(flows[0][1:], flows[1][1:]):
        assert rel_close(b, a)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(STRUCTURES))
def test_variables_without_slots_are_marginalised(name):
    _, pc = circuit(name)
    ids = torch.full((3, pc.num_vars, 2), -1, device="cuda")
    pc.init_param_flows(flows_memory=0.0)
    lls = pc(lm.TopLogits(ids, torch.zeros(3, pc.num_vars, 2, device="cuda")))
    # the root of a normalised circuit: log 1, but for the rounding of sums of probabilities
    assert float(lls.detach().abs().max()) < LL_ATOL
    pc.backward()
    for layer in pc.input_layer_group:
        assert bool((layer.param_flows == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["hclt", "hmm", "hmm-shadow", "hmm-vocabulary"])
def test_em_steps_between_teachers_and_categories(name):
    """A training loop that alternates both kinds of batches, long enough for its passes to be captured and replayed."""
    ns, pc = circuit(name)
    opt = pj.optim.MiniBatchEM(pc, step_size=0.3, pseudocount=0.1)
    C = cats_of(pc)
    for step in range(7):
        teacher = teacher_for(pc, 12 if step != 4 else 9, 3, seed=step)
        want, grads = reference(ns, pc, teacher)
        before = [layer.params.data.double().cpu().clone() for layer in pc.input_layer_group]
        lls = pc(teacher)
        lls.mean().backward()
        assert float((lls.detach().double().cpu() - want.t()).abs().max()) < LL_ATOL
        opt.step()
        for (i, start), grad in grads.items():
            old = before[i][start:start + grad.numel()].view(-1, C)
            new = 0.7 * old + 0.3 * (grad + 0.1 / C) / (grad.sum(1, keepdim=True) + 0.1)
            got = pc.input_layer_group[i].params.data[start:start + grad.numel()].view(-1, C).cpu()
            ok, err = rel_close(got, new, floor=1e-4)
            assert ok, f"step {step}: parameters rel err {err}"
        x = torch.randint(C, (12, pc.num_vars), generator=torch.Generator().manual_seed(step)).cuda()
        pc(x).mean().backward()
        opt.step()
    pc.validate_tables()


@pytest.mark.gpu
def test_distillation_raises_the_objective():
    """EM on a fixed teacher never lowers its objective (the sum of the leaves' expected log-probabilities is a bound that the
    update maximises)."""
    _, pc = circuit("hmm")
    opt = pj.optim.FullBatchEM(pc)
    teacher = teacher_for(pc, 40, 4)
    last = NEG_INF
    for _ in range(6):
        lls = pc(teacher)
        lls.mean().backward()
        opt.step()
        now = float(lls.detach().double().sum())
        assert now > last - 40 * LL_ATOL
        last = now


@pytest.mark.gpu
def test_teachers_of_other_widths_types_and_places():
    ns, pc = circuit("hmm")
    a = teacher_for(pc, 6, 4)
    want = pc(a).detach()
    for other in (lm.TopLogits(a.ids.int(), a.logits), lm.TopLogits(a.ids.cpu(), a.logits.cpu()),
                  lm.TopLogits(torch.cat([a.ids, a.ids], 1), torch.cat([a.logits, a.logits], 1)),       # variables beyond the circuit's
                  lm.TopLogits(torch.cat([a.ids, torch.full_like(a.ids, -1)], 2), torch.cat([a.logits, a.logits], 2)),
                  lm.TopLogits(a.ids.transpose(0, 1).contiguous().transpose(0, 1), a.logits)):
        assert torch.equal(pc(other).detach(), want)
    check(ns, pc, lm.TopLogits(a.ids, a.logits.bfloat16()))
    assert pc(lm.TopLogits(a.ids[:0], a.logits[:0])).shape == (0, 1)
    # a backward pass on another batch than the forward pass's own object
    pc(a)
    pc.init_param_flows(flows_memory=0.0)
    pc.backward(lm.TopLogits(a.ids.clone(), a.logits.clone()))
    first = [layer.param_flows.clone() for layer in pc.input_layer_group]
    pc.init_param_flows(flows_memory=0.0)
    pc.backward(a)
    for f, layer in zip(first, pc.input_layer_group):
        assert torch.equal(f, layer.param_flows)


@pytest.mark.gpu
def test_refusals_of_a_circuit():
    _, pc = circuit("hmm")
    ids = torch.zeros(4, pc.num_vars, 2, dtype=torch.int64, device="cuda")
    x = torch.zeros(4, pc.num_vars, 2, device="cuda")
    for bad in (lm.TopLogits(ids[:, :-1], x[:, :-1]), lm.TopLogits(ids[..., 0], x[..., 0]), lm.TopLogits(ids[..., :0], x[..., :0]),
                lm.TopLogits(ids, x[:2]), lm.TopLogits(ids, x, 0.0)):
        with pytest.raises(ValueError):
            pc(bad)
    with pytest.raises(TypeError):
        pc(lm.TopLogits(ids.float(), x))
    layer = pc.input_layer_group[0]
    with pytest.raises(ValueError):
        layer.forward(lm.Entries(lm._prepare(lm.TopLogits(ids.transpose(0, 1), x.transpose(0, 1)), pc.num_vars)), torch.zeros(pc.num_nodes, 32, device="cuda"))


def test_tables_of_the_leaf_vectors():
    """Vectors, groups and sets of a circuit with tied and untied vectors (host)."""
    for name in STRUCTURES:
        torch.manual_seed(4)
        random.seed(4)
        pc = pj.compile(STRUCTURES[name](), verbose=False)
        for layer in pc.input_layer_group:
            t = lm.LeafTables(layer._vectors, layer.num_parameters, "cpu")
            seg = t._held[0].numpy().view(np.dtype([("var", "i4"), ("M", "i4"), ("C", "i4"), ("col", "i4"), ("row0", "i8"), ("table", "i8"), ("flow_col", "i8")]))
            grp = t._held[1].numpy().view(np.dtype([("set", "i4"), ("M", "i4"), ("C", "i4"), ("col", "i4"), ("out", "i8"), ("flow_col", "i8")]))
            first, vars_ = t._held[2].numpy().view(np.int32), t._held[3].numpy().view(np.int32)
            rows = np.concatenate([np.arange(s["row0"], s["row0"] + s["M"]) for s in seg])
            a, b = layer._output_ind_range
            assert sorted(rows.tolist()) == list(range(a, b))                                # every leaf row once
            for s in seg:
                n = np.arange(s["row0"], s["row0"] + s["M"]) - a
                assert (layer.vids.numpy()[n, 0] == s["var"]).all() and (layer.node_cats.numpy()[n] == s["C"]).all()
                assert (layer.s_pids.numpy()[n] == s["table"] + np.arange(s["M"]) * s["C"]).all()
            at = 0
            for g in grp:
                members = vars_[first[g["set"]]:first[g["set"] + 1]]
                assert g["flow_col"] == seg["flow_col"][at] and (seg["var"][at:at + len(members)] == members).all()
                assert len(set(seg["table"][at:at + len(members)])) == 1
                source = layer.source_nids.numpy()
                own = [n for n in source if layer.s_pids.numpy()[n] == seg["table"][at]]
                assert len(own) == 1 and layer.s_pfids.numpy()[own[0]] == g["out"]
                at += len(members)
            assert at == len(seg) == t.sizes["n_segs"] and t.sizes["total_vars"] == len(vars_) == first[-1]
            assert t.sizes["flow_cols"] == sum(-(-int(s["M"]) // 4) * 4 for s in seg)
