"""Calls of the encoder block's operators that their documentation allows and tests/test_gpu_encoder_block.py does not make: outputs beside the main ones, graphs and optimizers in
states that a program reaches, inputs at the ends of their ranges.  Bounds: tests/encoder_block_reference.py."""
import math
from unittest import mock

import pytest
import torch

import encoder_block_reference as R
import test_gpu_encoder_block as T
from test_gpu_encoder_block import G, H, dev  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
F32, BF16, F16 = T.F32, T.BF16, T.F16


# ------------------------------------------------------------------------------------------------ neighbour attention
@pytest.mark.parametrize("heads,kv,dim,kind", [(4, 4, 25, F32), (8, 2, 64, BF16), (1, 1, 1, F16)])
@pytest.mark.parametrize("masked", [None, 2, 6])
def test_log_sum_exp_beside_the_output(H, dev, masked, heads, kv, dim, kind):
    """the log-sum-exp of every list: the sum of its two statistics, rounded once; -inf where nothing is live; short lists, none, one that is cut and joined.  The other
    results are those of the call without it."""
    index, offsets = T.lists(6, 30, [5, 0, 400, 30, 1, 2], 3)
    bias = None if masked is None else T.relation_bias(heads, 7, masked)(index.numel()).to(dev)
    q, k, v = T.rows_of(6, heads, dim, kind, dev, 1), T.rows_of(30, kv, dim, kind, dev, 2), T.rows_of(30, kv, dim, kind, dev, 3)
    plan = H.NeighborPlan(index.to(dev), offsets.to(dev), 30)
    out, stats, lse = H.neighbor_attention(q, k, v, plan, None, bias, return_lse=True)
    assert lse.shape == (6, heads) and lse.dtype == F32 and torch.equal(lse, stats[..., 0] + stats[..., 1])
    assert all(torch.equal(a, b) for a, b in zip((out, stats), H.neighbor_attention(q, k, v, plan, None, bias)))
    rows, owner = R.lists_of(index, offsets, 6)
    value, mag = R.attention(q, k, v, rows, owner, dim ** -0.5, None if bias is None else bias.cpu())["stats"]
    R.close(lse, value.sum(-1), mag.sum(-1), 1, "lse")
    assert bool((lse[1] == -math.inf).all()) and (masked != 6 or bool((lse == -math.inf).all()))


# ------------------------------------------------------------------------------------------------ graphs
def test_plans_are_of_mapped_lists(H, G, dev):
    """a graph whose lists are not mapped yet has no plan (it would leave every target alone with itself); mapping new lists drops the plan of the old ones, mapping again what is
    mapped keeps it: an encoder takes a graph that its caller has mapped, and takes it twice"""
    make = lambda: T.sampled(G, dev, 100, 900, [5], True, True, 20, 2)  # noqa: E731
    graph, other = make(), T.sampled(G, dev, 100, 900, [9], True, True, 20, 7)
    for call in (graph.neighborPlan, lambda: graph.entryRelations(5)):
        with pytest.raises(H.MariusHipError, match="performMap"):
            call()
    graph.performMap()
    plan, edges = graph.neighborPlan(), graph.src_sorted_edges_.size(0) + graph.dst_sorted_edges_.size(0)
    assert plan.num_entries == edges + 20 and edges > 100 and graph.neighborPlan() is plan
    enc = G.GraphAttentionEncoder(8, 16, 3, 1, 4, num_relations=5, device=dev)
    features = torch.randn(100, 8, generator=torch.Generator().manual_seed(1)).to(dev)
    want = enc(features[: make().node_ids_.numel()], make())
    for mapped in (graph, graph):
        assert torch.equal(enc(features[: graph.node_ids_.numel()], mapped), want)
    graph.hop_offsets_, graph.node_ids_, graph.graph_ = other.hop_offsets_, other.node_ids_, other.graph_
    graph.in_offsets_, graph.out_offsets_, graph.in_neighbors_vec_, graph.out_neighbors_vec_ = other.in_offsets_, other.out_offsets_, other.in_neighbors_vec_, other.out_neighbors_vec_
    graph.performMap()
    assert graph.neighborPlan() is not plan and graph.neighborPlan().num_entries == graph.src_sorted_edges_.size(0) + graph.dst_sorted_edges_.size(0) + 20


@pytest.mark.parametrize("out_edges", [[[2, 1, 3]], []])
@pytest.mark.parametrize("in_edges", [[[3, 0, 2], [2, 4, 1], [1, 2, 0]], [[3, 3, 2]], []])
def test_encoder_over_layers_whose_lists_run_out(H, G, dev, in_edges, out_edges):
    """a chain 3 -> 2 -> 1 -> 0 whose later layers have no neighbours in one direction or in both (dropout sampling leaves such graphs): a target without any has itself.
    Bound as for the other encoder steps: 4000 roundings of fp32 at a tensor's largest entry."""
    i64 = lambda v, shape=(-1,): torch.tensor(v, dtype=torch.int64).reshape(shape).to(dev)  # noqa: E731

    def make():
        ends = lambda edges, col: [0, *(sum(e[col] >= t for e in edges) for t in (2, 1))]  # noqa: E731  (lists of the targets 2, 1, 0)
        vec = lambda edges: [i64(edges, (-1, 3))] if edges else []  # noqa: E731
        base = i64([[0, 0, 1]], (1, 3))
        return G.DENSEGraph(torch.tensor([0, 1, 2, 3, 4]).to(dev), i64([3, 2, 1, 0]), i64(ends(in_edges, 2)), vec(in_edges), i64(ends(out_edges, 0)), vec(out_edges), G.MariusGraph(base, base, 4))

    torch.manual_seed(2)
    enc = G.GraphAttentionEncoder(6, 16, 3, 3, 4, kv_heads=2, num_relations=5, residual_scale=0.9, device=dev)
    with torch.no_grad():
        for layer in enc.layers:
            layer.relation_bias.copy_(torch.randn(6, 4, generator=torch.Generator().manual_seed(4)))
    features = torch.randn(4, 6, generator=torch.Generator().manual_seed(3))
    leaves = {n: p.detach().cpu().double().requires_grad_(True) for n, p in enc.named_parameters()}
    want = T.encoder_reference(enc, features.double(), make(), leaves)
    want.square().sum().backward()
    got = enc(features.to(dev), make())
    got.square().sum().backward()
    assert got.shape == (1, 3) and float((got.detach().cpu().double() - want.detach()).abs().max()) <= 4000 * R.U * float(want.abs().max())
    for n, p in enc.named_parameters():
        g = leaves[n].grad
        assert float((p.grad.cpu().double() - g).abs().max()) <= 4000 * R.U * float(g.abs().max()) + 1e-12, n


# ------------------------------------------------------------------------------------------------ AdamW
def refusals_of_a_step(dev):
    """(what is wrong with it, parameters, what makes it wrong) of optimizer steps that are refused at their last call or argument"""
    two = lambda: torch.ones(2, device=dev)  # noqa: E731
    return [("one float32", [F32], lambda ps, opt: dict(grad_scale=two())),
            ("not a dense tensor", [F32, BF16], lambda ps, opt: setattr(ps[1], "grad", ps[1].grad.to_sparse())),
            ("betas in", [F32, F16], lambda ps, opt: setattr(opt, "betas", (0.9, 1.0))),
            ("no longer what", [F32, BF16], lambda ps, opt: setattr(ps[1], "data", torch.ones(9, device=dev, dtype=BF16)))]


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("what", range(4))
def test_a_refused_step_changes_nothing(H, dev, what, capturable):
    """whichever of a step's calls is refused: no parameter, no state and no count is changed, and the step that follows is the first"""
    from marius_amd.optim import AdamW

    message, kinds, spoil = refusals_of_a_step(dev)[what]
    ps = [torch.nn.Parameter(torch.ones(8, device=dev, dtype=kind)) for kind in kinds]
    fresh = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, other = AdamW(ps, capturable=capturable), AdamW(fresh, capturable=capturable)
    for p in ps + fresh:
        p.grad = torch.full_like(p, 0.5)
    kept = [(p, p.detach().clone(), p.grad) for p in ps]
    with pytest.raises(H.MariusHipError, match=message):
        opt.step(**(spoil(ps, opt) or {}))
    assert opt.state_dict()["num_steps"] == 0 and not any(bool(t.any()) for t in opt.exp_avg + opt.exp_avg_sq)
    assert all(torch.equal(p, before) for p, before, _ in kept if p.numel() == 8)
    opt.betas = (0.9, 0.999)
    for p, before, g in kept:
        p.data, p.grad = before, g
    opt.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(ps, fresh)) and bool((ps[0] < 1).all())


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_every_parameter_counts_its_own_steps(H, dev, bits, capturable):
    """gradients that come late, now and then, always: every parameter moves as it does in an optimizer of its own that steps when it has a gradient (the same bits), and by the
    definition with its own number of steps; the counts are saved and loaded"""
    from marius_amd.optim import AdamW

    hy = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    make = lambda: [torch.nn.Parameter(torch.randn(s, generator=torch.Generator().manual_seed(s)).to(k).to(dev)) for s, k in ((300, F32), (5, F32), (700, F32), (9, BF16))]  # noqa: E731
    ps, alone = make(), make()
    opt, single = AdamW(ps, state_bits=bits, capturable=capturable, **hy), [AdamW([p], state_bits=bits, capturable=capturable, **hy) for p in alone]
    when = [lambda t: t >= 6, lambda t: True, lambda t: t % 3 == 1, lambda t: t >= 6]
    counts = [0] * 4
    for t in range(12):
        before = [(p.detach().clone(), m.detach().clone(), v.detach().clone()) for p, m, v in zip(ps, opt.exp_avg, opt.exp_avg_sq)]
        for i, (p, q) in enumerate(zip(ps, alone)):
            g = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * t + i)).to(p.dtype).to(dev)
            p.grad, q.grad = (g, g.clone()) if when[i](t) else (None, None)
        if t == 8:  # a program that ends and goes on
            opt, old = AdamW(ps, state_bits=bits, capturable=capturable), opt
            opt.load_state_dict(old.state_dict())
        opt.step()
        for i, s in enumerate(single):
            counts[i] += when[i](t)
            if when[i](t):
                s.step()
            if bits == 32 and when[i](t):
                (want, mag), _, _ = R.adamw(before[i][0], ps[i].grad, before[i][1], before[i][2], counts[i], 1e-2, 0.9, 0.99, 1e-8, 0.1)
                R.close(ps[i].detach(), want, mag, 1, "parameter %d at %d" % (i, t))
        assert all(torch.equal(a, b) for a, b in zip(ps, alone)), t
        assert all(torch.equal(a.float(), s.exp_avg[0].float()) for a, s in zip(opt.exp_avg, single)), t
        assert opt.steps == counts and opt.num_steps == max(counts)
    assert counts == [6, 12, 4, 6] and opt.state_dict()["steps"] == counts
    old = opt.state_dict()
    del old["steps"]                                                            # a state of one count for all
    opt.load_state_dict(old)
    assert opt.steps == [12] * 4


@pytest.mark.parametrize("count", [3, 70])
def test_a_step_on_the_device_for_every_tensor(H, dev, count):
    """one call over tensors whose steps differ: each gets what a call for it alone gives it; gradients that are absent in between; more tensors than one launch's arguments hold"""
    sizes = [1 + 37 * (i % 5) for i in range(count)]
    ps, gs, ms, vs, _, _ = T.adamw_case(H, dev, sizes, F32, F32, 32, 5)
    qs, _, ns, ws, _, _ = T.adamw_case(H, dev, sizes, F32, F32, 32, 5)
    steps = torch.arange(1, count + 1).to(dev)
    there = [None if i % 7 == 2 else g for i, g in enumerate(gs)]
    H.adamw_step(H.AdamWTensors(ps, ms, vs), there, steps)
    for i in range(count):
        if there[i] is not None:
            H.adamw_step(H.AdamWTensors([qs[i]], [ns[i]], [ws[i]]), [gs[i]], steps[i:i + 1])
    for a, b in ((ps, qs), (ms, ns), (vs, ws)):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for bad in (steps[:2], steps.repeat(2), steps.repeat_interleave(2)[::2][:2]):
        with pytest.raises(H.MariusHipError, match="one int64, or one for each"):
            H.adamw_step(H.AdamWTensors(ps, ms, vs), there, bad)


def test_steps_of_tensors_far_apart_in_a_long_list(H, dev):
    """200,000 tensors of which a few have gradients, over 65,536 places apart: the step of each is its own"""
    n, far = 200_000, [0, 1, 65_535, 65_536, 65_600, 140_000, 199_999]
    flat = [torch.full((n,), x, device=dev) for x in (1.0, 0.0, 0.0)]
    grads = [None] * n
    for i in far:
        grads[i] = torch.full((1,), 0.5, device=dev)
    steps = torch.zeros(n, dtype=torch.int64, device=dev)
    steps[far] = torch.tensor([1, 2, 3, 4, 50, 60, 70]).to(dev)
    tensors = H.AdamWTensors(*(list(f.split(1)) for f in flat))
    for live in (far, [5, 199_999]):
        for i in far:
            grads[i] = torch.full((1,), 0.5, device=dev) if i in live else None
        before = [f.clone() for f in flat]
        H.adamw_step(tensors, grads, steps, weight_decay=0.0)
        moved = [i for i in live if i in far]
        assert sorted((flat[0] != before[0]).nonzero().flatten().tolist()) == moved
        for i in moved:
            (want, mag), _, _ = R.adamw(before[0][i], grads[i], before[1][i], before[2][i], int(steps[i]), 1e-3, 0.9, 0.999, 1e-8, 0.0)
            R.close(flat[0][i:i + 1], want.reshape(1), mag.reshape(1), 1, str(i))


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_contiguous(H, dev, bits):
    """a column, a transposed matrix, a broadcast number: the step of a contiguous copy, in parameters and states"""
    sizes, runs = [200, 600, 64], []
    wide = torch.randn(200, 2, generator=torch.Generator().manual_seed(1)).to(dev)
    grads = [wide[:, 0], torch.randn(30, 20, generator=torch.Generator().manual_seed(2)).to(dev).t(), torch.full((1,), 0.25, device=dev).expand(64)]
    for copied in (False, True):
        ps, _, ms, vs, sm, sv = T.adamw_case(H, dev, sizes, F32, F32, bits, 1)
        start = [p.clone() for p in ps]
        tensors = H.AdamWTensors([p.view(20, 30) if i == 1 else p for i, p in enumerate(ps)], ms, vs, sm, sv)
        H.adamw_step(tensors, [g.contiguous() if copied else g for g in grads], 4)
        assert not any(torch.equal(p, s) for p, s in zip(ps, start))
        runs.append([t.float() for ts in (ps, ms, vs, sm or [], sv or []) for t in ts])
    assert not any(g.is_contiguous() for g in grads) and all(torch.equal(a, b) for a, b in zip(*runs))


def test_optimizer_captured_with_a_parameter_that_has_no_gradient(H, dev):
    """AdamW.step captured and replayed with eager work between the replays: the counts, states and parameters of the eager optimizer, the one without a gradient untouched"""
    from marius_amd.optim import AdamW

    make = lambda: [torch.nn.Parameter(torch.randn(s, generator=torch.Generator().manual_seed(s)).to(dev)) for s in (300, 5, 700)]  # noqa: E731
    ps, qs = make(), make()
    opt, eager = AdamW(ps, capturable=True), AdamW(qs, capturable=True)
    grads = [torch.zeros(300, device=dev), None, torch.zeros(700, device=dev)]
    for p, q, g in zip(ps, qs, grads):
        p.grad, q.grad = g, None if g is None else g.clone()
    for t in range(2):                                                          # eager steps first
        for o in (opt, eager):
            o.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for r in range(3):
        for g, q in zip(grads, qs):
            if g is not None:
                g.normal_()
                q.grad.copy_(g)
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert opt.steps == eager.steps == [3 + r, 0, 3 + r]
        assert all(torch.equal(a, b) for one, two in ((ps, qs), (opt.exp_avg, eager.exp_avg), (opt.exp_avg_sq, eager.exp_avg_sq)) for a, b in zip(one, two)), r


# ------------------------------------------------------------------------------------------------ residual norm
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("gate", ["channel", "element"])
def test_sigmoid_gates_far_from_zero(H, dev, gate, kind):
    """the gradient of a gate that is almost open or almost shut: sigmoid's slope is as small on one side as on the other, and as exact (a (1 - a) from a rounded a is zero from
    17 on); at +-90 it is below fp32's normal numbers, and at +-200 zero"""
    n, d = 7, 60
    x, z, _, pw, pb, w, b, gy, gh = T.norm_inputs(n, d, F32, kind, None, True, True, dev, 4)
    far = torch.tensor([s * v for s in (-1, 1) for v in (8, 9.5, 11, 12, 13, 14, 15, 15.5, 16, 16.5, 17, 18, 20, 25, 30, 40, 60, 80)] + [0, -0.5, 0.5, 4, -4, 2] * 4)
    g = far.to(kind).to(dev) if gate == "element" else far.to(dev)
    g = g.expand(n, d).contiguous() if gate == "element" else g
    how = dict(post_norm=True, kind="LAYER", eps=1e-3, residual_scale=1.0, gate_activation="SIGMOID")
    params = (g, pw, pb, w, b)
    y = H.residual_norm(x, z, *params, **how)[0]
    got = H.residual_norm_backward(gy, gh, y, z, *params, **how)
    # (sigmoid (1 - sigmoid) cancels in 64 bits, too: 2^-53 beside a slope of 1.4e-11 at 25 are 130 roundings of fp32, from 37 on the difference is zero)
    with mock.patch.object(R, "slope", lambda v, name: torch.exp(-v.abs()) / (1 + torch.exp(-v.abs())) ** 2):
        R.check_residual_norm_backward(got, gy, gh, y, z, *params, True, True, "LAYER", 1e-3, 1.0, "SIGMOID")
    small = got["dgate"].reshape(-1, d)[:, torch.tensor([10, 28])].abs().float()
    assert bool((small > 0).all())                                             # at -17 and 17
    for v in (90.0, -90.0, 200.0, -200.0):
        edge = H.residual_norm_backward(gy, gh, y, z, torch.full_like(g, v), *params[1:], **how)["dgate"]
        assert bool(edge.isfinite().all()) and float(edge.abs().max()) < 1e-30


# ------------------------------------------------------------------------------------------------ streams
def test_launches_follow_the_current_stream(H, dev):
    """inputs that are written on a side stream behind some 10 ms of products, by calls on that stream: a launch on any other stream would find the old ones.  The old inputs are
    valid too, and their results differ."""
    n, rows, heads, dim = 50, 60, 4, 32
    old_lists = [t.to(dev) for t in T.lists(n, rows, [(i + 1) % 9 for i in range(n - 4)] + [40, 80, 0, 80], 1)]
    new_lists = [(old_lists[0] * 7 + 3) % rows, old_lists[1]]
    shapes = dict(q=(n, heads, dim), k=(rows, heads, dim), v=(rows, heads, dim), g=(n, heads, dim), x=(rows, 128), z=(rows, 128), p=(500,), grad=(500,))
    rnd = lambda seed: {name: torch.randn(s, generator=torch.Generator().manual_seed(seed + i)).to(dev) for i, (name, s) in enumerate(shapes.items())}  # noqa: E731
    old, new, w = rnd(0), rnd(100), torch.linspace(0.5, 1.5, 128, device=dev)
    plan, bins = H.NeighborPlan(*new_lists, rows), torch.arange(rows).to(dev) % 7

    def calls(t, lists):
        made = H.NeighborPlan(*lists, rows)
        out, stats, lse = H.neighbor_attention(t["q"], t["k"], t["v"], plan, return_lse=True)
        y, h = H.residual_norm(t["x"], t["z"], w, pre_weight=w, post_norm=True)
        back = H.residual_norm_backward(t["x"], t["z"], y, t["z"], w, pre_weight=w, post_norm=True)
        m, v = torch.zeros_like(t["p"]), torch.zeros_like(t["p"])
        H.adamw_step(H.AdamWTensors([t["p"]], [m], [v]), [t["grad"]], 3)
        return [made.index, made._r_owner[:made.num_entries], out, stats, lse, *H.neighbor_attention_backward(t["g"], t["q"], t["k"], t["v"], stats, plan)[:3], y, h,
                *(g for g in back.values() if g is not None), H.bin_sum(t["x"], bins, 7), t["p"], m, v]

    want, stale = (calls({k: v.clone() for k, v in t.items()}, lists) for t, lists in ((new, new_lists), (old, old_lists)))
    assert not any(torch.equal(a, b) for a, b in zip(want, stale))
    inputs, lists = {k: v.clone() for k, v in old.items()}, [t.clone() for t in old_lists]
    big = torch.randn(4096, 4096, device=dev)
    side = torch.cuda.Stream(device=dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(10):
            big @ big
        for name, t in inputs.items():
            t.copy_(new[name])
        for t, fresh in zip(lists, new_lists):
            t.copy_(fresh)
        # the plan first: its readbacks wait for the products, so a second delay stands in front of the others
        made = H.NeighborPlan(*lists, rows)
        assert torch.equal(made.index, want[0]) and torch.equal(made._r_owner[:made.num_entries], want[1])
        for name, t in inputs.items():
            t.copy_(old[name])
        side.synchronize()
        for _ in range(10):
            big @ big
        for name, t in inputs.items():
            t.copy_(new[name])
        delayed = not side.query()
        out, stats, lse = H.neighbor_attention(inputs["q"], inputs["k"], inputs["v"], plan, return_lse=True)
        y, h = H.residual_norm(inputs["x"], inputs["z"], w, pre_weight=w, post_norm=True)
        back = H.residual_norm_backward(inputs["x"], inputs["z"], y, inputs["z"], w, pre_weight=w, post_norm=True)
        sums = H.bin_sum(inputs["x"], bins, 7)
        m, v = torch.zeros(500, device=dev), torch.zeros(500, device=dev)
        H.adamw_step(H.AdamWTensors([inputs["p"]], [m], [v]), [inputs["grad"]], 3)
        got = [out, stats, lse, *H.neighbor_attention_backward(inputs["g"], inputs["q"], inputs["k"], inputs["v"], stats, plan)[:3], y, h,
               *(g for g in back.values() if g is not None), sums, inputs["p"], m, v]
    side.synchronize()
    assert delayed and len(got) == len(want) - 2 and all(torch.equal(a, b) for a, b in zip(got, want[2:]))


# ------------------------------------------------------------------------------------------------ plans
def test_a_plan_in_use_on_another_stream_is_recorded_whole(H, dev):
    """record_stream reaches every tensor that the plan holds, what `places` reads among them"""
    index, offsets = T.lists(4, 9, [2, 0, 3, 1], 1)
    plan = H.NeighborPlan(index.to(dev), offsets.to(dev), 9, index.to(dev), offsets.to(dev), 5)
    seen = set()
    with mock.patch.object(torch.Tensor, "record_stream", lambda t, stream: seen.add(t.data_ptr())):
        plan.record_stream(None)
    held, todo = [], list(vars(plan).values())
    while todo:
        x = todo.pop()
        todo += list(x) if isinstance(x, (list, tuple)) else []
        held += [x] if torch.is_tensor(x) else []
    assert len(held) >= 9 and {t.data_ptr() for t in held if t.numel() > 0} <= seen


def test_a_plan_keeps_no_hold_on_the_lists_it_was_made_of(H, dev):
    """a program that samples into the same buffers batch after batch: the plan, and where its entries lie, stay those of the lists that it was made of"""
    a, oa = T.lists(4, 9, [2, 0, 3, 1], 1)
    b, ob = T.lists(4, 9, [0, 4, 1, 0], 2)
    for second in (False, True):
        for own in (None, 5):
            buffers = [t.to(dev) for t in ((a, oa, b, ob) if second else (a, oa))]
            plan = H.NeighborPlan(buffers[0], buffers[1], 9, *buffers[2:], self_offset=own)
            for t in buffers:
                t.zero_()
            assert torch.equal(plan.index[plan.places(0)].cpu().long(), a)
            assert not second or torch.equal(plan.index[plan.places(1)].cpu().long(), b)
            every = [plan.places(p) for p in ([0, 1] if second else [0]) + ([] if own is None else ["own"])]
            assert torch.equal(torch.cat(every).sort()[0].cpu(), torch.arange(plan.num_entries))


def test_parameters_given_one_memory_after_their_optimizer_was_made(H, dev):
    """new memory between two steps is read at the next one; the memory of another parameter or of a state is refused: two workgroups would write one element"""
    from marius_amd.optim import AdamW

    p, q, r = (torch.nn.Parameter(torch.ones(300, device=dev)) for _ in range(3))
    opt = AdamW([p, q, r])
    for t in (p, q, r):
        t.grad = torch.ones_like(t)
    opt.step()
    own, flat = q.data, torch.ones(500, device=dev)
    for bad in (p.data, opt.exp_avg[2].data, opt.exp_avg_sq[0].data):
        q.data = bad
        with pytest.raises(H.MariusHipError, match="appears twice, or overlaps"):
            opt.step()
    p.data, q.data = flat[:300], flat[200:]
    with pytest.raises(H.MariusHipError, match="appears twice, or overlaps"):
        opt.step()
    q.data, p.data = own, torch.ones(300, device=dev)
    opt.step()
    fresh = torch.ones(300, device=dev)
    r.data = fresh
    opt.step()
    assert opt.num_steps == 3 and r.data_ptr() == fresh.data_ptr() and bool((fresh < 1).all()) and bool((p < 1).all()) and bool((q < 1).all())


def test_states_given_new_memory(H, dev):
    """a state whose tensor is given other memory (loaded from elsewhere, say) is read and written there; memory that does not fit is refused"""
    ps, gs, ms, vs, sm, sv = T.adamw_case(H, dev, [300, 700], F32, F32, 8, 3)
    qs, hs, ns, ws, tm, tv = T.adamw_case(H, dev, [300, 700], F32, F32, 8, 3)
    one, two = H.AdamWTensors(ps, ms, vs, sm, sv), H.AdamWTensors(qs, ns, ws, tm, tv)
    H.adamw_step(one, gs, 1)
    H.adamw_step(two, hs, 1)
    for t in (ns[1], ws[0], tm[1]):
        old = t.data
        t.data = old.clone()
        old.zero_()
    H.adamw_step(one, gs, 2)
    H.adamw_step(two, hs, 2)
    assert all(torch.equal(a.float(), b.float()) for x, y in ((ps, qs), (ms, ns), (vs, ws), (sm, tm), (sv, tv)) for a, b in zip(x, y))
    for t, bad in ((ns[0], ns[0][:200].clone()), (tm[0], tm[0][:1].clone()), (ws[1], torch.zeros(700, 2, device=dev).to(torch.float8_e4m3fn)[:, 0]), (ns[0], ns[0][:200])):
        kept, t.data = t.data, bad
        with pytest.raises(H.MariusHipError, match="of its size|one for 256|contiguous"):
            H.adamw_step(two, hs, 3)
        t.data = kept
    H.adamw_step(two, hs, 3)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite_spoil_no_more_than_they_have_to(H, dev, bits):
    """a NaN its element, an infinity its element or, as the scale of an 8-bit block, its block; every other element of the tensor and the tensors beside it are those of a step
    without them"""
    runs = []
    for spoilt in (False, True):
        ps, gs, ms, vs, sm, sv = T.adamw_case(H, dev, [1000, 300], F32, F32, bits, 2)
        if spoilt:
            gs[0][10], gs[0][600] = math.nan, math.inf
        tensors = H.AdamWTensors(ps, ms, vs, sm, sv)
        for step in (1, 2):
            H.adamw_step(tensors, gs, step)
        runs.append(ps)
    bad = torch.zeros(1000, dtype=torch.bool)
    bad[10], bad[600] = True, True
    if bits == 8:
        bad[512:768] = True
    got, want = runs[1][0].cpu(), runs[0][0].cpu()
    assert bool((got[bad] != want[bad]).all()) and not bool(got[bad].isfinite().any()) and torch.equal(got[~bad], want[~bad]) and torch.equal(runs[1][1], runs[0][1])
