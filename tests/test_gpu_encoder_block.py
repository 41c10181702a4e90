"""The operators of an attention encoder's training block on the GPU against plain forms in 64 bits (tests/encoder_block_reference.py, which says where the bounds come
from): the norms around a residual (norm.hip), attention over neighbour lists (nbr_plan.hip, nbr_attention.hip), the AdamW step over many tensors (adamw.hip)."""
import math

import pytest
import torch

import encoder_block_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def H():
    from marius_amd import hip

    hip.lib()
    return hip


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ------------------------------------------------------------------------------------------------ residual norm
NORM_SHAPES = [(1, 1), (3, 2), (1, 64), (5, 100), (64, 128), (7, 257), (300, 33), (2, 1000), (19, 1032), (3, 2047), (2, 4096), (2, 8192), (1, 8191)]
NORM_FORMS = [  # post, pre, gate, activation, weights, biases, residual scale
    (False, True, None, "NONE", True, False, 1.0), (True, True, "channel", "NONE", True, True, 0.5), (True, True, "element", "SIGMOID", True, False, 1.0),
    (True, False, "channel", "RELU", True, True, 2.0), (False, True, "element", "RELU", False, False, -1.0), (True, True, "channel", "SIGMOID", False, False, 1.0),
    (True, False, None, "NONE", False, False, 1.0)]


def norm_inputs(n, d, stream, kind, gate, weights, biases, dev, seed, param=F32):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, z = (rnd(n, d) * 2 + 0.5).to(stream).to(dev), rnd(n, d).to(kind).to(dev)
    gt = None if gate is None else rnd(d).to(param).to(dev) if gate == "channel" else rnd(n, d).to(kind).to(dev)
    w = [(1 + 0.2 * rnd(d)).to(param).to(dev) if weights else None for _ in range(2)]
    b = [(0.2 * rnd(d)).to(param).to(dev) if biases else None for _ in range(2)]
    return x, z, gt, w[0], b[0], w[1], b[1], rnd(n, d).to(stream).to(dev), rnd(n, d).to(kind).to(dev)


@pytest.mark.parametrize("norm", ["RMS", "LAYER"])
@pytest.mark.parametrize("stream,kind", [(F32, F32), (F32, BF16), (BF16, BF16), (F32, F16), (F16, F16)])
@pytest.mark.parametrize("n,d", NORM_SHAPES)
def test_residual_norm_both_ways(H, dev, n, d, stream, kind, norm):
    for i, (post, pre, gate, a, weights, biases, scale) in enumerate(NORM_FORMS):
        x, z, gt, pw, pb, w, b, gy, gh = norm_inputs(n, d, stream, kind, gate, weights, biases, dev, 100 * n + d + i)
        pw, pb = (pw, pb) if post else (None, None)
        w, b = (w, b) if pre else (None, None)
        how = dict(post_norm=post, pre_norm=pre, kind=norm, eps=1e-3, residual_scale=scale, gate_activation=a)
        params = (gt, pw, pb, w, b)
        R.check_residual_norm(H.residual_norm(x, z, *params, **how), x, z, *params, post, pre, norm, 1e-3, scale, a)
        got = H.residual_norm_backward(gy, gh if pre else None, x, z, *params, **how)
        R.check_residual_norm_backward(got, gy, gh if pre else None, x, z, *params, post, pre, norm, 1e-3, scale, a)


@pytest.mark.parametrize("norm", ["RMS", "LAYER"])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_residual_norm_alone_strided_and_of_other_parameter_types(H, dev, kind, norm):
    """no block (h = norm(x)), rows of a wider tensor at an odd offset, parameters of the block's type, gradients left out, no rows at all"""
    n, d = 37, 75
    x, z, gt, pw, pb, w, b, gy, gh = norm_inputs(n, d, kind, kind, "channel", True, True, dev, 3, param=kind)
    y, h = H.residual_norm(x, pre_weight=w, pre_bias=b, kind=norm, eps=1e-5)
    assert y is x
    R.check_residual_norm((y, h), x, None, None, None, None, w, b, False, True, norm, 1e-5, 1.0, "NONE")
    for dy, dh in ((None, gh), (gy, gh), (gy, None)):
        got = H.residual_norm_backward(dy, dh, x, pre_weight=w, pre_bias=b, kind=norm, eps=1e-5)
        R.check_residual_norm_backward(got, dy, dh, x, None, None, None, None, w, b, False, True, norm, 1e-5, 1.0, "NONE")
    wide = [torch.full((n, d + 13), 7.0, dtype=kind, device=dev) for _ in range(4)]
    for t, v in zip(wide, (x, z, gy, gh)):
        t[:, 5:5 + d] = v
    xs, zs, gys, ghs = (t[:, 5:5 + d] for t in wide)
    how = dict(post_norm=True, kind=norm, eps=1e-5, residual_scale=0.7)
    for a, c in zip(H.residual_norm(xs, zs, gt, pw, pb, w, b, **how), H.residual_norm(x, z, gt, pw, pb, w, b, **how)):
        assert torch.equal(a, c)
    strided = H.residual_norm_backward(gys, ghs, xs, zs, gt, pw, pb, w, b, **how)
    R.check_residual_norm_backward(strided, gy, gh, x, z, gt, pw, pb, w, b, True, True, norm, 1e-5, 0.7, "NONE")
    again = H.residual_norm_backward(gys, ghs, xs, zs, gt, pw, pb, w, b, **how)
    assert all(torch.equal(strided[k], again[k]) for k in strided)              # the same bits on every run
    assert H.residual_norm_backward(gy, gh, x, z, gt, pw, pb, w, b, need_dx=False, **how)["dx"] is None
    none = H.residual_norm_backward(gy[:0], gh[:0], x[:0], z[:0], gt, pw, pb, w, b, **how)
    assert none["dx"].shape == (0, d) and all(not none[k].any() for k in ("dgate", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias"))
    spread = gh[:1].expand(n, d)                                                 # a gradient whose rows are one row (a sum's gradient)
    got = H.residual_norm_backward(gy, spread, x, z, gt, pw, pb, w, b, **how)
    R.check_residual_norm_backward(got, gy, spread, x, z, gt, pw, pb, w, b, True, True, norm, 1e-5, 0.7, "NONE")


def test_residual_norm_rows_apart(H, dev):
    """a row of zeros, one with an infinity and one with a NaN: the others' results are those they have alone"""
    x, z, gt, pw, pb, w, b, gy, gh = norm_inputs(9, 100, F32, F32, "channel", True, True, dev, 5)
    z[2], x[2], z[4, 7], x[6, 99] = 0, 0, math.inf, math.nan
    y, h = H.residual_norm(x, z, gt, pw, pb, w, b, post_norm=True)
    ok = [0, 1, 2, 3, 5, 7, 8]
    R.check_residual_norm((y[ok], h[ok]), x[ok], z[ok], gt, pw, pb, w, b, True, True, "RMS", 1e-6, 1.0, "NONE")
    assert not torch.isfinite(h[6]).any() and h[4].isnan().any()


def test_residual_norm_gradient_against_differences(H, dev):
    """the whole pass y, h -> scalar: its directional derivative in fp32 central differences (relative 1e-2: h^2 of the step 2^-6 and rounding / step)"""
    n, d = 6, 48
    x, z, gt, pw, pb, w, b, gy, gh = norm_inputs(n, d, F32, F32, "element", True, True, dev, 9)
    how = dict(post_norm=True, kind="LAYER", eps=1e-3, residual_scale=0.6, gate_activation="SIGMOID")
    f = lambda *t: sum(float((o.double() * g.double()).sum()) for o, g in zip(H.residual_norm(*t, **how), (gy, gh)))  # noqa: E731
    args = (x, z, gt, pw, pb, w, b)
    y, _ = H.residual_norm(*args, **how)
    got = H.residual_norm_backward(gy, gh, y, *args[1:], **how)
    names = ("dx", "dblock", "dgate", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias")
    for i, name in enumerate(names):
        v = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).to(dev)
        up, down = ([t if j != i else t + e * v for j, t in enumerate(args)] for e in (2.0 ** -6, -(2.0 ** -6)))
        want = (f(*up) - f(*down)) * 2.0 ** 5
        have = float((got[name].double() * v.double()).sum())
        assert abs(have - want) <= 1e-2 * float((got[name].double() * v.double()).norm()) * math.sqrt(d), (name, have, want)


# ------------------------------------------------------------------------------------------------ neighbour attention
def lists(n, rows, lengths, seed):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.tensor(lengths, dtype=torch.int64)
    return torch.randint(max(rows, 1), (int(lengths.sum()),), generator=g), lengths.cumsum(0) - lengths


def rows_of(n, h, d, kind, dev, seed):
    return torch.randn(n, h, d, generator=torch.Generator().manual_seed(seed)).to(kind).to(dev)


LENGTHS = {"one": [1], "none": [0, 0, 0], "single entry": [1, 0, 1], "ordinary": [0, 3, 17, 1, 0, 64, 65, 5], "long": [700, 0, 257, 256, 1, 2], "first empty": [0, 0, 9], "last empty": [9, 0]}


def both_ways(H, dev, index, offsets, rows, heads, kv, dim, kind, bias=None, seed=0, scale=None, second=None, self_offset=None, check=True):
    n = offsets.numel()
    q, k, v, g = rows_of(n, heads, dim, kind, dev, seed), rows_of(rows, kv, dim, kind, dev, seed + 1), rows_of(rows, kv, dim, kind, dev, seed + 2), rows_of(n, heads, dim, kind, dev, seed + 3)
    index_b, offsets_b = second or (None, None)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    plan = H.NeighborPlan(to(index), to(offsets), rows, to(index_b), to(offsets_b), self_offset)
    at, owner = R.lists_of(index, offsets, n, index_b, offsets_b, self_offset)
    assert plan.num_entries == at.numel() and torch.equal(plan.index.cpu().long(), at) and torch.equal(plan.owner.cpu().long(), owner)
    bias = bias(at.numel()) if callable(bias) else bias
    out, stats = H.neighbor_attention(q, k, v, plan, scale, to(bias))
    dq, dk, dv, db = H.neighbor_attention_backward(g, q, k, v, stats, plan, scale, to(bias))
    if check:
        want = R.attention(q, k, v, at, owner, dim ** -0.5 if scale is None else scale, bias, g)
        R.check_attention({"out": out, "stats": stats, "dq": dq, "dk": dk, "dv": dv, "dbias": db}, want)
    assert (db is None) == (bias is None)
    return plan, (q, k, v, g), (out, stats, dq, dk, dv, db)


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 1), (4, 4, 25), (4, 4, 32), (8, 2, 64), (3, 3, 20), (6, 2, 33), (2, 1, 128), (1, 1, 256), (16, 16, 8), (12, 1, 100), (65, 5, 7)])
@pytest.mark.parametrize("shape", sorted(LENGTHS))
def test_neighbor_attention_both_ways(H, dev, shape, heads, kv, dim, kind):
    rows = 40
    index, offsets = lists(len(LENGTHS[shape]), rows, LENGTHS[shape], len(shape))
    both_ways(H, dev, index, offsets, rows, heads, kv, dim, kind, seed=dim)


def relation_bias(heads, seed, masked=1):
    def make(entries):
        g = torch.Generator().manual_seed(seed)
        table = torch.randn(6, heads, generator=g)
        table[:masked] = -math.inf
        return table[torch.randint(6, (entries,), generator=g)]
    return make


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 32), (8, 2, 64), (3, 1, 25), (2, 2, 256)])
@pytest.mark.parametrize("masked", [0, 1, 5, 6])
def test_neighbor_attention_with_a_bias_that_masks(H, dev, masked, heads, kv, dim, kind):
    """relation biases, -inf among them: some, most, all entries masked; long lists too"""
    index, offsets = lists(6, 30, [5, 0, 400, 30, 1, 2], masked)
    both_ways(H, dev, index, offsets, 30, heads, kv, dim, kind, relation_bias(heads, 7, masked), seed=masked)


@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_neighbor_attention_lowest_value_and_masked_garbage(H, dev, kind):
    """a bias of the type's lowest value: lists that carry nothing else are uniform over their entries (as the formula says), gradients with them; keys and values that are
    infinite or NaN in masked places leave no trace; rows that no list names get zero gradients"""
    heads, dim, rows = 4, 32, 12
    index = torch.tensor([0, 1, 2, 3, 4, 5, 6, 0, 7, 7, 7, 2])
    offsets = torch.tensor([0, 4, 9, 10])
    low = torch.finfo(kind).min
    bias = torch.zeros(12, heads)
    bias[0:4] = low                    # a list of lowest values only
    bias[4:6] = low                    # some in a list
    _, _, got = both_ways(H, dev, index, offsets, rows, heads, heads, dim, kind, bias, seed=3)
    assert not got[3][8:].any() and not got[4][8:].any()
    bias = torch.zeros(12, heads)
    bias[[1, 5, 8, 9, 10]] = -math.inf
    q, k, v, g = (rows_of(m, heads, dim, kind, dev, 5 + i) for i, m in enumerate((4, rows, rows, 4)))
    plan = H.NeighborPlan(index.to(dev), offsets.to(dev), rows)
    clean = H.neighbor_attention(q, k, v, plan, None, bias.to(dev))
    clean += H.neighbor_attention_backward(g, q, k, v, clean[1], plan, None, bias.to(dev))
    for at in (1, 5, 7):
        k[at, :, ::2], v[at, :, 1::2], v[at, 0, 0] = math.inf, math.nan, -math.inf
    dirty = H.neighbor_attention(q, k, v, plan, None, bias.to(dev))
    dirty += H.neighbor_attention_backward(g, q, k, v, dirty[1], plan, None, bias.to(dev))
    assert all(torch.equal(a, b) for a, b in zip(clean, dirty))


def test_neighbor_attention_two_lists_and_own_rows(H, dev):
    """outgoing entries, then incoming ones, then the target's own row; either list may be empty"""
    a, oa = lists(5, 20, [3, 0, 4, 0, 7], 1)
    b, ob = lists(5, 20, [0, 0, 2, 300, 1], 2)
    for first, second, own in (((a, oa), (b, ob), None), ((a, oa), (b, ob), 15), ((a, oa), None, 0), ((b, ob), (a[:0], oa * 0), 3), ((a[:0], oa * 0), (b, ob), None),
                               ((a[:0], oa * 0), None, 10)):
        both_ways(H, dev, *first, 20, 4, 2, 16, F32, second=second, self_offset=own, seed=4)


def test_neighbor_attention_hubs_strides_and_repeats(H, dev):
    """one row in every list (a reverse list of 5000), q, k, v and the gradient as slices of wider tensors, a scale of one's own; the same bits on every run"""
    n, rows, heads, kv, dim = 900, 300, 4, 2, 24
    index, offsets = lists(n, rows, [6] * n, 8)
    index[::6], index[1::6] = 7, 7
    index = torch.cat([index, torch.full((3200,), 7)])
    plan, (q, k, v, g), got = both_ways(H, dev, index, offsets, rows, heads, kv, dim, F32, seed=2, scale=0.3)
    again = H.neighbor_attention(q, k, v, plan, 0.3)
    again += H.neighbor_attention_backward(g, q, k, v, again[1], plan, 0.3)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, again))
    packed = torch.zeros(rows, kv, 2 * dim + 3, device=dev)                     # k and v packed in one tensor
    packed[:, :, 1:1 + dim], packed[:, :, 1 + dim:1 + 2 * dim] = k, v
    ks, vs = packed[:, :, 1:1 + dim], packed[:, :, 1 + dim:1 + 2 * dim]
    qs, gs = (torch.zeros(heads, n, dim + 1, device=dev).transpose(0, 1)[:, :, :dim] for _ in range(2))   # heads outside
    qs.copy_(q)
    gs.copy_(g)
    strided = H.neighbor_attention(qs, ks, vs, plan, 0.3)
    strided += H.neighbor_attention_backward(gs, qs, ks, vs, strided[1], plan, 0.3)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, strided))


def test_neighbor_attention_gradient_against_differences(H, dev):
    index, offsets = lists(5, 9, [4, 0, 1, 12, 3], 6)
    bias = torch.randn(20, 4, generator=torch.Generator().manual_seed(1))
    plan, (q, k, v, g), (_, stats, dq, dk, dv, db) = both_ways(H, dev, index, offsets, 9, 4, 2, 16, F32, bias, seed=1)
    args, got = (q, k, v, bias.to(dev)), (dq, dk, dv, db)
    f = lambda q, k, v, b: float((H.neighbor_attention(q, k, v, plan, None, b)[0].double() * g.double()).sum())  # noqa: E731
    for i, name in enumerate(("dq", "dk", "dv", "dbias")):
        w = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).to(dev)
        up, down = ([t if j != i else t + e * w for j, t in enumerate(args)] for e in (2.0 ** -6, -(2.0 ** -6)))
        want, have = (f(*up) - f(*down)) * 2.0 ** 5, float((got[i].double() * w.double()).sum())
        # (third derivatives times the step's square, a softmax of few entries: below a hundredth of the terms' norm)
        assert abs(have - want) <= 1e-2 * float((got[i].double() * w.double()).norm()) * 4, (name, have, want)


# ------------------------------------------------------------------------------------------------ AdamW
def adamw_case(H, dev, sizes, param, grad, bits, seed, clip=None):
    g = torch.Generator().manual_seed(seed)
    ps = [(torch.randn(s, generator=g) * 0.3).to(param).to(dev) for s in sizes]
    gs = [(torch.randn(s, generator=g) * 0.05).to(grad).to(dev) for s in sizes]
    ms = [torch.randn(s, generator=g) * 0.01 for s in sizes]
    rs = [(torch.randn(s, generator=g) * 0.04).abs() for s in sizes]
    for r, m in zip(rs, ms):
        if r.numel() > 5:                          # weights that were never touched, and gradients far below their block's
            r[1], m[1] = 0, 0
            r[3], m[3] = 1e-9, 1e-12
    if bits == 32:
        return ps, gs, [m.to(dev) for m in ms], [(r * r).to(dev) for r in rs], None, None
    qm, qr = [R.quantise(m) for m in ms], [R.quantise(r, True) for r in rs]
    to = lambda pairs, i: [p[i].to(dev) for p in pairs]  # noqa: E731
    return ps, gs, to(qm, 0), to(qr, 0), to(qm, 1), to(qr, 1)


@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [0, 5, 0, 2048, 2049], [3] * 70, [10000, 1, 4096], [7, 8, 9, 1000]])
@pytest.mark.parametrize("param,grad", [(F32, F32), (BF16, BF16), (F32, BF16), (F16, F32), (BF16, F16)])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_step(H, dev, bits, param, grad, sizes):
    """three steps: every parameter, both moments; the 8-bit codes and scales are those of the fp32 formulas bit for bit; more than 64 tensors; empty ones; clipping"""
    hyper = dict(lr=3e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)
    hy = (3e-3, 0.9, 0.99, 1e-8, 0.1)
    ps, gs, ms, vs, sm, sv = adamw_case(H, dev, sizes, param, grad, bits, sum(sizes))
    clip = torch.tensor([0.37], device=dev)
    tensors = H.AdamWTensors(ps, ms, vs, sm, sv)
    for step in (1, 2, 40):
        c = None if step == 2 else clip
        before = [[t.cpu().clone() for t in ts] for ts in (ps, ms, vs)]
        scales = [[t.cpu().clone() for t in ts] for ts in (sm or [], sv or [])]
        H.adamw_step(tensors, gs, step, grad_scale=c, **hyper)
        for i in range(len(sizes)):
            p0, m0, v0 = (b[i] for b in before)
            if bits == 8:
                m0, v0 = R.dequantise(m0, scales[0][i]), R.dequantise(v0, scales[1][i])
                v0 = v0 * v0
            (p1, mp), (m1, mm), (v1, mv) = R.adamw(p0, gs[i], m0, v0, step, *hy, grad_scale=c)
            R.close(ps[i], p1, mp, 1, "parameter %d" % i)
            f = R.adamw_fp32(p0, gs[i], m0, v0, step, *hy, grad_scale=c)
            if bits == 32:
                R.close(ms[i], m1, mm, 1, "first moment %d" % i)
                R.close(vs[i], v1, mv, 1, "second moment %d" % i)
                assert torch.equal(ms[i].cpu(), f[0]) and torch.equal(vs[i].cpu(), f[1])
            else:
                for codes, scale, (wc, ws) in ((ms[i], sm[i], R.quantise(f[0])), (vs[i], sv[i], R.quantise(R.root(f[1]), True))):
                    assert torch.equal(codes.cpu().view(torch.uint8), wc.view(torch.uint8)) and torch.equal(scale.cpu(), ws)
                assert bool(((vs[i].cpu().float() > 0) | (f[1] == 0)).all())   # a second moment above zero stays above zero


def test_adamw_leaves_out_what_has_no_gradient_and_steps_by_a_device_counter(H, dev):
    ps, gs, ms, vs, _, _ = adamw_case(H, dev, [100, 200, 3000], F32, F32, 32, 1)
    qs, _, ns, ws, _, _ = adamw_case(H, dev, [100, 200, 3000], F32, F32, 32, 1)
    keep = [t[1].clone() for t in (ps, ms, vs)]
    H.adamw_step(H.AdamWTensors(ps, ms, vs), [gs[0], None, gs[2]], 7)
    assert all(torch.equal(a, t[1]) for a, t in zip(keep, (ps, ms, vs)))
    H.adamw_step(H.AdamWTensors(qs, ns, ws), gs, torch.tensor([7], device=dev))
    for a, b in ((ps, qs), (ms, ns), (vs, ws)):
        for i in (0, 2):
            # (the device's power of beta is in 64 bits, as the host's: at most the last bit of the two fp32 factors differs)
            assert torch.equal(a[i], b[i]) if a is not ps else float((a[i] - b[i]).abs().max()) <= 4 * R.U * float(a[i].abs().max())
    with torch.no_grad():
        H.adamw_step(H.AdamWTensors(ps, ms, vs), [None] * 3, 8)                 # nothing to do
        strided = torch.randn(200, 2, device=dev)[:, 0]
        H.adamw_step(H.AdamWTensors(ps, ms, vs), [None, strided, None], 8)
        H.adamw_step(H.AdamWTensors(qs, ns, ws), [None, strided.contiguous(), None], 8)


# ------------------------------------------------------------------------------------------------ together: the attention encoder
@pytest.fixture(scope="module")
def G():
    from marius_amd import gnn

    return gnn


def sampled(G, dev, num_nodes, E, fan, inc, out, seeds, seed):
    g = torch.Generator().manual_seed(seed)
    edges = torch.stack([torch.randint(num_nodes, (E,), generator=g), torch.randint(5, (E,), generator=g), torch.randint(num_nodes, (E,), generator=g)], 1)
    edges[: E // 5, 2] = 3
    src, dst = (edges[edges[:, c].argsort(stable=True)].to(dev) for c in (0, 2))
    graph = G.MariusGraph(src, dst, num_nodes)
    draw = lambda i, incoming, t: torch.randint(1 << 40, (t,), generator=torch.Generator().manual_seed(seed + 2 * i + int(incoming))).to(dev)  # noqa: E731
    return G.LayeredNeighborSampler(graph, fan, inc, out).getNeighbors(torch.arange(seeds).to(dev), rand=draw)


def encoder_reference(enc, features, graph, params):
    """the encoder in plain 64-bit torch operations over the graph's own lists; `params`: name -> leaf"""
    x = features @ params["project"].t()
    norm = lambda v, w: v * (v.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * w  # noqa: E731
    h = norm(x, params["first.pre_weight"])
    graph.performMap()
    for i, layer in enumerate(enc.layers):
        first = graph.getLayerOffset()
        n, p = x.size(0) - first, "layers.%d." % i
        rows, owner, rel = [], [], []
        for m, offs, edges in ((graph.out_neighbors_mapping_, graph.out_offsets_, graph.src_sorted_edges_), (graph.in_neighbors_mapping_, graph.in_offsets_, graph.dst_sorted_edges_)):
            if m is not None:
                rows.append(m.cpu())
                owner.append(torch.searchsorted(offs.cpu(), torch.arange(m.numel()), right=True) - 1)
                rel.append(edges[:, 1].cpu())
        rows, owner = torch.cat(rows + [torch.arange(first, first + n)]), torch.cat(owner + [torch.arange(n)])
        rel = torch.cat(rel + [torch.full((n,), 5)])
        R_ = layer.heads // layer.kv_heads
        q = (h[first:] @ params[p + "wq"].t()).view(n, layer.heads, layer.dim)
        kv = (h @ params[p + "wkv"].t()).view(-1, 2, layer.kv_heads, layer.dim).repeat_interleave(R_, 2)
        s = (q[owner] * kv[rows, 0]).sum(-1) * layer.dim ** -0.5 + params[p + "relation_bias"][rel]
        e = torch.exp(s)
        total = torch.zeros(n, layer.heads, dtype=torch.float64).index_add(0, owner, e)
        a = torch.zeros(n, layer.heads, layer.dim, dtype=torch.float64).index_add(0, owner, (e / total[owner]).unsqueeze(-1) * kv[rows, 1])
        block = a.reshape(n, -1) @ params[p + "wo"].t()
        w = "norms.%d." % i
        x = 0.9 * x[first:] + params[w + "gate"] * norm(block, params[w + "post_weight"])
        h = norm(x, params[w + "pre_weight"])
        if i < len(enc.layers) - 1:
            graph.prepareForNextLayer()
    return h @ params["classify"].t()


@pytest.mark.parametrize("inc,out", [(True, False), (True, True)])
@pytest.mark.parametrize("bits", [32, 8])
def test_attention_encoder_steps(H, G, dev, bits, inc, out):
    """sampling -> projections -> norms -> neighbour attention with relation biases -> gated residuals -> cross-entropy -> backward -> AdamW over all parameters: loss, outputs
    and every gradient against 64 bits, then the optimizer moves every parameter against its gradient.  Bound: 4000 roundings of fp32 at a tensor's largest entry (three layers of
    products over 32 columns, two norms each, sums over lists of up to a thousand entries)."""
    from marius_amd.optim import AdamW

    torch.manual_seed(1)
    enc = G.GraphAttentionEncoder(20, 32, 4, 2, 4, kv_heads=2, num_relations=5, residual_scale=0.9, device=dev)
    with torch.no_grad():
        for name, p in enc.named_parameters():
            if p.dim() == 1 or "relation" in name:
                p.add_(0.3 * torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())).to(dev))
    opt = AdamW(enc.parameters(), lr=1e-2, weight_decay=0.0, state_bits=bits)
    for step in range(2):
        make = lambda: sampled(G, dev, 400, 3000, [6, 5], inc, out, 40, 10 * step + 1)  # noqa: E731
        graph = make()
        features = torch.randn(graph.node_ids_.numel(), 20, generator=torch.Generator().manual_seed(step))
        labels = torch.randint(4, (40,), generator=torch.Generator().manual_seed(step))
        leaves = {n: p.detach().cpu().double().requires_grad_(True) for n, p in enc.named_parameters()}
        before = {n: p.detach().clone() for n, p in enc.named_parameters()}
        y = encoder_reference(enc, features.double(), make(), leaves)
        loss = torch.nn.functional.cross_entropy(y, labels, reduction="sum")
        loss.backward()
        got_loss, got_y = G.node_classification_step(enc, features.to(dev), graph, labels.to(dev), 0.0, optimizer=opt)
        assert abs(float(got_loss) - float(loss)) <= 4000 * R.U * float(loss)
        assert float((got_y.cpu().double() - y.detach()).abs().max()) <= 4000 * R.U * float(y.abs().max())
        for n, p in enc.named_parameters():
            want = leaves[n].grad
            assert float((p.grad.cpu().double() - want).abs().max()) <= 4000 * R.U * float(want.abs().max()), n
            moved, g = (p.detach() - before[n]).flatten(), p.grad.flatten()
            if step == 0:  # the first step from zero states: lr against the sign wherever the gradient is not tiny
                big = g.abs() > 1e-4 * g.abs().max()
                assert torch.allclose(moved[big], -1e-2 * g[big].sign(), rtol=1e-2), n


def test_attention_plan_places_of_two_lists(H, dev):
    a, oa = lists(4, 9, [2, 0, 3, 1], 1)
    b, ob = lists(4, 9, [0, 4, 1, 0], 2)
    for own in (None, 5):
        plan = H.NeighborPlan(a.to(dev), oa.to(dev), 9, b.to(dev), ob.to(dev), own)
        assert torch.equal(plan.index[plan.places(0)].cpu().long(), a) and torch.equal(plan.index[plan.places(1)].cpu().long(), b)
        every = [plan.places(0), plan.places(1)] + ([plan.places("own")] if own is not None else [])
        assert torch.equal(torch.cat(every).sort()[0].cpu(), torch.arange(plan.num_entries))
    one = H.NeighborPlan(a.to(dev), oa.to(dev), 9)
    assert torch.equal(one.places(0).cpu(), torch.arange(6))
    for part in (1, "own"):
        with pytest.raises(H.MariusHipError):
            one.places(part)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_block_captured_and_replayed(H, dev, kind):
    """norm -> attention -> gated residual -> their backward -> AdamW by a device counter, captured once and replayed on new inputs with eager work between the replays: the
    eager results bit for bit.  A step whose number is the host's is refused while capturing."""
    n, rows, heads, dim = 200, 300, 4, 16
    index, offsets = lists(n, rows, [(i * 7) % 13 for i in range(n - 1)] + [600], 3)
    plan = H.NeighborPlan(index.to(dev), offsets.to(dev), rows)
    d = heads * dim
    w = [torch.ones(d, device=dev) for _ in range(3)]
    param, m, v, m8, v8 = torch.randn(3000, device=dev), torch.zeros(3000, device=dev), torch.zeros(3000, device=dev), *(torch.zeros(12, device=dev) for _ in range(2))
    codes = [torch.zeros(3000, device=dev).to(torch.float8_e4m3fn) for _ in range(2)]
    tensors, tensors8 = H.AdamWTensors([param], [m], [v]), H.AdamWTensors([param], [codes[0]], [codes[1]], [m8], [v8])
    step = torch.zeros(1, dtype=torch.int64, device=dev)
    x, g = torch.empty(rows, d, device=dev), torch.empty(n, d, dtype=kind, device=dev)

    def block():
        _, h = H.residual_norm(x.to(kind), pre_weight=w[0])
        kv = h.view(rows, heads, dim)
        out, stats = H.neighbor_attention(kv[rows - n:], kv, kv, plan)
        z = out.view(n, d)
        y, h2 = H.residual_norm(x[rows - n:], z, w[1], w[2], pre_weight=w[0], post_norm=True)
        back = H.residual_norm_backward(None, g, y, z, w[1], w[2], pre_weight=w[0], post_norm=True)
        grads = H.neighbor_attention_backward(back["dblock"].view(n, heads, dim), kv[rows - n:], kv, kv, stats, plan)
        step.add_(1)
        flat = grads[1].reshape(-1)[:3000]
        H.adamw_step(tensors, [flat], step)
        H.adamw_step(tensors8, [flat], step)
        return [y, h2, back["dx"], back["dgate"], back["dpost_weight"], back["dpre_weight"], *grads[:3]]

    state = [param, m, v, m8, v8, codes[0], codes[1], step]
    x.normal_()
    g.normal_()
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(H.MariusHipError, match="captured step"):
            H.adamw_step(tensors, [m], 1)
        with pytest.raises(H.MariusHipError, match="before a capture"):
            H.NeighborPlan(plan.index.long(), plan.offsets[:-1].long(), rows)
        captured = block()
    torch.cuda.synchronize()
    for r in range(3):
        x.normal_()
        g.normal_()
        before = [t.clone() for t in state]
        graph.replay()
        torch.cuda.synchronize()
        got, after = [t.clone() for t in captured], [t.clone() for t in state]
        for t, b in zip(state, before):
            t.copy_(b)
        want = block()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), r
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(after, state)), r


def test_operators_on_another_stream(H, dev):
    """a stream of one's own: the launches go to the current stream, results are those of the default one"""
    index, offsets = lists(50, 60, [i % 9 for i in range(50)], 1)
    plan = H.NeighborPlan(index.to(dev), offsets.to(dev), 60)
    q, k, g = rows_of(50, 4, 32, F32, dev, 0), rows_of(60, 4, 32, F32, dev, 1), rows_of(50, 4, 32, F32, dev, 2)

    def calls():
        out, stats = H.neighbor_attention(q, k, k, plan)
        return [out, *H.neighbor_attention_backward(g, q, k, k, stats, plan)[:3], H.residual_norm(k.view(60, 128))[1]]

    want = calls()
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = calls()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_optimizer_state_is_saved_and_loaded(H, dev):
    from marius_amd.optim import AdamW

    for bits in (32, 8):
        a = [torch.randn(s, generator=torch.Generator().manual_seed(s)).to(dev).requires_grad_(True) for s in (5, 700)]
        b = [t.detach().clone().requires_grad_(True) for t in a]
        one, two = AdamW(a, state_bits=bits), AdamW(b, state_bits=bits, capturable=True)
        for t in a:
            t.grad = torch.ones_like(t) * 0.1
        one.step()
        two.load_state_dict(one.state_dict())
        for s, t in zip(a, b):
            t.data.copy_(s.data)
            t.grad = s.grad.clone()
        one.step()
        two.step()
        assert two.state_dict()["num_steps"] == one.num_steps == 2
        assert all(float((s - t).abs().max()) <= 4 * R.U * float(s.abs().max()) for s, t in zip(a, b))
        two.zero_grad()
        two.step()                                                              # nothing to do: no gradients
        with pytest.raises(H.MariusHipError):
            AdamW(a, state_bits=40 - bits).load_state_dict(one.state_dict())


def test_residual_norm_of_tiny_rows_without_eps(H, dev):
    """rows whose squares are subnormal numbers, eps = 0: the mean square is off by 2^-149 an element, 2e-6 of it here, and its root by half of that"""
    x = torch.randn(5, 64, generator=torch.Generator().manual_seed(3)) * 3e-20
    h = H.residual_norm(x.to(dev), eps=0.0)[1].cpu().double()
    want = x.double() / x.double().pow(2).mean(1, keepdim=True).sqrt()
    assert float((h - want).abs().max()) <= 1e-5 * float(want.abs().max())


def test_second_derivatives_are_refused(H, G, dev):
    x = torch.randn(3, 8, device=dev, requires_grad=True)
    norm = G.ResidualNorm(8, device=dev)
    (g,) = torch.autograd.grad(norm(x)[1].pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    plan = H.NeighborPlan(torch.tensor([0, 1, 2], device=dev), torch.tensor([0, 1], device=dev), 3)
    q, k = torch.randn(2, 2, 4, device=dev, requires_grad=True), torch.randn(3, 2, 4, device=dev)
    (g,) = torch.autograd.grad(G.neighbor_attention(q, k, k, plan).pow(2).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_gradient_of_a_sum_reaches_every_operand(H, G, dev):
    """a gradient whose strides are all zero (a sum's), single-element rows, heads and lists"""
    q, k = torch.randn(2, 2, 4, device=dev, requires_grad=True), torch.randn(3, 1, 4, device=dev, requires_grad=True)
    plan = H.NeighborPlan(torch.tensor([0, 1, 2], device=dev), torch.tensor([0, 1], device=dev), 3)
    G.neighbor_attention(q, k, k, plan).sum().backward()
    want = R.attention(q.detach(), k.detach(), k.detach(), torch.tensor([0, 1, 2]), torch.tensor([0, 1, 1]), 0.5, None, torch.ones(2, 2, 4))
    R.close(q.grad, *want["dq"], 1, "dq")
    R.close(k.grad, want["dk"][0] + want["dv"][0], want["dk"][1] + want["dv"][1], 2, "dk + dv")
    x = torch.randn(5, 1, device=dev, requires_grad=True)
    y, h = G.ResidualNorm(1, post_norm=True, bias=True, device=dev)(x, torch.randn(5, 1, device=dev))
    (y.sum() + h.sum()).backward()
    assert torch.isfinite(x.grad).all()


def test_views_of_one_row_may_have_any_stride(H, dev):
    """a dimension of size one says nothing with its stride"""
    plan = H.NeighborPlan(torch.tensor([0, 0], device=dev), torch.tensor([0], device=dev), 1)
    q, k, grad = (torch.randn(1, 2, 8, device=dev) for _ in range(3))
    far = lambda t: t.as_strided((1, 2, 8), (1 << 40, 8, 1))  # noqa: E731
    out, stats = H.neighbor_attention(far(q), far(k), far(k), plan)
    assert torch.equal(out, H.neighbor_attention(q, k, k, plan)[0])
    for a, b in zip(H.neighbor_attention_backward(far(grad), far(q), far(k), far(k), stats, plan), H.neighbor_attention_backward(grad, q, k, k, stats, plan)):
        assert a is b is None or torch.equal(a, b)


@pytest.mark.parametrize("gate", ["channel", "element"])
def test_nan_goes_through_a_relu_gate(H, dev, gate):
    x, z, g = torch.randn(3, 8, device=dev), torch.randn(3, 8, device=dev), torch.randn(8, device=dev)
    g[2], g[3] = float("nan"), -1.0
    g = g if gate == "channel" else g.expand(3, 8).contiguous()
    how = dict(pre_norm=False, gate_activation="RELU")
    y = H.residual_norm(x, z, g, **how)[0]
    assert y[:, 2].isnan().all() and torch.equal(y[:, 3], x[:, 3])
    got = H.residual_norm_backward(torch.ones_like(x), None, y, z, g, **how)
    assert got["dblock"][:, 2].isnan().all() and (got["dblock"][:, 3] == 0).all()


def test_norm_without_a_gradient_of_its_stream(H, G, dev):
    """the last block's y is not used: its gradient is absent, not zeros"""
    norm = G.ResidualNorm(16, device=dev)
    grads = []
    for use in (0.0, None):
        x, z = (torch.linspace(-1, 2, 48, device=dev).view(3, 16).sin().requires_grad_(True) for _ in range(2))
        y, h = norm(x, z)
        ((h * h).sum() if use is None else (h * h).sum() + use * y.sum()).backward()
        grads.append((x.grad, z.grad))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_adamw_step_is_seen_by_graphs_that_saved_the_parameter(H, dev):
    from marius_amd.optim import AdamW

    p, q = (torch.nn.Parameter(torch.randn(4, device=dev)) for _ in range(2))
    opt = AdamW([p, q])
    loss = (p * p).sum()
    p.grad, before = torch.ones_like(p), (p._version, q._version)
    opt.step()
    assert (p._version, q._version) == (before[0] + 1, before[1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("rows,kind", [(20000, BF16), (900000, F32)])
def test_neighbor_attention_over_a_million_entries(H, dev, rows, kind):
    """a plan whose work items are the longer ones: a hub, many ordinary lists, empty ones; rows in many lists, or in one or none"""
    g = torch.Generator().manual_seed(rows)
    lengths = torch.randint(0, 70, (31000,), generator=g)
    lengths[17] = 40000
    index, offsets = lists(lengths.numel(), rows, lengths.tolist(), 4)
    assert index.numel() > 1 << 20
    both_ways(H, dev, index, offsets, rows, 2, 1, 16, kind, relation_bias(2, 3), seed=5)


def test_neighbor_attention_rows_behind_four_gib(H, dev):
    """k and v of 4.6 GB each: the rows that lie behind 2^32 bytes give what the same rows give alone"""
    rows, n, dim = 9_000_000, 40, 128
    near = torch.randint(0, 64, (n * 9,), generator=torch.Generator().manual_seed(1)).to(dev)
    offsets = (torch.arange(n) * 9).to(dev)
    q, g, k = rows_of(n, 2, dim, F32, dev, 1), rows_of(n, 2, dim, F32, dev, 2), rows_of(64, 1, dim, F32, dev, 3)
    small = H.NeighborPlan(near, offsets, 64)
    out, stats = H.neighbor_attention(q, k, k, small)
    want = H.neighbor_attention_backward(g, q, k, k, stats, small)
    wide = torch.zeros(rows, 1, dim, device=dev)
    wide[rows - 64:] = k
    plan = H.NeighborPlan(near + (rows - 64), offsets, rows)
    far, far_stats = H.neighbor_attention(q, wide, wide, plan)
    dq, dk, dv, _ = H.neighbor_attention_backward(g, q, wide, wide, far_stats, plan)
    assert torch.equal(far, out) and torch.equal(far_stats, stats) and torch.equal(dq, want[0])
    assert torch.equal(dk[rows - 64:], want[1]) and torch.equal(dv[rows - 64:], want[2])
    assert not bool(dk[:rows - 64].any()) and not bool(dv[:rows - 64].any())


def test_adamw_of_many_tensors_in_two_graphs_of_one_pool(H, dev):
    """a list that goes through a table in workspace, captured twice into one pool and replayed in turn: every replay is the eager step"""
    sizes = [300] * 70
    runs = [adamw_case(H, dev, sizes, F32, F32, 32, seed) for seed in (1, 2)]
    eager = [adamw_case(H, dev, sizes, F32, F32, 32, seed) for seed in (1, 2)]
    tensors, plain = ([H.AdamWTensors(ps, ms, vs) for ps, _, ms, vs, _, _ in rs] for rs in (runs, eager))
    step, pool, graphs = torch.zeros(1, dtype=torch.int64, device=dev), torch.cuda.graph_pool_handle(), []
    torch.cuda.synchronize()
    for t, (_, gs, *_) in zip(tensors, runs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            H.adamw_step(t, gs, step)
    for r in range(3):
        step.add_(1)
        for graph, p, (_, gs, *_) in zip(graphs, plain, eager):
            graph.replay()
            H.adamw_step(p, gs, step)
        torch.cuda.synchronize()
        for a, b in zip(runs, eager):
            assert all(torch.equal(x, y) for k in (0, 2, 3) for x, y in zip(a[k], b[k])), r


def test_a_refused_optimizer_step_does_not_count(H, dev):
    from marius_amd.optim import AdamW

    p = torch.nn.Parameter(torch.ones(8, device=dev))
    opt = AdamW([p])
    p.grad = torch.ones_like(p)
    with pytest.raises(H.MariusHipError):
        opt.step(grad_scale=torch.ones(2, device=dev))
    opt.step()
    assert opt.num_steps == 1 and bool((p < 1).all())


def test_encoder_gradients_are_the_same_on_every_run(H, G, dev):
    """every gradient of a whole encoder, the relation biases' among them (many entries share a row), bit for bit"""
    torch.manual_seed(3)
    enc = G.GraphAttentionEncoder(16, 32, 4, 2, 4, kv_heads=2, num_relations=5, device=dev)
    runs = []
    for _ in range(4):
        enc.zero_grad()
        graph = sampled(G, dev, 3000, 60000, [12, 9], True, True, 400, 3)
        features = torch.randn(graph.node_ids_.numel(), 16, generator=torch.Generator().manual_seed(1)).to(dev)
        enc(features, graph).square().sum().backward()
        runs.append([p.grad.clone() for p in enc.parameters()])
    for again in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], again))


@pytest.mark.parametrize("T,heads,bins", [(0, 3, 5), (1, 1, 1), (9, 4, 6), (1000, 8, 6), (777, 5, 256), (3000, 64, 7), (300, 100, 3), (2049, 33, 41), (50000, 8, 6)])
def test_bin_sum(H, dev, T, heads, bins):
    """sums by bins against 64 bits, entries of no bin left out, strided values, the same bits again.  Bound: a sum of N products of one has N roundings of the running sum, each
    at most half a step of the sum of magnitudes: N lanes, workgroups and entries together stay below T / 64 + 200 of them in a row."""
    g = torch.Generator().manual_seed(T + heads)
    v, b = torch.randn(T, heads, generator=g), torch.randint(-1, bins + 1, (T,), generator=g)
    b = torch.where(torch.rand(T, generator=g) < 0.5, torch.zeros_like(b), b)
    inside = (b >= 0) & (b < bins)
    want, size = (torch.zeros(bins, heads, dtype=torch.float64).index_add(0, b[inside], x[inside].double()) for x in (v, v.abs()))
    got = H.bin_sum(v.to(dev), b.to(dev), bins)
    assert got.shape == (bins, heads) and bool(((got.cpu().double() - want).abs() <= (T / 64 + 200) * R.U * size).all())
    wide = torch.zeros(T, heads + 3, device=dev)
    wide[:, 1:1 + heads] = v.to(dev)
    assert torch.equal(got, H.bin_sum(wide[:, 1:1 + heads], b.to(dev), bins))


def test_attention_layer_with_more_relations_than_bins(H, G, dev):
    """300 relations: the gradient of the relation biases is that of the same entries' biases, summed"""
    layer = G.GraphAttentionLayer(8, 8, 2, num_relations=300, device=dev)
    few = G.GraphAttentionLayer(8, 8, 2, num_relations=5, device=dev)
    graph = sampled(G, dev, 100, 900, [5], True, True, 20, 2)
    graph.performMap()
    x = torch.randn(graph.node_ids_.numel(), 8, generator=torch.Generator().manual_seed(0)).to(dev)
    with torch.no_grad():
        for a, b in ((few.wq, layer.wq), (few.wo, layer.wo), (few.wkv, layer.wkv)):
            a.copy_(b)
    outs = [m(x, graph) for m in (layer, few)]
    assert torch.equal(*outs)
    for o in outs:
        o.square().sum().backward()
    a, b = layer.relation_bias.grad, few.relation_bias.grad
    assert float((a[[0, 1, 2, 3, 4, 300]] - b).abs().max()) <= 400 * R.U * float(b.abs().max()) + 1e-7 and not bool(a[5:300].any())


def test_attention_layer_in_bfloat16(H, G, dev):
    """a layer whose weights are bfloat16 takes bfloat16 rows, but its relation biases have to stay float32: refused, not read as if they were"""
    graph = sampled(G, dev, 100, 900, [5], True, True, 20, 2)
    graph.performMap()
    x = torch.randn(graph.node_ids_.numel(), 8, device=dev).bfloat16()
    plain = G.GraphAttentionLayer(8, 8, 2, device=dev).bfloat16()
    assert plain(x, graph).dtype == BF16
    layer = G.GraphAttentionLayer(8, 8, 2, num_relations=5, device=dev).bfloat16()
    with pytest.raises(H.MariusHipError, match="bias is float32"):
        layer(x, graph)
    layer.relation_bias.data = layer.relation_bias.data.float()
    out = layer(x, graph)
    out.float().square().sum().backward()
    assert out.dtype == BF16 and layer.relation_bias.grad.dtype == F32 and bool(layer.wq.grad.isfinite().all())
