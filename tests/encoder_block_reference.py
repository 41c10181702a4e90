"""64-bit plain forms of the encoder block's operators (residual norm, neighbour attention, AdamW), and how far a kernel that computes in fp32 and rounds once at
the end may be from them.

Bounds: u = 2^-24 is half a step of fp32, `half(t)` half a step of the output's type.  A result is allowed  half(t) |result| + k u * mag  (+ the type's smallest step,
for results below its normal range), mag being the result's formula with every term taken by its magnitude and k a count of roundings on the longest path:
  row statistics      sums of up to 8192 squares over lanes: <= 8 * 4 in a lane, 6 + 8 across lanes, and a division, a root: 64 covers them twice (value and weight)
  sums over rows      rows of a lane (<= 8 here), lanes that own a column (<= 128), workgroups (<= 1024 / 8 + 8): 512
  scores              8 products in a lane, 6 shuffles, scale, bias: 20;  exp(x): 2 + |x| (its argument is rounded)
  sums over a list    256 entries of a work item at most one after the other, then its parts: 400"""
import math

import numpy as np
import torch

U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def half(t):
    return torch.finfo(t).eps / 2


def close(got, want, mag, k, what=""):
    """|got - want| within half a step of got's type plus k roundings of fp32 at magnitude `mag`; infinities and NaN at the same places"""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    got64, want = got.detach().cpu().double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got64)), what + ": values that are not finite"
    assert torch.equal(got64[~fine & ~want.isnan()], want[~fine & ~want.isnan()]) and torch.equal(got64.isnan(), want.isnan()), what
    tol = half(got.dtype) * want.abs() + k * U * (1 + half(got.dtype)) * mag + TINY[got.dtype]
    off = ((got64 - want).abs() - tol)[fine]
    assert not off.numel() or float(off.max()) <= 0, (what, "off by %.3g beyond the bound" % float(off.max()), "largest error %.3g" % float((got64 - want)[fine].abs().max()))


# ------------------------------------------------------------------------------------------------ residual norm
def act(g, name):
    return torch.sigmoid(g) if name == "SIGMOID" else g.clamp(min=0) if name == "RELU" else g


def slope(g, name):
    return torch.sigmoid(g) * (1 - torch.sigmoid(g)) if name == "SIGMOID" else (g > 0).double() if name == "RELU" else torch.ones_like(g)


def norm_rows(v, kind, eps):
    """(normalised rows, 1 / deviation, the normalised rows' terms by magnitude)"""
    mu = v.mean(1, keepdim=True) if kind == "LAYER" else torch.zeros(v.size(0), 1, dtype=v.dtype)
    r = (((v - mu) ** 2).mean(1, keepdim=True) + eps).rsqrt()
    return (v - mu) * r, r, (v.abs() + (v.abs().mean(1, keepdim=True) if kind == "LAYER" else 0)) * r


def opt(t, missing):
    return missing if t is None else t.cpu().double()


def check_residual_norm(got, x, block, gate, pw, pb, w, b, post, pre, kind, eps, scale, activation):
    y_got, h_got = got
    x64, z = x.cpu().double(), None if block is None else block.cpu().double()
    y, my = x64, x64.abs()
    if z is not None:
        if post:
            zn, _, mz = norm_rows(z, kind, eps)
            u, mu = zn * opt(pw, 1.0) + opt(pb, 0.0), mz * (abs(opt(pw, 1.0))) + abs(opt(pb, 0.0))
        else:
            u, mu = z, z.abs()
        open_ = 1.0 if gate is None else act(gate.cpu().double(), activation)
        y, my = scale * x64 + open_ * u, abs(scale) * x64.abs() + (abs(open_) if gate is not None else 1.0) * mu
        close(y_got, y, my, 64, "y")
    if pre:
        yn, r, mn = norm_rows(y, kind, eps)
        # an error e of y moves a normalised row by r (e + mean e) and, through its deviation, by |yn| r rms(e)
        moved = (my + my.mean(1, keepdim=True) + mn * (my ** 2).mean(1, keepdim=True).sqrt()) * r
        close(h_got, yn * opt(w, 1.0) + opt(b, 0.0), (moved + mn) * abs(opt(w, 1.0)) + abs(opt(b, 0.0)), 64, "h")
    else:
        assert h_got is None


def norm_back(a, ma, vn, mv, r, kind):
    """gradient of norm_rows' input from that of its output, and its terms by magnitude"""
    out, mag = a - vn * (a * vn).mean(1, keepdim=True), ma + mv * (ma * mv).mean(1, keepdim=True)
    if kind == "LAYER":
        out, mag = out - a.mean(1, keepdim=True), mag + ma.mean(1, keepdim=True)
    return out * r, mag * r


def check_residual_norm_backward(got, gy, gh, y, block, gate, pw, pb, w, b, post, pre, kind, eps, scale, activation):
    y64, z = y.cpu().double(), None if block is None else block.cpu().double()
    dt = torch.zeros_like(y64) if gy is None else gy.cpu().double()
    mt = dt.abs()
    if pre and gh is not None:
        dh = gh.cpu().double()
        yn, r, mn = norm_rows(y64, kind, eps)
        d, m = norm_back(dh * opt(w, 1.0), dh.abs() * abs(opt(w, 1.0)), yn, mn, r, kind)
        dt, mt = dt + d, mt + m
    else:
        dh, yn, mn = torch.zeros_like(y64), torch.zeros_like(y64), torch.zeros_like(y64)
    if w is not None:
        close(got["dpre_weight"], (dh * yn).sum(0), (dh.abs() * mn).sum(0), 512, "dpre_weight")
    if b is not None:
        close(got["dpre_bias"], dh.sum(0), dh.abs().sum(0), 512, "dpre_bias")
    s = scale if block is not None else 1.0
    if got["dx"] is not None:
        close(got["dx"], s * dt, abs(s) * mt, 128, "dx")
    if z is None:
        return
    zn, rz, mz = norm_rows(z, kind, eps) if post else (z, None, z.abs())
    u, mu = (zn * opt(pw, 1.0) + opt(pb, 0.0), mz * abs(opt(pw, 1.0)) + abs(opt(pb, 0.0))) if post else (z, z.abs())
    if gate is not None:
        g = gate.cpu().double()
        o, sl = act(g, activation), slope(g, activation)
        if gate.dim() == 1:
            close(got["dgate"], (dt * u).sum(0) * sl, (mt * mu).sum(0) * sl.abs(), 640, "dgate")
        else:
            close(got["dgate"], dt * u * sl, mt * mu * sl.abs(), 256, "dgate")
        dt, mt = dt * o, mt * o.abs()
    if post:
        if pw is not None:
            close(got["dpost_weight"], (dt * zn).sum(0), (mt * mz).sum(0), 640, "dpost_weight")
        if pb is not None:
            close(got["dpost_bias"], dt.sum(0), mt.sum(0), 640, "dpost_bias")
        dt, mt = norm_back(dt * opt(pw, 1.0), mt * abs(opt(pw, 1.0)), zn, mz, rz, kind)
    close(got["dblock"], dt, mt, 256, "dblock")


# ------------------------------------------------------------------------------------------------ neighbour attention
def lists_of(index, offsets, n, index_b=None, offsets_b=None, self_offset=None):
    """(row, owner) of every entry in a plan's order"""
    rows, owner = [], []
    cut = lambda i, idx, off: idx[int(off[i]):int(off[i + 1]) if i + 1 < n else idx.numel()].tolist()  # noqa: E731
    for i in range(n):
        mine = cut(i, index, offsets) if index.numel() else []
        if index_b is not None and index_b.numel():
            mine = mine + cut(i, index_b, offsets_b)
        if self_offset is not None:
            mine = mine + [self_offset + i]
        rows += mine
        owner += [i] * len(mine)
    return torch.tensor(rows, dtype=torch.int64), torch.tensor(owner, dtype=torch.int64)


def attention(q, k, v, rows, owner, scale, bias, grad=None):
    """out, stats and (with grad) dq, dk, dv, dbias in 64 bits, each with its terms by magnitude and the factor k of its bound folded in: {name: (value, magnitude)}"""
    n, H, D = q.shape
    R, E = H // k.size(1), rows.numel()
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    b = torch.zeros(E, H, dtype=torch.float64) if bias is None else bias.cpu().double()
    live = b > -math.inf
    kh, vh = k.repeat_interleave(R, 1), v.repeat_interleave(R, 1)
    ke, ve, qe = kh[rows], vh[rows], q[owner]
    dead = ~live.unsqueeze(-1)
    ke, ve = ke.masked_fill(dead, 0.0), ve.masked_fill(dead, 0.0)           # a masked entry's key and value are not used, whatever they hold
    s = ((qe * ke).sum(-1) * scale + b).masked_fill(~live, -math.inf)
    ms = (qe * ke).abs().sum(-1) * abs(scale) + b.masked_fill(~live, 0.0).abs()
    top = torch.full((n, H), -math.inf, dtype=torch.float64)
    own = owner.unsqueeze(-1).expand(E, H)
    top = top.scatter_reduce(0, own, s, "amax")
    ref = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - ref[owner])
    total = torch.zeros(n, H, dtype=torch.float64).index_add(0, owner, p)
    safe = torch.where(total > 0, total, 1.0)
    logl = torch.log(safe)
    p = p / safe[owner]
    add = lambda x, to=owner, size=n: torch.zeros(size, *x.shape[1:], dtype=torch.float64).index_add(0, to, x)  # noqa: E731
    most = lambda x: torch.zeros(n, H, dtype=torch.float64).scatter_reduce(0, own, x, "amax")  # noqa: E731
    # relative error of a probability, in units of u: its score (twice: as its own and inside m and log l), the exp of it, the sum over the list
    far = (s - ref[owner]).abs().masked_fill(~live | (p == 0), 0.0)
    rel = 2 * most(20 * ms + 4 * far) + 4 * logl.abs() + 400
    re = rel[owner].unsqueeze(-1)
    pe = p.unsqueeze(-1)
    got = {"out": (add(pe * ve), add(re * pe * ve.abs())),
           "stats": (torch.stack([top, logl], -1), torch.stack([most(20 * ms), rel + most(20 * ms)], -1))}
    if grad is None:
        return got
    g = grad.cpu().double()
    ge = g[owner]
    d, md = (ge * ve).sum(-1), (ge * ve).abs().sum(-1)
    delta, mdelta = add(p * d), add(p * md)
    ds = p * (d - delta[owner])
    mds = (re.squeeze(-1) + 100) * p * (md + mdelta[owner])
    rows_n = k.size(0)
    group = lambda x: x.view(E, H // R, R, D).sum(2)  # noqa: E731
    got["dq"] = (scale * add(ds.unsqueeze(-1) * ke), abs(scale) * add(mds.unsqueeze(-1) * ke.abs()))
    got["dk"] = (scale * add(group(ds.unsqueeze(-1) * qe), rows, rows_n), abs(scale) * add(group(mds.unsqueeze(-1) * qe.abs()), rows, rows_n))
    got["dv"] = (add(group(pe * ge), rows, rows_n), add(group(re * pe * ge.abs()), rows, rows_n))
    got["dbias"] = (ds, mds)
    return got


def check_attention(got, want):
    for name, t in got.items():
        if t is not None:
            value, mag = want[name]
            close(t, value, mag, 1, name)


# ------------------------------------------------------------------------------------------------ AdamW
def adamw(p, g, m, v, step, lr, b1, b2, eps, wd, grad_scale=None):
    """(p, m, v) in 64 bits and their bounds' magnitudes (k folded in)"""
    p, g, m, v = (t.cpu().double() for t in (p, g, m, v))
    g = g if grad_scale is None else g * float(grad_scale)
    m1, mm = b1 * m + (1 - b1) * g, 6 * (b1 * m.abs() + (1 - b1) * g.abs())
    v1, mv = b2 * v + (1 - b2) * g * g, 8 * (b2 * v + (1 - b2) * g * g)
    root = (v1 / (1 - b2 ** step)).sqrt() + eps
    move = lr / (1 - b1 ** step) / root
    return (p * (1 - lr * wd) - move * m1, 4 * p.abs() + move * (mm + 16 * m1.abs())), (m1, mm), (v1, mv)


def adamw_fp32(p, g, m, v, step, lr, b1, b2, eps, wd, grad_scale=None):
    """the moments in single fp32 operations, in the order the kernel does them: the same bits"""
    g = g.cpu().float()
    g = g if grad_scale is None else g * grad_scale.cpu()
    m, v = m.cpu(), v.cpu()
    m1 = m * torch.tensor(b1, dtype=torch.float32) + g * torch.tensor(1.0 - b1, dtype=torch.float32)
    v1 = v * torch.tensor(b2, dtype=torch.float32) + (g * torch.tensor(1.0 - b2, dtype=torch.float32)) * g
    return m1, v1


def root(v):
    """fp32 square roots, correctly rounded (numpy's are; torch's on the CPU are up to a step off)"""
    return torch.from_numpy(np.sqrt(v.numpy()))


def quantise(x, root=False):
    """an 8-bit state from fp32 values: (codes, scales), blocks of 256 with one scale each"""
    n = x.numel()
    x = torch.nn.functional.pad(x.flatten(), (0, -n % 256)).view(-1, 256)
    top = x.abs().amax(1, keepdim=True)
    top = torch.where(top < 2.0 ** -100, torch.zeros_like(top), top)
    inv = torch.where(top > 0, (torch.ones_like(top) / top) * 448.0, torch.zeros_like(top))
    y = x * inv
    if root:
        y = torch.where((y > 0) & (y < 2.0 ** -9), torch.full_like(y, 2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn).flatten()[:n], (top * torch.tensor(1.0 / 448.0, dtype=torch.float32)).flatten()


def dequantise(codes, scales):
    n = codes.numel()
    x = torch.nn.functional.pad(codes.cpu().float(), (0, -n % 256)).view(-1, 256)
    return (x * scales.cpu().view(-1, 1)).flatten()[:n]
