"""Kept rows at the edges of what is documented: values that are not finite next to the end of the rows,
modules whose parameters are made on the fly, kinks at the end of the codes' range, rows and layers that
do not fit, no rows, long sums of one sign.

Tolerances as in test_gpu_kept_rows: u = 2^-24 per float32 operation, times the sum of magnitudes."""
import numpy as np
import pytest
import torch
from torch.nn.utils import parametrize, prune

import kept_rows_reference as ref
import test_gpu_kept_rows as base

pytestmark = pytest.mark.gpu
U = base.U
T = base.T
within = base.within


# ---- a value that is not finite in the last, cut tile -----------------------------------------------
SHAPES = [(64, 64), (64, 40), (32, 8), (16, 56), (8, 24), (33, 9)]


@pytest.mark.parametrize("I,O", SHAPES)
@pytest.mark.parametrize("rows", [5, 3001])
def test_linear_nan_in_the_last_row(rows, I, O):
    """The last value of the last row is NaN, the one three columns before it infinite: their columns of
    the weight gradient are NaN, and no others (the lanes past the last row must not bring them back)."""
    from mvfusion import training as tr
    g = np.random.default_rng(rows + I)
    lin = torch.nn.Linear(I, O).cuda()
    x = g.normal(size=(rows, I)).astype(np.float32)
    x[rows - 1, I - 1], x[rows - 1, I - 4] = np.nan, np.inf
    bad = [I - 4, I - 1]
    gy = g.normal(size=(rows, O)).astype(np.float32)
    xt = T(x).cuda().requires_grad_(True)
    y = tr.linear(lin, xt, keep="int8")
    gx, gw, gb = (t.cpu().numpy() for t in torch.autograd.grad(y, (xt, lin.weight, lin.bias), T(gy).cuda()))
    good = np.setdiff1d(np.arange(I), bad)
    xq = ref.unpack(*ref.pack(x))[:, good]
    g64, w64 = gy.astype(np.float64), lin.weight.detach().cpu().double().numpy()
    within(gw[:, good], g64.T @ xq, base.xty_bound(g64, xq, rows), "weight")
    assert np.isnan(gw[:, bad]).all()
    within(gx, g64 @ w64, (O + 2) * U * (np.abs(g64) @ np.abs(w64)), "x")
    within(gb, g64.sum(0), 64 * U * np.abs(g64).sum(0), "bias")


@pytest.mark.parametrize("training", [False, True])
@pytest.mark.parametrize("I,O", SHAPES)
def test_block_nan_in_the_last_row(I, O, training):
    """The same behind BatchNorm: in train mode the statistics make the whole column NaN, and only it.
    512 u: the sums of 3000 rows as in test_block_kinks_and_nan."""
    from mvfusion import packed, training as tr
    rows = 3001
    g = np.random.default_rng(I + O)
    bn, lin = torch.nn.BatchNorm1d(I).cuda().train(training), torch.nn.Linear(I, O).cuda()
    gamma, beta = (1 + 0.3 * g.normal(size=I)).astype(np.float32), (0.3 * g.normal(size=I)).astype(np.float32)
    with torch.no_grad():
        bn.weight.copy_(T(gamma))
        bn.bias.copy_(T(beta))
    z = base.rows_of(rows, I, 11)
    z[rows - 1, I - 1] = np.nan
    x = T(z).cuda().requires_grad_(True)
    gy = T(g.normal(size=(rows, O)).astype(np.float32)).cuda()
    state = {k: v.clone() for k, v in bn.state_dict().items()}
    y = tr.batch_norm_act_linear(x, bn, torch.nn.LeakyReLU(0.25), lin, keep="int8")
    gx, dgamma, dbeta, dw = (t.cpu().numpy() for t in
                             torch.autograd.grad(y, (x, bn.weight, bn.bias, lin.weight), gy))
    bn.load_state_dict(state)
    _, codes, exps, invstd = tr._bn8_forward(x.detach(), bn.weight.detach(), bn.bias.detach(), bn.running_mean,
                                             bn.running_var, bn.eps, 0.25, training, 0.1, None, None)
    zq = packed.unpack_rows(codes, exps).double().cpu().numpy()
    good = np.arange(I - 1)
    t = np.where(ref.bn_on(zq, gamma, beta), 1.0, 0.25)
    g64, w64 = gy.double().cpu().numpy(), lin.weight.detach().double().cpu().numpy()
    gh, mag = (t * (g64 @ w64))[:, good], (np.abs(g64) @ np.abs(w64))[:, good]
    v = (t * (gamma.astype(np.float64) * zq + beta))[:, good]
    zq = zq[:, good]
    vmag = np.abs(gamma[good] * zq) + np.abs(beta[good])
    within(dw[:, good], g64.T @ v, 512 * U * (np.abs(g64).T @ vmag), "dw")
    assert np.isnan(dw[:, I - 1]).all() and np.isnan(dgamma[I - 1])
    within(dbeta[good], gh.sum(0), 512 * U * mag.sum(0), "dbeta")
    within(dgamma[good], (gh * zq).sum(0), 512 * U * (mag * np.abs(zq)).sum(0), "dgamma")
    k = (gamma.astype(np.float64) * invstd.cpu().double().numpy())[good]
    if training:
        want = (gh - gh.mean(0) - zq * (gh * zq).mean(0)) * k
        mag = mag + mag.mean(0) + np.abs(zq) * (mag * np.abs(zq)).mean(0)
    else:
        want = gh * k
        assert np.isfinite(gx).all()
    within(gx[:, good], want, 512 * U * mag * np.abs(k), "gx")


# ---- parameters that are made on the fly -------------------------------------------------------------
class Doubled(torch.nn.Module):
    def forward(self, w):
        return 2 * w


def made(bn, how):
    """bn with a weight that is no entry of its own parameters."""
    if how == "parametrized":
        parametrize.register_parametrization(bn, "weight", Doubled())
    elif how == "pruned":
        prune.random_unstructured(bn, "weight", 0.5)
    elif how == "replica":
        (bn,) = torch.nn.parallel.replicate(bn, [0])
    return bn


@pytest.mark.parametrize("keep", ["float32", "int8"])
@pytest.mark.parametrize("how", ["parametrized", "pruned", "replica"])
def test_batch_norm_with_a_made_weight(how, keep):
    """The kernels take a BatchNorm whose weight is parametrized, pruned or a replica's copy: what a plain
    module with the same weight gives, and the gradient of the parameter underneath."""
    from mvfusion import training as tr
    torch.manual_seed(4)
    source, act, lin = torch.nn.BatchNorm1d(40).cuda(), torch.nn.LeakyReLU(0.2), torch.nn.Linear(40, 8).cuda()
    with torch.no_grad():
        source.weight.uniform_(0.5, 2)
        source.bias.uniform_(-1, 1)
    bn = made(source, how)
    plain = torch.nn.BatchNorm1d(40).cuda()
    with torch.no_grad():
        plain.weight.copy_(bn.weight)
        plain.bias.copy_(bn.bias)
    x, gy = torch.randn(5000, 40, device="cuda", requires_grad=True), torch.randn(5000, 40, device="cuda")
    under = next(p for n, p in source.named_parameters() if "weight" in n)
    (factor,) = torch.autograd.grad(bn.weight.sum(), under, retain_graph=True)
    y, want = tr.batch_norm_act(x, bn, act, keep=keep), tr.batch_norm_act(x, plain, act, keep=keep)
    assert torch.equal(y, want)
    gx, gw = torch.autograd.grad(y, (x, under), gy, retain_graph=True)   # (pruning makes the weight once)
    wx, ww = torch.autograd.grad(want, (x, plain.weight), gy)
    assert torch.equal(gx, wx) and torch.equal(gw, ww * factor)
    assert torch.equal(bn.running_mean, plain.running_mean) and int(bn.num_batches_tracked) == 1
    y, want = tr.batch_norm_act_linear(x, bn, act, lin, keep=keep), tr.batch_norm_act_linear(x, plain, act, lin, keep=keep)
    assert torch.equal(y, want)
    assert torch.equal(torch.autograd.grad(y, x, gy[:, :8])[0], torch.autograd.grad(want, x, gy[:, :8])[0])


# ---- no rows ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("keep", ["float32", "int8"])
def test_pool_of_points_without_views(keep):
    """A sample none of whose points has a view, in eval mode with a graph: zeros, and zero gradients of
    whatever the views go through."""
    from mvfusion import training as tr
    pool = base.make_pool().eval()
    x = [torch.randn(s, device="cuda", requires_grad=True) for s in ((7, 24), (0, 64), (0, 8))]
    ptr = torch.zeros(8, dtype=torch.int64, device="cuda")
    with tr.keep_activations(keep):
        out = pool(x[0], x[1], x[2], ptr)
    assert out.shape == (7, 64) and not out.any()
    grads = torch.autograd.grad(out.sum(), x + list(pool.parameters()), allow_unused=True)
    assert all(g is None or not g.any() for g in grads)


@pytest.mark.parametrize("keep", ["float32", "int8"])
def test_layers_without_rows(keep):
    """Every layer of the training path on no rows, in eval mode."""
    from mvfusion import training as tr
    from mvfusion.dense import MLP
    lin, bn, act = torch.nn.Linear(64, 32).cuda(), torch.nn.BatchNorm1d(64).cuda().eval(), torch.nn.LeakyReLU(0.2)
    seq = MLP([40 + 24, 32, 16], bias=False).cuda().eval()
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    ptr = torch.zeros(5, dtype=torch.int64, device="cuda")
    with tr.keep_activations(keep):
        assert tr.linear(lin, x).shape == (0, 32) and tr.batch_norm_act(x, bn, act).shape == (0, 64)
        assert tr.batch_norm_act_linear(x, bn, act, lin).shape == (0, 32) and tr.mlp(seq, x).shape == (0, 16)
        y = tr.mlp_on_rows_and_sets(seq, x[:, :40], torch.randn(4, 24, device="cuda"), ptr)
        assert y.shape == (0, 16)
    (gw,) = torch.autograd.grad(y.sum(), seq[0][0].weight)
    assert gw.shape == (32, 64) and not gw.any()


# ---- layers that do not fit the rows ------------------------------------------------------------------
@pytest.mark.parametrize("keep", ["float32", "int8"])
@pytest.mark.parametrize("rows", [40, 5000])
def test_widths_that_do_not_fit(rows, keep):
    """A layer of another width than the rows is the module's to refuse: no kernel runs on it."""
    from mvfusion import _lib, training as tr
    x = torch.randn(rows, 32, device="cuda", requires_grad=True)
    act, bn = torch.nn.LeakyReLU(0.2), torch.nn.BatchNorm1d(32).cuda()
    for width in (16, 64):
        lin, other = torch.nn.Linear(width, 8).cuda(), torch.nn.BatchNorm1d(width).cuda()
        for call in (lambda: tr.linear(lin, x, keep=keep), lambda: tr.batch_norm_act(x, other, act, keep=keep),
                     lambda: tr.batch_norm_act_linear(x, bn, act, lin, keep=keep),
                     lambda: tr.batch_norm_act_linear(x, other, act, torch.nn.Linear(32, 8).cuda(), keep=keep),
                     lambda: tr.linear(lin.cpu(), x, keep=keep)):
            with pytest.raises(RuntimeError) as e:
                call()
            assert not isinstance(e.value, _lib.MvfError)


@pytest.mark.parametrize("keep", ["float32", "int8"])
def test_sets_that_do_not_fit(keep):
    """The split first Linear of the set encoder: the halves have to fit rows and sets, and parameters on
    the host are refused rather than read."""
    from mvfusion import training as tr
    from mvfusion.dense import MLP
    seq = MLP([64, 32, 16], bias=False).cuda().eval()
    ptr = torch.tensor([0, 3, 3, 20], device="cuda")
    x, sets = torch.randn(20, 32, device="cuda", requires_grad=True), torch.randn(3, 32, device="cuda")
    with tr.keep_activations(keep):
        want = tr.mlp(seq, torch.cat((x, sets.repeat_interleave(ptr.diff(), dim=0)), 1))
        assert torch.allclose(tr.mlp_on_rows_and_sets(seq, x, sets, ptr), want, rtol=1e-5, atol=1e-5)
        for bad in ((x, sets[:, :16]), (x[:, :16], sets), (x, torch.randn(3, 48, device="cuda"))):
            with pytest.raises(RuntimeError):
                tr.mlp_on_rows_and_sets(seq, *bad, ptr)
        with pytest.raises(RuntimeError):
            tr.mlp_on_rows_and_sets(seq.cpu(), x, sets, ptr)


# ---- the reduction over packed rows by itself -----------------------------------------------------------
@pytest.mark.parametrize("tail", [False, True])
def test_xty8_layouts(tail):
    """Rows, codes and parameters that are not contiguous give what contiguous ones do; no rows give zeros."""
    from mvfusion import packed, training as tr
    torch.manual_seed(6)
    x, y = torch.randn(1000, 24, device="cuda"), torch.randn(1000, 50, device="cuda")
    w, b = torch.randn(2, 50, device="cuda")
    p = packed.pack_rows(y)
    args = (w, b, 0.2) if tail else None
    want, sums = tr.xty8(x, p.codes, p.exps, args, want_sums=True)
    v = p.unpack().double()
    if tail:
        v = v * w.double() + b.double()
        v = torch.where(v > 0, v, v * float(np.float32(0.2)))
    g = x.double()
    mag = (g.abs().t().contiguous() @ (p.unpack().double().abs() * (w.double().abs() if tail else 1)
                                       + (b.double().abs() if tail else 0))).cpu().numpy()
    within(want.cpu().numpy(), (g.t().contiguous() @ v).cpu().numpy(), 512 * U * mag)
    within(sums.cpu().numpy(), g.sum(0).cpu().numpy(), 64 * U * g.abs().sum(0).cpu().numpy())
    spread = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731
    got, again = tr.xty8(spread(x), spread(p.codes), spread(p.exps), (spread(w), spread(b), 0.2) if tail else None,
                         want_sums=True)
    assert torch.equal(got, want) and torch.equal(again, sums)
    none, sums = tr.xty8(x[:0], p.codes[:0], p.exps[:0], args, want_sums=True)
    assert none.shape == (24, 50) and not none.any() and not sums.any()


# ---- kinks at the end of the codes' range --------------------------------------------------------------
def sided_codes(zh, gamma, beta):
    """(codes, exps) of normalised rows: the code nearest to the value on its own side of the kink; a group in
    which a value of at least 127 steps meets a kink of 127 to 128 steps takes the next step."""
    C = zh.shape[1]
    t = (-beta.astype(np.float32) / gamma.astype(np.float32)).astype(np.float64)
    on, up = zh * gamma + beta > 0, gamma > 0
    zf = zh.astype(np.float32)
    e = ref.exponents(zf)
    at = np.ldexp(np.broadcast_to(t, zh.shape), ref.BIAS - ref.spread(e, C))
    past = np.zeros((zh.shape[0], e.shape[1] * ref.GROUP), bool)
    past[:, :C] = (np.abs(zf) >= np.ldexp(127.0, ref.spread(e, C) - ref.BIAS)) & (np.floor(np.abs(at)) == 127)
    e = e + past.reshape(*e.shape, ref.GROUP).any(2)
    q = np.clip(ref.codes_of(zh, e), -127, 127)
    at = np.ldexp(np.broadcast_to(t, zh.shape), ref.BIAS - ref.spread(e, C))
    q = np.where(on, np.where(up, np.fmax(q, np.floor(at) + 1), np.fmin(q, np.ceil(at) - 1)),
                 np.where(up, np.fmin(q, np.floor(at)), np.fmax(q, np.ceil(at))))
    assert np.abs(q).max() <= 127
    return q.astype(np.int8), e.astype(np.uint8)


def rows_at_the_end(rows, C, g):
    """(z, gamma, beta): kinks of either sign between 127 and 127.5 steps of 1/64, some at the ends of that range
    and some elsewhere, and rows whose largest values lie on both sides of them."""
    gamma = np.where(g.random(C) < 0.5, -1.0, 1.0) * 2.0 ** g.integers(-1, 2, C)
    kink = (127 + g.choice([0.0, 0.03, 0.2, 0.4, 0.49, 0.5], C)) / 64 * np.where(g.random(C) < 0.5, -1, 1)
    kink[::3] = g.normal(size=len(kink[::3]))
    beta = (-kink * gamma).astype(np.float32)
    z = g.uniform(-1.9, 1.9, (rows, C))
    near = g.random((rows, C)) < 0.1
    z = np.where(near, np.sign(kink) * (127 + g.uniform(-0.6, 0.5, (rows, C))) / 64, z)
    z = np.where(g.random((rows, C)) < 0.02, kink, z)
    z *= 2.0 ** np.where(g.random((rows, 1)) < 0.1, -1, 0)
    return z.astype(np.float32), gamma.astype(np.float32), beta


@pytest.mark.parametrize("rows,C,O", [(40, 33, 0), (900, 64, 0), (3000, 50, 0), (2500, 32, 0), (5000, 6, 0), (3001, 8, 8),
                                      (3001, 16, 40), (3001, 32, 16), (3001, 64, 64), (3001, 33, 9)])
def test_kept_side_at_the_end_of_the_range(rows, C, O):
    """Eval mode with statistics that make the normalised value z itself.  Bounds: the product, the slope and the
    scale are three float32 operations behind g, or behind g W with O + 2."""
    from mvfusion import training as tr
    g = np.random.default_rng(rows + C)
    z, gamma, beta = rows_at_the_end(rows, C, g)
    bn = torch.nn.BatchNorm1d(C, eps=0.0).cuda().eval()
    with torch.no_grad():
        bn.weight.copy_(T(gamma))
        bn.bias.copy_(T(beta))
    codes, exps = sided_codes(z.astype(np.float64), gamma.astype(np.float64), beta.astype(np.float64))
    plain = ref.exponents(z)
    assert 0 < (exps > plain).sum() < 0.8 * exps.size
    x, act = T(z).cuda().requires_grad_(True), torch.nn.LeakyReLU(0.125)
    if O:
        lin = torch.nn.Linear(C, O).cuda()
        y = tr.batch_norm_act_linear(x, bn, act, lin, keep="int8")
        w64 = lin.weight.detach().cpu().double().numpy()
    else:
        y, w64 = tr.batch_norm_act(x, bn, act, keep="int8"), np.eye(C)
    got = [t.cpu().numpy() for t in y.grad_fn.saved_tensors[:2]]
    assert np.array_equal(got[0], codes) and np.array_equal(got[1], exps)
    zq, on = ref.unpack(codes, exps), z.astype(np.float64) * gamma + beta > 0
    assert np.array_equal(ref.bn_on(zq, gamma.astype(np.float64), beta.astype(np.float64)), on)
    assert np.all(np.abs(zq - z) <= np.ldexp(1.0, ref.spread(exps.astype(np.int64), C) - ref.BIAS))
    gy = g.normal(size=(rows, O or C)).astype(np.float32)
    gx, dgamma, dbeta = (t.cpu().numpy() for t in torch.autograd.grad(y, (x, bn.weight, bn.bias), T(gy).cuda()))
    t = np.where(on, 1.0, 0.125)
    gh, mag = t * (gy.astype(np.float64) @ w64), np.abs(gy.astype(np.float64)) @ np.abs(w64)
    within(gx, gh * gamma, (O + 5) * U * mag * np.abs(gamma), "z")
    within(dbeta, gh.sum(0), 1024 * U * mag.sum(0), "beta")
    within(dgamma, (gh * zq).sum(0), 1024 * U * (mag * np.abs(zq)).sum(0), "gamma")


def test_idle_columns_take_no_part_in_a_group():
    """Lanes past the last column hold no value: they must not send their group to the next step."""
    from mvfusion import training as tr
    for rows in (300, 2000):
        z = np.full((rows, 5), 0.5, np.float32)
        bn = torch.nn.BatchNorm1d(5, eps=0.0).cuda().eval()
        with torch.no_grad():
            bn.running_mean[4], bn.running_var[4] = -1e4, 1.0       # (an idle column would read as 1e4)
            bn.bias[4] = -50.0
        z[:, 4] = -1e4
        y = tr.batch_norm_act(T(z).cuda().requires_grad_(True), bn, torch.nn.LeakyReLU(0.2), keep="int8")
        codes, exps = (t.cpu().numpy() for t in y.grad_fn.saved_tensors[:2])
        assert (codes[:, :4] == 64).all() and not codes[:, 4].any() and (exps == 126).all()


# ---- long sums -----------------------------------------------------------------------------------------
def over_rows(g, v):
    out = torch.zeros(g.shape[1], v.shape[1], dtype=torch.float64, device="cuda")
    for k in range(0, g.shape[0], 1 << 18):
        out += g[k:k + (1 << 18)].double().t().contiguous() @ v[k:k + (1 << 18)].double()
    return out


def long_sums(op, x, gy, lin, bn):
    """(weight gradient and, for the block, BatchNorm's gradients, what they are in float64)."""
    from mvfusion import packed, training as tr
    if op == "linear":
        y = tr.linear(lin, x, keep="int8")
        _, gw = torch.autograd.grad(y, (x, lin.weight), gy)
        return [gw], [over_rows(gy, packed.pack_rows(x).unpack())]
    y = tr.batch_norm_act_linear(x, bn, torch.nn.LeakyReLU(0.25), lin, keep="int8")
    _, gw, db = torch.autograd.grad(y, (x, lin.weight, bn.bias), gy)
    beta = bn.bias.detach()
    _, codes, exps, _ = tr._bn8_forward(x.detach(), bn.weight.detach(), beta, None, None, bn.eps, 0.25, True, 0.0, None, None)
    zq = packed.unpack_rows(codes, exps)
    t = torch.where(zq > -beta, 1.0, 0.25)
    want, wb = torch.zeros_like(gw, dtype=torch.float64), torch.zeros_like(db, dtype=torch.float64)
    for k in range(0, x.shape[0], 1 << 18):
        part = slice(k, k + (1 << 18))
        want += over_rows(gy[part], (zq[part].double() + beta.double()) * t[part])
        wb += ((gy[part].double() @ lin.weight.detach().double()) * t[part]).sum(0)
    return [gw, db], [want, wb]


@pytest.mark.parametrize("op", ["linear", "block"])
@pytest.mark.parametrize("I,O", [(64, 64), (32, 32), (64, 40), (33, 9)])
def test_long_sums_of_one_sign(I, O, op):
    """2^23 positive terms a sum.  Its last rounding is u; a wave adds N = 256 parts (of 16 rows) to the nearest,
    each off by at most u of a sum that grows evenly: a deviation of u sqrt(N) / 3 of the wave's sum, and for the
    mean of 1024 waves or more 0.17 u; what the matrix instructions cut off, always downwards, odd and even waves
    turn opposite ways.  2 u leaves six deviations."""
    rows = 1 << 23
    torch.manual_seed(7)
    x = 1 + 0.2 * torch.randn(rows, I, device="cuda").abs_()
    gy = 0.5 + torch.rand(rows, O, device="cuda")
    lin, bn = torch.nn.Linear(I, O, bias=False).cuda(), torch.nn.BatchNorm1d(I).cuda()
    with torch.no_grad():
        lin.weight.abs_()
        bn.bias.fill_(2.5)
    for got, want in zip(*long_sums(op, x.requires_grad_(True), gy, lin, bn)):
        assert float(want.min()) > 0
        assert float(((got.double() - want) / want).abs().max()) <= 2 * U


@pytest.mark.parametrize("op", ["linear", "block"])
@pytest.mark.parametrize("I,O", [(64, 64), (64, 40), (33, 9)])
def test_long_sums_of_both_signs(I, O, op):
    """2 M terms of both signs: sums grow as the root of their terms, so N additions a wave leave a deviation of
    u sqrt(N / 6) of the result's spread: 1024 waves (two steps of 16 rows a tile) at least, N = 123 at most."""
    rows = 2_000_000
    torch.manual_seed(8)
    x, gy = torch.randn(rows, I, device="cuda", requires_grad=True), torch.randn(rows, O, device="cuda")
    lin, bn = torch.nn.Linear(I, O, bias=False).cuda(), torch.nn.BatchNorm1d(I).cuda()
    got, want = (t[0] for t in long_sums(op, x, gy, lin, bn))
    waves = 1024 if op == "block" and O > 32 and I % 8 == 0 else 2048
    n = 2 * rows / 32 / waves
    err, spread = got.double() - want, want.square().mean().sqrt()
    assert float(err.std()) <= ((n / 6) ** 0.5 + 1) * U * float(spread)
    assert abs(float(err.mean())) <= 0.5 * float(err.std())
