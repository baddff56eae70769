"""8-bit kept rows against float64: packing bit for bit; BatchNorm + LeakyReLU, Linear and both as a
block with gradients within the rounding of their float32 arithmetic.

Tolerances: u = 2^-24 is the rounding of one float32 operation relative to its result.  A result
made by k operations from terms t_i is off by at most about k u sum |t_i|; the tests form that sum
of magnitudes in float64 and count the operations."""
import numpy as np
import pytest
import torch

import kept_rows_reference as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
T = torch.from_numpy


def within(got, want, bound, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, what
    over = np.abs(got - want) - bound
    assert np.all(over <= 0), f"{what}: {np.abs(got - want).max()} against {np.max(bound)}"


# ---- packing -------------------------------------------------------------------------------------
KINDS = {"float32": (torch.float32, 254), "bfloat16": (torch.bfloat16, 254), "float16": (torch.float16, 142)}


def rows_of(rows, C, seed):
    g = np.random.default_rng(seed)
    x = g.normal(size=(rows, C)) * np.exp(g.normal(size=(1, C)))
    x[g.random((rows, C)) < 0.1] = 0
    return x.astype(np.float32)


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("rows,C", [(1, 1), (1, 64), (3, 5), (257, 33), (1000, 50), (33, 1024), (19, 1031), (5000, 32),
                                    (4099, 40), (2, 2500)])
def test_pack_rows(rows, C, kind):
    from mvfusion import packed
    dtype, most = KINDS[kind]
    x = T(rows_of(rows, C, rows + C)).to(dtype)
    codes, exps = ref.pack(x.float().numpy(), most)
    p = packed.pack_rows(x.cuda())
    assert p.shape == (rows, C) and p.dtype == dtype and p.nbytes == codes.size + exps.size
    assert np.array_equal(p.codes.cpu().numpy(), codes)
    assert np.array_equal(p.exps.cpu().numpy(), exps)
    back = p.unpack()
    assert back.dtype == dtype
    assert np.array_equal(back.cpu().double().numpy(), ref.unpack(codes, exps))
    # half a step, at most amax / 127.5
    wide = ref.spread(exps.astype(np.int64), C)
    within(back.cpu().float().numpy(), x.float().numpy(), np.ldexp(0.5, wide - ref.BIAS))


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_pack_special_values(kind):
    """Infinities and NaN, the largest and smallest numbers, ties, groups of nothing."""
    from mvfusion import packed
    dtype, most = KINDS[kind]
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    sub = tiny * torch.finfo(dtype).eps
    x = torch.zeros(10, 70)
    x[0, :4] = torch.tensor([float("inf"), 1.0, -2.5, float("nan")])
    x[1, :3] = torch.tensor([top, -top, 1.0])
    x[2, :3] = torch.tensor([tiny, -sub, 3 * sub])
    x[3, :] = float("nan")
    x[4, 32:64] = float("-inf")
    x[5, :8] = torch.tensor([127.5, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5])
    x[6, :4] = torch.tensor([127.75, 0.75, 1.0, -127.75])
    x[7, 69] = -64.0
    x[8, :33] = torch.linspace(-1, 1, 33)
    x = x.to(dtype)
    codes, exps = ref.pack(x.float().numpy(), most)
    p = packed.pack_rows(x.cuda())
    assert np.array_equal(p.codes.cpu().numpy(), codes)
    assert np.array_equal(p.exps.cpu().numpy(), exps)
    back = p.unpack().float().cpu().numpy()
    assert np.array_equal(back, ref.unpack(codes, exps).astype(np.float32), equal_nan=True)
    assert np.array_equal(np.isnan(back), ~np.isfinite(x.float().numpy()))


def test_pack_layouts():
    """No rows, rows that are not contiguous or not aligned, another stream."""
    from mvfusion import packed
    assert packed.pack_rows(torch.empty(0, 7, device="cuda")).unpack().shape == (0, 7)
    x = T(rows_of(130, 48, 5)).cuda()
    want = packed.pack_rows(x).unpack()
    assert torch.equal(packed.pack_rows(x.t().contiguous().t()).unpack(), want)
    assert torch.equal(packed.pack_rows(torch.cat([x, x], 1)[:, 48:]).unpack(), want)
    shifted = torch.empty(x.numel() + 1, device="cuda")[1:].view(130, 48)
    shifted.copy_(x)
    assert shifted.data_ptr() % 16 != 0
    assert torch.equal(packed.pack_rows(shifted).unpack(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = packed.pack_rows(x).unpack()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_pack_more_than_2_31_values():
    from mvfusion import packed
    rows, C = (1 << 31) // 64 + 37, 64
    x = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    last = T(rows_of(50, C, 9)).to(torch.bfloat16)
    x[-50:] = last.cuda()
    back = packed.pack_rows(x).unpack()
    assert torch.equal(back[-50:].cpu(), packed.pack_rows(last.cuda()).unpack().cpu())
    assert int(torch.count_nonzero(back[:1000])) == 0


def test_refused_rows():
    from mvfusion import packed
    with pytest.raises(TypeError):
        packed.pack_rows(torch.zeros(3, 4, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError):
        packed.pack_rows(torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        packed.pack_rows(torch.zeros(4, 0, device="cuda"))
    p = packed.pack_rows(torch.zeros(3, 40, device="cuda"))
    with pytest.raises(ValueError):
        packed.unpack_rows(p.codes, p.exps[:, :1])
    with pytest.raises(ValueError):
        packed.unpack_rows(p.codes.float(), p.exps)
    with pytest.raises(TypeError):
        p.unpack(torch.float64)


# ---- BatchNorm + LeakyReLU -----------------------------------------------------------------------
def bn_module(C, g, affine=True, training=True):
    bn = torch.nn.BatchNorm1d(C, momentum=0.1, affine=affine)
    if affine:
        gamma = (1 + 0.4 * g.normal(size=C)).astype(np.float32)
        gamma[g.random(C) < 0.3] *= -1
        beta = (0.4 * g.normal(size=C)).astype(np.float32)
        if C > 3:
            gamma[1] = gamma[2] = 0
            beta[1], beta[2] = 0.5, -0.5
            beta[3] = 0
        bn.weight.data, bn.bias.data = T(gamma), T(beta)
    bn.running_mean.copy_(T(g.normal(size=C).astype(np.float32)))
    bn.running_var.copy_(T((0.5 + g.random(C)).astype(np.float32)))
    return bn.cuda().train(training)


def bn_reference(z, bn, act, training):
    """(zq, on, gamma, beta, invstd) of the float64 restatement."""
    C = z.shape[1]
    gamma = np.ones(C) if bn.weight is None else bn.weight.detach().cpu().double().numpy()
    beta = np.zeros(C) if bn.bias is None else bn.bias.detach().cpu().double().numpy()
    if training:
        mean, invstd = ref.bn_stats(z, bn.eps)
    else:
        mean = bn.running_mean.cpu().double().numpy()
        invstd = 1 / np.sqrt(bn.running_var.cpu().double().numpy() + np.float64(np.float32(bn.eps)))
    codes, exps = ref.bn_pack(z, mean, invstd, gamma, beta, act)
    zq = ref.unpack(codes, exps)
    return codes, exps, zq, ref.bn_on(zq, gamma, beta), gamma, beta, invstd


def bn_backward_reference(gy, err, zq, on, gamma, invstd, act, slope, training):
    """Gradients from gy (known to err) and their bounds."""
    f = np.where(on, 1.0, slope) if act else np.ones_like(gy)
    g, e = gy * f, (err + 2 * U * np.abs(gy)) * np.abs(f)
    n = g.shape[0]
    db, dw = g.sum(0), (g * zq).sum(0)
    # float64 sums of float32 terms: the terms' own error, and one rounding
    e_db, e_dw = e.sum(0) + U * np.abs(db), (e * np.abs(zq)).sum(0) + U * np.abs(dw)
    k = gamma * invstd
    if not training:
        return g * k, (e + 4 * U * np.abs(g)) * np.abs(k), dw, e_dw, db, e_db
    gz = (g - db / n - zq * dw / n) * k
    mag = np.abs(g) + np.abs(db) / n + np.abs(zq * dw) / n
    bound = (e + e_db / n + np.abs(zq) * e_dw / n + 8 * U * mag) * np.abs(k)
    return gz, bound, dw, e_dw, db, e_db


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("act", [True, False])
@pytest.mark.parametrize("rows,C,affine", [(2, 4, True), (17, 1, True), (300, 33, True), (1025, 64, True),
                                           (4099, 50, True), (20011, 32, False), (130, 300, True), (40, 1100, True)])
def test_batch_norm_act(rows, C, affine, act, training):
    from mvfusion import training as tr
    g = np.random.default_rng(rows + C)
    z = (g.normal(size=(rows, C)) * np.exp(0.7 * g.normal(size=C)) + g.normal(size=C)).astype(np.float32)
    gy = g.normal(size=(rows, C)).astype(np.float32)
    bn = bn_module(C, g, affine, training)
    slope = 0.2
    layer = torch.nn.LeakyReLU(slope) if act else torch.nn.Identity()
    codes, exps, zq, on, gamma, beta, invstd = bn_reference(z.astype(np.float64), bn, act, training)
    before = {k: v.clone() for k, v in bn.state_dict().items()}
    got = {}
    for keep in ("float32", "int8"):
        bn.load_state_dict(before)
        zt = T(z).cuda().requires_grad_(True)
        leaves = [zt] + list(bn.parameters())
        y = tr.batch_norm_act(zt, bn, layer, keep=keep)
        if keep == "int8":
            saved = y.grad_fn.saved_tensors if act else y.grad_fn.saved_tensors
            assert np.array_equal(saved[1].cpu().numpy(), exps)
            assert np.array_equal(saved[0].cpu().numpy(), codes)
        got[keep] = (y, torch.autograd.grad(y, leaves, T(gy).cuda()), {k: v.clone() for k, v in bn.state_dict().items()})
    assert torch.equal(got["int8"][0], got["float32"][0])
    for k, v in got["float32"][2].items():
        assert torch.equal(v, got["int8"][2][k]), k
    gz, bound, dw, e_dw, db, e_db = bn_backward_reference(
        gy.astype(np.float64), 0.0, zq, on, gamma, invstd, act, slope, training)
    grads = [t.cpu().numpy() for t in got["int8"][1]]
    within(grads[0], gz, bound, "z")
    if affine:
        within(grads[1], dw, e_dw, "gamma")
        within(grads[2], db, e_db, "beta")


def test_kept_side_of_the_kink():
    """Values close to the kink read back on their own side of it, at most one step away."""
    from mvfusion import training as tr
    g = np.random.default_rng(3)
    rows, C = 6000, 32
    z = g.normal(size=(rows, C)).astype(np.float32)
    bn = bn_module(C, g, True, False)
    with torch.no_grad():
        bn.running_mean.zero_()
        bn.running_var.fill_(1)
    gamma, beta = bn.weight.detach().cpu().double().numpy(), bn.bias.detach().cpu().double().numpy()
    invstd = 1 / np.sqrt(1 + np.float64(np.float32(bn.eps)))
    with np.errstate(divide="ignore", invalid="ignore"):
        kink = np.where(gamma != 0, -beta / gamma, 0)
    near = g.random((rows, C)) < 0.5
    z = np.where(near, kink / invstd + g.normal(size=(rows, C)) * 10.0 ** g.integers(-7, -1, (rows, C)), z).astype(np.float32)
    zt = T(z).cuda().requires_grad_(True)
    y = tr.batch_norm_act(zt, bn, torch.nn.LeakyReLU(0.1), keep="int8")
    codes, exps = (t.cpu().numpy() for t in y.grad_fn.saved_tensors[:2])
    zq = ref.unpack(codes, exps)
    on = gamma * (z.astype(np.float64) * invstd) + beta > 0
    assert np.array_equal(ref.bn_on(zq, gamma, beta), on)
    assert np.all(np.abs(zq - z.astype(np.float64) * invstd) <= np.ldexp(1.0, ref.spread(exps.astype(np.int64), C) - 133))
    plain = np.abs(zq - z.astype(np.float64) * invstd) > np.ldexp(0.5, ref.spread(exps.astype(np.int64), C) - 133)
    assert 0 < plain.sum() < 0.5 * near.sum()


def test_batch_norm_act_not_finite_rows():
    """Outside train mode a value that is not finite stays with itself: NaN reads back, every other
    gradient of z is that of the finite values."""
    from mvfusion import training as tr
    g = np.random.default_rng(4)
    z = g.normal(size=(50, 40)).astype(np.float32)
    bn = bn_module(40, g, True, False)
    gy = T(g.normal(size=(50, 40)).astype(np.float32)).cuda()

    def step(v):
        zt = T(v).cuda().requires_grad_(True)
        return torch.autograd.grad(tr.batch_norm_act(zt, bn, torch.nn.LeakyReLU(0.2), keep="int8"), zt, gy)[0]
    clean = step(z)
    z[3, 5], z[20, 39], z[21, 0] = np.inf, np.nan, -np.inf
    got = step(z)
    bad = torch.zeros(50, 40, dtype=torch.bool)
    bad[3, :32] = bad[20, 32:] = bad[21, :32] = True        # (their groups may have another step)
    assert torch.equal(got[~bad.cuda()], clean[~bad.cuda()])
    assert torch.isfinite(got).all()


# ---- Linear and the block ------------------------------------------------------------------------
def xty_bound(a, b, rows):
    """Bound of sum |a||b| roundings of the kernels: per wave and step of 16 rows up to six matrix
    instructions, each one rounding of the running sum and about 16 inside; a workgroup of four waves
    has at least 128 rows (256 workgroups at most), so a wave takes at most
    ceil(rows / (16 * 4 * workgroups)) + 1 steps."""
    wgs = min(256, -(-rows // 256))
    steps = -(-rows // (64 * wgs)) + 1
    return (6 * steps + 16 + 4) * U * (np.abs(a).T @ np.abs(b))


def same_kernel(lin, y8, y32):
    """From 4096 rows on both forms run the same product where mvf_linear_rows takes the shape."""
    from mvfusion import _lib
    if y8.shape[0] >= 4096 and _lib.load().mvf_linear_rows_supported(lin.in_features, lin.out_features):
        assert torch.equal(y8, y32)


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("rows,I,O", [(1, 8, 8), (31, 64, 64), (33, 16, 24), (4097, 64, 64), (40001, 32, 32), (5000, 8, 40),
                                      (4128, 64, 8), (1, 8, 4), (15, 5, 3), (16, 32, 32), (33, 64, 64), (257, 40, 48), (1000, 33, 65),
                                      (4099, 64, 32), (9000, 7, 63), (5000, 50, 34), (700, 200, 130)])
def test_linear(rows, I, O, bias):
    from mvfusion import training as tr
    g = np.random.default_rng(rows + I + O)
    lin = torch.nn.Linear(I, O, bias=bias).cuda()
    x = (g.normal(size=(rows, I)) * np.exp(g.normal(size=I))).astype(np.float32)
    gy = (g.normal(size=(rows, O)) * np.exp(2 * g.normal(size=(rows, 1)))).astype(np.float32)
    xt = T(x).cuda().requires_grad_(True)
    leaves = [xt, lin.weight] + ([lin.bias] if bias else [])
    y = tr.linear(lin, xt, keep="int8")
    grads = torch.autograd.grad(y, leaves, T(gy).cuda())
    same_kernel(lin, y, tr.linear(lin, xt, keep="float32"))
    xq = ref.unpack(*ref.pack(x))
    g64, x64, w64 = gy.astype(np.float64), x.astype(np.float64), lin.weight.detach().cpu().double().numpy()
    b64 = lin.bias.detach().cpu().double().numpy() if bias else np.zeros(O)
    within(y.detach().cpu().numpy(), x64 @ w64.T + b64, (I + 2) * U * (np.abs(x64) @ np.abs(w64).T + np.abs(b64)), "y")
    within(grads[0].cpu().numpy(), g64 @ w64, (O + 2) * U * (np.abs(g64) @ np.abs(w64)), "x")
    within(grads[1].cpu().numpy(), g64.T @ xq, xty_bound(g64, xq, rows), "weight")
    if bias:
        steps = -(-rows // 64) + 12
        within(grads[2].cpu().numpy(), g64.sum(0), min(steps, 64) * U * np.abs(g64).sum(0), "bias")


def test_linear_same_bits_and_layouts():
    from mvfusion import training as tr
    g = np.random.default_rng(8)
    lin = torch.nn.Linear(64, 48).cuda()
    x = T(g.normal(size=(5001, 64)).astype(np.float32)).cuda().requires_grad_(True)
    gy = T(g.normal(size=(5001, 48)).astype(np.float32)).cuda()
    first = torch.autograd.grad(tr.linear(lin, x, keep="int8"), (lin.weight, lin.bias), gy)
    for grad in (gy.clone(), gy.t().contiguous().t(), torch.cat([gy, gy], 1)[:, 48:]):
        again = torch.autograd.grad(tr.linear(lin, x, keep="int8"), (lin.weight, lin.bias), grad)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    # a gradient that is one value everywhere (expanded, stride 0)
    y = tr.linear(lin, x, keep="int8")
    (gw,) = torch.autograd.grad(y.sum(), lin.weight)
    xq = ref.unpack(*ref.pack(x.detach().cpu().numpy()))
    ones = np.ones((5001, 48))
    within(gw.cpu().numpy(), ones.T @ xq, xty_bound(ones, xq, 5001))
    # only one of the gradients, and none of the weight
    (gb,) = torch.autograd.grad(tr.linear(lin, x, keep="int8"), lin.bias, gy)
    assert torch.allclose(gb, first[1], rtol=0, atol=float(64 * U * gy.abs().sum(0).max()))
    lin.weight.requires_grad_(False)
    y = tr.linear(lin, x, keep="int8")
    assert y.grad_fn.saved_tensors[0] is None
    gx, gb = torch.autograd.grad(y, (x, lin.bias), gy)
    assert torch.equal(gx, torch.autograd.grad(tr.linear(lin, x, keep="float32"), x, gy)[0])


def test_linear_gradient_magnitudes():
    """Gradients from the smallest to large numbers, and zeros: bf16 parts lose nothing."""
    from mvfusion import training as tr
    g = np.random.default_rng(10)
    lin = torch.nn.Linear(32, 40, bias=False).cuda()
    x = g.normal(size=(2000, 32)).astype(np.float32)
    for power in (-30, -8, 0, 20, 30):
        gy = (g.normal(size=(2000, 40)) * 10.0 ** power).astype(np.float32)
        gy[::3] = 0
        xt = T(x).cuda().requires_grad_(True)
        (gw,) = torch.autograd.grad(tr.linear(lin, xt, keep="int8"), lin.weight, T(gy).cuda())
        xq = ref.unpack(*ref.pack(x))
        g64 = gy.astype(np.float64)
        within(gw.cpu().numpy(), g64.T @ xq, xty_bound(g64, xq, 2000), str(power))


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("rows,I,O,bias", [(16, 8, 4, False), (250, 33, 20, True), (1031, 64, 64, False), (5003, 32, 48, True),
                                           (31, 64, 8, True), (4096, 8, 16, False), (4129, 64, 64, True), (30011, 32, 32, False),
                                           (65, 16, 40, True), (4500, 16, 33, False), (600, 100, 70, True)])
def test_block(rows, I, O, bias, training):
    """BatchNorm + LeakyReLU + Linear from one packed copy of the normalised rows."""
    from mvfusion import training as tr
    g = np.random.default_rng(rows + I)
    z = (g.normal(size=(rows, I)) * np.exp(0.7 * g.normal(size=I)) + g.normal(size=I)).astype(np.float32)
    go = g.normal(size=(rows, O)).astype(np.float32)
    bn = bn_module(I, g, True, training)
    lin = torch.nn.Linear(I, O, bias=bias).cuda()
    act, slope = torch.nn.LeakyReLU(0.2), 0.2
    _, _, zq, on, gamma, beta, invstd = bn_reference(z.astype(np.float64), bn, True, training)
    zt = T(z).cuda().requires_grad_(True)
    before = {k: v.clone() for k, v in bn.state_dict().items()}
    y32 = tr.batch_norm_act_linear(zt, bn, act, lin, keep="float32")
    after = {k: v.clone() for k, v in bn.state_dict().items()}
    bn.load_state_dict(before)
    y = tr.batch_norm_act_linear(zt, bn, act, lin, keep="int8")
    same_kernel(lin, y, y32)
    assert all(torch.equal(v, after[k]) for k, v in bn.state_dict().items())
    leaves = [zt, bn.weight, bn.bias, lin.weight] + ([lin.bias] if bias else [])
    grads = [t.cpu().numpy() for t in torch.autograd.grad(y, leaves, T(go).cuda())]
    go64, w = go.astype(np.float64), lin.weight.detach().cpu().double().numpy()
    zh = (z.astype(np.float64) - (ref.bn_stats(z.astype(np.float64), bn.eps)[0] if training
                                  else bn.running_mean.cpu().double().numpy())) * invstd
    a = zh * gamma + beta
    act64 = np.where(a > 0, a, slope * a)
    # four roundings of the normalised value (its mean and spread among them), then the product's
    mag = (np.abs(zh) + np.abs(z - zh / invstd) * invstd + np.abs(z) * invstd) * np.abs(gamma) + np.abs(beta)
    b64 = lin.bias.detach().cpu().double().numpy() if bias else np.zeros(O)
    within(y.detach().cpu().numpy(), act64 @ w.T + b64, (I + 8) * U * (mag @ np.abs(w).T + np.abs(b64)), "y")
    gy = go64 @ w
    err = (O + 2) * U * (np.abs(go64) @ np.abs(w))
    gz, bound, dw, e_dw, db, e_db = bn_backward_reference(gy, err, zq, on, gamma, invstd, True, slope, training)
    within(grads[0], gz, bound, "z")
    within(grads[1], dw, e_dw, "gamma")
    within(grads[2], db, e_db, "beta")
    a = zq * gamma + beta
    yq = np.where(on, a, slope * a)
    # the activated value itself: three roundings of float32
    mag = np.abs(zq * gamma) + np.abs(beta)
    within(grads[3], go64.T @ yq, xty_bound(go64, yq, rows) + 4 * U * (np.abs(go64).T @ mag), "weight")
    if bias:
        within(grads[4], go64.sum(0), 64 * U * np.abs(go64).sum(0), "bias")


def test_gradients_against_differences():
    """The Linear's weight gradient on rows that 8 bits hold exactly, against differences of the
    loss (linear in the weight, so any step is exact up to rounding), and the tail's gradient of z on
    rows whose normalised values are codes."""
    from mvfusion import training as tr
    g = np.random.default_rng(12)
    x = (g.integers(-127, 128, (64, 32)) / 64).astype(np.float32)
    x[:, 0] = 127 / 64
    lin = torch.nn.Linear(32, 8).cuda()
    v = T(g.normal(size=(64, 8)).astype(np.float32)).cuda()
    xt = T(x).cuda().requires_grad_(True)
    (gw,) = torch.autograd.grad((tr.linear(lin, xt, keep="int8") * v).sum(), lin.weight)
    w, step = lin.weight.detach().double(), T(g.normal(size=(8, 32))).cuda()
    loss = lambda p: float(((T(x).cuda().double() @ p.t()) * v.double()).sum())  # noqa: E731
    diff = (loss(w + step) - loss(w - step)) / 2
    assert abs(float((gw.double() * step).sum()) - diff) <= 100 * U * float((gw.double().abs() * step.abs()).sum() + 1)
    # eval mode: zhat = z * invstd with invstd a power of two
    bn = torch.nn.BatchNorm1d(32, eps=0.0).cuda().eval()
    with torch.no_grad():
        bn.weight.copy_(T(g.normal(size=32).astype(np.float32)))
        bn.bias.copy_(T(g.normal(size=32).astype(np.float32)))
        bn.running_var.fill_(0.25)
    act = torch.nn.LeakyReLU(0.3)
    (gz,) = torch.autograd.grad((tr.batch_norm_act(xt, bn, act, keep="int8")[:, :8] * v).sum(), xt)
    w64, b64 = (t.detach().cpu().double() for t in (bn.weight, bn.bias))
    z64, d = T(x).double(), T(g.normal(size=(64, 32)))
    f = lambda z: float((act(z * 2 * w64 + b64)[:, :8] * v.cpu().double()).sum())  # noqa: E731
    h = 1e-7        # far below the distance of any value from its kink
    diff = (f(z64 + h * d) - f(z64 - h * d)) / (2 * h)
    assert abs(float((gz.cpu().double() * d).sum()) - diff) <= 1e-6 * float((gz.cpu().double().abs() * d.abs()).sum())


# ---- the path ------------------------------------------------------------------------------------
def make_pool(seed=0):
    from mvfusion.pooling import QKVBimodalCSRPool
    torch.manual_seed(seed)
    return QKVBimodalCSRPool(in_main=24, in_map=8, in_mod=64, nc_qk=8, num_groups=4).cuda().train()


def pool_inputs(points=6000, seed=1):
    g = np.random.default_rng(seed)
    sizes = g.poisson(4, points)
    sizes[g.random(points) < 0.2] = 0
    ptr = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
    V = int(ptr[-1])
    x = [T(g.normal(size=s).astype(np.float32)).cuda().requires_grad_(True) for s in ((points, 24), (V, 64), (V, 8))]
    return x, T(ptr).cuda()


def relative(a, b):
    return float((a - b).double().norm() / b.double().norm().clamp_min(1e-30))


def test_pool_training_step_with_kept_rows():
    """A training step of the attentive pool: the same outputs and running statistics, gradients
    close to those of float32 rows (half a step of 1 / 64 of a group's largest value, about 1 % of a
    value's spread, enters every weight gradient once), and less memory held for the backward."""
    from mvfusion import training as tr
    x, ptr = pool_inputs()
    res = {}
    for keep in ("float32", "int8"):
        pool = make_pool()
        with tr.keep_activations(keep):
            out = pool(x[0], x[1], x[2], ptr)
        w = torch.linspace(-1, 1, out.numel(), device="cuda").view_as(out)
        grads = torch.autograd.grad((out * w).sum(), x + [p for p in pool.parameters()])
        res[keep] = out.detach(), grads, pool.state_dict()
    assert torch.equal(res["int8"][0], res["float32"][0])
    for k, v in res["float32"][2].items():
        if "running" in k or "num_batches" in k:
            assert torch.equal(v, res["int8"][2][k]), k
    for a, b in zip(res["int8"][1], res["float32"][1]):
        assert relative(a, b) < 0.05 or float(b.norm()) < 1e-4 * float(res["float32"][1][0].norm())


def test_mlp_keeps_less_memory():
    from mvfusion import training as tr
    from mvfusion.dense import MLP
    torch.manual_seed(0)
    seq = MLP([64, 64, 64, 64], bias=False).cuda().train()
    x = torch.randn(40000, 64, device="cuda")
    held = {}
    for keep in ("float32", "int8"):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with tr.keep_activations(keep):
            y = tr.mlp(seq, x)
        held[keep] = torch.cuda.memory_allocated() - before - 4 * y.numel()
        y.sum().backward()
        del y
    rows = 40000 * 64
    # float32: the inputs of three BatchNorms and of two Linears beside x; int8: four packed rows
    assert held["float32"] >= 5 * 4 * rows
    assert held["int8"] <= 4 * (rows + rows // 32) + (1 << 16)


def test_step_in_a_graph():
    """A captured training step, replayed with eager work between the replays, gives the eager
    step's gradients every time."""
    from mvfusion import training as tr
    from mvfusion.dense import MLP
    torch.manual_seed(0)
    seq = MLP([32, 64, 48], bias=False).cuda().train()
    x = torch.randn(5000, 32, device="cuda")
    gy = torch.randn(5000, 48, device="cuda")
    params = list(seq.parameters())

    def step():
        with tr.keep_activations("int8"):
            y = tr.mlp(seq, x)
        grads = torch.autograd.grad(y, params, gy)
        return (y.detach(),) + grads        # (no eager graph of the same leaves may live during a capture)
    state = {k: v.clone() for k, v in seq.state_dict().items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    seq.load_state_dict(state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        x.copy_(torch.randn(5000, 32, device="cuda"))
        seq.load_state_dict(state)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        stats = {n: v.clone() for n, v in seq.state_dict().items()}
        seq.load_state_dict(state)
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k
        assert all(torch.equal(v, stats[n]) for n, v in seq.state_dict().items()), k


def test_two_steps_on_two_streams():
    from mvfusion import training as tr
    lin = torch.nn.Linear(64, 64).cuda()
    xs = [torch.randn(30000, 64, device="cuda", requires_grad=True) for _ in range(2)]
    gy = torch.randn(30000, 64, device="cuda")
    want = [torch.autograd.grad(tr.linear(lin, x, keep="int8"), lin.weight, gy)[0] for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            got.append(torch.autograd.grad(tr.linear(lin, x, keep="int8"), lin.weight, gy)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("I,O", [(64, 64), (64, 40), (16, 56), (32, 8), (8, 24), (33, 9)])
@pytest.mark.parametrize("act", [True, False])
def test_block_kinks_and_nan(I, O, act):
    """Scales of both signs and zero, shifts that put whole columns on one side, rows of NaN and infinities
    (eval mode), against the formulas on the same codes in float64.

    A sum of 3000 rows is made of at most 6 matrix instructions a tile and 2 tiles a wave, each cutting
    16 products and the sum off at a step of the largest (17 steps of 2 u), joined by 8 float32
    additions and in float64: 12 * 34 + 8 < 512 u of the magnitudes."""
    from mvfusion import packed, training as tr
    rows = 3001
    g = np.random.default_rng(I + O)
    gamma, beta = g.normal(size=I), g.normal(size=I)
    gamma[::5], gamma[3::7], beta[4::6] = 0.0, -gamma[3::7], 9.0 * np.sign(beta[4::6])
    gamma, beta = gamma.astype(np.float32), beta.astype(np.float32)
    z = rows_of(rows, I, 11)
    z[5, 1], z[900, I - 1], z[rows - 1, 2] = np.nan, np.inf, -np.inf
    bad = [1, I - 1, 2]
    bn, lin = torch.nn.BatchNorm1d(I).cuda().eval(), torch.nn.Linear(I, O).cuda()
    with torch.no_grad():
        bn.weight.copy_(T(gamma))
        bn.bias.copy_(T(beta))
    slope = 0.25 if act else 1.0
    x = T(z).cuda().requires_grad_(True)
    gy = T(g.normal(size=(rows, O)).astype(np.float32)).cuda()
    y = tr.batch_norm_act_linear(x, bn, torch.nn.LeakyReLU(slope), lin, keep="int8")
    gx, dgamma, dbeta, dw, db = torch.autograd.grad(y, (x, bn.weight, bn.bias, lin.weight, lin.bias), gy)
    _, codes, exps, invstd = tr._bn8_forward(x.detach(), bn.weight.detach(), bn.bias.detach(), bn.running_mean,
                                             bn.running_var, bn.eps, slope, False, 0.0, None, None)
    zq = packed.unpack_rows(codes, exps).double().cpu().numpy()
    on = ref.bn_on(zq, gamma, beta)
    t = np.where(on, 1.0, slope)
    g64, w64 = gy.double().cpu().numpy(), lin.weight.detach().double().cpu().numpy()
    gh = t * (g64 @ w64)
    v = t * (gamma.astype(np.float64) * zq + beta)
    good = np.setdiff1d(np.arange(I), bad)
    within(dw.cpu().numpy()[:, good], (g64.T @ v)[:, good],
           512 * U * (np.abs(g64).T @ (np.abs(gamma * zq) + np.abs(beta)))[:, good], "dw")
    assert torch.isnan(dw[:, bad]).all() and torch.isnan(dgamma[bad]).all()
    within(db.cpu().numpy(), g64.sum(0), 512 * U * np.abs(g64).sum(0), "db")
    mag = np.abs(g64) @ np.abs(w64)
    within(dbeta.cpu().numpy(), gh.sum(0), 512 * U * mag.sum(0), "dbeta")
    within(dgamma.cpu().numpy()[good], (gh * zq).sum(0)[good], 512 * U * (mag * np.abs(zq)).sum(0)[good], "dgamma")
    k = gamma.astype(np.float64) * invstd.cpu().double().numpy()
    within(gx.cpu().numpy(), gh * k, 512 * U * mag * np.abs(k), "gx")


@pytest.mark.parametrize("O", [64, 60])
@pytest.mark.parametrize("tail", [False, True])
def test_weight_gradient_has_no_common_shift(tail, O):
    """Sums of many zero-mean terms: the matrix cores' rounding, which goes one way, must not move all of
    them together.  The errors of the 64 O sums share 64 and O columns, so the mean of unbiased
    ones is within about std / 7.7 of zero; half the deviation is nearly four times that."""
    from mvfusion import training as tr
    rows = 1 << 20
    torch.manual_seed(5)
    lin, bn, act = torch.nn.Linear(64, O).cuda(), torch.nn.BatchNorm1d(64).cuda(), torch.nn.LeakyReLU(0.2)
    x, gy = torch.randn(rows, 64, device="cuda", requires_grad=True), torch.randn(rows, O, device="cuda")
    y = tr.batch_norm_act_linear(x, bn, act, lin, keep="int8") if tail else tr.linear(lin, x, keep="int8")
    _, gw = torch.autograd.grad(y, (x, lin.weight), gy)
    from mvfusion import packed
    if tail:
        _, codes, exps, _ = tr._bn8_forward(x.detach(), bn.weight.detach(), bn.bias.detach(), None, None, bn.eps, 0.2,
                                            True, 0.0, None, None)
        v = packed.unpack_rows(codes, exps).double()
        v = torch.where(v > 0, v, v * float(np.float32(0.2)))
    else:
        v = packed.pack_rows(x).unpack().double()
    g = gy.double().view(-1, 512, O).transpose(1, 2).contiguous()
    err = gw.double() - torch.bmm(g, v.view(-1, 512, 64)).sum(0)
    assert abs(float(err.mean())) <= 0.5 * float(err.std())


@pytest.mark.parametrize("op,I,O", [("linear", 64, 64), ("linear", 65, 8), ("tail", 65, 0), ("block", 64, 64), ("block", 65, 8)])
def test_more_than_2_31_values(op, I, O):
    """The last 5000 of 2^25 and some rows as a call on them alone has them.  The other rows' gradients
    are zeros, which leaves the last rows' in the sums: both calls add the same 5000 terms a column,
    each off by 5000 u of their magnitudes at most, and the codes of both are the same."""
    from mvfusion import training as tr
    rows, last = (1 << 25) + 77, 5000
    torch.manual_seed(3)
    lin = torch.nn.Linear(I, O).cuda() if O else None
    bn = torch.nn.BatchNorm1d(I).cuda().eval()
    with torch.no_grad():
        bn.weight.uniform_(0.5, 2)
        bn.bias.uniform_(-1, 1)
        bn.running_mean.uniform_(-1, 1)
        bn.running_var.uniform_(0.5, 2)
    act = torch.nn.LeakyReLU(0.2)
    call = {"linear": lambda x: tr.linear(lin, x, keep="int8"),
            "tail": lambda x: tr.batch_norm_act(x, bn, act, keep="int8"),
            "block": lambda x: tr.batch_norm_act_linear(x, bn, act, lin, keep="int8")}[op]
    params = ([] if op == "linear" else [bn.weight, bn.bias]) + ([lin.weight, lin.bias] if O else [])
    x = torch.randn(rows, I, device="cuda", requires_grad=True)
    gy = torch.zeros(rows, O or I, device="cuda")
    gy[-last:].normal_()
    y = call(x)
    gx, *sums = torch.autograd.grad(y, [x] + params, gy)
    xl = x.detach()[-last:].clone().requires_grad_(True)
    yl = call(xl)
    gxl, *suml = torch.autograd.grad(yl, [xl] + params, gy[-last:])
    assert torch.equal(y[-last:], yl)
    assert torch.equal(gx[-last:], gxl)
    assert not gx[:1000].any() and not gx[-last - 1000:-last].any()
    mag = gy[-last:].abs().double().sum(0).max() * xl.detach().abs().double().max().clamp_min(1) * 4
    if op == "block":       # (BatchNorm's sums: of g W, at most the sum of the weights' magnitudes more)
        mag = mag * lin.weight.detach().abs().double().sum(0).max().clamp_min(1)
    for a, b in zip(sums, suml):
        assert float((a - b).abs().max()) <= 2 * last * U * float(mag)


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_block(reentrant):
    """A block that is run again during the backward, on autograd's thread, sets the form itself."""
    from torch.utils.checkpoint import checkpoint
    from mvfusion import training as tr
    lin, bn, act = torch.nn.Linear(64, 32).cuda(), torch.nn.BatchNorm1d(64).cuda().eval(), torch.nn.LeakyReLU(0.2)

    def block(x):
        with tr.keep_activations("int8"):
            return tr.batch_norm_act_linear(x, bn, act, lin)
    x = torch.randn(5000, 64, device="cuda", requires_grad=True)
    params = [x, bn.weight, bn.bias, lin.weight, lin.bias]
    gy = torch.randn(5000, 32, device="cuda")
    want = torch.autograd.grad(block(x), params, gy)
    checkpoint(block, x, use_reentrant=reentrant).backward(gy)
    assert all(torch.equal(p.grad, w) for p, w in zip(params, want))


def test_what_autograd_refuses():
    """No second derivative, and no parameter changed between forward and backward."""
    from mvfusion import training as tr
    lin = torch.nn.Linear(8, 8).cuda()
    x = torch.randn(20, 8, device="cuda", requires_grad=True)
    y = tr.linear(lin, x, keep="int8")
    (gx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
    bn = torch.nn.BatchNorm1d(8).cuda()
    y = tr.batch_norm_act(x, bn, torch.nn.LeakyReLU(0.2), keep="int8")
    with torch.no_grad():
        bn.weight.mul_(2)
    with pytest.raises(RuntimeError):
        y.sum().backward()
    with pytest.raises(ValueError):
        tr.batch_norm_act(x[:1], bn.train(), torch.nn.LeakyReLU(0.2), keep="int8")


def test_inputs_the_kernels_do_not_take():
    """Modules take over as without kept rows: no graph, other types, other activations."""
    from mvfusion import training as tr
    bn = torch.nn.BatchNorm1d(16).cuda()
    x = torch.randn(40, 16, device="cuda", requires_grad=True)
    with torch.no_grad():
        assert tr.batch_norm_act(x, bn, torch.nn.LeakyReLU(0.2), keep="int8").grad_fn is None
    xd = x.detach().double().requires_grad_(True)
    lin = torch.nn.Linear(16, 4).double().cuda()
    y = tr.linear(lin, xd, keep="int8")
    assert y.dtype == torch.float64
    y.sum().backward()
    y = tr.batch_norm_act_linear(x, bn, torch.nn.GELU(), torch.nn.Linear(16, 4).cuda(), keep="int8")
    y.sum().backward()
    assert torch.isfinite(x.grad).all()
