"""The gated residual norm against float64.

Tolerances: u = 2^-24 is the rounding of one float32 operation.  kept_rows_reference.Residual forms
for every result the sum of the magnitudes it is made of, the statistics' errors included; a value
passes through at most about 64 operations (a lane's up to 16 channels, 8 exchanges, the
statistics and the products, both norms), column sums through as many rows of a lane before
they are folded in float64.  16-bit results have one rounding more, finfo(t).eps / 2 of the value
(half the smallest step below the normal range)."""
import itertools

import numpy as np
import pytest
import torch

import kept_rows_reference as ref

pytestmark = pytest.mark.gpu
U = 64 * 2.0 ** -24
T = torch.from_numpy
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
MOST = {"float32": 254, "bfloat16": 254, "float16": 142}


def norm_module(kind, C, g, eps=1e-5):
    if kind is None:
        return None
    m = (torch.nn.RMSNorm if kind == "rms" else torch.nn.LayerNorm)(C, eps=eps)
    m.weight.data = T((1 + 0.3 * g.normal(size=C)).astype(np.float32))
    if kind == "layer":
        m.bias.data = T((0.3 * g.normal(size=C)).astype(np.float32))
    return m.cuda()


def norm_ref(m):
    if m is None:
        return None
    d = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    return ("layer" if isinstance(m, torch.nn.LayerNorm) else "rms", d(m.weight), d(getattr(m, "bias", None)), m.eps)


def rounding(dtype, want):
    if dtype == torch.float32:
        return 0.0
    f = torch.finfo(dtype)
    return want.abs().clamp_min(f.smallest_normal) * (f.eps / 2)


def within(got, want, mag, what, u=U):
    want = want.double()
    bound = u * mag
    if got.dtype != torch.float32:
        bound = bound + rounding(got.dtype, want) * (1 + u)
    over = (got.detach().cpu().double() - want).abs() - bound
    assert torch.isfinite(got).all(), what
    assert float(over.max()) <= 0 if over.numel() else True, f"{what}: over by {float(over.max())}"


def make(rows, C, kind, post, pre, G, scale, seen, seed=0):
    g = np.random.default_rng(seed + rows * 7 + C)
    dt = TYPES[kind]
    s = {}
    spread = np.exp(0.5 * g.normal(size=C))
    s["x"] = T((g.normal(size=(rows, C)) * spread + 0.5).astype(np.float32)).to(dt).cuda().requires_grad_(True)
    s["f"] = T((g.normal(size=(rows, C)) * spread - 0.3).astype(np.float32)).to(dt).cuda().requires_grad_(True)
    s["gate"] = None if G == 0 else T(g.random((rows, G)).astype(np.float32)).cuda().requires_grad_(True)
    s["scale"] = T((0.4 + 0.2 * g.normal(size=C)).astype(np.float32)).cuda().requires_grad_(True) if scale else None
    s["seen"] = T(g.random(rows) > 0.3).cuda() if seen else None
    s["post"], s["pre"] = norm_module(post, C, g), norm_module(pre, C, g)
    s["d_out"] = T(g.normal(size=(rows, C)).astype(np.float32)).to(dt).cuda()
    s["d_h"] = T(g.normal(size=(rows, C)).astype(np.float32)).to(dt).cuda()
    return s


def f64(t):
    return None if t is None else t.detach().cpu().double()


def reference(s, kind, keep):
    x, f = f64(s["x"]), f64(s["f"])
    xq = fq = None
    if keep == "int8":
        xq, fq = (T(ref.unpack(*ref.pack(t.float().numpy(), MOST[kind]))) for t in (x, f))
    return ref.Residual(x, f, xq, fq, norm_ref(s["post"]), norm_ref(s["pre"]), f64(s["gate"]), f64(s["scale"]),
                        None if s["seen"] is None else s["seen"].cpu())


def run(s, keep):
    from mvfusion.residual import residual_norm
    got = residual_norm(s["x"], s["f"], post=s["post"], pre=s["pre"], gate=s["gate"], scale=s["scale"], seen=s["seen"],
                        keep=keep)
    return got if s["pre"] is not None else (got, None)


def check(s, kind, keep, use=(True, True)):
    out, h = run(s, keep)
    r = reference(s, kind, keep)
    within(out, r.out, r.M_out, "out")
    if h is not None:
        within(h, r.h, r.M_h, "h")
    pairs = [(o, d) for o, d, u in ((out, s["d_out"], use[0]), (h, s["d_h"], use[1])) if o is not None and u]
    names = {"x": s["x"], "f": s["f"], "gate": s["gate"], "scale": s["scale"]}
    for n in ("post", "pre"):
        if s[n] is not None:
            names["w_" + n] = s[n].weight
            names["b_" + n] = getattr(s[n], "bias", None)
    names = {k: v for k, v in names.items() if v is not None}
    grads = torch.autograd.grad([o for o, _ in pairs], list(names.values()), [d for _, d in pairs], allow_unused=True)
    want, mag = r.backward(f64(s["d_out"]) if use[0] else None, f64(s["d_h"]) if use[1] and h is not None else None)
    for (k, v), got in zip(names.items(), grads):
        if got is None:
            assert float(want[k].abs().max()) == 0
            continue
        assert got.dtype == v.dtype and got.shape == v.shape, k
        within(got, want[k].view(v.shape), mag[k].view(v.shape), k)


# every norm on either side, with every width of a lane team
@pytest.mark.parametrize("keep", ["float32", "int8"])
@pytest.mark.parametrize("post,pre", list(itertools.product([None, "rms", "layer"], repeat=2)))
def test_norms(post, pre, keep):
    check(make(203, 64, "float32", post, pre, 4, True, True), "float32", keep)


@pytest.mark.parametrize("keep", ["float32", "int8"])
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows,C,G", [(1, 1, 1), (1, 64, 4), (5, 7, 7), (33, 30, 2), (65, 32, 8), (70, 50, 5), (41, 128, 0),
                                      (29, 100, 4), (37, 200, 8), (19, 256, 64), (23, 500, 1), (11, 510, 17), (9, 1000, 8),
                                      (5, 1024, 2), (7, 1030, 10), (6, 2048, 16), (3, 4096, 1), (2, 4095, 0)])
def test_shapes(rows, C, G, kind, keep):
    check(make(rows, C, kind, "layer" if C > 1 else "rms", "rms", G, True, C % 3 == 0), kind, keep)


# every team of lanes, with whole pieces of 16 bytes and with every size of a cut one
@pytest.mark.parametrize("keep", ["float32", "int8"])
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("C", [16, 24, 27, 61, 64, 94, 96, 125, 183, 190, 192, 253, 382, 384, 511, 760, 767, 1022, 1024, 1049,
                               1528, 1534, 2042, 2045])
def test_teams(C, kind, keep):
    check(make(37, C, kind, "rms", "layer", 1, True, True), kind, keep)


@pytest.mark.parametrize("keep", ["float32", "int8"])
@pytest.mark.parametrize("kind,rows,C,G", [("float32", 20003, 64, 4), ("bfloat16", 3001, 512, 1), ("float16", 40001, 24, 2)])
def test_many_rows(kind, rows, C, G, keep):
    check(make(rows, C, kind, "rms", "layer", G, True, True), kind, keep)


@pytest.mark.parametrize("use", [(True, False), (False, True)])
def test_one_output_used(use):
    check(make(50, 64, "float32", "rms", "layer", 2, True, True), "float32", "int8", use)


@pytest.mark.parametrize("keep", ["float32", "int8"])
def test_without_gate_scale_or_mask(keep):
    check(make(50, 48, "float32", "rms", "rms", 0, False, False), "float32", keep)
    check(make(50, 48, "float32", None, None, 0, False, False), "float32", keep)


def test_rows_without_a_view():
    """No row seen, and f (NaN and infinities) reaches nothing there."""
    s = make(64, 96, "float32", "layer", "rms", 3, True, False)
    s["seen"] = torch.zeros(64, dtype=torch.bool, device="cuda")
    for keep in ("float32", "int8"):
        with torch.no_grad():
            s["f"].fill_(float("nan"))
            s["gate"][5] = float("inf")
        out, h = run(s, keep)
        assert torch.equal(out, s["x"])
        g = torch.autograd.grad((out, h), [s["x"], s["f"], s["gate"], s["scale"], s["post"].weight, s["post"].bias],
                                (s["d_out"], s["d_h"]))
        assert torch.isfinite(g[0]).all()
        assert all(float(t.abs().max()) == 0 for t in g[1:])


def test_rows_of_zeros_and_closed_gates():
    s = make(40, 64, "float32", "layer", "layer", 4, True, False)
    with torch.no_grad():
        s["x"][3] = 0
        s["f"][3] = 0
        s["f"][9] = 2.5         # no spread
        s["gate"][11] = 0
    for keep in ("float32", "int8"):
        check(s, "float32", keep)
    out, _ = run(s, "int8")
    assert torch.equal(out[11], s["x"][11])


def test_not_finite_rows_stay_alone():
    s = make(40, 64, "float32", "rms", "rms", 4, True, False)
    clean = run(s, "int8")
    with torch.no_grad():
        s["f"][7, 3] = float("inf")
        s["x"][8, 60] = float("nan")
    got = run(s, "int8")
    rest = torch.ones(40, dtype=torch.bool, device="cuda")
    rest[7] = rest[8] = False
    for a, b in zip(clean, got):
        assert torch.equal(a[rest], b[rest])
        assert not torch.isfinite(b[7]).all() and torch.isnan(b[8]).any()
    d = torch.autograd.grad(got, (s["x"], s["f"], s["gate"]), (s["d_out"], s["d_h"]))
    assert all(torch.isfinite(t[rest]).all() for t in d)


def test_first_norm_and_forward_only():
    """f = None is the norm in front of the first branch; without a graph nothing is kept."""
    from mvfusion.residual import residual_norm
    g = np.random.default_rng(1)
    x = T(g.normal(size=(77, 128)).astype(np.float32)).cuda().requires_grad_(True)
    for kind in ("rms", "layer"):
        m = norm_module(kind, 128, g)
        for keep in ("float32", "int8"):
            out, h = residual_norm(x, None, pre=m, keep=keep)
            assert torch.equal(out, x)
            r = ref.Residual(f64(x), torch.zeros(77, 128).double(), pre=norm_ref(m),
                             xq=T(ref.unpack(*ref.pack(x.detach().cpu().numpy()))) if keep == "int8" else None)
            within(h, r.h, r.M_h, "h")
            d = T(g.normal(size=(77, 128)).astype(np.float32)).cuda()
            gx, gw = torch.autograd.grad(h, (x, m.weight), d)
            want, mag = r.backward(None, f64(d))
            within(gx, want["x"], mag["x"], "x")
            within(gw, want["w_pre"], mag["w_pre"], "w")
        with torch.no_grad():
            out, h = residual_norm(x, None, pre=m)
            assert out.grad_fn is None and h.grad_fn is None


def test_layouts_leading_dimensions_and_scalars():
    from mvfusion.residual import residual_norm
    s = make(60, 64, "float32", "rms", "layer", 1, False, True)
    want = residual_norm(s["x"], s["f"], s["post"], s["pre"], gate=s["gate"], scale=torch.full((64,), 0.5, device="cuda"),
                         seen=s["seen"])
    x3, f3 = s["x"].view(3, 20, 64), s["f"].view(3, 20, 64)
    for gate in (s["gate"].view(3, 20), s["gate"].view(3, 20, 1)):
        for scale in (0.5, torch.tensor([0.5], device="cuda"), torch.tensor(0.5, device="cuda")):
            got = residual_norm(x3, f3, s["post"], s["pre"], gate=gate, scale=scale, seen=s["seen"].view(3, 20))
            assert all(torch.equal(a.view(60, 64), b) for a, b in zip(got, want))
    got = residual_norm(s["x"].t().contiguous().t(), torch.cat([s["f"], s["f"]], 1)[:, 64:], s["post"], s["pre"],
                        gate=s["gate"], scale=0.5, seen=s["seen"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # bases off by one element: the same values by another path of loads
    flat = torch.empty(60 * 64 + 1, device="cuda")[1:].view(60, 64)
    flat.copy_(s["x"].detach())
    got = residual_norm(flat, s["f"], s["post"], s["pre"], gate=s["gate"], scale=0.5, seen=s["seen"])
    assert all(torch.allclose(a, b, rtol=1e-5, atol=1e-5) for a, b in zip(got, want))
    # one learned scale for all channels
    one = torch.tensor(0.5, device="cuda", requires_grad=True)
    vec = torch.full((64,), 0.5, device="cuda", requires_grad=True)
    grads = []
    for scale in (one, vec):
        out, h = residual_norm(s["x"], s["f"], s["post"], s["pre"], gate=s["gate"], scale=scale, seen=s["seen"])
        grads.append(torch.autograd.grad((out, h), scale, (s["d_out"], s["d_h"]))[0])
    assert torch.allclose(grads[0], grads[1].sum(), rtol=1e-5, atol=1e-4)
    # no rows
    empty = s["x"][:0]
    out, h = residual_norm(empty, s["f"][:0], s["post"], s["pre"], gate=s["gate"][:0], scale=vec, seen=s["seen"][:0])
    assert out.shape == (0, 64)
    gw, gs = torch.autograd.grad((out.sum() + h.sum()), (s["post"].weight, vec))
    assert float(gw.abs().max()) == 0 and float(gs.abs().max()) == 0


def test_parameters_of_16_bits():
    """Modules in the rows' own type: gradients come back in that type."""
    from mvfusion.residual import residual_norm
    s = make(30, 64, "bfloat16", "rms", "layer", 4, True, True)
    for n in ("post", "pre"):
        s[n] = s[n].to(torch.bfloat16)
    s["gate"] = s["gate"].detach().to(torch.bfloat16).requires_grad_(True)
    check(s, "bfloat16", "int8")


def test_gradients_against_differences():
    """Directional differences of a float64 evaluation of the same function."""
    s = make(12, 40, "float32", "layer", "rms", 2, True, True)
    out, h = run(s, "float32")
    leaves = [s["x"], s["f"], s["gate"], s["scale"], s["post"].weight, s["post"].bias, s["pre"].weight]
    grads = torch.autograd.grad((out, h), leaves, (s["d_out"], s["d_h"]))
    g = np.random.default_rng(2)
    base = [f64(t) for t in leaves]

    def loss(v):
        r = ref.Residual(v[0], v[1], post=("layer", v[4], v[5], 1e-5), pre=("rms", v[6], None, 1e-5), gate=v[2], scale=v[3],
                         seen=s["seen"].cpu())
        return float((r.out * f64(s["d_out"])).sum() + (r.h * f64(s["d_h"])).sum())
    for i, grad in enumerate(grads):
        d = T(g.normal(size=tuple(base[i].shape)))
        step = 1e-5
        up, down = ([v + k * step * d if j == i else v for j, v in enumerate(base)] for k in (1, -1))
        diff = (loss(up) - loss(down)) / (2 * step)
        # truncation step^2 of a smooth function, cancellation 1e-16 / step, float32 gradients
        assert abs(float((f64(grad) * d).sum()) - diff) <= 1e-5 * float((f64(grad).abs() * d.abs()).sum()), i


def test_same_bits_other_streams_and_replays():
    s = make(5000, 96, "float32", "rms", "rms", 3, True, True)
    leaves = [s["x"], s["f"], s["gate"], s["scale"], s["post"].weight, s["pre"].weight]

    def step():
        # (outputs without their graph: a backward must not be captured while an eager graph of the
        # same leaves is alive, its nodes belong to a stream outside the capture)
        out, h = run(s, "int8")
        grads = torch.autograd.grad((out, h), leaves, (s["d_out"], s["d_h"]))
        return (out.detach(), h.detach()) + grads
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        with torch.no_grad():
            s["x"].copy_(torch.randn_like(s["x"]))
            s["f"].copy_(torch.randn_like(s["f"]))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


@pytest.mark.parametrize("keep", ["float32", "int8"])
def test_one_tensor_on_both_sides(keep):
    """f the tensor x itself, one norm on both sides: the sums of what two of each get."""
    from mvfusion.residual import residual_norm
    torch.manual_seed(2)
    x = torch.randn(300, 48, device="cuda", requires_grad=True)
    f = x.detach().clone().requires_grad_(True)
    m, m2 = torch.nn.LayerNorm(48).cuda(), torch.nn.LayerNorm(48).cuda()
    d = torch.randn(2, 300, 48, device="cuda")
    one = torch.autograd.grad(residual_norm(x, x, post=m, pre=m, keep=keep), (x, m.weight, m.bias), list(d))
    two = torch.autograd.grad(residual_norm(x, f, post=m2, pre=m, keep=keep),
                              (x, f, m2.weight, m.weight, m2.bias, m.bias), list(d))
    for k in range(3):
        assert torch.equal(one[k], two[2 * k] + two[2 * k + 1])


def test_more_than_2_31_values():
    from mvfusion.residual import residual_norm
    rows, C = (1 << 31) // 64 + 5, 64
    x = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    f = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    x[-3:], f[-3:] = 1.0, torch.arange(64, device="cuda").to(torch.bfloat16)
    m = torch.nn.RMSNorm(C).cuda()
    with torch.no_grad():
        out, h = residual_norm(x, f, post=m, pre=m)
        want = residual_norm(x[-3:], f[-3:], post=m, pre=m)
    assert torch.equal(out[-3:], want[0]) and torch.equal(h[-3:], want[1])
    assert int(torch.count_nonzero(out[:1000])) == 0


def test_block_with_kept_rows_inside_an_mlp():
    """The operators as a program uses them: an MLP's output, gated, added to a point's feature
    and normalised for the next branch, in kept 8-bit rows, against float32 rows: the same outputs,
    gradients within the half steps of 1 / 64 of a group's largest value that enter them."""
    from mvfusion import training as tr
    from mvfusion.dense import MLP
    from mvfusion.residual import residual_norm
    torch.manual_seed(0)
    seq, head = MLP([48, 64, 64], bias=False).cuda().train(), torch.nn.Linear(64, 16).cuda()
    post, pre = torch.nn.RMSNorm(64).cuda(), torch.nn.LayerNorm(64).cuda()
    scale = torch.full((64,), 0.5, device="cuda", requires_grad=True)
    v = torch.randn(6000, 48, device="cuda", requires_grad=True)
    x = torch.randn(6000, 64, device="cuda", requires_grad=True)
    gate = torch.rand(6000, 4, device="cuda", requires_grad=True)
    seen = torch.rand(6000, device="cuda") > 0.2
    params = [v, x, gate, scale] + [p for m in (seq, head, post, pre) for p in m.parameters()]
    state = {k: t.clone() for k, t in seq.state_dict().items()}
    d = torch.randn(6000, 16, device="cuda")
    res = {}
    for keep in ("float32", "int8"):
        seq.load_state_dict(state)
        with tr.keep_activations(keep):
            out, h = residual_norm(x, tr.mlp(seq, v), post=post, pre=pre, gate=gate, scale=scale, seen=seen)
            y = tr.linear(head, h)
        res[keep] = (out, h, y), torch.autograd.grad(y, params, d)
    assert all(torch.equal(a, b) for a, b in zip(res["float32"][0], res["int8"][0]))
    for a, b in zip(res["int8"][1], res["float32"][1]):
        assert float((a - b).norm() / b.norm().clamp_min(1e-20)) < 0.05


def test_refusals():
    from mvfusion.residual import residual_norm
    x, f = torch.randn(10, 24, device="cuda"), torch.randn(10, 24, device="cuda")
    rms = torch.nn.RMSNorm(24).cuda()
    bad = [
        (ValueError, dict(f=f[:5])), (ValueError, dict(f=f.half())), (ValueError, dict(f=f.cpu())),
        (ValueError, dict(f=None)), (ValueError, dict(f=None, pre=rms, gate=torch.rand(10, device="cuda"))),
        (TypeError, dict(f=f, post=torch.nn.BatchNorm1d(24).cuda())), (ValueError, dict(f=f, post=torch.nn.RMSNorm(12).cuda())),
        (ValueError, dict(f=f, post=torch.nn.RMSNorm((10, 24)).cuda())), (ValueError, dict(f=f, pre=torch.nn.LayerNorm(24))),
        (ValueError, dict(f=f, gate=torch.rand(10, 5, device="cuda"))), (ValueError, dict(f=f, gate=torch.rand(9, 4, device="cuda"))),
        (ValueError, dict(f=f, gate=torch.rand(10, 4))), (ValueError, dict(f=f, gate=torch.ones(10, 4, dtype=torch.int32, device="cuda"))),
        (ValueError, dict(f=f, scale=torch.rand(12, device="cuda"))), (ValueError, dict(f=f, scale=torch.rand(24))),
        (ValueError, dict(f=f, seen=torch.ones(10, dtype=torch.uint8, device="cuda"))),
        (ValueError, dict(f=f, seen=torch.ones(9, dtype=torch.bool, device="cuda"))),
        (ValueError, dict(f=f, keep="fp8")),
    ]
    for error, args in bad:
        with pytest.raises(error):
            residual_norm(x, **args)
    with pytest.raises(TypeError):
        residual_norm(x.double(), f.double())
    wide = torch.zeros(2, 4097, device="cuda")
    with pytest.raises(ValueError):
        residual_norm(wide, wide)
    y, h = residual_norm(x.requires_grad_(True), f, pre=rms)
    (gx,) = torch.autograd.grad(h.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
