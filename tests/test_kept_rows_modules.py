"""Which modules the training path's layers accept, without a GPU."""
import pytest
import torch
from torch.nn.utils import parametrize, prune

from mvfusion import packed, residual, training


@pytest.mark.parametrize("keep", [None, "float32", "int8"])
@pytest.mark.parametrize("norm", [torch.nn.Identity(), torch.nn.LayerNorm(4), torch.nn.Tanh()])
def test_other_modules_in_place_of_the_norm(norm, keep):
    """Modules with other parameters or none take over as they are."""
    act, lin = torch.nn.LeakyReLU(0.2), torch.nn.Linear(4, 3)
    x = torch.randn(6, 4, requires_grad=True)
    want = act(norm(x))
    assert torch.equal(training.batch_norm_act(x, norm, act, keep=keep), want)
    assert torch.equal(training.batch_norm_act(x, norm, torch.nn.ReLU(), keep=keep), torch.relu(norm(x)))
    y = training.batch_norm_act_linear(x, norm, act, lin, keep=keep)
    assert torch.equal(y, lin(want))
    y.sum().backward()
    with pytest.raises(ValueError):
        training.batch_norm_act(x, norm, act, keep="bits")
    with pytest.raises(ValueError):
        training.batch_norm_act_linear(x, norm, act, lin, keep="bits")


class Doubled(torch.nn.Module):
    def forward(self, w):
        return 2 * w


def test_residual_norms_with_made_weights():
    """The norms' parameters are read as attributes: parametrized and pruned ones, and none at all."""
    rows = torch.zeros(3, 8)
    norm = torch.nn.LayerNorm(8, eps=1e-3)
    parametrize.register_parametrization(norm, "weight", Doubled())
    prune.random_unstructured(norm, "bias", 0.5)
    kind, weight, bias, eps = residual._norm_args(norm, 8, rows, "post")
    assert kind == residual._LAYER and eps == 1e-3
    assert torch.equal(weight, 2 * torch.ones(8)) and weight.requires_grad and torch.equal(bias, norm.bias)
    rms = torch.nn.RMSNorm(8)
    parametrize.register_parametrization(rms, "weight", Doubled())
    kind, weight, bias, eps = residual._norm_args(rms, 8, rows, "pre")
    assert kind == residual._RMS and bias is None and eps == torch.finfo(torch.float32).eps
    assert torch.equal(weight, 2 * torch.ones(8))
    for none in (torch.nn.LayerNorm(8, elementwise_affine=False), torch.nn.RMSNorm(8, elementwise_affine=False)):
        assert residual._norm_args(none, 8, rows, "pre")[1:3] == (None, None)
    assert residual._norm_args(torch.nn.LayerNorm(8, bias=False), 8, rows, "pre")[2] is None


class Rows:
    """Rows as the choice of a kernel sees them: on a device, without values."""

    def __init__(self, *shape, dtype=torch.float32, device="cuda:0"):
        self.shape, self.dtype, self.device, self.is_cuda = torch.Size(shape), dtype, torch.device(device), True

    def dim(self):
        return len(self.shape)


def test_kernels_are_chosen_by_width_type_and_device():
    x, w = Rows(5, 32), Rows(8, 32)
    assert training._fits(x, w, None) and training._fits(x, w, Rows(8))
    for bad in (Rows(8, 16), Rows(8, 64), Rows(8, 32, dtype=torch.float16), Rows(8, 32, device="cuda:1"), torch.zeros(8, 32)):
        assert not training._fits(x, bad, None)
    for bias in (Rows(8, dtype=torch.float16), Rows(8, device="cuda:1"), torch.zeros(8)):
        assert not training._fits(x, w, bias)
    for rows in (Rows(0, 32), Rows(5, 2, 32), Rows(5, 32, dtype=torch.float64)):
        assert not training._fits(rows, w, None)
    assert training._takes_bn(x, torch.nn.BatchNorm1d(32)) and not training._takes_bn(x, torch.nn.BatchNorm1d(16))
    assert not training._takes_bn(Rows(0, 32), torch.nn.BatchNorm1d(32))
    host, bn = Rows(5, 32, device="cpu"), torch.nn.BatchNorm1d(32).eval()
    assert training._bn_plan(host, bn, bn.weight, bn.bias) is not None
    bn.running_mean = torch.zeros(16)
    assert training._bn_plan(host, bn, bn.weight, bn.bias) is None


def test_what_xty8_and_pack_codes_refuse():
    """The reduction over packed rows reads only what is there: rows, types and devices have to agree."""
    x, w = torch.zeros(6, 5), torch.ones(40)
    codes, exps = torch.zeros(6, 40, dtype=torch.int8), torch.zeros(6, 2, dtype=torch.uint8)
    for error, args in [
            (TypeError, (x.double(), codes, exps)), (ValueError, (x[0], codes, exps)), (ValueError, (x[:, :0], codes, exps)),
            (ValueError, (x, codes[:5], exps[:5])), (ValueError, (x, codes, exps[:, :1])), (ValueError, (x, codes, exps[:5])),
            (ValueError, (x, codes.float(), exps)), (ValueError, (x, codes, exps.int())), (ValueError, (x, codes[0], exps[0])),
            (ValueError, (x, Codes(6, 40), exps)), (ValueError, (x, codes, exps, (w[:39], None, 0.2))),
            (ValueError, (x, codes, exps, (w, w.double(), 0.2))), (ValueError, (x, codes, exps, (None, Rows(40), None))),
            (RuntimeError, (x, codes, exps)), (RuntimeError, (x, codes, exps, (w, None, 0.2)))]:
        with pytest.raises(error):
            training.xty8(*args)
    with pytest.raises(RuntimeError):
        packed.pack_codes(x)
    with pytest.raises(TypeError):
        packed.pack_codes(Rows(6, 5, dtype=torch.float64))
    with pytest.raises(ValueError):
        packed.pack_codes(Rows(5))


class Codes(Rows):
    def __init__(self, *shape):
        super().__init__(*shape, dtype=torch.int8)


def test_column_sums_that_do_not_fit():
    """The statistics' kernel reads n rows of 2 C float64 sums."""
    z, sums = torch.zeros(6, 8), torch.zeros(4, 2, 8, dtype=torch.float64)
    assert training._sums_for(z, sums) is sums and training._sums_for(z, None) is None
    for bad in (sums.float(), sums[:, :, :4], sums[:, :1], sums[:0], sums[0], torch.zeros(4, 2, 9, dtype=torch.float64),
                sums.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(ValueError):
            training._sums_for(z, bad)
