"""Which modules the training path's layers accept, without a GPU."""
import pytest
import torch

from mvfusion import training


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
