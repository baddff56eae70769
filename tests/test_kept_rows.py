"""Kept rows and the residual norm without a GPU: what is refused, and the choice of the kept form."""
import threading

import pytest
import torch

from mvfusion import packed, residual, training


def test_keep_activations_is_scoped_and_per_thread():
    assert training.kept_form() == "float32"
    with training.keep_activations("int8"):
        assert training.kept_form() == "int8"
        assert training.kept_form("float32") == "float32"
        with training.keep_activations("float32"):
            assert training.kept_form() == "float32"
        seen = []
        t = threading.Thread(target=lambda: seen.append(training.kept_form()))
        t.start()
        t.join()
        assert seen == ["float32"] and training.kept_form() == "int8"
    assert training.kept_form() == "float32"
    with pytest.raises(KeyError):
        with training.keep_activations("int8"):
            raise KeyError
    assert training.kept_form() == "float32"


def test_unknown_forms():
    with pytest.raises(ValueError):
        with training.keep_activations("int4"):
            pass
    with pytest.raises(ValueError):
        training.kept_form("fp8")
    with pytest.raises(ValueError):
        training.linear(torch.nn.Linear(4, 4), torch.zeros(3, 4), keep="bits")
    with pytest.raises(ValueError):
        training.batch_norm_act(torch.zeros(3, 4), torch.nn.BatchNorm1d(4), torch.nn.LeakyReLU(), keep="bits")


def test_modules_on_the_cpu_take_over():
    lin, bn = torch.nn.Linear(4, 3), torch.nn.BatchNorm1d(4)
    x = torch.randn(6, 4, requires_grad=True)
    with training.keep_activations("int8"):
        y = training.batch_norm_act_linear(x, bn, torch.nn.LeakyReLU(0.2), lin)
    want = lin(torch.nn.LeakyReLU(0.2)(torch.nn.BatchNorm1d(4)(x)))
    assert torch.allclose(y, want, atol=1e-6)
    y.sum().backward()


def test_no_cpu_fallback():
    with pytest.raises(RuntimeError):
        packed.pack_rows(torch.zeros(3, 4))
    with pytest.raises(RuntimeError):
        packed.unpack_rows(torch.zeros(3, 4, dtype=torch.int8), torch.zeros(3, 1, dtype=torch.uint8))
    with pytest.raises(RuntimeError):
        residual.residual_norm(torch.zeros(3, 4), torch.zeros(3, 4))
