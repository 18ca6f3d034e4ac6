"""Distillation without a GPU: the reference form against differences of its own loss, and every
refusal that needs no device."""

import ctypes

import numpy as np
import pytest
import torch

from rusticide_b200 import InvalidShape, TensorError, _lib, distill_loss, sampler
from rusticide_b200.sampler import Engine

from . import distill_ref as R


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0])
def test_reference_gradient_is_the_slope_of_the_reference_loss(tail, temperature):
    """Central differences of steps that are exact in binary32 (multiples of 2^-12 on logits of
    that grid): the truncation error is h^2 / 6 times a third derivative below 1."""
    rng = np.random.default_rng(5)
    x = (np.round(rng.normal(size=24) * 64) / 64).astype(np.float32)
    ids = np.array([3, 7, 8, 20, 7, -1, 99], np.int32)
    y = np.log(np.array([0.3, 0.1, 0.2, 0.15, 0.05, 0.5, 0.5])).astype(np.float32)
    h = 2.0 ** -10
    _, grad, _, _ = R.row(x, ids, y, temperature, tail)
    for j in range(len(x)):
        up, down = x.copy(), x.copy()
        up[j] += h
        down[j] -= h
        slope = (R.row(up, ids, y, temperature, tail)[0] - R.row(down, ids, y, temperature, tail)[0]) / (2 * h)
        # Binary32 rounding of v = x / T moves a term by at most 2^-24 * 8.
        assert abs(slope - grad[j]) < h * h * 8 + (0 if temperature == 1 else 2 ** -21 / h * 0.25)


def test_reference_agrees_with_plain_cross_entropy_and_kl():
    rng = np.random.default_rng(6)
    x = rng.normal(size=10).astype(np.float32)
    logp = torch.log_softmax(torch.from_numpy(x).double(), 0)
    loss, grad, _, _ = R.row(x, np.array([4]), np.array([0.0], np.float32))
    assert abs(loss + float(logp[4])) < 1e-12          # one token: cross entropy
    t = torch.softmax(torch.from_numpy(rng.normal(size=10)), 0)
    y = t.log().numpy().astype(np.float32)
    loss, _, _, _ = R.row(x, np.arange(10), y)
    want = torch.nn.functional.kl_div(logp, torch.from_numpy(y).double(), reduction="sum", log_target=True)
    assert abs(loss - float(want)) < 1e-6              # every token: KL (y rounded to binary32)


@pytest.fixture(autouse=True)
def no_stream(monkeypatch):
    monkeypatch.setattr(sampler, "_stream_ptr", lambda device: 0)


def cpu_engine() -> Engine:
    e = Engine.__new__(Engine)
    e.device, e.lib, e._h = torch.device("cpu"), _lib.lib(), ctypes.c_void_p()
    e.max_rows = e.max_vocab = 0
    e._index = -1  # Tensor.get_device() on the CPU
    return e


def arguments(rows=3, v=10, k=2):
    return dict(logits=torch.zeros(rows, v), ids=torch.zeros(rows, k, dtype=torch.int32),
                logprobs=torch.zeros(rows, k))


BAD = [
    ("logits", torch.zeros(3, 10, dtype=torch.float64), TensorError),
    ("logits", torch.zeros(2, 10), InvalidShape),
    ("logits", torch.zeros(()), InvalidShape),
    ("ids", torch.zeros(3, 2, dtype=torch.int64), TensorError),
    ("ids", torch.zeros(3, dtype=torch.int32), InvalidShape),
    ("ids", torch.zeros(2, 3, dtype=torch.int32).t(), ValueError),
    ("logprobs", torch.zeros(3, 3), InvalidShape),
    ("logprobs", torch.zeros(3, 2, dtype=torch.bfloat16), TensorError),
    ("n", torch.zeros(4, dtype=torch.int32), InvalidShape),
    ("n", torch.zeros(3), TensorError),
]


@pytest.mark.parametrize("name,value,error", BAD)
def test_calls_refuse(name, value, error):
    kw = {**arguments(), name: value}
    with pytest.raises(error):
        cpu_engine().distill_forward(**kw)
    with pytest.raises(error):
        cpu_engine().distill_step(row_grads=torch.zeros(3), **kw)
    with pytest.raises(error):
        cpu_engine().distill_backward(state=torch.zeros(3, 4), row_grads=torch.zeros(3), **kw)


@pytest.mark.parametrize("kw,error", [
    (dict(row_grads=torch.zeros(2)), InvalidShape),
    (dict(row_grads=torch.zeros(3, dtype=torch.float64)), TensorError),
    (dict(row_grads=torch.zeros(3), out=torch.zeros(3, 9)), InvalidShape),
    (dict(row_grads=torch.zeros(3), out=torch.zeros(3, 10, dtype=torch.bfloat16)), TensorError),
    (dict(row_grads=torch.zeros(3), out=torch.zeros(10, 3).t()), ValueError),
])
def test_step_refuses(kw, error):
    with pytest.raises(error):
        cpu_engine().distill_step(**arguments(), **kw)


def test_replacing_logits_of_another_layout_is_refused():
    a = arguments()
    a["logits"] = torch.zeros(10, 3).t()
    with pytest.raises(ValueError):
        cpu_engine().distill_step(row_grads=torch.zeros(3), out=a["logits"], **a)


def test_good_arguments_reach_the_library():
    a = arguments()
    for call in (lambda e: e.distill_forward(**a),
                 lambda e: e.distill_step(row_grads=torch.zeros(3), **a),
                 lambda e: e.distill_step(row_grads=torch.zeros(3), out=a["logits"], **a),
                 lambda e: e.distill_backward(state=torch.zeros(3, 4), row_grads=torch.zeros(3), **a)):
        with pytest.raises(_lib.RscError) as err:
            call(cpu_engine())
        assert err.value.code == _lib.RSC_ERR_NOT_INITIALIZED


def test_distill_loss_needs_a_gpu():
    if torch.cuda.is_available():
        pytest.skip("this machine has one")
    with pytest.raises(RuntimeError):
        distill_loss(**arguments())


@pytest.mark.parametrize("name", ["logits", "logprobs"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(name, grad):
    """A tangent must not be dropped: a dual tensor has no requires_grad of its own to go by."""
    with torch.autograd.forward_ad.dual_level():
        a = arguments()
        a[name] = torch.autograd.forward_ad.make_dual(a[name].requires_grad_(grad), torch.ones_like(a[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            distill_loss(**a)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="CUDA"):  # no tangent: the call goes on
            distill_loss(**arguments())
