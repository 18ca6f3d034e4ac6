"""Draft verification without a GPU: the reference form against the property it exists for, and
every refusal that needs no device."""

import ctypes

import numpy as np
import pytest
import torch

from rusticide_b200 import InvalidShape, SamplingParams, TensorError, _lib, sampler
from rusticide_b200.sampler import Engine

from . import verify_ref as R


def test_reference_form_keeps_the_target_distribution():
    """P(first token = j) summed over drafts, tests and draws is exactly p_j: integrate the
    uniforms on a grid instead of sampling them."""
    rng = np.random.default_rng(3)
    x, y = rng.normal(size=(1, 2, 6)), rng.normal(size=(1, 1, 6))
    x, y = x.astype(np.float32), y.astype(np.float32)
    p, q = R.softmax(x[0, 0]), R.softmax(y[0, 0])
    grid = (np.arange(200) + 0.5) / 200
    got = np.zeros(6)
    for t in range(6):
        for u0 in grid:
            for u1 in grid[::8]:
                toks, acc, _ = R.verify_batch(x, y, np.array([[t]]), None,
                                              np.array([[u0, u1]]), 1.0)
                got[toks[0, 0]] += q[t] / (len(grid) * len(grid[::8]))
    # Each test's and draw's edge is known to one grid step of its uniform.
    assert np.abs(got - p).max() < 1 / 200 + 1 / 25


@pytest.fixture(autouse=True)
def no_stream(monkeypatch):
    monkeypatch.setattr(sampler, "_stream_ptr", lambda device: 0)


def cpu_engine() -> Engine:
    """An engine without a handle on the CPU device: its argument checks run, and the C call
    answers that the handle is missing."""
    e = Engine.__new__(Engine)
    e.device, e.lib, e._h = torch.device("cpu"), _lib.lib(), ctypes.c_void_p()
    e.max_rows = e.max_vocab = 0
    e._index = -1  # Tensor.get_device() on the CPU
    return e


def arguments(b=2, d=3, v=10):
    return dict(target_logits=torch.zeros(b, d + 1, v), draft_tokens=torch.zeros(b, d, dtype=torch.int32),
                draft_logits=torch.zeros(b, d, v), n_draft=torch.zeros(b, dtype=torch.int32),
                uniforms=torch.zeros(b, d + 1))


@pytest.mark.parametrize("name,value,error", [
    ("target_logits", torch.zeros(2, 3, 10), InvalidShape),
    ("target_logits", torch.zeros(8, 10), InvalidShape),
    ("target_logits", torch.zeros(2, 4, 10, dtype=torch.float16), TensorError),
    ("target_logits", torch.zeros(2, 4, 20)[:, :, ::2], ValueError),
    ("draft_tokens", torch.zeros(2, 3, dtype=torch.int64), TensorError),
    ("draft_tokens", torch.zeros(6, dtype=torch.int32), InvalidShape),
    ("draft_tokens", torch.zeros(3, 2, dtype=torch.int32).t(), ValueError),
    ("draft_logits", torch.zeros(2, 4, 10), InvalidShape),
    ("draft_logits", torch.zeros(2, 3, 11), InvalidShape),
    ("n_draft", torch.zeros(3, dtype=torch.int32), InvalidShape),
    ("n_draft", torch.zeros(2, dtype=torch.int64), TensorError),
    ("uniforms", torch.zeros(2, 3), InvalidShape),
    ("uniforms", torch.zeros(2, 4, dtype=torch.float64), TensorError),
    ("rng_states", torch.zeros(3, dtype=torch.int64), InvalidShape),
    ("out", (torch.zeros(2, 3, dtype=torch.int32),) * 3, InvalidShape),
])
def test_verify_refuses(name, value, error):
    with pytest.raises(error):
        cpu_engine().verify(params=SamplingParams(1.0, 0, 1.0), **{**arguments(), name: value})


def test_verify_reaches_the_library_with_good_arguments():
    for kw in (arguments(), {**arguments(), "draft_logits": None, "n_draft": None}):
        with pytest.raises(_lib.RscError) as e:
            cpu_engine().verify(params=SamplingParams(1.0, 0, 1.0), **kw)
        assert e.value.code == _lib.RSC_ERR_NOT_INITIALIZED


def record(rows, cap, dtype=torch.float32):
    return (torch.zeros(rows, dtype=torch.int32), torch.zeros(rows, cap, dtype=torch.int32),
            torch.zeros(rows, cap, dtype=dtype))


@pytest.mark.parametrize("target,draft,error", [
    (record(7, 4), None, InvalidShape),
    (record(8, 4, torch.float64), None, TensorError),
    (record(8, 4), record(8, 4), InvalidShape),
    ((record(8, 4)[0], torch.zeros(8, 5, dtype=torch.int32), record(8, 4)[2]), None, InvalidShape),
    (record(8, 4) + (torch.zeros(7, dtype=torch.int32),), None, InvalidShape),
    (record(8, 4), record(6, 4), _lib.RscError),
])
def test_verify_survivors_refuses(target, draft, error):
    a = arguments()
    with pytest.raises(error):
        cpu_engine().verify_survivors(target, a["draft_tokens"], uniforms=a["uniforms"], draft=draft)


def test_workspace_grows_with_the_batch():
    size = _lib.lib().rsc_verify_workspace_bytes
    assert size(0, 4, 1000) == 0
    assert size(1, 0, 1000) >= 16 and size(1, 0, 1000) % 16 == 0
    assert size(8, 4, 151936) == 8 * size(1, 4, 151936)
    assert size(8, 4, 151936) >= size(8, 4, 1000)
