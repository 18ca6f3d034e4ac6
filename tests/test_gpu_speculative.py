"""Drafting, verifying and training a draft model, together as a decode loop would: the draft's tokens
come from the sampler, the target's rows verify them, and the same rows' survivor records train the
draft's output layer. Each stage is held to its own reference form on the values that the stage before
it left on the device."""

import numpy as np
import pytest
import torch

from rusticide_b200 import SamplingParams, distill_loss, engine

from . import distill_ref, verify_ref

pytestmark = pytest.mark.gpu


def host(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


@pytest.mark.parametrize("params", [SamplingParams(1.0, 0, 1.0), SamplingParams(0.8, 40, 0.95),
                                    SamplingParams(0.0, 0, 1.0)])
def test_a_few_steps_of_speculative_decoding(params):
    b, d, v, dim = 6, 3, 4001, 64
    e = engine(0)
    g = torch.Generator(device="cuda").manual_seed(5)
    hidden = torch.randn((b, d + 1, dim), generator=g, device="cuda")
    w_target = torch.randn((v, dim), generator=g, device="cuda") / 3
    w_draft = (w_target + 0.05 * torch.randn((v, dim), generator=g, device="cuda")).requires_grad_()
    target = (hidden @ w_target.t()).contiguous()
    teacher = SamplingParams(1.0, 40, 0.95)
    states = e.rng_seed(torch.arange(b))
    for step in range(3):
        # The draft proposes a token for every position but the last.
        draft = (hidden[:, :d] @ w_draft.t()).contiguous()
        tokens, status, _ = e.pick(draft.detach().reshape(b * d, v), params,
                                   uniforms=torch.rand(b * d, generator=g, device="cuda"))
        assert not status.bitwise_and(0xFF).any()
        tokens = tokens.reshape(b, d)
        # The target verifies them; the sequences' generators advance.
        before = [int(s) & ((1 << 64) - 1) for s in states]
        out, accepted, status = e.verify(target, tokens, params, rng_states=states,
                                         draft_logits=draft.detach())
        assert not status.any()
        x, y, t = host(target), host(draft), host(tokens)
        u = np.zeros((b, d + 1), np.float32)
        for i in range(b):
            us = verify_ref.wyrand_uniforms(before[i], d + 1)
            u[i, :d] = us[:d]
            a = int(accepted[i])
            u[i, d] = us[a + (a < d)]
        if params.temperature == 0:
            want = verify_ref.greedy_batch(x, t, None)
            assert [int(s) & ((1 << 64) - 1) for s in states] == before
        elif params.top_k == 0:
            want = verify_ref.verify_batch(x, y, t, None, u, params.temperature)
        else:
            def records(rows):
                o = e.sample_ex(rows.reshape(-1, v), params, survivor_cap=64,
                                uniforms=torch.zeros(rows.numel() // v, device="cuda"))
                return [host(o[k]) for k in (3, 4, 5)]
            want = verify_ref.verify_records(records(target), records(draft.detach()), v, t, None, u)
        np.testing.assert_array_equal(host(out), want[0])
        np.testing.assert_array_equal(host(accepted), want[1])
        # The target's records train the draft on the positions that were verified.
        rec = e.sample_ex(target.reshape(-1, v), teacher, survivor_cap=64, logprobs=True,
                          uniforms=torch.zeros(b * (d + 1), device="cuda"))
        n, ids, logp = (rec[k].reshape((b, d + 1) + rec[k].shape[1:])[:, :d].contiguous()
                        for k in (3, 4, 8))
        counts = (torch.arange(d, device="cuda") <= accepted[:, None]).float()
        upstream = counts / counts.sum()
        loss = distill_loss(draft, ids, logp, n=n, tail=True)
        dlogits, = torch.autograd.grad(loss, draft, upstream, retain_graph=True)
        grad, = torch.autograd.grad((loss * upstream).sum(), w_draft)
        ref = distill_ref.batch(y.reshape(b * d, v), host(ids).reshape(b * d, -1),
                                host(logp).reshape(b * d, -1), host(n).reshape(-1), 1.0, True)
        up = host(upstream).reshape(-1)
        # As in test_gpu_distill.py.
        assert (np.abs(host(loss).reshape(-1) - ref[0]) < 1.5e-5 + 2e-7 * np.abs(ref[0])).all()
        value = ref[1] * up[:, None]
        limit = up[:, None] * (1.3e-5 * ref[2] + 2e-7 * ref[3]) + 2.0 ** -24 * np.abs(value) + 1e-37
        assert (np.abs(host(dlogits).reshape(b * d, v) - value) <= limit).all()
        # The weights' gradient is the same rows through the matrix product (binary32, possibly
        # with TF32 off: b * d products a sum, each rounded once).
        h = host(hidden[:, :d]).reshape(b * d, dim).astype(np.float64)
        whole = value.T @ h
        room = (limit.T @ np.abs(h)) + 2.0 ** -24 * (b * d + 1) * (np.abs(value).T @ np.abs(h))
        assert not torch.backends.cuda.matmul.allow_tf32
        assert (np.abs(host(grad) - whole) <= room + 1e-30).all()
        # The step form gives the same loss and gradient without a graph, in place of the logits.
        spare = draft.detach().clone()
        step_loss, step_grad = e.distill_step(spare, ids, logp, upstream, n=n, tail=True, out=spare)
        assert (np.abs(host(step_loss).reshape(-1) - ref[0]) < 1.5e-5 + 2e-7 * np.abs(ref[0])).all()
        assert (np.abs(host(step_grad).reshape(b * d, v) - value) <= limit).all()
        with torch.no_grad():
            w_draft -= 0.5 * grad
