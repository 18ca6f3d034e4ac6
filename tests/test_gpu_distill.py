"""Distillation on the GPU against the binary64 form of distill_ref.py.

Tolerances, from the arithmetic (rsc_rowsum.cuh): a sum of exponentials is within 6e-6 relative, so a
log of it within 6e-6, and the loss, which holds at most two of them with weights that add up to
1 + r <= 2, within 1.2e-5, plus a binary32 rounding of t (2^-24 relative of terms that add up to less
than 40 here) and of the result. A gradient's p has |v - m| 7.3e-8 + 2^-22 from its exponential
(|v - m| < 88 where p is a normal number: 6.7e-6), 6e-6 from the sum and four roundings (2.4e-7):
1.3e-5 relative, and so has the tail's r exp(v) / S_tail. Exponentials below 2^-126 are flushed to 0,
and both sums are at least 1 against the largest term: 2^-126 of either, times the row's factor. The result is rounded to its type by at most half a step, relative eps / 2
or half the smallest subnormal."""

import numpy as np
import pytest
import torch

from rusticide_b200 import SamplingParams, _lib, distill_loss, engine

from . import distill_ref as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def case(rows, v, k, seed, dtype=torch.float32, ordered=True, spread=2.0, held=0.9):
    """Student logits of the type, and k entries a row whose probabilities add up to `held`."""
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.normal(size=(rows, v)) * spread).to(dtype)
    k = min(k, v)
    ids = np.stack([rng.choice(v, size=k, replace=False) for _ in range(rows)]).astype(np.int32) \
        if rows else np.zeros((0, k), np.int32)
    if ordered:
        ids.sort(axis=1)
    t = rng.dirichlet(np.ones(k), size=rows) if k else np.zeros((rows, 0))
    return x, ids, np.log(t * held + 1e-30).astype(np.float32)


def dev(a):
    if a is None:
        return None
    return (a if isinstance(a, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(a))).cuda()


def close_loss(got, want):
    got = got.float().cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    ok = np.isfinite(want)
    np.testing.assert_array_less(np.abs(got[ok] - want[ok]), 1.5e-5 + 2e-7 * np.abs(want[ok]))


def close_grad(got, want, up, temperature, tail):
    """`want`: what R.batch returned."""
    info = torch.finfo(got.dtype)
    g = got.float().cpu().numpy().astype(np.float64)
    _, grad, size, t = want
    value = grad * up[:, None]
    s = np.abs(up[:, None] * float(R.inverse(temperature)))
    rel = 1.3e-5 * size + 2e-7 * t
    tiny = float(info.smallest_normal * info.eps)
    limit = s * (rel + 2 * 2.0 ** -126) + np.abs(value) * info.eps / 2 * 1.001 + max(tiny, 1e-37)
    assert np.array_equal(np.isnan(g), np.isnan(value))
    ok = np.isfinite(value)
    bad = np.abs(g[ok] - value[ok]) > limit[ok]
    assert not bad.any(), (np.abs(g[ok] - value[ok]) / limit[ok]).max()


def check(x, ids, y, n=None, temperature=1.0, tail=False, up=None):
    """Every call on the same rows: the loss alone, the step, forward and backward, autograd."""
    rows = len(x)
    up = np.linspace(0.5, 2.0, rows).astype(np.float32) if up is None else up
    want = R.batch(x.float().numpy(), ids, y, n, temperature, tail)
    want[1] = np.where(up[:, None] == 0, 0.0, want[1]) if rows else want[1].reshape(x.shape)
    e, a = engine(0), (dev(x), dev(ids), dev(y))
    kw = dict(n=dev(n), temperature=temperature, tail=tail)
    loss, state = e.distill_forward(*a, **kw)
    close_loss(loss, want[0])
    assert torch.equal(loss, e.distill_forward(*a, want_state=False, **kw)[0]) or loss.isnan().any()
    both, grad = e.distill_step(*a, dev(up), **kw)
    assert grad.dtype == x.dtype
    close_loss(both, want[0])
    if rows:
        close_grad(grad, want, up, temperature, tail)
    back = e.distill_backward(*a, state, dev(up), **kw)
    if rows:
        close_grad(back, want, up, temperature, tail)
    z = dev(x).requires_grad_()
    out = distill_loss(z, *a[1:], **kw)
    auto, = torch.autograd.grad(out, z, dev(up))
    same = (auto == back) | (auto.isnan() & back.isnan())
    assert same.all()
    replaced = dev(x).clone()
    _, g = e.distill_step(replaced, *a[1:], dev(up), out=replaced, **kw)
    assert g is replaced
    assert ((g == grad) | (g.isnan() & grad.isnan())).all()
    return loss, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,v,k", [(1, 1, 1), (1, 2, 1), (3, 7, 7), (2, 31, 5), (5, 33, 33), (1, 1000, 20),
                                      (4, 2049, 1), (7, 4097, 64), (3, 8192, 100), (1, 50001, 128)])
def test_sizes(rows, v, k, dtype, tail):
    check(*case(rows, v, k, seed=rows * 7 + v, dtype=dtype), tail=tail)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_rows(dtype):
    check(*case(2, 151936, 64, seed=3, dtype=dtype), tail=True, temperature=2.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_vocabularies(dtype):
    """Segments far above 104 and 320 KB, at the largest cluster."""
    check(*case(2, 1500003, 1024, seed=5, dtype=dtype), tail=True)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows", [149, 700])
def test_many_rows(rows, tail):
    """More rows than CTAs fit the GPU at once: a row is no longer spread over a cluster."""
    rng = np.random.default_rng(rows)
    x, ids, y = case(rows, 1501, 20, seed=rows, dtype=torch.bfloat16)
    n = rng.integers(0, 23, size=rows).astype(np.int32)
    up = (rng.random(rows) * (rng.random(rows) < 0.8)).astype(np.float32)
    check(x, ids, y, n=n, tail=tail, up=up, temperature=0.7)


@pytest.mark.parametrize("tail", [False, True])
def test_no_rows_and_no_entries(tail):
    check(*case(0, 10, 3, seed=1), tail=tail)
    x, ids, y = case(4, 100, 3, seed=2)
    x[2] = float("nan")                       # not looked at: the row has no entry
    n = np.array([0, 3, 0, 1], np.int32)
    loss, grad = check(x, ids, y, n=n, tail=tail)
    assert loss[0] == 0 and loss[2] == 0 and not grad[0].any() and not grad[2].any()
    check(x[:2], np.zeros((2, 0), np.int32), np.zeros((2, 0), np.float32), tail=tail)
    ids[1], y[3] = -1, -np.inf                # padding, and entries of no probability
    check(x, ids, y, tail=tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_negative_count_is_an_empty_list(dtype, tail):
    x, ids, y = case(6, 3000, 8, seed=28, dtype=dtype)
    n = np.array([-1, 8, -2 ** 31, 0, 9, 3], np.int32)
    loss, grad = check(x, ids, y, n=n.clip(0), tail=tail)
    e, a = engine(0), (dev(x), dev(ids), dev(y))
    kw, up = dict(n=dev(n), tail=tail), dev(np.linspace(0.5, 2.0, 6).astype(np.float32))
    got, state = e.distill_forward(*a, **kw)
    assert torch.equal(got, loss) and not got[[0, 2, 3]].any()
    both, step = e.distill_step(*a, up, **kw)
    assert torch.equal(step, grad) and not step[[0, 2, 3]].any()
    assert not e.distill_backward(*a, state, up, **kw)[[0, 2, 3]].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_lists_out_of_order_and_with_repeats(dtype, tail):
    x, ids, y = case(6, 500, 40, seed=11, dtype=dtype, ordered=False, held=0.5)
    ids[1, 5:9] = ids[1, 0]                   # one token five times
    ids[2, :] = ids[2, 0]                     # one token alone
    ids[3, ::3] = -1
    ids[4, 7] = 500                           # just outside the vocabulary
    ids[4, 8] = 2 ** 31 - 1
    ids[5, 1::2] = ids[5, 0::2]
    check(x, ids, y, tail=tail)


@pytest.mark.parametrize("tail", [False, True])
def test_masked_logits_nan_and_infinities(tail):
    x, ids, y = case(12, 700, 8, seed=21)
    rng = np.random.default_rng(22)
    x[rng.random(x.shape) < 0.3] = float("-inf")
    for r in range(12):
        x[r, ids[r].astype(np.int64)] = 0.5
    x[0, int(ids[0, 2])] = float("-inf")      # a listed token of no student mass: loss inf
    x[1] = float("-inf")                      # no distribution
    x[2, 5] = float("nan")
    x[3, 6] = float("inf")
    x[4] = float("-inf")                      # the listed tokens alone are left
    x[4, ids[4].astype(np.int64)] = 1.0
    x[5] = torch.finfo(torch.float32).min     # masks of the type's lowest value
    x[5, ids[5].astype(np.int64)] = 0.0
    y[6, 1] = np.nan
    y[7, :] = -np.inf
    up = np.ones(12, np.float32)
    up[2] = 0.0                               # a row that does not count has no gradient
    check(x, ids, y, tail=tail, up=up)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_masks_nan_and_infinities_in_long_rows(dtype, tail):
    """Segments of several batches of 16-byte words, on their way through shared memory."""
    v = 131077 * (1 if dtype is torch.float32 else 2)
    x, ids, y = case(12, v, 8, seed=23, dtype=dtype)
    g = torch.Generator().manual_seed(24)
    x[torch.rand(x.shape, generator=g) < 0.3] = float("-inf")
    for r in range(12):
        x[r, ids[r].astype(np.int64)] = 0.5
    x[0, int(ids[0, 2])] = float("-inf")
    x[1] = float("-inf")
    x[2, v // 2] = float("nan")
    x[3, v - 1] = float("inf")
    x[4] = float("-inf")
    x[4, ids[4].astype(np.int64)] = 1.0
    x[5] = torch.finfo(dtype).min
    x[5, ids[5].astype(np.int64)] = 0.0
    x[6, v // 3:] = float("-inf")             # whole segments without a logit
    x[6, ids[6].astype(np.int64)] = 0.5
    y[7, :] = -np.inf
    n = np.full(12, 8, np.int32)
    n[8], n[9] = 0, 3
    up = np.linspace(0.5, 1.5, 12).astype(np.float32)
    up[2], up[10] = 0.0, 0.0
    check(x, ids, y, n=n, tail=tail, up=up)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_the_loss_is_the_same_with_and_without_the_state(dtype, tail):
    """Bit for bit, in rows of NaN and infinite loss as in the others."""
    x, ids, y = case(12, 40001, 8, seed=29, dtype=dtype)
    x[1] = float("-inf")
    x[2, 5] = float("nan")
    x[3, 6] = float("inf")
    x[4, int(ids[4, 1])] = float("-inf")
    y[5, 1] = np.nan
    e, a = engine(0), (dev(x), dev(ids), dev(y))
    loss, state = e.distill_forward(*a, tail=tail)
    alone, none = e.distill_forward(*a, tail=tail, want_state=False)
    assert state is not None and none is None
    assert torch.equal(loss.view(torch.int32), alone.view(torch.int32))
    assert loss.isnan().tolist() == [r in (1, 2, 3, 5) for r in range(12)] and loss[4].isinf()


@pytest.mark.parametrize("v", [700, 131077])
@pytest.mark.parametrize("tail", [False, True])
def test_logits_next_to_the_largest_number(v, tail):
    """Logits whose product with log2(e) leaves binary32; their neighbours are 2e31 away."""
    x, ids, y = case(4, v, 8, seed=25)
    for r, top in enumerate((3e38, 2.5e38, -3e38, 1e30)):
        x[r] = -3.3e38
        x[r, ::3] = top
        x[r, ids[r].astype(np.int64)] = top
    check(x, ids, y, tail=tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("base", [3e4, 1e6, 1.1e7, 1.2e7, 3e7, 1e9, -1e6, -2e7])
def test_logits_far_from_zero(base, tail):
    """A common offset, on both sides of 2^24 / log2(e); the logits are what binary32 leaves of them."""
    x, ids, y = case(6, 3001, 8, seed=26, spread=4.0)
    check(x + base, ids, y, tail=tail, temperature=1.0)
    check(x + base, ids, y, tail=tail, temperature=2.0)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [1e-4, 0.03, 0.3, 1.5, 70.0, 1e6, 1e30])
@pytest.mark.parametrize("base", [0.0, 1000.0, -1e6])
def test_temperatures(temperature, base, tail):
    """v = x / T is rounded once, for listed and unlisted tokens alike."""
    x, ids, y = case(6, 3001, 8, seed=27)
    check(x + base, ids, y, tail=tail, temperature=temperature)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment_of_long_rows(dtype):
    rows, v = 3, 131077 * (1 if dtype is torch.float32 else 2)
    x, ids, y = case(rows, v, 12, seed=52, dtype=dtype)
    up = np.ones(rows, np.float32)
    want = R.batch(x.float().numpy(), ids, y, None, 1.0, True)
    e = engine(0)
    for offset in (0, 1, 4, 7):
        buf = torch.full((rows * (v + 21) + 16,), float("nan"), dtype=dtype, device="cuda")
        view = torch.as_strided(buf, (rows, v), (v + 21, 1), offset)
        view.copy_(x)
        loss, grad = e.distill_step(view, dev(ids), dev(y), dev(up), tail=True)
        close_loss(loss, want[0])
        close_grad(grad, want, up, 1.0, True)
        e.distill_step(view, dev(ids), dev(y), dev(up), tail=True, out=view)
        assert torch.equal(view, grad)
        gap = torch.ones_like(buf, dtype=torch.bool)
        torch.as_strided(gap, (rows, v), (v + 21, 1), offset).fill_(False)
        assert buf[gap].isnan().all()


def test_rows_far_apart():
    """Row offsets that pass 32 bits, in elements and in bytes."""
    rows, v, pitch = 3, 5003, 1200000007
    x, ids, y = case(rows, v, 12, seed=53, dtype=torch.bfloat16)
    up = np.ones(rows, np.float32)
    want = R.batch(x.float().numpy(), ids, y, None, 1.0, False)
    buf = torch.empty(2 * pitch + v, dtype=torch.bfloat16, device="cuda")
    view = torch.as_strided(buf, (rows, v), (pitch, 1))
    view.copy_(x)
    loss, grad = engine(0).distill_step(view, dev(ids), dev(y), dev(up))
    close_loss(loss, want[0])
    close_grad(grad, want, up, 1.0, False)
    engine(0).distill_step(view, dev(ids), dev(y), dev(up), out=view)
    assert torch.equal(view, grad)


def test_nearly_all_mass_on_the_listed_tokens():
    """The unlisted share is 1e-9 to 1e-13: it is summed as such, not as 1 minus the rest."""
    x, ids, y = case(4, 3000, 10, seed=31, spread=1.0, held=1 - 1e-6)
    for r in range(4):
        x[r, ids[r].astype(np.int64)] += 25.0 + 2 * r
    check(x, ids, y, tail=True)


def test_probabilities_that_add_up_to_more_than_one():
    x, ids, y = case(3, 400, 10, seed=41, held=1.0)
    y[0] += 0.3
    y[1] += 1e-6
    check(x, ids, y, tail=True)
    y[2] += 500.0                             # logits of any offset, renormalised
    check(x, ids, y, tail=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    rows, v, k = 5, 1003, 12
    x, ids, y = case(rows, v, k, seed=51, dtype=dtype)
    up = np.ones(rows, np.float32)
    want = R.batch(x.float().numpy(), ids, y, None, 1.0, True)
    e = engine(0)
    for offset in range(0, 9):
        buf = torch.full((rows * (v + 21) + 16,), float("nan"), dtype=dtype, device="cuda")
        view = torch.as_strided(buf, (rows, v), (v + 21, 1), offset)
        view.copy_(x)
        loss, grad = e.distill_step(view, dev(ids), dev(y), dev(up), tail=True)
        close_loss(loss, want[0])
        close_grad(grad, want, up, 1.0, True)
        before = buf.clone()
        e.distill_step(view, dev(ids), dev(y), dev(up), tail=True, out=view)
        assert ((view == grad) | (view.isnan() & grad.isnan())).all()
        # What lies between the rows is left as it was.
        gap = torch.ones_like(buf, dtype=torch.bool)
        torch.as_strided(gap, (rows, v), (v + 21, 1), offset).fill_(False)
        assert torch.equal(buf[gap].isnan(), before[gap].isnan())
    # Leading dimensions, and one row broadcast to many.
    z = dev(x[0]).requires_grad_()
    wide = z.expand(2, rows, v)
    loss = distill_loss(wide, dev(ids).expand(2, -1, -1).contiguous(), dev(y).expand(2, -1, -1).contiguous(),
                        tail=True)
    assert loss.shape == (2, rows)
    loss.sum().backward()
    one = R.batch(np.repeat(x[:1].float().numpy(), rows, 0), ids, y, None, 1.0, True)
    # Ten row gradients, each rounded to the type, added up in it: twenty roundings, of at most
    # half the smallest subnormal where the values are that small (in f16, below 6e-5).
    total = 2 * one[1].sum(0)
    limit = 20 * (1.3e-5 + torch.finfo(dtype).eps) * (np.abs(one[1]).sum(0) + 1e-6)
    limit += 20 * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    assert (np.abs(z.grad.float().cpu().numpy() - total) < limit).all()


@pytest.mark.parametrize("tail", [False, True])
def test_gradient_is_the_slope_of_the_loss(tail):
    """Along a direction d with |d| <= 1, central differences of step h = 1/16 are off by at most
    h^2 / 6 of a third derivative below 1, and by 1.5e-5 / h from the losses' own error."""
    x, ids, y = case(8, 600, 16, seed=61)
    d = torch.from_numpy(np.random.default_rng(62).uniform(-1, 1, size=x.shape)).float()
    h = 1 / 16
    e = engine(0)
    a = (dev(ids), dev(y))
    up = e.distill_forward(dev(x + h * d), *a, tail=tail)[0].double()
    down = e.distill_forward(dev(x - h * d), *a, tail=tail)[0].double()
    _, grad = e.distill_step(dev(x), *a, torch.ones(8, device="cuda"), tail=tail)
    slope = (grad.double() * dev(d).double()).sum(1)
    assert ((up - down) / (2 * h) - slope).abs().max() < h * h / 6 + 1.5e-5 / h + 1e-4


def test_results_do_not_depend_on_the_batch_or_the_run():
    x, ids, y = case(40, 9001, 32, seed=71, dtype=torch.bfloat16)
    e = engine(0)
    up = torch.ones(40, device="cuda")
    loss, grad = e.distill_step(dev(x), dev(ids), dev(y), up, tail=True)
    again = e.distill_step(dev(x), dev(ids), dev(y), up, tail=True)
    assert torch.equal(loss, again[0]) and torch.equal(grad, again[1])
    # A row alone is spread over more CTAs: the same to the tolerance of its sums.
    want = R.batch(x.float().numpy(), ids, y, None, 1.0, True)
    for i in range(0, 40, 13):
        l1, g1 = e.distill_step(dev(x[i:i + 1]), dev(ids[i:i + 1]), dev(y[i:i + 1]), up[:1], tail=True)
        one = [w[i:i + 1] for w in want]
        close_loss(l1, one[0])
        close_grad(g1, one, np.ones(1, np.float32), 1.0, True)


def test_streams_and_graphs():
    e = engine(0)
    sets = [[dev(a) for a in case(9, 6007, 24, seed=81 + k, dtype=torch.bfloat16)] for k in range(2)]
    up = torch.full((9,), 0.25, device="cuda")
    want = [e.distill_step(*s, up, tail=True) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, a in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append(e.distill_step(*a, up, tail=True))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    # Loss and backward captured through autograd, two graphs replayed in turn.
    graphs = []
    for a in sets:
        z = a[0].clone().requires_grad_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss = distill_loss(z, *a[1:], tail=True)
            grad, = torch.autograd.grad(loss, z, up)
        graphs.append((g, loss, grad))
    for _ in range(2):
        for g, _, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for (_, loss, grad), a, w in zip(graphs, sets, want):
        eager, state = e.distill_forward(*a, tail=True)
        assert torch.equal(loss, eager)
        assert torch.equal(grad, e.distill_backward(*a, state, up, tail=True))


def test_replacing_logits_that_a_graph_keeps_is_noticed():
    x, ids, y = case(3, 500, 8, seed=41)
    x, a = x.cuda().requires_grad_(), (dev(ids), dev(y))
    logits = x * 1.0
    loss = distill_loss(logits, *a)
    with torch.no_grad():
        engine(0).distill_step(logits, *a, torch.ones(3, device="cuda"), out=logits)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.sum().backward()


def test_teacher_records_of_the_sampler():
    """The lists come from sample_ex as they are: survivors, their log-probabilities, their count."""
    rows, v = 6, 4001
    rng = np.random.default_rng(91)
    teacher = torch.from_numpy((rng.normal(size=(rows, v)) * 3).astype(np.float32)).cuda()
    student = teacher + torch.from_numpy(rng.normal(size=(rows, v)).astype(np.float32)).cuda()
    e = engine(0)
    out = e.sample_ex(teacher, SamplingParams(1.5, 40, 0.9), uniforms=torch.zeros(rows, device="cuda"),
                      survivor_cap=64, logprobs=True)
    n, ids, logprobs = out[3], out[4], out[8]
    for tail in (False, True):
        up = torch.full((rows,), 1 / rows, device="cuda")
        loss, grad = e.distill_step(student, ids, logprobs, up, n=n, temperature=1.5, tail=tail)
        want = R.batch(student.cpu().numpy(), ids.cpu().numpy(), logprobs.cpu().numpy(),
                       n.cpu().numpy(), 1.5, tail)
        close_loss(loss, want[0])
        close_grad(grad, want, up.cpu().numpy(), 1.5, tail)


def test_refusals_of_the_library():
    import ctypes
    e = engine(0)
    x, ids, y = (dev(a) for a in case(3, 64, 4, seed=1))
    up, loss = torch.ones(3, device="cuda"), torch.empty(3, device="cuda")
    state, grad = torch.empty(3, 4, device="cuda"), torch.empty(3, 64, device="cuda")

    def call(loss=loss.data_ptr(), state=state.data_ptr(), up=up.data_ptr(), grad=grad.data_ptr(),
             stride=64, back=False, **fields):
        b = _lib.RscDistillBatch(3, 64, x.data_ptr(), 64, _lib.RSC_F32, 0, 1.0, 4, None, ids.data_ptr(),
                                 y.data_ptr())
        for k, v in fields.items():
            setattr(b, k, v)
        if back:
            return e.lib.rsc_distill_backward(e.handle, ctypes.byref(b), state, up, grad, stride, None)
        return e.lib.rsc_distill(e.handle, ctypes.byref(b), loss, state, up, grad, stride, None)

    arg, shape = _lib.RSC_ERR_INVALID_ARGUMENT, _lib.RSC_ERR_INVALID_SHAPE
    assert call() == _lib.RSC_OK
    assert call(back=True) == _lib.RSC_OK
    assert call(rows=0, d_logits=None) == _lib.RSC_OK
    assert call(state=None) == _lib.RSC_OK
    assert call(loss=None) == arg
    assert call(up=None) == arg
    assert call(state=state.data_ptr() + 4) == arg
    assert call(back=True, state=None) == arg
    assert call(back=True, grad=None) == arg
    assert call(dtype=3) == arg
    assert call(d_logits=None) == arg
    assert call(d_logits=x.data_ptr() + 2) == arg
    assert call(grad=grad.data_ptr() + 1) == arg
    assert call(d_ids=None) == arg
    assert call(d_logprobs=None) == arg
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-45):
        assert call(temperature=t) == arg
    assert call(row_stride=63) == shape
    assert call(stride=63) == shape
    assert call(grad=x.data_ptr(), stride=65) == shape
    assert call(vocab=0) == shape
    assert call(vocab=(1 << 23) + 1) == _lib.RSC_ERR_VOCAB_TOO_LARGE
    assert call(cap=1025) == _lib.RSC_ERR_CAPACITY
    assert call(rows=(1 << 27) + 1) == _lib.RSC_ERR_CAPACITY
    torch.cuda.synchronize()
