"""Draft verification on the GPU against the binary64 form of verify_ref.py. Tokens, accepted counts
and statuses are whole numbers and have to be equal: the device decides as exact arithmetic does up
to 1e-13 relative, and of the at most 1e4 decisions below, each with uniforms that are multiples of
2^-24 or 2^-32, none is expected within that of an edge."""

import numpy as np
import pytest
import torch

from rusticide_b200 import Sampler, SamplingParams, _lib, engine

from . import verify_ref as R

pytestmark = pytest.mark.gpu

FULL = SamplingParams(1.0, 0, 1.0)


def case(b, d, v, seed, draft=True, spread=2.0, noise=0.5):
    """Logits, drafts and uniforms of a batch; tokens drawn from the draft's rows."""
    rng = np.random.default_rng(seed)
    x = (rng.normal(size=(b, d + 1, v)) * spread).astype(np.float32)
    y = (x[:, :d] + noise * rng.normal(size=(b, d, v))).astype(np.float32)
    g = rng.gumbel(size=(b, d, v))
    t = (y + g).argmax(2).astype(np.int32) if d else np.zeros((b, 0), np.int32)
    u = rng.random((b, d + 1), dtype=np.float32)
    return x, (y if draft else None), t, u


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def run(x, y, t, u, params=FULL, n=None, **kw):
    out = engine(0).verify(dev(x), dev(t), params, uniforms=dev(u), draft_logits=dev(y),
                           n_draft=dev(n), **kw)
    torch.cuda.synchronize()
    return [o.cpu().numpy() for o in out]


def same(got, want):
    for g, w, what in zip(got, want, ("tokens", "accepted", "status")):
        np.testing.assert_array_equal(g, w, err_msg=what)


@pytest.mark.parametrize("v", [1, 2, 3, 31, 33, 1000, 2049, 4097, 50001])
@pytest.mark.parametrize("b,d", [(1, 1), (3, 4), (2, 0), (1, 20)])
@pytest.mark.parametrize("draft", [True, False])
def test_sizes(b, d, v, draft):
    x, y, t, u = case(b, d, v, seed=b * 1000 + d * 100 + v, draft=draft)
    same(run(x, y, t, u), R.verify_batch(x, y, t, None, u, 1.0))


@pytest.mark.parametrize("temperature", [0.25, 0.8, 1.3, 7.0])
@pytest.mark.parametrize("draft", [True, False])
def test_ragged_batches(temperature, draft):
    b, d, v = 40, 6, 3001
    x, y, t, u = case(b, d, v, seed=5, draft=draft)
    n = np.random.default_rng(6).integers(-2, d + 3, size=b).astype(np.int32)
    want = R.verify_batch(x, y, t, n, u, temperature)
    # What lies behind a sequence's drafts is not looked at.
    for i in range(b):
        k = int(np.clip(n[i], 0, d))
        x[i, k + 1:] = np.nan
        t[i, k:] = -7
        if draft:
            y[i, k:] = np.inf
    same(run(x, y, t, u, SamplingParams(temperature, 0, 1.0), n=n), want)
    # More sequences than the GPU has SMs: one CTA draws for a sequence.
    reps = 10
    big = [np.concatenate([a] * reps) if a is not None else None for a in (x, y, t, u, n)]
    got = run(*big[:4], SamplingParams(temperature, 0, 1.0), n=big[4])
    same(got, [np.concatenate([w] * reps) for w in want])


def test_flat_rows_are_drawn_exactly():
    """Equal weights over a large vocabulary: the drawn index is floor(u * V), whose neighbours are
    1 / V away, far below binary32's reach in a running sum of this length."""
    b, v = 64, 151936
    x = np.zeros((b, 1, v), np.float32)
    u = np.random.default_rng(0).random((b, 1), dtype=np.float32)
    got = run(x, None, np.zeros((b, 0), np.int32), u)
    edge = u[:, 0].astype(np.float64) * v
    assert np.abs(edge - np.round(edge)).min() > 1e-4
    np.testing.assert_array_equal(got[0][:, 0], np.floor(edge).astype(np.int32))


def test_residual_over_a_large_flat_vocabulary():
    b, d, v = 4, 1, 151936
    x, y, t, u = case(b, d, v, seed=9, spread=0.5, noise=0.5)
    u[:, 0] = np.float32(1 - 2.0 ** -24)  # refuse whatever can be refused
    want = R.verify_batch(x, y, t, None, u, 1.0)
    assert (want[1] == 0).any()
    same(run(x, y, t, u), want)


def test_equal_distributions_accept_every_token():
    """p = q: u < 1 accepts, by a margin of 2^-24 that the binary32 sums cannot see."""
    b, d, v = 5, 6, 20011
    x, _, t, u = case(b, d, v, seed=11)
    y = x[:, :d].copy()
    u[:, :d] = np.float32(1 - 2.0 ** -24)
    got = run(x, y, t, u)
    same(got, R.verify_batch(x, y, t, None, u, 1.0))
    assert (got[1] == d).all()


@pytest.mark.parametrize("v", [6, 15, 42, 1003, 20001])
def test_equal_rows_leave_nothing_whatever_their_alignment(v):
    """A token outside the vocabulary is refused; where the draft's row is the target's, nothing is
    left of it and the last token is drawn from the row itself."""
    b, d = 24, 3
    rng = np.random.default_rng(v)
    for spread in (0.05, 0.7, 6.0):
        x = (rng.normal(size=(b, d + 1, v)) * spread).astype(np.float32)
        y = x[:, :d].copy()
        t = rng.integers(0, v, size=(b, d)).astype(np.int32)
        t[np.arange(b), rng.integers(0, d, size=b)] = [-1, v] * (b // 2)
        u = rng.random((b, d + 1), dtype=np.float32)
        same(run(x, y, t, u, SamplingParams(0.7, 0, 1.0)), R.verify_batch(x, y, t, None, u, 0.7))


def test_edges_of_a_test():
    """u exactly at p / q refuses (the test is strict); one step below accepts."""
    v = 4
    x = np.log(np.array([1, 2, 4, 1], np.float64) / 8).astype(np.float32)
    x = np.zeros((1, 2, v), np.float32)          # p = 1/4 each, exactly
    y = np.full((1, 1, v), -np.inf, np.float32)
    y[0, 0, 2] = 3.0                             # q = 1 at token 2
    t = np.array([[2]], np.int32)
    for u0, accepted in ((0.25, 0), (np.nextafter(np.float32(0.25), np.float32(0)), 1), (0.0, 1)):
        u = np.array([[u0, 0.5]], np.float32)
        for q in (y, None):
            got = run(x, q, t, u)
            assert got[1][0] == accepted
            same(got, R.verify_batch(x, q, t, None, u, 1.0))


def test_masked_tokens_nan_and_infinities():
    b, d, v = 12, 3, 777
    x, y, t, u = case(b, d, v, seed=21)
    rng = np.random.default_rng(22)
    x[rng.random(x.shape) < 0.5] = -np.inf
    y[rng.random(y.shape) < 0.5] = -np.inf
    x[rng.random(x.shape) < 0.05] = np.nan
    x[0, 0] = -np.inf                 # no distribution at the first test
    x[1, 0, 5] = np.inf               # nor with a logit of +inf
    y[2, 0] = np.nan                  # nor for the draft
    y[3, 0, 7] = np.inf
    x[4, 2] = -np.inf                 # needed only if two tokens pass
    x[5, :, :] = -np.inf
    x[5, :, 3] = 1.0                  # one token left: it is drawn
    y[5, :, :] = -np.inf
    y[5, :, 3] = 1.0
    t[5] = 3
    x[6] = np.finfo(np.float32).min   # masks of the type's lowest value
    x[6, :, 9] = 0.0
    x[7] = np.finfo(np.float32).max   # differences that leave binary32
    x[7, :, ::2] = np.finfo(np.float32).min
    t[8] = [v, v + 5, -1]             # outside the vocabulary
    t[9, 0] = np.int32(2 ** 31 - 1)
    y[10] = x[10, :d]                 # equal rows, a token outside both
    x[10, 0, t[10, 0]] = y[10, 0, t[10, 0]] = -np.inf
    for q in (y, None):
        same(run(x, q, t, u), R.verify_batch(x, q, t, None, u, 1.0))


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_strides_and_alignment(offset):
    b, d, v = 3, 2, 5003
    x, y, t, u = case(b, d, v, seed=31)
    want = R.verify_batch(x, y, t, None, u, 1.0)
    eng = engine(0)

    def spread(a, order):
        """The values at `offset` floats into a wider allocation, sequences or rows slowest."""
        s0, s1, _ = a.shape
        pitch = v + 13 + offset
        buf = torch.full((s0 * s1 * pitch + 8,), float("nan"), device="cuda")
        strides = (s1 * pitch, pitch, 1) if order else (pitch, s0 * pitch, 1)
        view = torch.as_strided(buf, a.shape, strides, offset)
        view.copy_(torch.from_numpy(a))
        return view

    for order in (True, False):
        out = eng.verify(spread(x, order), dev(t), FULL, uniforms=dev(u),
                         draft_logits=spread(y, not order))
        same([o.cpu().numpy() for o in out], want)


@pytest.mark.parametrize("base", [3e4, 1e6, 3e7, 1e9, -2e7, 1e30])
def test_logits_far_from_zero(base):
    """A common offset of all logits, which binary32 rounds to ever coarser steps."""
    x, y, t, u = case(4, 3, 3001, seed=34, spread=4.0)
    x, y = (x + np.float32(base)).astype(np.float32), (y + np.float32(base)).astype(np.float32)
    same(run(x, y, t, u), R.verify_batch(x, y, t, None, u, 1.0))
    same(run(x, None, t, u), R.verify_batch(x, None, t, None, u, 1.0))


def far_case(top, v, seed, below):
    """Rows whose largest logit is `top`; the others are binary32 numbers below it, a step of
    `below` apart and more, and a third of them masked. Drafts are the draft's likeliest token, a
    masked one or, in two sequences, a token at the target's maximum."""
    b, d = 8, 2
    rng = np.random.default_rng(seed)
    top = np.float32(top)

    def rows(n):
        gap = np.abs(rng.normal(size=(b, n, v))) * below + below
        x = np.minimum(top - gap.astype(np.float32), np.nextafter(top, np.float32(-np.inf)))
        x = x.astype(np.float32)
        x[rng.random(x.shape) < 1 / 3] = -np.inf
        at = rng.integers(0, v, size=(b, n, 3))     # the maximum, three times
        np.put_along_axis(x, at, top, 2)
        return x, at

    x, at_x = rows(d + 1)
    y, at_y = rows(d)
    y[4:6, 0] = x[4:6, 0]                           # equal rows: accepted
    at_y[4:6, 0] = at_x[4:6, 0]
    t = at_y[:, :, 0].astype(np.int32)
    t[6] = at_x[6, :d, 1]
    masked = np.isneginf(x[2:4, 0])                 # of no probability, whatever the test draws
    t[2:4, 0] = masked.argmax(1)
    y[2, 0, t[2, 0]] = -np.inf                      # nor in the draft
    u = rng.random((b, d + 1), dtype=np.float32) * np.float32(0.98) + np.float32(0.01)
    u[7, :d] = np.float32(2.0 ** -24)
    return x, y, t, u


@pytest.mark.parametrize("v", [777, 40003])
@pytest.mark.parametrize("top", [2.0 ** 29, 2.0 ** 30, 1.7e9, 2.0 ** 31, 2.2e9, 3e9, 4.2e9, 2.0 ** 32,
                                 5e9, 8e9, 2.0 ** 33, 1e10, 2.0 ** 40, 1e20, 3.4e38, -1.7e9,
                                 -2.0 ** 31, -3e9, -2.0 ** 32, -5e9, -2.0 ** 33, -1e10, -2.0 ** 40])
def test_maxima_whose_neighbours_are_far_apart(top, v):
    """Binary32 numbers are 64 apart and more here. Tokens a step below the maximum, masked ones and
    the padding behind a row have no weight beside it, and none is drawn or accepted."""
    x, y, t, u = far_case(top, v, seed=35, below=abs(top) * 2e-7)
    for q in (y, None):
        want = R.verify_batch(x, q, t, None, u, 1.0)
        assert len(set(want[1])) > 1
        same(run(x, q, t, u), want)


@pytest.mark.parametrize("temperature", [1e-9, 1e-8, 1e-6, 1e-4, 1e-3])
@pytest.mark.parametrize("top", [2.2, 4.0, 10.0, 25.0, 42.9, -3.0])
def test_temperatures_near_zero(temperature, top):
    """Almost greedy sampling of ordinary logits."""
    for v in (1, 3001):
        x, y, t, u = far_case(top, v, seed=36, below=0.25)
        for q in (y, None):
            same(run(x, q, t, u, SamplingParams(temperature, 0, 1.0)),
                 R.verify_batch(x, q, t, None, u, temperature))


@pytest.mark.parametrize("low,high", [(-2.0 ** 33, -2.0 ** 33 + 512), (2.0 ** 33 - 512, 2.0 ** 33),
                                      (2.0 ** 33, 2.0 ** 33 + 1024), (2.0 ** 32 - 256, 2.0 ** 32)])
def test_equal_maxima_met_early_and_late(low, high):
    """Two tokens share the maximum; a warp meets one of them behind its first block of a row of
    neighbouring numbers, another warp in its first block. Each has half of p."""
    v = 151936
    x = np.full((4, 1, v), low, np.float32)
    x[:2, 0, [700, 2433]] = high
    x[2:, 0, [1, 150000]] = high
    u = np.array([[0.25], [0.75], [0.25], [0.75]], np.float32)
    got = run(x, None, np.zeros((4, 0), np.int32), u)
    assert got[0][:, 0].tolist() == [700, 2433, 1, 150000] and not got[2].any()


@pytest.mark.parametrize("v", [40003, 151936])
@pytest.mark.parametrize("copies", [1, 40])
def test_tokens_without_weight_are_not_drawn_for_their_number(v, copies):
    """465 below the maximum a token has no probability, and neither have a hundred thousand of them.
    A draw of u = 0 takes the first token of any probability, which is the last one here; masked
    tokens stand in front."""
    x = np.full((3, 2, v), -465.0, np.float32)
    x[:, :, :5000] = -np.inf
    x[:, :, v - 1] = 0.0
    x[1:, 0, v // 2] = 0.0                      # sequences 1 and 2: half of p each, one refused
    y = np.full((3, 1, v), -np.inf, np.float32)
    y[:, 0, v // 2] = 0.0
    t = np.full((3, 1), v // 2, np.int32)
    u = np.array([[0.5, 0.0], [0.75, 0.0], [0.75, 0.0]], np.float32)
    n = np.array([0, 1, 1], np.int32)
    many = [np.concatenate([a] * copies) for a in (x, y, t, u, n)]
    for q in (many[1], None):
        tokens, accepted, status = run(many[0], q, *many[2:4], n=many[4])
        assert not accepted.any() and not status.any()
        assert (tokens[:, 0] == v - 1).all() and (tokens[:, 1] == -1).all()


@pytest.mark.parametrize("copies", [1, 40])
def test_what_counts_as_weight_is_measured_from_the_largest_logit(copies):
    """480 below it a token has no probability, however early in the row and wherever the maximum
    stands: a draw of u = 0 passes over it."""
    v, places = 151936, [0, 600, 1500, 9000, 100100, 151935]
    x = np.zeros((len(places), 1, v), np.float32)
    for i, at in enumerate(places):
        x[i, 0, at] = 480.0
    x = np.concatenate([x] * copies)
    u = np.zeros((len(x), 1), np.float32)
    tokens, _, status = run(x, None, np.zeros((len(x), 0), np.int32), u)
    assert not status.any()
    assert tokens[:, 0].tolist() == places * copies


@pytest.mark.parametrize("v", [1003, 151936])
@pytest.mark.parametrize("copies", [1, 60])
def test_where_weight_ends(v, copies):
    """1e-200 of the largest, between 460 and 461 below it, in draws and tests of u = 0, wherever
    the maximum stands and however a row is cut."""
    for shift in (0.0, -1000.0, 77.25):
        x = np.full((4, 2, v), -np.inf, np.float32)
        for i, at in enumerate((v - 1, v // 2, v - 1, v // 3)):
            x[i, :, v // 4:] = shift - 3.0      # in front of the maximum and behind it
            x[i, :, at] = shift
            x[i, :, 1] = shift - (460.0 if i < 2 else 461.0)
        t = np.full((4, 1), 1, np.int32)
        many = [np.concatenate([a] * copies) for a in (x, t, np.zeros((4, 2), np.float32))]
        tokens, accepted, _ = run(many[0], None, *many[1:])
        want = [[1, 1], [1, 1], [v // 4, -1], [v // 4, -1]]
        assert tokens.tolist() == want * copies
        assert accepted.tolist() == [1, 1, 0, 0] * copies


def test_one_likely_token_in_both_rows():
    """A token that has all of p and all of q, to binary64's last place, leaves the unlikely ones."""
    b, v = 40, 3001
    rng = np.random.default_rng(44)
    x = (rng.normal(size=(b, 2, v)) * 2 - 60).astype(np.float32)
    y = (x[:, :1] + rng.normal(size=(b, 1, v))).astype(np.float32)
    at = rng.integers(0, v, size=b)
    for i in range(b):
        x[i, :, at[i]], y[i, 0, at[i]] = 10 * rng.random(), 10 * rng.random()
    t = np.full((b, 1), v, np.int32)            # outside: refused
    u = rng.random((b, 2), dtype=np.float32)
    want = R.verify_batch(x, y, t, None, u, 1.0)
    assert (want[0][:, 0] != at).any()
    same(run(x, y, t, u), want)


def test_rows_far_apart():
    """Offsets of sequences and rows that pass 32 bits, in elements and in bytes."""
    b, d, v, far = 2, 1, 5003, 2300000004
    x, y, t, u = case(b, d, v, seed=33)
    want = R.verify_batch(x, y, t, None, u, 1.0)
    buf = torch.empty(far + far // 2 + 3 * v, device="cuda")
    target = torch.as_strided(buf, (b, d + 1, v), (far, far // 2, 1), 0)
    draft = torch.as_strided(buf, (b, d, v), (far, v, 1), v)
    target.copy_(torch.from_numpy(x))
    draft.copy_(torch.from_numpy(y))
    out = engine(0).verify(target, dev(t), FULL, uniforms=dev(u), draft_logits=draft)
    same([o.cpu().numpy() for o in out], want)
    greedy = SamplingParams(0.0, 0, 1.0)
    out = engine(0).verify(target, dev(t), greedy)
    same([o.cpu().numpy() for o in out], R.greedy_batch(x, t, None))


@pytest.mark.parametrize("v", [1, 5, 4099, 151936])
def test_greedy(v):
    b, d = 9, 5
    rng = np.random.default_rng(v)
    x = rng.normal(size=(b, d + 1, v)).astype(np.float32)
    x[1] = np.round(x[1])                       # ties: the last index counts
    t = x[:, :d].argmax(2).astype(np.int32)
    t[1] = v - 1 - x[1, :d, ::-1].argmax(1)
    t[2, 2] = (t[2, 2] + 1) % v
    t[3, 0] = -1
    x[4, 1] = -np.inf
    x[5, 2] = np.nan
    x[6, :, 0] = np.inf                         # larger than any finite logit
    n = np.array([d, d, d, d, d, d, d, 2, 0], np.int32)
    want = R.greedy_batch(x, t, n)
    y = np.full((b, d, v), np.nan, np.float32)  # not read
    for params in (SamplingParams(0.0, 40, 0.9), SamplingParams(0.0, 0, 1.0)):
        out = engine(0).verify(dev(x), dev(t), params, n_draft=dev(n), draft_logits=dev(y))
        same([o.cpu().numpy() for o in out], want)
    # The tokens are those of the greedy call on the same rows.
    ids, _ = engine(0).greedy(dev(x).reshape(-1, v))
    ids = ids.cpu().numpy().reshape(b, d + 1)
    for i in range(b):
        if want[2][i] == 0:
            assert want[0][i, want[1][i]] == ids[i, want[1][i]]


@pytest.mark.parametrize("v", [1, 3, 4, 1027, 4096, 4097, 4098, 4099, 50001, 151936])
@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_greedy_takes_the_last_of_equal_maxima(v, offset):
    """Rows of one, two and three values, at every phase of their 16-byte words: the maximum stands
    in the head, the body and the tail of each part, and the last of them counts."""
    b, d = 6, 2
    rng = np.random.default_rng(v + offset)
    x = rng.integers(0, 3, size=(b, d + 1, v)).astype(np.float32)
    x[0] = 1.0                                  # all equal
    x[1] = np.minimum(x[1], 1.0)
    x[2] = np.where(x[2] == 2.0, np.float32(0.0), np.float32(-0.0))  # total_cmp: -0 is below +0
    x[3] = -np.inf
    x[3, :, ::2] = -4.5                         # the even tokens are left, all equal
    x[4] = np.finfo(np.float32).max             # +inf above finite logits, several times
    x[4, :, :: max(1, v // 5)] = np.inf
    x[4, :, 0] = 0.0
    pitch = v + 5 + offset
    buf = torch.zeros(b * (d + 1) * pitch + 8, device="cuda")
    view = torch.as_strided(buf, x.shape, ((d + 1) * pitch, pitch, 1), offset)
    view.copy_(torch.from_numpy(x))
    flat = torch.as_strided(buf, (b * (d + 1), v), (pitch, 1), offset)
    best = engine(0).greedy(flat)[0].cpu().numpy().reshape(b, d + 1)
    t = best[:, :d].copy()                      # drafts that have to stand
    t[5, 1] = (t[5, 1] + 1) % v if v > 1 else 1
    want = R.greedy_batch(x, t, None)
    for i in range(b):
        assert want[0][i, want[1][i]] == best[i, want[1][i]] and want[2][i] == 0
    assert (want[1][:5] == d).all()
    out = engine(0).verify(view, dev(t), SamplingParams(0.0))
    same([o.cpu().numpy() for o in out], want)


def test_top_k_of_one_is_greedy():
    b, d, v = 4, 3, 999
    x, y, t, u = case(b, d, v, seed=41)
    t[:2] = x[:2, :d].argmax(2)
    same(run(x, y, t, u, SamplingParams(0.7, 1, 0.9)), R.greedy_batch(x, t, None))


@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0, 3.0, 1e-30, -1.0])
def test_greedy_parameters_give_the_sampler_s_tokens(temperature):
    """The argmax branch of the sampler: T = 0 compares the logits themselves, top_k = 1 the scaled
    ones, where neighbouring logits can become equal and the last of them counts. What rsc_pick
    answers for a row is what its draft is compared with."""
    v, d = 1003, 1
    rng = np.random.default_rng(43)
    x = rng.normal(size=(300, d + 1, v)).astype(np.float32)
    high = (5 + 15 * rng.random(300)).astype(np.float32)
    at = np.sort(rng.choice(v, size=(300, 2)), axis=1)
    for i in range(200):                        # the two largest are neighbours, the larger one first
        x[i, :, at[i, 0]], x[i, :, at[i, 1]] = np.nextafter(high[i], np.float32(99)), high[i]
    x[200, 0, 5] = np.inf
    x[201] = -np.inf
    x[202, 0] = np.nan
    x[203, 0, ::2] = -np.inf
    x[204, 0] = 1e-45                           # equal after a product that underflows
    x[204, 0, 7] = 3e-45
    x[205, 0] = -np.inf
    x[205, 0, 3] = np.inf
    x[206] = 3e38
    params = SamplingParams(temperature, 1, 1.0)
    rows = dev(x).reshape(-1, v)
    ids, status, _ = engine(0).pick(rows, params, uniforms=torch.zeros(len(rows), device="cuda"))
    ids, status = ids.cpu().numpy().reshape(300, 2), status.cpu().numpy().reshape(300, 2) & 0xFF
    t = np.where(status[:, :1] == 0, ids[:, :1], 0).astype(np.int32)
    out = engine(0).verify(dev(x), dev(t), params)
    tokens, accepted, st = [o.cpu().numpy() for o in out]
    for i in range(300):
        a = 0 if status[i, 0] else 1
        assert accepted[i] == a and st[i] == status[i, a]
        want = [-1, -1]
        if a:
            want[0] = ids[i, 0]
        if not st[i]:
            want[a] = ids[i, a]
        assert tokens[i].tolist() == want


def test_generator_states():
    """Draws from per-sequence states equal the same draws given as uniforms, and a state advances
    by what its sequence consumed."""
    b, d, v = 30, 4, 2003
    x, y, t, _ = case(b, d, v, seed=51)
    x[3, 0] = -np.inf                     # no draw at all
    x[4, d] = -np.inf                     # tests only, if all pass
    seeds = list(range(100, 100 + b))
    for draft in (y, None):
        states = engine(0).rng_seed(torch.tensor(seeds))
        got = [o.cpu().numpy() for o in engine(0).verify(
            dev(x), dev(t), FULL, rng_states=states, draft_logits=dev(draft))]
        for i in range(b):
            u = R.wyrand_uniforms(seeds[i], d + 1)
            row, acc, st, used = R.verify_one(
                lambda k: R.softmax(R.scaled(x[i, k], 1.0)),
                None if draft is None else lambda k: R.softmax(R.scaled(draft[i, k], 1.0)),
                t[i], d, u, lambda k: u[k])
            assert got[0][i, :len(row)].tolist() == [int(r) for r in row]
            assert (got[0][i, len(row):] == -1).all()
            assert (got[1][i], got[2][i]) == (acc, st)
            state = (seeds[i] + used * 0x2d358dccaa6c78a5) & ((1 << 64) - 1)
            assert int(states[i]) & ((1 << 64) - 1) == state


def test_a_sequence_does_not_depend_on_its_batch():
    b, d, v = 17, 5, 9001
    x, y, t, u = case(b, d, v, seed=61)
    whole = run(x, y, t, u)
    for i in range(b):
        one = run(x[i:i + 1], y[i:i + 1], t[i:i + 1], u[i:i + 1])
        same(one, [w[i:i + 1] for w in whole])


def test_output_distribution():
    """Over many sequences of one position the first token follows p. With N = 200000 draws a share
    is off by more than 6 standard deviations, 6 sqrt(p (1 - p) / N), with odds below 1e-8."""
    n, v = 200000, 6
    rng = np.random.default_rng(71)
    x = rng.normal(size=(1, 2, v)).astype(np.float32)
    y = rng.normal(size=(1, 1, v)).astype(np.float32)
    p, q = R.softmax(x[0, 0]), R.softmax(y[0, 0])
    t = rng.choice(v, size=(n, 1), p=q).astype(np.int32)
    u = rng.random((n, 2), dtype=np.float32)
    out = engine(0).verify(dev(x).expand(n, 2, v).contiguous(), dev(t), FULL, uniforms=dev(u),
                           draft_logits=dev(y).expand(n, 1, v).contiguous())
    share = np.bincount(out[0][:, 0].cpu().numpy(), minlength=v) / n
    assert (np.abs(share - p) < 6 * np.sqrt(p * (1 - p) / n)).all()


@pytest.mark.parametrize("draft", [True, False])
def test_large_batches(draft):
    """Several waves of row parts; what lies behind a sequence's first refused position does not
    matter, NaN neither."""
    b, d, v = 24, 8, 50003
    x, y, t, u = case(b, d, v, seed=111, draft=draft)
    n = np.random.default_rng(112).integers(0, d + 1, size=b).astype(np.int32)
    t[3, 2] = v                                   # outside the vocabulary
    x[5, 1] = -np.inf
    t[7] = x[7, :d].argmax(1)
    u[7, :d] = 0.0                                # accepts to the end
    n[7] = d
    for i in range(12, b):
        u[i, :i % (d + 1)] = 0.0                  # accepts at least these
    want = R.verify_batch(x, y, t, n, u, 1.0)
    assert len(set(want[1])) > 3
    same(run(x, y, t, u, n=n), want)
    for i in range(b):
        x[i, want[1][i] + 1:] = np.nan
    same(run(x, y, t, u, n=n), want)
    t = np.where(np.random.default_rng(113).random(t.shape) < 0.7, np.nan_to_num(x[:, :d]).argmax(2), t).astype(np.int32)
    greedy = R.greedy_batch(x, t, n)
    out = engine(0).verify(dev(x), dev(t), SamplingParams(0.0), n_draft=dev(n))
    same([o.cpu().numpy() for o in out], greedy)


def test_streams_graphs_and_reused_outputs():
    b, d, v = 6, 3, 30011
    sets = [case(b, d, v, seed=81 + k) for k in range(2)]
    want = [R.verify_batch(*s[:3], None, s[3], 1.0) for s in sets]
    ins = [[dev(a) for a in s] for s in sets]
    eng = engine(0)
    torch.cuda.synchronize()
    # Two calls in flight on two streams.
    streams = [torch.cuda.Stream() for _ in sets]
    outs = []
    for s, (x, y, t, u) in zip(streams, ins):
        with torch.cuda.stream(s):
            outs.append(eng.verify(x, t, FULL, uniforms=u, draft_logits=y))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        same([a.cpu().numpy() for a in o], w)
    # Two captured calls, replayed in turn, with outputs and inputs that are the caller's.
    graphs = []
    for x, y, t, u in ins:
        out = tuple(torch.empty_like(o) for o in outs[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = eng.verify(x, t, FULL, uniforms=u, draft_logits=y, out=out)
        assert all(a is b_ for a, b_ in zip(got, out))
        graphs.append((g, out))
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for (_, o), w in zip(graphs, want):
        same([a.cpu().numpy() for a in o], w)
    # New inputs in the captured buffers.
    for a, b_ in zip(ins[0], ins[1]):
        a.copy_(b_)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    same([a.cpu().numpy() for a in graphs[0][1]], want[1])


# ---------------------------------------------------------------------------
# Survivor records
# ---------------------------------------------------------------------------
def records(rng, rows, vocab, cap, empty=False):
    n = rng.integers(0 if empty else 1, min(cap, vocab) + 1, size=rows).astype(np.int32)
    ids = np.full((rows, cap), -1, np.int32)
    probs = np.full((rows, cap), np.nan, np.float32)
    for r in range(rows):
        k = int(n[r])
        ids[r, :k] = np.sort(rng.choice(vocab, size=k, replace=False))
        w = rng.random(k) ** 3 + 1e-3
        probs[r, :k] = (w / w.sum()).astype(np.float32) if k else 0
    return n, ids, probs


@pytest.mark.parametrize("b,d,vocab,cap", [(1, 1, 4, 1), (1, 4, 40, 16), (50, 3, 64, 40),
                                           (20, 9, 300, 152), (3, 2, 5000, 1500), (5, 0, 30, 8)])
@pytest.mark.parametrize("with_draft", [True, False])
def test_records(b, d, vocab, cap, with_draft):
    rng = np.random.default_rng(b * 100 + d + cap)
    target = records(rng, b * (d + 1), vocab, cap)
    draft = records(rng, b * d, vocab, cap) if with_draft else None
    t = rng.integers(0, vocab, size=(b, d)).astype(np.int32)
    for i in range(b):  # most tokens come from the target's list, some from neither
        for k in range(d):
            if rng.random() < 0.8:
                row = i * (d + 1) + k
                t[i, k] = target[1][row, rng.integers(0, target[0][row])]
    u = rng.random((b, d + 1), dtype=np.float32)
    n = rng.integers(0, d + 1, size=b).astype(np.int32)
    out = engine(0).verify_survivors([dev(a) for a in target], dev(t), uniforms=dev(u),
                                     draft=None if draft is None else [dev(a) for a in draft],
                                     n_draft=dev(n))
    same([o.cpu().numpy() for o in out], R.verify_records(target, draft, vocab, t, n, u))


def test_records_that_hold_no_distribution():
    rng = np.random.default_rng(1)
    b, d, vocab, cap = 6, 2, 50, 8
    target, draft = records(rng, b * (d + 1), vocab, cap), records(rng, b * d, vocab, cap)
    t = np.tile(target[1].reshape(b, d + 1, cap)[:, :d, 0], 1).astype(np.int32)
    u = np.zeros((b, d + 1), np.float32)  # u = 0 accepts every listed token
    status = np.zeros(b * (d + 1), np.int32)
    target[0][0] = 0                        # sequence 0, row 0: empty
    target[0][1 * 3 + 1] = cap + 1          # sequence 1, row 1: more survivors than slots
    status[2 * 3 + 2] = 0x102               # sequence 2, last row: a status, with a flag above it
    draft[0][3 * 2 + 1] = cap + 3           # sequence 3, draft row 1
    target[2][4 * 3 + 2, :] = 0.0           # sequence 4, last row: no weight
    out = engine(0).verify_survivors([dev(a) for a in target] + [dev(status)], dev(t),
                                     uniforms=dev(u), draft=[dev(a) for a in draft])
    tokens, accepted, st = [o.cpu().numpy() for o in out]
    assert accepted.tolist() == [0, 1, 2, 1, 2, 2]
    assert st.tolist() == [_lib.RSC_ROW_NO_VALID_TOKENS, _lib.RSC_ROW_INTERNAL, 2,
                           _lib.RSC_ROW_INTERNAL, _lib.RSC_ROW_NO_VALID_TOKENS, 0]
    for i in range(5):
        assert tokens[i, :accepted[i]].tolist() == t[i, :accepted[i]].tolist()
        assert (tokens[i, accepted[i]:] == -1).all()


@pytest.mark.parametrize("params", [SamplingParams(0.8, 40, 0.95), SamplingParams(1.0, 0, 0.9),
                                    SamplingParams(1.2, 100, 1.0)])
@pytest.mark.parametrize("draft", [True, False])
def test_filtered_parameters(params, draft):
    """Engine.verify with top-k and top-p: the distributions are the sampler's own survivors."""
    b, d, v = 8, 4, 3001
    x, y, t, u = case(b, d, v, seed=91, draft=draft, spread=3.0)
    eng = engine(0)

    def survivors(a):
        rows = a.reshape(-1, v)
        out = eng.sample_ex(dev(rows), params, uniforms=torch.zeros(len(rows), device="cuda"),
                            survivor_cap=v)
        return [o.cpu().numpy() for o in (out[3], out[4], out[5])]

    want = R.verify_records(survivors(x), survivors(y) if draft else None, v, t, None, u)
    same(run(x, y, t, u, params), want)
    states = eng.rng_seed(torch.arange(b))
    st0 = states.clone()
    out = eng.verify(dev(x), dev(t), params, rng_states=states,
                     draft_logits=dev(y) if draft else None)
    u2 = np.zeros((b, d + 1), np.float32)
    for i in range(b):  # the last draw takes the uniform behind the tests
        us = R.wyrand_uniforms(int(st0[i]), d + 1)
        u2[i, :d] = us[:d]
        acc = int(out[1][i])
        u2[i, d] = us[acc + (acc < d)]
    same([o.cpu().numpy() for o in out],
         R.verify_records(survivors(x), survivors(y) if draft else None, v, t, None, u2))


def test_sampler_verify_follows_the_generator():
    v, d = 500, 3
    x, y, t, _ = case(1, d, v, seed=101)
    s = Sampler(7)
    first = s.verify(dev(x[0]), t[0].tolist(), FULL, draft_logits=dev(y[0]))
    u = R.wyrand_uniforms(7, 2 * (d + 1))
    row, _, _, used = R.verify_one(lambda k: R.softmax(x[0, k]), lambda k: R.softmax(y[0, k]),
                                   t[0], d, u, lambda k: u[k])
    assert first == [int(r) for r in row]
    second = s.verify(dev(x[0]), t[0].tolist(), FULL, draft_logits=dev(y[0]))
    row, _, _, _ = R.verify_one(lambda k: R.softmax(x[0, k]), lambda k: R.softmax(y[0, k]), t[0],
                                d, u[used:], lambda k: u[used + k])
    assert second == [int(r) for r in row]
    assert s.verify(dev(x[0, :1]), [], SamplingParams(0.0)) == [int(x[0, 0].argmax())]
    assert len(s.verify(dev(x[0]), t[0].tolist(), SamplingParams())) >= 1


@pytest.mark.parametrize("params", [SamplingParams(-1.0, 0, 1.0), SamplingParams(float("inf"), 0, 1.0),
                                    SamplingParams(float("nan"), 0, 1.0), SamplingParams(1e-45, 0, 1.0)])
def test_parameters_without_a_distribution_are_refused(params):
    x, y, t, u = case(1, 1, 8, seed=1)
    with pytest.raises(_lib.RscError) as e:
        run(x, y, t, u, params)
    assert e.value.code == _lib.RSC_ERR_INVALID_ARGUMENT


def test_refusals_of_the_library():
    import ctypes
    eng = engine(0)
    x, y, t, u = (dev(a) for a in case(2, 2, 64, seed=1))
    lib, work = eng.lib, torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    o = torch.empty(64, dtype=torch.int32, device="cuda")

    def call(params=FULL, uniforms=u.data_ptr(), states=None, wptr=work.data_ptr(), wbytes=1 << 16,
             out=o.data_ptr(), **fields):
        b = _lib.RscDraftBatch(2, 2, 64, x.data_ptr(), 3 * 64, 64, y.data_ptr(), 2 * 64, 64,
                               t.data_ptr(), None)
        for k, v in fields.items():
            setattr(b, k, v)
        c = params.to_c()
        return lib.rsc_verify(eng.handle, ctypes.byref(b), ctypes.byref(c), uniforms, states, wptr,
                              wbytes, out, out, out, None)

    assert call() == _lib.RSC_OK
    assert call(n_seqs=0, d_target=None) == _lib.RSC_OK
    arg, shape = _lib.RSC_ERR_INVALID_ARGUMENT, _lib.RSC_ERR_INVALID_SHAPE
    assert call(SamplingParams(1.0, 40, 1.0)) == arg        # a filtered distribution
    assert call(SamplingParams(1.0, 0, 0.9)) == arg
    assert call(uniforms=None) == arg
    assert call(wbytes=16) == arg
    assert call(wptr=None) == arg
    assert call(wptr=work.data_ptr() + 4) == arg
    assert call(out=None) == arg
    assert call(d_target=None) == arg
    assert call(d_target=x.data_ptr() + 1) == arg
    assert call(d_draft=y.data_ptr() + 2) == arg
    assert call(d_draft_tokens=None) == arg
    assert call(vocab=0) == shape
    assert call(target_row_stride=63) == shape
    assert call(target_seq_stride=63) == shape
    assert call(draft_row_stride=0) == shape
    assert call(draft_seq_stride=0) == shape
    assert call(vocab=1 << 31) == _lib.RSC_ERR_VOCAB_TOO_LARGE
    assert call(n_seqs=1 << 27) == _lib.RSC_ERR_CAPACITY
    assert call(n_seqs=1 << 40, max_drafts=1 << 40) == _lib.RSC_ERR_CAPACITY
    torch.cuda.synchronize()
