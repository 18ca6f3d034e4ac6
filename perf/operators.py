"""The operators around the sampler that serve and train a draft model, as cases to measure.

Three families of calls:

* verify: drafted tokens checked against the target model's logits (the whole vocabulary, at a
  temperature; greedy at temperature 0), the first refused one replaced by a draw from the residual;
* survivors: the same check on filtered distributions, given as the survivor records (ids,
  probabilities) that a sampling call with top-k and top-p writes;
* distill: the loss of a student's logits against a teacher's top log-probabilities, alone
  ("forward"), with its gradient in the same call ("step"), or through autograd ("autograd").

With `own` false, `run` computes each in elementary torch operations; with `own` true it makes the
calls a user makes of this package. `exact` states the same results once more, row by row, in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One stream, four drafted tokens: the latency of a single user's decode step.
        {"name": "verify one stream", "kind": "verify", "seqs": 1, "drafts": 4, "vocab": 32000,
         "temperature": 0.8, "draft_rows": True, "ragged": False},
        # A few concurrent streams on the vocabulary of the headline benchmark.
        {"name": "verify small batch", "kind": "verify", "seqs": 8, "drafts": 5, "vocab": 151936,
         "temperature": 1.0, "draft_rows": True, "ragged": False},
        # A serving batch in which every sequence drafted its own number of tokens.
        {"name": "verify serving batch", "kind": "verify", "seqs": 96, "drafts": 7,
         "vocab": 128256, "temperature": 0.7, "draft_rows": True, "ragged": True},
        # Drafts looked up in the prompt: no draft distribution; a vocabulary of odd size.
        {"name": "verify prompt lookup", "kind": "verify", "seqs": 32, "drafts": 8, "vocab": 50001,
         "temperature": 1.0, "draft_rows": False, "ragged": True},
        # Greedy decoding with drafts: the tokens must equal the rows' largest logits.
        {"name": "verify greedy", "kind": "verify", "seqs": 64, "drafts": 4, "vocab": 151936,
         "temperature": 0.0, "draft_rows": False, "ragged": False},
        # The default filter (top-k 40) for one stream: records of up to 64 survivors.
        {"name": "survivors one stream", "kind": "survivors", "seqs": 1, "drafts": 4,
         "vocab": 32000, "top_k": 40, "cap": 64, "draft_rows": True, "ragged": False},
        # A large batch at the widest streaming top-k.
        {"name": "survivors large batch", "kind": "survivors", "seqs": 512, "drafts": 6,
         "vocab": 151936, "top_k": 128, "cap": 152, "draft_rows": True, "ragged": True},
        # Evaluation of one position: the smallest call.
        {"name": "distill one row", "kind": "distill", "call": "forward", "rows": 1,
         "vocab": 32000, "top": 20, "dtype": "f32", "tail": False, "temperature": 1.0,
         "ragged": False},
        # A small micro-batch in half precision, odd sizes, lists of differing length.
        {"name": "distill f16 step", "kind": "distill", "call": "step", "rows": 37,
         "vocab": 50001, "top": 33, "dtype": "f16", "tail": True, "temperature": 2.0,
         "ragged": True},
        # Autograd in binary32 over an odd vocabulary, renormalised targets.
        {"name": "distill f32 autograd", "kind": "distill", "call": "autograd", "rows": 1000,
         "vocab": 32001, "top": 100, "dtype": "f32", "tail": False, "temperature": 1.0,
         "ragged": True},
        # Validation over a long batch: the loss alone, with the tail of the distribution.
        {"name": "distill bf16 forward", "kind": "distill", "call": "forward", "rows": 4096,
         "vocab": 128256, "top": 128, "dtype": "bf16", "tail": True, "temperature": 1.0,
         "ragged": False},
        # A training micro-batch: 2048 positions of the headline vocabulary.
        {"name": "distill bf16 step", "kind": "distill", "call": "step", "rows": 2048,
         "vocab": 151936, "top": 64, "dtype": "bf16", "tail": False, "temperature": 1.0,
         "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "survivors", "distill", "distill"])
    if kind == "verify":
        c = {"kind": kind, "seqs": _log_int(rng, 1, 128), "drafts": rng.randint(1, 8),
             "vocab": _log_int(rng, 1000, 160000),
             "temperature": rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]),
             "draft_rows": rng.random() < 0.6, "ragged": rng.random() < 0.5}
        c["draft_rows"] = c["draft_rows"] and c["temperature"] > 0
        # At most the largest listed case's bytes.
        while c["seqs"] * (2 * c["drafts"] + 1) * c["vocab"] > 96 * 15 * 128256:
            c["seqs"] = max(1, c["seqs"] // 2)
        return c
    if kind == "survivors":
        k = rng.randint(2, 128)
        return {"kind": kind, "seqs": _log_int(rng, 1, 512), "drafts": rng.randint(1, 6),
                "vocab": _log_int(rng, 1000, 160000), "top_k": k, "cap": k + rng.randint(0, 24),
                "draft_rows": rng.random() < 0.7, "ragged": rng.random() < 0.5}
    c = {"kind": kind, "call": rng.choice(["forward", "step", "autograd"]),
         "rows": _log_int(rng, 1, 4096), "vocab": _log_int(rng, 1000, 160000),
         "top": rng.randint(1, 128), "dtype": rng.choice(["f32", "bf16", "f16"]),
         "tail": rng.random() < 0.5, "temperature": rng.choice([1.0, 1.5, 2.0]),
         "ragged": rng.random() < 0.5}
    while c["rows"] * c["vocab"] * (2 if c["dtype"] == "f32" else 1) > 2048 * 151936:
        c["rows"] = max(1, c["rows"] // 2)
    return c


def _mean_drafts(case):
    """Drafted tokens a sequence has on average: ragged batches draw 0..D evenly."""
    return case["drafts"] / 2 if case["ragged"] else case["drafts"]


def work(case):
    if case["kind"] == "verify":
        # Every row of the call read once. A call may need fewer: the rows behind a sequence's
        # first refused token do not matter, and where that is depends on the data.
        n = _mean_drafts(case)
        rows = case["seqs"] * (n + 1 + (n if case["draft_rows"] else 0))
        outs = case["seqs"] * (case["drafts"] + 3) * 4
        return {"bytes": rows * case["vocab"] * 4 + outs, "flops": 3 * rows * case["vocab"]}
    if case["kind"] == "survivors":
        n = _mean_drafts(case)
        rows = case["seqs"] * (n + 1 + (n if case["draft_rows"] else 0))
        outs = case["seqs"] * (case["drafts"] + 3) * 4
        return {"bytes": rows * (case["top_k"] * 8 + 4) + outs, "flops": 2 * rows * case["top_k"]}
    size = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
    cells = case["rows"] * case["vocab"]
    reads = cells * size + case["rows"] * (case["top"] * 8 + 8)
    if case["call"] == "forward":
        return {"bytes": reads, "flops": 3 * cells}
    return {"bytes": reads + cells * size, "flops": 6 * cells}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _gumbel(shape, g):
    u = torch.rand(shape, generator=g, device=DEVICE).clamp_(1e-7, 1 - 1e-7)
    return u.log_().neg_().log_().neg_()


def _ascending_ids(rows, k, vocab, g):
    """[rows, k] distinct token ids in ascending order, spread over the vocabulary."""
    step = vocab // k
    first = torch.arange(k, device=DEVICE, dtype=torch.int64) * step
    return first + torch.randint(0, step, (rows, k), generator=g, device=DEVICE)


def _ragged_drafts(case, g):
    """Drafted tokens of each sequence, or None where all drafted the same number."""
    if not case["ragged"]:
        return None
    return torch.randint(0, case["drafts"] + 1, (case["seqs"],), generator=g, device=DEVICE,
                         dtype=torch.int32)


def _prepare_verify(case, g):
    b, d, v, t = case["seqs"], case["drafts"], case["vocab"], case["temperature"]
    # A language model's rows: a bulk of width 2 and 20 likely tokens well above it.
    target = torch.randn((b, d + 1, v), generator=g, device=DEVICE).mul_(2.0)
    spikes = torch.randint(0, v, (b, d + 1, 20), generator=g, device=DEVICE)
    boost = torch.rand((b, d + 1, 20), generator=g, device=DEVICE).mul_(7.0).add_(5.0)
    target.scatter_add_(2, spikes, boost)
    draft = None
    if case["draft_rows"]:
        # The draft model sees nearly the same logits; its tokens are drawn from its own rows.
        draft = target[:, :d] + 0.5 * torch.randn((b, d, v), generator=g, device=DEVICE)
        tokens = (draft / t + _gumbel((b, d, v), g)).argmax(2)
    else:
        tokens = (target[:, :d] + 0.5 * _gumbel((b, d, v), g)).argmax(2)
    return {"case": case, "target": target, "draft": draft, "tokens": tokens.to(torch.int32),
            "n_draft": _ragged_drafts(case, g),
            "uniforms": torch.rand((b, d + 1), generator=g, device=DEVICE) if t > 0 else None}


def _record(logits, ids, top_k, cap, n):
    """A survivor record: the `n` largest of each row's candidates (n a row, at most top_k), ids
    ascending, softmax over them; `cap` slots a row, the unused ones id -1 and probability 0."""
    rows, m = logits.shape
    order = logits.argsort(dim=1, descending=True)
    rank = torch.empty_like(order).scatter_(1, order, torch.arange(m, device=DEVICE)
                                            .expand(rows, m).contiguous())
    keep = rank < n[:, None]
    e = torch.where(keep, (logits - logits.amax(1, keepdim=True)).exp(), 0.0)
    p = e / e.sum(1, keepdim=True)
    slot = (keep.cumsum(1) - 1).masked_fill(~keep, cap)
    out_ids = torch.full((rows, cap + 1), -1, dtype=torch.int32, device=DEVICE)
    out_p = torch.zeros((rows, cap + 1), device=DEVICE)
    out_ids.scatter_(1, slot, torch.where(keep, ids, -1).to(torch.int32))
    out_p.scatter_(1, slot, torch.where(keep, p, 0.0))
    return n.to(torch.int32), out_ids[:, :cap].contiguous(), out_p[:, :cap].contiguous()


def _prepare_survivors(case, g):
    b, d, k, cap = case["seqs"], case["drafts"], case["top_k"], case["cap"]
    # The candidates of a position: half as many again as survive, so that the two models keep
    # overlapping but not equal sets; top-p then cuts each row to its own length.
    m = k + max(1, k // 2)
    ids = _ascending_ids(b * (d + 1), m, case["vocab"], g)
    logits = 3.0 * torch.randn((b * (d + 1), m), generator=g, device=DEVICE)
    n = torch.randint((k + 1) // 2, k + 1, (b * (d + 1),), generator=g, device=DEVICE)
    target = _record(logits, ids, k, cap, n)
    first = torch.arange(b * (d + 1), device=DEVICE).reshape(b, d + 1)[:, :d].reshape(-1)
    theirs = logits[first] + 0.5 * torch.randn((b * d, m), generator=g, device=DEVICE)
    n_d = torch.randint((k + 1) // 2, k + 1, (b * d,), generator=g, device=DEVICE)
    draft = _record(theirs, ids[first], k, cap, n_d)
    at = (draft[2].log() + _gumbel((b * d, cap), g)).argmax(1)
    tokens = draft[1].gather(1, at[:, None]).reshape(b, d)
    return {"case": case, "target": target, "draft": draft if case["draft_rows"] else None,
            "tokens": tokens, "n_draft": _ragged_drafts(case, g),
            "uniforms": torch.rand((b, d + 1), generator=g, device=DEVICE)}


def _prepare_distill(case, g):
    n, v, k = case["rows"], case["vocab"], case["top"]
    z = torch.randn((n, v), generator=g, device=DEVICE, dtype=TYPES[case["dtype"]]).mul_(2.0)
    ids = _ascending_ids(n, k, v, g)
    # The student half knows the teacher's tokens; the teacher's logits differ by a unit normal.
    boost = 3.0 + 7.0 * torch.rand((n, k), generator=g, device=DEVICE)
    z.scatter_add_(1, ids, boost.to(z.dtype))
    teacher = (boost + torch.randn((n, k), generator=g, device=DEVICE)) / case["temperature"]
    # Log-probabilities over the whole vocabulary: the listed tokens hold 70 to 99.9 % of it.
    held = 1.0 - 10.0 ** -(0.5 + 2.5 * torch.rand((n, 1), generator=g, device=DEVICE))
    logprobs = teacher.log_softmax(1) + held.log()
    count = None
    if case["ragged"]:
        # Lists cut by top-p, and one position in sixteen without a list (padding, prompt).
        count = torch.randint(1, k + 1, (n,), generator=g, device=DEVICE, dtype=torch.int32)
        count[torch.rand(n, generator=g, device=DEVICE) < 1 / 16] = 0
    # The upstream gradient of each row: the mean over the batch, with the loss scaling that half
    # precision needs.
    scale = 4096.0 if case["dtype"] == "f16" else 1.0
    upstream = torch.full((n,), scale / n, device=DEVICE)
    return {"case": case, "z": z.requires_grad_(case["call"] == "autograd"),
            "ids": ids.to(torch.int32), "logprobs": logprobs, "count": count,
            "upstream": upstream}


def prepare(case, seed):
    g = _generator(seed)
    return {"verify": _prepare_verify, "survivors": _prepare_survivors,
            "distill": _prepare_distill}[case["kind"]](case, g)


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _inverse(temperature):
    """1/T as the sampler has it: one binary32 division."""
    return float(np.float32(1.0) / np.float32(temperature))


def _scaled(x, temperature):
    """The sampler's scaled logits: one binary32 product with 1/T."""
    return x.float() * _inverse(temperature)


def _emit(tokens, accepted, final):
    """[b, d + 1] tokens: the accepted drafts, the final token, then -1."""
    b, d = tokens.shape
    place = torch.arange(d + 1, device=tokens.device)
    drafts = torch.cat([tokens, tokens.new_zeros((b, 1))], 1).long()
    out = torch.where(place < accepted[:, None], drafts, -1)
    out = torch.where(place == accepted[:, None], final[:, None], out)
    return out.to(torch.int32)


def _first_refused(ok, n):
    """The number of leading accepted tests of each row of `ok`, at most n."""
    b, d = ok.shape
    ok = ok & (torch.arange(d, device=ok.device) < n[:, None])
    return ok.to(torch.int64).cumprod(1).sum(1)


def _pick(w, u):
    """The first index whose running sum exceeds u times the whole, else the last of weight."""
    c = w.cumsum(1)
    at = (c <= u[:, None] * c[:, -1:]).sum(1)
    place = torch.arange(w.shape[1], device=w.device)
    last = torch.where(w > 0, place, 0).amax(1)
    return torch.minimum(at, last)


def _plain_verify(s):
    case, target, tokens = s["case"], s["target"], s["tokens"].long()
    b, d = tokens.shape
    n = s["n_draft"].long() if s["n_draft"] is not None else tokens.new_full((b,), d)
    rows = torch.arange(b, device=target.device)
    status = torch.zeros(b, dtype=torch.int32, device=target.device)
    if case["temperature"] == 0:
        # The last of equal maxima.
        best = target.shape[2] - 1 - target.flip(2).argmax(2)
        accepted = _first_refused(best[:, :d] == tokens, n)
        return {"tokens": _emit(tokens, accepted, best[rows, accepted]),
                "accepted": accepted.to(torch.int32), "status": status}
    v = _scaled(target, case["temperature"])
    v = v - v.amax(2, keepdim=True).double()
    lse = v.exp().sum(2).log()
    lp = v[:, :d].gather(2, tokens[:, :, None])[:, :, 0] - lse[:, :d]
    if s["draft"] is not None:
        q = _scaled(s["draft"], case["temperature"])
        q = q - q.amax(2, keepdim=True).double()
        lse_q = q.exp().sum(2).log()
        lq = q.gather(2, tokens[:, :, None])[:, :, 0] - lse_q
    else:
        lq = torch.zeros_like(lp)
    u = s["uniforms"].double()
    accepted = _first_refused(u[:, :d] * lq.exp() < lp.exp(), n)
    refused = accepted < n
    # The row that the last token comes from, minus what its draft already had.
    w = (v[rows, accepted] - lse[rows, accepted][:, None]).exp()
    at = accepted.clamp(max=d - 1)
    if s["draft"] is not None:
        had = (q[rows, at] - lse_q[rows, at][:, None]).exp()
        w = torch.where(refused[:, None], (w - had).clamp(min=0), w)
    else:
        t = tokens.gather(1, at[:, None])
        w = w.scatter(1, t, torch.where(refused[:, None], 0.0, w.gather(1, t)))
    return {"tokens": _emit(tokens, accepted, _pick(w, u[:, d])),
            "accepted": accepted.to(torch.int32), "status": status}


def _plain_survivors(s):
    tokens = s["tokens"].long()
    b, d = tokens.shape
    n = s["n_draft"].long() if s["n_draft"] is not None else tokens.new_full((b,), d)
    rows = torch.arange(b, device=tokens.device)
    count, ids, p = s["target"]
    cap = ids.shape[1]
    place = torch.arange(cap, device=ids.device)
    p = torch.where(place < count[:, None], p, 0.0).double().reshape(b, d + 1, cap)
    ids = torch.where(place < count[:, None], ids, -1).reshape(b, d + 1, cap)
    pt = torch.where(ids[:, :d] == tokens[:, :, None], p[:, :d], 0.0).sum(2)
    qt = torch.ones_like(pt)
    if s["draft"] is not None:
        count_q, ids_q, q = s["draft"]
        q = torch.where(place < count_q[:, None], q, 0.0).double().reshape(b, d, cap)
        ids_q = torch.where(place < count_q[:, None], ids_q, -2).reshape(b, d, cap)
        qt = torch.where(ids_q == tokens[:, :, None], q, 0.0).sum(2)
    u = s["uniforms"].double()
    accepted = _first_refused(u[:, :d] * qt < pt, n)
    refused = accepted < n
    at = accepted.clamp(max=d - 1)
    w, w_ids = p[rows, accepted], ids[rows, accepted]
    if s["draft"] is not None:
        same = w_ids[:, :, None] == ids_q[rows, at][:, None, :]
        had = torch.where(same, q[rows, at][:, None, :], 0.0).sum(2)
    else:
        had = torch.where(w_ids == tokens[rows, at][:, None], math.inf, 0.0)
    w = torch.where(refused[:, None], (w - had).clamp(min=0), w)
    final = w_ids.gather(1, _pick(w, u[:, d])[:, None])[:, 0].long()
    return {"tokens": _emit(tokens, accepted, final), "accepted": accepted.to(torch.int32),
            "status": torch.zeros(b, dtype=torch.int32, device=ids.device)}


def _plain_distill(s):
    case, z = s["case"], s["z"].detach()
    n, v = z.shape
    k = case["top"]
    scale = _inverse(case["temperature"])
    x = _scaled(z, case["temperature"])
    m = x.amax(1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(1, keepdim=True)
    ids = s["ids"].long()
    there = torch.ones_like(ids, dtype=torch.bool)
    if s["count"] is not None:
        there = torch.arange(k, device=z.device) < s["count"][:, None]
    y = torch.where(there, s["logprobs"], -math.inf)
    some = there.any(1, keepdim=True)
    logq = x.gather(1, ids) - m - total.log()
    if case["tail"]:
        t, logt = y.exp(), y
        rest = e.scatter(1, ids, torch.where(there, 0.0, e.gather(1, ids)))
        share = rest.sum(1, keepdim=True) / total
        # 1 minus a sum of up to 128 probabilities near 1: in 64 bits.
        held = t.double().sum(1, keepdim=True)
        r, mass = (1 - held).clamp(min=0).float(), held.clamp(min=1).float()
        tail = torch.where(r > 0, r * (r / share).log(), 0.0)
        coeff = mass - torch.where(r > 0, r / share, 0.0)
    else:
        top = torch.where(some, y.amax(1, keepdim=True), 0.0)
        z_t = (y - top).exp().sum(1, keepdim=True)
        logt = y - top - z_t.log()
        t = torch.where(there, logt.exp(), 0.0)
        tail, mass, coeff = 0.0, 1.0, torch.ones_like(total)
    terms = torch.where(t > 0, t * (logt - logq), 0.0)
    loss = torch.where(some, terms.sum(1, keepdim=True) + tail, 0.0)[:, 0]
    if case["call"] == "forward":
        return {"loss": loss}
    e /= total
    at = e.gather(1, ids)
    grad = e.mul_(coeff)
    grad.scatter_(1, ids, torch.where(there, at * mass - t, at * coeff))
    grad.mul_(torch.where(some, scale * s["upstream"][:, None], 0.0))
    return {"loss": loss, "grad": grad.to(z.dtype)}


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _own_verify(s):
    from rusticide_b200 import SamplingParams, engine
    tokens, accepted, status = engine(0).verify(
        s["target"], s["tokens"], SamplingParams(s["case"]["temperature"], 0, 1.0),
        uniforms=s["uniforms"], draft_logits=s["draft"], n_draft=s["n_draft"])
    return {"tokens": tokens, "accepted": accepted, "status": status}


def _own_survivors(s):
    from rusticide_b200 import engine
    tokens, accepted, status = engine(0).verify_survivors(
        s["target"], s["tokens"], uniforms=s["uniforms"], draft=s["draft"], n_draft=s["n_draft"])
    return {"tokens": tokens, "accepted": accepted, "status": status}


def _own_distill(s):
    from rusticide_b200 import distill_loss, engine
    case = s["case"]
    kw = {"n": s["count"], "temperature": case["temperature"], "tail": case["tail"]}
    if case["call"] == "autograd":
        loss = distill_loss(s["z"], s["ids"], s["logprobs"], **kw)
        grad, = torch.autograd.grad(loss, s["z"], s["upstream"])
        return {"loss": loss.detach(), "grad": grad}
    if case["call"] == "step":
        loss, grad = engine(0).distill_step(s["z"], s["ids"], s["logprobs"], s["upstream"], **kw)
        return {"loss": loss, "grad": grad}
    return {"loss": distill_loss(s["z"], s["ids"], s["logprobs"], **kw)}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"verify": _own_verify, "survivors": _own_survivors,
                "distill": _own_distill}[kind](state)
    return {"verify": _plain_verify, "survivors": _plain_survivors,
            "distill": _plain_distill}[kind](state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one row at a time
# ---------------------------------------------------------------------------
def _exact_draw(w, u):
    c = torch.cumsum(w, 0)
    if float(c[-1]) == 0.0:
        return None
    at = int(torch.searchsorted(c, u * c[-1], right=True))
    return min(at, int(w.nonzero()[-1]))


def _exact_verify(case, s):
    t = case["temperature"]
    b, d = s["tokens"].shape
    out = torch.full((b, d + 1), -1, dtype=torch.int32)
    accepted = torch.zeros(b, dtype=torch.int32)
    tokens = s["tokens"].tolist()
    counts = s["n_draft"].tolist() if s["n_draft"] is not None else [d] * b
    u = s["uniforms"].double().tolist() if s["uniforms"] is not None else None
    inverse = float(np.float32(1.0) / np.float32(t)) if t > 0 else None

    def probs(row):
        return torch.softmax((row * inverse).double(), 0)

    for i in range(b):
        final, a = None, 0
        while final is None:
            row = s["target"][i, a]
            if t == 0:
                best = int((row == row.max()).nonzero()[-1])
                if a < counts[i] and best == tokens[i][a]:
                    a += 1
                else:
                    final = best
                continue
            p = probs(row)
            if a == counts[i]:
                final = _exact_draw(p, u[i][d])
                continue
            tok = tokens[i][a]
            q = probs(s["draft"][i, a]) if s["draft"] is not None else None
            if u[i][a] * (float(q[tok]) if q is not None else 1.0) < float(p[tok]):
                a += 1
                continue
            if q is None:
                w = p.clone()
                w[tok] = 0.0
            else:
                w = torch.clamp(p - q, min=0.0)
            final = _exact_draw(w, u[i][d])
            final = _exact_draw(p, u[i][d]) if final is None else final
        out[i, :a] = torch.tensor(tokens[i][:a], dtype=torch.int32)
        out[i, a] = final
        accepted[i] = a
    return {"tokens": out, "accepted": accepted, "status": torch.zeros(b, dtype=torch.int32)}


def _exact_survivors(case, s):
    b, d = s["tokens"].shape
    tokens = s["tokens"].tolist()
    counts = s["n_draft"].tolist() if s["n_draft"] is not None else [d] * b
    u = s["uniforms"].double().tolist()

    def lists(record):
        n, ids, p = (x.cpu() for x in record)
        return [dict(zip(i[:m].tolist(), q[:m].double().tolist()))
                for m, i, q in zip(n.tolist(), ids, p)]

    target = lists(s["target"])
    draft = lists(s["draft"]) if s["draft"] is not None else None
    out = torch.full((b, d + 1), -1, dtype=torch.int32)
    accepted = torch.zeros(b, dtype=torch.int32)
    for i in range(b):
        a, had = 0, {}
        while a < counts[i]:
            tok = tokens[i][a]
            had = draft[i * d + a] if draft is not None else {tok: 1.0}
            if not u[i][a] * had.get(tok, 0.0) < target[i * (d + 1) + a].get(tok, 0.0):
                break
            a, had = a + 1, {}
        p = target[i * (d + 1) + a]
        keep = [(j, max(x - had.get(j, 0.0), 0.0)) for j, x in p.items()]
        if not sum(x for _, x in keep) > 0:
            keep = list(p.items())
        at = _exact_draw(torch.tensor([x for _, x in keep], dtype=torch.float64), u[i][d])
        out[i, :a] = torch.tensor(tokens[i][:a], dtype=torch.int32)
        out[i, a] = keep[at][0]
        accepted[i] = a
    return {"tokens": out, "accepted": accepted, "status": torch.zeros(b, dtype=torch.int32)}


def _exact_distill(case, s):
    z = s["z"].detach()
    rows = z.shape[0]
    scale = float(np.float32(1.0) / np.float32(case["temperature"]))
    counts = s["count"].tolist() if s["count"] is not None else [case["top"]] * rows
    loss = torch.zeros(rows, dtype=torch.float64, device=z.device)
    grad = None if case["call"] == "forward" else torch.zeros(z.shape, dtype=torch.float64,
                                                              device=z.device)
    for i in range(rows):
        c = counts[i]
        if c == 0:
            continue
        ids, y = s["ids"][i, :c].long(), s["logprobs"][i, :c].double()
        logs = torch.log_softmax(z[i].double() * scale, 0)
        share = logs.exp()
        t = y.exp() if case["tail"] else torch.softmax(y, 0)
        row = (t * (t.log() - logs[ids])).sum()
        d = share.clone()
        if case["tail"]:
            r, mass = (1 - t.sum()).clamp(min=0), t.sum().clamp(min=1)
            rest = share.clone()
            rest[ids] = 0.0
            left = rest.sum()
            row = row + torch.special.xlogy(r, r / left)
            d = share * mass - rest * (r / left)
        d[ids] -= t
        loss[i] = row
        if grad is not None:
            grad[i] = d * (scale * s["upstream"][i].double())
    return {"loss": loss} if grad is None else {"loss": loss, "grad": grad}


def exact(case, seed):
    s = prepare(case, seed)
    return {"verify": _exact_verify, "survivors": _exact_survivors,
            "distill": _exact_distill}[case["kind"]](case, s)
