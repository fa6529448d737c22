"""Operators over rows of scores: log probabilities of given tokens, distillation from a teacher's top logits, routing to experts.

`listed()` names the calls by which they are judged, `draw()` gives further ones from the same ranges.  `run()` makes a call: through
the public entry points of `cutile_b200` where `own` is true, else in plain torch operations in f32 (f64 where the order of two
values or a difference from one decides).  `exact()` gives the same outputs in f64 from the definitions, gradients by automatic
differentiation.  Index arrays are 1-based and 0 stands for "none", as everywhere in the package.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # One decoding step of a few sequences: the sampled tokens' log probabilities and five alternatives. Latency counts.
        dict(name="logprobs_step", kind="logprobs", dtype="f32", rows=4, vocab=32000, top=5, temperature=0.8, padding=0.0,
             train=False),
        # A decoding step of a full batch with the longest list of alternatives that serving programs usually offer.
        dict(name="logprobs_batch", kind="logprobs", dtype="bf16", rows=64, vocab=128000, top=20, temperature=1.0, padding=0.0,
             train=False),
        # Scoring of a prompt, no alternatives; a vocabulary of odd size, so that rows start anywhere.
        dict(name="logprobs_prompt", kind="logprobs", dtype="f16", rows=2048, vocab=50001, top=0, temperature=1.0, padding=0.0,
             train=False),
        # A step of policy training: log probabilities and entropies of a padded batch, and the gradient of both.
        dict(name="logprobs_policy", kind="logprobs", dtype="bf16", rows=2048, vocab=100003, top=0, temperature=0.7, padding=0.1,
             train=True),
        # f32 logits with the longest list of alternatives, and gradients through the list.
        dict(name="logprobs_alternatives", kind="logprobs", dtype="f32", rows=512, vocab=50001, top=32, temperature=1.0,
             padding=0.0, train=True),
        # Evaluation of a student on a few positions.
        dict(name="distill_probe", kind="distill", dtype="f32", teacher="f32", rows=32, vocab=32000, entries=16, tail=False,
             temperature=1.0, padding=0.0, mode="loss"),
        # A training step that knows the rows' weights beforehand: loss and gradient in one call.
        dict(name="distill_train", kind="distill", dtype="bf16", teacher="bf16", rows=4096, vocab=65536, entries=64, tail=False,
             temperature=2.0, padding=0.1, mode="train"),
        # The same with all that the teacher did not list as one more class; loss first, gradient later.
        dict(name="distill_tail", kind="distill", dtype="f32", teacher="f32", rows=1500, vocab=50001, entries=50, tail=True,
             temperature=1.0, padding=0.0, mode="split"),
        # Router of a decoding step. Latency counts.
        dict(name="route_step", kind="route", dtype="f16", tokens=8, experts=64, topk=8, score="softmax", bias=False, groups=1,
             topk_groups=1, group_top=1, renormalize=True, scale=1.0, train=False),
        # Router of a prompt: sigmoid scores, a bias that balances the experts, the better half of eight groups.
        dict(name="route_groups", kind="route", dtype="f32", tokens=4096, experts=256, topk=8, score="sigmoid", bias=True, groups=8,
             topk_groups=4, group_top=2, renormalize=True, scale=2.5, train=False),
        # Router of a training step, forward and backward.
        dict(name="route_train", kind="route", dtype="bf16", tokens=16384, experts=128, topk=4, score="softmax", bias=False,
             groups=1, topk_groups=1, group_top=1, renormalize=False, scale=1.0, train=True),
    ]


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_BYTES = 4096 * 65536 * 2  # of logits


def _draw_rows(rng, dtype):
    vocab = _log(rng, 1000, 262144)
    vocab = vocab if rng.random() < 0.5 else vocab // 64 * 64
    return vocab, max(1, min(_log(rng, 1, 8192), _MOST_BYTES // (vocab * BYTES[dtype])))


def _draw_logprobs(rng):
    dtype = rng.choice(("f32", "f16", "bf16"))
    vocab, rows = _draw_rows(rng, dtype)
    train = rng.random() < 0.5
    return dict(kind="logprobs", dtype=dtype, rows=rows, vocab=vocab, top=rng.choice((0, 1, 5, 20, rng.randint(1, 32))),
                temperature=rng.choice((1.0, 0.7, 1.3)), padding=0.2 if train and rng.random() < 0.5 else 0.0, train=train)


def _draw_distill(rng):
    dtype = rng.choice(("f32", "f16", "bf16"))
    vocab, rows = _draw_rows(rng, dtype)
    return dict(kind="distill", dtype=dtype, teacher=rng.choice(("f32", dtype)), rows=rows, vocab=vocab, entries=_log(rng, 1, 256),
                tail=rng.random() < 0.5, temperature=rng.choice((1.0, 2.0, 0.9)), padding=rng.choice((0.0, 0.2)),
                mode=rng.choice(("loss", "train", "train", "split")))


def _draw_route(rng):
    experts = rng.choice((8, 16, 32, 60, 64, 128, 160, 256, 384, 512))
    groups = rng.choice([1, 1] + [g for g in (2, 4, 5, 8, 16) if experts % g == 0 and experts // g >= 2])
    kept = rng.randint(1, groups)
    topk = rng.randint(1, min(16, kept * (experts // groups)))
    return dict(kind="route", dtype=rng.choice(("f32", "f16", "bf16")), tokens=min(_log(rng, 1, 32768), 2 ** 23 // experts),
                experts=experts, topk=topk, score=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.5, groups=groups,
                topk_groups=kept, group_top=rng.choice((1, 2)), renormalize=rng.random() < 0.7, scale=rng.choice((1.0, 2.5)),
                train=rng.random() < 0.5)


def draw(rng):
    return rng.choice((_draw_logprobs, _draw_distill, _draw_route))(rng)


# ------------------------------------------------------------------ shared
def _package():
    path = os.path.abspath("cutile.jl_b200")  # the package of the tree that is the working folder
    if path not in sys.path:
        sys.path.insert(0, path)
    import cutile_b200
    return cutile_b200


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _scores(g, rows, vocab):
    """Scores as a language model gives them: frequent tokens, with low ids, are likelier; values of every row differ by chance."""
    x = torch.randn(rows, vocab, device="cuda", generator=g).mul_(2.0)
    return x.sub_(torch.log(torch.arange(1, vocab + 1, device="cuda", dtype=torch.float32)).mul_(0.5))


def _chance(g, n):
    return torch.rand(n, device="cuda", generator=g)


# ------------------------------------------------------------------ log probabilities of given tokens
def _prepare_logprobs(c, g):
    rows, vocab = c["rows"], c["vocab"]
    x = _scores(g, rows, vocab).to(DTYPES[c["dtype"]])
    tokens = torch.exp(_chance(g, rows) * math.log(vocab)).long().clamp_(1, vocab)
    tokens[_chance(g, rows) < c["padding"]] = 0
    return dict(x=x, tokens=tokens, top=c["top"], temperature=c["temperature"], train=c["train"],
                d_logprobs=torch.randn(rows, device="cuda", generator=g) if c["train"] else None,
                d_entropy=torch.randn(rows, device="cuda", generator=g) * 0.1 if c["train"] else None,
                d_top=torch.randn(rows, c["top"], device="cuda", generator=g) if c["train"] and c["top"] else None)


def _own_logprobs(s):
    ops = _package().logprobs
    r = ops.token_logprobs(s["x"], s["tokens"], top=s["top"], temperature=s["temperature"])
    out = [r.logprobs, r.entropy, r.lse]
    if s["top"]:
        out += [r.top_logprobs, r.top_ids]
    if s["train"]:
        out.append(ops.token_logprobs_bwd(s["x"], s["tokens"], r.lse, r.entropy, s["d_logprobs"], s["d_entropy"], top_ids=r.top_ids,
                                          d_top_logprobs=s["d_top"], temperature=s["temperature"]))
    return out


def _plain_logprobs(s):
    x = s["x"].float()
    z = x / s["temperature"]
    row = s["tokens"] > 0  # rows without a token are padding
    at = (s["tokens"] - 1).clamp(min=0)[:, None]
    peak = z.amax(1, keepdim=True)
    e = torch.exp(z - peak)
    total = e.sum(1, keepdim=True)
    lse = peak + torch.log(total)
    p = e / total
    logp = (z - peak) - torch.log(total)
    entropy = -(p * logp).sum(1)
    out = [torch.where(row, v, 0.0) for v in (logp.gather(1, at)[:, 0], entropy, lse[:, 0])]
    if s["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
        out += [torch.where(row[:, None], logp.gather(1, ids), 0.0), torch.where(row[:, None], ids + 1, 0).int()]
    if s["train"]:
        weight = s["d_logprobs"] if not s["top"] else s["d_logprobs"] + s["d_top"].sum(1)
        d = -p * (weight[:, None] + s["d_entropy"][:, None] * (logp + entropy[:, None]))
        d.scatter_add_(1, at, s["d_logprobs"][:, None])
        if s["top"]:
            d.scatter_add_(1, ids, s["d_top"])
        out.append(torch.where(row[:, None], d / s["temperature"], 0.0).to(s["x"].dtype))
    return out


def _exact_logprobs(s):
    x = s["x"].double().requires_grad_(s["train"])
    row = s["tokens"] > 0
    at = (s["tokens"] - 1).clamp(min=0)[:, None]
    z = x / s["temperature"]
    logp = torch.log_softmax(z, 1)
    values = [logp.gather(1, at)[:, 0], -(logp.exp() * logp).sum(1)]
    terms = [values[0] * s["d_logprobs"], values[1] * s["d_entropy"]] if s["train"] else []
    values.append(torch.logsumexp(z.detach(), 1))
    out = [torch.where(row, v.detach(), 0.0) for v in values]
    if s["top"]:
        ids = torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :s["top"]]
        top = logp.gather(1, ids)
        out += [torch.where(row[:, None], top.detach(), 0.0), torch.where(row[:, None], ids + 1, 0).int()]
        if s["train"]:
            terms.append((top * s["d_top"]).sum(1))
    if s["train"]:
        torch.where(row, sum(terms), 0.0).sum().backward()
        out.append(x.grad)
    return out


def _work_logprobs(c):
    live = c["rows"] * (1 - c["padding"])
    elements, b = c["rows"] * c["vocab"], BYTES[c["dtype"]]
    reads = live * c["vocab"] * b
    small = c["rows"] * (8 + 12 + 8 * c["top"])
    if not c["train"]:
        return {"bytes": int(reads + small), "flops": int(6 * live * c["vocab"])}
    return {"bytes": int(2 * reads + elements * b + small + c["rows"] * (16 + 4 * c["top"])), "flops": int(12 * live * c["vocab"])}


# ------------------------------------------------------------------ distillation from a teacher's top logits
def _prepare_distill(c, g):
    rows, vocab, k, tau = c["rows"], c["vocab"], c["entries"], c["temperature"]
    taught = _scores(g, rows, vocab)
    x = (taught + torch.randn(rows, vocab, device="cuda", generator=g)).to(DTYPES[c["dtype"]])  # a student that has come near
    value, index = torch.topk(taught, k, dim=1)
    ids = (index + 1).int()
    used = torch.where(_chance(g, rows) < 0.2, (_chance(g, rows) * k).long() + 1, k)  # some lists are shorter
    used[_chance(g, rows) < c["padding"]] = 0
    ids[torch.arange(k, device="cuda")[None, :] >= used[:, None]] = 0
    return dict(x=x, ids=ids, values=value.to(DTYPES[c["teacher"]]), lse=torch.logsumexp(taught / tau, 1) if c["tail"] else None,
                d_loss=_chance(g, rows) / rows, temperature=tau, mode=c["mode"])


def _own_distill(s):
    ops = _package().distill
    if s["mode"] == "train":
        return list(ops.distill_fwd_bwd(s["x"], s["ids"], s["values"], s["d_loss"], teacher_lse=s["lse"], temperature=s["temperature"]))
    loss, saved = ops.distill_fwd(s["x"], s["ids"], s["values"], teacher_lse=s["lse"], temperature=s["temperature"])
    if s["mode"] == "loss":
        return [loss]
    return [loss, ops.distill_bwd(s["x"], s["ids"], s["values"], saved, s["d_loss"], temperature=s["temperature"])]


def _plain_distill(s):
    z = s["x"].float() / s["temperature"]
    used = s["ids"] > 0
    row = used.any(1)
    at = (s["ids"].long() - 1).clamp(min=0)
    # the teacher's side in f64: what its list leaves over is a difference from one
    u = torch.where(used, s["values"].double() / s["temperature"], -math.inf)
    norm = s["lse"].double()[:, None] if s["lse"] is not None else torch.log(torch.exp(u).sum(1, keepdim=True))
    logq = u - norm
    q = torch.where(row[:, None], torch.exp(logq), 0.0)
    self_part = torch.where(q > 0, q * logq, 0.0).sum(1)
    peak = z.amax(1, keepdim=True)
    e = torch.exp(z - peak)
    total = e.sum(1, keepdim=True)
    logp = (z - peak) - torch.log(total)
    loss = self_part - torch.where(q > 0, q * logp.gather(1, at), 0.0).sum(1)
    all_of_q = q.sum(1)
    if s["lse"] is not None:
        listed_ = torch.zeros_like(z).scatter_add_(1, at, used.float()) > 0
        rest = torch.where(listed_, 0.0, e).sum(1)
        left = (1 - all_of_q).clamp(min=0)
        all_of_q = all_of_q + left
        log_rest = torch.log(rest) - torch.log(total[:, 0])
        loss = loss + torch.where(left > 0, left * (torch.log(left) - log_rest), 0.0)
    loss = torch.where(row, loss, 0.0).float()
    if s["mode"] == "loss":
        return [loss]
    p = e / total
    if s["lse"] is not None:
        outside = (all_of_q - left * (total[:, 0] / rest)).float()
        d = torch.where(listed_, all_of_q.float()[:, None], outside[:, None]) * p
    else:
        d = p
    d = d.scatter_add(1, at, -q.float())
    d = torch.where(row[:, None], d * (s["d_loss"] / s["temperature"])[:, None], 0.0)
    return [loss, d.to(s["x"].dtype)]


def _exact_distill(s):
    train = s["mode"] != "loss"
    x = s["x"].double().requires_grad_(train)
    used = s["ids"] > 0
    row = used.any(1)
    at = (s["ids"].long() - 1).clamp(min=0)
    u = (s["values"].double() / s["temperature"]).masked_fill(~used, -1e6)  # e^-1e6 = 0
    logq = u - s["lse"].double()[:, None] if s["lse"] is not None else torch.log_softmax(u, 1)
    q = logq.exp() * used
    logp = torch.log_softmax(x / s["temperature"], 1)
    loss = (torch.xlogy(q, q) - q * logp.gather(1, at)).sum(1)
    if s["lse"] is not None:
        listed_ = torch.zeros_like(x, dtype=torch.bool)
        which = torch.arange(len(at), device=at.device)[:, None].expand_as(at)
        listed_[which[used], at[used]] = True
        left = (1 - q.sum(1)).clamp(min=0)
        loss = loss + torch.xlogy(left, left) - left * torch.logsumexp(logp.masked_fill(listed_, -math.inf), 1)
    loss = torch.where(row, loss, 0.0)
    if not train:
        return [loss]
    (loss * s["d_loss"]).sum().backward()
    return [loss.detach(), x.grad]


def _work_distill(c):
    live = c["rows"] * (1 - c["padding"])
    b, tb = BYTES[c["dtype"]], BYTES[c["teacher"]]
    reads, writes = live * c["vocab"] * b, c["rows"] * c["vocab"] * b
    small = c["rows"] * (c["entries"] * (4 + tb) + (4 if c["tail"] else 0) + 4)
    if c["mode"] == "loss":
        return {"bytes": int(reads + small), "flops": int(4 * live * c["vocab"])}
    passes = 1 if c["mode"] == "train" else 2  # the gradient of a later call has to read the logits again
    return {"bytes": int(passes * (reads + small) + writes + 4 * c["rows"]), "flops": int(8 * live * c["vocab"])}


# ------------------------------------------------------------------ routing to experts
_OPTIONS = ("score", "groups", "topk_groups", "group_top", "renormalize", "scale")


def _prepare_route(c, g):
    tokens, experts = c["tokens"], c["experts"]
    x = (torch.randn(tokens, experts, device="cuda", generator=g) * 1.5).to(DTYPES[c["dtype"]])
    return dict(x=x, topk=c["topk"], bias=torch.randn(experts, device="cuda", generator=g) * 0.05 if c["bias"] else None,
                options={k: c[k] for k in _OPTIONS}, train=c["train"],
                d_weights=torch.randn(c["topk"], tokens, device="cuda", generator=g) if c["train"] else None)


def _own_route(s):
    ops, o = _package().moe, s["options"]
    weights, ids = ops.moe_route(s["x"], s["topk"], bias=s["bias"], **o)
    if not s["train"]:
        return [weights, ids]
    return [weights, ids, ops.moe_route_bwd(s["x"], ids, s["d_weights"], score=o["score"], renormalize=o["renormalize"],
                                            scale=o["scale"])]


def _chosen(value, topk, groups, topk_groups, group_top):
    """Ids [tokens, topk], best first, ties to the lowest: the experts of the best groups, by f64 values."""
    tokens, experts = value.shape
    if topk_groups < groups:
        best = torch.sort(value.view(tokens, groups, -1), dim=2, descending=True).values[:, :, :group_top].sum(2)
        keep = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :topk_groups]
        allowed = torch.zeros(tokens, groups, dtype=torch.bool, device=value.device).scatter_(1, keep, True)
        value = torch.where(allowed.repeat_interleave(experts // groups, 1), value, -math.inf)
    return torch.sort(value, dim=1, descending=True, stable=True).indices[:, :topk]


def _plain_route(s):
    o, x = s["options"], s["x"].double()  # f64: which of two experts is better must not hang on a rounding
    if o["score"] == "softmax":
        e = torch.exp(x - x.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    ids = _chosen(score if s["bias"] is None else score + s["bias"].double(), s["topk"], o["groups"], o["topk_groups"], o["group_top"])
    mine = score.gather(1, ids)
    total = mine.sum(1, keepdim=True).clamp(min=1e-20) if o["renormalize"] else torch.ones_like(mine[:, :1])
    weights = o["scale"] * mine / total
    out = [weights.t().contiguous().half(), (ids + 1).int().t().contiguous()]
    if s["train"]:
        up = s["d_weights"].double().t() * o["scale"] / total
        if o["renormalize"]:
            up = up - (up * mine).sum(1, keepdim=True) / total
        d = torch.zeros_like(score).scatter_(1, ids, up)
        if o["score"] == "softmax":
            d = score * (d - (up * mine).sum(1, keepdim=True))
        else:
            d = d * score * (1 - score)
        out.append(d.to(s["x"].dtype))
    return out


def _exact_route(s):
    o = s["options"]
    x = s["x"].double().requires_grad_(s["train"])
    score = torch.softmax(x, 1) if o["score"] == "softmax" else torch.sigmoid(x)
    value = score.detach() + (0 if s["bias"] is None else s["bias"].double())
    ids = _chosen(value, s["topk"], o["groups"], o["topk_groups"], o["group_top"])
    weights = score.gather(1, ids)
    if o["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    weights = weights * o["scale"]
    out = [weights.detach().t(), (ids + 1).int().t()]
    if s["train"]:
        (weights * s["d_weights"].t()).sum().backward()
        out.append(x.grad)
    return out


def _work_route(c):
    t, e, k, b = c["tokens"], c["experts"], c["topk"], BYTES[c["dtype"]]
    nbytes = t * e * b + t * k * 6 + (4 * e if c["bias"] else 0)
    if not c["train"]:
        return {"bytes": nbytes, "flops": 6 * t * e}
    return {"bytes": nbytes + 2 * t * e * b + t * k * 8, "flops": 12 * t * e}


# ------------------------------------------------------------------ the interface
_PREPARE = {"logprobs": _prepare_logprobs, "distill": _prepare_distill, "route": _prepare_route}
_OWN = {"logprobs": _own_logprobs, "distill": _own_distill, "route": _own_route}
_PLAIN = {"logprobs": _plain_logprobs, "distill": _plain_distill, "route": _plain_route}
_EXACT = {"logprobs": _exact_logprobs, "distill": _exact_distill, "route": _exact_route}
_WORK = {"logprobs": _work_logprobs, "distill": _work_distill, "route": _work_route}


def prepare(case, seed):
    return dict(_PREPARE[case["kind"]](case, _generator(seed)), kind=case["kind"])


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def work(case):
    return _WORK[case["kind"]](case)


def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))
