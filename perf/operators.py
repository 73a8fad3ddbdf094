"""Timed cases of the operators that train a policy on preferences or rewards (internevo_amd/kernels.py):

  logprobs    token_logprobs: log-probability of every row's label and the row's log-sum-exp
  preference  preference_loss_fwd / preference_loss_bwd: paired log-ratio loss and its gradient in the logits
  policy      policy_loss_fwd_bwd (or policy_loss_fwd + policy_loss_bwd): clipped policy loss with a KL term and its gradient
  clip        grad_norm / clip_grad_norm_: L2 norm over a list of gradients, and the clipped gradients

``own`` false computes each in elementary torch operations in 32 bits, ``own`` true calls the kernels.
"""
import math
import random

import torch

own = False

IGNORE = -100
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_LOGIT_OPS = ("logprobs", "preference", "policy")


# ------------------------------------------------------------------------------------------------ cases
def _rows(op, name, tokens, vocab, dtype="bf16", seqs=1, prompt=0.4, layout=1, pad=0, tail=0, temperature=1.0, **kw):
    """A case over logits [tokens, vocab]: `seqs` packed sequences, the share `prompt` of each masked, `tail` rows behind the last
    sequence, `pad` unused columns behind every row; `layout` seeds the sequence lengths (a plan, not data)."""
    case = dict(op=op, tokens=tokens, vocab=vocab, dtype=dtype, seqs=seqs, prompt=prompt, layout=layout, pad=pad, tail=tail, temperature=temperature)
    if name:
        case["name"] = name
    case.update(kw)
    return case


def _pref(kind="sigmoid", average=False, reference=True, beta=0.1, smoothing=0.0, margin=0.0, train=True, empty=False):
    return dict(kind=kind, average=average, reference=reference, beta=beta, smoothing=smoothing, margin=margin, train=train, empty=empty)


def _policy(form="fused", by_sequence=False, kl=0.05, low=0.2, high=0.2):
    return dict(form=form, by_sequence=by_sequence, kl=kl, low=low, high=high)


def _clip(name, hidden, layers, ffn, vocab, kv, grads="bf16", out="bf16", form="clip", odd=False, max_norm=1.0):
    """A case over the gradients of a decoder: per layer wqkv, wo, w1, w3, w2 and two norms; embedding, final norm and head if vocab > 0."""
    case = dict(op="clip", hidden=hidden, layers=layers, ffn=ffn, vocab=vocab, kv=kv, grads=grads, out=out, form=form, odd=odd, max_norm=max_norm)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the last tokens of a few candidate answers, scored while they are sampled: the smallest call, its latency counts
        _rows("logprobs", "logprobs_candidates", 8, 32000, prompt=0.0),
        # the reference policy's pass over a packed batch of the 7B model: half of the rows are prompt
        _rows("logprobs", "logprobs_reference", 8192, 92544, seqs=8, prompt=0.5, layout=2, tail=100),
        # fp32 logits of an odd vocabulary in padded rows, sampled at a temperature
        _rows("logprobs", "logprobs_fp32_odd", 1501, 50021, dtype="fp32", seqs=5, prompt=0.2, layout=3, pad=7, temperature=0.7),
        # one short pair: a user's smallest training call
        _rows("preference", "preference_one_pair", 96, 32000, seqs=2, layout=4, **_pref()),
        # one 16 384-token packed batch of the 7B model's vocabulary: eight pairs, forward and backward
        _rows("preference", "preference_batch", 16384, 92544, seqs=16, prompt=0.4, layout=5, tail=200, **_pref(smoothing=0.1)),
        # evaluation (forward only), length-normalised, squared form, an odd vocabulary, one answer without a token
        _rows("preference", "preference_eval_odd", 3001, 32003, dtype="fp32", seqs=14, prompt=0.3, layout=6, tail=17,
              **_pref(kind="ipo", average=True, reference=False, beta=0.5, train=False, empty=True)),
        # one short rollout
        _rows("policy", "policy_short", 33, 32000, prompt=0.25, layout=7, **_policy()),
        # one packed batch of rollouts at the 7B model's vocabulary, mean over the tokens, with the KL term
        _rows("policy", "policy_batch", 16384, 92544, seqs=32, prompt=0.25, layout=8, tail=200, **_policy()),
        # mean per sequence, asymmetric clip, fp32 logits of an odd vocabulary in padded rows, forward and backward apart
        _rows("policy", "policy_sequences_odd", 2501, 32003, dtype="fp32", seqs=9, prompt=0.3, layout=9, pad=5, tail=3, temperature=0.9,
              **_policy(form="split", by_sequence=True, kl=0.0, low=0.2, high=0.28)),
        # the gradients of a small test model: launches count, not bytes
        _clip("clip_small_model", 128, 2, 384, 1024, 64),
        # an eighth of the 7B model's layers (one pipeline stage), bf16 gradients into the optimizer's fp32 ones
        _clip("clip_stage", 4096, 4, 14336, 0, 1024, out="fp32"),
        # norm only, hundreds of tensors of odd sizes at unaligned addresses, two types (fp32 norms beside bf16 weights)
        _clip("norm_many_odd", 251, 60, 701, 5003, 83, grads="mixed", form="norm", odd=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(_LOGIT_OPS + ("clip",))
    if op == "clip":
        odd = rng.random() < 0.5
        hidden = _spread(rng, 32, 4096)
        if not odd:
            hidden = hidden // 8 * 8
        ffn, kv = int(hidden * rng.uniform(2.0, 3.5)), max(1, hidden // rng.choice([1, 2, 4, 8]))
        layers = _spread(rng, 1, max(1, min(60, int(4.5e8 / (hidden * (2 * hidden + 2 * kv + 3 * ffn))))))
        vocab = rng.choice([0, _spread(rng, 100, max(101, min(92544, int(7e7 / hidden))))])
        return _clip(None, hidden, layers, ffn, vocab, kv, grads=rng.choice(["bf16", "fp32", "mixed"]),
                     out=rng.choice(["bf16", "fp32"]), form=rng.choice(["clip", "clip", "norm"]), odd=odd, max_norm=rng.choice([0.5, 1.0, 1e6]))
    vocab = rng.choice([32000, 92544, 103168, _spread(rng, 500, 131072), _spread(rng, 500, 131072)])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    tokens = _spread(rng, 1 if op != "preference" else 4, max(8, min(16384, int((7e8 if dtype == "bf16" else 3.5e8) / vocab))))
    seqs = max(1, min(64, tokens // rng.choice([16, 100, 400])))
    extra = {}
    if op == "preference":
        seqs = max(2, seqs // 2 * 2)
        average = rng.random() < 0.4
        extra = _pref(kind=rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"]), average=average, reference=not average or rng.random() < 0.5,
                      beta=rng.choice([0.05, 0.1, 0.5, 2.0]), train=rng.random() < 0.75, empty=rng.random() < 0.2)
        if extra["kind"] == "sigmoid":
            extra["smoothing"] = rng.choice([0.0, 0.1])
        if extra["kind"] != "ipo":
            extra["margin"] = rng.choice([0.0, 0.3])
    elif op == "policy":
        extra = _policy(form=rng.choice(["fused", "fused", "split", "forward"]), by_sequence=rng.random() < 0.5, kl=rng.choice([0.0, 0.01, 0.2]),
                        low=rng.choice([0.1, 0.2]), high=rng.choice([0.2, 0.28]))
    return _rows(op, None, tokens, vocab, dtype=dtype, seqs=seqs, prompt=rng.choice([0.0, 0.3, 0.6]),
                 layout=rng.randrange(1 << 20), pad=rng.choice([0, 0, rng.randrange(1, 64)]), tail=rng.choice([0, tokens // 20]),
                 temperature=rng.choice([1.0, 1.0, 0.7]), **extra)


# ------------------------------------------------------------------------------------------------ plans
def _sequences(case):
    """(start, first answer row, end) of every sequence, from the case alone."""
    rng = random.Random(case["layout"])
    n, total = case["seqs"], case["tokens"] - case["tail"]
    cuts = sorted(rng.randrange(1, total) for _ in range(n - 1)) if total > n else list(range(1, n))
    if total > 4 * n:   # half way to equal lengths: a batch's sequences differ, but not without bound
        cuts = [(c + (i + 1) * total // n) // 2 for i, c in enumerate(cuts)]
    ends = [min(c, total) for c in cuts] + [total]
    out, begin = [], 0
    for i, end in enumerate(ends):
        answer = begin + int(case["prompt"] * (end - begin))
        if case.get("empty") and i == n - 1:
            answer = end
        out.append((begin, answer, end))
        begin = end
    return out


def _valid_rows(case):
    return sum(end - answer for _, answer, end in _sequences(case))


def _shapes(case):
    h, f, kv = case["hidden"], case["ffn"], case["kv"]
    sizes = [("wqkv", h * (h + 2 * kv)), ("wo", h * h), ("w1", f * h), ("w3", f * h), ("w2", h * f), ("attention_norm", h), ("ffn_norm", h)] * case["layers"]
    if case["vocab"]:
        sizes = [("embedding", case["vocab"] * h)] + sizes + [("norm", h), ("head", case["vocab"] * h)]
    fp32 = {"bf16": lambda what: False, "fp32": lambda what: True, "mixed": lambda what: what.endswith("norm")}[case["grads"]]
    return [(size, _DTYPES["fp32" if fp32(what) else "bf16"]) for what, size in sizes]


# ------------------------------------------------------------------------------------------------ states
def _label_logps64(logits, labels, temperature):
    """Log-probabilities of the labels in 64 bits (0 where there is none), in pieces of rows."""
    out = torch.zeros(labels.shape, dtype=torch.float64, device=labels.device)
    step = max(1, (1 << 27) // logits.shape[1])
    for a in range(0, labels.numel(), step):
        z = logits[a:a + step].double() / temperature
        lab = labels[a:a + step]
        lp = z.gather(1, lab.clamp(min=0)[:, None])[:, 0] - torch.logsumexp(z, 1)
        out[a:a + step] = torch.where(lab >= 0, lp, torch.zeros_like(lp))
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    if case["op"] == "clip":
        grads = []
        shapes = _shapes(case)
        if case["odd"]:   # views into two flat buffers, each one element behind the last: most of them start at an unaligned address
            flats = {t: randn(sum(n + 1 for n, d in shapes if d == t) + 1, dtype=t).mul_(0.01) for t in {d for _, d in shapes}}
            at = dict.fromkeys(flats, 1)
            for n, t in shapes:
                grads.append(flats[t][at[t]:at[t] + n])
                at[t] += n + 1
        else:
            grads = [randn(n, dtype=t).mul_(0.01) for n, t in shapes]
        out = None
        if case["form"] == "clip":   # the optimizer's gradient buffers, kept from step to step
            out = [torch.empty(n, dtype=torch.float32 if case["out"] == "fp32" else t, device=dev) for n, t in shapes]
        return dict(case=case, grads=grads, out=out)

    T, V = case["tokens"], case["vocab"]
    dtype = _DTYPES[case["dtype"]]
    logits = randn(T, V + case["pad"], dtype=dtype).mul_(2.0)[:, :V]
    labels = torch.full((T,), IGNORE, dtype=torch.int64, device=dev)
    drawn = torch.randint(0, V, (T,), generator=g, device=dev)
    spans = _sequences(case)
    for _, answer, end in spans:
        labels[answer:end] = drawn[answer:end]
    # a trained model puts most of its weight on few tokens: the label's logit is raised by 0 to 14
    boost = torch.rand(T, generator=g, device=dev) * 14.0
    logits.scatter_add_(1, drawn[:, None], boost[:, None].to(dtype))
    cu = torch.tensor([0] + [end for _, _, end in spans], dtype=torch.int32, device=dev)
    st = dict(case=case, logits=logits, labels=labels, cu=cu)
    if case["op"] == "logprobs":
        return st
    st["dloss"] = torch.full((1,), 256.0, device=dev)   # the loss scale of the step
    lp = _label_logps64(logits, labels, case["temperature"])
    if case["op"] == "preference":
        # the reference model's log-probabilities of the sequences: the policy has moved from them by about one unit
        sums = torch.stack([lp[a:e].sum() for _, a, e in spans])
        if case["average"]:
            sums = sums / torch.tensor([max(1, e - a) for _, a, e in spans], device=dev)
        st["ref"] = (sums + randn(len(spans)).double() / case["beta"]).float() if case["reference"] else None
        return st
    # log-probabilities of the policy that made the rollouts and of the reference model, near the present ones.  A ratio within 1e-3 of
    # a clip border is moved off it: there the gradient jumps, and 32 and 64 bits may stand on different sides
    delta = randn(T).double() * 0.15
    for border in (math.log(1.0 - case["low"]), math.log(1.0 + case["high"])):
        delta = torch.where((delta - border).abs() < 1e-3, delta + 4e-3, delta)
    st["old"] = (lp - delta).float()
    st["ref"] = (lp + randn(T).double() * 0.2).float() if case["kl"] > 0 else None
    st["adv"] = randn(T)
    if case["by_sequence"]:   # one advantage for a whole answer
        for a, _, e in spans:
            if e > a:
                st["adv"][a:e] = st["adv"][a].clone()
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_softmax(logits, labels, temperature):
    z = logits.float() / temperature
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    s = e.sum(1, keepdim=True)
    lse = (m + torch.log(s))[:, 0]
    valid = labels >= 0
    logp = z.gather(1, labels.clamp(min=0)[:, None])[:, 0] - lse
    zero = torch.zeros_like(lse)
    return torch.where(valid, logp, zero), torch.where(valid, lse, zero), valid, e, s


def _plain_dlogits(logits, labels, valid, e, s, dlogp, temperature):
    d = e * (-dlogp / temperature)[:, None] / s
    d.scatter_add_(1, labels.clamp(min=0)[:, None], (dlogp / temperature)[:, None])
    return (d * valid[:, None]).to(logits.dtype)


def _plain_log_sigmoid(z):
    return -(torch.log1p(torch.exp(-z.abs())) + (-z).clamp(min=0))


def _plain_preference(st):
    c = st["case"]
    logp, lse, valid, e, s = _plain_softmax(st["logits"], st["labels"], c["temperature"])
    n = c["seqs"]
    seq = torch.bucketize(torch.arange(c["tokens"], device=logp.device, dtype=torch.int32), st["cu"], right=True, out_int32=True).long() - 1
    inside = valid & (seq < n)
    seq = seq.clamp(max=n - 1)
    total = torch.zeros(n, dtype=torch.float64, device=logp.device).index_add_(0, seq, (logp * inside).double())
    count = torch.zeros(n, dtype=torch.float64, device=logp.device).index_add_(0, seq, inside.double())
    if c["average"]:
        total = total / count.clamp(min=1)
    gain = total - (st["ref"].double() if c["reference"] else 0.0)
    h = gain[0::2] - gain[1::2]
    beta, eps = c["beta"], c["smoothing"]
    z = beta * h - c["margin"]
    if c["kind"] == "sigmoid":
        loss = -(1 - eps) * _plain_log_sigmoid(z) - eps * _plain_log_sigmoid(-z)
        dh = beta * (eps / (1 + torch.exp(-z)) - (1 - eps) / (1 + torch.exp(z)))
    elif c["kind"] == "hinge":
        loss = (1 - z).clamp(min=0)
        dh = -beta * (z < 1).double()
    else:
        loss = (h - 0.5 / beta) ** 2
        dh = 2 * (h - 0.5 / beta)
    out = [loss.mean().float().reshape(1), (beta * gain).float().reshape(-1, 2), total.float()]
    if c["train"]:
        w = torch.stack([dh, -dh], 1).reshape(-1) / (n // 2)
        if c["average"]:
            w = w / count.clamp(min=1)
        dlogp = (w[seq] * inside).float() * st["dloss"]
        out.append(_plain_dlogits(st["logits"], st["labels"], valid, e, s, dlogp, c["temperature"]))
    return out


def _plain_policy(st):
    c = st["case"]
    logp, lse, valid, e, s = _plain_softmax(st["logits"], st["labels"], c["temperature"])
    zero = torch.zeros_like(logp)
    if c["by_sequence"]:
        n = c["seqs"]
        seq = torch.bucketize(torch.arange(c["tokens"], device=logp.device, dtype=torch.int32), st["cu"], right=True, out_int32=True).long() - 1
        inside = valid & (seq < n)
        seq = seq.clamp(max=n - 1)
        count = torch.zeros(n, device=logp.device).index_add_(0, seq, inside.float())
        w = torch.where(inside, 1.0 / (n * count.clamp(min=1))[seq], zero)
    else:
        w = valid.float() / valid.float().sum().clamp(min=1)
    adv = torch.where(valid, st["adv"], zero)
    ratio = torch.exp(torch.where(valid, logp - st["old"], zero))
    low, high = 1 - c["low"], 1 + c["high"]
    clipped = ((adv > 0) & (ratio > high)) | ((adv < 0) & (ratio < low))
    surrogate = -torch.minimum(ratio * adv, ratio.clamp(low, high) * adv)
    dlogp = torch.where(clipped, zero, -ratio * adv)
    kl = zero
    if c["kl"] > 0:
        d = torch.where(valid, st["ref"] - logp, zero)
        kl = torch.exp(d) - d - 1
        dlogp = dlogp + c["kl"] * (1 - torch.exp(d))
    sums = [(w.double() * t.double()).sum() for t in (surrogate, kl, clipped)]
    stats = torch.stack([sums[0] + c["kl"] * sums[1], *sums]).float()
    out = [stats, logp]
    if c["form"] != "forward":
        out.append(_plain_dlogits(st["logits"], st["labels"], valid, e, s, dlogp * w * st["dloss"], c["temperature"]))
    return out


def _plain_clip(st):
    c = st["case"]
    total = torch.zeros(1, dtype=torch.float64, device=st["grads"][0].device)
    for t in st["grads"]:
        total += (t.float() ** 2).sum().double()
    norm = torch.sqrt(total).float()
    if c["form"] == "norm":
        return [norm]
    factor = (c["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for t, o in zip(st["grads"], st["out"]):
        o.copy_(t.float() * factor)
    return [norm, *st["out"]]


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    c = st["case"]
    if not own:
        if c["op"] == "logprobs":
            return list(_plain_softmax(st["logits"], st["labels"], c["temperature"])[:2])
        return {"preference": _plain_preference, "policy": _plain_policy, "clip": _plain_clip}[c["op"]](st)
    from internevo_amd import kernels as K

    if c["op"] == "clip":
        if c["form"] == "norm":
            return [K.grad_norm(st["grads"])]
        return [K.clip_grad_norm_(st["grads"], c["max_norm"], out=st["out"]), *st["out"]]
    x, labels, t = st["logits"], st["labels"], c["temperature"]
    if c["op"] == "logprobs":
        return list(K.token_logprobs(x, labels, temperature=t))
    if c["op"] == "preference":
        r = K.preference_loss_fwd(x, labels, st["cu"], st["ref"], beta=c["beta"], kind=c["kind"], label_smoothing=c["smoothing"], margin=c["margin"],
                                  average=c["average"], temperature=t)
        out = [r.loss, r.rewards, r.seq_logps]
        if c["train"]:
            out.append(K.preference_loss_bwd(x, labels, r, st["dloss"], temperature=t, dlogits=torch.empty_like(x)))
        return out
    args = dict(ref_logps=st["ref"], clip_low=c["low"], clip_high=c["high"], kl_coef=c["kl"], cu_seqlens=st["cu"] if c["by_sequence"] else None, temperature=t)
    if c["form"] == "fused":
        r, d = K.policy_loss_fwd_bwd(x, labels, st["old"], st["adv"], st["dloss"], dlogits=torch.empty_like(x), **args)
        return [r.stats, r.logp, d]
    r = K.policy_loss_fwd(x, labels, st["old"], st["adv"], **args)
    if c["form"] == "forward":
        return [r.stats, r.logp]
    return [r.stats, r.logp, K.policy_loss_bwd(x, labels, r, st["dloss"], temperature=t, dlogits=torch.empty_like(x))]


# ------------------------------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "clip":
        shapes = _shapes(case)
        bytes_ = sum(n * t.itemsize for n, t in shapes)
        elems = sum(n for n, _ in shapes)
        if case["form"] == "norm":
            return {"bytes": bytes_ + 4, "flops": 2 * elems}
        return {"bytes": bytes_ + sum(n * (4 if case["out"] == "fp32" else t.itemsize) for n, t in shapes) + 4, "flops": 3 * elems}
    T, V, size = case["tokens"], case["vocab"], _DTYPES[case["dtype"]].itemsize
    valid = _valid_rows(case)   # a masked row's logits decide nothing
    bytes_, flops = valid * V * size + T * 8, 3 * valid * V   # per logit: difference, exponential, sum
    if case["op"] == "logprobs":
        return {"bytes": bytes_ + T * 8, "flops": flops}
    train = case["train"] if case["op"] == "preference" else case["form"] != "forward"
    if case["op"] == "preference":
        bytes_ += case["seqs"] * 16
    else:
        bytes_ += T * (12 + (4 if case["kl"] > 0 else 0))
    if train:
        bytes_ += T * V * size
        flops += 2 * valid * V
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "clip":
        squares = [torch.dot(t.double(), t.double()) for t in st["grads"]]
        norm = torch.stack(squares).sum().sqrt()
        if case["form"] == "norm":
            return [norm.reshape(1)]
        factor = min(1.0, case["max_norm"] / (norm.item() + 1e-6))
        return [norm.reshape(1), *(t.double() * factor for t in st["grads"])]

    x, labels, tau = st["logits"], st["labels"], case["temperature"]
    T, V = x.shape
    spans = _sequences(case)
    rows = torch.nonzero(labels != IGNORE)[:, 0]
    lp, lse = torch.zeros(T, dtype=f64, device=x.device), torch.zeros(T, dtype=f64, device=x.device)
    pieces = rows.split(max(1, (1 << 27) // V))
    for r in pieces:
        z = x[r].double() / tau
        lse[r] = torch.logsumexp(z, 1)
        lp[r] = z[torch.arange(r.numel(), device=x.device), labels[r]] - lse[r]
    if case["op"] == "logprobs":
        return [lp, lse]
    weight = torch.zeros(T, dtype=f64, device=x.device)   # d loss / d log-probability, by hand from the definition
    scale = float(st["dloss"])
    if case["op"] == "preference":
        beta, P = case["beta"], case["seqs"] // 2
        sums = [lp[a:e].sum().item() / (max(1, e - a) if case["average"] else 1) for _, a, e in spans]
        ref = st["ref"].double().tolist() if case["reference"] else [0.0] * len(spans)
        loss, rewards = 0.0, []
        for i in range(P):
            win, lose = sums[2 * i] - ref[2 * i], sums[2 * i + 1] - ref[2 * i + 1]
            rewards.append([beta * win, beta * lose])
            h = win - lose
            z = beta * h - case["margin"]
            if case["kind"] == "sigmoid":
                softplus = lambda v: max(v, 0.0) + math.log1p(math.exp(-abs(v)))   # noqa: E731
                sigma = 0.5 * (1.0 + math.tanh(0.5 * z))
                loss += (1 - case["smoothing"]) * softplus(-z) + case["smoothing"] * softplus(z)
                slope = beta * (sigma - (1 - case["smoothing"]))
                if z > 0:   # 1 - sigma without cancellation
                    slope = beta * (case["smoothing"] - 1 / (1 + math.exp(min(z, 700.0))))
            elif case["kind"] == "hinge":
                loss += max(0.0, 1 - z)
                slope = -beta if z < 1 else 0.0
            else:
                loss += (h - 1 / (2 * beta)) ** 2
                slope = 2 * (h - 1 / (2 * beta))
            for sign, (_, a, e) in ((1, spans[2 * i]), (-1, spans[2 * i + 1])):
                if e > a:
                    weight[a:e] = sign * slope / P / ((e - a) if case["average"] else 1)
        out = [torch.tensor([loss / P], dtype=f64, device=x.device), torch.tensor(rewards, dtype=f64, device=x.device),
               torch.tensor(sums, dtype=f64, device=x.device)]
        if not case["train"]:
            return out
    else:
        mean = torch.zeros(T, dtype=f64, device=x.device)
        for _, a, e in spans:
            if e > a:
                mean[a:e] = 1.0 / (len(spans) * (e - a)) if case["by_sequence"] else 1.0 / rows.numel()
        adv, ratio = st["adv"][rows].double(), torch.exp(lp[rows] - st["old"][rows].double())
        bound = torch.where(adv > 0, torch.full_like(ratio, 1 + case["high"]), torch.full_like(ratio, 1 - case["low"]))
        cut = (adv != 0) & ((ratio - bound) * adv > 0)
        gain = torch.where(cut, bound, ratio) * adv
        slope = torch.where(cut, torch.zeros_like(ratio), -ratio * adv)
        kl = torch.zeros_like(ratio)
        if case["kl"] > 0:
            q = torch.exp(st["ref"][rows].double() - lp[rows])
            kl = q - q.log() - 1
            slope = slope + case["kl"] * (1 - q)
        m = mean[rows]
        parts = [-(m * gain).sum(), (m * kl).sum(), (m * cut).sum()]
        out = [torch.stack([parts[0] + case["kl"] * parts[1], *parts]), lp]
        if case["form"] == "forward":
            return out
        weight[rows] = slope * m
    d = torch.zeros(T, V, dtype=f64, device=x.device)
    for r in pieces:
        p = torch.exp(x[r].double() / tau - lse[r, None])
        p[torch.arange(r.numel(), device=x.device), labels[r]] -= 1
        d[r] = p * (-weight[r] * scale / tau)[:, None]
    return [*out, d]
