"""Log-probabilities, preference and policy losses with their gradients, and the norm / clip over a list of gradients, against plain 64-bit implementations.

Tolerances.  u = 2^-24.  A log-sum-exp sums V exponentials, at most V / 256 + 32 of them one after the other, each good to a few u plus u times its exponent; a
probability exp(z - lse) carries that error and u times its own exponent.  Rounding a value to its type costs eps / 2 of it.  Coefficients are compared with the
formula at the kernel's own log-probabilities, so that each stage is held to its own rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
IGNORE = -100


def K():
    from internevo_amd import kernels

    return kernels


def make(dev, rows, V, dtype, seed, pad=0, shift=0, mask=0.25, scale=3.0):
    """logits [rows, V] in rows of V + pad elements that start `shift` elements into a buffer, labels with a share of masked rows"""
    g = torch.Generator().manual_seed(seed)
    buf = torch.randn(rows * (V + pad) + shift, generator=g) * scale
    logits = buf.to(dtype).to(dev)[shift:].view(rows, V + pad)[:, :V]
    labels = torch.randint(0, V, (rows,), generator=g)
    labels[torch.rand(rows, generator=g) < mask] = IGNORE
    return logits, labels.to(dev)


def ref_logp(logits, labels, temperature=1.0, ignore=IGNORE):
    z = logits.detach().cpu().double() / temperature
    lab = labels.cpu()
    valid = (lab != ignore) & (lab >= 0) & (lab < z.shape[1])
    lse = torch.logsumexp(z, 1)
    lp = z.gather(1, torch.where(valid, lab, torch.zeros_like(lab))[:, None])[:, 0] - lse
    zero = torch.zeros_like(lp)
    return torch.where(valid, lp, zero), torch.where(valid, lse, zero), valid, z


def lp_tol(V, z):
    return U * (V / 256 + 64 + 4 * float(z[torch.isfinite(z)].abs().max()))


def check(got, ref, tol, what):
    got, ref = got.detach().cpu().double(), ref.cpu().double()
    assert got.shape == ref.shape, what
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    inf = ref.isinf()
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities"
    fin = ~(inf | ref.isnan())
    err = (got - ref).abs()[fin]
    tol = (tol.cpu() if torch.is_tensor(tol) else torch.full_like(ref, tol)).expand_as(ref)[fin]
    bad = err > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst error {float(err.max()):.3e}, {float((err / tol).max()):.2f} of its tolerance"


def check_dlogits(got, logits, labels, factor, what, temperature=1.0, ignore=IGNORE):
    """factor [rows], 64 bits: everything the row's gradient is multiplied by except 1 / temperature"""
    _, lse, valid, z = ref_logp(logits, labels, temperature, ignore)
    V = z.shape[1]
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(p)
    hot[torch.arange(p.shape[0])[valid], labels.cpu()[valid]] = 1.0
    g = (torch.where(valid, factor.cpu().double(), torch.zeros(())) / temperature)[:, None]
    ref = torch.where(g != 0, g * (hot - p), torch.zeros(()))
    eps = torch.finfo(got.dtype).eps / 2
    dist = torch.where(torch.isfinite(z), (z - lse[:, None]).abs(), torch.zeros(()))
    tol = (eps + 4 * U) * ref.abs() + g.abs() * p * (lp_tol(V, z) + U * (8 + 4 * dist)) + 2 * U * g.abs() * hot + 2.0 ** -125 * (1 + g.abs())
    check(got, ref, tol, what)


SIZES = [(1, 1), (3, 2), (5, 7), (4, 8), (2, 9), (7, 63), (3, 255), (33, 2047), (2, 2049), (9, 5003), (1, 32000), (3, 32003), (2, 92544), (2, 103168), (1, 131073)]
DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows, V", SIZES)
def test_token_logprobs_and_gradient(dev, rows, V, dtype):
    for pad, shift, temperature, mask in ((0, 0, 1.0, 0.0), (5, 1, 0.7, 0.3)):
        x, y = make(dev, rows, V, dtype, rows * 7919 + V, pad, shift, mask)
        logp, lse = K().token_logprobs(x, y, temperature=temperature)
        lp, ls, valid, z = ref_logp(x, y, temperature)
        check(logp, lp, lp_tol(V, z), "logp")
        check(lse, ls, lp_tol(V, z) + U * ls.abs(), "lse")
        c = torch.randn(rows, generator=torch.Generator().manual_seed(V)).to(dev)
        dloss = torch.full((1,), 8.0, device=dev)
        before = x.clone()
        d = K().token_logprobs_bwd(x, y, lse, c, dloss, 0.25, temperature=temperature, dlogits=torch.full_like(x, 7.0))
        assert torch.equal(x, before)
        check_dlogits(d, x, y, c.double() * 2.0, "dlogits", temperature)
        # in place over a strided buffer: the same bits, and nothing behind the rows is touched
        flat = torch.full((rows, V + 3), 5.0, dtype=dtype, device=dev)
        flat[:, :V] = x
        inplace = K().token_logprobs_bwd(flat[:, :V], y, lse, c, dloss, 0.25, temperature=temperature)
        assert inplace.data_ptr() == flat.data_ptr()
        assert torch.equal(flat[:, :V], d) and bool((flat[:, V:] == 5.0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
def test_masked_rows_are_never_read(dev, dtype):
    x, y = make(dev, 12, 1001, dtype, 1, mask=0.0)
    y[0], y[1], y[2], y[3] = IGNORE, -1, 1001, 1 << 40     # ignored, and three labels that are no column
    clean = x.clone()
    x[0], x[1], x[2], x[3] = math.nan, math.inf, -math.inf, math.nan
    logp, lse = K().token_logprobs(x, y)
    lp, ls, valid, z = ref_logp(clean, y)
    assert valid.tolist() == [False] * 4 + [True] * 8
    check(logp, lp, lp_tol(1001, z), "logp")
    d = K().token_logprobs_bwd(x, y, lse, torch.full((12,), math.nan, device=dev).masked_fill(torch.from_numpy(valid.numpy()).to(dev), 1.0))
    check_dlogits(d, clean, y, torch.ones(12), "dlogits")
    # another ignore_index: -100 is then a label that is no column, 5 is ignored
    y2 = torch.full((12,), 5, device=dev)
    y2[4] = 6
    logp, lse = K().token_logprobs(clean, y2, ignore_index=5)
    assert int((logp != 0).sum()) == 1
    # nothing valid at all
    none = torch.full((12,), IGNORE, device=dev)
    logp, lse = K().token_logprobs(x, none)
    assert not logp.any() and not lse.any()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
def test_infinite_and_nan_logits_in_live_rows(dev, dtype):
    V = 3000
    x, y = make(dev, 8, V, dtype, 2, mask=0.0)
    y[:] = torch.arange(8, device=dev) * 300 + 5
    lowest = torch.finfo(dtype).min
    x[0, 7:2900] = -math.inf                    # most of the vocabulary forbidden
    x[1] = lowest; x[1, 305] = 1.0              # ... by the type's lowest value
    x[2, 605] = -math.inf                       # the label itself forbidden
    x[3] = -math.inf                            # nothing allowed
    x[4, 11] = math.nan
    x[5, 12] = math.inf
    x[6] = lowest                               # uniform at the lowest value
    x[7, 2105] = 300.0                          # all of the probability on the label: logp 0
    logp, lse = K().token_logprobs(x, y)
    lp, ls, valid, z = ref_logp(x, y)
    tol = torch.full((8,), lp_tol(V, z[7:])).double()
    tol[6] = 2.0 ** 104 * 4                     # z of 3e38: its own rounding step
    lp[5] = math.nan                            # inf - inf
    got = logp.cpu().double()
    assert got[3].isnan() and got[4].isnan() and got[5].isnan() and got[2] == -math.inf
    check(got[[0, 1, 7]], lp[[0, 1, 7]], tol[[0, 1, 7]], "logp")
    assert abs(float(got[6]) + math.log(V)) <= lp_tol(V, torch.tensor([8.0]))
    sel = [0, 1, 7]
    d = K().token_logprobs_bwd(x, y, lse, torch.ones(8, device=dev), dlogits=torch.empty_like(x))
    check_dlogits(d[sel], x[sel], y[sel], torch.ones(3), "dlogits")
    assert bool(d[3].isnan().all()) and bool(d[4].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("centre, temperature", [(100.0, 1.0), (-300.0, 1.0), (5000.0, 1.0), (-40000.0, 3.0), (0.0, 0.01), (2.0, 1e-3)])
def test_gradient_of_rows_far_from_zero(dev, centre, temperature, dtype):
    """The gradient keeps its digits where the log-sum-exp is large.  A saved log-sum-exp below 128 (fp32 gradients) or 2048 (bf16) is off by 2^-18 or 2^-14 at
    most; everything else goes with the distance from it, not with its size."""
    for V in (90, 5003):
        x, y = make(dev, 9, V, dtype, V, 2, 1, 0.2, scale=3.0 * temperature)
        x += centre
        _, lse = K().token_logprobs(x, y, temperature=temperature)
        c = torch.linspace(0.5, 2.0, 9, device=dev)
        d = K().token_logprobs_bwd(x, y, lse, c, temperature=temperature, dlogits=torch.full_like(x, 7.0))
        _, ls, valid, z = ref_logp(x, y, temperature)
        p = torch.exp(z - ls[:, None])
        hot = torch.zeros_like(p)
        hot[torch.arange(9)[valid], y.cpu()[valid]] = 1.0
        g = (torch.where(valid, c.cpu().double(), torch.zeros(())) / temperature)[:, None]
        ref = torch.where(g != 0, g * (hot - p), torch.zeros(()))
        eps = torch.finfo(dtype).eps / 2
        share = U * (V / 256 + 64 + 8 + 4 * (z - ls[:, None]).abs()) + (2.0 ** -14 if dtype == torch.bfloat16 else 2.0 ** -18)
        check(d, ref, (eps + 4 * U) * ref.abs() + g.abs() * p * share + 2 * U * g.abs() * hot + 2.0 ** -125 * (1 + g.abs()), f"dlogits, {V} columns")
        inplace = x.clone()
        K().token_logprobs_bwd(inplace, y, lse, c, temperature=temperature)
        assert torch.equal(inplace, d)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
def test_log_probabilities_share_no_error(dev, dtype):
    """Answers of one row each and references next to their log-probabilities: the rewards then show what the log-probabilities are off before they are rounded to
    32 bits.  Each may be off by a few u; their mean over 8000 rows by 5 u / sqrt(8000) < u / 16 by chance and as much again by what all rows share: a sequence of n
    rows is off by n times that."""
    x, y = make(dev, 8000, 5003, dtype, 11, mask=0.0, scale=2.0)
    z = x.cpu().double()
    lp = z.gather(1, y.cpu()[:, None])[:, 0] - torch.logsumexp(z, 1)
    ref = lp.float()
    r = K().preference_loss_fwd(x, y, torch.arange(8001, dtype=torch.int32, device=dev), ref.to(dev), beta=1.0)
    off = r.rewards.cpu().double().reshape(-1) - (lp - ref.double())
    assert float(off.abs().max()) <= 8 * U and abs(float(off.mean())) <= U / 8


def pref_ref(logp, labels, cu, ref, beta, kind, eps, margin, average):
    """64-bit loss, rewards, sums and coefficients from given log-probabilities, and what the loss, the rewards and the coefficients may be off: the kernel sums its
    log-probabilities before they are rounded to 32 bits, u |lp| each and all of one sign, so that a sum may be off by u |sum|; the loss by its slope times that, a
    coefficient by the loss's second derivative times that -- at most beta^2 / 4, 0 and 2 of the three forms"""
    lp, lab = logp.cpu().double(), labels.cpu()
    S = len(cu) - 1
    sums = torch.zeros(S, dtype=torch.float64)
    live = []
    for s in range(S):
        idx = [t for t in range(cu[s], cu[s + 1]) if int(lab[t]) >= 0]
        live.append(idx)
        sums[s] = lp[idx].sum() / (max(1, len(idx)) if average else 1)
    h0 = (sums - ref.cpu().double()) if ref is not None else sums
    h0 = h0.clone().requires_grad_(True)
    h = h0[0::2] - h0[1::2]
    z = beta * h - margin
    if kind == "sigmoid":
        loss = -(1 - eps) * torch.nn.functional.logsigmoid(z) - eps * torch.nn.functional.logsigmoid(-z)
    elif kind == "hinge":
        loss = torch.relu(1 - z)
    else:
        loss = (h - 0.5 / beta) ** 2
    loss = loss.mean()
    loss.backward()
    coef = torch.zeros(lp.numel(), dtype=torch.float64)
    for s in range(S):
        if live[s]:
            coef[live[s]] = h0.grad[s] / (len(live[s]) if average else 1)
    off = U * sums.abs()
    bend = {"sigmoid": beta ** 2 / 4, "hinge": 0.0, "ipo": 2.0}[kind] / (S // 2) * (off[0::2] + off[1::2])
    coef_off = torch.zeros_like(coef)
    for s in range(S):
        coef_off[live[s]] = bend[s // 2] / (max(1, len(live[s])) if average else 1)
    tol = ((h0.grad.abs() * off).sum() + 2 * U * loss.detach().abs() + 1e-12, beta * off + 2 * U * (beta * h0.detach()).abs() + 1e-12,
           coef_off + 2 * U * coef.abs() + 2.0 ** -50)   # (the slope of a saturated sigmoid is a difference of 64-bit values: absolute 2^-50)
    return loss.detach(), beta * h0.detach(), sums, coef, tol


PREF = [dict(kind="sigmoid"), dict(kind="sigmoid", label_smoothing=0.2, margin=0.4), dict(kind="sigmoid", average=True, beta=2.0, margin=0.5), dict(kind="hinge", margin=0.3),
        dict(kind="ipo", average=True, beta=0.5), dict(kind="ipo"), dict(kind="sigmoid", beta=5.0)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("opt", PREF, ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()))
@pytest.mark.parametrize("cu", [[0, 1, 2], [0, 17, 40, 40, 61, 61, 61], [3, 9, 30, 55, 57], [0, 0, 0]], ids=["two-rows", "empty-answers", "rows-outside", "all-empty"])
def test_preference_loss(dev, cu, opt, dtype):
    rows, V = cu[-1] + (5 if cu[0] else 0) or 4, 517
    x, y = make(dev, rows, V, dtype, rows + len(cu), pad=1, mask=0.3 if rows > 4 else 0.0)
    S = len(cu) - 1
    base = K().token_logprobs(x, y)[0]
    g = torch.Generator().manual_seed(3)
    _, _, sums, _, _ = pref_ref(base, y, cu, None, 1.0, "sigmoid", 0, 0, opt.get("average", False))
    for with_ref in (True, False):
        ref = (sums + torch.randn(S, generator=g).double() / opt.get("beta", 0.1)).float().to(dev) if with_ref else None
        r = K().preference_loss_fwd(x, y, torch.tensor(cu, dtype=torch.int32, device=dev), ref, **opt)
        assert torch.equal(r.logp, base)
        args = (opt.get("beta", 0.1), opt["kind"], opt.get("label_smoothing", 0.0), opt.get("margin", 0.0), opt.get("average", False))
        loss, rewards, sums_, coef, tol = pref_ref(r.logp, y, cu, ref, *args)
        assert r.loss.shape == (1,) and r.rewards.shape == (S // 2, 2)
        check(r.loss, loss.reshape(1), tol[0], "loss")
        check(r.seq_logps, sums_, 2 * U * sums_.abs(), "seq_logps")
        check(r.rewards, rewards.reshape(-1, 2), tol[1].reshape(-1, 2), "rewards")
        check(r.coef, coef, tol[2], "coef")
        dloss = torch.full((1,), 64.0, device=dev)
        d = K().preference_loss_bwd(x, y, r, dloss, 0.5, dlogits=torch.empty_like(x))
        check_dlogits(d, x, y, r.coef.double() * 32.0, "dlogits")


def test_preference_loss_of_many_pairs_and_of_long_ones(dev):
    for rows, S in ((4000, 2 * 700), (5003, 4), (9000, 2)):
        x, y = make(dev, rows, 40, torch.float32, rows)
        g = torch.Generator().manual_seed(S)
        cu = [0] + sorted(torch.randint(0, rows + 1, (S - 1,), generator=g).tolist()) + [rows]
        ref = torch.randn(S, generator=g).to(dev)
        r = K().preference_loss_fwd(x, y, torch.tensor(cu, dtype=torch.int32, device=dev), ref, average=True)
        loss, rewards, sums, coef, tol = pref_ref(r.logp, y, cu, ref, 0.1, "sigmoid", 0.0, 0.0, True)
        check(r.loss, loss.reshape(1), tol[0], "loss")
        check(r.seq_logps, sums, 2 * U * sums.abs(), "seq_logps")
        check(r.coef, coef, tol[2], "coef")


def test_sums_of_a_long_sequence_keep_their_digits(dev):
    """3000 log-probabilities a sequence against 64 bits: their errors are rounding errors of 32-bit sums, independent from row to row (u sqrt(V / 256 + 64) each, five
    times the deviation of the sum allowed), and no common bias is left (the rounding of log2(e) alone would be 1.3e-8 of every row's mean distance from its maximum)."""
    rows, V = 6000, 3001
    x, y = make(dev, rows, V, torch.float32, 12, mask=0.0)
    r = K().preference_loss_fwd(x, y, torch.tensor([0, 3000, 6000], dtype=torch.int32, device=dev))
    lp = ref_logp(x, y)[0]
    for s in range(2):
        want = float(lp[3000 * s:3000 * s + 3000].sum())
        assert abs(float(r.seq_logps[s]) - want) <= U * abs(want) + 5 * U * math.sqrt(3000 * (V / 256 + 64)), (float(r.seq_logps[s]), want)


def test_broken_offsets_stay_inside_the_rows(dev):
    """Offsets that run backwards or past the rows are clamped: every output is written, nothing outside is touched (their values mean nothing)."""
    x, y = make(dev, 20, 64, torch.bfloat16, 5, mask=0.0)
    for cu in ([0, 30, 10], [-5, 12, 99], [15, 5, 20], [1 << 30, -(1 << 30), 7]):
        c = torch.tensor(cu, dtype=torch.int32, device=dev)
        r = K().preference_loss_fwd(x, y, c)
        assert bool(torch.isfinite(r.coef).all()) and bool(torch.isfinite(r.loss).all())
        p = K().policy_loss_fwd(x, y, r.logp, torch.ones(20, device=dev), cu_seqlens=c)
        assert bool(torch.isfinite(p.coef).all()) and bool(torch.isfinite(p.stats).all())


def policy_inputs(dev, x, y, seed, low, high, temperature=1.0):
    rows = x.shape[0]
    g = torch.Generator().manual_seed(seed)
    lp = ref_logp(x, y, temperature)[0]
    delta = torch.randn(rows, generator=g).double() * 0.3
    for b in (math.log(max(1 - low, 1e-9)), math.log(1 + high)):   # no ratio next to a border, where the gradient jumps
        delta = torch.where((delta - b).abs() < 1e-2, delta + 3e-2, delta)
    adv = torch.randn(rows, generator=g)
    adv[torch.rand(rows, generator=g) < 0.1] = 0.0
    return (lp - delta).float().to(dev), adv.to(dev), (lp + 0.4 * torch.randn(rows, generator=g).double()).float().to(dev)


def policy_ref(logp, labels, old, adv, ref, low, high, kl_coef, cu):
    lp = logp.cpu().double().requires_grad_(True)
    lab = labels.cpu()
    rows = lp.numel()
    w = torch.zeros(rows, dtype=torch.float64)
    if cu is None:
        live = lab >= 0
        w[live] = 1.0 / max(1, int(live.sum()))
    else:
        S = len(cu) - 1
        for s in range(S):
            idx = [t for t in range(cu[s], cu[s + 1]) if int(lab[t]) >= 0]
            if idx:
                w[idx] = 1.0 / (S * len(idx))
    on = w > 0
    zero = torch.zeros(rows, dtype=torch.float64)
    o, a = torch.where(on, old.cpu().double(), zero), torch.where(on, adv.cpu().double(), zero)
    ref = None if ref is None else torch.where(on, ref.cpu().double(), zero)
    r = torch.exp(lp - o)
    s = torch.where(on, -torch.minimum(r * a, r.clamp(1 - low, 1 + high) * a), torch.zeros(()))
    k = torch.zeros(rows, dtype=torch.float64)
    if ref is not None:
        q = ref - lp
        k = torch.where(on, torch.exp(q) - q - 1, torch.zeros(()))
    clipped = ((a > 0) & (r > 1 + high)) | ((a < 0) & (r < 1 - low))
    parts = [(w * s).sum(), (w * k).sum(), (w * clipped).sum()]
    loss = parts[0] + kl_coef * parts[1]
    if loss.requires_grad:
        loss.backward()
    coef = lp.grad if lp.grad is not None else torch.zeros(rows, dtype=torch.float64)
    size = w * (r.detach() * a.abs() + (kl_coef * (1 + torch.exp(ref - lp.detach())) if ref is not None else 0.0))
    err = U * (lp.detach().abs() + o.abs() + (ref.abs() if ref is not None else 0.0) + 16)
    return torch.stack([loss.detach(), *[t.detach() for t in parts]]), coef, torch.where(on, size * err, torch.zeros(())), float((w * k.detach() * 4 * U).sum())


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("kl", [None, 0.0, 0.1])
@pytest.mark.parametrize("rows, V, cu", [(1, 33, None), (37, 517, None), (1500, 65, None), (40, 1031, [0, 13, 13, 40]), (25, 32003, [2, 9, 20]), (3000, 40, list(range(0, 2701, 27))),
                                          (5000, 9, [3 + 3 * i - (i % 2) for i in range(1600)])],
                         ids=["one-row", "tokens", "many", "sequences", "rows-outside", "100-sequences", "1599-sequences"])
def test_policy_loss(dev, rows, V, cu, kl, dtype):
    low, high, tau = 0.2, 0.28, 0.8
    x, y = make(dev, rows, V, dtype, rows + V, pad=3, mask=0.3 if rows > 1 else 0.0)
    old, adv, ref = policy_inputs(dev, x, y, V, low, high, tau)
    masked = y < 0
    old[masked], adv[masked], ref[masked] = math.nan, math.inf, -math.inf        # masked rows' values decide nothing
    if kl is None:
        ref = None
    c = torch.tensor(cu, dtype=torch.int32, device=dev) if cu else None
    args = dict(ref_logps=ref, clip_low=low, clip_high=high, kl_coef=kl or 0.0, cu_seqlens=c, temperature=tau)
    f = K().policy_loss_fwd(x, y, old, adv, **args)
    lp, ls, valid, z = ref_logp(x, y, tau)
    check(f.logp, lp, lp_tol(V, z), "logp")
    stats, coef, tol, kl_tol = policy_ref(f.logp, y, old, adv, ref, low, high, kl or 0.0, cu)
    check(f.coef, coef, tol, "coef")
    check(f.stats, stats, 2 * U * stats.abs() + torch.tensor([float(tol.sum()) + kl_tol, float(tol.sum()), float(tol.sum()) + kl_tol, 4 * U]).double(), "stats")
    assert torch.equal(f.loss, f.stats[:1])
    dloss = torch.full((1,), 128.0, device=dev)
    d1 = K().policy_loss_bwd(x, y, f, dloss, 0.5, temperature=tau, dlogits=torch.empty_like(x))
    check_dlogits(d1, x, y, f.coef.double() * 64.0, "dlogits", tau)
    b, d2 = K().policy_loss_fwd_bwd(x, y, old, adv, dloss, 0.5, dlogits=torch.empty_like(x), **args)
    check(b.logp, lp, lp_tol(V, z), "logp (one pass)")
    stats, coef, tol, kl_tol = policy_ref(b.logp, y, old, adv, ref, low, high, kl or 0.0, cu)
    check(b.coef, coef, tol, "coef (one pass)")
    check(b.stats, stats, 2 * U * stats.abs() + torch.tensor([float(tol.sum()) + kl_tol, float(tol.sum()), float(tol.sum()) + kl_tol, 4 * U]).double(), "stats (one pass)")
    check_dlogits(d2, x, y, b.coef.double() * 64.0, "dlogits (one pass)", tau)
    x3 = x.clone()   # in place: the same bits
    b3, d3 = K().policy_loss_fwd_bwd(x3, y, old, adv, dloss, 0.5, **args)
    assert d3.data_ptr() == x3.data_ptr() and torch.equal(d3, d2) and torch.equal(b3.stats, b.stats)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows, V", SIZES + [(3, 9001), (2, 17001), (3, 45001), (2, 60007), (2, 70001)])
def test_policy_loss_in_one_pass_at_every_row_length(dev, rows, V, dtype):
    """Rows of every length class of the one-pass kernel (held whole, held in part, a rest behind the last whole vector), in place and apart, aligned and not."""
    for pad, shift, mask in ((0, 0, 0.0), (5, 1, 0.3)):
        x, y = make(dev, rows, V, dtype, rows * 31 + V, pad, shift, mask)
        old, adv, ref = policy_inputs(dev, x, y, V, 0.2, 0.2)
        dloss = torch.full((1,), 16.0, device=dev)
        before = x.clone()
        b, d = K().policy_loss_fwd_bwd(x, y, old, adv, dloss, dlogits=torch.full_like(x, 7.0), ref_logps=ref, kl_coef=0.1)
        lp, ls, valid, z = ref_logp(x, y)
        check(b.logp, lp, lp_tol(V, z), "logp")
        check(b.lse, ls, lp_tol(V, z) + U * ls.abs(), "lse")
        stats, coef, tol, kl_tol = policy_ref(b.logp, y, old, adv, ref, 0.2, 0.2, 0.1, None)
        check(b.coef, coef, tol, "coef")
        check_dlogits(d, x, y, b.coef.double() * 16.0, "dlogits")
        assert torch.equal(x, before)
        flat = torch.full((rows, V + 3), 5.0, dtype=dtype, device=dev)
        flat[:, :V] = x
        b2, d2 = K().policy_loss_fwd_bwd(flat[:, :V], y, old, adv, dloss, ref_logps=ref, kl_coef=0.1)
        assert torch.equal(flat[:, :V], d) and torch.equal(b2.stats, b.stats) and bool((flat[:, V:] == 5.0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", [3000, 60007, 92544])
def test_policy_loss_in_one_pass_with_infinite_and_lowest_logits(dev, dtype, V):
    """The rows of test_infinite_and_nan_logits_in_live_rows through the one-pass kernel: forbidden by -inf or by the type's lowest value, in part and as a whole."""
    x, y = make(dev, 6, V, dtype, 3, mask=0.0)
    y[:] = torch.arange(6, device=dev) * 300 + 5
    lowest = torch.finfo(dtype).min
    x[0, 7:2900] = -math.inf
    x[1] = lowest; x[1, 305] = 1.0
    x[2] = lowest                              # uniform at the lowest value
    x[3, 11] = math.nan
    x[4, 1205] = 300.0
    x[5, :] = -math.inf; x[5, 1505] = -2.0; x[5, 7] = -3.0
    zero, one = torch.zeros(6, device=dev), torch.ones(1, device=dev)
    want = K().token_logprobs(x, y)[0]
    old = torch.where(want.isnan(), zero, want)
    b, d = K().policy_loss_fwd_bwd(x, y, old, zero + 1.0, one, dlogits=torch.empty_like(x))
    f = K().policy_loss_fwd(x, y, old, zero + 1.0)
    e = K().policy_loss_bwd(x, y, f, one, dlogits=torch.empty_like(x))
    assert bool(b.logp[3].isnan()) and bool(d[3].isnan().all()) and bool(e[3].isnan().all())
    assert abs(float(b.logp[2]) + math.log(V)) <= lp_tol(V, torch.tensor([8.0]))
    sel = [0, 1, 4, 5]
    lp, ls, valid, z = ref_logp(x[sel], y[sel])
    check(b.logp[sel], lp, lp_tol(V, z), "logp")
    for got, r in ((d, b), (e, f)):
        check_dlogits(got[sel], x[sel], y[sel], r.coef[sel].double(), "dlogits")
        p = torch.full((V,), 1.0 / V, dtype=torch.float64)
        hot = torch.zeros(V, dtype=torch.float64)
        hot[605] = 1.0
        c = float(r.coef[2])
        check(got[2], c * (hot - p), (torch.finfo(dtype).eps / 2 + 16 * U) * abs(c) * (hot + p), "uniform row")


def test_policy_loss_without_a_token(dev):
    x, _ = make(dev, 6, 100, torch.bfloat16, 1)
    y = torch.full((6,), IGNORE, device=dev)
    z = torch.zeros(6, device=dev)
    for cu in (None, torch.tensor([0, 0, 6], dtype=torch.int32, device=dev)):
        r, d = K().policy_loss_fwd_bwd(x, y, z, z, torch.ones(1, device=dev), dlogits=torch.full_like(x, 3.0), cu_seqlens=cu)
        assert not r.stats.any() and not d.any() and not r.coef.any() and not r.logp.any()
    e = x[:0]
    r = K().policy_loss_fwd(e, y[:0], z[:0], z[:0])
    assert not r.stats.any()
    logp, lse = K().token_logprobs(e, y[:0])
    assert logp.numel() == 0
    p = K().preference_loss_fwd(e, y[:0], torch.tensor([0, 0, 0], dtype=torch.int32, device=dev))
    assert abs(float(p.loss) - math.log(2.0)) <= 2 * U


def test_gradients_against_differences(dev):
    """Central differences of the fp32 forward along a unit direction, step 1/64: truncation h^2 / 6 |L'''| <= 4e-5 x 4 (third derivatives of these losses along a
    unit direction stay below 4 at beta <= 0.5, |A| <= 3), rounding of the loss 2 u |L| / h <= 64 x 2^-23 x |L|."""
    rows, V, h = 24, 50, 1.0 / 64
    x, y = make(dev, rows, V, torch.float32, 9, mask=0.2, scale=1.0)
    g = torch.Generator().manual_seed(4)
    cu = torch.tensor([0, 5, 12, 20, 24], dtype=torch.int32, device=dev)
    old, adv, ref = policy_inputs(dev, x, y, 6, 0.2, 0.2)
    old, adv = ref_logp(x, y)[0].float().to(dev) + 0.02, adv.clamp(-3, 3)    # every ratio well inside the borders
    one = torch.ones(1, device=dev)
    cases = {
        "preference": (lambda t: K().preference_loss_fwd(t, y, cu, beta=0.5, label_smoothing=0.1, average=True).loss,
                       lambda t: K().preference_loss_bwd(t, y, K().preference_loss_fwd(t, y, cu, beta=0.5, label_smoothing=0.1, average=True), one)),
        "policy": (lambda t: K().policy_loss_fwd(t, y, old, adv, ref, kl_coef=0.2, cu_seqlens=cu).loss,
                   lambda t: K().policy_loss_fwd_bwd(t, y, old, adv, one, ref_logps=ref, kl_coef=0.2, cu_seqlens=cu)[1]),
    }
    for what, (loss, grad) in cases.items():
        d = grad(x.clone()).double()
        for i in range(6):
            v = torch.randn(rows, V, generator=g, dtype=torch.float64).to(dev)
            v = v / v.norm() if i else d / d.norm()
            up, down = float(loss((x.double() + h * v).float())), float(loss((x.double() - h * v).float()))
            slope = float((d * v).sum())
            assert abs((up - down) / (2 * h) - slope) <= 4e-5 * 4 + 64 * 2 * U * max(abs(up), abs(down)), (what, i, (up - down) / (2 * h), slope)


def test_rows_beyond_32_bit_offsets(dev):
    rows, V = 66000, 32800          # 2.16e9 elements; all rows but the last ones masked, so that only they are read
    x = torch.empty(rows, V, dtype=torch.bfloat16, device=dev)
    y = torch.full((rows,), IGNORE, device=dev)
    small, ysmall = make(dev, 3, V, torch.bfloat16, 8, mask=0.0)
    x[-3:], y[-3:] = small, ysmall
    old, adv, ref = policy_inputs(dev, small, ysmall, 2, 0.2, 0.2)
    z = torch.zeros(rows - 3, device=dev)
    one = torch.ones(1, device=dev)
    d = torch.empty_like(x)
    b, _ = K().policy_loss_fwd_bwd(x, y, torch.cat([z, old]), torch.cat([z, adv]), one, dlogits=d)
    bs, ds = K().policy_loss_fwd_bwd(small, ysmall, old, adv, one, dlogits=torch.empty_like(small))
    assert torch.equal(b.logp[-3:], bs.logp) and torch.equal(b.stats, bs.stats) and torch.equal(d[-3:], ds)
    assert not b.logp[:-3].any() and not any(part.any() for part in d[:-3].split(8192))
    d.fill_(1.0)
    K().token_logprobs_bwd(x, y, b.lse, b.coef, dlogits=d)
    assert not any(part.any() for part in d[:-3].split(8192))
    check_dlogits(d[-3:], small, ysmall, b.coef[-3:].double(), "dlogits")


# ------------------------------------------------------------------------------------------ gradient lists
def grad_list(dev, kind, seed, odd=True):
    g = torch.Generator().manual_seed(seed)
    sizes = {"few": [1, 7, 4096, 8, 65537], "empty": [0, 5, 0, 0, 3], "many": [1 + (i * 37) % 900 for i in range(300)], "chunks": [32768, 32769, 98303, 65536, 3]}[kind]
    out = []
    for i, n in enumerate(sizes):
        dtype = DTYPES[i % 2]
        t = (torch.randn(n + 3, generator=g) * 0.1).to(dtype).to(dev)
        out.append(t[1 + i % 3:1 + i % 3 + n] if odd else t[:n].clone())
    return out


@pytest.mark.parametrize("kind", ["few", "empty", "many", "chunks"])
def test_grad_norm_and_clip(dev, kind):
    ts = grad_list(dev, kind, 3)
    ref = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
    n = K().grad_norm(ts)
    assert n.shape == (1,) and abs(float(n) - ref) <= U * ref
    for max_norm in (0.3 * ref, 0.0, 10 * ref, math.inf):
        f = min(1.0, max_norm / (float(n) + 1e-6))
        outs = [torch.full((t.numel(),), 9.0, dtype=DTYPES[(i // 2) % 2], device=dev) for i, t in enumerate(ts)]
        before = [t.clone() for t in ts]
        got = K().clip_grad_norm_(ts, max_norm, out=outs)
        assert torch.equal(got, n) and all(torch.equal(a, b) for a, b in zip(ts, before))
        for t, o in zip(ts, outs):
            r = t.double() * f
            check(o, r, (torch.finfo(o.dtype).eps / 2 + 4 * U) * r.abs() + 1e-38, "out")
        mine = [t.clone() for t in ts]
        assert torch.equal(K().clip_grad_norm_(mine, max_norm), n)
        for t, o in zip(ts, mine):
            r = t.double() * f
            check(o, r, (torch.finfo(o.dtype).eps / 2 + 4 * U) * r.abs() + 1e-38, "in place")
            if f == 1.0:
                assert torch.equal(t, o)


def test_norm_of_one_tensor_many_times(dev):
    """more elements in all than one launch's chunks of the usual length hold (the tensors of a real list would not fit the card)"""
    t = torch.ones(1 << 30, dtype=torch.bfloat16, device=dev)
    assert float(K().grad_norm([t] * 300)) == pytest.approx(math.sqrt(300 * 2.0 ** 30), rel=2 * U)


def test_lists_without_an_element(dev):
    ts = [torch.empty(0, device=dev), torch.empty(0, dtype=torch.bfloat16, device=dev)]
    assert float(K().grad_norm(ts)) == 0.0 and float(K().clip_grad_norm_(ts, 1.0)) == 0.0


def test_clip_leaves_neighbours_alone(dev):
    flat = torch.ones(1000, dtype=torch.bfloat16, device=dev)
    K().clip_grad_norm_([flat[1:18], flat[19:500]], 1e-3)
    assert flat[0] == 1 and flat[18] == 1 and bool((flat[500:] == 1).all()) and float(flat[1]) < 1e-3 and float(flat[499]) < 1e-3


def test_norm_of_values_whose_squares_leave_fp32(dev):
    big = torch.full((5000,), 1e30, device=dev)
    assert abs(float(K().grad_norm([big, big[:10].bfloat16()])) / (1e30 * math.sqrt(5010)) - 1) <= 2.0 ** -8
    tiny = torch.full((40000,), 1e-30, device=dev)
    assert abs(float(K().grad_norm([tiny])) / 2e-28 - 1) <= 1e-6
    K().clip_grad_norm_([big], 1.0)
    assert abs(float(big[0]) * math.sqrt(5000) - 1) <= 1e-6


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_clip_with_non_finite_gradients(dev, bad):
    """torch.nn.utils.clip_grad_norm_'s rule: an infinite norm gives the factor 0, a NaN norm NaN."""
    ts = [torch.ones(100, device=dev), torch.ones(9, dtype=torch.bfloat16, device=dev)]
    ts[0][50] = bad
    n = K().clip_grad_norm_(ts, 1.0)
    if math.isnan(bad):
        assert bool(n.isnan()) and all(bool(t.isnan().all()) for t in ts)
    else:
        assert float(n) == math.inf and bool(ts[0][50].isnan()) and not ts[1].any() and int((ts[0] == 0).sum()) == 99


def test_clip_refuses_overlapping_tensors(dev):
    from internevo_amd._lib import InternEvoHipError

    t = torch.ones(100, device=dev)
    with pytest.raises(InternEvoHipError, match="overlap"):
        K().clip_grad_norm_([t, t], 1.0)
    with pytest.raises(InternEvoHipError, match="overlap"):
        K().clip_grad_norm_([t[:60], t[50:]], 1.0)
    with pytest.raises(InternEvoHipError, match="overlap"):
        K().clip_grad_norm_([t[:50], t[50:]], 1.0, out=[t[50:], torch.empty(50, device=dev)])
    assert bool((t == 1).all())
    assert abs(float(K().grad_norm([t, t])) - math.sqrt(200)) <= 1e-5    # the norm alone may see a tensor twice
    K().clip_grad_norm_([t], 1.0, out=[t])
    assert abs(float(t[0]) - 0.1) <= 1e-6


def test_gradient_longer_than_32_bit_offsets(dev):
    n = (1 << 32) + 12345
    t = torch.ones(n, dtype=torch.bfloat16, device=dev)
    assert abs(float(K().grad_norm([t])) / math.sqrt(n) - 1) <= 2 * U
    K().clip_grad_norm_([t], 0.5 * math.sqrt(n))
    assert bool((t[:1 << 20] == 0.5).all()) and bool((t[-(1 << 20):] == 0.5).all())


# ------------------------------------------------------------------------------------------ together, as a training step uses them
def test_alignment_step_end_to_end(dev):
    """Hidden states through the head product, the reference model's log-probabilities, the preference loss and the policy loss, their gradients through the head
    into its weight, and the clipped weight gradients -- against the same chain in 64 bits."""
    T, H, V = 96, 64, 1000
    g = torch.Generator().manual_seed(11)
    hid = torch.randn(T, H, generator=g).bfloat16().to(dev)
    w = (torch.randn(V, H, generator=g) * 0.2).bfloat16().to(dev)
    w_ref = (w.float() + 0.02 * torch.randn(V, H, generator=g).to(dev)).bfloat16()
    y = torch.randint(0, V, (T,), generator=g)
    cu = [0, 20, 45, 70, 90]
    for a, b in zip(cu, cu[1:]):
        y[a:a + 5] = IGNORE
    y[90:] = IGNORE
    y = y.to(dev)
    cud = torch.tensor(cu, dtype=torch.int32, device=dev)
    adv = torch.randn(T, generator=g).to(dev)
    logits, logits_ref = K().gemm(hid, w), K().gemm(hid, w_ref)
    ref_lp, _ = K().token_logprobs(logits_ref, y)
    ref_sums = torch.stack([ref_lp[a:b].sum() for a, b in zip(cu, cu[1:])])
    scale = torch.full((1,), 1024.0, device=dev)
    r = K().preference_loss_fwd(logits, y, cud, ref_sums, beta=0.3)
    d_pref = K().preference_loss_bwd(logits, y, r, scale, dlogits=torch.empty_like(logits))
    p, d_pol = K().policy_loss_fwd_bwd(logits, y, r.logp, adv, scale, dlogits=torch.empty_like(logits), ref_logps=ref_lp, kl_coef=0.1)
    grads = [K().gemm(d, hid, a_kmajor=True, b_kmajor=True) for d in (d_pref, d_pol)]
    clipped = [torch.empty(V, H, device=dev) for _ in grads]
    norm = K().clip_grad_norm_(grads, 5.0, out=clipped)
    # the same in 64 bits from the same logits
    x = logits.cpu().double().requires_grad_(True)
    lp = torch.log_softmax(x, 1).gather(1, y.cpu().clamp(min=0)[:, None])[:, 0] * (y.cpu() >= 0)
    sums = torch.stack([lp[a:b].sum() for a, b in zip(cu, cu[1:])]) - ref_sums.cpu().double()
    loss = -torch.nn.functional.logsigmoid(0.3 * (sums[0::2] - sums[1::2])).mean()
    dx1, = torch.autograd.grad(loss, x, retain_graph=True)
    live = y.cpu() >= 0
    q = ref_lp.cpu().double() - lp
    pol = ((-torch.exp(lp - r.logp.cpu().double()) * adv.cpu().double() + 0.1 * (torch.exp(q) - q - 1)) * live).sum() / int(live.sum())
    dx2, = torch.autograd.grad(pol, x)
    assert abs(float(r.loss) - float(loss)) <= 1e-4 and abs(float(p.loss) - float(pol)) <= 1e-4
    ws = [(dx * 1024.0).t() @ hid.cpu().double() for dx in (dx1, dx2)]
    n64 = math.sqrt(sum(float((t ** 2).sum()) for t in ws))
    # bf16 gradients in the logits and in the weight: half a step (2^-8) each, relative to the norm
    assert abs(float(norm) - n64) <= 2 * 2.0 ** -8 * n64
    f = min(1.0, 5.0 / n64)
    for got, t in zip(clipped, ws):
        err = float((got.cpu().double() - t * f).norm() / (t * f).norm())
        assert err <= 4 * 2.0 ** -8, err


def test_captured_calls_replay(dev):
    """One graph of the losses, their gradients and the clip; replayed with other inputs, eager work and synchronisation between the replays."""
    rows, V = 70, 2003
    xs = [make(dev, rows, V, torch.bfloat16, s)[0].clone() for s in range(4)]
    y = make(dev, rows, V, torch.bfloat16, 0)[1]
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device=dev)
    old, adv, ref = policy_inputs(dev, xs[0], y, 1, 0.2, 0.2)
    one = torch.ones(1, device=dev)
    x = xs[0].clone()
    d1, d2 = torch.empty_like(x), torch.empty_like(x)
    clipped = [torch.empty(rows, V, device=dev), torch.empty(rows, V, device=dev)]

    def step():
        r = K().preference_loss_fwd(x, y, cu)
        K().preference_loss_bwd(x, y, r, one, dlogits=d1)
        p, _ = K().policy_loss_fwd_bwd(x, y, old, adv, one, dlogits=d2, ref_logps=ref, kl_coef=0.1, cu_seqlens=cu)
        f = K().policy_loss_fwd(x, y, old, adv)
        norm = K().clip_grad_norm_([d1, d2], 0.01, out=clipped)
        return [r.loss, r.rewards, r.coef, p.stats, f.stats, norm, d1, d2, *clipped]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for s in (1, 2, 3, 1):
        x.copy_(xs[s])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_calls_on_a_side_stream_and_repeated(dev):
    x, y = make(dev, 400, 9001, torch.bfloat16, 3)
    old, adv, ref = policy_inputs(dev, x, y, 3, 0.2, 0.2)
    one = torch.ones(1, device=dev)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams * 2:
        with torch.cuda.stream(s):
            b, d = K().policy_loss_fwd_bwd(x, y, old, adv, one, dlogits=torch.empty_like(x), ref_logps=ref, kl_coef=0.1)
            outs.append((b.stats, d, K().grad_norm([d])))
    torch.cuda.synchronize()
    for a in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(outs[0], a))
