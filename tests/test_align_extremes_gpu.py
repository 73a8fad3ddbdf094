"""Preference and policy losses where logits, temperatures or given log-probabilities are extreme but finite, or infinite where the formulas still have a value.

Tolerances.  u = 2^-24.  The reference subtracts the row's maximum in 64 bits before it divides by the temperature, so that its log-probabilities keep their digits however
far from zero the logits lie.  A log-probability is off by its rounding, u of it, and by what the sum of exponentials is off: at most V / 256 + 32 of them added one
after the other, each good to a few u (u (V / 256 + 64) in all), and 4 u of every term's distance from the maximum, weighted with its probability."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
IGNORE = -100
DTYPES = [torch.bfloat16, torch.float32]


def K():
    from internevo_amd import kernels

    return kernels


def check(got, ref, tol, what):
    got, ref = got.detach().cpu().double(), ref.cpu().double()
    assert got.shape == ref.shape, what
    assert not got.isnan().any(), f"{what}: {int(got.isnan().sum())} NaN of {got.numel()}"
    inf = ref.isinf()
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities"
    tol = (tol.cpu() if torch.is_tensor(tol) else torch.tensor(tol)).double().expand_as(ref)[~inf]
    err = (got - ref).abs()[~inf]
    assert not (err > tol).any(), f"{what}: {int((err > tol).sum())} of {err.numel()} off, worst error {float(err.max()):.3e}, {float((err / tol).max()):.2f} of its tolerance"


class Ref:
    """64-bit log-probabilities, log-sum-exps and probabilities of rows that all have a label"""

    def __init__(self, x, y, temperature):
        z = x.cpu().double()
        top = z.amax(1, keepdim=True)
        self.z = (z - top) / temperature
        self.sum = torch.logsumexp(self.z, 1, keepdim=True)
        self.p = torch.exp(self.z - self.sum)
        self.hot = torch.zeros_like(self.p)
        self.hot[torch.arange(z.shape[0]), y.cpu()] = 1.0
        self.logp = (self.z - self.sum).gather(1, y.cpu()[:, None])[:, 0]
        self.dist = torch.where(torch.isfinite(self.z), self.z.abs(), torch.zeros(()))
        self.lse = (top / temperature + self.sum)[:, 0]
        self.sum_tol = U * (z.shape[1] / 256 + 64) + 4 * U * (self.p * self.dist).sum(1)
        self.logp_tol = self.sum_tol + U * self.logp.abs()
        self.temperature = temperature

    def check_dlogits(self, got, factor, what):
        """factor [rows]: what the row's gradient is multiplied by except 1 / temperature; rows of factor 0 are zeros"""
        g = (factor.cpu().double() / self.temperature)[:, None]
        ref = g * (self.hot - self.p)
        # a saved log-sum-exp of fp32 (bf16) logits within 128 (2048) of zero leaves 2^-18 (2^-14) of a probability
        share = self.sum_tol[:, None] + U * (8 + 4 * (self.dist + self.sum)) + (2.0 ** -14 if got.dtype == torch.bfloat16 else 2.0 ** -18)
        check(got, ref, (torch.finfo(got.dtype).eps / 2 + 4 * U) * ref.abs() + g.abs() * self.p * share + 2 * U * g.abs() * self.hot + 2.0 ** -125 * (1 + g.abs()), what)


def everything(dev, x, y, t):
    """Every forward, both backwards and the one-pass kernel over the same rows (eight, all with a label), against 64 bits"""
    rows, V = x.shape
    ref = Ref(x, y, t)
    logp, lse = K().token_logprobs(x, y, temperature=t)
    check(logp, ref.logp, ref.logp_tol, "logp")
    check(lse, ref.lse, ref.sum_tol + 2 * U * ref.lse.abs(), "lse")
    c = torch.linspace(-1.0, 1.5, rows, device=dev)
    d = K().token_logprobs_bwd(x, y, lse, c, temperature=t, dlogits=torch.full_like(x, 7.0))
    ref.check_dlogits(d, c, "dlogits")
    inplace = x.clone()
    assert torch.equal(K().token_logprobs_bwd(inplace, y, lse, c, temperature=t), d)
    # one pair
    one = torch.ones(1, device=dev)
    cut = rows // 2
    cu = torch.tensor([0, cut, rows], dtype=torch.int32, device=dev)
    r = K().preference_loss_fwd(x, y, cu, beta=0.1, temperature=t)
    sums = torch.stack([ref.logp[:cut].sum(), ref.logp[cut:].sum()])
    off = torch.stack([ref.sum_tol[:cut].sum(), ref.sum_tol[cut:].sum()]) + U * sums.abs()
    check(r.seq_logps, sums, off, "seq_logps")
    check(r.rewards, 0.1 * sums.reshape(1, 2), 0.1 * off.reshape(1, 2) + 2 * U * 0.1 * sums.abs().reshape(1, 2), "rewards")
    h = 0.1 * float(sums[0] - sums[1])
    loss = max(-h, 0.0) + math.log1p(math.exp(-abs(h)))
    slope = -0.1 * (1.0 / (1.0 + math.exp(h)) if h < 700 else 0.0)
    check(r.loss, torch.tensor([loss]), 0.1 * float(off.sum()) + 2 * U * loss + 1e-12, "loss")
    coef = torch.cat([torch.full((cut,), slope), torch.full((rows - cut,), -slope)]).double()
    check(r.coef, coef, 0.0025 * float(off.sum()) + 2 * U * coef.abs() + 2.0 ** -50, "coef")
    ref.check_dlogits(K().preference_loss_bwd(x, y, r, one, temperature=t, dlogits=torch.empty_like(x)), r.coef, "dlogits of the pair")
    # a policy near its own log-probabilities; rows whose label has next to no probability are left out (their ratio is that of two huge numbers)
    on = ref.logp > -50
    assert on.any()
    y = torch.where(on.to(dev), y, torch.full_like(y, IGNORE))
    old = (ref.logp - 0.02).float()
    other = (ref.logp + 0.1).float()
    adv = torch.linspace(-1.25, 2.0, rows)
    w = on.double() / int(on.sum())
    ratio, q = torch.exp(ref.logp - old.double()), other.double() - ref.logp
    coef = w * (-ratio * adv.double() + 0.3 * (1 - torch.exp(q)))
    tol = w * (ratio * adv.abs().double() + 0.3 * (1 + torch.exp(q))) * (ref.logp_tol + 16 * U) + 2.0 ** -120
    coef, tol = torch.where(on, coef, torch.zeros(())), torch.where(on, tol, torch.zeros(()))
    old, other, adv = old.to(dev), other.to(dev), adv.to(dev)
    args = dict(ref_logps=other, kl_coef=0.3, temperature=t)
    b, d = K().policy_loss_fwd_bwd(x, y, old, adv, one, dlogits=torch.full_like(x, 7.0), **args)
    f = K().policy_loss_fwd(x, y, old, adv, cu_seqlens=torch.tensor([0, rows], dtype=torch.int32, device=dev), **args)
    e = K().policy_loss_bwd(x, y, f, one, temperature=t, dlogits=torch.full_like(x, 7.0))
    for got, grad, what in ((b, d, "one pass"), (f, e, "forward, backward")):
        check(got.logp, torch.where(on, ref.logp, torch.zeros(())), ref.logp_tol, what + ": logp")
        check(got.coef, coef, tol, what + ": coef")
        assert bool(torch.isfinite(got.stats).all()), what
        ref.check_dlogits(grad, got.coef, what + ": dlogits")
    inplace = x.clone()
    _, d2 = K().policy_loss_fwd_bwd(inplace, y, old, adv, one, **args)
    assert torch.equal(d2, d)


WIDTHS = [90, 3001, 20011, 60007, 92544]   # 64, 256, 512 and 1024 threads a row, rows held whole and in part


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", WIDTHS)
@pytest.mark.parametrize("fill, t", [(-1e5, 1.0), (-1e7, 1.0), (-1e9, 1.0), (-1e9, 0.3), (-1e9, 0.1), (-1e10, 1.0), (-1e12, 1.0), (-1e20, 1.0), (-1e29, 1.0), (-1e29, 50.0)])
def test_finite_fill_values(dev, fill, t, V, dtype):
    """Parts of the vocabulary forbidden by a finite value: whole threads, single vectors, the row's last elements, the whole row, the label itself."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(8, V, generator=g) * 3).to(dtype).to(dev)
    y = torch.full((8,), V // 3 + 2, device=dev)
    column = torch.arange(V, device=dev)
    x[0] = torch.where((column >= V // 3) & (column < V // 3 + 5), x[0], fill)
    x[1] = torch.where((column // 8 % 2 == 0) & (column != V // 3 + 2), torch.full_like(x[1], fill), x[1])
    x[2, V - V % 8 - 8:] = fill
    x[3] = fill
    x[4] = fill
    x[4, V // 3 + 2] = fill * (1 - 2.0 ** -6)
    x[5, V // 3 + 2] = fill
    x[6] = torch.where(column < V // 2, torch.full_like(x[6], -fill), torch.full_like(x[6], fill))
    x[7] = torch.where(column < V // 2, torch.full_like(x[7], fill), torch.full_like(x[7], 2 * fill))
    everything(dev, x, y, t)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", WIDTHS)
@pytest.mark.parametrize("t", [1e-4, 1e-5, 1e-6, 1e-7, 1e-8, 1e-12, 1e-20, 1e-29])
def test_small_temperatures(dev, t, V, dtype):
    """Largest logits of 0, 11.2 and 20.3 that several columns share (fp32: with the next smaller numbers beside them), the label one of them in most rows"""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(8, V, generator=g).clamp(-4, 4) * 2 - 9).to(dtype)
    y = torch.zeros(8, dtype=torch.int64)
    for i, top in enumerate((0.0, 11.19, 20.3, -0.3, 11.19, 20.3, 1e-3, 3.0)):
        at = torch.randperm(V, generator=g)[:9]
        v = torch.tensor(top).to(dtype)
        x[i, at[:5]] = v
        if dtype == torch.float32:
            for a in at[5:]:
                v = torch.nextafter(v, torch.tensor(-math.inf))
                x[i, a] = v
        y[i] = at[0] if i != 4 else (at[8] + 1) % V
    everything(dev, x.to(dev), y.to(dev), t)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", WIDTHS)
@pytest.mark.parametrize("centre", [726817.4, -726817.4, 1453634.9, -1453634.9, 9.9e5, -9.9e5, 3e6, 1e9, -1e9, 1e20, -1e20])
def test_logits_far_from_zero(dev, centre, V, dtype):
    """Rows around one large value, logits of both sides of a power of two of log 2 among them (2^20 log 2 = 726817.4)."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(8, V, generator=g) * 3 + centre).to(dtype).to(dev)
    x[:4, :V // 3] -= abs(centre) / 16
    everything(dev, x, x.argmax(1), 1.0)


def pair_formula(kind, eps, beta, h):
    """loss and its slope in h of one pair, infinite log-ratios as limits"""
    z = beta * h
    sig = 0.0 if z == -math.inf else 1.0 / (1.0 + math.exp(-z)) if z > -700 else math.exp(z)
    if kind == "sigmoid":
        soft = [math.inf if v == math.inf else 0.0 if v == -math.inf else max(v, 0.0) + math.log1p(math.exp(-abs(v))) for v in (-z, z)]
        return (1 - eps) * soft[0] + (eps * soft[1] if eps else 0.0), beta * (eps * sig - (1 - eps) * (1.0 - sig))
    if kind == "hinge":
        return max(0.0, 1.0 - z), -beta if z < 1 else 0.0
    return (h - 0.5 / beta) ** 2, 2 * (h - 0.5 / beta)


FORMS = [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)]


@pytest.mark.parametrize("pairs", [1, 2, 3, 7, 9])
@pytest.mark.parametrize("kind, eps", FORMS)
@pytest.mark.parametrize("where, value", [(0, -math.inf), (0, math.inf), (1, -math.inf), (1, math.inf)])
def test_infinite_reference_log_probabilities(dev, where, value, kind, eps, pairs):
    """The log-ratio of the last pair is infinite: its loss is 0 or infinite, its slope a limit, and the other pairs are as they were."""
    rows, V, beta = 6 * pairs, 211, 0.4
    g = torch.Generator().manual_seed(pairs)
    x, y = torch.randn(rows, V, generator=g).to(dev), torch.randint(0, V, (rows,), generator=g).to(dev)
    cu = torch.arange(0, rows + 1, 3, dtype=torch.int32, device=dev)
    lp = Ref(x, y, 1.0)
    ref = lp.logp.reshape(-1, 3).sum(1).float() + torch.randn(2 * pairs, generator=g)
    ref[2 * pairs - 2 + where] = value
    r = K().preference_loss_fwd(x, y, cu, ref.to(dev), beta=beta, kind=kind, label_smoothing=eps)
    gain = lp.logp.reshape(-1, 3).sum(1) - ref.double()
    each = [pair_formula(kind, eps, beta, float(a - b)) for a, b in gain.reshape(-1, 2)]
    off = float(lp.logp_tol.reshape(-1, 6).sum(1).max())      # of a pair's log-ratio
    steep = max(abs(s) for _, s in each if math.isfinite(s)) if any(math.isfinite(s) for _, s in each) else 0.0
    loss = sum(v for v, _ in each) / pairs
    check(r.loss, torch.tensor([loss]), steep * off + 2 * U * abs(loss) + 1e-12, "loss")
    coef = torch.tensor([[s] * 3 + [-s] * 3 for _, s in each]).double().reshape(-1) / pairs
    bend = {"sigmoid": beta ** 2 / 4, "hinge": 0.0, "ipo": 2.0}[kind]
    check(r.coef, coef, (bend * off + 2 * U * coef.abs() + 2.0 ** -50), "coef")
    check(r.rewards.reshape(-1), beta * gain, beta * off + 2 * U * beta * gain.abs(), "rewards")


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("pairs", [1, 3, 9])
@pytest.mark.parametrize("average", [False, True], ids=["sums", "means"])
@pytest.mark.parametrize("kind, eps", FORMS)
@pytest.mark.parametrize("where", [0, 1], ids=["chosen", "rejected"])
def test_a_label_whose_logit_is_minus_infinity(dev, where, kind, eps, average, pairs, dtype):
    """One token of the first pair is impossible (log-probability -inf): its answer's sum is -inf, the pair's loss 0 or infinite with the slope's limit, and gradients of
    finite slopes are finite."""
    rows, V, beta = 6 * pairs, 1031, 0.4
    g = torch.Generator().manual_seed(pairs)
    x, y = (torch.randn(rows, V, generator=g) * 2).to(dtype).to(dev), torch.randint(0, V, (rows,), generator=g).to(dev)
    bad = 3 * where + 1
    x[bad, y[bad]] = -math.inf
    cu = torch.arange(0, rows + 1, 3, dtype=torch.int32, device=dev)
    n = 3 if average else 1
    r = K().preference_loss_fwd(x, y, cu, beta=beta, kind=kind, label_smoothing=eps, average=average)
    lp = Ref(x, y, 1.0)
    check(r.logp, lp.logp, lp.logp_tol, "logp")
    sums = lp.logp.reshape(-1, 3).sum(1) / n
    tol = lp.sum_tol.reshape(-1, 3).sum(1) + 2 * U * torch.where(torch.isfinite(sums), sums.abs(), torch.zeros(()))
    check(r.seq_logps, sums, tol, "seq_logps")
    check(r.rewards.reshape(-1), beta * sums, beta * tol + 2 * U * beta * sums.abs(), "rewards")
    each = [pair_formula(kind, eps, beta, float(a - b)) for a, b in sums.reshape(-1, 2)]
    off = float(tol.reshape(-1, 2).sum(1).max())
    steep = max([abs(s) for _, s in each if math.isfinite(s)] or [0.0])
    loss = sum(v for v, _ in each) / pairs
    check(r.loss, torch.tensor([loss]), steep * off + 2 * U * abs(loss) + 1e-12, "loss")
    coef = torch.tensor([[s] * 3 + [-s] * 3 for _, s in each]).double().reshape(-1) / pairs / n
    bend = {"sigmoid": beta ** 2 / 4, "hinge": 0.0, "ipo": 2.0}[kind]
    check(r.coef, coef, bend * off + 2 * U * coef.abs() + 2.0 ** -50, "coef")
    if kind != "ipo":
        d = K().preference_loss_bwd(x, y, r, torch.full((1,), 8.0, device=dev), dlogits=torch.full_like(x, 7.0))
        lp.check_dlogits(d, r.coef.double() * 8.0, "dlogits")


@pytest.mark.parametrize("rows", [1, 63, 1000, 4095, 4096])
def test_short_batches_weigh_every_row_alike(dev, rows):
    """The one workgroup that finishes a short batch counts its tokens and sums its terms in the same shared memory: every call gives the same bits, those of the batch as one
    sequence, whose weights 1 / (1 N) are the same numbers."""
    V = 17
    g = torch.Generator().manual_seed(rows)
    x, y = torch.randn(rows, V, generator=g).to(dev), torch.randint(0, V, (rows,), generator=g)
    y[torch.rand(rows, generator=g) < 0.3] = IGNORE
    y[0] = 3
    y = y.to(dev)
    old, adv, ref = (torch.randn(rows, generator=g).to(dev) for _ in range(3))
    old, ref = old * 0.1 - 2.8, ref * 0.1 - 2.8
    want = K().policy_loss_fwd(x, y, old, adv, ref, kl_coef=0.1, cu_seqlens=torch.tensor([0, rows], dtype=torch.int32, device=dev))
    for _ in range(50):
        got = K().policy_loss_fwd(x, y, old, adv, ref, kl_coef=0.1)
        assert torch.equal(got.coef, want.coef) and torch.equal(got.stats, want.stats)


def policy_forms(dev, x, y, old, adv, ref, kl_coef):
    """The same rows, one sequence, through every form"""
    cu = torch.tensor([0, x.shape[0]], dtype=torch.int32, device=dev)
    one = torch.ones(1, device=dev)
    args = dict(ref_logps=ref, kl_coef=kl_coef)
    yield "small batch", K().policy_loss_fwd(x, y, old, adv, cu_seqlens=cu, **args)
    long = 4097 - x.shape[0]      # masked rows behind the sequence: past the rows that one workgroup finishes
    more = lambda t, v: torch.cat([t, torch.full((long, *t.shape[1:]), v, dtype=t.dtype, device=dev)])   # noqa: E731
    yield "long batch", K().policy_loss_fwd(more(x, 0.0), more(y, IGNORE), more(old, 0.0), more(adv, 0.0), ref_logps=more(ref, 0.0), kl_coef=kl_coef, cu_seqlens=cu)
    yield "one pass", K().policy_loss_fwd_bwd(x, y, old, adv, one, dlogits=torch.empty_like(x), cu_seqlens=cu, **args)[0]


def policy_rows(dev, seed):
    rows, V = 6, 300
    g = torch.Generator().manual_seed(seed)
    x, y = torch.randn(rows, V, generator=g).to(dev), torch.randint(0, V, (rows,), generator=g).to(dev)
    lp = Ref(x, y, 1.0).logp
    return x, y, (lp - 0.05).float().to(dev), torch.tensor([0.5, 1.0, -1.0, 0.75, -0.5, 2.0], device=dev), (lp + 0.2).float().to(dev)


@pytest.mark.parametrize("kl_coef", [0.0, 0.1])
def test_kl_of_an_impossible_label(dev, kl_coef):
    """exp(q) - q - 1 of q = inf is inf, reported and in the loss; without a weight on it the loss and every coefficient stay as they are."""
    x, y, old, adv, ref = policy_rows(dev, 1)
    for what, base in policy_forms(dev, x, y, old, adv, ref, kl_coef):
        assert bool(torch.isfinite(base.stats).all()), what
    x[1, y[1]] = -math.inf
    for what, r in policy_forms(dev, x, y, old, adv, ref, kl_coef):
        assert float(r.logp[1]) == -math.inf and float(r.stats[2]) == math.inf, (what, r.stats)
        if kl_coef:
            assert float(r.stats[0]) == math.inf and float(r.coef[1]) == -math.inf, (what, r.stats)
        else:
            assert bool(torch.isfinite(r.stats[[0, 1, 3]]).all()) and float(r.coef[1]) == 0.0, (what, r.stats)
        rest = [0, 2, 3, 4, 5]
        assert bool(torch.isfinite(r.coef[rest]).all()) and bool((r.coef[rest] != 0).all()), what


def test_ratio_past_fp32_without_an_advantage(dev):
    """r A = 0 where A = 0, whatever the ratio is: the row adds its KL term alone."""
    x, y, old, adv, ref = policy_rows(dev, 2)
    adv[3] = 0.0
    want = {what: r for what, r in policy_forms(dev, x, y, old, adv, ref, 0.1)}
    old[3] = -200.0
    for what, r in policy_forms(dev, x, y, old, adv, ref, 0.1):
        assert torch.equal(r.coef, want[what].coef) and torch.equal(r.stats, want[what].stats), (what, r.stats, want[what].stats)
    x[3, 5] = math.nan
    for what, r in policy_forms(dev, x, y, old, adv, ref, 0.1):
        assert bool(r.stats[0].isnan()) and bool(r.coef[3].isnan()), what
