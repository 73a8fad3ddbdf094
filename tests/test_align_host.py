"""Refusals of the preference / policy losses and of the gradient-list norm, without a GPU: the wrappers' checks on host tensors, the C entries' on addresses that
are never dereferenced (every call here is refused before its first launch)."""
import ctypes

import pytest
import torch

FAKE = ctypes.c_void_p(4096)


@pytest.fixture(scope="module")
def K():
    from internevo_amd.build import build

    build(verbose=False)
    from internevo_amd import kernels

    return kernels


@pytest.fixture(scope="module")
def lib(K):
    return K._L()


def _logits(rows=4, V=16, dtype=torch.bfloat16):
    return torch.zeros(rows, V, dtype=dtype), torch.zeros(rows, dtype=torch.int64)


def test_host_tensors_are_refused(K):
    x, y = _logits()
    with pytest.raises(ValueError, match="no CPU fallback"):
        K.token_logprobs(x, y)
    with pytest.raises(ValueError, match="no CPU fallback"):
        K.preference_loss_fwd(x, y, torch.tensor([0, 2, 4], dtype=torch.int32))
    with pytest.raises(ValueError, match="no CPU fallback"):
        K.policy_loss_fwd(x, y, torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="no CPU fallback"):
        K.grad_norm([torch.zeros(3)])
    with pytest.raises(ValueError, match="no CPU fallback"):
        K.clip_grad_norm_([torch.zeros(3)], 1.0)


@pytest.mark.parametrize("change, match", [
    (dict(labels=torch.zeros(3, dtype=torch.int64)), "labels"),
    (dict(labels=torch.zeros(4, dtype=torch.int32)), "labels"),
    (dict(labels=torch.zeros(8, dtype=torch.int64)[::2]), "labels"),
    (dict(logits=torch.zeros(4, 16, dtype=torch.float16)), "dtype"),
    (dict(logits=torch.zeros(16, 4).t()), "unit column stride"),
    (dict(logits=torch.zeros(4, 4, 4)), "2-D"),
    (dict(logits=torch.zeros(4, 0)), "no columns"),
    (dict(temperature=0.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"),
])
def test_logit_arguments(K, change, match):
    x, y = _logits()
    kw = dict(logits=x, labels=y)
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        K.token_logprobs(**kw)
    with pytest.raises(ValueError, match=match):
        K.preference_loss_fwd(cu_seqlens=torch.tensor([0, 2, 4], dtype=torch.int32), **kw)
    with pytest.raises(ValueError, match=match):
        K.policy_loss_fwd(old_logps=torch.zeros(4), advantages=torch.zeros(4), **kw)


@pytest.mark.parametrize("change, match", [
    (dict(cu_seqlens=torch.tensor([0, 2], dtype=torch.int32)), "pairs"),
    (dict(cu_seqlens=torch.tensor([0, 2, 3, 4], dtype=torch.int32)), "pairs"),
    (dict(cu_seqlens=torch.tensor([0, 2, 4])), "cu_seqlens"),
    (dict(ref_logps=torch.zeros(3)), "ref_logps"),
    (dict(ref_logps=torch.zeros(2, dtype=torch.float64)), "ref_logps"),
    (dict(kind="logistic"), "kind"),
])
def test_preference_arguments(K, change, match):
    x, y = _logits()
    kw = dict(cu_seqlens=torch.tensor([0, 2, 4], dtype=torch.int32))
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        K.preference_loss_fwd(x, y, **kw)


@pytest.mark.parametrize("change, match", [
    (dict(old_logps=torch.zeros(3)), "old_logps"),
    (dict(advantages=torch.zeros(4, dtype=torch.bfloat16)), "advantages"),
    (dict(kl_coef=0.1), "ref_logps"),
    (dict(ref_logps=torch.zeros(5)), "ref_logps"),
    (dict(cu_seqlens=torch.tensor([0], dtype=torch.int32)), "cu_seqlens"),
    (dict(cu_seqlens=torch.tensor([0, 4])), "cu_seqlens"),
])
def test_policy_arguments(K, change, match):
    x, y = _logits()
    kw = dict(old_logps=torch.zeros(4), advantages=torch.zeros(4))
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        K.policy_loss_fwd(x, y, **kw)
    with pytest.raises(ValueError, match=match):
        K.policy_loss_fwd_bwd(x, y, dloss=torch.ones(1), **kw)


def test_backward_arguments(K):
    x, y = _logits()
    ok = torch.zeros(4)
    with pytest.raises(ValueError, match="lse"):
        K.token_logprobs_bwd(x, y, torch.zeros(3), ok)
    with pytest.raises(ValueError, match="dlogp"):
        K.token_logprobs_bwd(x, y, ok, torch.zeros(4, dtype=torch.float64))
    with pytest.raises(ValueError, match="dloss"):
        K.token_logprobs_bwd(x, y, ok, ok, torch.zeros(2))
    with pytest.raises(ValueError, match="dlogits"):
        K.token_logprobs_bwd(x, y, ok, ok, dlogits=torch.zeros(4, 16))
    with pytest.raises(ValueError, match="dlogits"):
        K.token_logprobs_bwd(x, y, ok, ok, dlogits=torch.zeros(4, 15, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="dloss"):
        K.policy_loss_fwd_bwd(x, y, ok, ok, None)


def test_gradient_list_arguments(K):
    t = torch.zeros(8)
    for f in (K.grad_norm, lambda ts: K.clip_grad_norm_(ts, 1.0)):
        with pytest.raises(ValueError, match="empty list"):
            f([])
        with pytest.raises(ValueError, match="contiguous"):
            f([t[::2]])
        with pytest.raises(ValueError, match="dtype"):
            f([t.half()])
    with pytest.raises(ValueError, match="negative"):
        K.clip_grad_norm_([t], -1.0)
    with pytest.raises(ValueError, match="negative"):
        K.clip_grad_norm_([t], float("nan"))
    with pytest.raises(ValueError, match="same length"):
        K.clip_grad_norm_([t], 1.0, out=[torch.zeros(7)])
    with pytest.raises(ValueError, match="same length"):
        K.clip_grad_norm_([t], 1.0, out=[])


def _refused(lib, rc, word):
    assert rc == -1, rc
    assert word in lib.ie_last_error().decode(), lib.ie_last_error()


def test_c_entries_refuse_bad_calls(lib):
    f = FAKE
    _refused(lib, lib.ie_logprob_fwd(None, 0, 8, f, f, f, 4, 8, -100, 1.0, None), "null")
    _refused(lib, lib.ie_logprob_fwd(f, 2, 8, f, f, f, 4, 8, -100, 1.0, None), "dtype")
    _refused(lib, lib.ie_logprob_fwd(f, 0, 7, f, f, f, 4, 8, -100, 1.0, None), "shape")
    _refused(lib, lib.ie_logprob_fwd(f, 0, 1 << 40, f, f, f, 4, 1 << 31, -100, 1.0, None), "shape")
    _refused(lib, lib.ie_logprob_fwd(f, 0, 8, f, f, f, 1 << 31, 8, -100, 1.0, None), "shape")
    _refused(lib, lib.ie_logprob_fwd(f, 0, 8, f, f, f, (1 << 26) - 3, 8, -100, 1.0, None), "shape")   # (one workgroup of four rows more than a launch may have)
    for t in (0.0, -1.0, float("nan"), float("inf")):
        _refused(lib, lib.ie_logprob_fwd(f, 0, 8, f, f, f, 4, 8, -100, t, None), "temperature")
    # a gradient that overlaps the logits without being them
    for off, ldd in ((2, 8), (0, 9), (62, 8)):
        _refused(lib, lib.ie_logprob_bwd(f, 0, 8, ctypes.c_void_p(4096 + off), ldd, f, f, f, None, 1.0, 4, 8, -100, 1.0, None), "apart")
    _refused(lib, lib.ie_logprob_bwd(f, 0, 8, ctypes.c_void_p(8192), 7, f, f, f, None, 1.0, 4, 8, -100, 1.0, None), "apart")

    def pref(kind=0, beta=0.1, smooth=0.0, margin=0.0, pairs=1, ws=f):
        return lib.ie_preference_loss_fwd(f, 0, 8, f, f, None, kind, beta, smooth, margin, 0, f, f, f, f, f, f, ws, 4, 8, pairs, -100, 1.0, None)

    _refused(lib, pref(ws=None), "null")
    _refused(lib, pref(ws=ctypes.c_void_p(4100)), "aligned")
    _refused(lib, pref(pairs=0), "pair")
    _refused(lib, pref(kind=3), "kind")
    for b in (0.0, -0.1, float("nan"), float("inf")):
        _refused(lib, pref(beta=b), "beta")
    for s in (-0.1, 0.6, float("nan")):
        _refused(lib, pref(smooth=s), "smoothing")
    _refused(lib, pref(kind=1, smooth=0.1), "smoothing")
    _refused(lib, pref(kind=2, margin=0.1), "margin")
    _refused(lib, pref(margin=float("nan")), "margin")

    def policy(d=None, dloss=None, ref=None, cu=None, seqs=0, low=0.2, high=0.2, kl=0.0):
        return lib.ie_policy_loss(f, 0, 8, d, 8, f, f, f, ref, cu, seqs, low, high, kl, dloss, 1.0, f, f, f, f, f, 4, 8, -100, 1.0, None)

    _refused(lib, policy(d=ctypes.c_void_p(8192)), "dloss")
    _refused(lib, policy(dloss=f), "dloss")
    _refused(lib, policy(d=ctypes.c_void_p(4098), dloss=f), "apart")
    _refused(lib, policy(cu=f), "sequences")
    _refused(lib, policy(seqs=2), "sequences")
    _refused(lib, policy(kl=0.1), "KL")
    _refused(lib, policy(ref=f, kl=-0.1), "KL")
    for low, high in ((-0.1, 0.2), (1.1, 0.2), (0.2, -0.1), (float("nan"), 0.2)):
        _refused(lib, policy(low=low, high=high), "clip")


def _arrays(ptrs, numels, dtypes):
    n = len(ptrs)
    return (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numels), (ctypes.c_int * n)(*dtypes)


def test_gradient_list_entries_refuse_bad_calls(lib):
    def norm(ptrs, numels, dtypes, n=None, ws=FAKE):
        return lib.ie_grad_norm(*_arrays(ptrs, numels, dtypes), len(ptrs) if n is None else n, ws, FAKE, None)

    _refused(lib, norm([4096], [8], [0], ws=None), "null")
    _refused(lib, norm([4096], [8], [0], ws=ctypes.c_void_p(4100)), "aligned")
    _refused(lib, norm([4096], [-1], [0]), "list")
    _refused(lib, norm([4096] * 1025, [1 << 38] * 1025, [0] * 1025), "list")
    _refused(lib, norm([None], [8], [0]), "list")
    _refused(lib, norm([4096], [8], [2]), "list")
    _refused(lib, norm([4096], [8], [0], n=-1), "list")
    _refused(lib, lib.ie_grad_norm(None, None, None, 1, FAKE, FAKE, None), "list")

    def clip(ptrs, numels, dtypes, outs=None, odt=None, max_norm=1.0, norm=FAKE):
        n = len(ptrs)
        o = (ctypes.c_void_p * n)(*outs) if outs else None
        d = (ctypes.c_int * n)(*odt) if odt else None
        return lib.ie_grad_clip(*_arrays(ptrs, numels, dtypes), o, d, n, max_norm, FAKE, norm, None)

    _refused(lib, clip([4096], [8], [0], norm=None), "null")
    _refused(lib, clip([4096], [8], [0], max_norm=-1.0), "max_norm")
    _refused(lib, clip([4096], [8], [0], max_norm=float("nan")), "max_norm")
    _refused(lib, clip([4096, 4096], [8, 8], [0, 0]), "overlap")                       # the same tensor twice
    _refused(lib, clip([4096, 8192, 4108], [8, 8, 8], [0, 0, 0]), "overlap")           # two bytes into the first's end
    _refused(lib, clip([4096, 8192], [8, 8], [1, 1], outs=[8192, 12288], odt=[1, 1]), "overlap")   # one's output is the other's input
    _refused(lib, clip([4096], [8], [0], outs=[4096], odt=[1]), "overlap")             # fp32 over its own bf16
    _refused(lib, clip([4096, 8192], [8, 8], [1, 1], outs=[12288, 12304], odt=[1, 1]), "overlap")  # two outputs
    _refused(lib, clip([4096], [8], [0], outs=[8192]), "null")
    _refused(lib, clip([4096], [8], [0], outs=[8192], odt=[5]), "output")


def test_workspace_sizes(lib):
    assert lib.ie_preference_loss_workspace(10, 3) == 64
    assert lib.ie_policy_loss_workspace(10, 0) == 41 * 4 and lib.ie_policy_loss_workspace(10, 4) == 44 * 4
    # one launch at least, and one more for every full set of tensors
    assert lib.ie_grad_norm_workspace(0) > 0 and lib.ie_grad_norm_workspace(1000) > lib.ie_grad_norm_workspace(1)
