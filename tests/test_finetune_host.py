"""The fine-tuning objectives' checks that need no GPU: the C entry points refuse bad arguments before any HIP call,
the modules refuse bad settings and CPU tensors."""
import ctypes as C
import math

import pytest
import torch


@pytest.fixture(scope="module")
def pkg():
    import d3pm_amd
    return d3pm_amd


def desc(L, data=1, dtype=0, V=8, B=2, length=3, sb=24, sl=8):
    return L.Logits(data, dtype, V, B, length, sb, sl)


def test_struct_layout(pkg):
    assert C.sizeof(pkg._lib.Logits) == 8 + 2 * 4 + 4 * 8


@pytest.mark.parametrize("bad", [dict(data=None), dict(dtype=3), dict(dtype=-1), dict(V=0), dict(V=(1 << 27) + 1), dict(B=-1),
                                 dict(length=-1), dict(B=1 << 20, length=1 << 20), dict(sb=-1), dict(sl=-8)])
def test_bad_logits(pkg, bad):
    L = pkg._lib
    z = desc(L, **bad)
    ws = L.lib.d3pm_objective_workspace(2, 3)
    for rc in (L.lib.d3pm_token_logprobs(C.byref(z), 1, 8, None, 1.0, 1, 16, None),
               L.lib.d3pm_token_grad(C.byref(z), 1, 8, 1.0, 16, 1, 1, 0, 1, None),
               L.lib.d3pm_topk_distill_loss(C.byref(z), 1, 0, 1, 8, 2, None, 1.0, 1.0, None, 0, 1, 1, 1, 8, ws, None),
               L.lib.d3pm_policy_loss(C.byref(z), 1, 8, 1, 1, 0, None, None, 1.0, 0.2, 0.2, 0.0, 1.0, None, 0, 1, 1, 1, 8, ws, None),
               L.lib.d3pm_preference_loss(C.byref(z), 1, 8, None, None, 0.1, 0.0, 0, 1.0, 1, 1, 16, 1, 8, ws, None)):
        assert rc == L.EINVAL
        with pytest.raises(ValueError):
            L.check(rc)


def test_bad_arguments(pkg):
    L = pkg._lib
    z = C.byref(desc(L))
    ws = L.lib.d3pm_objective_workspace(2, 3)
    lp = lambda tokens=1, tb=8, t=1.0, out=1: L.lib.d3pm_token_logprobs(z, tokens, tb, None, t, out, None, None)
    for rc in (lp(tokens=None), lp(tb=2), lp(t=0.0), lp(t=-1.0), lp(t=math.nan), lp(t=1e7), lp(out=None),
               L.lib.d3pm_token_logprobs(None, 1, 8, None, 1.0, 1, None, None)):
        assert rc == L.EINVAL
    grad = lambda tokens=1, st=16, u=1, per=1, only=0, out=1: L.lib.d3pm_token_grad(z, tokens, 8, 1.0, st, u, per, only, out, None)
    for rc in (grad(tokens=None), grad(st=None), grad(out=None), grad(per=1, only=1), grad(u=None, per=0, only=1)):
        assert rc == L.EINVAL
    dis = lambda tl=1, td=0, ti=1, ib=8, k=2, t=1.0, s=1.0, w=8, wb=ws: L.lib.d3pm_topk_distill_loss(
        z, tl, td, ti, ib, k, None, t, s, None, 0, 1, None, None, w, wb, None)
    for rc in (dis(tl=None), dis(td=7), dis(ti=None), dis(ib=1), dis(k=0), dis(k=257), dis(t=0.0), dis(s=math.inf), dis(w=None),
               dis(wb=ws - 1)):
        assert rc == L.EINVAL
    pol = lambda y=1, old=1, adv=1, ref=None, cl=0.2, ch=0.2, kl=0.0, s=1.0, wb=ws: L.lib.d3pm_policy_loss(
        z, y, 8, old, adv, 0, ref, None, 1.0, cl, ch, kl, s, None, 0, 1, 1, 1, 8, wb, None)
    for rc in (pol(y=None), pol(old=None), pol(adv=None), pol(kl=0.1), pol(cl=1.5), pol(cl=-0.1), pol(ch=-0.1), pol(kl=math.nan),
               pol(s=math.nan), pol(wb=0)):
        assert rc == L.EINVAL
    pre = lambda B=2, b=0.1, e=0.0, s=1.0, loss=1, rew=1, st=16, wb=ws: L.lib.d3pm_preference_loss(
        C.byref(desc(L, B=B)), 1, 8, None, None, b, e, 0, s, loss, rew, st, 1, 8, wb, None)
    for rc in (pre(B=0), pre(B=3), pre(b=math.nan), pre(e=1.5), pre(e=-0.1), pre(s=math.inf), pre(loss=None), pre(rew=None),
               pre(st=None), pre(wb=8)):
        assert rc == L.EINVAL


def test_modules_refuse(pkg):
    for make in (lambda: pkg.TopKDistillLoss(temperature=0.0), lambda: pkg.TopKDistillLoss(temperature=math.nan),
                 lambda: pkg.PreferenceLoss(label_smoothing=-0.5), lambda: pkg.PreferenceLoss(beta=math.inf),
                 lambda: pkg.PolicyLoss(clip_low=2.0), lambda: pkg.PolicyLoss(clip_high=math.nan),
                 lambda: pkg.PolicyLoss(kl_coeff=math.nan), lambda: pkg.PolicyLoss(temperature=1e9)):
        with pytest.raises(ValueError):
            make()
    z, y, f = torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3)
    for use in (lambda: pkg.token_logprobs(z, y), lambda: pkg.PreferenceLoss()(z, y), lambda: pkg.PolicyLoss()(z, y, f, f),
                lambda: pkg.TopKDistillLoss()(z, z, y[..., None])):
        with pytest.raises(RuntimeError):          # no CPU path
            use()
