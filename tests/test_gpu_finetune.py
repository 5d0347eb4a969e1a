"""The fine-tuning objectives (token log-probabilities, top-logits distillation, preference loss, policy loss) against
their definition in float64 on the CPU, the gradient by autograd there.

Tolerances, fixed by arithmetic.  eps = 2^-24.  An exponential exp((z - m) / tau) has a relative error of at most
|x| * 2 eps (two roundings of its exponent x, |x| <= 30 for what these tests draw) + 2 eps (the instruction), a sum
adds eps per addition of a lane's chain (at most 140 long: 64 pieces halved between two chains, the lanes' tree, the
waves) -> 210 eps on S; a log-probability inherits that and adds 4 roundings of its own value:
    TOL = 2^-24 * 240 = 1.5e-5 absolute, + 4 eps |lp|.
A gradient element c (t - p) is off by the type's rounding (finfo.eps / 2 of its value) and by c's and p's error:
cmag * 2 TOL * (p + t), cmag the sum of the absolute terms that c is made of (each is an exponential of lp or 1)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
TOL = 240 * EPS
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
OBJECTIVES = ["logprobs", "distill", "preference", "policy"]


@pytest.fixture(scope="module")
def pkg():
    import d3pm_amd
    return d3pm_amd


def make(seed, B, L, V, dtype, k=4, scale=2.0, mask=True, device="cuda"):
    """Inputs of all four objectives on the CPU (float32 and integers), logits rounded to their type."""
    g = torch.Generator().manual_seed(seed)
    d = {"logits": (torch.randn(B, L, V, generator=g) * scale).to(DTYPES[dtype]),
         "tokens": torch.randint(0, V, (B, L), generator=g)}
    lp = torch.log_softmax(d["logits"].double(), -1).gather(-1, d["tokens"][..., None])[..., 0]
    drift = 0.3 * torch.randn(B, L, generator=g)
    for edge in (math.log(0.8), math.log(1.25)):                    # no ratio within rounding of a clip's edge
        drift = torch.where((drift - edge).abs() < 1e-2, drift + 3e-2, drift)
    d["old"] = (lp - drift).float()
    d["ref"] = (lp + 0.3 * torch.randn(B, L, generator=g)).float()
    d["adv"] = torch.randn(B, L, generator=g)
    d["index"] = torch.randint(0, V, (B, L, k), generator=g)
    d["teacher"] = torch.randn(B, L, k, generator=g)
    d["up"] = torch.randn(B, L, generator=g)
    d["mask"] = None
    if mask:
        d["mask"] = torch.rand(B, L, generator=g) < 0.7
        d["mask"][0] = False                                         # a sequence that leaves nothing
    return d


def to_dev(d):
    return {k: (v.cuda() if torch.is_tensor(v) else v) for k, v in d.items()}


TAU = 1.7
CFG = dict(beta=0.3, smooth=0.1, lo=0.2, hi=0.25, kl=0.07)


def reference(name, d, average=False, scale=1.0):
    """(outputs, gradient, error bound of the gradient) in float64 from the definition."""
    z = d["logits"].double().requires_grad_(True)
    B, L, V = z.shape
    keep = torch.ones(B, L, dtype=torch.bool) if d["mask"] is None else d["mask"]
    rows = torch.where(keep[..., None], z, torch.zeros((), dtype=torch.float64))
    pick = lambda x: torch.where(keep, x.double(), torch.zeros((), dtype=torch.float64))
    w = keep.double()
    count = w.sum().clamp(min=1.0)
    tau = TAU if name in ("logprobs", "distill", "policy") else 1.0
    logp = torch.log_softmax(rows / tau, -1)
    target = torch.zeros(B, L, V, dtype=torch.float64)
    if name == "distill":
        t = d["teacher"].double()
        idx = d["index"]
        kept = (idx >= 0) & (t > -math.inf) & keep[..., None]
        tt = torch.where(kept, t / tau, torch.full((), -math.inf, dtype=torch.float64))
        anyk = kept.any(-1, keepdim=True)
        q = torch.where(anyk, torch.softmax(torch.where(anyk, tt, torch.zeros(())), -1), torch.zeros((), dtype=torch.float64))
        cls = idx.clamp(0, V - 1)
        term = torch.where(q > 0, q * (torch.log(q.clamp(min=1e-300)) - logp.gather(-1, cls)), torch.zeros((), dtype=torch.float64))
        per = tau * tau * term.sum(-1)
        loss = scale * (per * w).sum() / count
        loss.backward()
        target.scatter_add_(-1, cls, q)
        cmag = (scale * tau * w / count)[..., None]
        out = {"loss": loss, "per": per * w}
        # the terms q (log q - lp) and their number, per unit of which lp and log q are off by TOL
        out["loss_tol"] = abs(scale) * tau * tau * 3 * TOL + 8 * EPS * float((abs(scale) * (tau * tau * term.abs().sum(-1) * w).sum() / count).detach())
    else:
        lp = logp.gather(-1, d["tokens"].clamp(0, V - 1)[..., None])[..., 0]
        target.scatter_(-1, d["tokens"].clamp(0, V - 1)[..., None], 1.0)
        if name == "logprobs":
            (lp * w * pick(d["up"])).sum().backward()
            cmag = (pick(d["up"]).abs() * w / tau)[..., None]
            out = {"lp": lp * w}
        elif name == "preference":
            P = B // 2
            n = w.sum(1).clamp(min=1.0) if average else torch.ones(B, dtype=torch.float64)
            D = ((lp - pick(d["ref"])) * w).sum(1) / n
            m = CFG["beta"] * (D[:P] - D[P:])
            ls = torch.nn.functional.logsigmoid
            loss = scale * (-(1 - CFG["smooth"]) * ls(m) - CFG["smooth"] * ls(-m)).mean()
            loss.backward()
            cmag = (w * abs(scale) * CFG["beta"] / P / n[:, None])[..., None]
            # a row's lp is off by TOL, D by as much per counted row
            out = {"loss": loss, "rewards": CFG["beta"] * D}
            dtol = CFG["beta"] * (w.sum(1) / n).max() * TOL + EPS * (1 + float((CFG["beta"] * D).detach().abs().max()))
            out["rewards_tol"] = float(dtol)
            out["loss_tol"] = abs(scale) * (2 * float(dtol) + 4 * EPS * (float(loss.detach().abs()) / max(abs(scale), 1e-30) + 1))
        else:
            r = torch.exp(lp - pick(d["old"]))
            adv = d["adv"] if d["adv"].dim() == 2 else d["adv"][:, None].expand(B, L)
            A = pick(adv)
            x = pick(d["ref"]) - lp
            per = -torch.min(r * A, r.clamp(1 - CFG["lo"], 1 + CFG["hi"]) * A) + CFG["kl"] * (torch.exp(x) - x - 1)
            loss = scale * (per * w).sum() / count
            loss.backward()
            mag = (r * A).abs() + CFG["kl"] * (torch.exp(x) + 1)
            cmag = (abs(scale) * mag * w / count / tau).detach()[..., None]
            out = {"loss": loss, "lp": lp * w}
            out["loss_tol"] = abs(scale) * float(((mag * w).sum() / count).detach()) * 2 * TOL
        if "lp" in out:
            out["lp_tol"] = TOL + 4 * EPS * out["lp"].detach().abs()
    p = logp.detach().exp()
    bound = cmag * 2 * TOL * (p + target)
    return {k: (v.detach() if torch.is_tensor(v) else v) for k, v in out.items()}, z.grad, bound


def build(pkg, name, average=False):
    if name == "distill":
        return pkg.TopKDistillLoss(temperature=TAU)
    if name == "preference":
        return pkg.PreferenceLoss(beta=CFG["beta"], label_smoothing=CFG["smooth"], average=average)
    return pkg.PolicyLoss(clip_low=CFG["lo"], clip_high=CFG["hi"], kl_coeff=CFG["kl"], temperature=TAU)


def call(pkg, name, c, z, fn=None, scale=1.0):
    """One call on device inputs; (tensor to differentiate, outputs)."""
    if name == "logprobs":
        lp = pkg.token_logprobs(z, c["tokens"], mask=c["mask"], temperature=TAU)
        return lp, {"lp": lp}
    fn = fn or build(pkg, name)
    if name == "distill":
        loss = fn(z, c["teacher"], c["index"], mask=c["mask"], out_scale=scale)
        return loss, {"loss": loss, "per": fn.per_token}
    if name == "preference":
        loss = fn(z, c["tokens"], c["ref"], mask=c["mask"], out_scale=scale)
        return loss, {"loss": loss, "rewards": fn.rewards}
    loss = fn(z, c["tokens"], c["old"], c["adv"], c["ref"], mask=c["mask"], out_scale=scale)
    return loss, {"loss": loss, "lp": fn.logprobs}


def check_grad(got, want, bound, dtype, factor=1.0):
    fi = torch.finfo(dtype)
    got = got.detach().cpu().double()
    lim = (fi.eps / 2 + 4 * EPS) * want.abs() + (1 + fi.eps) * bound * abs(factor) + fi.smallest_normal * fi.eps / 2 + 1e-38
    bad = ~((got - want).abs() <= lim)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], lim[bad][:4])


def check(pkg, name, d, average=False, scale=1.0):
    out, grad, bound = reference(name, d, average, scale)
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    root, got = call(pkg, name, c, z, build(pkg, name, average) if name != "logprobs" else None, scale)
    for k in ("lp", "per", "rewards", "loss"):
        if k not in out:
            continue
        tol = out.get(k + "_tol", None)
        if k == "per":
            tol = TAU * TAU * 3 * TOL + 8 * EPS * (out["per"].abs() + 4 * TAU * TAU)
        diff = (got[k].detach().cpu().double() - out[k]).abs()
        assert got[k].dtype == torch.float32 and got[k].shape == out[k].shape
        assert bool((diff <= tol + EPS * out[k].abs()).all()), (name, k, float(diff.max()), tol if not torch.is_tensor(tol) else float(tol.max()))
    if name == "logprobs":
        up = c["up"] if c["mask"] is None else torch.where(c["mask"], c["up"], torch.zeros((), device="cuda"))
        root.backward(up)
    else:
        root.backward()
    assert z.grad.dtype == z.dtype and z.grad.shape == z.shape
    check_grad(z.grad, grad, bound, z.dtype)


# one or more sizes on each side of every shape of the row kernel, for 4 and 8 elements to a 16-byte piece
SIZES = [1, 2, 7, 8, 20, 22, 24, 31, 32, 33, 64, 65, 71, 100, 128, 255, 257, 513, 1000, 1025, 2049, 4099, 8200, 16390,
         20000, 32775]
WIDE = [32003, 65543, 100003, 131077]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("name", OBJECTIVES)
def test_against_definition(pkg, name, V, dtype):
    check(pkg, name, make(V, 4, 5, V, dtype, k=min(6, max(1, V))))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", WIDE)
@pytest.mark.parametrize("name", OBJECTIVES)
def test_wide_rows(pkg, name, V, dtype):
    check(pkg, name, make(V, 2, 2, V, dtype, k=64, mask=False))


@pytest.mark.parametrize("B,L", [(1, 1), (2, 1), (2, 4097), (300, 3), (6, 127)])
@pytest.mark.parametrize("name", OBJECTIVES)
def test_batch_shapes(pkg, name, B, L):
    if name == "preference" and B % 2:
        B += 1
    check(pkg, name, make(B + L, B, L, 22, "f32", mask=B > 2))
    check(pkg, name, make(B + L, B, L, 40, "bf16", mask=False))


@pytest.mark.parametrize("V", [24, 300, 5000, 70001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_rows_than_workgroups(pkg, V, dtype):
    """Row loops: more rows than one sweep of the grid (2048 workgroups of up to 32 rows, 8192 of one)."""
    rows = {24: 70000, 300: 9000, 5000: 8400, 70001: 8300}[V]
    g = torch.Generator(device="cuda").manual_seed(V)
    z = torch.randn(rows, V, generator=g, device="cuda").to(DTYPES[dtype])
    y = torch.randint(0, V, (rows,), generator=g, device="cuda")
    old = pkg.token_logprobs(z, y) - 0.05
    zz = z.detach().requires_grad_(True)
    fn = pkg.PolicyLoss()
    loss = fn(zz, y, old, torch.ones(rows, device="cuda"))
    loss.backward()
    assert abs(float(loss.detach()) + math.exp(0.05)) < 4 * TOL
    for sl in (slice(0, 3), slice(rows // 2, rows // 2 + 3), slice(rows - 3, rows)):
        lp64 = torch.log_softmax(z[sl].double(), -1)
        lp = lp64.gather(1, y[sl][:, None])
        assert bool(((fn.logprobs[sl].double() - lp[:, 0]).abs() <= TOL + 4 * EPS * lp[:, 0].abs()).all())
        p = lp64.exp()
        onehot = torch.zeros_like(p).scatter_(1, y[sl][:, None], 1.0)
        c = math.exp(0.05) / rows
        check_grad(zz.grad[sl], (c * (p - onehot)).cpu(), (c * 4 * TOL * (p + onehot)).cpu(), z.dtype)


@pytest.mark.parametrize("name", OBJECTIVES)
@pytest.mark.parametrize("V", [24, 3000, 70001])
def test_masked_places_hold_anything(pkg, name, V):
    d = make(3, 4, 6, V, "f32")
    clean = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in d.items()}
    off = ~d["mask"]
    junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min])
    d["logits"][off] = junk[torch.arange(int(off.sum()) * V) % 4].reshape(-1, V)
    d["tokens"][off] = -100
    for k in ("old", "ref", "adv", "up"):
        d[k][off] = math.nan
    d["teacher"][off] = math.nan
    d["index"][off] = 1 << 40
    c, cc = to_dev(d), to_dev(clean)
    za, zb = c["logits"].requires_grad_(True), cc["logits"].requires_grad_(True)
    (ra, oa), (rb, ob) = call(pkg, name, c, za), call(pkg, name, cc, zb)
    up = cc["up"] * cc["mask"] if name == "logprobs" else None
    ra.backward(up)
    rb.backward(up)
    for k in oa:
        assert torch.equal(oa[k], ob[k]), k
    assert torch.equal(za.grad, zb.grad)
    assert bool((za.grad[c["mask"].logical_not()] == 0).all())
    check(pkg, name, clean)


@pytest.mark.parametrize("name", OBJECTIVES)
def test_nothing_counted(pkg, name):
    d = make(5, 4, 6, 50, "f32")
    d["mask"][:] = False
    d["logits"][:] = math.nan
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    root, out = call(pkg, name, c, z)
    root.backward(torch.ones_like(root))
    want = math.log(2.0) if name == "preference" else 0.0
    assert abs(float(out["loss"] if "loss" in out else root.abs().max()) - want) <= 2 * EPS
    assert bool((z.grad == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [24, 600, 40000])
def test_extreme_logits(pkg, V, dtype):
    """Classes ruled out with -inf or with the type's lowest value, rows of nothing but the lowest, huge logits."""
    dt = DTYPES[dtype]
    low = torch.finfo(dt).min
    d = make(9, 4, 4, V, dtype, mask=False)
    z = d["logits"]
    z[0, :, ::2] = -math.inf
    z[1, :, 1::2] = low
    z[2, 0] = low
    z[2, 1] = torch.finfo(dt).max
    d["tokens"] = torch.where(torch.arange(4)[:, None] == 0, d["tokens"] // 2 * 2 + 1, d["tokens"] // 2 * 2).clamp(max=V - 1)
    d["tokens"][0] = 1
    lp64 = torch.log_softmax(z.double(), -1)
    lp = lp64.gather(-1, d["tokens"][..., None])[..., 0]
    zz = z.cuda().requires_grad_(True)
    got = pkg.token_logprobs(zz, d["tokens"].cuda())
    assert bool(((got.detach().cpu().double() - lp).abs() <= TOL + 4 * EPS * lp.abs()).all())
    got.sum().backward()
    p = lp64.exp()
    onehot = torch.zeros_like(p).scatter_(-1, d["tokens"][..., None], 1.0)
    check_grad(zz.grad, onehot - p, 2 * TOL * (p + onehot), dt)


@pytest.mark.parametrize("name", OBJECTIVES)
@pytest.mark.parametrize("V", [24, 600, 70001])
@pytest.mark.parametrize("bad", [math.nan, math.inf, "empty"])
def test_undefined_rows_are_nan_and_stay_in_their_row(pkg, name, V, bad):
    d = make(11, 2, 3, V, "f32", mask=False)
    d["tokens"][0, 1] = 0
    if bad == "empty":
        d["logits"][0, 1] = -math.inf
    else:
        d["logits"][0, 1, V // 2] = bad
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    root, out = call(pkg, name, c, z)
    root.backward(torch.ones_like(root))
    if "loss" in out:
        assert math.isnan(float(out["loss"]))
    if "lp" in out:
        assert bool(torch.isnan(out["lp"][0, 1])) and int(torch.isnan(out["lp"]).sum()) == 1
    assert bool(torch.isnan(z.grad[0, 1]).any())
    if name != "preference":                                 # there one NaN is in the pair's sum and so in its rows
        g = z.grad.clone()
        g[0, 1] = 0
        assert bool(torch.isfinite(g).all())


def test_impossible_token(pkg):
    """A token whose logit is -inf: log-probability -inf, ratio 0; the gradient of its log-probability is finite."""
    z = torch.randn(1, 3, 40, device="cuda")
    z[0, 1, 7] = -math.inf
    y = torch.tensor([[3, 7, 9]], device="cuda")
    zz = z.requires_grad_(True)
    lp = pkg.token_logprobs(zz, y)
    assert float(lp[0, 1]) == -math.inf and bool(torch.isfinite(lp[0, ::2]).all())
    lp.backward(torch.ones_like(lp))
    assert bool(torch.isfinite(zz.grad).all()) and float(zz.grad[0, 1, 7]) == 1.0


@pytest.mark.parametrize("name", OBJECTIVES)
@pytest.mark.parametrize("kind", ["shift", "transposed", "padded", "classes_apart", "expanded", "offset"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(pkg, name, kind, dtype):
    B, L, V = 4, 5, 37
    dt = DTYPES[dtype]
    d = make(21, B, L, V, dtype)
    if kind == "shift":
        base = torch.randn(B, L + 1, V).to(dt)
        view = lambda t: t[:, :-1]
    elif kind == "transposed":
        base = torch.randn(L, B, V).to(dt)
        view = lambda t: t.transpose(0, 1)
    elif kind == "padded":
        base = torch.randn(B, L, V + 3).to(dt)
        view = lambda t: t[..., 1:V + 1]
    elif kind == "classes_apart":
        base = torch.randn(B, V, L).to(dt)
        view = lambda t: t.transpose(1, 2)
    elif kind == "expanded":
        base = torch.randn(1, L, V).to(dt)
        view = lambda t: t.expand(B, L, V)
    else:
        base = torch.randn(B * L * V + 1).to(dt)
        view = lambda t: t[1:].view(B, L, V)
    d["logits"] = view(base).contiguous()
    c = to_dev(d)
    leaf = base.cuda().requires_grad_(True)
    z = view(leaf)
    z.retain_grad()
    root, out = call(pkg, name, c, z)
    if name == "logprobs":
        root.backward(c["up"] * c["mask"])
    else:
        root.backward()
    ref, grad, bound = reference(name, d)
    check_grad(z.grad, grad, bound, dt)
    b64 = base.double().requires_grad_(True)
    view(b64).backward(z.grad.cpu().double())
    assert leaf.grad.shape == base.shape
    if kind != "expanded":                                    # (expanded: torch sums the copies in its own order)
        assert torch.equal(leaf.grad.cpu().double(), b64.grad)


@pytest.mark.parametrize("name", OBJECTIVES)
def test_flat_and_image_shapes(pkg, name):
    d = make(31, 4, 6, 50, "f32")
    c = to_dev(d)
    a = c["logits"].clone().requires_grad_(True)
    b = c["logits"].clone().requires_grad_(True)
    r1, o1 = call(pkg, name, c, a)
    shape = (4, 2, 3)
    c2 = {k: (v.reshape(shape + v.shape[2:]) if torch.is_tensor(v) else v) for k, v in c.items()}
    r2, o2 = call(pkg, name, c2, b.reshape(4, 2, 3, 50))
    r1.backward(torch.ones_like(r1))
    r2.backward(torch.ones_like(r2))
    for k in o1:
        assert torch.equal(o1[k].reshape(-1), o2[k].reshape(-1))
    assert torch.equal(a.grad, b.grad)
    if name != "preference":
        c3 = {k: (v.reshape((24,) + v.shape[2:]) if torch.is_tensor(v) else v) for k, v in c.items()}
        r3, o3 = call(pkg, name, c3, c["logits"].reshape(24, 50).requires_grad_(True))
        for k in o1:
            assert torch.equal(o1[k].reshape(-1), o3[k].reshape(-1))


@pytest.mark.parametrize("name", OBJECTIVES)
def test_empty_batches(pkg, name):
    for B, L in ((0, 4), (2, 0)):
        if name == "preference" and B == 0:
            with pytest.raises(ValueError):
                pkg.PreferenceLoss()(torch.zeros(0, 4, 8, device="cuda"), torch.zeros(0, 4, dtype=torch.long, device="cuda"))
            continue
        c = to_dev({"logits": torch.zeros(B, L, 8), "tokens": torch.zeros(B, L, dtype=torch.long), "mask": None,
                    "old": torch.zeros(B, L), "ref": torch.zeros(B, L), "adv": torch.zeros(B, L),
                    "index": torch.zeros(B, L, 2, dtype=torch.long), "teacher": torch.zeros(B, L, 2)})
        z = c["logits"].requires_grad_(True)
        root, out = call(pkg, name, c, z)
        if name != "logprobs":
            assert abs(float(root) - (math.log(2.0) if name == "preference" else 0.0)) < 2 * EPS
        root.backward(torch.ones_like(root))
        assert z.grad.shape == z.shape


@pytest.mark.parametrize("V", [22, 300, 3000, 33000])
@pytest.mark.parametrize("k", [1, 5, 64, 65, 256])
@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_teacher_lists(pkg, V, k, index_dtype):
    """Duplicate classes, entries that are not there, entries of no mass, classes beyond the last, rows of neither."""
    d = make(V + k, 3, 5, V, "f32", k=k)
    d["index"] = (d["index"] % max(1, min(V, k // 2 + 1))).to(index_dtype)
    d["index"][1, 0] = -1
    d["teacher"][1, 1] = -math.inf
    if k > 4:
        d["index"][2, :, 1] = -7
        d["teacher"][2, :, 2] = -math.inf
        d["index"][2, :, 3] = V + 5
        d["teacher"][2, 2, :] = 80.0 * d["teacher"][2, 2, :]
    ref = {**d, "index": d["index"].long()}
    out, grad, bound = reference("distill", ref)
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    root, got = call(pkg, "distill", c, z)
    assert abs(float(root) - float(out["loss"])) <= out["loss_tol"] + 1e3 * EPS
    root.backward()
    check_grad(z.grad, grad, bound, z.dtype)
    assert float(got["per"][1, 0]) == 0.0 and float(got["per"][1, 1]) == 0.0


@pytest.mark.parametrize("tdtype", DTYPES)
def test_teacher_types(pkg, tdtype):
    d = make(41, 2, 7, 90, "bf16", k=8)
    d["teacher"] = d["teacher"].to(DTYPES[tdtype])
    check(pkg, "distill", d)


def test_advantage_per_sequence_and_average(pkg):
    d = make(43, 4, 9, 60, "f32")
    d["adv"] = d["adv"][:, 0].clone()
    check(pkg, "policy", d)
    check(pkg, "preference", make(44, 6, 9, 60, "f32"), average=True)
    d = make(45, 4, 9, 60, "f32")
    fn = pkg.PolicyLoss(clip_low=0.2, clip_high=0.25, kl_coeff=0.0, temperature=TAU)
    c = to_dev(d)
    old = CFG["kl"]
    try:
        CFG["kl"] = 0.0
        out, grad, bound = reference("policy", d)
    finally:
        CFG["kl"] = old
    z = c["logits"].requires_grad_(True)
    loss = fn(z, c["tokens"].int(), c["old"], c["adv"], mask=c["mask"])           # int32 tokens, no reference model
    assert abs(float(loss) - float(out["loss"])) <= out["loss_tol"]
    loss.backward()
    check_grad(z.grad, grad, bound, z.dtype)


def test_clip_holds_rows_exactly(pkg):
    """A row that the clip holds has a zero gradient, and the loss of one is -(1 +- clip) A."""
    z = torch.randn(1, 4, 30, device="cuda").requires_grad_(True)
    y = torch.zeros(1, 4, dtype=torch.long, device="cuda")
    lp = pkg.token_logprobs(z, y).detach()
    old = lp - torch.tensor([[0.5, -0.5, 0.5, -0.5]], device="cuda")
    adv = torch.tensor([[1.0, -1.0, -1.0, 1.0]], device="cuda")
    loss = pkg.PolicyLoss(clip_low=0.2, clip_high=0.3)(z, y, old, adv)
    want = (-1.3 + 0.8 + math.exp(0.5) - math.exp(-0.5)) / 4
    assert abs(float(loss) - want) <= 8 * TOL
    loss.backward()
    assert bool((z.grad[0, :2] == 0).all()) and bool((z.grad[0, 2:] != 0).any(-1).all())


@pytest.mark.parametrize("name", OBJECTIVES)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("V", [24, 2000])
def test_upstream_gradients(pkg, name, dtype, V):
    """An upstream gradient other than 1, a second backward, accumulation, out_scale."""
    d = make(51, 4, 6, V, dtype)
    out, grad, bound = reference(name, d)
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    root, _ = call(pkg, name, c, z)
    up = c["up"] * c["mask"] if name == "logprobs" else torch.ones((), device="cuda")
    factor = 512.0 if dtype == "f16" else 0.37
    root.backward(factor * up, retain_graph=True)
    first = z.grad.clone()
    check_grad(first, factor * grad, bound, z.dtype, factor)
    z.grad = None
    root.backward(factor * up, retain_graph=True)
    assert torch.equal(z.grad, first)                            # again, into a buffer of its own
    root.backward(up)
    one = torch.autograd.grad(call(pkg, name, c, z)[0], z, up)[0]
    assert torch.equal(z.grad, first + one)
    check_grad(one, grad, bound, z.dtype)
    if name != "logprobs":
        scaled, _ = call(pkg, name, c, z, scale=factor)
        assert abs(float(scaled) - factor * float(out["loss"])) <= factor * out["loss_tol"] + EPS * abs(factor * float(out["loss"]))
        g = torch.autograd.grad(scaled, z)[0]
        check_grad(g, factor * grad, bound, z.dtype, factor)


@pytest.mark.parametrize("name", OBJECTIVES)
def test_gradient_against_differences(pkg, name):
    """Central differences of the float32 loss itself: error h^2 / 6 of the third derivative (below 1e-2 h^2 at these
    sizes) and the loss' rounding over h."""
    d = make(61, 2, 3, 9, "f32", mask=False, scale=1.0)
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    weigh = (lambda r: (r * c["up"]).sum()) if name == "logprobs" else (lambda r: r)
    g = torch.autograd.grad(weigh(call(pkg, name, c, z)[0]), z)[0].flatten().cpu()
    h = 2.0 ** -5
    with torch.no_grad():
        for i in range(0, z.numel(), 5):
            step = torch.zeros(z.numel(), device="cuda")
            step[i] = h
            step = step.view_as(z)
            diff = (weigh(call(pkg, name, c, z + step)[0]) - weigh(call(pkg, name, c, z - step)[0])) / (2 * h)
            assert abs(float(diff) - float(g[i])) <= 10 * h * h + 4 * TOL / h, (i, float(diff), float(g[i]))


@pytest.mark.parametrize("name", OBJECTIVES)
@pytest.mark.parametrize("V", [24, 1000, 20000, 70001])
def test_repeatable_and_forward_only(pkg, name, V):
    d = make(71, 4, 40, V, "bf16")
    c = to_dev(d)
    runs = []
    for _ in range(2):
        z = c["logits"].clone().requires_grad_(True)
        root, out = call(pkg, name, c, z)
        root.backward(torch.ones_like(root))
        runs.append([v.detach() for v in out.values()] + [z.grad])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    with torch.no_grad():
        _, out = call(pkg, name, c, c["logits"].clone().requires_grad_(True))
    assert all(torch.equal(a, b) for a, b in zip(runs[0], out.values()))
    assert not any(v.requires_grad for v in out.values())


@pytest.mark.parametrize("V", [24, 3000, 70001])
def test_graph_capture(pkg, V):
    """All four with their backward in one graph, replayed on fresh data with eager work and synchronisation between
    the replays; a second graph captured beside it."""
    cs = [to_dev(make(81 + i, 4, 6, V, "bf16")) for i in range(3)]
    static = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in cs[0].items()}

    def everything(c, z):
        res = []
        for name in OBJECTIVES:
            z.grad = None
            root, out = call(pkg, name, c, z)
            root.backward(c["up"] * c["mask"] if name == "logprobs" else None)
            res += [v.detach() for v in out.values()] + [z.grad]
        z.grad = None
        return res

    graphs = []
    for _ in range(2):
        z = static["logits"].clone().requires_grad_(True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            everything(static, z)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = everything(static, z)
        graphs.append((g, z, res))
    for c in (cs[1], cs[2], cs[0], cs[1]):
        for k, v in c.items():
            if torch.is_tensor(v):
                static[k].copy_(v)
        for g, z, res in graphs:
            with torch.no_grad():
                z.copy_(c["logits"])
        for g, z, res in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = everything(c, c["logits"].clone().requires_grad_(True))
        for g, z, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_on_another_stream(pkg):
    d = to_dev(make(91, 4, 60, 5000, "bf16"))
    want = [torch.autograd.grad(call(pkg, n, d, z := d["logits"].clone().requires_grad_(True))[0], z,
                                d["up"] if n == "logprobs" else None)[0] for n in OBJECTIVES]
    streams = [torch.cuda.Stream() for _ in OBJECTIVES]
    got = []
    for n, s in zip(OBJECTIVES, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            z = d["logits"].clone().requires_grad_(True)
            got.append(torch.autograd.grad(call(pkg, n, d, z)[0], z, d["up"] if n == "logprobs" else None)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_beyond_32_bit_offsets(pkg):
    """More than 2^31 logits and 2^32 bytes: the last rows are the last rows."""
    V, N = 131072, 16500
    z = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    picks = [0, 8191, 8192, 16383, 16384, N - 1]
    for n in picks:
        z[n] = torch.randn(V, generator=g, device="cuda") * 2
    y = torch.randint(0, V, (N,), generator=g, device="cuda")
    zz = z.requires_grad_(True)
    idx = y[:, None]
    fn = pkg.TopKDistillLoss()
    for name in ("logprobs", "distill"):
        zz.grad = None
        if name == "logprobs":
            lp = pkg.token_logprobs(zz, y)
            lp.backward(torch.full_like(lp, -1.0))
            scale = 1.0
        else:
            loss = fn(zz, torch.zeros(N, 1, device="cuda"), idx, out_scale=float(N))
            loss.backward()
            lp, scale = -fn.per_token, 1.0
        for n in picks + [4000, 12000, N - 2]:
            lp64 = torch.log_softmax(z[n].detach().double(), -1)
            want = scale * lp64.exp()
            p = want.clone()
            want[y[n]] -= scale
            onehot = torch.zeros_like(p)
            onehot[y[n]] = 1.0
            assert abs(float(lp[n]) - float(lp64[y[n]])) <= TOL + 8 * EPS * abs(float(lp64[y[n]]))
            check_grad(zz.grad[n], want.cpu(), (2 * TOL * (p + onehot)).cpu(), torch.bfloat16)


def test_nothing_is_written_outside(pkg):
    """The C entry points on buffers inside larger ones: what lies before and behind stays as it was."""
    import ctypes as C
    from d3pm_amd._lib import lib, check as rc, ptr, stream_ptr, Logits
    for V in (22, 33, 300, 4099, 70001):
        for dtype, code, size in ((torch.float32, 0, 4), (torch.bfloat16, 2, 2)):
            B, L, pad = 2, 3, 64
            n = B * L * V
            z = torch.randn(n + 2 * pad, device="cuda").to(dtype)
            dz = torch.full((n + 2 * pad,), 7.0, device="cuda", dtype=dtype)
            y = torch.randint(0, V, (B, L), device="cuda")
            lp = torch.full((B * L + 2 * pad,), 7.0, device="cuda")
            st = torch.full((B * L * 4 + 2 * pad,), 7.0, device="cuda")
            up = torch.ones(B, L, device="cuda")
            desc = Logits(ptr(z) + pad * size, code, V, B, L, L * V, V)
            rc(lib.d3pm_token_logprobs(C.byref(desc), ptr(y), 8, None, 1.0, ptr(lp) + pad * 4, ptr(st) + pad * 4, stream_ptr()))
            rc(lib.d3pm_token_grad(C.byref(desc), ptr(y), 8, 1.0, ptr(st) + pad * 4, ptr(up), 1, 0, ptr(dz) + pad * size,
                                   stream_ptr()))
            first = dz.clone()
            dz.fill_(7.0)
            wsb = lib.d3pm_objective_workspace(B, L)
            ws = torch.full((wsb // 4 + 2 * pad,), 7.0, device="cuda")
            loss = torch.full((2 * pad,), 7.0, device="cuda")
            idx = y[..., None].contiguous()
            t = torch.zeros(B, L, 1, device="cuda")
            rc(lib.d3pm_topk_distill_loss(C.byref(desc), ptr(t), 0, ptr(idx), 8, 1, None, 1.0, float(-B * L), None, 0,
                                          ptr(loss) + pad * 4, None, ptr(dz) + pad * size, ptr(ws) + pad * 4, wsb,
                                          stream_ptr()))
            torch.cuda.synchronize()
            for buf, m in ((first, n), (dz, n), (lp, B * L), (st, 4 * B * L), (ws, wsb // 4), (loss, 1)):
                assert bool((buf[:pad] == 7.0).all()) and bool((buf[pad + m:] == 7.0).all())
            a, b = first[pad:pad + n].double(), dz[pad:pad + n].double()
            assert float((a - b).abs().max()) <= 4 * TOL + torch.finfo(dtype).eps


def test_refusals(pkg):
    dev = "cuda"
    z = torch.randn(4, 5, 30, device=dev, requires_grad=True)
    y = torch.zeros(4, 5, dtype=torch.long, device=dev)
    f = torch.zeros(4, 5, device=dev)
    ok = torch.ones(4, 5, dtype=torch.bool, device=dev)
    t, i = torch.zeros(4, 5, 3, device=dev), torch.zeros(4, 5, 3, dtype=torch.long, device=dev)
    with pytest.raises(RuntimeError):
        pkg.token_logprobs(z.cpu(), y)
    with pytest.raises(RuntimeError):
        pkg.token_logprobs(z, y.cpu())
    with pytest.raises(TypeError):
        pkg.token_logprobs(z, f)
    with pytest.raises(TypeError):
        pkg.token_logprobs(z.double(), y)
    with pytest.raises(TypeError):
        pkg.token_logprobs(z, y, mask=f)
    with pytest.raises(ValueError):
        pkg.token_logprobs(z, y[:, :4])
    with pytest.raises(ValueError):
        pkg.token_logprobs(z, y, mask=ok[:, :4])
    with pytest.raises(ValueError):
        pkg.token_logprobs(z, y, temperature=0.0)
    with pytest.raises(ValueError):
        pkg.token_logprobs(torch.zeros(4, 5, 0, device=dev), y)
    for bad in (dict(temperature=-1.0), dict(temperature=math.inf)):
        with pytest.raises(ValueError):
            pkg.TopKDistillLoss(**bad)
    fn = pkg.TopKDistillLoss()
    with pytest.raises(ValueError):
        fn(z, t[:, :4], i[:, :4])
    with pytest.raises(ValueError):
        fn(z, t, i[..., :2])
    with pytest.raises(ValueError):
        fn(z, t[..., :0], i[..., :0])
    with pytest.raises(ValueError):
        fn(z, torch.zeros(4, 5, 257, device=dev), torch.zeros(4, 5, 257, dtype=torch.long, device=dev))
    with pytest.raises(TypeError):
        fn(z, t.double(), i)
    with pytest.raises(ValueError):
        fn(z, t.clone().requires_grad_(True), i)
    with pytest.raises(ValueError):
        fn(z, t, i, out_scale=math.nan)
    for bad in (dict(label_smoothing=1.5), dict(beta=math.nan)):
        with pytest.raises(ValueError):
            pkg.PreferenceLoss(**bad)
    with pytest.raises(ValueError):
        pkg.PreferenceLoss()(z[:3], y[:3], f[:3])
    with pytest.raises(ValueError):
        pkg.PreferenceLoss()(z, y, f[:, :4])
    with pytest.raises(ValueError):
        pkg.PreferenceLoss()(z, y, f.clone().requires_grad_(True))
    for bad in (dict(clip_low=1.5), dict(clip_high=-0.1), dict(kl_coeff=math.inf), dict(temperature=0.0)):
        with pytest.raises(ValueError):
            pkg.PolicyLoss(**bad)
    with pytest.raises(ValueError):
        pkg.PolicyLoss(kl_coeff=0.1)(z, y, f, f)
    with pytest.raises(ValueError):
        pkg.PolicyLoss()(z, y, f, f[:3, 0].contiguous())
    with pytest.raises(ValueError):
        pkg.PolicyLoss()(z, y, f, f.clone().requires_grad_(True))
    # a buffer changed between forward and backward is noticed
    w = z * 1.0
    loss = pkg.PolicyLoss()(w, y, f, f)
    w.add_(1.0)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_together(pkg):
    """A small denoiser distilled from another's top logits, then tuned on pairs and on rewards with the distilled one as
    the reference model, each step's parameter gradients against float64 autograd of the same step."""
    V, Dm, B, L, k = 24, 16, 8, 13, 6
    torch.manual_seed(0)
    emb = torch.randn(V, Dm, device="cuda").requires_grad_(True)
    head = (torch.randn(Dm, V, device="cuda") / 4).requires_grad_(True)
    teacher = torch.randn(V, V, device="cuda")
    x = torch.randint(0, V, (B, L), device="cuda")
    y = torch.randint(0, V, (B, L), device="cuda")
    mask = torch.arange(L, device="cuda")[None] < torch.arange(L - B + 1, L + 1, device="cuda")[:, None]
    tl, ti = teacher[x].topk(k, -1)
    model = lambda e, h: e[x] @ h
    adv = torch.randn(B, device="cuda")
    opt = torch.optim.SGD([emb, head], lr=0.05)

    def step(loss_fn, loss64):
        opt.zero_grad(set_to_none=True)
        loss = loss_fn(model(emb, head))
        loss.backward()
        e, h = emb.detach().double().requires_grad_(True), head.detach().double().requires_grad_(True)
        want = loss64(torch.log_softmax(model(e, h), -1))
        want.backward()
        # float32 products of Dm = 16 terms each way on top of the losses' own error
        assert abs(float(loss) - float(want)) <= 1e-4 * (1 + abs(float(want)))
        for got, ref in ((emb.grad, e.grad), (head.grad, h.grad)):
            assert float((got.double() - ref).abs().max()) <= 1e-4 * float(ref.abs().max())
        opt.step()

    w = mask.double()
    distill, pref, policy = pkg.TopKDistillLoss(), pkg.PreferenceLoss(beta=0.5), pkg.PolicyLoss(kl_coeff=0.1)
    q = torch.softmax(tl.double(), -1)
    for _ in range(2):
        step(lambda z: distill(z, tl, ti, mask=mask),
             lambda lp: ((q * (q.log() - lp.gather(-1, ti))).sum(-1) * w).sum() / w.sum())
    with torch.no_grad():
        ref = pkg.token_logprobs(model(emb, head), y, mask=mask)
    assert bool((ref[~mask] == 0).all())
    for _ in range(2):
        def pair64(lp):
            D = ((lp.gather(-1, y[..., None])[..., 0] - ref.double()) * w).sum(1)
            return -torch.nn.functional.logsigmoid(0.5 * (D[:B // 2] - D[B // 2:])).mean()
        step(lambda z: pref(z, y, ref, mask=mask), pair64)
    with torch.no_grad():
        old = pkg.token_logprobs(model(emb, head), y, mask=mask)
    for _ in range(2):
        def policy64(lp):
            l = lp.gather(-1, y[..., None])[..., 0]
            r, xx, A = torch.exp(l - old.double()), ref.double() - l, adv.double()[:, None]
            per = -torch.min(r * A, r.clamp(0.8, 1.2) * A) + 0.1 * (torch.exp(xx) - xx - 1)
            return (per * w).sum() / w.sum()
        step(lambda z: policy(z, y, old, adv, ref, mask=mask), policy64)


@pytest.mark.parametrize("V,dtype", [(24, "f32"), (24, "bf16"), (60, "f32"), (100, "f16"), (250, "f32"), (255, "bf16"),
                                     (500, "f32"), (1000, "f32"), (1001, "bf16"), (2047, "f16")])
@pytest.mark.parametrize("B,L", [(2, 1), (4, 15), (6, 64), (2, 320), (4, 321)])
def test_pairs_of_any_size(pkg, V, dtype, B, L):
    """Preference pairs on both sides of what one workgroup takes."""
    check(pkg, "preference", make(V + L, B, L, V, dtype, mask=B > 2))
    check(pkg, "preference", make(V + L + 1, B, L, V, dtype, mask=False), average=True)


def test_pair_without_slope(pkg):
    """Smoothing 1/2 of an undecided pair: the slope is 0 and so is the gradient."""
    for V in (24, 5000):
        z = torch.randn(1, 7, V, device="cuda").repeat(2, 1, 1).requires_grad_(True)
        y = torch.randint(0, V, (1, 7), device="cuda").repeat(2, 1)
        loss = pkg.PreferenceLoss(beta=0.5, label_smoothing=0.5)(z, y)
        loss.backward()
        assert abs(float(loss.detach()) - math.log(2.0)) <= 2 * EPS and bool((z.grad == 0).all())


@pytest.mark.parametrize("name", ["distill", "policy"])
def test_masks_counted_by_the_row_launch_or_ahead_of_it(pkg, name):
    """16384 positions are the row launch's own to count; a mask that starts at an odd address, bytes of any value."""
    for N in (1, 15, 33, 16384, 16385, 20000):
        d = to_dev(make(N, 1, N + 1, 20, "f32", mask=True))
        d["mask"] = torch.rand(1, N + 1, device="cuda") < 0.5
        d["mask"][0, 1] = True
        cut = {k: (v[:, 1:].contiguous() if torch.is_tensor(v) else v) for k, v in d.items()}
        odd = torch.empty(N + 1, dtype=torch.uint8, device="cuda")
        odd[1:] = cut["mask"][0].to(torch.uint8) * 0x90
        cut["mask"] = odd[1:].view(torch.bool).view(1, N)
        keep = (odd[1:] != 0).view(1, N)
        per = {k: v for k, v in cut.items()}
        root, out = call(pkg, name, per, cut["logits"])
        terms = call(pkg, name, {**cut, "mask": None}, cut["logits"])[1]
        if name == "distill":
            want = (terms["per"].double() * keep).sum() / keep.sum()
            tol = N * EPS * float(terms["per"].abs().max()) / max(1, int(keep.sum())) + 4 * EPS * abs(float(want))
            assert abs(float(out["loss"]) - float(want)) <= tol
        assert torch.equal(out["per" if name == "distill" else "lp"], terms["per" if name == "distill" else "lp"] * keep)


def test_classes_that_share_a_place_of_the_table(pkg):
    """Classes a multiple of 16384 apart (the table's size), listed once and twice."""
    V, k = 60000, 12
    d = make(101, 2, 3, V, "bf16", k=k, mask=False)
    base = torch.randint(0, 5000, (2, 3, k // 3))
    d["index"] = torch.cat([base, base + 16384, base + 32768], -1)
    check(pkg, "distill", d)
    d["index"][0, :, 1] = d["index"][0, :, 0]
    check(pkg, "distill", d)


@pytest.mark.parametrize("name", OBJECTIVES)
def test_second_derivative_is_refused(pkg, name):
    d = make(103, 4, 3, 20, "f32", mask=False)
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    root, _ = call(pkg, name, c, z)
    g = torch.autograd.grad(root, z, torch.ones_like(root), create_graph=True)[0]
    assert bool(torch.isfinite(g).all())
    with pytest.raises(RuntimeError):
        g.sum().backward()
    root, _ = call(pkg, name, c, z)
    root.backward(torch.ones_like(root))
    with pytest.raises(RuntimeError):                            # the graph is gone
        root.backward(torch.ones_like(root))


@pytest.mark.parametrize("name", OBJECTIVES)
def test_modes_without_a_gradient(pkg, name):
    d = to_dev(make(105, 4, 3, 20, "f32"))
    want = call(pkg, name, d, d["logits"])[1]
    with torch.inference_mode():
        got = call(pkg, name, {k: (v.clone() if torch.is_tensor(v) else v) for k, v in d.items()}, d["logits"].clone())[1]
        assert all(torch.equal(want[k], got[k]) for k in want)
    for k in ("ref", "old", "adv"):                              # constants may require a gradient where none is recorded
        d[k].requires_grad_(True)
    with torch.no_grad():
        got = call(pkg, name, d, d["logits"].requires_grad_(True))[1]
    assert all(torch.equal(want[k], got[k]) for k in want)


def test_row_shapes_at_their_edges(pkg):
    """Widths around what each shape of the row kernel holds, for rows that start at every alignment."""
    for dtype, E in (("f32", 4), ("bf16", 8)):
        for pieces in (8, 16, 32, 64, 128, 256, 512, 1024, 2048, 4096):
            for V in (pieces * E - 1, pieces * E, pieces * E + E - 1, pieces * E + E):
                rows = 9
                g = torch.Generator(device="cuda").manual_seed(V)
                z = torch.randn(rows, V, generator=g, device="cuda").to(DTYPES[dtype]).requires_grad_(True)
                y = torch.randint(0, V, (rows,), generator=g, device="cuda")
                y[:3] = torch.tensor([0, V - 1, V // 2], device="cuda")
                lp64 = torch.log_softmax(z.detach().double(), -1)
                p, lp = lp64.exp(), lp64.gather(1, y[:, None])[:, 0]
                onehot = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
                c = torch.rand(rows, device="cuda") + 0.5
                got = pkg.token_logprobs(z, y)
                assert bool(((got.detach().double() - lp).abs() <= TOL + 4 * EPS * lp.abs()).all()), V
                got.backward(c)
                want, bound = c.double()[:, None] * (onehot - p), c.double()[:, None] * 2 * TOL * (p + onehot)
                check_grad(z.grad, want.cpu(), bound.cpu(), z.dtype)
                z.grad = None
                loss = pkg.PolicyLoss(clip_low=1.0, clip_high=1e6)(z, y, lp.float(), c)       # r = 1: the same gradient, over rows
                loss.backward()
                check_grad(z.grad, (-want / rows).cpu(), (2 * bound / rows).cpu(), z.dtype)


@pytest.mark.parametrize("name", OBJECTIVES)
def test_checkpointed_and_offloaded(pkg, name):
    """The head and its loss under a checkpoint (backward computes them again), or with saved tensors moved to the host:
    the gradients of the ordinary call, bit for bit."""
    from torch.utils.checkpoint import checkpoint
    d = to_dev(make(107, 4, 5, 40, "f32"))
    h = torch.randn(4 * 5, 16, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)
    w = torch.randn(16, 40, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_(True)

    def part(h, w):
        return call(pkg, name, d, (h @ w).view(4, 5, 40))[0]

    def grads(run):
        root = run()
        return torch.autograd.grad(root, (h, w), 1.5 * torch.ones_like(root))

    want = grads(lambda: part(h, w))
    again = grads(lambda: checkpoint(part, h, w, use_reentrant=False))

    def offloaded():
        with torch.autograd.graph.save_on_cpu():
            return part(h, w)

    for got in (again, grads(offloaded)):
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("L,V", [(4, 24), (700, 24), (3, 9000)])
def test_pair_whose_other_sequence_is_impossible(pkg, L, V):
    """-log sigmoid(inf) = 0 and its slope is 0: without label smoothing the infinite other term is not there."""
    d = to_dev(make(109, 2, L, V, "f32", mask=False))
    for side in (1, 0):
        z = d["logits"].clone()
        z[side, 1, int(d["tokens"][side, 1])] = -math.inf
        z.requires_grad_(True)
        fn = pkg.PreferenceLoss(beta=0.5, label_smoothing=1.0 - side)      # smoothing of 1: the other way round
        loss = fn(z, d["tokens"])
        loss.backward()
        assert float(loss) == 0.0 and int((z.grad != 0).sum()) == 0
        assert float(fn.rewards[side]) == -math.inf and math.isfinite(float(fn.rewards[1 - side]))


@pytest.mark.parametrize("name", OBJECTIVES)
@pytest.mark.parametrize("V", [24, 3000])
def test_backward_in_a_graph_of_its_own(pkg, name, V):
    """Forward and backward captured apart: the backward replayed again for other upstream gradients, with its result
    overwritten between, and for new logits after the forward's replay."""
    c = to_dev(make(111, 4, 6, V, "bf16"))
    z = c["logits"].clone().requires_grad_(True)

    def loss():
        return call(pkg, name, c, z)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        root = loss()
        u = torch.ones_like(root)
        torch.autograd.grad(root, z, u)
    torch.cuda.current_stream().wait_stream(side)
    del root
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        root = loss()
    with torch.cuda.graph(second, pool=first.pool()):
        grad, = torch.autograd.grad(root, z, u)
    for seed in (1, 2):
        with torch.no_grad():
            z.copy_(torch.randn(z.shape, generator=torch.Generator().manual_seed(seed)).cuda())
        first.replay()
        for factor in (2.0, 1.0, 1.0, -0.5):
            u.fill_(factor)
            grad.zero_()
            second.replay()
            torch.cuda.synchronize()
            fresh = call(pkg, name, c, z.detach().clone().requires_grad_(True))[0]
            zz = z.detach().clone().requires_grad_(True)
            want, = torch.autograd.grad(call(pkg, name, c, zz)[0], zz, u)
            assert torch.equal(grad, want) and torch.equal(root, fresh)
