"""The fine-tuning objectives where a call is allowed but unusual: upstream gradients that are no numbers at places that
are not counted, derivatives that these losses do not have, far log-probabilities, long sums and means, rows that start
anywhere, dispatch modes and transforms.  Inputs, definitions and tolerances as in test_gpu_finetune.py unless stated."""
import math

import pytest
import torch

from test_gpu_finetune import DTYPES, EPS, OBJECTIVES, call, check, check_grad, make, reference, to_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    import d3pm_amd
    return d3pm_amd


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [24, 300, 3000, 70001, 140001])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_upstream_of_a_place_that_is_not_counted(pkg, V, dtype, bad):
    """exp(lp - old) with a NaN at a pad, or a mean over no position, sends such an upstream gradient: the gradient there
    is 0 all the same, and the row is not looked at."""
    d = make(V, 4, 6, V, dtype)
    off = ~d["mask"]
    d["logits"][off] = math.nan
    d["tokens"][off] = -100
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    want, = torch.autograd.grad(pkg.token_logprobs(z, c["tokens"], mask=c["mask"]), z, c["up"] * c["mask"])
    got, = torch.autograd.grad(pkg.token_logprobs(z, c["tokens"], mask=c["mask"]), z,
                               torch.where(c["mask"], c["up"], torch.full((), bad, device="cuda")))
    assert bool((got[off.cuda()] == 0).all())
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", ["distill", "preference", "policy"])
@pytest.mark.parametrize("L,V", [(6, 24), (700, 24), (6, 3000), (6, 70001)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_loss_scale_that_is_no_number(pkg, name, L, V, bad):
    """An upstream gradient of inf or NaN is for the counted positions only."""
    d = make(V + L, 4, L, V, "f32")
    off = ~d["mask"]
    d["logits"][off] = math.nan
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    g, = torch.autograd.grad(call(pkg, name, c, z)[0], z, torch.full((), bad, device="cuda"))
    assert bool((g[off.cuda()] == 0).all())
    if math.isnan(bad):
        assert bool(torch.isnan(g[c["mask"]]).all())


@pytest.mark.parametrize("V,dtype", [(1001, "bf16"), (2001, "bf16"), (4099, "f16"), (9001, "bf16"), (16411, "bf16"),
                                     (32003, "bf16"), (65001, "f16"), (100003, "bf16"), (131077, "bf16"), (2051, "f32"),
                                     (33001, "f32"), (65543, "f32")])
@pytest.mark.parametrize("kind", ["shift", "padded"])
@pytest.mark.parametrize("name", OBJECTIVES)
def test_gradient_rows_that_start_elsewhere(pkg, name, kind, V, dtype):
    """Odd widths out of strided rows: a row of the gradient lies at another alignment than the logits' row."""
    B, L = 4, 3
    dt = DTYPES[dtype]
    d = make(V, B, L, V, dtype, k=16)
    base = torch.randn((B, L + 1, V) if kind == "shift" else (B, L, V + 2), generator=torch.Generator().manual_seed(V)).to(dt)
    view = (lambda t: t[:, :-1]) if kind == "shift" else (lambda t: t[..., 1:V + 1])
    d["logits"] = view(base).contiguous()
    out, grad, bound = reference(name, d)
    c = to_dev(d)
    z = view(base.cuda()).requires_grad_(True)
    assert not z.is_contiguous()
    root, got = call(pkg, name, c, z)
    g, = torch.autograd.grad(root, z, c["up"] * c["mask"] if name == "logprobs" else None)
    assert g.is_contiguous()
    check_grad(g, grad, bound, dt)
    # (not bit for bit a contiguous call's: the pieces begin elsewhere in the row, so its terms are added in another order)
    for k in ("lp", "rewards", "loss"):
        if k in out:
            diff = (got[k].detach().cpu().double() - out[k]).abs()
            assert bool((diff <= out[k + "_tol"] + EPS * out[k].abs()).all())


@pytest.mark.parametrize("name", OBJECTIVES)
def test_the_gradient_of_a_gradient_is_an_error(pkg, name):
    """Also where it is one term of a sum that has a gradient: not a silent zero."""
    c = to_dev(make(103, 4, 3, 20, "f32", mask=False))
    z = c["logits"].requires_grad_(True)

    def gradient():
        root, _ = call(pkg, name, c, z)
        return torch.autograd.grad(root, z, torch.ones_like(root), create_graph=True)[0]

    g = gradient()
    assert g.requires_grad and bool(torch.isfinite(g).all())
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()
    g = gradient()
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        (z.square().sum() + g.square().sum()).backward()
    plain, = torch.autograd.grad(call(pkg, name, c, z)[0], z, None if name != "logprobs" else torch.ones(4, 3, device="cuda"))
    assert torch.equal(plain, gradient().detach())


@pytest.mark.parametrize("name", OBJECTIVES)
def test_forward_mode_is_refused(pkg, name):
    """No tangent comes out, so none is taken: of the logits, and of the inputs that are constants."""
    import torch.autograd.forward_ad as fwd
    c = to_dev(make(113, 4, 3, 20, "f32", mask=False))
    floats = {"logprobs": [], "distill": ["teacher"], "preference": ["ref"], "policy": ["old", "ref", "adv"]}[name]
    for key in ["logits"] + floats:
        with fwd.dual_level():
            d = {**c, key: fwd.make_dual(c[key], torch.ones_like(c[key]))}
            with pytest.raises(NotImplementedError, match="forward"):
                call(pkg, name, d, d["logits"])
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
                call(pkg, name, d, d["logits"])
            call(pkg, name, c, c["logits"])                       # an ordinary call inside the level


@pytest.mark.parametrize("V,dtype", [(1 << 18, "f32"), ((1 << 20) + 5, "bf16"), ((1 << 22) + 3, "f32"), ((1 << 22) + 3, "bf16")])
def test_sums_of_long_rows(pkg, V, dtype):
    """Rows of equal classes behind M higher ones, which every lane meets first: every later term of the sum is the same
    number, so what the additions lose adds up (4096 float32 additions of exp(-87/128): 1010 eps).  S = M + (V - M) e,
    e = exp(-87/128): the exponent's rounding and the instruction's ulp make 1.5 + 2 eps of e, a lane's float32 additions
    (16 of them at most, the rest in 64 bits) 16 eps: 20 eps of log S, and |lp| eps for the output's rounding (the type's)."""
    M = 8208
    z = torch.full((2, 3, V), -87.0 / 128.0, dtype=DTYPES[dtype])     # (a number of all types)
    z[..., :M] = 0.0
    y = torch.tensor([[0, M // 2, M - 1], [1, 7, M - 2]])
    lp = -math.log(M + (V - M) * math.exp(-87.0 / 128.0))
    z, y = z.cuda(), y.cuda()
    assert float((pkg.token_logprobs(z, y).double() - lp).abs().max()) <= (20 + abs(lp)) * EPS
    fn = pkg.PreferenceLoss(beta=1.0)
    ref = torch.full((2, 3), lp, dtype=torch.float32, device="cuda")
    fn(z, y, ref)
    want = 3 * (lp - float(ref[0, 0]))
    assert float((fn.rewards.double() - want).abs().max()) <= 3 * 20 * EPS
    fn = pkg.PolicyLoss(clip_low=1.0, clip_high=1e6)
    loss = fn(z, y, ref, torch.ones(2, 3, device="cuda"))
    # the ratio: exp of a small number (2 eps), the mean's rounding; S and its logarithm as float32 (4 eps)
    assert abs(float(loss) + math.exp(lp - float(ref[0, 0]))) <= (20 + 8) * EPS


@pytest.mark.parametrize("L,V,dtype", [(263, 24, "f32"), (263, 24, "bf16"), (300, 60, "f32")])
def test_rewards_of_long_sequences(pkg, L, V, dtype):
    """A reward is a long sum of small differences of large terms.  Per row the instruction's error (within one ulp,
    2 eps, either way: at most 1 eps in the root mean square) is what is left of S in 64 bits, whatever its sign, and its
    mean is taken off: sqrt(L) eps over a sequence, in the root mean square over the sequences, + the reward's rounding."""
    d = make(L + V, 64, L, V, dtype, mask=False)
    d["ref"] = torch.log_softmax(d["logits"].double(), -1).gather(-1, d["tokens"][..., None])[..., 0].float()
    lp = torch.log_softmax(d["logits"].double(), -1).gather(-1, d["tokens"][..., None])[..., 0]
    want = (lp - d["ref"].double()).sum(1)
    c = to_dev(d)
    fn = pkg.PreferenceLoss(beta=1.0)
    fn(c["logits"], c["tokens"], c["ref"])
    err = fn.rewards.cpu().double() - want
    assert float(err.square().mean().sqrt()) <= math.sqrt(L) * EPS + EPS * float(want.abs().max())


@pytest.mark.parametrize("V", [24, 2000, 70001])
@pytest.mark.parametrize("tau", [0.3, 1.3, 1.7, 3.0])
def test_ratios_of_improbable_tokens(pkg, V, tau):
    """The log-probability's two parts hold (z - m) / tau whatever its size.  With old = lp rounded to float32 the ratio
    is exp of a difference of at most half a step of lp: its error is that of lp, log S (4 eps: the exponentials' ulp, the
    sum's rounding to float32, the logarithm's ulp) and 2 eps of the parts' own last additions, plus 2 eps of the
    exponential and 1 eps of the mean's rounding; a row's float32 additions (V > 256) add up to 35 eps."""
    g = torch.Generator().manual_seed(V)
    z = torch.randn(4, 8, V, generator=g)
    z[..., 0] = 30.0
    y = torch.randint(1, V, (4, 8), generator=g)
    t32 = float(torch.tensor(tau, dtype=torch.float32))           # tau as the library takes it
    lp = torch.log_softmax(z.double() / t32, -1).gather(-1, y[..., None])[..., 0]
    old = lp.float()
    fn = pkg.PolicyLoss(clip_low=1.0, clip_high=1e6, temperature=tau)
    loss = fn(z.cuda(), y.cuda(), old.cuda(), torch.ones(4, 8, device="cuda"))
    want = -torch.exp(lp - old.double()).mean()
    assert abs(float(loss) - float(want)) <= (9 + (35 if V > 256 else 0)) * EPS * float(want.abs())


@pytest.mark.parametrize("N", [16384, 16385, 50001])
@pytest.mark.parametrize("name", ["distill", "policy"])
def test_mean_over_many_counted_positions(pkg, name, N):
    """Masks that the row launch counts itself, and longer ones that a launch ahead of it counts; the backward with another
    upstream gradient finds that count again."""
    d = make(N, 1, N, 20, "f32")
    d["mask"] = torch.rand(1, N, generator=torch.Generator().manual_seed(N)) < 0.4
    check(pkg, name, d)
    out, grad, bound = reference(name, d)
    c = to_dev(d)
    z = c["logits"].requires_grad_(True)
    g, = torch.autograd.grad(call(pkg, name, c, z)[0], z, torch.full((), 0.37, device="cuda"))
    check_grad(g, float(torch.tensor(0.37)) * grad, bound, z.dtype, 0.37)


@pytest.mark.parametrize("name", OBJECTIVES)
@pytest.mark.parametrize("kind", ["classes_apart", "odd_middle"])
def test_backward_makes_no_second_copy(pkg, name, kind):
    """Logits that are copied into rows are copied once, in the forward call."""
    B, L, V = 4, 32, 4096
    d = make(115, B, L, V, "f32", mask=False)
    c = to_dev(d)
    if kind == "classes_apart":
        z = c["logits"].transpose(1, 2).contiguous().transpose(1, 2)
    else:                                                     # [B, L / 4, 4, V] whose middle dimensions are swapped
        c = {k: (v.reshape((B, L // 4, 4) + v.shape[2:]) if torch.is_tensor(v) else v) for k, v in c.items()}
        z = c["logits"].transpose(1, 2).contiguous().transpose(1, 2)
    z = z.detach().requires_grad_(True)
    size = z.numel() * z.element_size()
    up = c["up"] if name == "logprobs" else torch.ones((), device="cuda")
    flat = z.detach().contiguous().requires_grad_(True)
    want, = torch.autograd.grad(call(pkg, name, c, flat)[0], flat, up)
    root, _ = call(pkg, name, c, z)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got, = torch.autograd.grad(root, z, up)
    grown = torch.cuda.max_memory_allocated() - before
    assert torch.equal(got, want)
    assert grown < (1.5 if name == "logprobs" else 0.5) * size      # (a log-probability's gradient is made in backward)


@pytest.mark.parametrize("name", OBJECTIVES)
def test_seen_by_dispatch_modes(pkg, name):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.ops = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.ops.append(str(func))
            return func(*args, **(kwargs or {}))

    c = to_dev(make(117, 4, 3, 20, "f32"))
    z = c["logits"].requires_grad_(True)
    up = c["up"] * c["mask"] if name == "logprobs" else None
    want, = torch.autograd.grad(call(pkg, name, c, z)[0], z, up)
    with Seen() as seen:
        root, _ = call(pkg, name, c, z)
    assert any(op.startswith("d3pm_mi355x.") for op in seen.ops), seen.ops
    with Seen() as seen:
        got, = torch.autograd.grad(root, z, up)
    assert any(op.startswith("d3pm_mi355x.") for op in seen.ops), seen.ops
    with Seen() as seen, torch.no_grad():
        call(pkg, name, c, z)
    assert any(op.startswith("d3pm_mi355x.") for op in seen.ops), seen.ops
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", OBJECTIVES)
def test_selective_checkpoint(pkg, name):
    """A checkpoint that keeps what these operators returned: they do not run again."""
    from functools import partial
    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts
    d = to_dev(make(107, 4, 5, 40, "f32"))
    h = torch.randn(20, 16, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)
    w = torch.randn(16, 40, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_(True)
    ran = []

    def keep(ctx, op, *args, **kwargs):
        mine = str(op).startswith("d3pm_mi355x.")
        if mine:
            ran.append(ctx.is_recompute)
        return CheckpointPolicy.MUST_SAVE if mine else CheckpointPolicy.PREFER_RECOMPUTE

    def part(h, w):
        return call(pkg, name, d, (h @ w).view(4, 5, 40))[0]

    root = part(h, w)
    up = 1.5 * torch.ones_like(root)
    want = torch.autograd.grad(root, (h, w), up)
    root = checkpoint(part, h, w, use_reentrant=False, context_fn=partial(create_selective_checkpoint_contexts, keep))
    got = torch.autograd.grad(root, (h, w), up)
    assert ran and all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("name", OBJECTIVES)
def test_under_func_grad(pkg, name):
    c = to_dev(make(119, 4, 3, 20, "f32"))
    z = c["logits"].clone().requires_grad_(True)
    total = lambda z: (call(pkg, name, c, z)[0] * (c["up"] * c["mask"] if name == "logprobs" else 1.0)).sum()
    want, = torch.autograd.grad(total(z), z)
    assert torch.equal(torch.func.grad(total)(c["logits"]), want)
    with pytest.raises(RuntimeError):                            # a gradient of the gradient
        torch.func.grad(lambda z: torch.func.grad(total)(z).square().sum())(c["logits"])
