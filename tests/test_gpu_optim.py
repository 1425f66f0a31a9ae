"""GPU: optimizer operators over a list of tensors (superresolution_amd/optim.py) against the 64-bit oracle, with tolerances
from the roundings of a single-precision evaluation (oracle/optim_ref.py: ``AdamWRef.step`` returns them)."""
import numpy as np
import pytest
import torch

from oracle import optim_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZES = {
    "one": [1],
    "blocks": [31, 32, 33, 64, 1, 0, 3],
    "chunks": [4095, 4096, 4097, 8192, 5],
    "many": [1 + (37 * i) % 301 for i in range(300)],                # several launches
    "mixed": [96 * 96 * 9, 96, 1, 13, 0, 20001],
}


def _f64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def _hash_floats(n, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g)) * scale


def _make(sizes, pdt, gdt, seed=0, gap=1):
    """Parameters and gradients as views of flat buffers, ``gap`` elements apart: starts of every alignment."""
    out = []
    for dt, s, scale in ((pdt, seed, 0.1), (gdt, seed + 1, 1e-2)):
        n = sum(sizes) + gap * (len(sizes) + 1)
        flat = _hash_floats(n, s, scale).to(dt).cuda()
        views, at = [], gap
        for k in sizes:
            views.append(flat[at:at + k])
            at += k + gap
        out.append((flat, views))
    return out


def _refs(opt, params, bits, seed=0):
    g, mo = opt.param_groups[0], opt.moments[0]
    return [R.AdamWRef(_f64(p), bits=bits, lr=float(g["lr"]), betas=g["betas"], eps=g["eps"], wd=g["weight_decay"], offset=o, seed=seed,
                       bf16=p.dtype == torch.bfloat16) for p, o in zip(params, mo.offsets)]


def _check(opt, params, refs, tols):
    mo = opt.moments[0]
    for i, (p, ref, (tp, tm, tv)) in enumerate(zip(params, refs, tols)):
        a, n = mo.offsets[i], mo.numels[i]
        if n == 0:
            continue
        if mo.bits == 32:
            np.testing.assert_array_less(np.abs(_f64(mo.exp_avg[a:a + n]) - ref.m), tm + 1e-300)
            np.testing.assert_array_less(np.abs(_f64(mo.exp_avg_sq[a:a + n]) - ref.v), tv + 1e-300)
            assert not mo.exp_avg[a + n:a + R.padded(n)].any() and not mo.exp_avg_sq[a + n:a + R.padded(n)].any()
        else:
            # evaluated in 64 bits on both sides: a value within 2^-50 of a border is the only one that could differ
            k = R.padded(n)
            for got, want in ((mo.exp_avg, ref.m8[0]), (mo.root, ref.r8[0])):
                np.testing.assert_array_equal(_f64(got[a:a + k].float()), want)
            for got, want in ((mo.exp_avg_scale, ref.m8[1]), (mo.root_scale, ref.r8[1])):
                np.testing.assert_array_equal(_f64(got[a // 32:(a + k) // 32].float()), want)
        got = _f64(p)
        if ref.bf16:
            lo, hi = ref.ends
            assert ((got >= np.minimum(lo, hi)) & (got <= np.maximum(lo, hi))).all(), i
            assert (got != ref.p).mean() <= 0.01 + 2.0 / n      # (a border within tol_p is rare: tol_p is 2^-15 of a bf16 step)
        else:
            assert (np.abs(got - ref.p) <= tp).all(), (i, np.abs(got - ref.p).max())


def _sync_ref(params, refs, mo):
    """The oracle goes on from what the kernel stored: one step's roundings are judged at a time."""
    for i, (p, ref) in enumerate(zip(params, refs)):
        a, n = mo.offsets[i], mo.numels[i]
        ref.p = _f64(p)
        if mo.bits == 32:
            ref.m, ref.v = _f64(mo.exp_avg[a:a + n]), _f64(mo.exp_avg_sq[a:a + n])


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("pdt, gdt", [("fp32", "fp32"), ("bf16", "bf16")])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_steps(bits, pdt, gdt, sizes):
    from superresolution_amd import optim
    sizes = SIZES[sizes]
    (flat, views), (gflat, gviews) = _make(sizes, DT[pdt], DT[gdt])
    before = flat.clone()
    params = [torch.nn.Parameter(v) for v in views]
    opt = optim.AdamW(params, lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05, state_bits=bits, seed=5)
    refs = _refs(opt, params, bits, seed=5)
    versions = [p._version for p in params]
    for s in range(3):
        gflat.copy_(_hash_floats(gflat.numel(), 100 + s, 10.0 ** -s).to(gflat.dtype))
        for p, g in zip(params, gviews):
            p.grad = g
        keep = gflat.clone()
        opt.step()
        tols = [r.step(_f64(g)) for r, g in zip(refs, gviews)]
        _check(opt, params, refs, tols)
        _sync_ref(params, refs, opt.moments[0])
        assert torch.equal(gflat, keep)                             # gradients are only read
    assert all(p._version >= v + 3 for p, v in zip(params, versions))        # (views of one buffer share their counter)
    inside = torch.zeros_like(flat, dtype=torch.bool)
    at = 1
    for k in sizes:
        inside[at:at + k] = True
        at += k + 1
    assert torch.equal(flat[~inside], before[~inside])              # nothing outside the tensors is written
    assert opt.moments[0].steps() == [3 if k else 0 for k in sizes]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pdt, gdt", [("fp32", "bf16"), ("bf16", "fp32")])
def test_adamw_mixed_types(bits, pdt, gdt):
    """Gradients of another type than the parameter's, through the C ABI's list (torch itself refuses such a .grad)."""
    from array import array
    from superresolution_amd import _lib, optim
    sizes = [1000, 37]
    (_, views), (_, gviews) = _make(sizes, DT[pdt], DT[gdt], seed=3)
    mo = optim.Moments(sizes, bits, torch.device("cuda", 0))
    refs = [R.AdamWRef(_f64(v), bits=bits, lr=1e-2, eps=1e-6, wd=0.0, offset=o, bf16=pdt == "bf16") for v, o in zip(views, mo.offsets)]
    args = _lib.srgen_adamw_args(1e-2, 0.9, 0.999, 1e-6, 0.0)
    code = {"fp32": 0, "bf16": 1}
    mo.update(array("Q", [v.data_ptr() for v in views]), array("Q", [v.data_ptr() for v in gviews]), array("i", [code[pdt]] * 2),
              array("i", [code[gdt]] * 2), args, torch.cuda.current_stream().cuda_stream)
    tols = [r.step(_f64(g)) for r, g in zip(refs, gviews)]

    class Holder:
        moments = [mo]
    _check(Holder, views, refs, tols)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("over", [dict(weight_decay=0.0), dict(maximize=True), dict(betas=(0.0, 0.0)), dict(eps=1e-3, lr=0.5), dict(lr=0.0)])
def test_adamw_hyperparameters(bits, over):
    from superresolution_amd import optim
    (_, views), (_, gviews) = _make([5000, 3], torch.float32, torch.float32, seed=9)
    params = [torch.nn.Parameter(v) for v in views]
    opt = optim.AdamW(params, state_bits=bits, **over)
    refs = _refs(opt, params, bits)
    sign = -1.0 if over.get("maximize") else 1.0
    for s in range(2):
        for p, g in zip(params, gviews):
            p.grad = g
        opt.step()
        _check(opt, params, refs, [r.step(sign * _f64(g)) for r, g in zip(refs, gviews)])
        _sync_ref(params, refs, opt.moments[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_without_gradients_keep_their_own_step(bits):
    from superresolution_amd import optim
    (_, views), (_, gviews) = _make([100, 5000, 7], torch.float32, torch.float32, seed=2)
    params = [torch.nn.Parameter(v) for v in views]
    opt = optim.AdamW(params, lr=1e-2, state_bits=bits)
    refs = _refs(opt, params, bits)
    mo = opt.moments[0]
    for turn in ((0,), (0, 2), (0, 1, 2), ()):
        for i, p in enumerate(params):
            p.grad = gviews[i] if i in turn else None
        before = [p.detach().clone() for p in params]
        opt.step()
        for i, p in enumerate(params):
            if i not in turn:
                assert torch.equal(p, before[i])
        used = [i for i in turn]
        tols = {i: refs[i].step(_f64(gviews[i])) for i in used}
        zero = (0.0, np.zeros(1), np.zeros(1))
        if bits == 8 or len(used) == 3:
            _check(opt, params, refs, [tols.get(i, (1e-300, 0.0, 0.0)) for i in range(3)])
        _sync_ref(params, refs, mo)
    assert mo.steps() == [3, 1, 2]


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite_gradients(bits):
    """A NaN or infinite gradient spoils its own element (and no other, not even in its block), for good, as in torch."""
    from superresolution_amd import optim
    n = 200
    p0, g0 = _hash_floats(n, 1), _hash_floats(n, 2, 1e-2)
    got = []
    for bad in (False, True):
        p, g = torch.nn.Parameter(p0.clone().cuda()), g0.clone().cuda()
        if bad:
            g[[5, 70, 199]] = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")
        opt = optim.AdamW([p], lr=1e-2, state_bits=bits)
        p.grad = g
        opt.step()
        got.append([p.detach().clone(), *opt.moments[0].read()])
        p.grad = g0.clone().cuda()
        opt.step()
        got[-1] += [p.detach().clone(), *opt.moments[0].read()]
    clean, spoilt = got
    for k, (a, b) in enumerate(zip(clean, spoilt)):
        a, b = a[:n], b[:n]
        isbad = torch.zeros(n, dtype=torch.bool, device="cuda")
        isbad[[5, 70, 199]] = True
        if k % 3 == 2 and bits == 32:
            # (an infinite gradient leaves an infinite second moment: not finite, not NaN)
            assert not torch.isfinite(b[isbad]).any()
        elif k % 3 != 2:
            assert not torch.isfinite(b[isbad]).any()
        if bits == 32:
            assert torch.equal(a[~isbad], b[~isbad])
        else:
            # the blocks of the spoilt elements take their scales without them: those may differ, within a step of the value
            blocks = torch.zeros(n, dtype=torch.bool, device="cuda")
            for i in (5, 70, 199):
                blocks[i // 32 * 32:i // 32 * 32 + 32] = True
            assert torch.equal(a[~blocks], b[~blocks])
            assert torch.isfinite(b[~isbad]).all()


def test_found_inf_and_grad_scale_as_the_grad_scaler_sets_them():
    from superresolution_amd import optim
    p = torch.nn.Parameter(_hash_floats(5000, 4).cuda())
    q = torch.nn.Parameter(p.detach().clone())
    a, b = optim.AdamW([p], lr=1e-2), optim.AdamW([q], lr=1e-2)
    g = _hash_floats(5000, 6, 1e-2).cuda()
    p.grad, q.grad = g * 1024.0, g.clone()
    a.grad_scale, a.found_inf = torch.tensor(1024.0, device="cuda"), torch.tensor(0.0, device="cuda")
    a.step()
    b.step()
    assert torch.equal(p, q)                                           # the scale is a power of two: the same bits
    keep = p.detach().clone()
    a.found_inf = torch.tensor(1.0, device="cuda")
    p.grad.fill_(float("nan"))
    a.step()
    assert torch.equal(p, keep) and a.moments[0].steps() == [1] and torch.isfinite(a.moments[0].exp_avg).all()


def test_grad_scaler_drives_it():
    from superresolution_amd import optim
    torch.manual_seed(0)
    model = torch.nn.Linear(16, 4).cuda()
    opt = optim.AdamW(model.parameters(), lr=1e-2, state_bits=8)
    scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 10)
    for k in range(3):
        opt.zero_grad()
        x = torch.randn(8, 16, device="cuda")
        loss = model(x).square().mean() * (float("inf") if k == 1 else 1.0)
        scaler.scale(loss).backward()
        before = model.weight.detach().clone()
        scaler.step(opt)
        scaler.update()
        assert torch.equal(before, model.weight) == (k == 1)
    assert opt.moments[0].steps() == [2, 2]


def test_grad_scaler_and_clipping():
    """Clipping inside the step wants unscaled gradients: refused otherwise, and the skipped step still tells its norm."""
    from superresolution_amd import optim
    torch.manual_seed(0)
    model = torch.nn.Linear(16, 4).cuda()
    twin = torch.nn.Linear(16, 4).cuda()
    twin.load_state_dict(model.state_dict())
    opt, ref = (optim.AdamW(m.parameters(), lr=1e-2, max_grad_norm=0.1) for m in (model, twin))
    scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 12)
    x = torch.randn(8, 16, device="cuda")
    scaler.scale(model(x).square().mean()).backward()
    with pytest.raises(RuntimeError, match="unscale_"):
        scaler.step(opt)
    opt.zero_grad()
    scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 12)
    for k in range(3):
        opt.zero_grad()
        ref.zero_grad()
        scaler.scale(model(x).square().mean() * (float("nan") if k == 1 else 1.0)).backward()
        scaler.unscale_(opt)
        scaler.step(opt)
        scaler.update()
        if k != 1:
            twin(x).square().mean().backward()
            ref.step()
            assert torch.equal(model.weight, twin.weight) and torch.equal(opt.last_grad_norm, ref.last_grad_norm)
        else:
            assert torch.isnan(opt.last_grad_norm)


def test_a_refused_group_keeps_the_others_from_stepping():
    from superresolution_amd import optim
    a, b = (torch.nn.Parameter(torch.ones(40, device="cuda")) for _ in range(2))
    opt = optim.AdamW([{"params": [a]}, {"params": [b]}], lr=1e-2)
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.param_groups[1]["lr"] = torch.tensor(1e-2, dtype=torch.float64, device="cuda")
    with pytest.raises(RuntimeError, match="fp32 scalar"):
        opt.step()
    assert torch.equal(a, torch.ones_like(a)) and opt.moments[0].steps() == [0]
    opt.param_groups[1]["lr"] = torch.tensor(1e-2, device="cuda")
    opt.step()
    assert torch.equal(a, b) and not torch.equal(a, torch.ones_like(a))


def test_hooks_and_profiler_see_the_step():
    from torch.optim.optimizer import register_optimizer_step_post_hook
    from superresolution_amd import optim
    p = torch.nn.Parameter(torch.ones(40, device="cuda"))
    opt = optim.AdamW([p], lr=1e-2)
    p.grad = torch.ones_like(p)
    seen = []
    pre = opt.register_step_pre_hook(lambda o, a, k: seen.append("pre"))
    post = opt.register_step_post_hook(lambda o, a, k: seen.append("post"))
    opt.step()
    assert seen == ["pre", "post"]
    pre.remove()
    post.remove()
    everywhere = register_optimizer_step_post_hook(lambda o, a, k: seen.append("all"))
    opt.step()
    everywhere.remove()
    assert seen == ["pre", "post", "all"]
    loss = opt.step(lambda: (p * 2.0).sum())
    assert float(loss) > 0 and len(seen) == 3 and opt.moments[0].steps() == [3]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("lr", [0.0, 1e-44, 1e-39, 1e-30])
def test_vanishing_learning_rates_and_zero_gradients(bits, lr):
    """Elements whose gradients have always been zero stay where they are (0 / eps), for any step size down to 0."""
    from superresolution_amd import optim
    p = torch.nn.Parameter(torch.ones(100, device="cuda"))
    opt = optim.AdamW([p], lr=lr, weight_decay=0.0, state_bits=bits)
    for _ in range(2):
        p.grad = torch.zeros_like(p)
        p.grad[::3] = 1e-3
        opt.step()
    assert torch.equal(p, torch.ones_like(p))


@pytest.mark.parametrize("bits", [32, 8])
def test_vanishing_eps_and_zero_gradients(bits):
    """0 / eps is 0 for the smallest eps too."""
    from superresolution_amd import optim
    p = torch.nn.Parameter(torch.ones(100, device="cuda"))
    opt = optim.AdamW([p], lr=0.5, eps=1e-42, weight_decay=0.0, state_bits=bits)
    for _ in range(2):
        p.grad = torch.zeros_like(p)
        opt.step()
    assert torch.equal(p, torch.ones_like(p))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_clip_inside_the_step(bits, max_norm):
    from superresolution_amd import optim
    sizes = SIZES["many"]
    (_, views), (_, gviews) = _make(sizes, torch.float32, torch.float32, seed=12)
    params = [torch.nn.Parameter(v) for v in views]
    opt = optim.AdamW(params, lr=1e-2, state_bits=bits, max_grad_norm=max_norm)
    refs = _refs(opt, params, bits)
    for p, g in zip(params, gviews):
        p.grad = g
    keep = [g.clone() for g in gviews]
    opt.step()
    want = np.sqrt(sum((_f64(g) ** 2).sum() for g in gviews))
    norm = float(opt.last_grad_norm)
    assert abs(norm - want) <= 1.01 * R.U24 * want
    coef = float(np.float32(min(1.0, max_norm / (norm + 1e-6))))
    assert (coef < 1.0) == (max_norm == 0.5)
    # (32 bits: the product with the coefficient is one more rounding, which tol_m already counts)
    _check(opt, params, refs, [r.step(_f64(g), coef) for r, g in zip(refs, gviews)])
    assert all(torch.equal(a, b) for a, b in zip(keep, gviews))


@pytest.mark.parametrize("sizes", [[5_000_003, 7], [100] * 1100, [0, 0]])
def test_clip_inside_the_step_with_more_partial_sums_than_a_wave_adds(sizes):
    """More than 1,024 partial sums take a launch of their own; a list of empty tensors has norm 0.  Against clipping in place."""
    from superresolution_amd import optim
    ps = [torch.nn.Parameter(_hash_floats(n, i).cuda()) for i, n in enumerate(sizes)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for i, (p, q) in enumerate(zip(ps, qs)):
        p.grad = _hash_floats(p.numel(), 5000 + i, 1e-2).cuda()
        q.grad = p.grad.clone()
    a, b = optim.AdamW(ps, lr=1e-2, max_grad_norm=0.5), optim.AdamW(qs, lr=1e-2)
    a.step()
    norm = optim.clip_grad_norm_(qs, 0.5)
    b.step()
    assert torch.equal(a.last_grad_norm, norm) and all(torch.equal(p, q) for p, q in zip(ps, qs))
    want = np.sqrt(sum((_f64(p.grad) ** 2).sum() for p in ps))
    assert abs(float(norm) - want) <= 1.01 * R.U24 * want


def test_clipping_norm_where_the_first_tensors_have_no_gradient_or_the_step_is_skipped():
    from superresolution_amd import optim
    ps = [torch.nn.Parameter(_hash_floats(50, i).cuda()) for i in range(300)]
    for i in (7, 299):
        ps[i].grad = _hash_floats(50, 70 + i).cuda()
    want = optim.total_norm([ps[7].grad, ps[299].grad])
    opt = optim.AdamW(ps, lr=1e-2, max_grad_norm=0.1)
    assert opt.last_grad_norm is None
    for _ in range(3):                                                  # (the buffer's earlier contents do not help)
        torch.full((4096,), float("nan"), device="cuda")
        opt.step()
        assert torch.equal(opt.last_grad_norm, want)
    keep = ps[7].detach().clone()
    opt.found_inf = torch.ones((), device="cuda")
    torch.full((4096,), float("nan"), device="cuda")
    opt.step()
    assert torch.equal(opt.last_grad_norm, want) and torch.equal(ps[7], keep)
    assert opt.moments[0].steps()[7] == 3 and opt.moments[0].steps()[0] == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_follows_the_learning_rate_and_counts(bits):
    """A captured step replayed five times, with eager work and synchronisation between, against eager steps; the learning
    rate lives on the device and changes; two optimizers' graphs do not disturb each other."""
    from superresolution_amd import optim
    sizes = [5000, 33, 1]

    def build(lr):
        (_, views), (_, gviews) = _make(sizes, torch.float32, torch.float32, seed=21)
        params = [torch.nn.Parameter(v) for v in views]
        for p, g in zip(params, gviews):
            p.grad = g
        return params, gviews, optim.AdamW(params, lr=lr, state_bits=bits, max_grad_norm=0.3)

    lr = [torch.tensor(1e-2, device="cuda") for _ in range(3)]
    eager, g0, opt0 = build(lr[0])
    one, g1, opt1 = build(lr[1])
    two, g2, opt2 = build(lr[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for opt in (opt1, opt2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                opt.step()
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(5):
        fresh = [_hash_floats(n, 50 + k * 3 + i, 1e-2).cuda() for i, n in enumerate(sizes)]
        for gs in (g0, g1, g2):
            for a, b in zip(gs, fresh):
                a.copy_(b)
        for t in lr:
            t.fill_(1e-2 / (k + 1))
        opt0.step()
        for graph in graphs:
            graph.replay()
        (torch.randn(64, 64, device="cuda") @ torch.randn(64, 64, device="cuda")).sum().item()
        for other, opt in ((one, opt1), (two, opt2)):
            assert all(torch.equal(a, b) for a, b in zip(eager, other)), k
            assert torch.equal(opt0.last_grad_norm, opt.last_grad_norm)
            for a, b in zip(opt0.moments[0].read(), opt.moments[0].read()):
                assert torch.equal(a, b)
    assert opt1.moments[0].steps() == [5, 5, 5]


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(bits):
    """Dense parameters of other orders than C's, gradients of another order than the parameter's, expanded gradients."""
    from superresolution_amd import optim
    w = _hash_floats(6 * 5 * 3 * 3, 1).view(6, 5, 3, 3).cuda()
    g = _hash_floats(6 * 5 * 3 * 3, 2, 1e-2).view(6, 5, 3, 3).cuda()
    plain = torch.nn.Parameter(w.clone())
    plain.grad = g.clone()
    a = optim.AdamW([plain], lr=1e-2)
    last = torch.nn.Parameter(w.clone(memory_format=torch.channels_last))
    b = optim.AdamW([last], lr=1e-2)
    last.grad = g.clone()                                              # C order beside a channels-last parameter
    ones = torch.nn.Parameter(w.clone())
    c = optim.AdamW([ones], lr=1e-2, state_bits=bits)
    ones.sum().backward()
    assert ones.grad.stride() == (0, 0, 0, 0) or ones.grad.is_contiguous()
    for o in (a, b, c):
        o.step()
    assert torch.equal(plain, last)
    x = torch.nn.Parameter(w.clone())
    x.grad = torch.ones_like(w)
    d = optim.AdamW([x], lr=1e-2, state_bits=bits)
    d.step()
    assert torch.equal(x, ones)
    sa, sb = a.state_dict()["state"][0], b.state_dict()["state"][0]
    assert torch.equal(sa["exp_avg"], sb["exp_avg"]) and torch.equal(sa["exp_avg_sq"], sb["exp_avg_sq"])
    b2 = optim.AdamW([last], lr=1e-2)
    b2.load_state_dict(a.state_dict())
    assert torch.equal(b2.moments[0].exp_avg, b.moments[0].exp_avg)


def test_parameters_that_change_under_the_optimizer():
    """Taken out of its group, of another order, or with a gradient of another size: refused, and nothing is written."""
    from superresolution_amd import optim
    w = _hash_floats(6 * 5 * 3 * 3, 1).view(6, 5, 3, 3).cuda()
    a, b = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.clone())
    opt = optim.AdamW([a, b], lr=1e-2)
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.step()
    kept = b.detach().clone()
    out = opt.param_groups[0]["params"].pop()
    with pytest.raises(RuntimeError, match="number of elements"):
        opt.step()
    assert torch.equal(out, kept)
    opt.param_groups[0]["params"].append(out)
    opt.step()
    assert torch.equal(a, b) and not torch.equal(b, kept)

    for first, then in ((torch.contiguous_format, torch.channels_last), (torch.channels_last, torch.contiguous_format)):
        p = torch.nn.Parameter(w.clone(memory_format=first))
        opt = optim.AdamW([p], lr=1e-2)
        p.grad = torch.ones_like(p)
        opt.step()
        p.data = p.data.contiguous(memory_format=then)
        with pytest.raises(RuntimeError, match="another order"):
            opt.step()
        p.data = p.data.contiguous(memory_format=first)
        opt.step()
        assert opt.moments[0].steps() == [2] and torch.equal(p, a)

    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = optim.AdamW([p], lr=1e-2)
    p.data = torch.ones(4, device="cuda")
    p.grad = torch.ones(4, device="cuda")
    p.data = torch.ones(8, device="cuda")
    with pytest.raises(RuntimeError, match="gradient of shape"):
        opt.step()


def test_lazily_negated_gradients():
    from superresolution_amd import optim
    g = _hash_floats(70, 2).cuda()
    a, b = (torch.nn.Parameter(torch.ones(70, device="cuda")) for _ in range(2))
    a.grad, b.grad = -g, torch._neg_view(g)
    for p in (a, b):
        optim.AdamW([p], lr=1e-2).step()
    assert torch.equal(a, b)
    assert torch.equal(optim.total_norm([a.grad]), optim.total_norm([b.grad]))
    with pytest.raises(RuntimeError, match="negated"):
        p = torch.nn.Parameter(torch._neg_view(torch.ones(70, device="cuda")))
        p.grad = torch.ones_like(p)
        optim.AdamW([p], lr=1e-2).step()


def test_loaded_groups_are_copies():
    from superresolution_amd import optim
    lr = torch.tensor(1e-2, device="cuda")
    a, b = (optim.AdamW([torch.nn.Parameter(torch.ones(8, device="cuda"))], lr=lr) for _ in range(2))
    b.load_state_dict(a.state_dict())
    lr.fill_(1.0)
    assert float(b.param_groups[0]["lr"]) == float(torch.tensor(1e-2))
    sd = a.state_dict()
    sd["param_groups"][0]["decoupled_weight_decay"] = False
    with pytest.raises(ValueError, match="weight decay"):
        b.load_state_dict(sd)


def test_a_group_with_bad_numbers_keeps_the_others_from_stepping():
    from superresolution_amd import optim
    a, b = (torch.nn.Parameter(torch.ones(40, device="cuda")) for _ in range(2))
    opt = optim.AdamW([{"params": [a]}, {"params": [b]}], lr=1e-2)
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    for key, bad in (("lr", -1.0), ("betas", (0.9, 1.0)), ("eps", float("nan")), ("weight_decay", -1.0)):
        good = opt.param_groups[1][key]
        opt.param_groups[1][key] = bad
        with pytest.raises(ValueError, match="Invalid"):
            opt.step()
        opt.param_groups[1][key] = good
    assert torch.equal(a, torch.ones_like(a)) and opt.moments[0].steps() == [0]


def test_refusals_on_the_device():
    from superresolution_amd import optim
    t = torch.zeros(64, device="cuda")
    with pytest.raises(RuntimeError, match="share memory"):
        optim.AdamW([torch.nn.Parameter(t[:40]), torch.nn.Parameter(t[32:])])
    p = torch.nn.Parameter(t)
    with pytest.raises((RuntimeError, ValueError), match="twice|duplicate|share memory"):
        optim.AdamW([p, p])
    with pytest.raises(RuntimeError, match="fp32 or bf16 parameters"):
        optim.AdamW([torch.nn.Parameter(t.half())])
    with pytest.raises(RuntimeError, match="gaps or overlaps"):
        optim.AdamW([torch.nn.Parameter(t[::2])])
    opt = optim.AdamW([p])
    p.data = torch.zeros(32, device="cuda")
    p.grad = torch.zeros(32, device="cuda")
    with pytest.raises(RuntimeError, match="number of elements"):
        opt.step()
    p.data = torch.zeros(64, device="cuda", dtype=torch.half)
    p.grad = None
    with pytest.raises(RuntimeError, match="fp32 or bf16 parameters"):
        opt.step()
    with pytest.raises(RuntimeError, match="state_dict"):
        import copy
        copy.deepcopy(opt)
    q = torch.nn.Parameter(torch.zeros(64, device="cuda"))
    with pytest.raises(ValueError, match="match the size"):
        opt.load_state_dict(optim.AdamW([q, torch.nn.Parameter(torch.zeros(3, device="cuda"))]).state_dict())
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        optim.total_norm([torch.zeros(3, device="cuda", dtype=torch.float64)])
    g = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    g.grad = torch.zeros(1, device="cuda").expand(4)
    with pytest.raises(RuntimeError, match="gaps or overlaps"):
        optim.clip_grad_norm_([g], 1.0)
    with pytest.raises(RuntimeError, match="non-finite"):
        g.grad = torch.full((4,), float("nan"), device="cuda")
        optim.clip_grad_norm_([g], 1.0, error_if_nonfinite=True)


def test_another_stream():
    """Everything is enqueued on the caller's stream: steps on a side stream behind work that is not done yet."""
    from superresolution_amd import optim
    p = torch.nn.Parameter(torch.zeros(1 << 20, device="cuda"))
    q = torch.nn.Parameter(torch.zeros(1 << 20, device="cuda"))
    a, b = optim.AdamW([p], lr=1e-2, max_grad_norm=1.0), optim.AdamW([q], lr=1e-2, max_grad_norm=1.0)
    g = _hash_floats(1 << 20, 3).cuda()
    big = torch.randn(4096, 4096, device="cuda")
    q.grad = g.clone()
    b.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-2
        p.grad = torch.zeros_like(g)
        p.grad.copy_(g)
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(p, q) and torch.equal(a.last_grad_norm, b.last_grad_norm)


def test_steps_repeat_bit_for_bit_and_seeds_matter():
    from superresolution_amd import optim

    def run(seed):
        (_, views), (_, gviews) = _make([30000, 11], torch.bfloat16, torch.bfloat16, seed=31)
        params = [torch.nn.Parameter(v) for v in views]
        opt = optim.AdamW(params, lr=1e-3, state_bits=8, max_grad_norm=1.0, seed=seed)
        for _ in range(3):
            for p, g in zip(params, gviews):
                p.grad = g
            opt.step()
        return [p.detach().clone() for p in params] + [opt.moments[0].exp_avg.view(torch.uint8).clone(), opt.last_grad_norm]
    a, b, c = run(1), run(1), run(2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert not torch.equal(a[0], c[0]) and not torch.equal(a[2], c[2])


def test_stochastic_rounding_follows_a_mean_that_nearest_would_not():
    """beta2 = 0.999 moves the second moment by at most 0.1 % a step, an e4m3 step is 6 to 12 %: rounded to nearest it would
    stay where it is.  After 2,000 steps of a constant gradient the mean over 4,096 elements has moved as the 32-bit one."""
    from superresolution_amd import optim
    n = 4096
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = optim.AdamW([p], lr=0.0, weight_decay=0.0, state_bits=8)
    sd = opt.state_dict()
    sd["state"] = {0: {"step": torch.tensor(1.0), "exp_avg": torch.full((n,), 0.01), "exp_avg_sq": torch.full((n,), 1e-4)}}
    opt.load_state_dict(sd)
    start = float(opt.moments[0].read()[1][:n].mean())
    p.grad = torch.full((n,), 0.02, device="cuda")                     # the second moment goes from 1e-4 towards 4e-4
    for _ in range(2000):
        opt.step()
    v = opt.moments[0].read()[1][:n]
    w = 0.999 ** 2000
    want = w * start + (1 - w) * 4e-4
    # One rounding of the root r has variance at most (step of r)^2 / 4 * (change / step) ... bounded by change * step: with
    # change <= 5e-4 * 1.5 r and step <= r / 8 that is 1e-4 r^2 a step, forgotten at rate 1e-3 of r^2: 2e-1 relative at the most
    # for one element's v, 5 standard errors of 4,096 elements are 1.6 %; squaring adds the variance of r, under 5 %
    assert abs(float(v.mean()) / want - 1.0) < 0.07
    assert float(v.mean()) > 2.5 * start


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_moves_between_torch_and_here(bits):
    from superresolution_amd import optim
    sizes = [300, 5, 4097]
    ps = [torch.nn.Parameter(_hash_floats(n, i).cuda()) for i, n in enumerate(sizes)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    t, a = torch.optim.AdamW(ps, lr=1e-2), optim.AdamW(qs, lr=1e-2, state_bits=bits)
    gs = [_hash_floats(n, 60 + i, 1e-2).cuda() for i, n in enumerate(sizes)]
    for p, g in zip(ps, gs):
        p.grad = g.clone()
    t.step()
    a.load_state_dict(t.state_dict())                                   # torch -> here
    assert a.moments[0].steps() == [1, 1, 1]
    sd = a.state_dict()
    for i, p in enumerate(ps):
        for key in ("exp_avg", "exp_avg_sq"):
            want, got = t.state[p][key], sd["state"][i][key]
            # 8 bits: to nearest, half a step of e4m3 (2^-4 of the value, the square root's doubled), or half the smallest step
            # of its block (2^-10 of the scale, which is at most 2^-8 of the block's largest)
            if bits == 32:
                assert torch.equal(want, got)
            else:
                tol = 2.0 ** -4 if key == "exp_avg" else 2.0 ** -3 + 2.0 ** -8
                ends = torch.cat([want, want.new_zeros(R.padded(want.numel()) - want.numel())]).view(-1, 32).abs().amax(1)
                big = ends.repeat_interleave(32)[:want.numel()]
                low = big * 2.0 ** -18 if key == "exp_avg" else big * 2.0 ** -16
                assert ((want - got).abs() <= want.abs() * tol + low).all()
    b = optim.AdamW([torch.nn.Parameter(q.detach().clone()) for q in qs], lr=5e-2, state_bits=8)
    b.load_state_dict(sd)                                               # here -> here, through fp32
    if bits == 8:
        for x, y in ((a, b),):
            assert torch.equal(x.moments[0].read()[0], y.moments[0].read()[0]) and torch.equal(x.moments[0].read()[1], y.moments[0].read()[1])
    assert b.param_groups[0]["lr"] == 1e-2
    u = torch.optim.AdamW(qs, lr=1e-2)
    u.load_state_dict(sd)                                               # here -> torch
    for q, g in zip(qs, gs):
        q.grad = g.clone()
    u.step()
    assert all(torch.isfinite(q).all() for q in qs)


def test_matches_torch_adamw_over_several_steps():
    """32 bits against torch.optim.AdamW, five steps: both round in fp32, so twice the oracle's tolerance a step."""
    from superresolution_amd import optim
    sizes = [20000, 77, 1]
    ps = [torch.nn.Parameter(_hash_floats(n, i).cuda()) for i, n in enumerate(sizes)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    t, a = torch.optim.AdamW(ps, lr=1e-2, weight_decay=0.1), optim.AdamW(qs, lr=1e-2, weight_decay=0.1)
    refs = _refs(a, qs, 32)
    total = [0.0] * 3
    for s in range(5):
        for i, (p, q) in enumerate(zip(ps, qs)):
            p.grad = _hash_floats(sizes[i], 10 * s + i, 1e-2).cuda()
            q.grad = p.grad.clone()
            total[i] = total[i] + refs[i].step(_f64(p.grad))[0]
        t.step()
        a.step()
    for i, (p, q) in enumerate(zip(ps, qs)):
        # (errors of the moments are carried from step to step: four times the sum covers them)
        assert (np.abs(_f64(p) - _f64(q)) <= 4 * total[i]).all()


def test_two_groups_and_scheduler():
    from superresolution_amd import optim
    p, q = (torch.nn.Parameter(_hash_floats(5000, i).cuda()) for i in (1, 2))
    p2, q2 = (torch.nn.Parameter(x.detach().clone()) for x in (p, q))
    a = optim.AdamW([dict(params=[p], lr=1e-2), dict(params=[q], weight_decay=0.0)], lr=1e-3, max_grad_norm=0.1)
    b = [optim.AdamW([p2], lr=1e-2), optim.AdamW([q2], lr=1e-3, weight_decay=0.0)]
    sched = torch.optim.lr_scheduler.CosineAnnealingLR(a, T_max=10)
    for s in range(3):
        for x, y, k in ((p, p2, 1), (q, q2, 2)):
            x.grad = _hash_floats(5000, 7 * s + k).cuda()
            y.grad = x.grad.clone()
        for o, g in zip(b, a.param_groups):
            o.param_groups[0]["lr"] = g["lr"]
        norm = optim.clip_grad_norm_([p2, q2], 0.1)
        a.step()
        for o in b:
            o.step()
        sched.step()
        assert torch.equal(norm, a.last_grad_norm)
    # clipping in place rounds the gradients to fp32 as the step's product does: the same bits
    assert torch.equal(p, p2) and torch.equal(q, q2)
    assert a.param_groups[0]["lr"] < 1e-2
    a.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(9, device="cuda"))]))
    assert len(a.moments) == 3


@pytest.mark.parametrize("bits", [8, 32])
def test_positions_that_pass_32_bits(bits):
    """A bf16 parameter of 2^32 + 100 elements: offsets, the position's high word in the random bits, the last ragged block."""
    from superresolution_amd import optim
    n = (1 << 32) + 100
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    tail = 4096 + 100
    p[-tail:], g[-tail:] = _hash_floats(tail, 1, 0.1).cuda().bfloat16(), _hash_floats(tail, 2, 1e-2).cuda().bfloat16()
    p[:4096], g[:4096] = _hash_floats(4096, 3, 0.1).cuda().bfloat16(), _hash_floats(4096, 4, 1e-2).cuda().bfloat16()
    param = torch.nn.Parameter(p)
    param.grad = g
    opt = optim.AdamW([param], lr=1e-2, state_bits=bits, seed=3, max_grad_norm=1e9)
    want = np.sqrt((_f64(g[-tail:]) ** 2).sum() + (_f64(g[:4096]) ** 2).sum())
    for lo, hi in ((n - tail, n), (0, 4096)):
        ref = R.AdamWRef(_f64(p[lo:hi]), bits=bits, lr=1e-2, seed=3, bf16=True, first=lo)
        if lo:
            opt.step()
            assert abs(float(opt.last_grad_norm) - want) <= 1.01 * R.U24 * want
            after = param.detach()
        else:
            ref.p = _hash_floats(4096, 3, 0.1).bfloat16().double().numpy()
        ref.step(_f64(g[lo:hi]))
        lo_, hi_ = ref.ends
        got = _f64(after[lo:hi])
        assert ((got >= np.minimum(lo_, hi_)) & (got <= np.maximum(lo_, hi_))).all()
        assert (got != ref.p).mean() <= 0.01
        if bits == 8:
            k = R.padded(hi - lo)
            np.testing.assert_array_equal(_f64(opt.moments[0].exp_avg[lo:lo + k].float()), ref.m8[0])
            np.testing.assert_array_equal(_f64(opt.moments[0].root_scale[lo // 32:(lo + k) // 32].float()), ref.r8[1])
    assert not after[4096:1 << 20].any()


def test_a_chunk_that_crosses_the_32_bit_position():
    """The second tensor starts at position 32: one of its chunks has elements on both sides of position 2^32."""
    from superresolution_amd import optim
    n = (1 << 32) + 5000
    q, p, g = (torch.zeros(k, device="cuda", dtype=torch.bfloat16) for k in (7, n, n))
    lo = (1 << 32) - 32 - 4064 - 4096                                   # 32 + lo is the start of a chunk, two before the crossing one
    p[lo:], g[lo:] = _hash_floats(n - lo, 1, 0.1).cuda().bfloat16(), _hash_floats(n - lo, 2, 1e-2).cuda().bfloat16()
    params = [torch.nn.Parameter(q), torch.nn.Parameter(p)]
    params[0].grad, params[1].grad = torch.ones_like(q), g
    opt = optim.AdamW(params, lr=1e-2, state_bits=8, seed=9)
    ref = R.AdamWRef(_f64(p[lo:]), bits=8, lr=1e-2, seed=9, bf16=True, offset=32, first=lo)
    opt.step()
    ref.step(_f64(g[lo:]))
    k = R.padded(n - lo)
    np.testing.assert_array_equal(_f64(opt.moments[0].exp_avg[32 + lo:32 + lo + k].float()), ref.m8[0])
    np.testing.assert_array_equal(_f64(opt.moments[0].root[32 + lo:32 + lo + k].float()), ref.r8[0])
    a, b = ref.ends
    got = _f64(params[1][lo:])
    assert ((got >= np.minimum(a, b)) & (got <= np.maximum(a, b))).all()


# ---- total norm, clipping ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", list(SIZES))
def test_total_norm(dt, sizes):
    from superresolution_amd import optim
    (_, views), _ = _make(SIZES[sizes], dt, dt, seed=40)
    want = np.sqrt(sum((_f64(v) ** 2).sum() for v in views))
    got = [optim.total_norm(views) for _ in range(2)]
    assert torch.equal(got[0], got[1]) and got[0].dtype == torch.float32 and got[0].dim() == 0
    # sums in 64 bits (their rounding is 2^-40 of it at the most), one rounding to fp32
    assert abs(float(got[0]) - want) <= 1.01 * R.U24 * want


def test_total_norm_large_and_ends_of_the_range():
    from superresolution_amd import optim
    x = torch.randn(50_000_003, device="cuda")
    want = float(x.double().norm())
    assert abs(float(optim.total_norm([x[1:], x[:1]])) - want) <= 1.01 * R.U24 * want
    for scale in (1e30, 1e-30, 1e-40):                                  # squares leave fp32's range, the norm does not
        t = torch.full((1000,), scale, device="cuda")
        want = float(t.double().norm())
        assert abs(float(optim.total_norm(t)) - want) <= 1.01 * R.U24 * want + 2.0 ** -150
    t = torch.ones(100, device="cuda")
    t[3] = float("inf")
    assert float(optim.total_norm([t])) == float("inf")
    t[5] = float("nan")
    assert np.isnan(float(optim.total_norm([t])))
    assert float(optim.total_norm([torch.zeros(0, device="cuda")])) == 0.0
    assert float(optim.total_norm(torch.full((7, 5), 2.0, device="cuda").t())) == pytest.approx(2.0 * 35 ** 0.5, rel=1e-6)
    assert float(optim.total_norm(torch.full((8, 4), 1.0, device="cuda")[:, ::2])) == 4.0


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("max_norm", [0.7, 1e5])
def test_clip_grad_norm(dt, max_norm):
    from superresolution_amd import optim
    sizes = SIZES["many"] + [9001]
    (flat, views), _ = _make(sizes, dt, dt, seed=50)
    flat.mul_(10.0)
    params = []
    for v in views:
        p = torch.nn.Parameter(torch.zeros_like(v))
        p.grad = v
        params.append(p)
    before = flat.clone()
    want = np.sqrt(sum((_f64(v) ** 2).sum() for v in views))
    versions = [v._version for v in views]
    norm = optim.clip_grad_norm_(params, max_norm)
    assert abs(float(norm) - want) <= 1.01 * R.U24 * want
    assert torch.equal(optim.grad_norm(torch.nn.ParameterList(params)), optim.total_norm(views))
    coef = min(1.0, max_norm / (float(norm) + 1e-6))
    if coef == 1.0:
        assert torch.equal(flat, before)
        return
    gap = torch.ones_like(flat, dtype=torch.bool)
    at = 1
    for k in sizes:
        gap[at:at + k] = False
        at += k + 1
    assert torch.equal(flat[gap], before[gap])
    x = before[~gap].double() * coef
    # coefficient to fp32, product to fp32, then to the gradients' type (half a step each; fp16 has subnormals)
    half = torch.finfo(dt).eps / 2
    assert ((flat[~gap].double() - x).abs() <= x.abs() * (2 * R.U24 + half * (1 + 2 * R.U24)) + (2.0 ** -25 if dt == torch.float16 else 0.0)).all()
    assert all(v._version > w for v, w in zip(views, versions) if v.numel())


def test_clip_with_a_norm_that_is_not_finite_is_torchs():
    from superresolution_amd import optim
    for bad in (float("inf"), float("nan")):
        g = torch.tensor([1.0, bad, -2.0, 0.0], device="cuda")
        p, q = (torch.nn.Parameter(torch.zeros(4, device="cuda")) for _ in range(2))
        p.grad, q.grad = g.clone(), g.clone()
        a = optim.clip_grad_norm_([p], 1.0)
        b = torch.nn.utils.clip_grad_norm_([q], 1.0)
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(torch.nan_to_num(p.grad, nan=7.0), torch.nan_to_num(q.grad, nan=7.0))


# ---- moments in 8 bits -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 31, 32, 33, 1024, 100_003])
def test_pack_and_unpack(n):
    from superresolution_amd import optim
    m = _hash_floats(n, 1) * torch.exp(4 * torch.randn(n, generator=torch.Generator().manual_seed(3)))
    v = _hash_floats(n, 2).square()
    m[:: 17], v[:: 13] = 0.0, 0.0
    big = torch.cat([torch.zeros(1), m]).cuda()
    m8, me, r8, re = optim.pack_moments(big[1:], v.cuda())              # (4-byte aligned only)
    want = R.pack(m.numpy(), v.numpy())
    for got, w in zip((m8, me, r8, re), want):
        np.testing.assert_array_equal(_f64(got.float()), w)
    a, b = optim.unpack_moments(m8, me, r8, re, n)
    np.testing.assert_array_equal(_f64(a), R.values(want[0], want[1])[:n])
    np.testing.assert_array_equal(_f64(b), R.values(want[2], want[3])[:n] ** 2)
    again = optim.pack_moments(a, b)
    c, d = optim.unpack_moments(*again, n)
    assert torch.equal(a, c) and torch.equal(b, d)                     # what 8 bits hold comes back as it was


def test_pack_ends_of_the_range():
    """Blocks of zeros, subnormals, the largest values, magnitudes around 1.75 * 2^k, ties, infinities and NaN, negative zero."""
    from superresolution_amd import optim
    top = float(np.finfo(np.float32).max)
    rows = [np.zeros(32), np.full(32, 1e-45), np.linspace(0, 1e-38, 32), np.full(32, top), np.geomspace(1e-38, top, 32),
            1.75 * (1 + np.linspace(-1e-6, 1e-6, 32)), 2.0 - np.geomspace(1e-7, 0.2, 32), np.arange(32) / 16.0 + 1 / 32.0,
            np.where(np.arange(32) % 5 == 0, np.inf, np.arange(32)), np.where(np.arange(32) == 7, np.nan, 3.0), np.full(32, -0.0),
            np.full(32, np.nan), np.geomspace(1.0, 2.0 ** -20, 32)]
    m = torch.tensor(np.concatenate(rows), dtype=torch.float32)
    sign = torch.where(torch.arange(m.numel()) % 2 == 0, 1.0, -1.0)
    v = m.abs()
    got = optim.pack_moments((m * sign).cuda(), v.cuda())
    for x, w in zip(got, R.pack((m * sign).numpy(), v.numpy())):
        np.testing.assert_array_equal(_f64(x.float()), w)
    a, b = optim.unpack_moments(*got, m.numel())
    ok = torch.isfinite(m)
    assert torch.isfinite(a.cpu()[ok]).all() and torch.isnan(a.cpu()[~ok]).all()
    assert (b.cpu()[ok & (v >= 1e-37)] > 0).all()                      # a root that is not zero is not stored as zero


def test_unpack_refuses():
    from superresolution_amd import optim
    m8, me, r8, re = optim.pack_moments(torch.ones(64, device="cuda"), torch.ones(64, device="cuda"))
    with pytest.raises(RuntimeError, match="of 64 elements"):
        optim.unpack_moments(m8, me, r8, re, 65)
    with pytest.raises(RuntimeError, match="e8m0 scale"):
        optim.unpack_moments(m8, me[:1], r8, re, 64)
    with pytest.raises(RuntimeError, match="e8m0 scale"):
        optim.unpack_moments(m8, me.view(torch.uint8), r8, re, 64)
    with pytest.raises(RuntimeError, match="4-byte aligned"):
        optim.unpack_moments(m8[1:33], me[:1], r8[1:33], re[:1], 32)
    with pytest.raises(RuntimeError, match="flat contiguous fp32"):
        optim.pack_moments(torch.ones(4, 4, device="cuda"), torch.ones(4, 4, device="cuda"))


# ---- as they are used together -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_the_reference_loop_with_these_operators(bits):
    """Two iterations of the reference's pre-train loop body on the drop-in generator (train.py:90-97), with the optimizer,
    the clipping and the logged norm of this module, then a checkpoint: against torch's optimizer on the same gradients."""
    from superresolution_amd import Generator, optim, pixel_loss
    torch.manual_seed(0)
    gen = Generator().cuda().train()
    opt = optim.AdamW(gen.parameters(), lr=1e-4, state_bits=bits, max_grad_norm=0.05)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in gen.parameters()]
    ref = torch.optim.AdamW(twin, lr=1e-4)
    lr_img, hr = torch.rand(2, 3, 64, 64, device="cuda"), torch.rand(2, 3, 125, 125, device="cuda")
    for _ in range(2):
        loss = pixel_loss(gen(lr_img), hr)
        opt.zero_grad()
        loss.backward()
        for p, t in zip(gen.parameters(), twin):
            t.grad = p.grad.clone()
        want = torch.nn.utils.clip_grad_norm_(twin, 0.05)
        logged = optim.grad_norm(gen)
        opt.step()
        ref.step()
        assert torch.equal(logged, opt.last_grad_norm)
        assert abs(float(logged) - float(want)) <= 1e-5 * float(want)     # torch adds in fp32
    moved = rel = 0.0
    for p, t in zip(gen.parameters(), twin):
        rel = max(rel, float((p - t).abs().max()))
        moved = max(moved, float((t - p.detach()).abs().max()))
    # a step moves a parameter by at most about lr; 8-bit moments scatter it by less than that each of the two steps
    assert rel <= (1e-6 if bits == 32 else 2e-4)
    gen.eval()
    with torch.no_grad():
        assert torch.isfinite(gen(lr_img)).all()                          # (the weights are uploaded again)
    sd = opt.state_dict()
    assert len(sd["state"]) == 167 and float(sd["state"][0]["step"]) == 2.0


def test_flat_adamw_with_8_bit_moments():
    """training.FlatAdamW(state_bits=8) is the list's step on its one flat buffer; its checkpoints are those of 32 bits."""
    from superresolution_amd import optim
    from superresolution_amd.training import FlatAdamW
    sizes = [300, 1, 5000]
    init = [_hash_floats(n, i).cuda() for i, n in enumerate(sizes)]
    ps = [torch.nn.Parameter(x.clone()) for x in init]
    a = FlatAdamW(ps, lr=1e-3, state_bits=8, seed=4)
    one = torch.nn.Parameter(torch.cat(init))
    b = optim.AdamW([one], lr=1e-3, weight_decay=0.01, state_bits=8, seed=4)
    for s in range(3):
        g = _hash_floats(sum(sizes), 20 + s, 1e-2).cuda()
        a.zero_grad()
        a.flat_grad.copy_(g)
        one.grad = g.clone()
        before = [p._version for p in ps]
        a.step()
        b.step()
        assert all(p._version > v for p, v in zip(ps, before))
    assert torch.equal(a.flat, one) and torch.equal(a.moments.exp_avg.view(torch.uint8), b.moments[0].exp_avg.view(torch.uint8))
    sd = a.state_dict()
    assert float(sd["state"][0]["step"]) == 3.0 and sd["state"][2]["exp_avg"].shape == (5000,)
    c = FlatAdamW([torch.nn.Parameter(x.clone()) for x in init], lr=1.0, state_bits=8)
    c.load_state_dict(sd)
    assert c.steps == 3 and c.param_groups[0]["lr"] == 1e-3 and c.moments.steps() == [3]
    assert all(torch.equal(x, y) for x, y in zip(a.moments.read(), c.moments.read()))
    d = FlatAdamW([torch.nn.Parameter(x.clone()) for x in init], lr=1.0)          # 8 -> 32 bits -> torch
    d.load_state_dict(sd)
    assert torch.equal(d.exp_avg, a.moments.read()[0][:sum(sizes)])
    torch.optim.AdamW([torch.nn.Parameter(x.clone()) for x in init], lr=1.0).load_state_dict(d.state_dict())
    e = FlatAdamW([torch.nn.Parameter(x.clone()) for x in init], lr=1.0, state_bits=8)
    e.load_state_dict({"step": 3, "exp_avg": d.exp_avg, "exp_avg_sq": d.exp_avg_sq, "param_groups": sd["param_groups"]})
    assert all(torch.equal(x, y) for x, y in zip(a.moments.read(), e.moments.read()))


def test_fused_training_steps_with_8_bit_moments():
    """PretrainStep and GanStep with state_bits=8: the first step's gradients are those of 32 bits, the update's sizes are alike."""
    from superresolution_amd import Discriminator, Generator
    from superresolution_amd.gan_training import GanStep
    from superresolution_amd.training import PretrainStep
    lr_img, hr = torch.rand(2, 3, 64, 64, device="cuda"), torch.rand(2, 3, 125, 125, device="cuda")
    flats = []
    for bits in (32, 8):
        torch.manual_seed(3)
        gen = Generator().cuda().train()
        step = PretrainStep(gen, lr=1e-4, state_bits=bits)
        start = step.optimizer.flat.clone()
        step.step(lr_img, hr)
        flats.append((start, step.optimizer.flat_grad.clone(), step.optimizer.flat.clone()))
    assert torch.equal(flats[0][1], flats[1][1])
    # From zero moments m = (1 - b1) g and v = (1 - b2) g^2 before they are stored, so the first update is that of 32 bits but for
    # fp32 roundings: 1 - b2 in FlatAdamW's kernel is a float's (5e-5 of it off), which is 3e-5 of an update of lr
    moved = (flats[0][2] - flats[0][0]).abs().max()
    assert float((flats[0][2] - flats[1][2]).abs().max()) <= 1e-4 * float(moved) + 2e-8
    torch.manual_seed(3)
    gan = GanStep(Generator().cuda().train(), Discriminator().cuda().train(), state_bits=8)
    for _ in range(2):
        out = gan.step(lr_img, hr)
    assert all(torch.isfinite(v) for v in out.values()) and gan.opt_g.moments.steps() == [2] and gan.opt_d.moments.steps() == [2]
    assert torch.isfinite(gan.opt_g.flat).all() and torch.isfinite(gan.opt_d.flat).all()
    assert gan.opt_d.moments.nbytes < 0.27 * 8 * gan.opt_d.flat.numel()
