"""GPU: lists that take several launches, lists of both parameter types, and other memory orders, step by step against the 64-bit
oracle."""
import numpy as np
import pytest
import torch

from oracle import optim_ref as R
from test_gpu_optim import _check, _f64, _hash_floats, _make, _refs, _sync_ref

pytestmark = pytest.mark.gpu

# 1,050 tensors of up to three chunks of 4,096 elements (some empty): four launches of a step, four of a norm
LONG = [(7919 * i) % 9001 if i % 50 else 0 for i in range(1050)]



@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_of_lists_that_take_several_launches(bits, dt, clip):
    from superresolution_amd import optim
    (flat, views), (gflat, gviews) = _make(LONG, dt, dt, seed=7)
    before = flat.clone()
    params = [torch.nn.Parameter(v) for v in views]
    opt = optim.AdamW(params, lr=3e-3, betas=(0.9, 0.99), weight_decay=0.05, state_bits=bits, seed=5, max_grad_norm=clip)
    refs = _refs(opt, params, bits, seed=5)
    for s in range(2):
        gflat.copy_(_hash_floats(gflat.numel(), 100 + s, 1e-2).to(gflat.dtype))
        for p, g in zip(params, gviews):
            p.grad = g
        opt.step()
        coef = 1.0
        if clip:
            want = np.sqrt(sum((_f64(g) ** 2).sum() for g in gviews))
            assert abs(float(opt.last_grad_norm) - want) <= 1.01 * R.U24 * want
            coef = float(np.float32(min(1.0, clip / (float(opt.last_grad_norm) + 1e-6))))
            assert coef < 1.0
        _check(opt, params, refs, [r.step(_f64(g), coef) for r, g in zip(refs, gviews)])
        _sync_ref(params, refs, opt.moments[0])
    inside = torch.zeros_like(flat, dtype=torch.bool)
    at = 1
    for k in LONG:
        inside[at:at + k] = True
        at += k + 1
    assert torch.equal(flat[~inside], before[~inside])
    assert opt.moments[0].steps() == [2 if k else 0 for k in LONG]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_and_clipping_of_lists_that_take_several_launches(dt):
    from superresolution_amd import optim
    (flat, views), _ = _make(LONG, dt, dt, seed=50)
    params = [torch.nn.Parameter(torch.zeros_like(v)) for v in views]
    for p, v in zip(params, views):
        p.grad = v
    before = flat.clone()
    want = np.sqrt(sum((_f64(v) ** 2).sum() for v in views))
    assert abs(float(optim.total_norm(views)) - want) <= 1.01 * R.U24 * want
    norm = optim.clip_grad_norm_(params, 0.7)
    assert abs(float(norm) - want) <= 1.01 * R.U24 * want
    coef = min(1.0, 0.7 / (float(norm) + 1e-6))
    assert coef < 1.0
    inside = torch.zeros_like(flat, dtype=torch.bool)
    at = 1
    for k in LONG:
        inside[at:at + k] = True
        at += k + 1
    assert torch.equal(flat[~inside], before[~inside])
    # the coefficient to fp32, the product to fp32, then half a step of the gradients' type (fp16: of its subnormals at least)
    x, half = before[inside].double() * coef, torch.finfo(dt).eps / 2
    assert ((flat[inside].double() - x).abs() <= x.abs() * (2 * R.U24 + half * (1 + 2 * R.U24)) + (2.0 ** -25 if dt == torch.float16 else 0.0)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_lists_of_both_parameter_types(bits):
    """fp32 and bf16 parameters in turn, in one optimizer, gradients of each one's type."""
    from superresolution_amd import optim
    sizes = [5, 4096, 4097, 0, 9000, 33, 1, 12289, 64, 31]
    dts = [torch.float32, torch.bfloat16]
    params = [torch.nn.Parameter(_hash_floats(n + 1, 60 + i, 0.1).to(dts[i % 2]).cuda()[1:]) for i, n in enumerate(sizes)]
    opt = optim.AdamW(params, lr=3e-3, weight_decay=0.05, state_bits=bits, seed=8, max_grad_norm=2.0)
    refs = _refs(opt, params, bits, seed=8)
    for s in range(3):
        for i, p in enumerate(params):
            p.grad = _hash_floats(p.numel(), 300 + 10 * s + i, 1e-2).to(p.dtype).cuda()
        opt.step()
        norm = np.sqrt(sum((_f64(p.grad) ** 2).sum() for p in params))
        assert abs(float(opt.last_grad_norm) - norm) <= 1.01 * R.U24 * norm
        coef = float(np.float32(min(1.0, 2.0 / (float(opt.last_grad_norm) + 1e-6))))
        _check(opt, params, refs, [r.step(_f64(p.grad), coef) for r, p in zip(refs, params)])
        _sync_ref(params, refs, opt.moments[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_channels_last_parameters(bits):
    """Moments and random bits go by the parameter's memory; the gradient is in C order."""
    from superresolution_amd import optim
    w = torch.randn(6, 5, 3, 3, generator=torch.Generator().manual_seed(1)).cuda()
    p = torch.nn.Parameter(w.clone(memory_format=torch.channels_last))
    opt = optim.AdamW([p], lr=1e-2, state_bits=bits)

    def in_memory(t):
        return t.detach().permute(0, 2, 3, 1).reshape(-1)
    ref = R.AdamWRef(_f64(in_memory(p)), bits=bits, lr=1e-2)
    for s in range(3):
        p.grad = _hash_floats(p.numel(), 40 + s, 1e-2).view(p.shape).cuda()
        opt.step()
        assert p.is_contiguous(memory_format=torch.channels_last)
        _check(opt, [in_memory(p)], [ref], [ref.step(_f64(in_memory(p.grad)))])
        _sync_ref([in_memory(p)], [ref], opt.moments[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_expanded_gradients(bits):
    from superresolution_amd import optim
    p = torch.nn.Parameter(_hash_floats(4100, 1).view(41, 100).cuda())
    opt = optim.AdamW([p], lr=1e-2, state_bits=bits)
    (ref,) = _refs(opt, [p], bits)
    p.grad = _hash_floats(100, 2, 1e-2).cuda().expand(41, 100)
    assert p.grad.stride() == (0, 1)
    opt.step()
    _check(opt, [p], [ref], [ref.step(_f64(p.grad))])


def test_32_bit_moments_of_parameters_without_gradients_at_every_turn():
    from superresolution_amd import optim
    (_, views), (_, gviews) = _make([100, 5000, 7], torch.float32, torch.float32, seed=2)
    params = [torch.nn.Parameter(v) for v in views]
    opt = optim.AdamW(params, lr=1e-2)
    refs, mo = _refs(opt, params, 32), opt.moments[0]
    for turn in ((0,), (0, 2), (1,), (0, 1, 2), ()):
        for i, p in enumerate(params):
            p.grad = gviews[i] if i in turn else None
        before = [(p.detach().clone(), mo.exp_avg[a:a + n].clone(), mo.exp_avg_sq[a:a + n].clone())
                  for p, a, n in zip(params, mo.offsets, mo.numels)]
        opt.step()
        for i, (p, a, n) in enumerate(zip(params, mo.offsets, mo.numels)):
            got = (p.detach(), mo.exp_avg[a:a + n], mo.exp_avg_sq[a:a + n])
            if i not in turn:
                assert all(torch.equal(x, y) for x, y in zip(got, before[i]))
                continue
            tols = refs[i].step(_f64(gviews[i]))
            for x, want, tol in zip(got, (refs[i].p, refs[i].m, refs[i].v), tols):
                assert (np.abs(_f64(x) - want) <= tol).all(), (turn, i)
        _sync_ref(params, refs, mo)
    assert mo.steps() == [3, 2, 2]


def test_the_reference_loop_with_8_bit_moments_against_the_oracle():
    """Three iterations of the pre-train loop's body on the drop-in generator, clipped: every code, scale and parameter as the
    oracle has them from the same gradients, and parameters that have moved."""
    from superresolution_amd import Generator, optim, pixel_loss
    torch.manual_seed(0)
    gen = Generator().cuda().train()
    params = list(gen.parameters())
    opt = optim.AdamW(params, lr=1e-4, state_bits=8, max_grad_norm=0.05)
    refs = _refs(opt, params, 8)
    lr_img, hr = torch.rand(2, 3, 64, 64, device="cuda"), torch.rand(2, 3, 125, 125, device="cuda")
    for _ in range(3):
        start = [p.detach().clone() for p in params]
        loss = pixel_loss(gen(lr_img), hr)
        opt.zero_grad()
        loss.backward()
        opt.step()
        coef = float(np.float32(min(1.0, 0.05 / (float(opt.last_grad_norm) + 1e-6))))
        assert coef < 1.0
        _check(opt, params, refs, [r.step(_f64(p.grad), coef) for r, p in zip(refs, params)])
        _sync_ref(params, refs, opt.moments[0])
        assert all(not torch.equal(a, p) for a, p in zip(start, params) if p.grad.any())
