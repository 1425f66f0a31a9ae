"""CPU: argument checks of the optimizer operators over a list of tensors (C ABI and Python mirror), and the 64-bit oracle
against torch.optim.AdamW."""
import ctypes
from array import array

import numpy as np
import pytest
import torch

from oracle import optim_ref as R


def _lib():
    from superresolution_amd import _lib as L
    return L


def _adamw(numel=(64,), offset=(0,), p=(4096,), g=(8192,), pd=(0,), gd=(0,), count=None, **over):
    """srgen_adamw_many with addresses that are never followed: every call here is refused before anything is launched."""
    L = _lib()
    mo = L.srgen_moments(32, 0, 1 << 20, 1 << 21, None, None, 1 << 22, 1 << 23, 64, 1)
    args = L.srgen_adamw_args(1e-3, 0.9, 0.999, 1e-8, 0.0)
    for k, v in over.items():
        setattr(mo if hasattr(mo, k) else args, k, v)
    a = [array("Q", p), array("Q", g), array("Q", numel), array("Q", offset), array("i", pd), array("i", gd)]
    rc = L.lib().srgen_adamw_many(len(numel) if count is None else count, *[x.buffer_info()[0] for x in a], mo, args, None)
    return rc, L.lib().srgen_last_error().decode()


@pytest.mark.parametrize("kw, rc, text", [
    (dict(count=-1), -1, "count"),
    (dict(p=(0,)), -1, "parameter 0 is NULL"),
    (dict(p=(4097,)), -1, "not aligned"),
    (dict(p=(4098,)), -1, "not aligned"),
    (dict(g=(8193,), gd=(1,)), -1, "not aligned"),
    (dict(pd=(2,)), -6, "type 2"),
    (dict(gd=(2,)), -6, "type 2"),
    (dict(pd=(7,)), -6, "type 7"),
    (dict(bits=16), -6, "16 bits"),
    (dict(offset=(16,)), -1, "offset"),
    (dict(offset=(32,)), -1, "end behind their buffer"),
    (dict(numel=(65,)), -1, "end behind their buffer"),
    (dict(chunks=0), -1, "chunks"),
    (dict(chunks=2), -1, "chunks"),
    (dict(p=(1 << 50,)), -6, "48 bits"),
    (dict(table=None), -1, "NULL moments"),
    (dict(table=(1 << 23) + 8), -1, "misaligned"),
    (dict(numel=(1 << 40,)), -6, "elements"),
    (dict(m=None), -1, "NULL moments"),
    (dict(step=None), -1, "NULL moments"),
    (dict(bits=8), -1, "NULL moments"),                      # no scales
    (dict(m=(1 << 20) + 4), -1, "misaligned"),
    (dict(lr=-1.0), -1, "lr"),
    (dict(lr=float("nan")), -1, "lr"),
    (dict(beta1=1.0), -1, "betas"),
    (dict(beta2=-0.1), -1, "betas"),
    (dict(eps=-1.0), -1, "eps"),
    (dict(weight_decay=float("nan")), -1, "weight decay"),
    (dict(norm_coef2=64, max_norm=0.0), -1, "max_norm"),
    (dict(norm_coef2=64, max_norm=1.0, grad_mul=64), -1, "one of the two"),
    (dict(norm_coef2=66, max_norm=1.0), -1, "norm_coef2"),
    (dict(norm_coef2=64, max_norm=1.0), -1, "scratch"),
    (dict(norm_coef2=64, max_norm=1.0, norm_scratch=256, norm_scratch_bytes=4), -5, "scratch"),
])
def test_adamw_many_refuses(kw, rc, text):
    got, msg = _adamw(**kw)
    assert got == rc and text in msg, (got, msg)


def test_empty_lists_are_allowed():
    assert _adamw(numel=(), offset=(), p=(), g=(), pd=(), gd=(), chunks=0)[0] == 0
    assert _adamw(numel=(0, 0), offset=(0, 0), p=(0, 0), g=(0, 0), pd=(0, 0), gd=(0, 0), chunks=0)[0] == 0
    L = _lib().lib()
    z, d = array("Q", [0]), array("i", [0])
    assert L.srgen_scale_many(1, z.buffer_info()[0], z.buffer_info()[0], d.buffer_info()[0], 64, None) == 0
    assert L.srgen_moments_pack(None, None, 0, None, None, None, None, None) == 0


def test_counters_and_scratch():
    L = _lib().lib()
    n = array("Q", [0, 1, 4096, 4097])
    out = ctypes.c_uint64()
    assert L.srgen_adamw_chunk_count(4, n.buffer_info()[0], ctypes.byref(out)) == 0 and out.value == 0 + 1 + 1 + 2
    off, table = array("Q", [0, 0, 32, 4128]), array("I", bytes(64))
    assert L.srgen_adamw_chunk_table(4, n.buffer_info()[0], off.buffer_info()[0], table.buffer_info()[0], 4) == 0
    assert list(table) == [1, 0, 0, 1, 2, 0, 1, 4096, 3, 0, 129, 4096, 3, 1, 257, 1]
    assert L.srgen_adamw_chunk_table(4, n.buffer_info()[0], off.buffer_info()[0], table.buffer_info()[0], 3) == -1
    off[1] = 16
    assert L.srgen_adamw_chunk_table(4, n.buffer_info()[0], off.buffer_info()[0], table.buffer_info()[0], 4) == -1
    b = ctypes.c_size_t()
    assert L.srgen_total_norm_scratch_bytes(4, n.buffer_info()[0], ctypes.byref(b)) == 0 and b.value >= 4 * 8
    assert L.srgen_adamw_chunk_count(4, None, ctypes.byref(out)) == -1
    assert L.srgen_total_norm_scratch_bytes(-1, n.buffer_info()[0], ctypes.byref(b)) == -1


def test_norm_scale_pack_refuse():
    L = _lib().lib()
    kept = []                                        # (the lists have to outlive the calls)

    def ad(a):
        kept.append(a)
        return a.buffer_info()[0]

    n, d, p = array("Q", [8192]), array("i", [0]), array("Q", [4096])
    assert L.srgen_total_norm(1, ad(p), ad(n), ad(d), 1.0, None, 256, 256, None) == -1            # no output
    assert L.srgen_total_norm(1, ad(p), ad(n), ad(d), 1.0, 64, None, 256, None) == -1             # no scratch
    assert L.srgen_total_norm(1, ad(p), ad(n), ad(d), 1.0, 64, 260, 256, None) == -1              # misaligned scratch
    assert L.srgen_total_norm(1, ad(p), ad(n), ad(d), 1.0, 64, 256, 8, None) == -5                # too small
    assert L.srgen_total_norm(1, ad(p), ad(n), ad(array("i", [3])), 1.0, 64, 256, 256, None) == -6
    assert L.srgen_scale_many(1, ad(p), ad(n), ad(d), None, None) == -1
    assert L.srgen_scale_many(1, ad(array("Q", [4097])), ad(n), ad(array("i", [2])), 64, None) == -1
    assert L.srgen_moments_pack(256, 256, 4, None, 256, 256, 256, None) == -1
    assert L.srgen_moments_pack(258, 256, 4, 256, 256, 256, 256, None) == -1
    assert L.srgen_moments_unpack(256, 256, 257, 256, 256, 256, 4, None) == -1


def test_python_refuses_cpu_tensors_and_bad_arguments():
    from superresolution_amd import optim
    p = torch.nn.Parameter(torch.zeros(8))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        optim.AdamW([p])
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([p], state_bits=4)
    with pytest.raises(ValueError, match="max_grad_norm"):
        optim.AdamW([p], max_grad_norm=0.0)
    with pytest.raises(ValueError, match="beta parameter at index 1"):
        optim.AdamW([p], betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="learning rate"):
        optim.AdamW([p], lr=-1.0)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        optim.total_norm([torch.zeros(3)])
    with pytest.raises(NotImplementedError, match="L2"):
        optim.clip_grad_norm_([p], 1.0, norm_type=1.0)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        optim.pack_moments(torch.zeros(3), torch.zeros(3))
    # no gradients: as torch
    assert float(optim.clip_grad_norm_([p], 1.0)) == 0.0 and float(optim.grad_norm(torch.nn.Linear(2, 2))) == 0.0


def test_dense_and_overlap_checks():
    from superresolution_amd.optim import _dense, _no_overlap
    t = torch.zeros(4, 6, 5, 5)
    assert _dense(t) and _dense(t.to(memory_format=torch.channels_last)) and _dense(t.permute(3, 1, 0, 2)) and _dense(torch.zeros(3, 0))
    assert not _dense(t[:, ::2]) and not _dense(torch.zeros(1).expand(4)) and not _dense(t[:, :5])
    assert _dense(t[1:3]) and _dense(torch.zeros(()))
    _no_overlap(array("Q", [0, 16, 8, 4]), array("Q", [2, 2, 4, 0]), array("i", [0, 0, 1, 0]), "x")
    with pytest.raises(RuntimeError, match="share memory"):
        _no_overlap(array("Q", [0, 4]), array("Q", [2, 2]), array("i", [0, 0]), "x")
    with pytest.raises(RuntimeError, match="share memory"):
        _no_overlap(array("Q", [64, 64]), array("Q", [1, 1]), array("i", [1, 2]), "x")
    with pytest.raises(ValueError):
        _no_overlap(array("Q", [64, 128]), array("Q", [1]), array("i", [1, 2]), "x")


def test_oracle_against_torch_adamw():
    """Four steps of the 64-bit oracle against torch.optim.AdamW on float64 tensors: the same formula, so 1e-12 of the values."""
    torch.manual_seed(0)
    p = torch.randn(50, dtype=torch.float64)
    q = torch.nn.Parameter(p.clone())
    ref = R.AdamWRef(p.numpy(), lr=3e-3, betas=(0.8, 0.95), eps=1e-7, wd=0.1)
    opt = torch.optim.AdamW([q], lr=3e-3, betas=(0.8, 0.95), eps=1e-7, weight_decay=0.1)
    for _ in range(4):
        q.grad = torch.randn(50, dtype=torch.float64)
        ref.step(q.grad.numpy())
        opt.step()
    np.testing.assert_allclose(ref.p, q.detach().numpy(), rtol=1e-12, atol=1e-15)
    np.testing.assert_allclose(ref.v, opt.state[q]["exp_avg_sq"].numpy(), rtol=1e-12)


def test_oracle_e4m3_is_torchs_format_and_unbiased():
    """Values are e4m3 numbers (torch's own table of the 256 codes), rounded to a neighbour, and right on average."""
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    table = np.unique(table[np.isfinite(table)])
    rng = np.random.RandomState(1)
    x = (rng.randn(64 * 32) * np.exp(2 * rng.randn(64 * 32))).astype(np.float32)
    mean = np.zeros(x.size)
    rounds = 400
    for s in range(rounds):
        v, e = R.e4m3(x, R.random_bits(np.arange(x.size), 11, s)[0], False)
        assert np.isin(v, table).all()
        mean += R.values(v, e) / rounds
    y = np.abs(x.astype(np.float64)) / np.repeat(e, 32)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(y, 1e-9))), -6) - 3) * np.repeat(e, 32)
    # the mean of 400 roundings of variance <= step^2 / 4: five standard deviations, over 2,048 elements (p < 2e-3), plus the
    # 2^-16 of a step that 16 random bits do not resolve
    assert (np.abs(mean - x) <= step * (5 * 0.5 / np.sqrt(rounds) + 2.0 ** -16)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_update_refuses_other_lists(bits):
    """Arrays that are not one entry for each tensor, or of another type, would be read past their end."""
    from array import array
    from superresolution_amd import _lib, optim
    mo = optim.Moments([5, 40], bits, torch.device("cpu"))
    q, i, args = array("Q", [0, 0]), array("i", [0, 0]), _lib.srgen_adamw_args()
    for k in range(4):
        lists = [q, q, i, i]
        lists[k] = lists[k][:1]
        with pytest.raises(ValueError, match="2 tensors"):
            mo.update(*lists, args, 0)
        lists[k] = array("I", [0, 0]) if k < 2 else array("h", [0, 0])
        with pytest.raises(TypeError, match="type codes"):
            mo.update(*lists, args, 0)


def test_a_shorter_parameter_list_wants_a_closer_look():
    """The arrays still hold the addresses of a parameter that was taken out of its group: not to be launched with."""
    from array import array
    from superresolution_amd import _tensorlist
    q, i = (lambda n: array("Q", [7] * n)), (lambda n: array("i", [0] * n))
    assert _tensorlist.params([], 0, q(1), q(1), i(1), q(1), i(1)) == -1
    assert _tensorlist.params([], 0, q(0), q(0), i(0), q(0), i(0)) == 0


def _wrapper(n, dtype=torch.float32):
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls):
            return torch.Tensor._make_wrapper_subclass(cls, (n,), dtype=dtype, device="cuda:0")

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise NotImplementedError(str(func))

    return Wrapper()


def test_tensors_without_memory_are_refused():
    """A subclass that wraps another tensor has address 0, which stands for a tensor that is left out."""
    from superresolution_amd import optim
    for f in (optim.total_norm, lambda ts: optim.AdamW(ts)):
        with pytest.raises(RuntimeError, match="no memory of its own"):
            f([_wrapper(5)])


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_write_refuses_other_buffers(bits):
    from superresolution_amd import optim
    mo = optim.Moments([5, 40], bits, torch.device("cpu"))
    good = torch.zeros(mo.total)
    for bad in (torch.zeros(mo.total + 32), torch.zeros(1), good.double(), torch.zeros(2 * mo.total)[::2], good.to("meta")):
        for pair in ((bad, good), (good, bad)):
            with pytest.raises(RuntimeError, match="Moments.write"):
                mo.write(*pair)
