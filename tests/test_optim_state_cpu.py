"""CPU: what an optimizer over a list of tensors does around its steps -- groups that fail to be added, checkpoints and their
hooks, parameters that change under it -- with the moments in host memory (nothing is launched), and the tags by which the modules
know that weights have changed."""
import gc

import numpy as np
import pytest
import torch


@pytest.fixture
def optim(monkeypatch):
    """The module, with the check for a ROCm device put aside."""
    from superresolution_amd import optim
    monkeypatch.setattr(optim, "_one_device", lambda ts, what: torch.device("cpu"))
    return optim


def _filled(optim, params, **kw):
    """An optimizer that has taken three steps, its moments told apart by element."""
    opt = optim.AdamW(params, lr=1e-2, **kw)
    for mo in opt.moments:
        mo.set_steps([3] * len(mo.numels))
        mo.exp_avg.copy_(torch.arange(mo.total) + 1.0)
        mo.exp_avg_sq.copy_(torch.arange(mo.total) + 0.5)
    return opt


def test_a_group_whose_moments_do_not_fit_is_not_added(optim, monkeypatch):
    p, q = (torch.nn.Parameter(torch.ones(40)) for _ in range(2))
    opt = optim.AdamW([p], lr=1e-2)

    def full(*a):
        raise torch.OutOfMemoryError("no memory for them")
    monkeypatch.setattr(optim, "Moments", full)
    with pytest.raises(torch.OutOfMemoryError):
        opt.add_param_group(dict(params=[q]))
    assert len(opt.param_groups) == len(opt.moments) == 1
    monkeypatch.undo()
    monkeypatch.setattr(optim, "_one_device", lambda ts, what: torch.device("cpu"))
    opt.add_param_group(dict(params=[q]))                              # (and can be added afterwards)
    assert len(opt.param_groups) == len(opt.moments) == 2


@pytest.mark.parametrize("change", ["popped", "appended"])
def test_groups_without_moments_of_their_own_are_refused(optim, change):
    """A group put into the list, or taken out of it, by hand: the others would step with its moments, or it would not step."""
    p, q = (torch.nn.Parameter(torch.ones(40)) for _ in range(2))
    opt = _filled(optim, [dict(params=[p]), dict(params=[q])])
    sd = opt.state_dict()
    if change == "popped":
        opt.param_groups.pop(0)
    else:
        opt.param_groups.append(dict(opt.param_groups[1], params=[torch.nn.Parameter(torch.ones(40))]))
    for call in (opt.step, opt.state_dict, lambda: opt.load_state_dict(sd)):
        with pytest.raises(RuntimeError, match="add_param_group"):
            call()


def test_state_dict_hooks_are_called(optim):
    opt = _filled(optim, [torch.nn.Parameter(torch.ones(40))])
    seen = []

    def post(o, sd):
        seen.append("post")
        return {**sd, "extra": 7}
    handles = [opt.register_state_dict_pre_hook(lambda o: seen.append("pre")), opt.register_state_dict_post_hook(post)]
    sd = opt.state_dict()
    assert seen == ["pre", "post"] and sd["extra"] == 7
    for h in handles:
        h.remove()
    assert "extra" not in opt.state_dict() and len(seen) == 2

    def rename(o, given):
        seen.append("load pre")
        return {"state": given["mine"], "param_groups": given["param_groups"]}
    opt.register_load_state_dict_pre_hook(rename)
    opt.register_load_state_dict_post_hook(lambda o: seen.append(o.moments[0].steps()))
    given = {"mine": {0: {"step": torch.tensor(5.0), "exp_avg": torch.full((40,), 2.0), "exp_avg_sq": torch.ones(40)}},
             "param_groups": sd["param_groups"]}
    opt.load_state_dict(given)
    assert seen[2:] == ["load pre", [5]] and set(given) == {"mine", "param_groups"}
    assert torch.equal(opt.moments[0].exp_avg[:40], torch.full((40,), 2.0))


@pytest.mark.parametrize("first, then", [(torch.contiguous_format, torch.channels_last), (torch.channels_last, torch.contiguous_format)])
def test_checkpoints_of_a_parameter_of_another_memory_order(optim, first, then):
    """The moments keep the order that the parameter was added with; a checkpoint has them by element all the same."""
    w = torch.randn(6, 5, 3, 3)
    p = torch.nn.Parameter(w.clone(memory_format=first))
    opt = _filled(optim, [p])
    want = {k: v.clone() for k, v in opt.state_dict()["state"][0].items()}
    p.data = p.data.contiguous(memory_format=then)
    got = opt.state_dict()["state"][0]
    assert all(torch.equal(got[k], want[k]) for k in want)
    before = opt.moments[0].exp_avg.clone()
    opt.moments[0].exp_avg.zero_()
    opt.load_state_dict(opt.state_dict() | {"state": {0: want}})
    assert torch.equal(opt.moments[0].exp_avg[:270], before[:270])


def test_checkpoints_of_a_parameter_of_another_size_are_refused(optim):
    p, q = (torch.nn.Parameter(torch.ones(n)) for n in (40, 40))
    opt = _filled(optim, [p, q])
    sd = opt.state_dict()
    p.data = torch.ones(64)                                             # (its padded part and the next tensor's first moments)
    with pytest.raises(RuntimeError, match="number of elements"):
        opt.state_dict()
    with pytest.raises((RuntimeError, ValueError), match="number of elements|entries"):
        opt.load_state_dict(sd)
    p.data = torch.ones(5, 8)                                           # (another shape of the same memory)
    assert torch.equal(opt.state_dict()["state"][0]["exp_avg"].view(-1), sd["state"][0]["exp_avg"])
    opt.param_groups[0]["params"].pop()
    with pytest.raises(RuntimeError, match="number of elements"):
        opt.state_dict()


@pytest.mark.parametrize("break_it", [lambda st: st.pop("step"), lambda st: st.pop("exp_avg_sq"), lambda st: st.update(exp_avg=torch.ones(3)),
                                      lambda st: st.update(step="three")])
def test_a_checkpoint_that_is_refused_changes_nothing(optim, break_it):
    opt = _filled(optim, [dict(params=[torch.nn.Parameter(torch.ones(40))]), dict(params=[torch.nn.Parameter(torch.ones(33))])])
    sd = opt.state_dict()
    for st in sd["state"].values():
        st["exp_avg"] = st["exp_avg"] * 2.0
        st["step"] = torch.tensor(9.0)
    for g in sd["param_groups"]:
        g["lr"] = 1.0
    break_it(sd["state"][1])
    kept = [mo.exp_avg.clone() for mo in opt.moments]
    with pytest.raises((KeyError, ValueError)):
        opt.load_state_dict(sd)
    assert all(torch.equal(a, mo.exp_avg) and mo.steps() == [3] for a, mo in zip(kept, opt.moments))
    assert [g["lr"] for g in opt.param_groups] == [1e-2, 1e-2]


def test_tags_of_parameters_that_a_graph_writes():
    """A tag is the same again while nothing has written the tensor; never, where a replay may have, unseen by the host."""
    from superresolution_amd import versions

    class Owner:
        pass
    a, b = torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(3))
    assert versions.tag(a) == versions.tag(a) != versions.tag(b)
    was = versions.tag(a)
    with torch.no_grad():
        a.mul_(2.0)
    assert versions.tag(a) != was
    one, two = Owner(), Owner()
    versions.note_captured([a], one)
    versions.note_captured([a], two)
    assert versions.tag(a) != versions.tag(a) and versions.tag(b) == versions.tag(b)
    del one
    gc.collect()
    assert versions.tag(a) != versions.tag(a)
    last = versions.tag(a)
    del two                                                              # no graph may be replayed after its optimizer
    gc.collect()
    assert versions.tag(a) == versions.tag(a) != last


def test_modules_go_by_the_tags():
    """The signatures by which Generator and Discriminator know that their uploaded weights are still the parameters'."""
    from superresolution_amd import Discriminator, Generator, versions

    class Owner:
        pass
    for module in (Generator(), Discriminator()):
        assert module._signature() == module._signature()
        owner = Owner()
        versions.note_captured(list(module.parameters())[-1:], owner)
        assert module._signature() != module._signature()
        del owner
        gc.collect()
        assert module._signature() == module._signature()


def test_group_seeds_differ():
    """Same-position elements of two groups round with bits of their own; the first group's are the seed's."""
    from oracle import optim_ref as R
    from superresolution_amd import optim
    seeds = [optim.group_seed(5, k) for k in range(100)]
    assert seeds[0] == 5 and len(set(seeds)) == 100 and all(0 <= s < 1 << 32 for s in seeds)
    # 4,096 positions: equal bits by chance in 1 of 65,536 each, so that 8 or more of them have probability under 1e-14
    bits = [R.random_bits(np.arange(4096), s, 1) for s in seeds[:4]]
    for i in range(4):
        for j in range(i):
            assert all((x == y).sum() < 8 for x, y in zip(bits[i], bits[j]))
