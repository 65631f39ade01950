"""Gradient norm, clipping and ClippedAdamW without a GPU: what the calls refuse, and the argument checks of the C ABI."""
import copy
import ctypes as C
import math

import pytest
import torch

import pde_amd
from pde_amd import _lib


def _params(*grads):
    out = []
    for g in grads:
        p = torch.zeros_like(g).requires_grad_(True)
        p.grad = g
        out.append(p)
    return out


def test_nothing_to_do():
    assert float(pde_amd.get_total_norm([])) == 0.0
    total, each = pde_amd.get_total_norm([], per_tensor=True)
    assert float(total) == 0.0 and each.shape == (0,)
    bare = [torch.zeros(3, requires_grad=True)]
    assert float(pde_amd.clip_grad_norm_(bare, 1.0)) == 0.0      # no gradients
    assert float(pde_amd.clip_grad_norm_([], 1.0, error_if_nonfinite=True)) == 0.0
    assert pde_amd.clip_grads_with_norm_(bare, 1.0, torch.tensor(1.0)) is None


def test_arguments_are_those_of_torch():
    import inspect
    for name in ("get_total_norm", "clip_grad_norm_", "clip_grads_with_norm_"):
        theirs = list(inspect.signature(getattr(torch.nn.utils, name)).parameters.values())
        ours = list(inspect.signature(getattr(pde_amd, name)).parameters.values())[:len(theirs)]
        assert [(p.name, p.default, p.kind) for p in ours] == [(p.name, p.default, p.kind) for p in theirs]


def test_there_is_no_cpu_fallback():
    g = torch.ones(4)
    for call in (lambda: pde_amd.get_total_norm([g]), lambda: pde_amd.clip_grad_norm_(_params(g), 1.0),
                 lambda: pde_amd.clip_grads_with_norm_(_params(g), 1.0, torch.tensor(1.0)),
                 lambda: pde_amd.ClippedAdamW(_params(g)).step()):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    assert torch.equal(g, torch.ones(4))


@pytest.mark.parametrize("norm_type", [0, 3, -1, 0.5, -math.inf, math.nan])
def test_norm_types(norm_type):
    with pytest.raises(ValueError, match="norm_type"):
        pde_amd.get_total_norm([torch.ones(3)], norm_type)
    with pytest.raises(ValueError, match="norm_type"):
        pde_amd.clip_grad_norm_(_params(torch.ones(3)), 1.0, norm_type)


@pytest.mark.parametrize("max_norm", [-1.0, math.nan, -math.inf])
def test_limits(max_norm):
    with pytest.raises(ValueError, match="max_norm"):
        pde_amd.clip_grad_norm_(_params(torch.ones(3)), max_norm)
    with pytest.raises(ValueError, match="max_norm"):
        pde_amd.clip_grads_with_norm_(_params(torch.ones(3)), max_norm, torch.tensor(1.0))
    with pytest.raises(ValueError, match="max_norm"):
        pde_amd.ClippedAdamW(_params(torch.ones(3)), max_norm=max_norm)


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.complex64, torch.float8_e4m3fn])
def test_types(dtype):
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        pde_amd.get_total_norm([torch.ones(3), torch.ones(3).to(dtype)])
    if dtype in (torch.float64, torch.complex64):
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            pde_amd.clip_grad_norm_(_params(torch.ones(3, dtype=dtype)), 1.0)


def test_sparse_tensors_are_refused():
    with pytest.raises(TypeError, match="layout"):
        pde_amd.get_total_norm([torch.eye(3).to_sparse()])


def test_total_norm_of_a_given_norm():
    for bad in (1.0, None):
        with pytest.raises(TypeError, match="total_norm"):
            pde_amd.clip_grads_with_norm_(_params(torch.ones(3)), 1.0, bad)
    with pytest.raises(TypeError, match="total_norm"):
        pde_amd.ClippedAdamW(_params(torch.ones(3)), max_norm=1.0).step(total_norm=2.0)


def test_gradients_that_are_written_must_be_dense_and_apart():
    base = torch.ones(16)
    for grads in ([base[::2]], [torch.ones(1).expand(4)]):
        with pytest.raises(ValueError, match="dense in memory"):
            pde_amd.clip_grad_norm_(_params(*grads), 1.0)
    for grads in ([base, base], [base[:9], base[8:]], [base[8:], torch.ones(2), base[:9]]):
        with pytest.raises(ValueError, match="share memory"):
            pde_amd.clip_grad_norm_(_params(*grads), 1.0)
    p = _params(base)
    with pytest.raises(ValueError, match="share memory"):
        pde_amd.clip_grad_norm_(p + p, 1.0)
    with pytest.raises(RuntimeError, match="HIP device"):      # neighbours, in any order, are fine
        pde_amd.clip_grad_norm_(_params(base[8:], base[:8], base[:0]), 1.0)
    assert torch.equal(base, torch.ones(16))


def test_optimizer_arguments():
    p = [torch.zeros(3, requires_grad=True)]
    for kw in (dict(lr=-1.0), dict(lr=math.nan), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-0.1),
               dict(lr=torch.zeros(2))):
        with pytest.raises(ValueError):
            pde_amd.ClippedAdamW(p, **kw)
    with pytest.raises(ValueError, match="64 parameter groups"):
        pde_amd.ClippedAdamW([dict(params=[torch.zeros(1, requires_grad=True)]) for _ in range(65)])
    opt = pde_amd.ClippedAdamW(p)
    opt.param_groups[0]["lr"] = -0.5      # changed later: checked at the step
    with pytest.raises(ValueError):
        opt.step()


@pytest.mark.parametrize("make, error, match", [
    (lambda: torch.zeros(3, dtype=torch.float16), TypeError, "float32 or bfloat16"),
    (lambda: torch.zeros(3, dtype=torch.float64), TypeError, "float32 or bfloat16"),
    (lambda: torch.zeros(8)[::2], ValueError, "dense in memory"),
])
def test_optimizer_parameters(make, error, match):
    p = make().requires_grad_(True)
    p.grad = torch.zeros(p.shape, dtype=p.dtype)
    with pytest.raises(error, match=match):
        pde_amd.ClippedAdamW([p]).step()


def test_optimizer_parameters_must_not_share_memory():
    base = torch.zeros(16)
    ps = [base[:9].requires_grad_(True), base[8:].requires_grad_(True)]
    with pytest.raises(ValueError, match="share memory"):
        pde_amd.ClippedAdamW(ps).step()


def test_optimizer_state_is_checked():
    p = torch.zeros(4, 3, requires_grad=True)
    good = dict(step=torch.zeros(()), exp_avg=torch.zeros(4, 3), exp_avg_sq=torch.zeros(4, 3))
    for bad, match in ((dict(good, exp_avg=torch.zeros(12)), "laid out"), (dict(good, exp_avg_sq=torch.zeros(3, 4).t()), "laid out"),
                       (dict(good, exp_avg=torch.zeros(4, 3, dtype=torch.bfloat16)), "laid out"), (dict(good, step=torch.zeros(2)), "step counts"),
                       (dict(good, exp_avg_sq=good["exp_avg"]), "share memory"), (dict(step=torch.zeros(())), "must hold")):
        opt = pde_amd.ClippedAdamW([p])
        opt.state[p] = bad
        with pytest.raises(ValueError, match=match):
            opt.step()


def test_state_dict_keeps_float32_state():
    p = torch.randn(4, 3, dtype=torch.bfloat16).requires_grad_(True)
    q = torch.randn(5).requires_grad_(True)
    opt = pde_amd.ClippedAdamW([dict(params=[p], lr=0.5), dict(params=[q])], lr=0.25, betas=(0.8, 0.9), max_norm=2.0, skip_nonfinite=True)
    opt.state[p] = dict(step=torch.tensor(3.0), exp_avg=torch.randn(4, 3), exp_avg_sq=torch.rand(4, 3), master=torch.randn(4, 3))
    other = pde_amd.ClippedAdamW([dict(params=[p]), dict(params=[q])])
    other.load_state_dict(opt.state_dict())
    assert [g["lr"] for g in other.param_groups] == [0.5, 0.25] and other.param_groups[1]["betas"] == (0.8, 0.9)
    assert set(other.state) == {p}
    for k, v in opt.state[p].items():
        w = other.state[p][k]
        assert w.dtype == torch.float32 and torch.equal(w, v) and w.data_ptr() != v.data_ptr()
    with pytest.raises(ValueError):      # another parameter's shape
        pde_amd.ClippedAdamW([dict(params=[torch.zeros(2, requires_grad=True)]), dict(params=[q])]).load_state_dict(opt.state_dict())


def test_c_abi_checks_arguments_before_the_device():
    L = _lib.lib()
    n64, n32 = C.c_int64 * 2, C.c_int32 * 2
    ptrs = (C.c_void_p * 2)(4096, 8192)
    ws = C.c_void_p(1 << 20)
    size = L.pde_amd_multi_workspace_bytes(2)
    assert size > 0 and L.pde_amd_multi_workspace_bytes(-1) == 0
    assert L.pde_amd_multi_workspace_bytes(1000) > size
    total = C.c_void_p(1 << 21)
    ok = (ptrs, n64(3, 4), n32(0, 1), 2)

    def norm(*head, norm_type=2, total=total, ws=ws, size=size):
        return L.pde_amd_multi_norm(*head, norm_type, total, None, ws, size, None)

    assert norm(None, n64(3, 4), n32(0, 1), 2) == -1
    assert norm(*ok[:3], -1) == -1
    assert norm((C.c_void_p * 2)(4096, None), *ok[1:]) == -1
    assert norm(ptrs, n64(3, -4), n32(0, 1), 2) == -1
    assert norm(ptrs, n64(3, 4), n32(0, 3), 2) == -1
    assert norm(ptrs, n64(3, 1 << 62), n32(0, 1), 2) == -2      # ESHAPE
    assert norm(*ok, norm_type=3) == -1 and norm(*ok, total=None) == -1 and norm(*ok, ws=None) == -1
    assert norm(*ok, size=size - 1) == -3                        # EWORKSPACE
    assert L.pde_amd_multi_clip(*ok, -1.0, total, None) == -1 and L.pde_amd_multi_clip(*ok, math.nan, total, None) == -1
    assert L.pde_amd_multi_clip(*ok, 1.0, None, None) == -1
    assert L.pde_amd_multi_norm_clip(*ok, 2, -1.0, total, ws, size, None) == -1

    def table(**kw):
        row = dict(param=4096, exp_avg=8192, exp_avg_sq=12288, master=None, step=64, numel=5, dtype=0, group=0)
        row.update(kw)
        return (_lib.AdamWTensor * 1)(_lib.AdamWTensor(**row))

    group, lr = C.c_void_p(1 << 19), (C.c_float * 1)(1e-3)
    grads = (C.c_void_p * 1)(16384)

    def adamw(t, n=1, groups=group, n_groups=1, lr=lr, max_norm=1.0, total=total, size=size, device=ws):
        return L.pde_amd_multi_adamw(t, device, grads, n, groups, n_groups, lr, max_norm, 0, None, total, ws, size, None)

    for bad in (table(param=None), table(exp_avg=None), table(exp_avg_sq=None), table(step=None), table(numel=-1), table(dtype=2), table(group=1),
                table(group=-1), table(dtype=1)):
        assert adamw(bad) == -1
    assert adamw(table(numel=1 << 62)) == -2 and adamw(table(numel=1 << 40)) == -2
    assert adamw(table(), n=-1) == -1 and adamw(table(), n_groups=0) == -1 and adamw(table(), n_groups=65) == -1
    assert adamw(table(), groups=None) == -1 and adamw(table(), lr=None) == -1 and adamw(table(), max_norm=math.nan) == -1 and adamw(table(), total=None) == -1
    assert adamw(None) == -1 and adamw(table(), device=None) == -1 and adamw(table(), size=8) == -3


def test_struct_layouts():
    assert C.sizeof(_lib.AdamWTensor) == 56 and C.sizeof(_lib.AdamWGroup) == 32


def test_plans_that_a_graph_reads_are_kept(monkeypatch):
    """whatever makes an optimizer describe its tensors anew, a captured description stays"""
    import copy
    import pickle

    from pde_amd import optim

    class Extension:
        def adamw_captured(self, plan):
            return plan.startswith("captured")

    monkeypatch.setattr(optim, "_ext", Extension())
    opt = pde_amd.ClippedAdamW([torch.zeros(3, requires_grad=True)])
    opt._plan = "captured 1"
    opt.load_state_dict(opt.state_dict())
    assert opt._plan is None and opt._captured_plans == ["captured 1"]
    opt._plan = "eager"
    opt.add_param_group(dict(params=[torch.zeros(2, requires_grad=True)]))
    assert opt._plan is None and opt._captured_plans == ["captured 1"]
    opt._plan = "captured 2"
    opt.add_param_group(dict(params=[torch.zeros(2, requires_grad=True)]))
    assert opt._captured_plans == ["captured 1", "captured 2"]
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other._plan is None and other._captured_plans == []


def _with_state(cls, values, dtype=torch.float32):
    """an optimizer over 3-element parameters whose moments hold the values, and the parameters"""
    params = [torch.zeros(3, dtype=dtype, requires_grad=True) for _ in values]
    opt = cls(params)
    for p, x in zip(params, values):
        opt.state[p] = dict(step=torch.tensor(float(x)), exp_avg=torch.full((3,), float(x)), exp_avg_sq=torch.full((3,), float(x)))
    return opt, params


@pytest.mark.parametrize("cls", [torch.optim.AdamW, pde_amd.ClippedAdamW])
def test_load_state_dict_hooks(cls):
    """what a pre-hook returns is loaded, and what a post-hook sets stays"""
    opt, params = _with_state(cls, [1, 2])
    saved = opt.state_dict()

    def swap(o, sd):
        assert o is opt
        return {**sd, "state": {0: sd["state"][1], 1: sd["state"][0]}}

    opt.register_load_state_dict_pre_hook(swap)
    opt.load_state_dict(saved)
    assert [float(opt.state[p]["exp_avg"][0]) for p in params] == [2.0, 1.0]
    assert [float(opt.state[p]["step"]) for p in params] == [2.0, 1.0]

    def nine(o):
        o.state[params[0]]["exp_avg"] = torch.full((3,), 9.0)

    opt.register_load_state_dict_post_hook(nine)
    opt.load_state_dict(saved)
    assert [float(opt.state[p]["exp_avg"][0]) for p in params] == [9.0, 1.0]
    assert len(opt._optimizer_load_state_dict_pre_hooks) == len(opt._optimizer_load_state_dict_post_hooks) == 1


def test_load_state_dict_hooks_see_float32_state():
    """bfloat16 parameters: a post-hook finds the state as it is used afterwards"""
    opt, params = _with_state(pde_amd.ClippedAdamW, [1 + 2 ** -12], torch.bfloat16)
    seen = []
    opt.register_load_state_dict_post_hook(lambda o: seen.append({k: (v.dtype, v) for k, v in o.state[params[0]].items()}))
    opt.load_state_dict(opt.state_dict())
    assert set(seen[0]) == {"step", "exp_avg", "exp_avg_sq", "master"} and all(t is torch.float32 for t, _ in seen[0].values())
    assert float(seen[0]["exp_avg"][1][0]) == 1 + 2 ** -12
    assert all(opt.state[params[0]][k] is v for k, (_, v) in seen[0].items())


@pytest.mark.parametrize("cls", [torch.optim.AdamW, pde_amd.ClippedAdamW])
def test_load_state_dict_leaves_earlier_state_dicts_alone(cls):
    opt, (p, q) = _with_state(cls, [1, 2])
    best, _ = _with_state(cls, [7, 8])
    current = opt.state_dict()
    opt.load_state_dict(best.state_dict())
    assert [float(opt.state[x]["exp_avg"][0]) for x in (p, q)] == [7.0, 8.0]
    opt.load_state_dict(current)
    assert [float(opt.state[x]["exp_avg"][0]) for x in (p, q)] == [1.0, 2.0]
    assert [float(best.state[x]["step"]) for x in best.state] == [7.0, 8.0]


@pytest.mark.parametrize("captured", [False, True])
def test_load_state_dict_of_its_own_tensors(captured, monkeypatch):
    """the tensors of two parameters in each other's place; with a captured step they are written, not replaced"""
    from pde_amd import optim

    class Extension:
        def adamw_captured(self, plan):
            return captured

    monkeypatch.setattr(optim, "_ext", Extension())
    opt, (p, q) = _with_state(pde_amd.ClippedAdamW, [1, 2])
    opt._plan = "a plan"
    before = [dict(opt.state[x]) for x in (p, q)]
    saved = opt.state_dict()
    opt.load_state_dict({**saved, "state": {0: saved["state"][1], 1: saved["state"][0]}})
    for x, value, old in ((p, 2.0, before[0]), (q, 1.0, before[1])):
        for name in ("step", "exp_avg", "exp_avg_sq"):
            assert torch.equal(opt.state[x][name], torch.full_like(opt.state[x][name], value))
            assert (opt.state[x][name] is old[name]) == captured


@pytest.mark.parametrize("bad", [dict(exp_avg=torch.zeros(4)), dict(exp_avg_sq=torch.zeros(3, 1)), dict(step=torch.zeros(2)), dict(exp_avg=None),
                                 dict(step="three")])
def test_load_state_dict_refuses_before_it_changes_anything(bad):
    opt, (p, q) = _with_state(pde_amd.ClippedAdamW, [1, 2])
    other, (r, _) = _with_state(pde_amd.ClippedAdamW, [7, 8])
    saved = copy.deepcopy(other.state_dict())
    saved["state"][1].update(bad)
    saved["param_groups"][0]["lr"] = 0.5
    state = {x: dict(opt.state[x]) for x in (p, q)}
    with pytest.raises(ValueError, match="state"):
        opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 1e-3 and {x: dict(opt.state[x]) for x in (p, q)} == state
    assert [float(opt.state[x]["exp_avg"][0]) for x in (p, q)] == [1.0, 2.0]


def test_load_state_dict_of_other_groups_is_refused_as_in_torch():
    opt, _ = _with_state(pde_amd.ClippedAdamW, [1, 2])
    for cls in (torch.optim.AdamW, pde_amd.ClippedAdamW):
        other, _ = _with_state(cls, [1, 2, 3])
        with pytest.raises(ValueError, match="doesn't match"):
            opt.load_state_dict(other.state_dict())
        assert all(float(opt.state[p]["step"]) in (1.0, 2.0) for p in opt.state)


@pytest.mark.parametrize("cls", [torch.optim.AdamW, pde_amd.ClippedAdamW])
def test_load_state_dict_keeps_entries_of_the_user(cls):
    opt, (p, _) = _with_state(cls, [1, 2])
    opt.state[p].update(average=torch.full((3,), 4.0), note=7)
    other, (q, _) = _with_state(cls, [5, 6])
    other.load_state_dict(opt.state_dict())
    assert set(other.state[q]) == {"step", "exp_avg", "exp_avg_sq", "average", "note"}
    assert torch.equal(other.state[q]["average"], torch.full((3,), 4.0)) and other.state[q]["note"] == 7
    assert float(other.state[q]["exp_avg"][0]) == 1.0


@pytest.mark.parametrize("cls", [torch.optim.AdamW, pde_amd.ClippedAdamW])
def test_step_hooks_get_the_arguments_of_torch(cls, monkeypatch):
    """(optimizer, the call's arguments with the optimizer first, the call's keywords); there is nothing to update here"""
    from pde_amd import optim

    class Extension:
        def adamw_plan(self, *args):
            return "a plan"

        def adamw_step(self, *args):
            return None

    monkeypatch.setattr(optim, "_ext", Extension())
    p = torch.zeros(3, requires_grad=True)
    opt, seen = cls([p]), []
    remove = [opt.register_step_pre_hook(lambda o, args, kwargs: seen.append(("pre", o, args, kwargs))),
              opt.register_step_post_hook(lambda o, args, kwargs: seen.append(("post", o, args, kwargs)))]
    one, two = lambda: 1.0, lambda: 2.0
    for call, args, kwargs, loss in ((lambda: opt.step(), (opt,), {}, None), (lambda: opt.step(None), (opt, None), {}, None),
                                     (lambda: opt.step(one), (opt, one), {}, 1.0), (lambda: opt.step(closure=one), (opt,), {"closure": one}, 1.0)):
        del seen[:]
        assert call() == loss
        assert seen == [("pre", opt, args, kwargs), ("post", opt, args, kwargs)]
    for r in remove:
        r.remove()
    with_hook = lambda result: opt.register_step_pre_hook(lambda o, args, kwargs: result)      # noqa: E731
    for result, loss in ((((opt, two), {}), 2.0), (((opt,), {"closure": two}), 2.0), (((opt, None), {}), None)):
        r = with_hook(result)
        after = opt.register_step_post_hook(lambda o, args, kwargs: seen.append((args, kwargs)))
        del seen[:]
        assert opt.step(one) == loss
        assert seen == [result]      # the changed ones
        r.remove()
        after.remove()
    for result in (5, (opt,), [(opt,), {}], ((opt,), {}, None)):
        r = with_hook(result)
        with pytest.raises(RuntimeError, match="must return None or a tuple"):
            opt.step()
        r.remove()


def test_step_hooks_run_once_for_a_subclass(monkeypatch):
    from pde_amd import optim

    class Extension:
        def adamw_plan(self, *args):
            return "a plan"

        def adamw_step(self, *args):
            return None

    class Mine(pde_amd.ClippedAdamW):
        def step(self, closure=None):
            return super().step(closure)

    monkeypatch.setattr(optim, "_ext", Extension())
    opt, seen = Mine([torch.zeros(3, requires_grad=True)]), []
    opt.register_step_pre_hook(lambda o, args, kwargs: seen.append((args, kwargs)))
    opt.register_step_post_hook(lambda o, args, kwargs: seen.append((args, kwargs)))
    one = lambda: 1.0      # noqa: E731
    assert opt.step(one) == 1.0 and seen == [((opt, one), {})] * 2


def test_step_arguments():
    opt = pde_amd.ClippedAdamW([torch.zeros(3, requires_grad=True)])
    for hook in (False, True):
        for call in (lambda: opt.step(None, None), lambda: opt.step(1, 2, 3), lambda: opt.step(loss=3)):
            with pytest.raises(TypeError, match="argument"):
                call()
        opt.register_step_pre_hook(lambda o, args, kwargs: None)
    import inspect
    assert str(inspect.signature(opt.step)) == "(closure=None, *, total_norm: 'Optional[torch.Tensor]' = None)"


@pytest.mark.parametrize("max_norm", [-1, -0.5, math.nan, -math.inf])
def test_limit_that_is_changed_later(max_norm, monkeypatch):
    from pde_amd import optim

    class Extension:
        limits = []

        def adamw_plan(self, *args):
            return "a plan"

        def adamw_step(self, plan, groups, limit, *args):
            self.limits.append(limit)

    monkeypatch.setattr(optim, "_ext", Extension())
    opt = pde_amd.ClippedAdamW([torch.zeros(3, requires_grad=True)], max_norm=1.0)
    opt.step()
    opt.max_norm = max_norm
    with pytest.raises(ValueError, match="max_norm"):
        opt.step()
    opt.max_norm = 3
    opt.step()
    opt.max_norm = None
    opt.step()
    assert Extension.limits == [1.0, 3.0, -1.0]


def test_settings_of_other_optimizers_are_refused():
    """in a group that is made, and in one that is loaded (torch's Adam adds its weight decay to the gradients)"""
    p = torch.zeros(3, requires_grad=True)
    for bad in (dict(amsgrad=True), dict(maximize=True), dict(decoupled_weight_decay=False)):
        with pytest.raises(ValueError, match="ClippedAdamW has no"):
            pde_amd.ClippedAdamW([dict(params=[p], **bad)])
    pde_amd.ClippedAdamW([dict(params=[p], amsgrad=False, maximize=False, decoupled_weight_decay=True)])
    pde_amd.ClippedAdamW([dict(params=[p], weight_decay=0.0, decoupled_weight_decay=False)])
    opt = pde_amd.ClippedAdamW([p])
    opt.load_state_dict(torch.optim.Adam([p], weight_decay=0.1).state_dict())
    with pytest.raises(ValueError, match="added to the gradients"):
        opt.step()
    opt.load_state_dict(torch.optim.Adam([p]).state_dict())
    with pytest.raises(RuntimeError, match="HIP device"):
        opt.step()


def test_c_abi_checks_the_groups():
    L = _lib.lib()
    groups, device = (_lib.AdamWGroup * 2)(), C.c_void_p(4096)
    for n in (0, -1, 65):
        assert L.pde_amd_multi_adamw_groups(groups, n, device, None) == -1
    assert L.pde_amd_multi_adamw_groups(None, 2, device, None) == -1 and L.pde_amd_multi_adamw_groups(groups, 2, None, None) == -1


def test_tensors_that_do_not_hold_their_values():
    neg, zero = torch._neg_view, torch._efficientzerotensor
    with pytest.raises(ValueError, match="memory of their own"):
        p = torch.zeros(3, requires_grad=True)
        p.grad = zero(3)
        pde_amd.clip_grad_norm_([p], 1.0)
    for p in (neg(torch.ones(3)).requires_grad_(True), zero(3).requires_grad_(True)):
        with pytest.raises(ValueError, match="hold their values"):
            pde_amd.ClippedAdamW([p]).step()
    good = dict(step=torch.zeros(()), exp_avg=torch.zeros(3), exp_avg_sq=torch.zeros(3))
    p = torch.zeros(3, requires_grad=True)
    for name, match in (("exp_avg", "hold its values"), ("exp_avg_sq", "hold its values"), ("step", "step counts")):
        opt = pde_amd.ClippedAdamW([p])
        opt.state[p] = {**good, name: neg(good[name].clone())}
        with pytest.raises(ValueError, match=match):
            opt.step()


def test_lazy_clones_do_not_share_memory():
    base = torch.ones(16)
    with pytest.raises(RuntimeError, match="HIP device"):
        pde_amd.clip_grad_norm_(_params(base, torch._lazy_clone(base)), 1.0)
    p = torch.zeros(16)
    q = torch._lazy_clone(p)
    with pytest.raises(RuntimeError, match="HIP device"):
        pde_amd.ClippedAdamW(_params(base, base.clone())[:0] + [p.requires_grad_(True), q.requires_grad_(True)]).step()


def test_load_state_dict_takes_step_counts_of_any_kind():
    import numpy as np
    opt, (p, _) = _with_state(pde_amd.ClippedAdamW, [1, 2])
    for step in (3, 3.0, np.int64(3), np.float32(3), torch.tensor(3), torch.tensor([3.0], dtype=torch.float64)):
        saved = copy.deepcopy(opt.state_dict())
        saved["state"][0]["step"] = step
        other, (q, _) = _with_state(pde_amd.ClippedAdamW, [5, 6])
        other.load_state_dict(saved)
        assert other.state[q]["step"].dtype == torch.float32 and other.state[q]["step"].shape == () and float(other.state[q]["step"]) == 3.0
