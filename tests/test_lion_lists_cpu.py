"""The launches that a Lion step keeps for the next one, without a GPU: whatever they hold of a parameter, a
gradient or a momentum tensor is compared with the tensors of the step that issues them again.  The device calls are
replaced by a record of their arguments."""
import weakref

import pytest
import torch

from fast_ops_b200.lion import Lion, lion_optimizer


class Recorder:
    """Stands in for the library: the tensor lists of the steps, in order."""

    def __init__(self):
        self.steps = []

    def fo_lion_multi_tensor_step(self, params, grads, moms, numels, n, p_code, _g_code, m_code, *_rest):
        self.steps.append((list(params[:n]), list(grads[:n]), list(moms[:n]), list(numels[:n]), p_code, m_code))
        return 0

    fo_lion_multi_tensor_step_clipped = fo_lion_multi_tensor_step


class NormList:
    """Stands in for the gradient list of the norm."""

    calls = []

    def __init__(self, grads):
        self.numels = [g.numel() for g in grads]
        self.ptrs = [g.data_ptr() for g in grads]

    def launch(self, max_norm):
        NormList.calls.append((self.ptrs, self.numels))
        return torch.tensor(1.0), torch.tensor([1.0])


@pytest.fixture
def record(monkeypatch):
    rec = Recorder()
    check = lion_optimizer._check_triple

    class OnDevice(torch.Tensor):
        """The same tensor, said to be on the device."""
        is_cuda = True

    def check_triple(p, g, m):
        check(p.detach().as_subclass(OnDevice), g, m)

    monkeypatch.setattr(lion_optimizer, "_check_triple", check_triple)
    monkeypatch.setattr(lion_optimizer, "GradList", NormList)
    monkeypatch.setattr(lion_optimizer._lib, "load", lambda: rec)
    monkeypatch.setattr(lion_optimizer._lib, "check", lambda rc: None)
    monkeypatch.setattr(lion_optimizer._lib, "current_stream_ptr", lambda device: 0)
    NormList.calls = []
    return rec


def make(shapes, clip, dtype=torch.float32):
    params = [torch.nn.Parameter(torch.ones(s, dtype=dtype)) for s in shapes]
    for p in params:
        p.grad = torch.ones_like(p)
    return params, Lion(params, max_grad_norm=1.0 if clip else None)


def expect(step, params, opt):
    with_grad = [p for p in params if p.grad is not None]
    moms = [opt.state[p]["exp_avg"] for p in with_grad]
    assert step[0] == [p.data_ptr() for p in with_grad]
    assert step[1] == [p.grad.data_ptr() for p in with_grad]
    assert step[2] == [m.data_ptr() for m in moms]
    assert step[3] == [p.numel() for p in with_grad]
    assert step[4] == lion_optimizer._lib.dtype_code(params[0].dtype)
    assert step[5] == lion_optimizer._lib.dtype_code(moms[0].dtype)


both = pytest.mark.parametrize("clip", [False, True])


@both
def test_lists_are_kept_while_nothing_changes(record, clip, monkeypatch):
    params, opt = make([(7,), (3, 5)], clip)
    opt.step()
    made = []
    monkeypatch.setattr(opt, "_prepare_group", lambda *a: made.append(a))
    opt.step()
    assert not made and record.steps[0] == record.steps[1]
    expect(record.steps[1], params, opt)


@both
@pytest.mark.parametrize("change", ["new tensor", "other type", "new state dict", "state cleared", "swapped", "set data"])
def test_replaced_momentum_is_the_one_that_is_stepped(record, clip, change):
    params, opt = make([(7,), (7,)], clip)
    opt.step()
    old = [opt.state[p]["exp_avg"] for p in params]  # alive, so that no new tensor has their addresses
    if change == "new tensor":
        opt.state[params[1]]["exp_avg"] = torch.full((7,), 0.5)
    elif change == "other type":
        for p in params:
            opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"].bfloat16()
    elif change == "new state dict":
        opt.state[params[0]] = {"exp_avg": torch.zeros(7)}
    elif change == "state cleared":
        opt.state.clear()
    elif change == "swapped":
        opt.state[params[0]]["exp_avg"], opt.state[params[1]]["exp_avg"] = old[1], old[0]
    else:
        old = [m.detach() for m in old]
        opt.state[params[0]]["exp_avg"].data = torch.zeros(7)
    opt.step()
    expect(record.steps[-1], params, opt)
    opt.step()
    expect(record.steps[-1], params, opt)
    assert len(old) == 2


@both
def test_shorter_tensors_at_the_same_addresses(record, clip):
    params, opt = make([(70,), (20,)], clip)
    opt.step()
    p = params[0]
    p.data = p.data[:5]
    p.grad = p.grad[:5]
    with pytest.raises(RuntimeError, match="same number of elements"):
        opt.step()  # the momentum has 70
    opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"][:5]
    opt.step()
    expect(record.steps[-1], params, opt)
    assert record.steps[-1][3] == [5, 20]
    if clip:
        assert NormList.calls[-1][1] == [5, 20]


@both
def test_another_layout_at_the_same_address(record, clip):
    params, opt = make([(6, 6), (20,)], clip)
    opt.step()
    p = params[0]
    p.grad = p.grad.t()
    with pytest.raises(RuntimeError, match="memory layout"):
        opt.step()
    p.data = p.data.t()
    opt.step()
    expect(record.steps[-1], params, opt)


@both
def test_another_type_at_the_same_address(record, clip):
    params, opt = make([(8,), (8,)], clip, torch.float16)
    opt.step()
    for p in params:
        g = p.grad
        p.grad = None
        p.data = p.data.view(torch.bfloat16)
        p.grad = g.view(torch.bfloat16)
    opt.step()
    expect(record.steps[-1], params, opt)


@both
def test_another_parameter_on_the_same_memory(record, clip):
    params, opt = make([(8,), (8,)], clip)
    opt.step()
    new = torch.nn.Parameter(params[0].data)
    new.grad = params[0].grad
    opt.param_groups[0]["params"][0] = new
    opt.step()
    expect(record.steps[-1], [new, params[1]], opt)
    assert opt.state[new]["exp_avg"] is not opt.state[params[0]]["exp_avg"]


@both
def test_gradients_that_come_and_go(record, clip):
    params, opt = make([(8,), (9,), (10,)], clip)
    opt.step()
    kept, params[1].grad = params[1].grad, None
    opt.step()
    expect(record.steps[-1], params, opt)
    params[1].grad = kept
    opt.step()
    expect(record.steps[-1], params, opt)
    assert len(record.steps) == 3


@both
def test_groups_are_looked_at_apart(record, clip):
    params = [torch.nn.Parameter(torch.ones(n)) for n in (4, 5, 6)]
    for p in params:
        p.grad = torch.ones_like(p)
    opt = Lion([{"params": params[:1]}, {"params": params[1:], "lr": 1e-2}], max_grad_norm=1.0 if clip else None)
    opt.step()
    opt.state[params[2]]["exp_avg"] = torch.zeros(6)
    opt.step()
    expect(record.steps[-2], params[:1], opt)
    expect(record.steps[-1], params[1:], opt)
    if clip:
        assert NormList.calls[-1] == ([p.grad.data_ptr() for p in params], [4, 5, 6])


@both
def test_a_replaced_momentum_is_released_at_once(record, clip):
    """As where the state is moved to the host to make room on the device until the next step."""
    params, opt = make([(7,), (7,)], clip)
    opt.step()
    refs = [weakref.ref(opt.state[p]["exp_avg"]) for p in params]
    opt.state[params[0]]["exp_avg"] = opt.state[params[0]]["exp_avg"].double().float()
    del opt.state[params[1]]["exp_avg"]
    assert [r() for r in refs] == [None, None]
    opt.step()
    expect(record.steps[-1], params, opt)
