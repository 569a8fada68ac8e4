"""What optim.AdamW takes of other optimisers' state dicts; no step is made, no GPU asked."""
from __future__ import annotations

import copy

import pytest

torch = pytest.importorskip("torch")


def stepped(dtype=torch.float32, shape=(6, 4), **flags):
    """torch's optimiser after two steps."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(shape, generator=g).to(dtype).requires_grad_()
    opt = torch.optim.AdamW([x], lr=1e-2, **flags)
    for _ in range(2):
        x.grad = torch.randn(shape, generator=g).to(dtype)
        opt.step()
    return x, opt.state_dict()


@pytest.mark.parametrize("flag", [{"maximize": True}, {"amsgrad": True}, "decoupled_weight_decay", "bits"])
def test_state_dicts_that_ask_for_more_are_refused(flag):
    from sunnynet_b200.optim import AdamW
    x, saved = stepped(**(flag if isinstance(flag, dict) else {}))
    if flag == "decoupled_weight_decay":
        saved["param_groups"][0][flag] = False
    opt = AdamW([x.detach().clone().requires_grad_()], lr=0.5, state_bits=8 if flag == "bits" else 32)
    before = copy.deepcopy(opt.state_dict())
    with pytest.raises(ValueError, match="8 bits" if flag == "bits" else "not supported"):
        opt.load_state_dict(saved)
    assert opt.state_dict() == before


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_states_are_kept_in_float32(dtype):
    from sunnynet_b200.optim import AdamW
    x, saved = stepped(dtype)
    saved["state"][0]["exp_avg"] = saved["state"][0]["exp_avg"].t().contiguous().t()  # of another layout
    opt = AdamW([x])
    opt.load_state_dict(saved)
    s = opt.state[x]
    assert s["step"] == 2 and opt.param_groups[0]["lr"] == 1e-2
    for k in ("exp_avg", "exp_avg_sq"):
        assert s[k].dtype == torch.float32 and s[k].is_contiguous()
        assert torch.equal(s[k], saved["state"][0][k].float())
        assert s[k].data_ptr() != saved["state"][0][k].data_ptr()


def test_without_weight_decay_it_need_not_be_decoupled():
    from sunnynet_b200.optim import AdamW
    x, saved = stepped(weight_decay=0.0)
    saved["param_groups"][0]["decoupled_weight_decay"] = False
    opt = AdamW([x])
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["weight_decay"] == 0.0 and opt.state[x]["step"] == 2
