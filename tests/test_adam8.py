"""AdamW8bit's arguments, its place among the optimizers a runner can be given, and its state's types, without a GPU."""
import argparse

import pytest
import torch


def test_the_option_names_it():
    from pfeife.optim import AdamW8bit as through_the_alias
    from pfeife_amd.optim import AdamW8bit
    from pfeife_amd.option import PipeOption, get_optimizer_cls

    assert through_the_alias is AdamW8bit and get_optimizer_cls("AdamW8bit") is AdamW8bit
    args = PipeOption.add_arguments(argparse.ArgumentParser()).parse_args(["--optimizer_type", "adamw8bit"])
    option = PipeOption.from_args(args)
    opt = get_optimizer_cls(option.optimizer_type)([torch.nn.Parameter(torch.zeros(3))], **option.optimizer_kwargs)
    assert type(opt) is AdamW8bit and opt.param_groups[0]["lr"] == 1e-3


@pytest.mark.parametrize("kwargs", [{"lr": -1.0}, {"eps": -1e-8}, {"weight_decay": -0.1}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"min_8bit_size": -1}])
def test_bad_values(kwargs):
    from pfeife_amd.optim import AdamW8bit

    with pytest.raises(ValueError, match=next(iter(kwargs))):
        AdamW8bit([torch.nn.Parameter(torch.zeros(3))], **kwargs)


def test_refusals():
    from pfeife_amd.optim import AdamW8bit

    for dtype in (torch.float16, torch.bfloat16, torch.float64):
        with pytest.raises(RuntimeError, match="fp32"):
            AdamW8bit([torch.nn.Parameter(torch.zeros(3, dtype=dtype))])
    p = torch.nn.Parameter(torch.zeros(3))
    opt = AdamW8bit([p])
    opt.step()                    # (nothing has a gradient)
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="GPU"):
        opt.step()


def test_loading_keeps_the_codes_types():
    from pfeife_amd.optim import AdamW8bit

    p, q = (torch.nn.Parameter(torch.zeros(5000)) for _ in range(2))
    opt = AdamW8bit([p])
    st = opt._init_state(p, opt.param_groups[0])
    assert st["exp_avg"].dtype == st["exp_avg_sq_root"].dtype == torch.float8_e4m3fn and st["exp_avg_scale"].shape == (20,)
    st["exp_avg"].view(torch.uint8).fill_(0x41)
    st["exp_avg_scale"].fill_(0.5)
    other = AdamW8bit([q])
    other.load_state_dict(opt.state_dict())
    assert other.state[q]["step"] == 0
    for key, t in ((k, t) for k, t in st.items() if k != "step"):
        mine = other.state[q][key]
        assert mine.dtype == t.dtype and torch.equal(mine.float(), t.float()) and mine.data_ptr() != t.data_ptr(), key
