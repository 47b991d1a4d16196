"""Copies of the AdamW optimizers that are taken before their first step."""

import copy
import pickle

import pytest
import torch

from muonium_amd import AdamW, AdamWFp8


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
@pytest.mark.parametrize("block", [64, 256, 2048])
def test_a_copy_keeps_the_block_size(copied, block):
    p = torch.nn.Parameter(torch.zeros(8192))
    made = copied(AdamWFp8([p], lr=0.5, betas=(0.8, 0.9), block_size=block))
    q = made.param_groups[0]["params"][0]
    assert made.block_size == block and made._block(q) == block
    assert made.param_groups[0]["lr"] == 0.5 and made.param_groups[0]["betas"] == (0.8, 0.9)
    state = made._init_state(q)
    assert state["exp_avg"].block_size == block and state["exp_avg_sq_root"].scale.shape == (8192 // block,)


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_a_copy_of_adamw(copied):
    made = copied(AdamW([torch.nn.Parameter(torch.zeros(8192))], lr=0.5))
    state = made._init_state(made.param_groups[0]["params"][0])
    assert made.param_groups[0]["lr"] == 0.5 and state["exp_avg"].dtype == torch.float32


def test_a_copy_without_the_block_size_has_the_default():
    made = AdamWFp8([torch.nn.Parameter(torch.zeros(8192))], block_size=64)
    state = made.__getstate__()
    del state["block_size"]
    other = AdamWFp8.__new__(AdamWFp8)
    other.__setstate__(state)
    assert other.block_size == 256
