"""A step that would make or move its state while a graph is captured is refused: every replay would do it
again, and start from it. Whether a graph is captured is pretended here."""

import pytest
import torch

from muonium_amd import AdamW, AdamWFp8
from muonium_amd.optim import adamw


@pytest.fixture
def capturing(monkeypatch):
    monkeypatch.setattr(adamw, "_capturing", lambda p: True)


def param(*shape):
    p = torch.nn.Parameter(torch.zeros(shape))
    p.grad = torch.zeros(shape)
    return p


@pytest.mark.parametrize("kind", [AdamW, AdamWFp8])
def test_a_captured_step_makes_no_state(kind, capturing):
    p = param(4096)
    opt = kind([p])
    with pytest.raises(RuntimeError, match="no state while a graph is captured"):
        opt.step()
    assert not opt.state[p]


def test_a_captured_step_lays_no_moment_out_anew(monkeypatch):
    p = param(64, 128)
    opt = AdamW([p])
    opt._init_state(p)
    for name in ("exp_avg", "exp_avg_sq"):
        turned = torch.ones(128, 64).t()
        opt.state[p][name] = turned
        monkeypatch.setattr(adamw, "_capturing", lambda p: True)
        with pytest.raises(RuntimeError, match="unlike its parameter while a graph is captured"):
            opt.step()
        assert opt.state[p][name] is turned
        monkeypatch.setattr(adamw, "_capturing", lambda p: False)
        assert list(opt._collect([p]))  # and outside of one it is
        assert opt.state[p][name].stride() == p.stride() and (opt.state[p][name] == 1).all()


def test_a_captured_step_moves_no_counter(capturing):
    p = param(8)
    opt = AdamW([p])
    opt.state[p].update(step=torch.zeros((), device="meta"), exp_avg=torch.zeros(8), exp_avg_sq=torch.zeros(8))
    with pytest.raises(RuntimeError, match="another device while a graph is captured"):
        opt.step()
