"""Checks of the state-space policy layer's calls that come before anything is on a GPU."""
import pytest
import torch

from pufferlean_amd import device as D

T, B, C, N = 2, 3, 8, 4


def args(*lead):
    f = lambda *s: torch.zeros(*lead, *s)
    return f(C), f(C), torch.zeros(C, N), f(N), f(N)


@pytest.fixture(autouse=True)
def no_call(monkeypatch):
    """A refused call does not reach the library."""
    def call(name, *a):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(D.L, "call", call)


@pytest.mark.parametrize("lead", [(), (1, B), (T, B), (1, T, B)])
def test_step_takes_one_step(lead):
    """x[t:t + 1] of a sequence is [1, B, C], whose rows' stride is not the one that the outputs' rows would be given."""
    with pytest.raises(ValueError, match=r"x must be \[B, C\]"):
        D.ssm_step(*args(*lead), torch.zeros(B, C, N))


@pytest.mark.parametrize("lead", [(), (B,), (1, T, B)])
def test_scan_takes_sequences(lead):
    with pytest.raises(ValueError, match=r"x must be \[T, B, C\]"):
        D.ssm_scan(*args(*lead))
    with pytest.raises(ValueError, match=r"x must be \[T, B, C\]"):
        D.ssm_scan_grad(*args(*lead), torch.zeros(4), torch.zeros(*lead, C))


def test_decays_are_per_channel_and_state():
    x, delta, _, Bm, Cm = args(T, B)
    with pytest.raises(ValueError, match=r"A \[C, N\]"):
        D.ssm_scan(x, delta, torch.zeros(C), Bm, Cm)
