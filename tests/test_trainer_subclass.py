"""A trainer whose subclass builds its own module."""
import pytest
import torch

from artemis_amd.train import HeadTrainer


class Own(HeadTrainer):
    @staticmethod
    def build(num_features, fused):
        return torch.nn.Linear(num_features, 1 + fused)


def test_build_of_two_arguments():
    tr = Own(torch.device("cpu"), num_features=5)
    assert tr.module.weight.shape == (2, 5) and isinstance(tr.optimizer, torch.optim.Adamax)


def test_a_choice_that_build_does_not_know_is_not_dropped():
    with pytest.raises(TypeError):
        Own(torch.device("cpu"), num_features=5, encoder_ops="hip")
