"""What rollout.py settles without a device, where it is easily got wrong."""
import torch

from fp4_post_b200 import rollout


def test_frequencies_are_plain_tensors_whatever_mode_they_are_made_in():
    with torch.inference_mode():
        made = rollout.Rotary(64, device="cpu")
    assert not made.turns.is_inference() and torch.equal(made.turns, rollout.Rotary(64, device="cpu").turns)
