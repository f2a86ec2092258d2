"""CPU checks of what a served decay model keeps: the rotary frequencies on a device, and
the slots of a stream."""
import torch

from tencent_recommendation_2025_amd.model import Rotary


def test_frequencies_first_used_under_inference_mode_can_be_saved_for_a_backward():
    for rot in (Rotary(True, 64), Rotary({'dim': 16, 'layout': 'interleaved'}, 32)):
        for dev in ('meta', 'cpu'):
            positions = torch.zeros(3, dtype=torch.int64, device=dev)
            with torch.inference_mode():
                rot.at(positions)
            freqs = rot.at(positions)[1]
            assert not freqs.is_inference() and freqs.dtype == torch.float64 and freqs.device.type == dev
    with torch.inference_mode():
        made = Rotary(True, 64)
        made.at(torch.zeros(3))
    assert not made.at(torch.zeros(3))[1].is_inference()
