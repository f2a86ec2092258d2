"""CPU checks of what a served decay model keeps: the rotary frequencies on a device, the
slots of a stream, and the workspace of a step of many events."""
import torch

from tencent_recommendation_2025_amd import _lib as L
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


def test_step_workspace_is_linear_in_the_events():
    lib = L.lib()
    assert lib.grk_decay_attn_step_workspace(1 << 23, 0) == 0 == lib.grk_decay_attn_step_workspace(256, 1)
    for n in (257, 8192, 8193, 100_000, 1 << 23):
        assert 8 * n <= lib.grk_decay_attn_step_workspace(n, 1) <= 41 * n + 16384
    need = lib.grk_decay_attn_step_workspace(9000, 1)
    call = lambda ws, size: lib.grk_decay_attn_step(4096, 64, 4096, 64, 4096, 64, L.GRK_F32, 4096, 9000, 1, 64, 1.0, 4096,  # noqa: E731
                                                    9, 4096, L.GRK_I64, None, 4096, 64, ws, size, None)
    for ws, size, word in ((None, need, 'small'), (4096, need - 1, 'small'), (4100, need, 'aligned')):
        assert call(ws, size) == L.GRK_EINVAL and word in lib.grk_last_error().decode()
