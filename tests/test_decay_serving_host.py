"""CPU checks of what a served decay model keeps: the rotary frequencies on a device, the
slots of a stream, and the workspace of a step of many events."""
import pytest
import torch

from tencent_recommendation_2025_amd import _lib as L
from tencent_recommendation_2025_amd.model import DecayStream, Rotary


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


def stream(n, first, layers=2, hd=3):
    states = [torch.arange(first, first + n).float().mul(10).add(i)[:, None, None, None].repeat(1, 2, hd, hd)
              for i in range(layers)]
    return DecayStream(states, torch.arange(first, first + n))


def users(s):
    """Which user each slot holds, the same in every layer and in the positions."""
    for i, x in enumerate(s.states):
        assert torch.equal(x, (s.position * 10. + i * (s.position > 0))[:, None, None, None].expand_as(x))
    return s.position.tolist()


def test_a_negative_slot_names_no_user():
    s = stream(5, 1)
    s.place(torch.tensor([3, -1, 0]), stream(3, 7))
    assert users(s) == [9, 2, 3, 7, 5]
    s.clear(torch.tensor([-1, 1, -5]))
    assert users(s) == [9, 0, 3, 7, 5]
    s.place([-1, -2], stream(2, 20))
    s.clear([])
    assert users(s) == [9, 0, 3, 7, 5]


def test_slots_in_other_forms():
    s = stream(4, 1)
    s.clear(2)
    s.place(slice(0, 2), stream(2, 7))
    assert users(s) == [7, 8, 0, 4]
    s.place(torch.tensor([False, False, True, False]), stream(1, 9))
    s.clear(torch.tensor([True, False, False, False]))
    assert users(s) == [0, 8, 9, 4]
    s.place(torch.tensor([1, 2, 3, 0], dtype=torch.int32), s)   # its own users, moved round
    assert users(s) == [4, 0, 8, 9]


def test_slots_that_a_stream_does_not_have_are_refused_whole():
    s = stream(4, 1)
    for slots, other in (([0, 4], stream(2, 7)), ([0, 1], stream(3, 7)), ([1, 1], stream(2, 7)),
                         ([0, 1], stream(2, 7, layers=1)), ([0, 1], stream(2, 7, hd=4)), ([0.0, 1.0], stream(2, 7)),
                         (torch.tensor([True, True]), stream(2, 7))):
        with pytest.raises(ValueError):
            s.place(slots, other)
    for slots in (4, [0, 9], torch.tensor([True]), torch.tensor([0.5])):
        with pytest.raises(ValueError):
            s.clear(slots)
    assert users(s) == [1, 2, 3, 4]
