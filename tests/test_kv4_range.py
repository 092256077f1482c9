"""Arithmetic of the 4-bit cache at the ends of the values that it holds, on the CPU."""
import pytest
import torch

from ridgefill_data_b200.ops import oracle as ops


@pytest.mark.parametrize("exponent", range(-60, 56))
def test_probability_times_step_stays_inside_fp16(exponent):
    """P is at most 2^14 and multiplies a V row's steps in fp16. Rows whose largest value is the largest or the smallest of
    2^exponent's binade, both signs in one group (the largest step that a row can have) or one, beside groups of any smaller
    size."""
    big = torch.tensor([1.0, 2.0 - 2.0 ** -7]) * 2.0 ** exponent
    rows = []
    for top in big:
        for low in (-top, top * 0, top / 2, top):
            y = torch.empty(64)
            y[:32], y[32:] = top, low
            y[1:32:2] = low
            rows += [y, -y, torch.cat((y[:32], y[32:] * 2.0 ** -20))]
    y = torch.stack(rows).bfloat16()
    byte, s, m, c = ops.kv4_quantise(y)
    assert (byte != ops.KV4_MARK).all()
    fit = ops.kv4_fitted(byte, s, m)
    assert (2.0 ** 14 * fit[1] < 65504).all() and (fit[2].abs() <= 2).all() and torch.isfinite(fit[2]).all()
    # the same values: powers of two move between the parts, but for what fp16 cannot hold of a group 2^-24 and less of
    # its row: half a step of 2^-24 in m, and in s over 15 steps
    was, now = ops.kv4_values(byte, s, m, c), ops.kv4_values(*fit, c)
    assert ((was - now).abs() <= 16 * 2.0 ** -25 * torch.pow(2.0, fit[0].double() - 127)[:, None]).all()
    assert torch.equal(was, now) or exponent > 40


def test_a_row_of_zeros_has_the_smallest_size():
    """Beside rows of any size a row of zeros does not raise the running maximum (over score + exponent byte)."""
    y = torch.zeros(4, 64)
    y[1], y[2, 3], y[3, 40] = -0.0, 2.0 ** -40, -(2.0 ** -30)
    byte, _, _ = ops.kv4_fitted(*ops.kv4_quantise(y.bfloat16())[:3])
    assert byte.tolist() == [87, 87, 87, 97]
    byte, s, m = ops.kv4_fitted(torch.tensor([0, 255]), torch.zeros(2, 2), torch.zeros(2, 2))
    assert byte.tolist() == [87, 255] and not s.any() and not m.any()
