"""CPU: calls of the operators on device arrays that are refused before a device is looked at."""
import pytest

from test_q8_refusals import INVALID, P, _loss, _refused


@pytest.mark.parametrize("temperature", [4e36, 3e38])
def test_temperatures_over_which_a_difference_of_logits_overflows(trag, temperature):
    """The widest difference of two finite logits, 6.8e38, is an infinity in 32 bits: over a temperature of 1e36 its exponential
    is e^-680, 0 either way; over 3e38 it is e^-2.3, and the kernels would take it for 0."""
    _refused(trag, INVALID, "temperature", trag.distill_loss_device, **_loss(temperature=temperature))
    _refused(trag, INVALID, "temperature", trag.distill_grad_device, P, 100, 0, 2, 100, P, P, P, 10, temperature, P, P, P + 4096, 100)
