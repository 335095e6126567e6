"""CPU: calls of the operators on device arrays that are refused before a device is looked at."""
import pytest

from test_q8_refusals import INVALID, P, _loss, _norm, _refused


@pytest.mark.parametrize("temperature", [4e36, 3e38])
def test_temperatures_over_which_a_difference_of_logits_overflows(trag, temperature):
    """The widest difference of two finite logits, 6.8e38, is an infinity in 32 bits: over a temperature of 1e36 its exponential
    is e^-680, 0 either way; over 3e38 it is e^-2.3, and the kernels would take it for 0."""
    _refused(trag, INVALID, "temperature", trag.distill_loss_device, **_loss(temperature=temperature))
    _refused(trag, INVALID, "temperature", trag.distill_grad_device, P, 100, 0, 2, 100, P, P, P, 10, temperature, P, P, P + 4096, 100)


@pytest.mark.parametrize("value", [1 << 32, (1 << 32) + 2, -1])
def test_counts_that_do_not_fit_the_interface(trag, value):
    """Counts are 32 bits in the C interface: 2^32 rows must not be taken for none, nor -1 for 2^32 - 1."""
    for name in ("dtype", "n_rows", "dim"):
        _refused(trag, INVALID, "32 bits", trag.rmsnorm_q8_device, **_norm(**{name: value}))
    for at in (2, 3, 4):
        args = [P, 1 << 40, 0, 2, 64, P, 1 << 40, P]
        args[at] = value
        _refused(trag, INVALID, "32 bits", trag.quantize_q8_device, *args)
    for at in (6, 7, 8, 9):
        args = [P, 1 << 40, P, P, 1 << 40, P, 4, 4, 64, 0, P, 1 << 40]
        args[at] = value
        _refused(trag, INVALID, "32 bits", trag.matmul_q8_device, *args)
    for name in ("dtype", "n_rows", "n_cols", "k"):
        _refused(trag, INVALID, "32 bits", trag.distill_loss_device, **_loss(**{name: value, "logits_stride": 1 << 40, "grad_stride": 1 << 40}))
    for at in (2, 3, 4, 8):
        args = [P, 1 << 40, 0, 2, 100, P, P, P, 10, 1.0, P, P, P + 4096, 1 << 40]
        args[at] = value
        _refused(trag, INVALID, "32 bits", trag.distill_grad_device, *args)
    for args in ((value, 100_000), (4, value)):
        _refused(trag, INVALID, "32 bits", trag.distill_work_bytes, *args)
    _refused(trag, INVALID, "32 bits", trag.VectorStore.quantize_device, None, 0, value, P, 64, P)
