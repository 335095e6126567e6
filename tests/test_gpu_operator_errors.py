"""GPU: operators on device arrays in a program whose earlier runtime call failed."""
import pytest

pytestmark = pytest.mark.gpu


def test_an_earlier_error_is_named_not_lost(trag):
    """The call clears the runtime's record of the error, which its own launch would be taken for, and says so: its message is
    what trag_last_error has after the call, and a call that found none leaves the message of the last failure alone."""
    import torch
    x = torch.ones((3, 64), device="cuda")
    q8 = torch.empty((3, 64), dtype=torch.int8, device="cuda")
    scale = torch.empty(3, device="cuda")
    args = (x.data_ptr(), 64, 0, 3, 64, q8.data_ptr(), 64, scale.data_ptr(), 0, 0, torch.cuda.current_stream().cuda_stream)
    L = trag.lib()
    with pytest.raises(trag.TragError, match="dim is 0"):
        trag.quantize_q8_device(x.data_ptr(), 64, 0, 3, 0, q8.data_ptr(), 64, scale.data_ptr())
    trag.quantize_q8_device(*args)
    assert b"dim is 0" in L.trag_last_error()
    assert L.hipSetDevice(9999) != 0
    trag.quantize_q8_device(*args)
    message = L.trag_last_error()
    assert b"trag_quantize_q8_device" in message and b"earlier" in message and b"invalid device ordinal" in message, message
    torch.cuda.synchronize()
    assert (q8 == 127).all()
