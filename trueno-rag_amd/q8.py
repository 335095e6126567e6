"""Operators on device arrays: rows of 8-bit integers with scales, their product, and distillation of
scores from a teacher's best k (include/trag.h, "Operators on a caller's device arrays"). Like
`fusion.rrf_device`, every argument named *_ptr is a device address (0: none), strides count elements,
`stream` is a hipStream_t as an integer; calls are enqueued and return at once."""
import enum

from . import _abi


class DType(enum.IntEnum):
    """trag_dtype of include/trag.h."""
    F32 = 0
    F16 = 1
    BF16 = 2


def _too_large():
    """Counts and codes are 32 bits in the C interface, which would take 2^32 rows for none."""
    raise _abi.TragError(_abi.INVALID_ARG, "a count does not fit 32 bits")


def rmsnorm_q8_device(x_ptr: int, x_stride: int, residual_ptr: int, residual_stride: int, weight_ptr: int, eps: float,
                      dtype: int, n_rows: int, dim: int, sum_ptr: int, sum_stride: int, q8_ptr: int, q8_stride: int,
                      scale_ptr: int, values_ptr: int = 0, values_stride: int = 0, stream: int = 0) -> None:
    """Residual addition, root-mean-square norm and 8-bit rows with a scale each (trag_rmsnorm_q8_device)."""
    if (dtype | n_rows | dim) >> 32:
        _too_large()
    _abi.check(_abi.lib().trag_rmsnorm_q8_device(x_ptr, x_stride, residual_ptr, residual_stride, weight_ptr, eps, dtype,
                                                 n_rows, dim, sum_ptr, sum_stride, q8_ptr, q8_stride, scale_ptr,
                                                 values_ptr, values_stride, stream))


def quantize_q8_device(x_ptr: int, x_stride: int, dtype: int, n_rows: int, dim: int, q8_ptr: int, q8_stride: int,
                       scale_ptr: int, values_ptr: int = 0, values_stride: int = 0, stream: int = 0) -> None:
    """Rows as they are to 8-bit rows with a scale each (trag_quantize_q8_device)."""
    if (dtype | n_rows | dim) >> 32:
        _too_large()
    _abi.check(_abi.lib().trag_quantize_q8_device(x_ptr, x_stride, dtype, n_rows, dim, q8_ptr, q8_stride, scale_ptr,
                                                  values_ptr, values_stride, stream))


def matmul_q8_device(a_ptr: int, a_stride: int, a_scale_ptr: int, b_ptr: int, b_stride: int, b_scale_ptr: int, m: int,
                     n: int, dim: int, out_dtype: int, out_ptr: int, out_stride: int, stream: int = 0) -> None:
    """out (m, n) = (a b^T) a_scale b_scale for 8-bit rows a (m, dim) and b (n, dim) (trag_matmul_q8_device)."""
    if (m | n | dim | out_dtype) >> 32:
        _too_large()
    _abi.check(_abi.lib().trag_matmul_q8_device(a_ptr, a_stride, a_scale_ptr, b_ptr, b_stride, b_scale_ptr, m, n, dim,
                                                out_dtype, out_ptr, out_stride, stream))


def distill_work_bytes(n_rows: int, n_cols: int) -> int:
    """Bytes of workspace distill_loss_device needs for rows of this many columns."""
    if (n_rows | n_cols) >> 32:
        _too_large()
    return int(_abi.lib().trag_distill_work_bytes(n_rows, n_cols))


def distill_loss_device(logits_ptr: int, logits_stride: int, dtype: int, n_rows: int, n_cols: int, ids_ptr: int,
                        teacher_ptr: int, counts_ptr: int, k: int, temperature: float, loss_ptr: int, norm_ptr: int,
                        row_weight_ptr: int = 0, grad_ptr: int = 0, grad_stride: int = 0, work_ptr: int = 0,
                        work_bytes: int = 0, stream: int = 0) -> None:
    """Loss of every row against its teacher list, and, with grad_ptr, the gradient of the weighted
    sum of the losses (trag_distill_loss_device)."""
    if (dtype | n_rows | n_cols | k) >> 32:
        _too_large()
    _abi.check(_abi.lib().trag_distill_loss_device(logits_ptr, logits_stride, dtype, n_rows, n_cols, ids_ptr, teacher_ptr,
                                                   counts_ptr, k, temperature, loss_ptr, norm_ptr, row_weight_ptr,
                                                   grad_ptr, grad_stride, work_ptr, work_bytes, stream))


def distill_grad_device(logits_ptr: int, logits_stride: int, dtype: int, n_rows: int, n_cols: int, ids_ptr: int,
                        teacher_ptr: int, counts_ptr: int, k: int, temperature: float, norm_ptr: int,
                        row_weight_ptr: int, grad_ptr: int, grad_stride: int, stream: int = 0) -> None:
    """The gradient alone, from the norm the forward call saved (trag_distill_grad_device)."""
    if (dtype | n_rows | n_cols | k) >> 32:
        _too_large()
    _abi.check(_abi.lib().trag_distill_grad_device(logits_ptr, logits_stride, dtype, n_rows, n_cols, ids_ptr, teacher_ptr,
                                                   counts_ptr, k, temperature, norm_ptr, row_weight_ptr, grad_ptr,
                                                   grad_stride, stream))
