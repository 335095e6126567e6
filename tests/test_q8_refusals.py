"""CPU: what the operators on device arrays refuse, before they look at a device; and that without a GPU
a well-formed call fails loudly."""
import pytest

P = 1 << 20            # stands for a device address (never read: every call here is refused)
INVALID, UNSUPPORTED = 5, 6


def _refused(trag, status, words, fn, *args, **kw):
    with pytest.raises(trag.TragError) as e:
        fn(*args, **kw)
    assert e.value.status == status and words in str(e.value)


def _norm(**kw):
    a = dict(x_ptr=P, x_stride=64, residual_ptr=P, residual_stride=64, weight_ptr=P, eps=1e-6, dtype=0, n_rows=2, dim=64, sum_ptr=P + 4096,
             sum_stride=64, q8_ptr=P, q8_stride=64, scale_ptr=P, values_ptr=0, values_stride=0)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(dtype=3), "element type"), (dict(dim=0), "dim is 0"), (dict(x_ptr=0), "null"), (dict(q8_ptr=0), "null"), (dict(scale_ptr=0), "null"),
    (dict(x_ptr=P + 2), "aligned"), (dict(residual_ptr=P + 1), "aligned"), (dict(weight_ptr=P + 2), "aligned"), (dict(sum_ptr=P + 2), "aligned"),
    (dict(values_ptr=P + 2, values_stride=64), "aligned"), (dict(scale_ptr=P + 2), "aligned"), (dict(dtype=1, x_ptr=P + 1), "aligned"),
    (dict(x_stride=63), "stride"), (dict(residual_stride=63), "stride"), (dict(sum_stride=1), "stride"), (dict(q8_stride=63), "stride"),
    (dict(values_ptr=P + 8192, values_stride=63), "stride"), (dict(sum_ptr=P, sum_stride=80), "in place"), (dict(values_ptr=P, values_stride=65), "in place"),
    (dict(values_ptr=P + 4096, values_stride=64), "share"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps")])
def test_norm_refusals(trag, change, words):
    _refused(trag, INVALID, words, trag.rmsnorm_q8_device, **_norm(**change))


def test_norm_limits(trag):
    _refused(trag, UNSUPPORTED, "2^30", trag.rmsnorm_q8_device, **_norm(dim=(1 << 30) + 1))
    trag.rmsnorm_q8_device(**_norm(n_rows=0, x_ptr=0))          # no rows: nothing is looked at


@pytest.mark.parametrize("args,words", [
    ((P, 64, 7, 2, 64, P, 64, P), "element type"), ((P, 64, 0, 2, 0, P, 64, P), "dim is 0"), ((0, 64, 0, 2, 64, P, 64, P), "null"),
    ((P, 32, 0, 2, 64, P, 64, P), "stride"), ((P, 64, 0, 2, 64, P, 63, P), "stride"), ((P + 1, 64, 2, 2, 64, P, 64, P), "aligned")])
def test_quantize_refusals(trag, args, words):
    _refused(trag, INVALID, words, trag.quantize_q8_device, *args)


@pytest.mark.parametrize("args,words", [
    ((P, 64, P, P, 64, P, 4, 4, 64, 3, P, 4), "element type"), ((P, 64, P, P, 64, P, 4, 4, 0, 0, P, 4), "dim is 0"),
    ((0, 64, P, P, 64, P, 4, 4, 64, 0, P, 4), "null"), ((P, 64, P, 0, 64, P, 4, 4, 64, 0, P, 4), "null"), ((P, 64, P, P, 64, P, 4, 4, 64, 0, 0, 4), "null"),
    ((P, 63, P, P, 64, P, 4, 4, 64, 0, P, 4), "stride"), ((P, 64, P, P, 63, P, 4, 4, 64, 0, P, 4), "stride"), ((P, 64, P, P, 64, P, 4, 4, 64, 0, P, 3), "stride"),
    ((P, 64, P + 1, P, 64, P, 4, 4, 64, 0, P, 4), "aligned"), ((P, 64, P, P, 64, P + 2, 4, 4, 64, 0, P, 4), "aligned"),
    ((P, 64, P, P, 64, P, 4, 4, 64, 0, P + 2, 4), "aligned"), ((P, 64, P, P, 64, P, 4, 4, 64, 1, P + 1, 4), "aligned")])
def test_product_refusals(trag, args, words):
    _refused(trag, INVALID, words, trag.matmul_q8_device, *args)


def test_product_limits(trag):
    _refused(trag, UNSUPPORTED, "131071", trag.matmul_q8_device, P, 131072, P, P, 131072, P, 4, 4, 131072, 0, P, 4)
    big = 1 << 29
    _refused(trag, UNSUPPORTED, "2^22 tiles", trag.matmul_q8_device, P, 64, P, P, 64, P, 200, big, 64, 0, P, big)
    trag.matmul_q8_device(0, 0, 0, 0, 0, 0, 0, 4, 64, 0, 0, 0)
    trag.matmul_q8_device(0, 0, 0, 0, 0, 0, 4, 0, 64, 0, 0, 0)


def _loss(**kw):
    a = dict(logits_ptr=P, logits_stride=100, dtype=0, n_rows=2, n_cols=100, ids_ptr=P, teacher_ptr=P, counts_ptr=P, k=10, temperature=1.0, loss_ptr=P,
             norm_ptr=P, row_weight_ptr=P, grad_ptr=P + 4096, grad_stride=100, work_ptr=0, work_bytes=0)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(dtype=3), "element type"), (dict(n_cols=0), "0 columns"), (dict(logits_ptr=0), "null"), (dict(ids_ptr=0), "null"), (dict(teacher_ptr=0), "null"),
    (dict(loss_ptr=0), "null"), (dict(norm_ptr=0), "null"), (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(temperature=1e-40), "temperature"), (dict(temperature=float("inf")), "temperature"), (dict(logits_stride=99), "stride"),
    (dict(grad_stride=99), "stride"), (dict(grad_ptr=P, grad_stride=101), "in place"), (dict(logits_ptr=P + 2), "aligned"), (dict(ids_ptr=P + 2), "aligned"),
    (dict(norm_ptr=P + 1), "aligned"), (dict(grad_ptr=P + 2), "aligned"), (dict(n_cols=80000, logits_stride=80000, grad_stride=80000), "workspace"),
    (dict(n_cols=80000, logits_stride=80000, grad_stride=80000, work_ptr=P, work_bytes=8), "workspace")])
def test_distill_refusals(trag, change, words):
    _refused(trag, INVALID, words, trag.distill_loss_device, **_loss(**change))


def test_distill_limits(trag):
    _refused(trag, UNSUPPORTED, "1024", trag.distill_loss_device, **_loss(k=1025))
    trag.distill_loss_device(**_loss(n_rows=0, logits_ptr=0))
    a = (P, 100, 0, 2, 100, P, P, P, 10, 1.0)
    _refused(trag, INVALID, "null", trag.distill_grad_device, *a, 0, P, P, 100)
    _refused(trag, INVALID, "null", trag.distill_grad_device, *a, P, P, 0, 100)
    _refused(trag, INVALID, "stride", trag.distill_grad_device, *a, P, P, P + 4096, 99)
    assert trag.distill_work_bytes(5, 65536) == 0 and trag.distill_work_bytes(0, 1 << 20) == 0
    for rows, cols in ((1, 65537), (4096, 100_000), (64, 1_000_000), (1, (1 << 32) - 1), (1 << 20, 1 << 20)):
        need = trag.distill_work_bytes(rows, cols)
        assert need >= 8 * rows * -(-cols // 16384) and need % 8 == 0


def test_without_a_gpu_calls_fail_loudly(trag):
    import torch
    if torch.cuda.is_available():
        return
    for fn, args in ((trag.rmsnorm_q8_device, _norm()), (trag.distill_loss_device, _loss())):
        with pytest.raises(trag.TragError) as e:
            fn(**args)
        assert e.value.status == 3 and "no HIP device" in str(e.value)
    with pytest.raises(trag.TragError, match="no HIP device"):
        trag.matmul_q8_device(P, 64, P, P, 64, P, 4, 4, 64, 0, P, 4)
