"""GPU: distillation from a teacher's best k (trag_distill_loss_device, trag_distill_grad_device) against the
formula in 64 bits and against differences, and the 8-bit first stage as it is used: encoder states ->
8-bit queries -> scores over an 8-bit corpus -> loss against the lists of an exact search.

Tolerances, derived. With E the largest |z - max| / T * log2(e) of a row (at most 150: smaller terms are 0), an
exponential of the kernel is off by the roundings of z - max, of the two products and of the hardware's exp2:
(4 E + 4) 2^-24 relative; a thread adds up to 64 of them (64 roundings), the rest is summed in 64 bits. So the
logarithm of the sum is off by at most S = (4 E + 70) 2^-24, the loss by T^2 S plus its own rounding, and a
gradient by |weight T| (q (2 S + 8 2^-24) + p 8 2^-24) plus the rounding to its type, eps / 2 relative, or half the
type's smallest step. The hardware's exp2 has no subnormal results: an exponential below 2^-126 is 0, which a gradient
feels as at most |weight T| 2^-126 (its divisor, the sum, is at least 1)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

CODE = {"f32": 0, "f16": 1, "bf16": 2}
U = 2.0 ** -24
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def _torch():
    import torch
    return torch


def _types():
    torch = _torch()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _teacher64(ids, teacher, counts, k, cols, temp):
    torch = _torch()
    there = torch.arange(k, device="cuda")[None] < counts[:, None].clamp(max=k)
    there &= (ids.long() >= 0) & (ids.long() < cols)
    t = torch.where(there, teacher.double() / temp, -float("inf"))
    some = (t > -float("inf")).any(1)
    p = torch.where(some[:, None], torch.softmax(torch.where(some[:, None], t, 0.0), 1), 0.0)
    return p, there, some


def _reference(z, ids, teacher, counts, temp, weight):
    """loss, norm, gradient in 64 bits, and the tolerances of loss and gradient"""
    torch = _torch()
    rows, cols = z.shape
    k = ids.shape[1]
    zd = z.double()
    top = zd.amax(1, keepdim=True)
    ln = torch.logsumexp((zd - top) / temp, 1, keepdim=True)
    logq = (zd - top) / temp - ln
    q = logq.exp()
    p, there, some = _teacher64(ids, teacher, counts, k, cols, temp)
    safe = torch.where(there, ids.long(), 0)
    terms = torch.where(p > 0, p * (torch.log(p) - logq.gather(1, safe)), 0.0)
    loss = temp ** 2 * terms.sum(1)
    q = torch.where(some[:, None], q, 0.0)
    dense = torch.zeros_like(zd).scatter_add_(1, safe, p)
    g = weight.double()[:, None] * temp
    grad = g * (q - dense)
    e = torch.where(zd > -float("inf"), (zd - top).abs() / temp * 1.4427, 0.0).amax(1).clamp(max=150.0)
    s = (4 * e + 70) * U
    tol_loss = temp ** 2 * s + 2 * U * loss.abs()
    tol_grad = g.abs() * (q * (2 * s + 8 * U)[:, None] + dense * 8 * U + 2.0 ** -126)
    return loss, torch.cat([top, ln], 1), grad, tol_loss, s, tol_grad


def _filled(values, dt, pad, offset):
    torch = _torch()
    rows, cols = values.shape
    buf = torch.full((rows * (cols + pad) + offset + 64,), 77.0, dtype=dt, device="cuda")
    v = buf[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    v.copy_(values)
    return buf, v


def _loss(trag, t, z, ids, teacher, counts, temp, weight, loss, norm, grad=None, stream=None, work=None):
    torch = _torch()
    rows, cols = z.shape
    need = trag.distill_work_bytes(rows, cols)
    if work is None:
        work = torch.empty(max(need, 4), dtype=torch.uint8, device="cuda")
    trag.distill_loss_device(z.data_ptr(), z.stride(0), CODE[t], rows, cols, ids.data_ptr() if ids.numel() else 0, teacher.data_ptr() if ids.numel() else 0,
                             0 if counts is None else counts.data_ptr(), ids.shape[1], temp, loss.data_ptr(), norm.data_ptr(),
                             0 if weight is None else weight.data_ptr(), 0 if grad is None else grad.data_ptr(),
                             0 if grad is None else grad.stride(0), work.data_ptr(), work.numel(),
                             (stream or torch.cuda.current_stream()).cuda_stream)
    return work


def _grad(trag, t, z, ids, teacher, counts, temp, norm, weight, grad, stream=None):
    torch = _torch()
    rows, cols = z.shape
    trag.distill_grad_device(z.data_ptr(), z.stride(0), CODE[t], rows, cols, ids.data_ptr() if ids.numel() else 0, teacher.data_ptr() if ids.numel() else 0,
                             0 if counts is None else counts.data_ptr(), ids.shape[1], temp, norm.data_ptr(),
                             0 if weight is None else weight.data_ptr(), grad.data_ptr(), grad.stride(0),
                             (stream or torch.cuda.current_stream()).cuda_stream)


def _case(rows, cols, k, seed, spread=2.0):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = spread * torch.randn((rows, cols), generator=g, device="cuda")
    ids = torch.randint(0, cols, (rows, k), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)     # (repeats among them)
    teacher = torch.sort(2 * torch.randn((rows, k), generator=g, device="cuda"), 1, descending=True).values.contiguous() if k else torch.empty((rows, 0), device="cuda")
    counts = torch.randint(0, k + 3, (rows,), generator=g, device="cuda").to(torch.int32)                      # (0, and more than k, among them)
    weight = torch.randn(rows, generator=g, device="cuda")
    return z, ids, teacher, counts, weight


def _check_grad(got, want, tol, t):
    torch = _torch()
    eps = torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs()
    assert (off <= tol + eps * (want.abs() + tol) + TINY[t]).all(), (off.max().item(), (off - tol - eps * want.abs()).max().item())


COLS = [1, 2, 7, 8, 9, 100, 1021, 2047, 2048, 2049, 4096, 4100, 8192, 8193, 16384, 16390, 32000, 32768, 32769, 40000, 65536, 65537, 70001, 152064]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", COLS)
def test_loss_and_gradient_match_the_formula(trag, t, cols):
    torch = _torch()
    dt = _types()[t]
    for rows, k, pad, offset, temp in ((1, 1, 0, 0, 1.0), (9, 10, 3, 1, 2.0), (4, 100, 0, 0, 0.5), (3, 1000, 8, 8, 3.0)):
        z0, ids, teacher, counts, weight = _case(rows, cols, k, cols + rows)
        zb, z = _filled(z0, dt, pad, offset)
        gb, grad = _filled(torch.full((rows, cols), 5.0, device="cuda"), dt, pad + 2, offset)
        want_loss, want_norm, want_grad, tol_loss, s, tol_grad = _reference(z, ids, teacher, counts, temp, weight)
        loss = torch.full((rows + 1,), 77.0, device="cuda")
        norm = torch.full((rows + 1, 2), 77.0, device="cuda")
        _loss(trag, t, z, ids, teacher, counts, temp, weight, loss, norm, grad)
        assert ((loss[:rows].double() - want_loss).abs() <= tol_loss + 2.0 ** -149).all(), (loss, want_loss)
        assert torch.equal(norm[:rows, 0].double(), want_norm[:, 0])
        assert ((norm[:rows, 1].double() - want_norm[:, 1]).abs() <= s + 2 * U * want_norm[:, 1].abs()).all()
        _check_grad(grad, want_grad, tol_grad, t)
        # the loss alone gives the same bits; the gradient alone the same gradient
        alone, norm2 = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda")
        _loss(trag, t, z, ids, teacher, counts, temp, None, alone, norm2)
        assert torch.equal(alone, loss[:rows]) and torch.equal(norm2, norm[:rows])
        gb2, grad2 = _filled(torch.full((rows, cols), 5.0, device="cuda"), dt, pad, offset)
        _grad(trag, t, z, ids, teacher, counts, temp, norm2, weight, grad2)
        # (the saved logarithm has been rounded to 32 bits)
        _check_grad(grad2, want_grad, tol_grad + want_grad.abs() * 0 + (weight.double()[:, None] * temp).abs() * want_norm[:, 1:].abs() * 2 * U, t)
        # in place
        z2b, z2 = _filled(z0, dt, pad, offset)
        _loss(trag, t, z2, ids, teacher, counts, temp, weight, alone, norm2, z2)
        assert torch.equal(z2, grad) and torch.equal(alone, loss[:rows])
        z3b, z3 = _filled(z0, dt, pad, offset)
        _grad(trag, t, z3, ids, teacher, counts, temp, norm2, weight, z3)
        assert torch.equal(z3, grad2)
        assert loss[rows] == 77 and (norm[rows] == 77).all()
        for buf, v, p in ((gb, grad, pad + 2), (gb2, grad2, pad), (z2b, z2, pad), (z3b, z3, pad)):
            inside = torch.zeros_like(buf, dtype=torch.bool)
            inside[offset:offset + rows * (cols + p)].view(rows, cols + p)[:, :cols] = True
            assert (buf[~inside].float() == 77).all()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1100, 1900), (1025, 4001), (2561, 25003), (2 ** 20 + 77, 5), (1, 2_200_003), (3, 700_001)])
def test_many_rows(trag, t, rows, cols):
    """The forms for many rows, more rows than one launch takes, and rows of more parts than the gradient joins."""
    torch = _torch()
    z0, ids, teacher, counts, weight = _case(rows, cols, 4, cols)
    zb, z = _filled(z0, _types()[t], 1, 1)
    want_loss, _, want_grad, tol_loss, _, tol_grad = _reference(z, ids, teacher, counts, 1.5, weight)
    loss, norm, grad = torch.full((rows,), 77.0, device="cuda"), torch.full((rows, 2), 77.0, device="cuda"), torch.full_like(z, 77.0)
    _loss(trag, t, z, ids, teacher, counts, 1.5, weight, loss, norm, grad)
    assert ((loss.double() - want_loss).abs() <= tol_loss + 2.0 ** -149).all()
    _check_grad(grad, want_grad, tol_grad, t)


def test_more_chunks_than_one_launch_takes(trag):
    torch = _torch()
    rows, cols, k = 116_600, 65_537, 3
    z = torch.empty((rows, cols), dtype=torch.float16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    _, ids, teacher, counts, weight = _case(rows, 1, k, 2)
    ids = torch.randint(0, cols, (rows, k), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda", dtype=torch.int64).to(torch.int32)
    some = torch.cat([torch.arange(20), torch.arange(rows - 200, rows, 5)]).cuda()
    want_loss, _, want_grad, tol_loss, _, tol_grad = _reference(z[some], ids[some], teacher[some], counts[some], 2.0, weight[some])
    loss, norm = torch.full((rows,), 77.0, device="cuda"), torch.full((rows, 2), 77.0, device="cuda")
    _loss(trag, "f16", z, ids, teacher, counts, 2.0, weight, loss, norm, z)
    assert ((loss[some].double() - want_loss).abs() <= tol_loss + 2.0 ** -149).all()
    _check_grad(z[some], want_grad, tol_grad, "f16")


def test_gradient_against_differences(trag):
    """Central differences of the 64-bit loss (step h: off by h^2 / 6 times a third derivative below 2 T, plus
    2^-52 / h times the loss), for rows with repeated ids, ids that are no column, and short lists."""
    torch = _torch()
    rows, cols, k, temp, h = 4, 23, 6, 1.7, 1e-4
    z, ids, teacher, counts, _ = _case(rows, cols, k, 3)
    counts[:] = torch.tensor([6, 4, 1, 6])
    ids[0, 2] = ids[0, 4]
    ids[3, 1] = cols
    ids[3, 5] = -1                                 # 0xFFFFFFFF
    one = torch.ones(rows, device="cuda")
    loss, norm, grad = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda"), torch.empty((rows, cols), device="cuda")
    _loss(trag, "f32", z, ids, teacher, counts, temp, None, loss, norm, grad)
    _, _, _, _, _, tol = _reference(z, ids, teacher, counts, temp, one)
    for c in range(cols):
        zp, zm = z.double(), z.double()
        zp, zm = zp.clone(), zm.clone()
        zp[:, c] += h
        zm[:, c] -= h
        diff = (_reference(zp, ids, teacher, counts, temp, one)[0] - _reference(zm, ids, teacher, counts, temp, one)[0]) / (2 * h)
        assert ((grad[:, c].double() - diff).abs() <= tol[:, c] + U * diff.abs() + 2 * temp * h * h + 1e-10).all()


@pytest.mark.parametrize("cols", [300, 1500, 5000, 30000, 50000, 90000])
def test_masked_and_empty_rows(trag, cols):
    torch = _torch()
    inf, low = float("inf"), torch.finfo(torch.float32).min
    rows, k, temp = 9, 5, 0.7
    z, ids, teacher, counts, weight = _case(rows, cols, k, 11)
    counts[:] = k
    ids[:] = torch.arange(k, device="cuda", dtype=torch.int32) * 3
    z[0, 20:] = -inf                              # most of a row masked
    z[1, 20:] = low
    z[2] = low                                    # all of it, with the type's lowest value: every column alike
    counts[3] = 0                                 # no list, whatever the logits
    z[3, 7] = float("nan")
    teacher[4] = -inf                             # a list without probability
    teacher[5, 2:] = -inf                         # part of a list
    ids[6] = cols + 5                             # no id is a column
    z[7, 3] = -inf                                # a taught column that the student has ruled out: infinite loss, finite gradient
    z[8, :] = 1e30                                # large, equal
    loss, norm = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda")
    grad, grad2 = torch.empty((rows, cols), device="cuda"), torch.empty((rows, cols), device="cuda")
    _loss(trag, "f32", z, ids, teacher, counts, temp, weight, loss, norm, grad)
    _grad(trag, "f32", z, ids, teacher, counts, temp, norm, weight, grad2)
    for r in (3, 4, 6):
        assert loss[r] == 0 and (grad[r] == 0).all() and (grad2[r] == 0).all()
    assert loss[7] == inf
    zz = z.clone()
    zz[3] = 0
    want_loss, want_norm, want_grad, tol_loss, s, tol_grad = _reference(zz, ids, teacher, counts, temp, weight)
    for r in (0, 1, 2, 5, 8):
        assert abs(loss[r].double() - want_loss[r]) <= tol_loss[r], r
    for r in (0, 1, 2, 5, 7, 8):
        for g in (grad, grad2):
            extra = abs(weight[r].double()) * temp * want_norm[r, 1].abs() * 2 * U
            assert ((g[r].double() - want_grad[r]).abs() <= tol_grad[r] + extra + U * want_grad[r].abs()).all(), r
    # NaN and +inf among the logits of a row with a list reach its loss
    z[0, 5], z[1, 5] = float("nan"), inf
    teacher[5, 0] = float("nan")
    _loss(trag, "f32", z, ids, teacher, counts, temp, weight, loss, norm, grad)
    assert torch.isnan(loss[0]) and torch.isnan(loss[1]) and torch.isnan(loss[5])
    assert torch.isnan(grad[0]).all() and torch.isnan(grad[1]).any()


@pytest.mark.parametrize("cols", [64, 40000, 80000])
def test_empty_lists_of_length_zero_and_missing_counts(trag, cols):
    torch = _torch()
    z, ids, teacher, _, _ = _case(3, cols, 0, 1)
    loss, norm, grad = torch.full((3,), 5.0, device="cuda"), torch.empty((3, 2), device="cuda"), torch.full((3, cols), 5.0, device="cuda")
    _loss(trag, "f32", z, ids, teacher, None, 1.0, None, loss, norm, grad)
    assert (loss == 0).all() and (grad == 0).all()
    grad.fill_(5.0)
    _grad(trag, "f32", z, ids, teacher, None, 1.0, norm, None, grad)
    assert (grad == 0).all()
    z, ids, teacher, _, _ = _case(3, cols, 20, 1)
    full = torch.full((3,), 20, dtype=torch.int32, device="cuda")
    a, b = torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    _loss(trag, "f32", z, ids, teacher, None, 1.0, None, a, norm)
    _loss(trag, "f32", z, ids, teacher, full, 1.0, None, b, norm)
    assert torch.equal(a, b)


def test_a_row_past_32_bit_offsets(trag):
    """Rows whose offsets pass 2^32 bytes, and a row of ten million columns."""
    torch = _torch()
    rows, cols, k = 450, 10_000_000, 10
    z = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda").normal_()
    ids = torch.randint(0, cols, (rows, k), device="cuda", dtype=torch.int64).to(torch.int32)
    teacher = torch.randn((rows, k), device="cuda")
    counts = torch.full((rows,), k, dtype=torch.int32, device="cuda")
    loss, norm = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda")
    _loss(trag, "bf16", z, ids, teacher, counts, 1.0, None, loss, norm)
    weight = torch.ones(rows, device="cuda")
    for r in (0, 230, 449):
        part = slice(r, r + 1)
        want, _, _, tol, _, _ = _reference(z[part], ids[part], teacher[part], counts[part], 1.0, weight[part])
        assert abs(loss[r].double() - want[0]) <= tol[0]
    last = z[449:].clone()
    want = _reference(last, ids[449:], teacher[449:], counts[449:], 1.0, weight[449:])
    _grad(trag, "bf16", z, ids, teacher, counts, 1.0, norm, weight, z)      # in place, the whole of it
    _check_grad(z[449:], want[2], want[5] + want[1][:, 1:].abs() * 2 * U, "bf16")


@pytest.mark.parametrize("cols", [3000, 60000, 120000])
def test_streams_and_graphs(trag, cols):
    """A captured step replayed with new logits, two captured steps with a workspace each on two streams."""
    torch = _torch()
    rows, k, temp = 12, 9, 2.0
    sets = []
    for seed in (1, 2):
        z, ids, teacher, counts, weight = _case(rows, cols, k, seed)
        s = dict(z=z, ids=ids, teacher=teacher, counts=counts, weight=weight, loss=torch.empty(rows, device="cuda"), norm=torch.empty((rows, 2), device="cuda"),
                 grad=torch.empty_like(z), work=torch.empty(max(4, trag.distill_work_bytes(rows, cols)), dtype=torch.uint8, device="cuda"), stream=torch.cuda.Stream())
        s["graph"] = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(s["graph"], stream=s["stream"]):
            _loss(trag, "f32", z, ids, teacher, counts, temp, weight, s["loss"], s["norm"], s["grad"], s["stream"], s["work"])
        sets.append(s)
    for it in range(4):
        for s in sets:
            s["z"].normal_(generator=torch.Generator(device="cuda").manual_seed(100 * it + cols))
            s["grad"].fill_(float("nan"))
            s["loss"].fill_(float("nan"))
        torch.cuda.synchronize()
        for s in sets:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
        torch.cuda.synchronize()
        for s in sets:
            loss, norm, grad = torch.empty_like(s["loss"]), torch.empty_like(s["norm"]), torch.empty_like(s["grad"])
            _loss(trag, "f32", s["z"], s["ids"], s["teacher"], s["counts"], temp, s["weight"], loss, norm, grad)
            assert torch.equal(loss, s["loss"]) and torch.equal(grad, s["grad"]) and torch.equal(norm, s["norm"])


def test_the_first_stage_and_its_training_step(trag):
    """Encoder states -> 8-bit queries; store rows -> 8-bit corpus; their product = the student's scores; the store's exact
    search = the teacher's lists, taken from device memory as they are; loss and gradient over the whole corpus. Compared with
    the same chain in 64 bits on the 8-bit values."""
    torch = _torch()
    n, d, B, k, temp = 50_000, 384, 6, 20, 0.05
    store = trag.VectorStore(trag.VectorStoreConfig(dimension=d, metric=trag.DistanceMetric.DotProduct, reserve_rows=n))
    store.fill_synthetic(n, 21)
    g = torch.Generator(device="cuda").manual_seed(4)
    hidden, residual = (torch.randn((B, d), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    w = (torch.rand(d, generator=g, device="cuda") + 0.5).to(torch.bfloat16)
    st = torch.cuda.current_stream().cuda_stream
    q8, qs = torch.empty((B, d), dtype=torch.int8, device="cuda"), torch.empty(B, device="cuda")
    new_sum = torch.empty_like(hidden)
    trag.rmsnorm_q8_device(hidden.data_ptr(), d, residual.data_ptr(), d, w.data_ptr(), 1e-6, CODE["bf16"], B, d, new_sum.data_ptr(), d, q8.data_ptr(), d,
                           qs.data_ptr(), stream=st)
    c8, cs = torch.empty((n, d), dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    store.quantize_device(0, n, c8.data_ptr(), d, cs.data_ptr(), st)
    scores = torch.empty((B, n), device="cuda")
    trag.matmul_q8_device(q8.data_ptr(), d, qs.data_ptr(), c8.data_ptr(), d, cs.data_ptr(), B, n, d, CODE["f32"], scores.data_ptr(), n, st)
    # the teacher searches with the unquantised query
    h = hidden.float() + residual.float()
    full = (h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * w.float()).contiguous()
    rows, best = torch.empty((B, k), dtype=torch.int32, device="cuda"), torch.empty((B, k), device="cuda")
    found, status = torch.empty(B, dtype=torch.int32, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
    store.search_device(full.data_ptr(), B, k, rows.data_ptr(), best.data_ptr(), found.data_ptr(), status.data_ptr(), st)
    loss, norm, grad = torch.empty(B, device="cuda"), torch.empty((B, 2), device="cuda"), torch.empty((B, n), device="cuda")
    work = _loss(trag, "f32", scores, rows, best, found, temp, None, loss, norm, grad)
    torch.cuda.synchronize()
    assert status.tolist() == [0] * B and found.tolist() == [k] * B and work.numel() >= trag.distill_work_bytes(B, n)
    corpus = torch.from_numpy(store.read_rows(0, n)).cuda().double()
    # the 8-bit scores are within the grids' own steps of the exact ones: |error| <= (||q|| / 127-step part + corpus part)
    exact = full.double() @ corpus.t()
    step = 0.5 * (qs.double()[:, None] * corpus.abs().sum(1)[None] + cs.double()[None] * full.double().abs().sum(1)[:, None]
                  + 0.5 * d * qs.double()[:, None] * cs.double()[None])
    assert ((scores.double() - exact).abs() <= step * (1 + 1e-5)).all()
    assert torch.equal(scores, (c8.double() @ q8.double().t()).t().float() * qs[:, None] * cs[None])
    want_loss, _, want_grad, tol_loss, _, tol_grad = _reference(scores, rows, best, found, temp, torch.ones(B, device="cuda"))
    assert ((loss.double() - want_loss).abs() <= tol_loss).all()
    _check_grad(grad, want_grad, tol_grad, "f32")
    # probabilities moved, none made: a row's gradient sums to zero
    assert (grad.double().sum(1).abs() <= (tol_grad + U * want_grad.abs()).sum(1)).all()
    store.close()
