"""GPU: distillation at the edges of its inputs, against the formula in 64 bits."""
import pytest

from test_gpu_distill import U, _case, _check_grad, _grad, _loss, _reference, _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temp", [0.7, 3.0])
@pytest.mark.parametrize("rows,cols", [(64, 40), (64, 5000), (24, 40000), (24, 70001), (2, 2_200_003)])
def test_probabilities_of_a_repeated_id_add_up(trag, rows, cols, temp):
    """Lists of 1024 entries, the longest, that name a few columns hundreds of times, at columns where the student has nothing:
    the gradient there is -weight T sum p. Bound: an entry's exponential is off by the rounding of its argument, below one half
    (2^-26 ln 2), and one unit of the hardware's exp2 (2 U), together 3 U; the sum they are divided by is a 64-bit sum of the
    same, 3 U; the probability's own rounding U, weight T U, their product U: (3 + 3 + 1 + 1 + 1) U, whatever the number of
    repeats. Where every entry names the same column, the probability is a sum over itself, exactly 1: 2 U."""
    torch = _torch()
    k = 1024
    g = torch.Generator(device="cuda").manual_seed(cols)
    z = torch.randn((rows, cols), generator=g, device="cuda")
    first = cols // 3
    z[:, first:first + 8] = -1000.0          # (the student's share is e^-333 and less: 0)
    teacher = torch.sort(2 * torch.randn((rows, k), generator=g, device="cuda"), 1, descending=True).values.contiguous()
    ids = torch.full((rows, k), first, dtype=torch.int32, device="cuda")                     # rows 0, 4, ...: one column
    j = torch.arange(k, device="cuda", dtype=torch.int32)
    ids[1::4] = first + j % 2                                                                # two, in turn
    ids[2::4] = first + torch.clamp(j // 128, max=7).to(torch.int32)                         # eight, in runs
    ids[3::4] = first + (torch.randint(0, 8, (1, k), generator=g, device="cuda")).to(torch.int32)
    counts = torch.full((rows,), k, dtype=torch.int32, device="cuda")
    weight = torch.randn(rows, generator=g, device="cuda")
    loss, norm, grad, alone = (torch.empty(s, device="cuda") for s in ((rows,), (rows, 2), (rows, cols), (rows, cols)))
    _loss(trag, "f32", z, ids, teacher, counts, temp, weight, loss, norm, grad)
    _grad(trag, "f32", z, ids, teacher, counts, temp, norm, weight, alone)
    temp = torch.tensor(temp).double().item()    # (what the call takes: its argument is 32 bits)
    p = torch.softmax(teacher.double() / temp, 1)
    dense = torch.zeros((rows, 8), dtype=torch.float64, device="cuda").scatter_add_(1, ids.long() - first, p)
    want = -(weight.double() * temp)[:, None] * dense
    bound = torch.full((rows, 1), 9.0 * U, dtype=torch.float64, device="cuda")
    bound[0::4] = 2.0 * U
    for got in (grad, alone):
        off = (got[:, first:first + 8].double() - want).abs()
        assert (off <= bound * want.abs() * (1 + 1e-6)).all(), ((off / want.abs().clamp_min(1e-300)).max(1).values / U).tolist()


@pytest.mark.parametrize("cols", [3000, 60000, 120000])
def test_captured_steps_that_differ(trag, cols):
    """Two captured steps and two captured gradients alone on two streams, a workspace each, whose logits differ in every
    column and in their spread, so that maxima and sums of one would be wrong for the other; every replay against the formula.
    The logarithm of a row's sum is off by the exponential's own error, (4 E + 4) U as derived beside _reference, and one U for
    each addition in 32 bits that a term goes through: up to 8 + 16 in a row held in registers, 33 and the sum's rounding in a chunk."""
    torch = _torch()
    slack = (66 - (24 if cols <= 65536 else 34)) * U     # (_reference allows for 66)
    rows, k, temp = 12, 9, 2.0
    sets = []
    for i in range(2):
        z, ids, teacher, counts, weight = _case(rows, cols, k, 50 + i)
        s = dict(z=z, lists=(ids, teacher, counts), weight=weight, loss=torch.empty(rows, device="cuda"), norm=torch.empty((rows, 2), device="cuda"),
                 grad=torch.empty_like(z), alone=torch.empty_like(z), spread=(1.0, 6.0)[i], stream=torch.cuda.Stream(),
                 work=torch.empty(max(4, trag.distill_work_bytes(rows, cols)), dtype=torch.uint8, device="cuda"), graph=torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(s["graph"], stream=s["stream"]):
            _loss(trag, "f32", z, *s["lists"], temp, weight, s["loss"], s["norm"], s["grad"], s["stream"], s["work"])
            _grad(trag, "f32", z, *s["lists"], temp, s["norm"], weight, s["alone"], s["stream"])
        sets.append(s)
    for it in range(4):
        for i, s in enumerate(sets):
            g = torch.Generator(device="cuda").manual_seed(10 * it + i)
            s["z"].copy_(s["spread"] * torch.randn((rows, cols), generator=g, device="cuda") + 3.0 * i)
            for name in ("loss", "norm", "grad", "alone"):
                s[name].fill_(float("nan"))
        torch.cuda.synchronize()
        for s in sets:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
        torch.cuda.synchronize()
        for s in sets:
            want_loss, want_norm, want_grad, tol_loss, tol, tol_grad = _reference(s["z"], *s["lists"], temp, s["weight"])
            assert ((s["loss"].double() - want_loss).abs() <= tol_loss - temp ** 2 * slack).all()
            assert torch.equal(s["norm"][:, 0].double(), want_norm[:, 0])
            assert ((s["norm"][:, 1].double() - want_norm[:, 1]).abs() <= tol - slack + 2 * U * want_norm[:, 1].abs()).all()
            _check_grad(s["grad"], want_grad, tol_grad, "f32")
            # (the saved logarithm has been rounded to 32 bits)
            _check_grad(s["alone"], want_grad, tol_grad + (s["weight"].double()[:, None] * temp).abs() * want_norm[:, 1:].abs() * 2 * U, "f32")


@pytest.mark.parametrize("t,cols", [("f32", 60), ("bf16", 3000), ("f16", 30000), ("f32", 60000), ("bf16", 120000), ("f32", 2_200_003)])
def test_rows_of_logits_that_leave_nothing(trag, t, cols):
    """A row of minus infinities has no distribution: loss and gradient are NaN, 0 where the list is empty too; its neighbours
    are what they are without it."""
    torch = _torch()
    inf, rows, k, temp = float("inf"), 4, 6, 1.5
    dt = dict(f32=torch.float32, f16=torch.float16, bf16=torch.bfloat16)[t]
    z, ids, teacher, counts, weight = _case(rows, cols, k, 8)
    z = z.to(dt)
    counts[:] = k
    z[1], z[2] = -inf, -inf
    counts[2] = 0
    loss, norm = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda")
    grad, alone = torch.zeros_like(z), torch.zeros_like(z)
    _loss(trag, t, z, ids, teacher, counts, temp, weight, loss, norm, grad)
    _grad(trag, t, z, ids, teacher, counts, temp, norm, weight, alone)
    assert torch.isnan(loss[1]) and torch.isnan(grad[1]).all() and torch.isnan(alone[1]).all()
    assert loss[2] == 0 and (grad[2] == 0).all() and (alone[2] == 0).all()
    assert (norm[1:3] == -inf).all()
    fine = [0, 3]
    want_loss, want_norm, want_grad, tol_loss, _, tol_grad = _reference(z[fine], ids[fine], teacher[fine], counts[fine], temp, weight[fine])
    assert ((loss[fine].double() - want_loss).abs() <= tol_loss + 2.0 ** -149).all()
    _check_grad(grad[fine], want_grad, tol_grad, t)
    _check_grad(alone[fine], want_grad, tol_grad + (weight[fine].double()[:, None] * temp).abs() * want_norm[:, 1:].abs() * 2 * U, t)
