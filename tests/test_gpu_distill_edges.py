"""GPU: distillation at the edges of its inputs, against the formula in 64 bits."""
import pytest

from test_gpu_distill import U, _grad, _loss, _torch

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
