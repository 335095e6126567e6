"""GPU: rows of 8-bit integers with scales (trag_rmsnorm_q8_device, trag_quantize_q8_device) and their
product (trag_matmul_q8_device) against plain forms in 64 bits. Integers, sums and products are
compared bit for bit: they are functions of the inputs alone. Scales are 64-bit results rounded once to
f32 (half a step, 2^-24 relative)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_F32 = 2.0 ** -24 * (1 + 1e-6)      # a rounding to f32; the 64-bit arithmetic in front of it is off by 1e-13 at most
FILL = 77                               # what the bytes around an output hold


def _torch():
    import torch
    return torch


def _types():
    torch = _torch()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


CODE = {"f32": 0, "f16": 1, "bf16": 2}


def _strided(rows, cols, pad, dtype, offset=0):
    """(rows, cols) view whose rows lie cols + pad apart, `offset` elements behind an aligned address; the rest
    of the buffer holds FILL."""
    torch = _torch()
    buf = torch.full((rows * (cols + pad) + offset + 64,), FILL, dtype=dtype, device="cuda")
    return buf, buf[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]


def _untouched(buf, view, offset=0):
    """Everything in the buffer outside the view still holds FILL."""
    torch = _torch()
    mask = torch.ones_like(buf, dtype=torch.bool)
    rows, cols = view.shape
    stride = view.stride(0) if rows > 1 else cols
    inner = mask[offset:offset + (rows - 1) * stride + cols]
    idx = (torch.arange(rows, device="cuda")[:, None] * stride + torch.arange(cols, device="cuda")[None]).reshape(-1)
    inner[idx] = False
    return bool((buf[mask].float() == FILL).all())


def _reference(x, r, w, eps, norm=True):
    """integers and scale in 64 bits"""
    torch = _torch()
    h = x.double() + (r.double() if r is not None else 0)
    p = h * w.double() if w is not None else h
    top = p.abs().amax(1, keepdim=True)
    q = torch.round(p * 127 / top)
    scale = top / 127
    if norm:
        scale = scale / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    zero = top == 0
    return torch.where(zero, 0, q).to(torch.int8), torch.where(zero, 0, scale).squeeze(1)


def _run_norm(trag, t, x, r, w, eps, s_sum, q8, scale, values, stream=None):
    torch = _torch()
    trag.rmsnorm_q8_device(x.data_ptr(), x.stride(0), 0 if r is None else r.data_ptr(), 0 if r is None else r.stride(0),
                           0 if w is None else w.data_ptr(), eps, CODE[t], x.shape[0], x.shape[1],
                           0 if s_sum is None else s_sum.data_ptr(), 0 if s_sum is None else s_sum.stride(0), q8.data_ptr(), q8.stride(0),
                           scale.data_ptr(), 0 if values is None else values.data_ptr(), 0 if values is None else values.stride(0),
                           (stream or torch.cuda.current_stream()).cuda_stream)


def _check_rows(x, r, w, eps, q8, scale, norm=True):
    eq, es = _reference(x, r, w, eps, norm)
    assert (q8 == eq).all(), ((q8 != eq).nonzero()[:3].tolist())
    assert ((scale.double() - es).abs() <= HALF_F32 * es + 2.0 ** -150).all()


DIMS = [1, 2, 7, 8, 9, 63, 64, 65, 384, 511, 512, 513, 1021, 1024, 1025, 2048, 2049, 4096, 4100, 8192, 8193, 16384, 16391,
        32768, 32769, 40001]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", DIMS)
def test_norm_matches_the_formula(trag, t, dim):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(dim)
    dt = _types()[t]
    for rows, pad, offset, residual, weight in ((1, 0, 0, True, True), (5, 3, 1, True, True), (37, 0, 0, False, True), (6, 16, 8, True, False)):
        xb, x = _strided(rows, dim, pad, dt, offset)
        rb, r = _strided(rows, dim, pad + 1, dt, offset)
        x.copy_(torch.randn((rows, dim), generator=g, device="cuda") * torch.exp(torch.randn((rows, 1), generator=g, device="cuda")))
        r.copy_(torch.randn((rows, dim), generator=g, device="cuda"))
        w = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dt) if weight else None
        if not residual:
            r = None
        sb, s_sum = _strided(rows, dim, pad, dt, offset)
        qb, q8 = _strided(rows, dim, pad + 5, torch.int8, offset)
        vb, values = _strided(rows, dim, pad, dt, offset)
        scale = torch.full((rows + 3,), float(FILL), device="cuda")
        _run_norm(trag, t, x, r, w, 1e-5, s_sum, q8, scale, values)
        _check_rows(x, r, w, 1e-5, q8, scale[:rows])
        want = x.float() + r.float() if r is not None else x.float()
        assert torch.equal(s_sum, want.to(dt))
        assert torch.equal(values, (q8.float() * scale[:rows, None]).to(dt))
        assert _untouched(sb, s_sum, offset) and _untouched(qb, q8, offset) and _untouched(vb, values, offset)
        assert (scale[rows:] == FILL).all()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [1, 8, 65, 384, 768, 1000, 4096, 33001])
def test_quantize_matches_the_formula(trag, t, dim):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(dim)
    dt = _types()[t]
    for rows, pad, offset in ((1, 0, 0), (130, 2, 1), (7, 8, 0)):
        _, x = _strided(rows, dim, pad, dt, offset)
        x.copy_(torch.randn((rows, dim), generator=g, device="cuda"))
        qb, q8 = _strided(rows, dim, pad, torch.int8, offset)
        scale = torch.full((rows + 1,), float(FILL), device="cuda")
        trag.quantize_q8_device(x.data_ptr(), x.stride(0), CODE[t], rows, dim, q8.data_ptr(), q8.stride(0), scale.data_ptr(),
                                stream=torch.cuda.current_stream().cuda_stream)
        _check_rows(x, None, None, 0.0, q8, scale[:rows], norm=False)
        assert _untouched(qb, q8, offset) and scale[rows] == FILL


def test_ties_go_to_even(trag):
    """Rows of whole numbers whose quotients fall on the middle between two integers, for largest elements
    127 j whose reciprocal is not exact: 127 p / (127 j) = p / j = n + 1/2."""
    torch = _torch()
    for j in (2, 6, 10, 14, 22, 26, 38, 46, 58, 74):
        p = torch.arange(-127 * j, 127 * j + 1, dtype=torch.float32, device="cuda")[None].contiguous()
        dim = p.shape[1]
        q8 = torch.empty((1, dim), dtype=torch.int8, device="cuda")
        scale = torch.empty(1, device="cuda")
        trag.quantize_q8_device(p.data_ptr(), dim, 0, 1, dim, q8.data_ptr(), dim, scale.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
        whole = p.cpu().to(torch.int64)[0].tolist()
        want = []
        for v in whole:                       # nearest(v / j), ties to even, in whole numbers
            lo, rest = divmod(v, j)
            want.append(lo + (1 if 2 * rest > j or (2 * rest == j and lo % 2) else 0))
        assert q8[0].cpu().tolist() == want, j
        assert scale.item() == float(j)


@pytest.mark.parametrize("dim", [40, 600, 4096, 33000])
def test_rows_of_zeros_infinities_and_nans(trag, dim):
    torch = _torch()
    x = torch.randn((8, dim), device="cuda")
    x[1] = 0
    x[2, dim // 2] = float("inf")
    x[3, dim - 1] = float("nan")
    x[4, 0] = -float("inf")
    x[5] = torch.finfo(torch.float32).min        # the type's lowest value: finite, its square is not in 32 bits
    x[6] = 1e-30
    w = torch.ones(dim, device="cuda")
    w[1] = 0
    q8 = torch.full((8, dim), FILL, dtype=torch.int8, device="cuda")
    scale = torch.empty(8, device="cuda")
    values = torch.empty((8, dim), device="cuda")
    _run_norm(trag, "f32", x, None, w, 1e-6, None, q8, scale, values)
    fine = [0, 1, 5, 6, 7]
    _check_rows(x[fine], None, w, 1e-6, q8[fine], scale[fine])
    assert scale[1] == 0 and (q8[1] == 0).all() and (values[1] == 0).all()
    for r in (2, 3, 4):
        assert torch.isnan(scale[r]) and (q8[r] == 0).all() and torch.isnan(values[r]).all()
    trag.quantize_q8_device(x.data_ptr(), dim, 0, 8, dim, q8.data_ptr(), dim, scale.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    _check_rows(x[fine], None, None, 0.0, q8[fine], scale[fine], norm=False)
    assert torch.isnan(scale[[2, 3, 4]]).all()
    # eps 0 on a row of zeros
    _run_norm(trag, "f32", x, None, w, 0.0, None, q8, scale, values)
    assert scale[1] == 0 and (values[1] == 0).all()


@pytest.mark.parametrize("t,dim", [("bf16", 4096), ("f16", 1001), ("f32", 384), ("bf16", 36000)])
def test_sum_and_values_in_place(trag, t, dim):
    torch = _torch()
    dt = _types()[t]
    rows = 9
    x, r = (torch.randn((rows, dim), device="cuda").to(dt) for _ in range(2))
    w = torch.rand(dim, device="cuda").to(dt)
    eq, es = _reference(x, r, w, 1e-5)
    want = (x.float() + r.float()).to(dt)
    q8 = torch.empty((rows, dim), dtype=torch.int8, device="cuda")
    scale = torch.empty(rows, device="cuda")
    for sum_in, values_in in ((0, 1), (1, 0), (0, None), (1, None)):
        pair = [x.clone(), r.clone()]
        _run_norm(trag, t, pair[0], pair[1], w, 1e-5, pair[sum_in], q8, scale, None if values_in is None else pair[values_in])
        assert (q8 == eq).all() and torch.equal(pair[sum_in], want)
        if values_in is not None:
            assert torch.equal(pair[values_in], (q8.float() * scale[:, None]).to(dt))


def test_many_short_rows(trag):
    """More rows than one sweep of workgroups, rows of one element among them."""
    torch = _torch()
    rows = (1 << 22) + 5
    x = torch.randn((rows, 1), device="cuda")
    q8 = torch.empty((rows, 1), dtype=torch.int8, device="cuda")
    scale = torch.empty(rows, device="cuda")
    trag.quantize_q8_device(x.data_ptr(), 1, 0, rows, 1, q8.data_ptr(), 1, scale.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    assert torch.equal(q8, (127 * torch.sign(x)).to(torch.int8))   # (a single element is its own maximum)
    # (the quotient in 64 bits, rounded once)
    assert torch.equal(scale, (x.abs().double() / 127).float().squeeze(1))


# ---- the product

def _int8(rows, cols, pad, offset, g, extreme=False):
    torch = _torch()
    buf, v = _strided(rows, cols, pad, torch.int8, offset)
    v.copy_(torch.randint(-128, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int16).to(torch.int8))
    if extreme:
        v[0] = -128
    return v


def _product(trag, a, b, sa, sb, out, t, stream=None):
    torch = _torch()
    trag.matmul_q8_device(a.data_ptr(), a.stride(0), 0 if sa is None else sa.data_ptr(), b.data_ptr(), b.stride(0),
                          0 if sb is None else sb.data_ptr(), a.shape[0], b.shape[0], a.shape[1], CODE[t], out.data_ptr(), out.stride(0),
                          (stream or torch.cuda.current_stream()).cuda_stream)


def _expect(a, b, sa, sb, dt):
    """the whole-number sums, rounded to f32 and scaled there in the documented order"""
    acc = a.double() @ b.double().t()       # whole numbers below 2^53: exact
    c = acc.float()
    c = c * sa[:, None] if sa is not None else c
    c = c * sb[None] if sb is not None else c
    return c.to(dt)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(r, d) for r in (1030, 2051, 4103) for d in (100, 201, 300, 505, 700, 1000, 1300, 2001)] + [(520, 5001), (1030, 9000)])
def test_forms_for_many_rows(trag, t, rows, dim):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(rows + dim)
    dt = _types()[t]
    xb, x = _strided(rows, dim, 3, dt, 1)
    x.copy_(torch.randn((rows, dim), generator=g, device="cuda"))
    r = torch.randn((rows, dim), generator=g, device="cuda").to(dt)
    w = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dt)
    want = (x.float() + r.float()).to(dt)
    x0 = x.clone()
    qb, q8 = _strided(rows, dim, 5, torch.int8, 1)
    scale = torch.full((rows + 3,), float(FILL), device="cuda")
    values = torch.empty((rows, dim), dtype=dt, device="cuda")
    _run_norm(trag, t, x, r, w, 1e-5, x, q8, scale, values)      # (the sum in place)
    _check_rows(x0, r, w, 1e-5, q8, scale[:rows])
    assert torch.equal(x, want) and torch.equal(values, (q8.float() * scale[:rows, None]).to(dt))
    assert _untouched(xb, x, 1) and _untouched(qb, q8, 1) and (scale[rows:] == FILL).all()


def test_more_rows_than_one_launch_takes(trag):
    torch = _torch()
    rows = 2 ** 24 + 35
    g = torch.Generator(device="cuda").manual_seed(5)
    x, r = (torch.randn((rows, 3), generator=g, device="cuda") for _ in range(2))
    q8, scale, s = torch.full((rows, 3), FILL, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros((rows, 3), device="cuda")
    _run_norm(trag, "f32", x, r, None, 1e-6, s, q8, scale, None)
    _check_rows(x, r, None, 1e-6, q8, scale)
    assert torch.equal(s, x + r)


SHAPES = [(1, 1, 1), (1, 5, 16), (1, 1000, 384), (2, 129, 15), (3, 64, 17), (7, 300, 64), (8, 257, 768), (16, 4096, 1024),
          (17, 100, 63), (31, 513, 65), (32, 64, 128), (33, 4097, 96), (64, 640, 2048), (65, 130, 129), (100, 999, 250),
          (128, 128, 64), (129, 127, 144), (200, 2000, 384), (256, 256, 512), (257, 511, 400), (300, 1030, 777), (512, 768, 1040),
          (1000, 300, 4096), (1025, 513, 48), (5, 3, 20000), (300, 2000, 15), (2100, 2050, 1), (16, 4096, 4096), (33, 70, 4112),
          (600, 4100, 2064), (1100, 4096, 1040), (2000, 9000, 272), (2050, 8200, 128), (70, 33000, 400), (40, 70, 131071), (1, 40, 131071), (300, 300, 9000)]


@pytest.mark.parametrize("m,n,dim", SHAPES)
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_product_is_exact(trag, m, n, dim, t):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(m * 7 + n)
    dt = _types()[t]
    for pad, offset, opad in ((0, 0, 0), (16, 16, 8), (3, 1, 5)):
        a, b = _int8(m, dim, pad, offset, g, True), _int8(n, dim, pad, offset, g, True)
        # (keeps the largest sums inside f16)
        sa = torch.rand(m, generator=g, device="cuda") / 128
        sb = torch.rand(n, generator=g, device="cuda") / (2 * dim)
        ob, out = _strided(m, n, opad, dt)
        _product(trag, a, b, sa, sb, out, t)
        assert torch.equal(out, _expect(a, b, sa, sb, dt)), (pad, offset)
        assert _untouched(ob, out)


@pytest.mark.parametrize("m,n,dim", [(3421, 2373, 432), (791, 10075, 438), (489, 1399, 409), (2377, 201, 405), (65, 33717, 624), (2325, 2467, 429),
                                     (915, 261, 704), (2927, 1221, 426), (273, 997, 400), (113, 1067, 432), (1129, 101, 576), (701, 397, 551),
                                     (2563, 405, 400), (111, 297, 448), (69, 28779, 480), (19, 23123, 496), (855, 303, 411), (331, 8661, 1184),
                                     (3491, 1705, 34), (2997, 495, 33), (611, 4355, 33), (4, 65, 192), (177, 161, 320), (13, 35, 1111)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_product_in_every_tile(trag, m, n, dim, t):
    """Sizes between them reach every tile, with rows at multiples of 16 bytes and at any byte."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(m * 7 + n)
    for pad, offset in ((0, 0), (5, 1)):
        a, b = _int8(m, dim, pad, offset, g, True), _int8(n, dim, pad, offset, g, True)
        sa, sb = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
        ob, out = _strided(m, n, 3, _types()[t])
        _product(trag, a, b, sa, sb, out, t)
        assert torch.equal(out, _expect(a, b, sa, sb, _types()[t])), (pad, offset)
        assert _untouched(ob, out)


def test_product_without_scales_and_with_nan_scales(trag):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(5)
    for m, n in ((1, 700), (12, 700), (150, 700), (600, 700)):
        a, b = _int8(m, 384, 0, 0, g), _int8(n, 384, 0, 0, g)
        out = torch.empty((m, n), device="cuda")
        _product(trag, a, b, None, None, out, "f32")
        assert torch.equal(out, _expect(a, b, None, None, torch.float32))
        sa, sb = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
        sb[3] = float("nan")
        a[0] = 0
        _product(trag, a, b, sa, sb, out, "f32")
        assert torch.isnan(out[:, 3]).all() and not torch.isnan(out[:, :3]).any() and not torch.isnan(out[:, 4:]).any()


@pytest.mark.parametrize("m", [1, 20, 300])
def test_product_past_32_bit_offsets(trag, m):
    """A corpus of more than 4 GiB, and an output whose offsets pass 2^32 bytes."""
    torch = _torch()
    dim, n = 1040, 4_200_000
    g = torch.Generator(device="cuda").manual_seed(1)
    b = torch.randint(-127, 128, (n, dim), generator=g, device="cuda", dtype=torch.int8)
    a = _int8(m, dim, 0, 0, g)
    out = torch.empty((m, n), device="cuda")
    _product(trag, a, b, None, None, out, "f32")
    for lo in (0, n // 2 - 500, n - 1000):
        assert torch.equal(out[:, lo:lo + 1000], _expect(a, b[lo:lo + 1000], None, None, torch.float32)), lo


def test_product_of_rows_far_apart(trag):
    """Strides of 2^24 bytes and more: offsets inside a tile pass 32 bits."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(2)
    far = (1 << 24) + 16
    for m, n, dim in ((1, 300, 384), (70, 300, 100), (300, 40, 96)):
        wide = torch.empty(300 * far + 512, dtype=torch.int8, device="cuda")
        rows = torch.as_strided(wide, (300, dim), (far, 1))
        rows.copy_(_int8(300, dim, 0, 0, g))
        near = _int8(300, dim, 0, 0, g)
        for a, b in ((near[:m], rows[:n]), (rows[:m], near[:n])):
            out = torch.empty((m, n), device="cuda")
            _product(trag, a, b, None, None, out, "f32")
            assert torch.equal(out, _expect(a, b, None, None, torch.float32))


@pytest.mark.parametrize("m,n,dim", [(2 ** 28 + 1000, 2, 3), (2, 2 ** 28 + 1000, 16)])
def test_product_of_very_many_rows(trag, m, n, dim):
    """More rows than one grid of the smallest tiles covers, rows of the other operand 2^24 bytes apart where it is the wide one."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(m + n)
    few, many = (n, m) if m > n else (m, n)
    far = 2 ** 24 if m < n else dim
    big = torch.randint(-128, 128, (many, dim), generator=g, device="cuda", dtype=torch.int8)
    small = torch.empty(far * (few - 1) + dim, dtype=torch.int8, device="cuda").as_strided((few, dim), (far, 1))
    small.copy_(torch.randint(-128, 128, (few, dim), generator=g, device="cuda", dtype=torch.int8))
    scale = torch.rand(many, generator=g, device="cuda")
    out = torch.full((m, n), float("nan"), device="cuda")
    a, b = (big, small) if m > n else (small, big)
    sa, sb = (scale, None) if m > n else (None, scale)
    _product(trag, a, b, sa, sb, out, "f32")
    for i in range(few):
        s = torch.zeros(many, dtype=torch.int32, device="cuda")
        for c in range(dim):
            s += big[:, c].int() * small[i, c].int()
        got = out[:, i] if m > n else out[i]
        assert torch.equal(got, s.float() * scale), i


def test_an_earlier_error_of_the_program_is_not_the_call_s(trag):
    """A runtime call of the program that failed leaves an error behind; an operator that is launched after it succeeds."""
    torch = _torch()
    x = torch.ones((3, 64), device="cuda")
    q8 = torch.empty((3, 64), dtype=torch.int8, device="cuda")
    scale = torch.empty(3, device="cuda")
    assert trag.lib().hipSetDevice(9999) != 0   # (the runtime that the library is linked to)
    trag.quantize_q8_device(x.data_ptr(), 64, 0, 3, 64, q8.data_ptr(), 64, scale.data_ptr(), 0, 0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (q8 == 127).all()


def test_two_threads_at_once(trag):
    """The calls keep nothing: two threads on streams of their own, one of them the thread's default stream, get what one gets."""
    import threading
    torch = _torch()
    per_thread = 2   # hipStreamPerThread
    g = torch.Generator(device="cuda").manual_seed(4)
    work, errors = [], []
    for m, n, dim in ((5, 700, 384), (130, 257, 1000)):
        x = torch.randn((m, dim), generator=g, device="cuda")
        b = _int8(n, dim, 0, 0, g)
        q8 = torch.zeros((m, dim), dtype=torch.int8, device="cuda")
        work.append((x, b, q8, torch.zeros(m, device="cuda"), torch.zeros((m, n), device="cuda")))
    streams = [torch.cuda.Stream().cuda_stream, per_thread]
    torch.cuda.synchronize()

    def run(i):
        try:
            x, b, q8, scale, out = work[i]
            for _ in range(50):
                trag.quantize_q8_device(x.data_ptr(), x.stride(0), 0, x.shape[0], x.shape[1], q8.data_ptr(), q8.stride(0), scale.data_ptr(), 0, 0, streams[i])
                trag.matmul_q8_device(q8.data_ptr(), q8.stride(0), scale.data_ptr(), b.data_ptr(), b.stride(0), 0, x.shape[0], b.shape[0], x.shape[1], 0,
                                      out.data_ptr(), out.stride(0), streams[i])
        except Exception as e:   # noqa: BLE001 (handed to the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for x, b, q8, scale, out in work:
        _check_rows(x, None, None, 0.0, q8, scale, norm=False)
        assert torch.equal(out, _expect(q8, b, scale, None, torch.float32))


def test_operators_on_other_streams_and_in_graphs(trag):
    """A chain norm -> product on a side stream, then captured and replayed with new inputs, with eager work
    between the replays: every replay gives what the eager chain gives."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(9)
    for m, n, dim in ((1, 3000, 384), (20, 1000, 768), (300, 512, 1024)):
        x = torch.randn((m, dim), generator=g, device="cuda").to(torch.bfloat16)
        r = torch.randn((m, dim), generator=g, device="cuda").to(torch.bfloat16)
        w = torch.rand(dim, generator=g, device="cuda").to(torch.bfloat16)
        b = _int8(n, dim, 0, 0, g)
        sb = torch.rand(n, generator=g, device="cuda")
        q8 = torch.empty((m, dim), dtype=torch.int8, device="cuda")
        scale = torch.empty(m, device="cuda")
        out = torch.empty((m, n), device="cuda")

        def chain(st):
            _run_norm(trag, "bf16", x, r, w, 1e-6, None, q8, scale, None, st)
            _product(trag, q8, b, scale, sb, out, "f32", st)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        chain(side)
        side.synchronize()
        eq, es = _reference(x, r, w, 1e-6)
        assert (q8 == eq).all() and torch.equal(out, _expect(q8, b, scale, sb, torch.float32))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            chain(torch.cuda.current_stream())
        for k in range(4):
            x.copy_(torch.randn((m, dim), generator=g, device="cuda"))
            out.fill_(float("nan"))
            q8.fill_(99)
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            chain(torch.cuda.current_stream())
            torch.cuda.synchronize()
            assert torch.equal(got, out), k
            eq, _ = _reference(x, r, w, 1e-6)
            assert (q8 == eq).all() and torch.equal(out, _expect(q8, b, scale, sb, torch.float32))


def test_host_memory_is_refused(trag):
    torch = _torch()
    x = np.zeros((2, 64), dtype=np.float32)
    d = torch.zeros((2, 64), device="cuda")
    q8 = torch.zeros((2, 64), dtype=torch.int8, device="cuda")
    sc = torch.zeros(2, device="cuda")
    with pytest.raises(trag.TragError, match="not device memory"):
        trag.quantize_q8_device(x.ctypes.data, 64, 0, 2, 64, q8.data_ptr(), 64, sc.data_ptr())
    with pytest.raises(trag.TragError, match="not device memory"):
        trag.matmul_q8_device(q8.data_ptr(), 64, 0, x.ctypes.data, 64, 0, 2, 2, 64, 0, d.data_ptr(), 64)
    torch.cuda.synchronize()


def test_store_rows_as_8_bits(trag):
    """trag_store_quantize_device writes what quantize_q8_device writes for the rows of the store, small
    inserts included, on any stream; then the product against them is the scores' 8-bit form."""
    torch = _torch()
    d = 200
    rng = np.random.default_rng(3)
    rows = rng.standard_normal((5000, d)).astype(np.float32)
    store = trag.VectorStore(trag.VectorStoreConfig(dimension=d, metric=trag.DistanceMetric.DotProduct))
    store.insert_rows(rows[:4900])
    for i in range(4900, 5000):                      # (deferred small inserts)
        store.insert_rows(rows[i:i + 1])
    side = torch.cuda.Stream()
    for row0, n, st in ((0, 5000, None), (4890, 110, side), (17, 1, None), (5000, 0, None)):
        q8 = torch.full((max(n, 1), d + 8), FILL, dtype=torch.int8, device="cuda")
        scale = torch.full((max(n, 1),), float(FILL), device="cuda")
        torch.cuda.synchronize()
        store.quantize_device(row0, n, q8.data_ptr(), d + 8, scale.data_ptr(), 0 if st is None else st.cuda_stream)
        torch.cuda.synchronize()
        if n:
            x = torch.from_numpy(rows[row0:row0 + n]).cuda()
            _check_rows(x, None, None, 0.0, q8[:, :d], scale, norm=False)
        assert (q8[:, d:] == FILL).all()
    # a row that is replaced while its quantisation still waits on a busy stream: the call has the row it was given
    busy = torch.randn((8192, 8192), device="cuda")
    q8 = torch.empty((5000, d), dtype=torch.int8, device="cuda")
    scale = torch.empty(5000, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(10):
            busy @ busy
    store.quantize_device(0, 5000, q8.data_ptr(), d, scale.data_ptr(), side.cuda_stream)
    trag._abi.check(trag.lib().trag_store_overwrite(store.handle, 17, (100 * rows[17]).ctypes.data_as(trag._abi._fp), d))
    torch.cuda.synchronize()
    _check_rows(torch.from_numpy(rows).cuda(), None, None, 0.0, q8, scale, norm=False)
    trag._abi.check(trag.lib().trag_store_overwrite(store.handle, 17, rows[17].ctypes.data_as(trag._abi._fp), d))
    with pytest.raises(trag.TragError, match="out of bounds"):
        store.quantize_device(4999, 2, q8.data_ptr(), d, scale.data_ptr())
    with pytest.raises(trag.TragError, match="stride"):
        store.quantize_device(0, 1, q8.data_ptr(), d - 1, scale.data_ptr())
    with pytest.raises(trag.TragError, match="not device memory"):
        store.quantize_device(0, 1, rows.ctypes.data, d, scale.data_ptr())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(trag.TragError, match="capture"):
            store.quantize_device(0, 1, q8.data_ptr(), d, scale.data_ptr(), torch.cuda.current_stream().cuda_stream)
    store.close()
