"""GPU: products of 8-bit rows whose offsets inside a tile come close to 32 bits."""
import pytest

from test_gpu_q8 import _expect, _int8, _product, _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,far", [(272, 2 ** 24 - 16), (300, 2 ** 24 - 16), (300, 2 ** 24 - 1)])
def test_rows_just_below_2_24_bytes_apart(trag, dim, far):
    """The largest strides that go through tiles: from row 128 of a tile of 256 on, a row's offset from the tile's first passes
    2^31, at row 255 it is 2^32 less 2^24 and a little. Sizes at which the choice is that tile (272: transfers straight into LDS,
    300: through registers), the far rows on either side."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(dim)
    few, many = 300, 30_000
    wide = torch.empty((few - 1) * far + dim, dtype=torch.int8, device="cuda")
    rows = torch.as_strided(wide, (few, dim), (far, 1))
    rows.copy_(_int8(few, dim, 0, 0, g, True))
    near = _int8(many, dim, 0, 0, g, True)
    for a, b in ((rows, near), (near, rows)):
        sa, sb = torch.rand(a.shape[0], generator=g, device="cuda"), torch.rand(b.shape[0], generator=g, device="cuda")
        out = torch.full((a.shape[0], b.shape[0]), float("nan"), device="cuda")
        _product(trag, a, b, sa, sb, out, "f32")
        assert torch.equal(out, _expect(a, b, sa, sb, torch.float32))
