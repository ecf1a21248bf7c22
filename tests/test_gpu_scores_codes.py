"""What quantize_rows' codes and scales are by definition, whichever way the scale is rounded."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_by_definition(dtype):
    """The scale is the fp32 product with 1 / 127 and lies within two units of the quotient; a code is nearest to x / scale but
    for the fp32 quotient's own rounding, 127 * 2^-24; torch's expression on the GPU gives the same."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import octex_amd as O

    x = torch.randn((3000, 512), generator=torch.Generator().manual_seed(4)).to(TYPES[dtype])
    codes, scales = O.quantize_rows(x.cuda())
    top = x.float().abs().amax(1).numpy()
    product, quotient = top * (np.float32(1) / np.float32(127)), top / np.float32(127)
    assert (product != quotient).sum() > 50, "rows on which the two differ"
    assert np.array_equal(scales.cpu().numpy(), product)
    assert (np.abs(product.astype(np.float64) - top.astype(np.float64) / 127) <= 2 * np.spacing(quotient)).all()
    exact = x.double() / scales.cpu().double()[:, None]
    assert ((exact - codes.cpu().double()).abs() <= 0.5 + 127 * 2.0**-24).all()
    assert (codes.cpu().abs().amax(1) == 127).all()
    xg = x.cuda().float()
    s = xg.abs().amax(1) / 127
    assert torch.equal(s, scales) and torch.equal(torch.round(xg / s[:, None]).to(torch.int8), codes)
