"""AdapterLinear at the ends of the number range: results that the type holds are not lost on the
way to them, whatever the number of rows."""
import pytest
import torch

rv = pytest.importorskip("ruvector_amd")
from heads_ref import F32, TINY, assert_within  # noqa: E402
from test_gpu_adapters import run  # noqa: E402
from heads_ref import to_buffer  # noqa: E402

pytestmark = pytest.mark.gpu


def spread(g, *shape):
    """Values of either sign with magnitudes in [1/2, 1)."""
    v = torch.rand(*shape, generator=g) * 0.5 + 0.5
    return torch.where(torch.rand(*shape, generator=g) < 0.5, -v, v)


@pytest.mark.parametrize("n", [1, 64, 65, 200, 700])
@pytest.mark.parametrize("xe,we", [(-61, -61), (-20, -102), (-102, -20), (-58, -64), (60, 60), (100, -126), (-126, 100)])
@pytest.mark.parametrize("inp,out", [(100, 70), (4100, 40)])
def test_f32_products_near_the_ends(n, xe, we, inp, out):
    """max |x| max |W| from 2^-122 to 2^120: sums of such products are ordinary numbers."""
    g = torch.Generator().manual_seed(n * 1000 + xe + inp)
    x, w = spread(g, n, inp) * 2.0 ** xe, spread(g, out, inp) * 2.0 ** we
    layer = rv.AdapterLinear(inp, out, to_buffer(w), max_adapters=0)
    got = run(layer, x, None)
    x, w = x.double(), w.double()
    want, size = x @ w.T, x.abs() @ w.abs().T
    # sums of `in` products in 32 bits (no partial sum needs a step below the type's smallest), and each
    # product within 3 2^-22 of the two rows' largest values
    most = x.abs().amax(1)[:, None] * w.abs().amax(1)
    assert_within(got, want, size * F32 * (inp + 4) + inp * (3 * 2.0 ** -22 * most + TINY["f32"]))
