"""GPU tests of the gated feed-forward block's stores where one tile mixes TMA stores with plain ones: a
tile's last, narrower group of columns, and outputs of which only some have addresses that TMA can take.
The projections have to be the same bits in every run, and the bits that plain stores alone write: the tile
widths, and so the order of every sum, do not depend on where the outputs lie."""
import pytest
import torch

import xspmm_b200 as xs

pytestmark = pytest.mark.gpu

f16, bf16 = torch.float16, torch.bfloat16
NAMES = ("y", "gate", "up")


def problem(rows, K, F, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [(torch.randn(r, K, generator=g, device="cuda") * s).to(dtype)
            for r, s in ((rows, 1.0), (F, 1.5 * K ** -0.5), (F, 1.5 * K ** -0.5))]


def placed(rows, cols, dtype, start):
    """A contiguous rows x cols tensor that begins `start` elements past an aligned address."""
    return torch.full((rows * cols + 16,), 7.0, dtype=dtype, device="cuda")[start:start + rows * cols].view(rows, cols)


def forward(executor, operands, starts):
    x, wg, wu = operands
    out = [placed(x.shape[0], wg.shape[0], x.dtype, s) for s in starts]
    xs.gated_ffn(executor, x, wg, wu, out[0], "silu", out[1], out[2])
    return out


# narrower last groups (tiles of 80, 112, 120 columns), and whole ones
SIZES = [(64, 4096, 11008), (512, 4096, 11008), (30000, 128, 120), (4000, 256, 80), (512, 1024, 2816),
         (2048, 1024, 4096), (20000, 64, 128)]


@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("rows,K,F", SIZES)
def test_kept_projections_repeat_and_equal_plain_stores(executor, rows, K, F, dtype):
    operands = problem(rows, K, F, dtype)
    plain = forward(executor, operands, (1, 1, 1))
    for starts in [(0, 0, 0)] * 8 + [(0, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)] * 3:
        for a, b, name in zip(forward(executor, operands, starts), plain, NAMES):
            assert torch.equal(a, b), (name, starts)


@pytest.mark.parametrize("rows,K,F", [(700, 360, 120), (5000, 200, 264), (300, 4096, 80)])
def test_gradients_repeat_and_equal_plain_stores(executor, rows, K, F):
    """dx and the weights' gradients, of widths that end in narrower groups."""
    x, wg, wu = problem(rows, K, F, bf16)
    _, gate, up = forward(executor, (x, wg, wu), (0, 0, 0))
    dy = problem(rows, F, 1, bf16, seed=3)[0]

    def backward(starts):
        dx, dwg, dwu = (placed(r, K, bf16, s) for r, s in zip((rows, F, F), starts))
        xs.gated_ffn_backward(executor, dy, x, wg, wu, gate, up, dx, dwg, dwu)
        return dx, dwg, dwu

    plain = backward((1, 1, 1))
    for starts in [(0, 0, 0)] * 8 + [(0, 1, 0), (1, 0, 1)] * 3:
        for a, b, name in zip(backward(starts), plain, ("dx", "dw_gate", "dw_up")):
            assert torch.equal(a, b), (name, starts)
