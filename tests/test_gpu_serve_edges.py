"""The serving operators on calls at the edge of what the header allows (include/imi_cuda.h), each way of the attention among
them, against their restatement in 64 bits (tests/serve_plain.py)."""
import pytest

from test_gpu_serve_ops import attn_case, run_attn

pytestmark = pytest.mark.gpu

# rows of 2 kv heads with 4 query heads each: few query rows (registers), one tile of them, several tiles (tensor cores)
ROWS = [3, 9, 40, 130]


def lengths(rows, unused=()):
    return [-1 if i in unused else (7 * i) % 50 for i in range(rows)]


# ------------------------------------------------------------------------------------------------------- the scale
@pytest.mark.parametrize("dt,d", [("f16", 64), ("bf16", 64), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("scale", [0.0, -0.25])
def test_attn_scale_zero_and_negative(rows, dt, d, scale):
    """Scale 0: equal weights, with a ragged end of the prompt, a window and a missing page as well; a negative scale turns the
    scores around."""
    c = attn_case(rows, 2, 4, d, dt, 16, 1400, lengths(rows), seed=rows)
    run_attn(c, scale=scale)
    run_attn(c, scale=scale, window=1000)
    c["prefix"][33] = -1
    run_attn(c, scale=scale, status_want=1)
    run_attn(attn_case(rows, 2, 4, d, dt, 16, 1408, lengths(rows), seed=rows), scale=scale)
