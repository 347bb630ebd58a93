"""Layer normalisation's backward of more than one cluster's rows in double and fp16: several groups a block, partial rows,
a second kernel that adds them."""
import pytest
import torch

import transformer_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float64, torch.float16])
@pytest.mark.parametrize("rows,cols", [(30000, 24), (4099, 136), (2500, 260), (1201, 1544), (200, 3001)])
def test_many_rows(t, rows, cols):
    from nnv_b200 import ops
    g = torch.Generator().manual_seed(rows)

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)
    x, dy = (r(rows, cols) + 0.3).to(t).cuda(), r(rows, cols).to(t).cuda()
    s, o = (1 + 0.2 * r(cols)).to(t).cuda(), r(cols).to(t).cuda()
    y, mean, rstd = ops.layer_norm(x, s, o, return_stats=True)
    want, _, _, tol = R.layer_norm(x, s, o, 1e-5, t)
    R.check("y", y, want, tol)
    wants, tols = R.layer_norm_backward(dy, x, s, 1e-5, t)
    for name, a, b, c in zip(("dx", "dscale", "doffset"), ops.layer_norm_backward(dy, x, s, mean, rstd), wants, tols):
        R.check(name, a, b, c)
