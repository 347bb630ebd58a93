"""Layer normalisation on device tensors against 64 bits, with bounds derived from the roundings made."""
import pytest
import torch

import transformer_reference as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


def _rows(t, rows, cols, seed=0, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, dtype=torch.float64) * (0.5 + torch.rand(rows, 1, generator=g, dtype=torch.float64))
    return (x + mean).to(t).cuda()


def _weights(t, cols, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.2 * torch.randn(cols, generator=g)).to(t).cuda(), (0.2 * torch.randn(cols, generator=g)).to(t).cuda()


# the edges of every variant: one column, a part of a 16-byte access, a full group of 8 / 32 / 128 / 512 threads with
# 16-byte accesses and one more, and rows wider than a block holds
WIDTHS = [1, 2, 7, 8, 64, 65, 96, 256, 257, 768, 1024, 1032, 2049, 4096, 4104, 8193, 16384, 16392, 20011]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_forward_and_backward(t, cols):
    from nnv_b200 import ops
    rows = 37 if cols < 4096 else 5
    x, dy = _rows(t, rows, cols), _rows(t, rows, cols, 2, 0.0)
    s, o = _weights(t, cols)
    y, mean, rstd = ops.layer_norm(x, s, o, 1e-5, return_stats=True)
    want, m, r, tol = R.layer_norm(x, s, o, 1e-5, t)
    R.check("y", y, want, tol)
    assert mean.dtype == rstd.dtype == (torch.float64 if t is torch.float64 else torch.float32)
    assert torch.equal(ops.layer_norm(x, s, o, 1e-5), y)
    got = ops.layer_norm_backward(dy, x, s, mean, rstd)
    wants, tols = R.layer_norm_backward(dy, x, s, 1e-5, t)
    for name, a, b, c in zip(("dx", "dscale", "doffset"), got, wants, tols):
        R.check(name, a, b, c)
    again = ops.layer_norm_backward(dy, x, s, mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip(got, again))          # a fixed order of additions


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 768), (5000, 24), (4099, 136), (2500, 260), (1201, 1544)])
def test_many_rows(t, rows, cols):
    from nnv_b200 import ops
    x, dy = _rows(t, rows, cols), _rows(t, rows, cols, 2, 0.0)
    s, o = _weights(t, cols)
    y, mean, rstd = ops.layer_norm(x, s, o, return_stats=True)
    want, _, _, tol = R.layer_norm(x, s, o, 1e-5, t)
    R.check("y", y, want, tol)
    wants, tols = R.layer_norm_backward(dy, x, s, 1e-5, t)
    for name, a, b, c in zip(("dx", "dscale", "doffset"), ops.layer_norm_backward(dy, x, s, mean, rstd), wants, tols):
        R.check(name, a, b, c)


@pytest.mark.parametrize("t", TYPES)
def test_without_weights_and_batched_shapes(t):
    from nnv_b200 import ops
    x = _rows(t, 12, 40).reshape(3, 4, 40)
    y, mean, rstd = ops.layer_norm(x, None, None, 0.0, return_stats=True)
    assert y.shape == x.shape and mean.shape == (3, 4)
    want, _, _, tol = R.layer_norm(x.reshape(12, 40), None, None, 0.0, t)
    R.check("y", y.reshape(12, 40), want, tol)
    dy = _rows(t, 12, 40, 5, 0.0).reshape(3, 4, 40)
    got = ops.layer_norm_backward(dy, x, None, mean, rstd)
    wants, tols = R.layer_norm_backward(dy.reshape(12, 40), x.reshape(12, 40), None, 0.0, t)
    R.check("dx", got[0].reshape(12, 40), wants[0], tols[0])
    R.check("dscale", got[1], wants[1], tols[1])
    R.check("doffset", got[2], wants[2], tols[2])


@pytest.mark.parametrize("cut", [(0, 64), (1, 65), (8, 72), (3, 60)])
def test_strided_and_misaligned_rows(cut):
    from nnv_b200 import ops
    full = _rows(torch.bfloat16, 33, 100)
    x = full[:, cut[0]:cut[1]]
    s, o = _weights(torch.bfloat16, x.shape[1])
    y, mean, rstd = ops.layer_norm(x, s, o, return_stats=True)
    assert torch.equal(y, ops.layer_norm(x.contiguous(), s, o)) or x.shape[1] % 8
    want, _, _, tol = R.layer_norm(x, s, o, 1e-5, torch.bfloat16)
    R.check("y", y, want, tol)
    dy = _rows(torch.bfloat16, 33, 120, 3, 0.0)[:, :x.shape[1]]
    wants, tols = R.layer_norm_backward(dy, x, s, 1e-5, torch.bfloat16)
    for name, a, b, c in zip(("dx", "dscale", "doffset"), ops.layer_norm_backward(dy, x, s, mean, rstd), wants, tols):
        R.check(name, a, b, c)
    z = _rows(torch.float32, 20, 16).t()                              # columns side by side: copied
    want, _, _, tol = R.layer_norm(z, None, None, 1e-5, torch.float32)
    R.check("y", ops.layer_norm(z), want, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(20, 256), (600, 72)])
def test_rows_past_32_bits(t, rows, cols):
    """Rows so far apart that the last one begins more than 2^31 elements behind the first."""
    from nnv_b200 import ops
    x, dy = _rows(t, rows, cols), _rows(t, rows, cols, 2, 0.0)
    s, o = _weights(t, cols)
    step = (1 << 31) // (rows - 3) // 64 * 64
    far = torch.empty(step * rows, dtype=t, device="cuda")
    xf, df = (far.as_strided((rows, cols), (step, 1), i * 1024) for i in range(2))
    xf.copy_(x)
    df.copy_(dy)
    y, mean, rstd = ops.layer_norm(xf, s, o, 1e-5, return_stats=True)
    assert torch.equal(y, ops.layer_norm(x, s, o, 1e-5))
    assert all(torch.equal(a, b) for a, b in zip(ops.layer_norm_backward(df, xf, s, mean, rstd),
                                                 ops.layer_norm_backward(dy, x, s, mean, rstd)))


def test_large_mean_keeps_the_variance():
    from nnv_b200 import ops
    x = _rows(torch.float32, 9, 1000, mean=1e4)
    want, _, _, tol = R.layer_norm(x, None, None, 1e-5, torch.float32)
    y = ops.layer_norm(x)
    R.check("y", y, want, tol)
    assert abs(float(y.double().var(1, unbiased=False).mean()) - 1) < 1e-2


def test_constant_rows_and_nan_stays_in_its_row():
    from nnv_b200 import ops
    x = torch.full((4, 50), 3.0, device="cuda")
    x[1] = torch.randn(50, device="cuda")
    x[2, 7] = float("nan")
    y = ops.layer_norm(x)
    assert torch.equal(y[0], torch.zeros(50, device="cuda")) and torch.equal(y[3], y[0])
    assert y[2].isnan().all() and y[1].isfinite().all()


def test_no_rows():
    from nnv_b200 import ops
    x = torch.empty(0, 12, device="cuda")
    y, mean, rstd = ops.layer_norm(x, return_stats=True)
    dx, ds, do = ops.layer_norm_backward(torch.empty_like(x), x, None, mean, rstd)
    assert y.shape == dx.shape == (0, 12) and torch.equal(ds, torch.zeros(12, device="cuda")) and torch.equal(do, ds)


def test_gradient_against_differences():
    from nnv_b200 import ops
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 11, generator=g, dtype=torch.float64).cuda()
    dy = torch.randn(3, 11, generator=g, dtype=torch.float64).cuda()
    s, o = (torch.randn(11, generator=g, dtype=torch.float64).cuda() for _ in range(2))
    _, mean, rstd = ops.layer_norm(x, s, o, return_stats=True)
    dx, ds, do = ops.layer_norm_backward(dy, x, s, mean, rstd)
    step = 1e-5              # central differences: error step^2 / 6 * third derivative, plus 1e-16 / step
    for arg, grad in ((x, dx), (s, ds), (o, do)):
        flat, gflat = arg.view(-1), grad.reshape(-1)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + step
            up = (ops.layer_norm(x, s, o) * dy).sum().item()
            flat[i] = keep - step
            down = (ops.layer_norm(x, s, o) * dy).sum().item()
            flat[i] = keep
            assert abs((up - down) / (2 * step) - gflat[i].item()) < 1e-7


def test_on_another_stream_and_captured():
    from nnv_b200 import ops
    x, dy = _rows(torch.bfloat16, 300, 512), _rows(torch.bfloat16, 300, 512, 2)
    s, o = _weights(torch.bfloat16, 512)
    y, mean, rstd = ops.layer_norm(x, s, o, return_stats=True)
    ref = ops.layer_norm_backward(dy, x, s, mean, rstd)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y2 = ops.layer_norm(x, s, o)
    side.synchronize()
    assert torch.equal(y, y2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got_y, m, r = ops.layer_norm(x, s, o, return_stats=True)
        got = ops.layer_norm_backward(dy, x, s, m, r)
    for turn in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got_y, y) and all(torch.equal(a, b) for a, b in zip(got, ref))
