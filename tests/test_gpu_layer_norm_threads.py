"""Layer normalisation called from several host threads at once: the calls keep no state that another call could meet."""
import threading

import pytest
import torch

from nnv_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("backward", [False, True])
def test_threads_with_different_row_counts(backward):
    """One width, so one kernel: calls with many rows take all the shared memory of an SM, calls with few rows little.
    The C entries are called in tight loops, which release the interpreter lock."""
    lib = _lib.load()
    cols, turns = 768, 10000
    g = torch.Generator().manual_seed(0)
    w = torch.randn(cols, generator=g).cuda()
    calls, failed = [], []
    for rows in (8, 6000, 8, 6000):
        x, dy = (torch.randn(rows, cols, generator=g).cuda() for _ in range(2))
        y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        stream = torch.cuda.Stream()
        fwd = (stream.cuda_stream, _lib.F32, rows, cols, x.data_ptr(), cols, w.data_ptr(), w.data_ptr(), 1e-5, y.data_ptr(),
               cols, mean.data_ptr(), rstd.data_ptr())
        need = lib.nnvb_layer_norm_workspace(_lib.F32, rows, cols)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        dw = torch.empty(2, cols, device="cuda")
        bwd = (stream.cuda_stream, _lib.F32, rows, cols, dy.data_ptr(), cols, x.data_ptr(), cols, w.data_ptr(),
               mean.data_ptr(), rstd.data_ptr(), y.data_ptr(), cols, dw[0].data_ptr(), dw[1].data_ptr(), ws.data_ptr(), need)
        calls.append((fwd, bwd, (x, dy, y, mean, rstd, ws, dw, stream)))
    torch.cuda.synchronize()
    for fwd, _, _ in calls:
        assert lib.nnvb_layer_norm_forward(*fwd) == 0
    torch.cuda.synchronize()
    start = threading.Barrier(len(calls))

    def run(fwd, bwd, keep):
        fn, args = (lib.nnvb_layer_norm_backward, bwd) if backward else (lib.nnvb_layer_norm_forward, fwd)
        start.wait()
        bad = sum(fn(*args) != 0 for _ in range(turns))
        if bad:
            failed.append("%d of %d calls with %d rows: %s" % (bad, turns, args[2], lib.nnvb_last_error().decode()))
    threads = [threading.Thread(target=run, args=c) for c in calls]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed, failed
