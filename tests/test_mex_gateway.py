"""The MEX gateway called through stand-ins for MATLAB's functions: what it refuses (no GPU: refused before a context is
made), and networks with layer normalisation and attention evaluated through it."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

from nnv_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Gateway:
    def __init__(self, lib):
        self.lib = lib
        for f in ("fake_doubles", "fake_text", "fake_structs"):
            getattr(lib, f).restype = C.c_void_p
        lib.fake_call.restype = C.c_char_p

    def value(self, x):
        if isinstance(x, str):
            return self.lib.fake_text(x.encode())
        if isinstance(x, list) and isinstance(x[0], dict):      # a struct array
            s = self.lib.fake_structs(C.c_size_t(len(x)))
            for i, fields in enumerate(x):
                for k, v in fields.items():
                    self.lib.mxSetField(C.c_void_p(s), C.c_size_t(i), k.encode(), C.c_void_p(self.value(v)))
            return s
        a = np.asarray(x)
        shape = a.shape if a.ndim >= 2 else (1, a.size)
        flat = np.ascontiguousarray(np.real(a).astype(np.float64).ravel(order="F"))
        return self.lib.fake_doubles(len(shape), (C.c_size_t * len(shape))(*shape), flat.ctypes.data_as(C.c_void_p),
                                     int(np.iscomplexobj(a)))

    def __call__(self, *args):
        """The result's numbers as a flat array; RuntimeError with the gateway's message."""
        vals = (C.c_void_p * len(args))(*[self.value(a) for a in args])
        out = C.c_void_p()
        err = self.lib.fake_call(len(args), vals, C.byref(out)).decode()
        if err:
            raise RuntimeError(err)
        if not out.value:
            return None
        self.lib.mxGetNumberOfElements.restype = C.c_size_t
        self.lib.mxGetDoubles.restype = C.POINTER(C.c_double)
        n = self.lib.mxGetNumberOfElements(out)
        return np.ctypeslib.as_array(self.lib.mxGetDoubles(out), (n,)).copy()


@pytest.fixture(scope="module")
def gateway(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    _lib.load()
    so = str(tmp_path_factory.mktemp("mex") / "gateway.so")
    pkg = os.path.join(ROOT, "nnv_b200")
    subprocess.run([gxx, "-std=c++17", "-O1", "-fPIC", "-shared", "-I", os.path.join(ROOT, "include", "mex_stub"),
                    os.path.join(pkg, "csrc", "nnvb200_mex.cpp"), os.path.join(ROOT, "tests", "mex_runtime.cpp"),
                    "-L", pkg, "-l:libnnvb200.so", "-Wl,-rpath," + pkg, "-o", so], check=True)
    return Gateway(C.CDLL(so))


def _attention(heads=4, keys=(8, 2, 5), values=(8, 2, 5), **more):
    return {"Type": "attention", "NumHeads": heads, "Keys": np.ones(keys), "Values": np.ones(values), **more}


@pytest.mark.parametrize("layer,word", [
    (_attention(values=(2, 8, 5)), "one size"), (_attention(values=(8, 2, 4)), "one size"), (_attention(keys=(8, 2, 5, 2), values=(8, 2, 5, 2)), "one size"),
    (_attention(heads=2.5), "whole"), (_attention(heads=-2), "whole"), (_attention(heads=float("nan")), "whole"),
    (_attention(heads=1e12), "whole"),
    ({"Type": "attention", "NumHeads": 2, "Keys": np.ones((4, 2, 3)) * 1j, "Values": np.ones((4, 2, 3))}, "one size"),
    ({"Type": "attention", "NumHeads": 2, "Keys": np.ones((4, 2, 3))}, "one size"),
    ({"Type": "layernorm", "NumChannels": 3.5}, "whole"), ({"Type": "layernorm", "NumChannels": 0}, "whole"),
    ({"Type": "layernorm"}, "NumChannels"), ({"Type": "layernorm", "NumChannels": 4, "Scale": np.ones(3)}, "size"),
    ({"Type": "layernorm", "NumChannels": 4, "Offset": np.ones(5)}, "size")])
def test_layers_that_the_gateway_refuses(gateway, layer, word):
    with pytest.raises(RuntimeError, match=word):
        gateway("create_net", [layer], [32, 3, 1])


@pytest.mark.gpu
def test_layers_evaluated_through_the_gateway(gateway):
    from nnv_b200 import nn
    rng = np.random.default_rng(0)
    c, heads, hk, S, T, n = 8, 4, 2, 33, 3, 5
    D = c * heads
    s, o = rng.standard_normal(D), rng.standard_normal(D)
    K, V = rng.standard_normal((c, hk, S)), rng.standard_normal((c, hk, S))
    X = rng.standard_normal((D * T, n))
    h = gateway("create_net", [{"Type": "layernorm", "NumChannels": D, "Scale": s, "Offset": o, "Epsilon": 1e-6},
                               {"Type": "attention", "NumHeads": heads, "Keys": K, "Values": V, "AttentionScale": 0.3},
                               {"Type": "layernorm", "NumChannels": D}], [D, T, 1])
    got = gateway("evaluate", h, X).reshape(D * T, n, order="F")
    net = nn.NN([nn.LayerNormalizationLayer(D, s, o, 1e-6), nn.AttentionLayer(heads, K, V, Scale=0.3), nn.LayerNormalizationLayer(D)])
    want = net.evaluate([x.reshape(D, T, 1, order="F") for x in X.T])
    for i in range(n):
        assert np.array_equal(got[:, i], np.asarray(want[i]).ravel(order="F"))
    for bad in (X[:-1], X[:, :1].reshape(D, T, order="F"), X[:1]):      # other sizes would read behind the array
        with pytest.raises(RuntimeError, match="rows"):
            gateway("evaluate", h, bad)
    with pytest.raises(RuntimeError, match="heads"):                   # the layer does not fit the input
        gateway("create_net", [_attention(heads=6)], [D, T, 1])
    gateway("destroy", h)
