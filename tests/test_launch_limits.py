"""Sizes whose launch would need 2^32 threads or more are refused by the library (descriptors alone: no GPU)."""
import ctypes
from concurrent.futures import ThreadPoolExecutor

from nerfhip import _lib, fp8, muon


def test_sizes_beyond_a_launch_are_refused():
    """(In a thread of its own: the last error is kept for each thread.)"""
    def run():
        L = _lib.lib()
        one = ctypes.c_void_p(1 << 20)      # (never read: the sizes are refused first)

        def said(rc, what):
            assert rc == 1001 and what in L.nerf_last_error().decode(), L.nerf_last_error()

        N = 1 << 29
        d = fp8._Fp8Linear(one, 128, 1, None, 1, 1, 1, 1, 0, 1, N, 128, one, one, None, None, one, N)
        said(L.nerf_fp8_linear(ctypes.addressof(d), None, 0, None), "too many columns")
        M = (1 << 31) - 1
        d = fp8._Fp8Linear(one, 512, M, None, 1, 1, 1, 1, 0, M, 129, 512, one, one, None, None, one, 129)
        need = L.nerf_fp8_linear_workspace(M, 129, 512, 1, 0)
        said(L.nerf_fp8_linear(ctypes.addressof(d), one, need, None), "too many tiles")
        g = (muon._Group * 32)(*[muon._Group(one, one, None, 70, 1000, (1 << 20) - 1, 0, 0)] * 32)
        o = muon._Options(0, 0, 0, 5, 0.0, 0.0, 0.0, 1e-7, -1.0, None)
        at = ctypes.addressof(g)
        said(L.nerf_muon(at, 32, ctypes.addressof(o), one, L.nerf_muon_workspace(at, 32), None), "too many tiles")

    with ThreadPoolExecutor(1) as ex:
        ex.submit(run).result()
