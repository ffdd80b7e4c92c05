"""CPU checks of what the header promises about the sequence operators' queries."""
from ctypes import byref

import numpy as np


def test_scan_workspace_does_not_depend_on_the_element_type():
    """The query's answer follows from the sizes it names, so a buffer of that size serves every type."""
    from sed_amd import _lib as L
    rng = np.random.default_rng(0)
    for k in range(2000):
        B, n, D = (int(round(np.exp(rng.uniform(0, np.log(most))))) for most in (512, 40000, 2048))
        N = int(rng.choice([1, 3, 8, 16, 16, 32]))
        for ragged in (None, 16):
            for back in (0, 1):
                asked = {t: L.lib.sed_gated_scan_workspace(byref(L.ScanArgs(B=B, L=n, D=D, N=N, G=1, dtype=t, frames=ragged)), back) for t in (L.F32, L.BF16, L.F16, 0)}
                assert len(set(asked.values())) == 1, (B, n, D, N, ragged, back, asked)
    # a shape whose gradient takes more chunks in 16 bits than in 32
    asked = [L.lib.sed_gated_scan_workspace(byref(L.ScanArgs(B=1, L=16385, D=384, N=16, G=1, dtype=t)), 1) for t in (L.F32, L.BF16)]
    assert asked[0] == asked[1] >= 29195520
