"""Programs with the transformer operators through the lowering, interpreted on the CPU (results and workspaces poisoned
before an operand is read), against the oracle."""
import numpy as np
import pytest

import operator_programs
from test_plan_interp_cpu import _Both, _interpret_or_refused


@pytest.mark.parametrize("chunk", range(2))
def test_random_operator_programs(hostcheck, tmp_path, chunk):
    refused = ran = 0
    for seed in range(chunk * 40, chunk * 40 + 40):
        dev = _Both()
        kept = operator_programs.build(seed)(dev)
        tol = operator_programs.tolerance(kept)
        if tol is None:
            continue
        for flags in (0, 1, 2):
            got = _interpret_or_refused(hostcheck, tmp_path, dev.blobs[-1], flags, f"op{seed}_{flags}")
            if got is None:
                refused += 1
                break
            ran += 1
            for k, v in kept.items():
                dims, data = got[k]
                assert dims == list(v.dim)
                assert np.abs(data - np.asarray(v.data, np.float64)).max(initial=0) <= tol[k], (seed, flags, k)
    assert ran >= 60 and refused <= 20, (ran, refused)
