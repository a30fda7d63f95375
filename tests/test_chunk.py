"""The division of paged_chunk_attn's work, under host sanitizers, and its oracle."""
import os
import shutil
import subprocess
import tempfile

import numpy as np
import pytest

from conftest import ROOT
from oracle import paged as op


def test_division_under_host_sanitizers():
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    tmp = tempfile.mkdtemp()
    try:
        exe = os.path.join(tmp, "chunk_fuzz")
        subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-Wno-unknown-pragmas",
                        "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                        "-I", os.path.join(ROOT, "varlenabsorbflashattn_amd", "csrc"),
                        os.path.join(ROOT, "tests", "host_fuzz", "chunk_fuzz.cpp"), "-o", exe],
                       check=True, capture_output=True, text=True)
        for seed in (3, 99):
            r = subprocess.run([exe, "300", str(seed)], capture_output=True, text=True, timeout=300)
            assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
            assert "0 failed checks" in r.stdout
    finally:
        shutil.rmtree(tmp, ignore_errors=True)


@pytest.mark.parametrize("window", [None, 1, 7, 100])
def test_oracle_is_masked_attention(window):
    """The oracle's chunk against a causal softmax over a whole sequence's rows."""
    rng = np.random.default_rng(4)
    H, Hk, D, page, n = 4, 2, 16, 4, 23
    k, v = rng.standard_normal((2, 8, page, Hk, D))
    table = np.array([[5, 0, 7, 2, 1, 6]])
    q = rng.standard_normal((9, H, D))
    out, mag, _ = op.chunk(q, k, v, table, [n], [1, 8], 0.3, softcap=4.0, window=window)
    rows = table[0, np.arange(n) // page], np.arange(n) % page
    for t in range(1, 8):
        p = n - 8 + t
        for h in range(H):
            z = 4.0 * np.tanh(0.3 * (k[rows][:, h // 2] @ q[t, h]) / 4.0)
            j = np.arange(n)
            hidden = (j > p) | (j <= p - window if window else False)
            e = np.where(hidden, 0.0, np.exp(z))
            assert np.allclose(out[t, h], (e / e.sum()) @ v[rows][:, h // 2])
    assert not out[0].any() and not out[8].any() and (np.abs(out) <= mag + 1e-12).all()
