"""The tile loop's loads and prefetches stay inside their operands, and leave
nothing of them out: walked on the host (tests/ranges/gemm_ranges.hip)."""

import os
import subprocess

import pytest

from graspo_amd import build as B

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("ranges") / "gemm_ranges")
    flags = [f for f in B.HIP_FLAGS if f != "-fPIC"]
    subprocess.run([B._hipcc(), *flags, "--cuda-host-only",
                    os.path.join(HERE, "ranges", "gemm_ranges.hip"), "-o", out], check=True,
                   capture_output=True)
    return out


# K % 128 in 1 .. 64 above 128: the prefetch runs a whole step past K
@pytest.mark.parametrize("K", [8, 64, 72, 128, 136, 192, 200, 256, 264, 320, 328, 2880])
@pytest.mark.parametrize("outer", [1, 7, 255, 257])
def test_rows_along_k(walk, outer, K):
    """Rows without a gap, with one, and the right half of wider rows: the
    operand's memory ends with its last row's K."""
    for ld in (K, K + 8, K + 64, 2 * K):
        r = subprocess.run([walk, "along", str(outer), str(K), str(ld)], capture_output=True, text=True)
        assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("K", [0, 1, 5, 130, 135, 261, 390])
def test_a_last_chunk_along_k(walk, K):
    """The logits' gradient by the number of listed rows: whole chunks of 8 lie
    in its rows."""
    for outer in (1, 300):
        for ld in ((K + 7) // 8 * 8 + 8, 512):
            r = subprocess.run([walk, "along", str(outer), str(K), str(ld)], capture_output=True,
                               text=True)
            assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("K", [0, 1, 7, 64, 65, 129, 192, 261, 700])
@pytest.mark.parametrize("outer", [8, 64, 256, 264, 520])
def test_columns_across_k(walk, outer, K):
    for ld in (outer, outer + 8, 2 * outer):
        r = subprocess.run([walk, "across", str(outer), str(K), str(ld)], capture_output=True, text=True)
        assert r.returncode == 0, r.stdout
