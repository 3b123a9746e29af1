"""The even shares of a request's tiles (share_begin of mi_internal.h), compiled for the host.

Share k of n covers [k total / n, (k + 1) total / n); a request of 2^26 tiles cut in
hundreds has products beyond 32 bits.
"""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "mstar_amd" / "csrc"


@pytest.fixture(scope="module")
def share(tmp_path_factory):
    text = (CSRC / "mi_internal.h").read_text()
    part = re.search(r"__host__ __device__ (inline int share_begin\(.*?\n})", text, re.S).group(1)
    tmp = tmp_path_factory.mktemp("share")
    (tmp / "share.cpp").write_text(part + '\nextern "C" int at(int k, int n, int total) { return share_begin(k, n, total); }\n')
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-ftrapv", "-o", tmp / "share.so", tmp / "share.cpp"], check=True)
    return ctypes.CDLL(str(tmp / "share.so")).at


@pytest.mark.parametrize("n", [1, 2, 3, 7, 16, 61, 255, 512, 768, 1024])
def test_shares_are_the_quotients(share, n):
    """-ftrapv ends the process on a sum or product that passes 32 bits."""
    for total in [*range(0, 40), 1000, 1023, 4097, (1 << 22) - 1, 1 << 22, (1 << 22) + 5, (1 << 26) - 1, 1 << 26, 2**31 - 1]:
        for k in {0, 1, n // 3, n // 2, n - 1, n}:
            assert share(k, n, total) == k * total // n, (k, n, total)


def test_kernels_take_their_shares_by_it():
    """No kernel forms the product of a share's index with the tiles or steps of a request."""
    for name in ("mi_decode_kernel.h", "mi_prefill_kernel.h", "mi_prefill_rs.h"):
        text = (CSRC / name).read_text()
        assert text.count("share_begin(") == 2, name
        assert not re.search(r"(kidx|un\.k)( \+ 1\))? \* (span\.total|n_kt)", text), name
