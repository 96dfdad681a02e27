"""The streaming kernels' division of their list of weight rows, compiled for the host (no GPU needed)."""
import ctypes as C
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "iree_b200", "csrc")


@pytest.fixture(scope="module")
def share(tmp_path_factory):
    folder = tmp_path_factory.mktemp("list")
    source, lib = folder / "list.cc", folder / "list.so"
    source.write_text('#include "w4a16_stream_list.h"\n'
                      'extern "C" int64_t share(int64_t total, uint32_t parts) { return b200::list_share(total, parts); }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, "-o", str(lib), str(source)], check=True)
    f = C.CDLL(str(lib)).share
    f.restype, f.argtypes = C.c_int64, [C.c_int64, C.c_uint32]
    return f


def test_every_row_is_in_a_part(share):
    """Up to 1024 experts of one row and 2^31 weight rows each: also where rows + parts - 1 passes 2^32 (771 x 5570645 = 2^32 - 1)."""
    rng = random.Random(3)
    totals = [0, 1, 147, 148, 149, 771 * 5570645, 255 * 16843009, (1 << 32) - 147, (1 << 32) - 148, 1 << 32, (1 << 32) + 1, 1024 << 31]
    totals += [rng.randrange(1 << rng.randint(1, 41)) for _ in range(2000)]
    totals += [(1 << 32) + d for d in range(-300, 300)]
    for total in totals:
        for parts in (1, 2, 20, 132, 148):
            assert share(total, parts) == -(-total // parts), (total, parts)
