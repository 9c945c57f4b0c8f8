"""Which tiles the vocabulary loss's products are computed in, on the host."""
import os
import subprocess

from saga_b200.build import CSRC, _nvcc

PROGRAM = r'''
#include <cstdio>
#include "tc_gemm.cuh"

using namespace b200;

int main()
{
    // rows, columns, k, whether tiles of 512 columns are the faster ones on 148 SMs (both measured)
    const struct { long long m, n, k; bool wide; } cases[] = {
        {16384, 4096, 512, false}, {16384, 4096, 1024, false}, {16384, 4096, 2048, true}, {16384, 4096, 8192, true},
        {50021, 2048, 64, false}, {50021, 2048, 512, false}, {50021, 2048, 768, false}, {50021, 2048, 2048, true},
        {48640, 2048, 512, false}, {15360, 4096, 2048, false}, {15360, 4096, 8192, true}, {32000, 1024, 4096, false},
    };
    int wrong = 0;
    for(auto &c : cases)
        if(tc_wide(c.m, c.n, c.k, 148) != c.wide) {
            printf("%lld x %lld x %lld\n", c.m, c.n, c.k);
            wrong++;
        }
    // a GPU of one SM pair or less divides by nothing
    tc_wide(1, 8, 1 << 20, 1);
    return wrong;
}
'''


def test_wide_tiles_where_they_are_faster(tmp_path):
    src, exe = tmp_path / "tiles.cu", tmp_path / "tiles"
    src.write_text(PROGRAM)
    res = subprocess.run([_nvcc(), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, str(src),
                          "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout
