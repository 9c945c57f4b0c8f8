"""The arithmetic that the embedding gradient's kernels and their launches share, on the host:
how the rows are dealt to blocks and how far the threads step, up to the largest table."""
import os
import subprocess

from saga_b200.build import CSRC, _nvcc

PROGRAM = r'''
#include <cstdio>
#include "embedding.cu"

#define CHECK(c) do { if(!(c)) { printf("vocab %zu: %s\n", vocab, #c); return 1; } } while(0)

int main()
{
    for(size_t vocab : {(size_t)1, (size_t)148, (size_t)149, (size_t)75776, (size_t)75777, (size_t)262144,
                        (size_t)262145, (size_t)0x7ffffe00, (size_t)0x7ffffe01, B200OPT_LM_MAX}) {
        const Work w(129, vocab, 1);
        CHECK(w.blocks >= 1 && w.blocks <= vocab && w.blocks <= 0xffffffffu);
        CHECK((vocab + w.blocks - 1) / w.blocks <= (size_t)kDigits);  // rows of a block
        // every step of a loop over what is left is as long as all blocks' threads together
        CHECK((unsigned long long)order_step((uint32_t)w.blocks) == (unsigned long long)w.blocks * 1024ull);
    }
    printf("fine\n");
    return 0;
}
'''


def test_blocks_and_steps_up_to_the_largest_table(tmp_path):
    src, exe = tmp_path / "plan.cu", tmp_path / "plan"
    src.write_text(PROGRAM)
    # the program launches nothing: its device code is compiled without optimisation, to be quick
    res = subprocess.run([_nvcc(), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-Xcicc", "-O0",
                          "-Xptxas", "-O0", "-I", CSRC, str(src), "-o", str(exe)],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout == "fine\n", res.stdout
