"""The multiply-high that stands for a division by the block size (gvirt_amd/csrc/block_magic.h), compiled for the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "block_magic.h"
int main()
{
    for (uint32_t bs = 1; bs <= 4096; bs = bs < 300 ? bs + 1 : bs * 3 / 2) {
        for (uint64_t positions : std::initializer_list<uint64_t>{bs, (5000 / bs + 1) * bs, ((1ull << 32) - 1) / bs, 1ull << 31}) {
            const uint32_t m = xlite::block_magic(bs, positions);
            if ((m == 0) != (bs == 1 || positions * bs >= (1ull << 32))) {
                printf("block size %u, %llu positions: magic %u\n", bs, (unsigned long long)positions, m);
                return 1;
            }
            auto off = [&](uint64_t p) { return m != 0 && p < positions && static_cast<uint32_t>(p * m >> 32) != p / bs; };
            for (uint64_t p = 0; p < positions; p += 1 + p / 64) {
                // the positions around a block's border are where a quotient goes wrong
                for (uint64_t q : std::initializer_list<uint64_t>{p, p / bs * bs, p / bs * bs + bs - 1, positions - 1 - p}) {
                    if (off(q)) {
                        printf("block size %u, position %llu\n", bs, (unsigned long long)q);
                        return 1;
                    }
                }
            }
        }
    }
    return 0;
}
"""


def test_the_magic_divides_or_is_not_there(tmp_path):
    source = tmp_path / "magic.cpp"
    source.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "gvirt_amd", "csrc"), str(source), "-o", str(tmp_path / "magic")])
    r = subprocess.run([str(tmp_path / "magic")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
