"""The shared memory of an eviction's selecting CTAs, on the CPU: every key that
a thread reads lies inside what the launcher asks for, at every width of table
and every length of sequence. A thread reads whole runs of keys, so the
arithmetic of evict_keys.h is walked as the kernel walks it."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

PROBE = r"""
#include "evict_keys.h"
#include <cstdio>
#include <cstdlib>
using namespace fer::evict;

// One behind the last word that a CTA of `each` slots touches.
static int touched(int each, int threads) {
    const int run = slots_of_thread(each, threads);
    if (run * threads < each || run % 4 || run > kMostKeys) return 1 << 30;   // every slot has a thread
    int most = word_of(each - 1) + 1;                                         // keys written
    for (int t = 0; t < threads && run * t < each; ++t)
        for (int i = 0; i < run; i += 4)
            if (word_of(run * t + i) + 4 > most) most = word_of(run * t + i) + 4;   // 16 bytes read
    return most;
}

int main(int, char** argv) {
    const int threads = atoi(argv[1]), most = kMostKeys * threads;
    int over = 0, over_exact = 0, beyond = 0;
    for (int width = 128; width <= most; width += 128) {
        int reach = 0;
        for (int each = 128; each <= width; each += 128) {   // what a shorter sequence makes of it
            const int n = touched(each, threads);
            if (n > reach) reach = n;
        }
        over += reach > words_of_cta(width, threads);
        over_exact += reach > width / 32 * 36;               // room for the keys alone
        beyond += words_of_cta(width, threads) > words_of_cta(most, threads);
    }
    // a CTA of any cluster has no more slots than its part of the widest table
    int wide = 0;
    for (int ctas = 1; ctas <= 8; ctas *= 2)
        for (int n = 1; n <= ctas * most; n += 61) {
            const int each = slots_of_cta(n, ctas);
            wide += each % 128 != 0 || each > most || static_cast<long long>(each) * ctas < n;
        }
    printf("%d %d %d %d %d\n", over, over_exact, beyond, wide, words_of_cta(most, threads));
}
"""


@pytest.mark.parametrize("threads,narrow", [(1024, 94), (256, 22)])
def test_every_key_lies_in_the_shared_memory_asked_for(tmp_path, threads, narrow):
    (tmp_path / "probe.cpp").write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT}/fercuda_b200/csrc/kernels", str(tmp_path / "probe.cpp"), "-o",
                    str(tmp_path / "probe")], check=True)
    out = subprocess.run([str(tmp_path / "probe"), str(threads)], capture_output=True, text=True, check=True).stdout
    over, over_exact, beyond, wide, words = map(int, out.split())
    assert (over, beyond, wide) == (0, 0, 0)
    assert over_exact == narrow      # widths at which room for the keys alone is passed: the walk sees such a fault
    assert words <= threads * 36     # 4 words of padding behind every 32 keys
