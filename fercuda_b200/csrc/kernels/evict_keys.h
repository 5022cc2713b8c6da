// Where the selecting CTAs of an eviction hold their keys in shared memory.
// Plain arithmetic, shared by the kernel, its launcher and a test on the host.
#pragma once

#ifdef __CUDACC__
#define FER_EVICT_FN __host__ __device__ constexpr
#else
#define FER_EVICT_FN constexpr
#endif

namespace fer::evict {

constexpr int kMostKeys = 32;   // keys a thread holds at most

// Slots of each of `ctas` CTAs that share a head of n.
FER_EVICT_FN int slots_of_cta(int n, int ctas) { return ((n - 1) / ctas + 1 + 127) & ~127; }
// Slots of a thread: whole 16-byte pieces.
FER_EVICT_FN int slots_of_thread(int each, int threads) { return ((each - 1) / threads + 4) & ~3; }
// Word of the key of a CTA's slot j: 4 words of padding behind every 32 keys, so
// that threads read runs of keys in 16-byte pieces without bank conflicts.
FER_EVICT_FN int word_of(int j) { return j + j / 32 * 4; }
// Words that a CTA of `each` slots reads and writes. Threads walk whole runs,
// and a run of 12, 20, 24 or 28 slots does not divide `each`, so the last one
// may end behind it. Words never become fewer as `each` grows: a CTA's keys
// fit what is asked for the widest sequence.
FER_EVICT_FN int words_of_cta(int each, int threads) {
    const int run = slots_of_thread(each, threads);
    return word_of((each + run - 1) / run * run - 1) + 1;
}

}  // namespace fer::evict
