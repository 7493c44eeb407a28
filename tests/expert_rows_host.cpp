// The loads of expert weight rows on the CPU, built with AddressSanitizer: every group of every row, by every lane
// group, from a tensor in memory of exactly its size.  A load outside it ends the program.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>

// The headers' device functions for the host, and the one builtin that a load uses.
#undef __device__
#define __device__ __attribute__((host)) __attribute__((device))
static inline uint32_t join_bytes(uint32_t hi, uint32_t lo, uint32_t n) {
    return (uint32_t)((((uint64_t)hi << 32) | lo) >> (8 * (n & 3)));
}
#define __builtin_amdgcn_alignbyte join_bytes
#include "moe_formats.h"

using namespace exq;

template <class F>
static void read_all(const char *name, int unit, int experts, int rows, int n) {
    const int nblk = n / unit;
    const size_t row_bytes = (size_t)nblk * F::kBytes, size = row_bytes * rows * experts;
    uint8_t *t = (uint8_t *)malloc(size);
    memset(t, 1, size);
    printf("%s: %d experts of %d rows of %d\n", name, experts, rows, n);
    fflush(stdout);
    unsigned sum = 0;
    for (int r = 0; r < rows * experts; ++r)
        for (int u = 0; u < moe_groups(n); ++u)
            for (int g = 0; g < 4; ++g) {
                typename F::W w;
                F::load_w(w, t + r * row_bytes, u, nblk, g);
                unsigned char b[sizeof(w)];
                memcpy(b, &w, sizeof(w));
                for (unsigned char c : b) sum += c;
            }
    printf("%u\n", sum);
    free(t);
}

int main() {
    const int shapes[][2] = {{1, 1}, {5, 17}, {2, 3}, {4, 4}};
    for (const auto &s : shapes) {
        for (int n : {256, 512, 768}) {
            read_all<MoeQ4K>("Q4_K", 256, s[0], s[1], n);
            read_all<MoeQ5K>("Q5_K", 256, s[0], s[1], n);
            read_all<MoeQ6K>("Q6_K", 256, s[0], s[1], n);
        }
        for (int n : {32, 96, 256, 608}) {
            read_all<MoeQ80>("Q8_0", 32, s[0], s[1], n);
            read_all<MoeQ40>("Q4_0", 32, s[0], s[1], n);
            read_all<MoeQ50>("Q5_0", 32, s[0], s[1], n);
        }
    }
    puts("all in bounds");
    return 0;
}
