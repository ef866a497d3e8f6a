// The lookup gradient's kernels where the sort cannot finish: one of two sorting blocks is never launched, so the other's
// bounded wait for it runs out. The workspace's keys and positions are valid places throughout.
#include "../lookatmyquant_b200/csrc/embed.cu"

// keys, pos: n entries each, twice; counts: kMaxSorters x kMaxBins; head, tail: a partial per chunk; words: two zeros.
extern "C" int gradient_with_a_block_missing(const float *dy, const long long *ids, int64_t n, int64_t rows, int d, float *dE,
                                             uint32_t *keys, uint32_t *pos, uint32_t *counts, float *head, float *tail,
                                             unsigned *words, int *status) {
    SortedParams p{};
    p.g = GradParams{ids, 1, n, rows, -1, d, d, d / 4, 1.f, 1, status};
    p.sorters = 2;
    p.passes = 1;
    p.bits = kMaxDigitBits;
    p.per_sorter = (n / 2 + kTile - 1) / kTile * kTile;
    for (int i = 0; i < 2; ++i) p.keys[i] = keys + i * n, p.pos[i] = pos + i * n;
    p.counts = counts;
    p.chunk = chunk_tokens(n);
    p.chunks = layout_of(n, d).chunks;
    p.head = head;
    p.tail = tail;
    p.barrier = words;
    p.gave_up = words + 1;
    const int slices = (p.g.packs + 31) / 32;
    gradient_sort_kernel<float, 4><<<1, kThreads>>>(dE, p);
    gradient_sum_kernel<float, 4><<<dim3((unsigned)p.chunks, slices), 32>>>(dy, dE, p, keys, pos);
    gradient_join_kernel<float, 4><<<(unsigned)(p.chunks * slices), kSumThreads>>>(dE, p, keys, slices);
    return (int)cudaDeviceSynchronize();
}
