// What the calls on a cache in pages have in common: pages of a length, and the ring of free pages with its {first, count}.
#pragma once

#include "common.h"

__device__ __forceinline__ int plan_pages(int n, int shift) { return n > 0 ? ((n - 1) >> shift) + 1 : 0; }
__device__ __forceinline__ int plan_wrap(uint32_t i, int pool) { return i >= (uint32_t)pool ? (int)(i - pool) : (int)i; }   // i < 2 * pool

struct plan_state {
    int head, count, tail;                       // (a state that no ring can have is an empty ring)
    __device__ __forceinline__ plan_state(const int32_t *p, int pool) {
        head = p[0];
        count = p[1];
        if (head < 0 || head >= pool || count < 0 || count > pool) head = count = 0;
        tail = plan_wrap((uint32_t)head + count, pool);
    }
};
