// paged.h -- a KV cache in pages that several requests share: the handle behind mg_paged and the launchers of its kernels.
#pragma once
#include <hip/hip_runtime.h>

#include "paged_rules.h"

namespace mg {

struct PagedTables {
    const int *newLens, *lens, *ringState;
    int *lensOut, *table, *ring, *ringStateOut, *rowStart, *slots, *positions, *counts;
    int nReqs, rows, nPages, pageShift, width, maxLen;
};
hipError_t launch_paged_tables(const PagedTables& p, hipStream_t s);

struct PagedStore {
    const float *q, *k, *v, *cosTab, *sinTab;
    float* qOut;
    void *K, *V;
    const int *slots, *positions;
    int ldq, ldk, ldv, ldqOut, rows, tableRows, nHeads, nKVHeads, headDim, kvHalf, nSlots;
};
hipError_t launch_paged_store(const PagedStore& p, hipStream_t s);

// What a step's attention calls share, copied when the plan is made: the requests' rows, lengths and prefixes.
struct PagedPlan {
    const int *rowStart, *lens, *prefixLens;      // the caller's
    int* reqs;                                    // the handle's: 4 ints a request {first row, rows, length, prefix}
    int nReqs, rows, window, maxLen;
};
hipError_t launch_paged_plan(const PagedPlan& p, hipStream_t s);

struct PagedAttention {
    const float *q, *slopes;
    const void *K, *V;
    const int *table, *reqs;
    float* out;
    float scale, softcap;
    int ldq, ldo, rows, nReqs, window;
    PagedGeo g;
};
hipError_t launch_paged_attention(const PagedAttention& p, hipStream_t s);

}  // namespace mg
